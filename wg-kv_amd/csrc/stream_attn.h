// The windowed decode attention for batches of many heads (stream_attn.hip),
// as the entry point in decode_attn.hip calls it.
#pragma once

#include "wgkv_common.h"

struct StreamWindow {
  const uint16_t* q;
  int64_t q_sb, q_sh;
  const uint16_t* kc;
  const uint16_t* vc;
  int64_t num_pages;
  int page_shift;  // page_size = 16 << page_shift
  const int32_t* len;
  int64_t len_sb;
  const int32_t* bt;
  int64_t bt_sb, bt_sh;
  int cap;  // tokens a row of the table has room for
  uint16_t* out;
  int64_t out_sb, out_sh;
  int B, H, G, D, window, sinks;
  float scale_log2;
  uint32_t q_and, q_xor;
};

size_t wgkv_stream_window_bytes(int B, int H, int G, int D);
int wgkv_stream_window(const StreamWindow& w, void* scratch, hipStream_t st);
