// The 4-bit cache's number format and page layout (gfx950).
//
// A row of D values (a token's key or value of one head) is held in groups of
// 32.  A group keeps a step s and a middle m, both bf16, and a code c in
// 0..15 per value:
//   s = bf16((max - min) / 15), 0 where that is below 2^-126
//   m = bf16((max + min) / 2)
//   (both quotients rounded to fp32 first)
//   c = round((x - m) / s + 7.5) clamped to 0..15 (ties to even; 0 if s = 0)
//   a value reads as m + s * (c - 7.5)
// A group that holds a NaN or an infinity (or whose m is one) gets
// s = m = NaN: all of it reads as NaN rather than as plausible numbers.  bf16
// steps have the inputs' range (a fp16 step would overflow where bf16 keys do
// not), and the codes are chosen for the rounded s and m, so their rounding
// costs nothing but range at the ends: |error| <= s/2 plus half a bf16 step
// of m.
//
// 16 tokens form a tile of 10*D bytes; a page is page_size/16 tiles.  With
// t = token % 16 and q = t / 4:
//   keys   16-bit word (t, d/8, d%2)      codes d%8 = d%2 + {0, 2, 4, 6}
//   values 16-bit word (q, r, t%4/2, half, t%2)
//                                         codes d = (D/16)*r + 4*half + {0..3}
//   then, for both, (s, m) pairs (q, g, t%4) of group g = d/32
// (first code in the lowest bits, index lists outermost first).  So the
// matrix core's operands come out of 16-byte loads without a shuffle: for
// keys a lane's 8 consecutive d of a token, two neighbours in one dword's
// halves, and for values one d of the tokens (t, t+1), so that
// (w >> 4*i) & 0x000f000f is an operand pair in both.  All of it is byte
// addressed per token: writing a token never reads or rewrites another's.
#pragma once

#include "wgkv_common.h"

constexpr int kKv4Group = 32;
constexpr int kKv4Tile = 16;

__host__ __device__ constexpr int kv4_tile_bytes(int D) { return 10 * D; }
WGKV_DEVICE constexpr int kv4_scales_at(int D) { return 8 * D; }

// A caller's paged 4-bit cache (all entry points share these checks).
struct Kv4Pages {
  int64_t num_pages;
  int page_size, page_shift;  // page_size = 16 << page_shift
  const int32_t* bt;
  int64_t bt_sb, bt_sh;
  int max_pages;
};

__host__ __device__ inline int64_t kv4_capacity(const Kv4Pages& p) { return (int64_t)p.max_pages * p.page_size; }

// First byte of tile `tile` (position / 16) of a head, or -1 where its page
// is outside the pool.
template <int D>
WGKV_DEVICE int64_t kv4_tile_at(const Kv4Pages& p, const int32_t* bt_row, int tile) {
  const int pg = bt_row[tile >> p.page_shift];
  if (pg < 0 || pg >= p.num_pages) return -1;
  const int within = tile & ((1 << p.page_shift) - 1);
  return (((int64_t)pg << p.page_shift) + within) * kv4_tile_bytes(D);
}

inline int kv4_pages(Kv4Pages* p, int64_t num_pages, int32_t page_size, const int32_t* bt, int64_t sb, int64_t sh,
                     int32_t max_pages) {
  if (!bt || num_pages <= 0 || max_pages <= 0) return WGKV_ERR_ARG;
  if (page_size != 16 && page_size != 32 && page_size != 64) return WGKV_ERR_UNSUPPORTED;
  // positions are 32-bit
  if ((int64_t)max_pages * page_size > 0x7fffff00) return WGKV_ERR_UNSUPPORTED;
  *p = Kv4Pages{num_pages, page_size, page_size == 16 ? 0 : page_size == 32 ? 1 : 2, bt, sb, sh, max_pages};
  return WGKV_OK;
}

// Whether two rows of `row` elements, spread over four dimensions of these
// sizes and strides, share an element (an output's rows are written by
// workgroups that do not wait for each other).  Layouts whose every stride
// spans what the smaller ones reach cannot; of others, the differences of two
// rows' places are gone through in three dimensions and solved for the largest.
inline bool kv4_rows_meet(const int64_t (&sizes)[4], const int64_t (&strides)[4], int64_t row) {
  typedef __int128 wide;
  wide n[4], s[4];
  int dims = 0;
  for (int i = 0; i < 4; ++i) {
    if (sizes[i] <= 1) continue;
    const wide st = strides[i] < 0 ? -(wide)strides[i] : (wide)strides[i];  // a difference's sign does not matter
    int j = dims++;
    for (; j > 0 && s[j - 1] > st; --j) s[j] = s[j - 1], n[j] = n[j - 1];
    s[j] = st, n[j] = sizes[i];
  }
  wide reach = row;
  bool nested = true;
  for (int i = 0; i < dims; ++i) {
    nested = nested && s[i] >= reach;
    reach += (n[i] - 1) * s[i];
  }
  if (nested) return false;
  int most = 0;
  for (int i = 1; i < dims; ++i)
    if (n[i] > n[most]) most = i;
  const wide step = s[most], far = n[most] - 1;
  if (step < row) return true;  // neighbours in this dimension
  wide d[4];
  for (int i = 0; i < dims; ++i) d[i] = 1 - n[i];
  for (;;) {
    wide x = 0;
    bool same = true;
    for (int i = 0; i < dims; ++i) {
      if (i == most) continue;
      x += d[i] * s[i];
      same = same && d[i] == 0;
    }
    if (!same) {  // the two multiples of `step` next to -x, within reach
      wide k = -x / step - (-x % step < 0 ? 1 : 0);
      for (int i = 0; i < 2; ++i, ++k) {
        const wide c = k < -far ? -far : k > far ? far : k, y = x + c * step;
        if (y < row && -y < row) return true;
      }
    }
    int i = 0;
    for (; i < dims; ++i) {
      if (i == most) continue;
      if (++d[i] < n[i]) break;
      d[i] = 1 - n[i];
    }
    if (i == dims) return false;
  }
}

// Whether a block's 8-byte words fit the 32-bit arguments they become.
template <typename... I>
inline bool kv4_narrow(const int64_t* a, I... at) {
  return ((a[at] == (int32_t)a[at]) && ...);
}

// ---- element types of the rows quantised or read back -------------------------
enum Kv4Type { kKv4Bf16 = 0, kKv4F32 = 1, kKv4F16 = 2 };

// Eight consecutive values of a row as they are in memory.
template <int TY>
struct Kv4Raw {
  u32x4_t w[TY == kKv4F32 ? 2 : 1];
};

// Every row is read once: non-temporally where one access takes it (a 128K
// prompt's append 53 -> 45 us; the two accesses of an fp32 row share a line,
// which the first must leave in the cache).
template <int TY>
WGKV_DEVICE void kv4_fetch(const void* p, int64_t off, Kv4Raw<TY>& r) {
  if constexpr (TY == kKv4F32) {
    r.w[0] = *(const u32x4_t*)((const float*)p + off);
    r.w[1] = *(const u32x4_t*)((const float*)p + off + 4);
  } else {
    r.w[0] = __builtin_nontemporal_load((const u32x4_t*)((const uint16_t*)p + off));
  }
}

template <int TY>
WGKV_DEVICE void kv4_widen(const Kv4Raw<TY>& r, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (TY == kKv4F32) {
      x[i] = __uint_as_float(r.w[0][i]);
      x[4 + i] = __uint_as_float(r.w[1][i]);
    } else if constexpr (TY == kKv4Bf16) {
      x[2 * i] = bf16lo(r.w[0][i]);
      x[2 * i + 1] = bf16hi(r.w[0][i]);
    } else {
      x[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(r.w[0][i] & 0xffffu));
      x[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(r.w[0][i] >> 16));
    }
  }
}

// Eight fp32 values rounded once to the row's type.  Non-temporal: 24K rows
// of 64 heads written 192.6 -> 186.2 us.
template <int TY>
WGKV_DEVICE void kv4_store8(void* p, int64_t off, const float (&x)[8]) {
  if constexpr (TY == kKv4F32) {
    __builtin_nontemporal_store(((f32x4_t){x[0], x[1], x[2], x[3]}), (f32x4_t*)((float*)p + off));
    __builtin_nontemporal_store(((f32x4_t){x[4], x[5], x[6], x[7]}), (f32x4_t*)((float*)p + off + 4));
  } else {
    u32x4_t w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (TY == kKv4Bf16) {
        w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
      } else {
        w[i] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x[2 * i]) |
               (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x[2 * i + 1]) << 16;
      }
    }
    __builtin_nontemporal_store(w, (u32x4_t*)((uint16_t*)p + off));
  }
}
