// Writing and reading a paged cache held in 4 bits (gfx950): the tokens a
// gate admits are quantised as they are appended to each head's pages, and
// rows are read back as dense bf16 / fp16 / fp32 tensors.  The number format
// and the tiles' layout are in kv4.h.
//
// Both kernels give a lane the same piece of the cache: 8 consecutive d of a
// quad of 4 consecutive positions.  D/8 lanes share a quad, a wave takes
// 64/(D/8) quads at a time, every row of the dense side is read or written
// whole by neighbouring lanes, and the values' words of a quad are one
// 16-byte access.  Both are bound by memory.
#include "kv4.h"

namespace {

constexpr int kTile = 64;          // source tokens per append workgroup (one wave)
constexpr int kSegment = 4096;     // flags per counting workgroup
constexpr int kSegTiles = kSegment / kTile;

struct AppendArgs {
  const void* src[2];
  int64_t s_b[2], s_t[2], s_h[2];
  const uint8_t* mask;  // or null: every token
  int64_t m_b, m_h;
  const int32_t* len;
  int64_t len_sb;
  int32_t* new_len;
  int64_t new_sb;
  uint8_t* cache[2];
  Kv4Pages pg;
  int B, T, H;
  int32_t* status;  // or null
  // more than one tile: the lengths before the call (B*H), the admitted
  // tokens of each segment (B*H, segments) and those before each tile within
  // its segment (B*H, tiles)
  int32_t *ws_len, *ws_seg, *ws_tile;
  int tiles, segments;
};

WGKV_DEVICE int clamped_len(const AppendArgs& a, int b, int h) {
  const int64_t n = a.len[(int64_t)b * a.len_sb + h], cap = kv4_capacity(a.pg);
  return (int)(n < 0 ? 0 : n > cap ? cap : n);
}

// Admitted tokens per tile and segment, and a copy of the lengths (the append
// may write the new ones over them).  One workgroup per segment and head,
// 16 flags per thread.
__global__ __launch_bounds__(256) void kv4_count_kernel(AppendArgs a) {
  __shared__ int s_tmp[4];
  const int seg = blockIdx.x, bh = blockIdx.y;
  const int b = bh / a.H, h = bh - b * a.H;
  const int t0 = seg * kSegment + threadIdx.x * 16;
  const int n = min(16, a.T - t0);
  int c = max(n, 0);
  if (a.mask && n > 0) {
    const uint8_t* m = a.mask + (int64_t)b * a.m_b + (int64_t)h * a.m_h + t0;
    c = 0;
    if (n == 16) {
      u32x4_t w;
      __builtin_memcpy(&w, m, 16);  // rows of odd length start anywhere
#pragma unroll
      for (int i = 0; i < 4; ++i)  // bit 7 of each nonzero byte
        c += __builtin_popcount((((w[i] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w[i]) & 0x80808080u);
    } else {
      for (int i = 0; i < n; ++i) c += m[i] != 0;
    }
  }
  int total = 0;
  const int before = block_exclusive_scan_256(c, s_tmp, &total);
  constexpr int per = kTile / 16;  // threads per tile
  const int tile = seg * kSegTiles + (int)threadIdx.x / per;
  if (threadIdx.x % per == 0 && tile < a.tiles) a.ws_tile[(int64_t)bh * a.tiles + tile] = before;
  if (threadIdx.x == 0) {
    a.ws_seg[(int64_t)bh * a.segments + seg] = total;
    if (seg == 0) a.ws_len[bh] = clamped_len(a, b, h);
  }
}

WGKV_DEVICE float quad_max(float x) {
  x = fmaxf(x, dpp_f32<WGKV_DPP_QP_1032>(x));
  return fmaxf(x, dpp_f32<WGKV_DPP_QP_2301>(x));
}
WGKV_DEVICE float quad_min(float x) {
  x = fminf(x, dpp_f32<WGKV_DPP_QP_1032>(x));
  return fminf(x, dpp_f32<WGKV_DPP_QP_2301>(x));
}

// Nearest bf16 of an fp32 value, in integers: a conversion instruction after
// one from fp64 is folded into a single rounding from fp64, another number
// where the fp32 value lies halfway between two bf16 ones.
WGKV_DEVICE float bf16_of(float x) { return __uint_as_float((uint32_t)f32_to_bf16(x) << 16); }

// Quantises a lane's 8 values of a group that four neighbouring lanes share.
// Returns (s, m) as a packed pair; codes 0..3 and 4..7 in c[0..7].
WGKV_DEVICE uint32_t quantise8(const float (&x)[8], uint32_t (&c)[8]) {
  float hi = x[0], lo = x[0], finite = x[0] * 0.f;
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    hi = fmaxf(hi, x[i]);
    lo = fminf(lo, x[i]);
    finite = fmaf(x[i], 0.f, finite);  // NaN once a value is not finite
  }
  hi = quad_max(hi);
  lo = quad_min(lo);
  finite += dpp_f32<WGKV_DPP_QP_1032>(finite);
  finite += dpp_f32<WGKV_DPP_QP_2301>(finite);
  // In 64 bits, as a multiplication: 1/15 in fp64 is 2^-56 off, too little
  // to move the quotient across a border of fp32 or bf16.
  float s = bf16_of((float)(((double)hi - (double)lo) * (1.0 / 15.0)));
  const float m = bf16_of(0.5f * hi + 0.5f * lo);
  if (!(s >= 0x1p-126f)) s = 0.f;
  const bool bad = finite != 0.f || !(fabsf(m) <= 0x1.fep127f);
  // code = 8 + k for x beyond m + k s, 7 + k below it, the even one on it,
  // for an integer k next to (x - m) / s: that need not be the nearest, so
  // the quotient may be approximate, and the side is decided by an exact
  // residue (fp64 holds x - m and k s).  A rounded fp32 quotient would put
  // values near a border on the wrong side.
  const float inv = __builtin_amdgcn_rcpf(s);
  const double md = (double)m, sd = (double)s;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float k = rintf((x[i] - m) * inv);
    const double r = fma(-(double)k, sd, (double)x[i] - md);
    const int ki = (int)fminf(fmaxf(k, -9.f), 9.f);
    const int up = r > 0.0 || (r == 0.0 && !(ki & 1));
    const int code = min(15, max(0, ki + 7 + up));
    c[i] = s == 0.f || bad ? 0u : (uint32_t)code;
  }
  const uint32_t w = (__float_as_uint(s) >> 16) | (__float_as_uint(m) & 0xffff0000u);
  return bad ? 0x7fc07fc0u : w;
}

template <int D, int TY>
__global__ __launch_bounds__(64) void kv4_append_kernel(AppendArgs a) {
  constexpr int LPR = D / 8;        // lanes per quad
  constexpr int QPW = 64 / LPR;     // quads per step
  constexpr int NG = D / kKv4Group;
  __shared__ uint8_t s_src[kTile];
  const int tile = blockIdx.x, bh = blockIdx.y;
  const int b = bh / a.H, h = bh - b * a.H;
  const int lane = threadIdx.x;
  const int t0 = tile * kTile;

  bool f = t0 + lane < a.T;
  if (f && a.mask) f = a.mask[(int64_t)b * a.m_b + (int64_t)h * a.m_h + t0 + lane] != 0;
  const uint64_t bits = __builtin_amdgcn_ballot_w64(f);
  if (f) s_src[__builtin_popcountll(bits & ((1ull << lane) - 1))] = (uint8_t)lane;
  wave_lds_sync();
  const int n_adm = __builtin_popcountll(bits);

  // positions [p0, p1) take the tile's admitted tokens
  int64_t first;
  if (a.tiles > 1) {
    const int seg = tile / kSegTiles;
    int before = 0;
    for (int i = lane; i < seg; i += 64) before += a.ws_seg[(int64_t)bh * a.segments + i];
    first = (int64_t)a.ws_len[bh] + wave_sum_int(before) + a.ws_tile[(int64_t)bh * a.tiles + tile];
  } else {
    first = clamped_len(a, b, h);
  }
  const int64_t cap = kv4_capacity(a.pg);
  const int p0 = (int)min(first, cap), p1 = (int)min(first + n_adm, cap);
  bool lost = first + n_adm > cap;
  if (tile == max(a.tiles, 1) - 1 && lane == 0) a.new_len[(int64_t)b * a.new_sb + h] = p1;

  const int32_t* bt_row = a.pg.bt + (int64_t)b * a.pg.bt_sb + (int64_t)h * a.pg.bt_sh;
  const int L = lane % LPR, slot = lane / LPR;
  const int q0 = p0 >> 2, nq = p1 > p0 ? ((p1 - 1) >> 2) - q0 + 1 : 0;
  // items: keys and values of each quad in turn, so that a single token's
  // key and value are quantised side by side
  for (int it = slot; it < 2 * nq; it += QPW) {
    const int quad = q0 + (it >> 1), kind = it & 1;
    const int64_t at = kv4_tile_at<D>(a.pg, bt_row, quad >> 2);
    if (at < 0) {
      lost = true;
      continue;
    }
    uint32_t w[4][2], sm[4];
    bool ok[4];
    float x[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = quad * 4 + i;
      ok[i] = p >= p0 && p < p1;
      const int src = t0 + s_src[min(max(p - p0, 0), n_adm - 1)];
      kv4_load8<TY>(a.src[kind], (int64_t)b * a.s_b[kind] + (int64_t)src * a.s_t[kind] + (int64_t)h * a.s_h[kind] + L * 8,
                    x[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t c[8];
      sm[i] = quantise8(x[i], c);
      if (kind == 0) {
        w[i][0] = c[0] | c[2] << 4 | c[4] << 8 | c[6] << 12;
        w[i][1] = c[1] | c[3] << 4 | c[5] << 8 | c[7] << 12;
      } else {
        w[i][0] = c[0] | c[1] << 4 | c[2] << 8 | c[3] << 12;
        w[i][1] = c[4] | c[5] << 4 | c[6] << 8 | c[7] << 12;
      }
    }
    uint8_t* tp = a.cache[kind] + at;
    const int qi = quad & 3;
    const bool whole = ok[0] && ok[1] && ok[2] && ok[3];
    if (kind == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (ok[i]) *(uint32_t*)(tp + (qi * 4 + i) * (D / 2) + L * 4) = w[i][0] | w[i][1] << 16;
    } else {
      // words of lane L: D = 128: row r = L, halves 0 and 1; D = 64: rows
      // 2L and 2L + 1.  Both are 16 consecutive bytes of the quad.
      uint8_t* vp = tp + qi * (2 * D) + L * 16;
      constexpr int kWord = D == 128 ? 4 : 8, kPair = D == 128 ? 8 : 4;  // strides of w[.][1] and of t%4/2
      if (whole) {
        u32x4_t v;
#pragma unroll
        for (int pr = 0; pr < 2; ++pr)
#pragma unroll
          for (int j = 0; j < 2; ++j) v[(pr * kPair + j * kWord) / 4] = w[2 * pr][j] | w[2 * pr + 1][j] << 16;
        *(u32x4_t*)vp = v;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (ok[i]) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
              *(uint16_t*)(vp + (i >> 1) * kPair + j * kWord + (i & 1) * 2) = (uint16_t)w[i][j];
          }
      }
    }
    if (L % 4 == 0) {
      uint32_t* sp = (uint32_t*)(tp + kv4_scales_at(D)) + (qi * NG + L / 4) * 4;
      if (whole) {
        *(u32x4_t*)sp = (u32x4_t){sm[0], sm[1], sm[2], sm[3]};
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (ok[i]) sp[i] = sm[i];
      }
    }
  }
  if (a.status && lost) atomicMax(a.status, WGKV_ERR_CAPACITY);
}

struct ReadArgs {
  const uint8_t* cache[2];
  Kv4Pages pg;
  const int32_t* len;
  int64_t len_sb;
  const int32_t* start;  // or null: 0
  int64_t start_sb;
  void* out[2];
  int64_t o_b, o_t, o_h;
  int B, rows, H;
};

// One wave per 64 positions of a head's keys or values.
constexpr int kReadTile = 64;

template <int D, int TY>
__global__ __launch_bounds__(64) void kv4_read_kernel(ReadArgs a) {
  constexpr int LPR = D / 8, QPW = 64 / LPR, NG = D / kKv4Group;
  const int bh = blockIdx.y, kind = blockIdx.z;
  const int b = bh / a.H, h = bh - b * a.H;
  const int64_t cap = kv4_capacity(a.pg);
  int64_t len = a.len[(int64_t)b * a.len_sb + h];
  len = len < 0 ? 0 : len > cap ? cap : len;
  const int start = a.start ? max(a.start[(int64_t)b * a.start_sb + h], 0) : 0;
  const int64_t end = (int64_t)start + a.rows;
  const int32_t* bt_row = a.pg.bt + (int64_t)b * a.pg.bt_sb + (int64_t)h * a.pg.bt_sh;
  const int lane = threadIdx.x, L = lane % LPR, slot = lane / LPR;
  const int64_t quad0 = (int64_t)(start >> 2) + (int64_t)blockIdx.x * (kReadTile / 4);
  const int64_t ob = (int64_t)b * a.o_b + (int64_t)h * a.o_h + L * 8;
#pragma unroll 2
  for (int i0 = slot; i0 < kReadTile / 4; i0 += QPW) {
    const int64_t quad = quad0 + i0, p = quad * 4;
    if (p >= end) break;
    float x[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] = 0.f;
    const int64_t at = p < len ? kv4_tile_at<D>(a.pg, bt_row, (int)(quad >> 2)) : -1;
    if (at >= 0) {
      const uint8_t* tp = a.cache[kind] + at;
      const int qi = (int)(quad & 3);
      const u32x4_t sm = *(const u32x4_t*)(tp + kv4_scales_at(D) + (qi * NG + L / 4) * 16);
      uint32_t w[4][2];  // codes of token i: K even / odd d, V first / second four
      if (kind == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t v = *(const uint32_t*)(tp + (qi * 4 + i) * (D / 2) + L * 4);
          w[i][0] = v & 0xffffu;
          w[i][1] = v >> 16;
        }
      } else {
        const u32x4_t v = *(const u32x4_t*)(tp + qi * (2 * D) + L * 16);
        constexpr int kWord = D == 128 ? 1 : 2, kPair = D == 128 ? 2 : 1;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) w[i][j] = (v[(i >> 1) * kPair + j * kWord] >> (16 * (i & 1))) & 0xffffu;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (p + i >= len) continue;
        const float s = bf16lo(sm[i]), m = bf16hi(sm[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float c0 = (float)(w[i][0] >> (4 * j) & 15u) - 7.5f, c1 = (float)(w[i][1] >> (4 * j) & 15u) - 7.5f;
          x[i][kind == 0 ? 2 * j : j] = fmaf(s, c0, m);
          x[i][kind == 0 ? 2 * j + 1 : 4 + j] = fmaf(s, c1, m);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = p + i - start;
      if (row >= 0 && row < a.rows) kv4_store8<TY>(a.out[kind], ob + row * a.o_t, x[i]);
    }
  }
}

template <int D>
void launch_append(const AppendArgs& a, int ty, hipStream_t st) {
  const dim3 g(max(a.tiles, 1), a.B * a.H);
  if (ty == kKv4Bf16) hipLaunchKernelGGL((kv4_append_kernel<D, kKv4Bf16>), g, dim3(64), 0, st, a);
  else if (ty == kKv4F32) hipLaunchKernelGGL((kv4_append_kernel<D, kKv4F32>), g, dim3(64), 0, st, a);
  else hipLaunchKernelGGL((kv4_append_kernel<D, kKv4F16>), g, dim3(64), 0, st, a);
}

template <int D>
void launch_read(const ReadArgs& a, int ty, hipStream_t st) {
  // one workgroup more than rows / 64: the first row may lie inside a quad
  const dim3 g((a.rows + 3 + kReadTile - 1) / kReadTile, a.B * a.H, 2);
  if (ty == kKv4Bf16) hipLaunchKernelGGL((kv4_read_kernel<D, kKv4Bf16>), g, dim3(64), 0, st, a);
  else if (ty == kKv4F32) hipLaunchKernelGGL((kv4_read_kernel<D, kKv4F32>), g, dim3(64), 0, st, a);
  else hipLaunchKernelGGL((kv4_read_kernel<D, kKv4F16>), g, dim3(64), 0, st, a);
}

int tiles_of(int T) { return (T + kTile - 1) / kTile; }
int segments_of(int T) { return (T + kSegment - 1) / kSegment; }

constexpr int kMaxBH = 65535;  // grid y

}  // namespace

extern "C" size_t wgkv_kv4_append_workspace_bytes(int32_t batch, int32_t num_kv_heads, int32_t tokens) {
  if (batch <= 0 || num_kv_heads <= 0 || tokens <= kTile) return 0;
  return ((size_t)1 + segments_of(tokens) + tiles_of(tokens)) * batch * num_kv_heads * sizeof(int32_t);
}

extern "C" int wgkv_kv4_append(
    const void* key, int64_t k_stride_b, int64_t k_stride_t, int64_t k_stride_h,
    const void* value, int64_t v_stride_b, int64_t v_stride_t, int64_t v_stride_h, int32_t dtype,
    const uint8_t* g_mask, int64_t gm_stride_b, int64_t gm_stride_h,
    const int32_t* lengths, int64_t len_stride_b, int32_t* new_lengths, int64_t new_stride_b,
    void* k_cache, void* v_cache, int64_t num_pages, int32_t page_size,
    const int32_t* block_table, int64_t bt_stride_b, int64_t bt_stride_h, int32_t max_pages,
    int32_t batch, int32_t tokens, int32_t num_kv_heads, int32_t head_dim,
    int32_t* status, void* workspace, size_t workspace_bytes, void* stream) {
  if (!lengths || !new_lengths || !k_cache || !v_cache) return WGKV_ERR_ARG;
  if (tokens < 0 || batch <= 0 || num_kv_heads <= 0 || (tokens > 0 && (!key || !value))) return WGKV_ERR_ARG;
  if (head_dim != 64 && head_dim != 128) return WGKV_ERR_UNSUPPORTED;
  if (dtype != kKv4Bf16 && dtype != kKv4F32 && dtype != kKv4F16) return WGKV_ERR_UNSUPPORTED;
  if ((int64_t)batch * num_kv_heads > kMaxBH || tokens > (1 << 30)) return WGKV_ERR_UNSUPPORTED;
  AppendArgs a{};
  const int st = kv4_pages(&a.pg, num_pages, page_size, block_table, bt_stride_b, bt_stride_h, max_pages);
  if (st != WGKV_OK) return st;
  // 16-byte loads of the rows and accesses of the tiles
  const int64_t unit = dtype == kKv4F32 ? 3 : 7;
  if (((uintptr_t)key | (uintptr_t)value | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) return WGKV_ERR_UNSUPPORTED;
  if ((k_stride_b | k_stride_t | k_stride_h | v_stride_b | v_stride_t | v_stride_h) & unit) return WGKV_ERR_UNSUPPORTED;
  a.src[0] = key;
  a.src[1] = value;
  a.s_b[0] = k_stride_b, a.s_t[0] = k_stride_t, a.s_h[0] = k_stride_h;
  a.s_b[1] = v_stride_b, a.s_t[1] = v_stride_t, a.s_h[1] = v_stride_h;
  a.mask = g_mask;
  a.m_b = gm_stride_b;
  a.m_h = gm_stride_h;
  a.len = lengths;
  a.len_sb = len_stride_b;
  a.new_len = new_lengths;
  a.new_sb = new_stride_b;
  a.cache[0] = (uint8_t*)k_cache;
  a.cache[1] = (uint8_t*)v_cache;
  a.B = batch;
  a.T = tokens;
  a.H = num_kv_heads;
  a.status = status;
  a.tiles = tiles_of(tokens);
  a.segments = segments_of(tokens);
  hipStream_t s = (hipStream_t)stream;
  if (a.tiles > 1) {
    if (!workspace || ((uintptr_t)workspace & 3) ||
        workspace_bytes < wgkv_kv4_append_workspace_bytes(batch, num_kv_heads, tokens))
      return WGKV_ERR_WORKSPACE;
    const int64_t bh = (int64_t)batch * num_kv_heads;
    a.ws_len = (int32_t*)workspace;
    a.ws_seg = a.ws_len + bh;
    a.ws_tile = a.ws_seg + bh * a.segments;
    hipLaunchKernelGGL(kv4_count_kernel, dim3(a.segments, (unsigned)bh), dim3(256), 0, s, a);
    if (hipGetLastError() != hipSuccess) return WGKV_ERR_HIP;
  }
  if (head_dim == 128) launch_append<128>(a, dtype, s);
  else launch_append<64>(a, dtype, s);
  return hipGetLastError() == hipSuccess ? WGKV_OK : WGKV_ERR_HIP;
}

extern "C" int wgkv_kv4_read(
    const void* k_cache, const void* v_cache, int64_t num_pages, int32_t page_size,
    const int32_t* block_table, int64_t bt_stride_b, int64_t bt_stride_h, int32_t max_pages,
    const int32_t* lengths, int64_t len_stride_b, const int32_t* starts, int64_t start_stride_b,
    void* key, void* value, int64_t out_stride_b, int64_t out_stride_t, int64_t out_stride_h, int32_t dtype,
    int32_t batch, int32_t rows, int32_t num_kv_heads, int32_t head_dim, void* stream) {
  if (!k_cache || !v_cache || !lengths || !key || !value) return WGKV_ERR_ARG;
  if (batch <= 0 || num_kv_heads <= 0 || rows <= 0) return WGKV_ERR_ARG;
  if (head_dim != 64 && head_dim != 128) return WGKV_ERR_UNSUPPORTED;
  if (dtype != kKv4Bf16 && dtype != kKv4F32 && dtype != kKv4F16) return WGKV_ERR_UNSUPPORTED;
  if ((int64_t)batch * num_kv_heads > kMaxBH || rows > (1 << 30)) return WGKV_ERR_UNSUPPORTED;
  ReadArgs a{};
  const int st = kv4_pages(&a.pg, num_pages, page_size, block_table, bt_stride_b, bt_stride_h, max_pages);
  if (st != WGKV_OK) return st;
  const int64_t unit = dtype == kKv4F32 ? 3 : 7;
  if (((uintptr_t)key | (uintptr_t)value | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) return WGKV_ERR_UNSUPPORTED;
  if ((out_stride_b | out_stride_t | out_stride_h) & unit) return WGKV_ERR_UNSUPPORTED;
  a.cache[0] = (const uint8_t*)k_cache;
  a.cache[1] = (const uint8_t*)v_cache;
  a.len = lengths;
  a.len_sb = len_stride_b;
  a.start = starts;
  a.start_sb = start_stride_b;
  a.out[0] = key;
  a.out[1] = value;
  a.o_b = out_stride_b;
  a.o_t = out_stride_t;
  a.o_h = out_stride_h;
  a.B = batch;
  a.rows = rows;
  a.H = num_kv_heads;
  if (head_dim == 128) launch_read<128>(a, dtype, (hipStream_t)stream);
  else launch_read<64>(a, dtype, (hipStream_t)stream);
  return hipGetLastError() == hipSuccess ? WGKV_OK : WGKV_ERR_HIP;
}
