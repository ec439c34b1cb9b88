// Writing and reading a paged cache held in 4 bits (gfx950): the tokens a
// gate admits are quantised as they are appended to each head's pages, and
// rows are read back as dense bf16 / fp16 / fp32 tensors.  The number format
// and the tiles' layout are in kv4.h.
//
// Both kernels give a lane the same piece of the cache: 8 consecutive d of a
// quad of 4 consecutive positions.  D/8 lanes share a quad, a wave takes
// 64/(D/8) quads at a time, every row of the dense side is read or written
// whole by neighbouring lanes, and the values' words of a quad are one
// 16-byte access.  The read-back is bound by its writes (24K rows of 64 heads,
// 994 MB, 186 us, 5.35 TB/s; a copy reaches 4.9).  The append is bound by
// nothing alone (26K admitted rows of a 128K prompt in 8 heads, 143 MB moved:
// 45 us, of which 30 are vector instructions' issue, the rounding's above all):
// a tile with a fifth of its tokens admitted is one step, whose flags, page
// id, rows and arithmetic follow each other.  460 instructions less per wave
// took 8 us off; registers for more waves spill (87 us for both calls instead
// of 79).
#include <string.h>

#include "kv4.h"

namespace {

constexpr int kFew = 64;           // up to this many tokens a call is one-wave workgroups
constexpr int kTile = 256;         // source tokens per append workgroup otherwise
constexpr int kSegment = 4096;     // flags per counting workgroup
constexpr int kSegTiles = kSegment / kTile;
// Up to this many tokens a workgroup counts the flags in front of its tile
// itself; beyond, kv4_count_kernel does, in a launch before.
constexpr int kCountsItself = 16384;

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
  // what kv4_count_kernel leaves, or null: the lengths before the call
  // (B*H), the admitted tokens of each segment (B*H, segments) and those
  // before each tile within its segment (B*H, tiles)
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

// NaN-propagating maximum and minimum (v_maximum3 / v_minimum3), over a
// lane's values and then its quad of lanes.
WGKV_DEVICE float quad_maximum(float x) {
  x = __builtin_elementwise_maximum(x, dpp_f32<WGKV_DPP_QP_1032>(x));
  return __builtin_elementwise_maximum(x, dpp_f32<WGKV_DPP_QP_2301>(x));
}
WGKV_DEVICE float quad_minimum(float x) {
  x = __builtin_elementwise_minimum(x, dpp_f32<WGKV_DPP_QP_1032>(x));
  return __builtin_elementwise_minimum(x, dpp_f32<WGKV_DPP_QP_2301>(x));
}

// Nearest bf16 of a finite fp32 value, in integers: a conversion instruction
// after one from fp64 is folded into a single rounding from fp64, another
// number where the fp32 value lies halfway between two bf16 ones.
WGKV_DEVICE float bf16_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return __uint_as_float((u + 0x7fffu + (u >> 16 & 1u)) & 0xffff0000u);
}

// A group's step, middle and reciprocal step; the step is 0 where the group
// has none (all values alike, or one not finite: `pair` says which).
struct Group {
  float s, m, inv;
  uint32_t pair;  // (s, m) as they are stored
};

WGKV_DEVICE Group group_of(float hi, float lo) {
  // In 64 bits, as a multiplication: 1/15 in fp64 is 2^-56 off, too little
  // to move the quotient across a border of fp32 or bf16.
  const float sf = (float)(((double)hi - (double)lo) * (1.0 / 15.0));
  Group g;
  g.s = bf16_of(sf);
  // The sum in 64 bits too: half of an odd fp32 subnormal is not an fp32 number.
  g.m = bf16_of((float)(((double)hi + (double)lo) * 0.5));
  const bool bad = !(sf < INFINITY) || !(fabsf(g.m) < INFINITY);
  if (!(g.s >= 0x1p-126f) || bad) g.s = 0.f;
  g.inv = __builtin_amdgcn_rcpf(g.s);
  g.pair = bad ? 0x7fc07fc0u : (__float_as_uint(g.s) >> 16) | __float_as_uint(g.m);
  return g;
}

// The code of x is k + 7.5 rounded to even for x = m + k s, k + 8 beyond it
// and k + 7 below, for an integer k next to (x - m) / s.  That need not be the
// nearest, so the quotient may be approximate (v_rcp is good to 2^-23), and
// the side is decided by the sign of an exact residue (k here is k + 7, and m7
// its zero):
//   * 16-bit inputs: x - (m + k s).  The border m + k s is exact in fp32 for
//     the |k| <= 8 that matter: m has 8 bits and k s 12, m is 0 or at least
//     2^-13 of the range (a sum of two 11-bit numbers), and s is at least
//     2^-15 of m (values that differ do so by a unit of their 11 bits).
//   * fp32: (x - m) - k s with the two-sum error of x - m, which counts only
//     where the rounded difference equals k s (a nonzero residue is at least
//     one ulp of it).
template <int TY>
WGKV_DEVICE void exact_codes(const float (&x)[8], float s, float m, float inv, float (&c)[8]) {
  const float nb = fmaf(-m, inv, 7.f), m7 = fmaf(-7.f, s, m);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float k, r;
    if constexpr (TY == kKv4F32) {
      const float d = x[i] - m;
      k = rintf(d * inv);
      const float bb = d - x[i];
      r = (fmaf(-k, s, d) + ((x[i] - (d - bb)) - (m + bb))) * inv * 0x1p-97f;
      k += 7.f;
    } else {
      k = rintf(fmaf(x[i], inv, nb));
      r = x[i] - fmaf(k, s, m7);
    }
    // 0, 0.5 or 1 by the residue's sign: for 16-bit inputs any (the least is
    // 2^-133, at steps of 2^-126), for fp32 those above 2^-51 of a step, which
    // arithmetic in 64 bits tells from a border too.
    const float side = __builtin_amdgcn_fmed3f(fmaf(r, 0x1p127f, 0.5f), 0.f, 1.f);
    c[i] = rintf(__builtin_amdgcn_fmed3f(k + side, 0.f, 15.f));
  }
}

// The codes of a lane's 8 values, as numbers.
template <int TY>
WGKV_DEVICE void codes_of(const float (&x)[8], float s, float m, float inv, float (&c)[8]) {
  if constexpr (TY == kKv4F32) {
    // (x - m) / s + 7.5 by one fma is within 2^-24 (|bias| + 32) of itself.
    // Rows of a wave with a value that near to a border between two codes are
    // taken exactly.  (Not for 16-bit inputs: 0.7 % of bf16 values lie on a
    // border, some in every wave.)
    const float bias = fmaf(-m, inv, 7.5f);
    float far = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float t = fmaf(x[i], inv, bias), r = rintf(t);
      far = fmaxf(far, fabsf(t - r));
      c[i] = __builtin_amdgcn_fmed3f(r, 0.f, 15.f);
    }
    const bool near = far >= 0.5f - 0x1p-23f * (fabsf(bias) + 32.f);
    if (__builtin_amdgcn_ballot_w64(near && s != 0.f)) exact_codes<TY>(x, s, m, inv, c);
  } else {
    exact_codes<TY>(x, s, m, inv, c);
  }
}

template <int I>
WGKV_DEVICE float quad_lane(float x) {  // lane I of each four
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), I * 0x55, 0xf, 0xf, true));
}

// Four codes as a 16-bit word, the first in the lowest bits.
WGKV_DEVICE uint32_t pack4(float a, float b, float c, float d) {
  return (uint32_t)fmaf(d, 4096.f, fmaf(c, 256.f, fmaf(b, 16.f, a)));
}

// One quad of positions quantised and written: kKeys or values, the four
// tokens' values x, those of them that are there (ok).
template <int D, int TY, bool kKeys>
WGKV_DEVICE void write_quad(uint8_t* tile, int qi, int L, const Kv4Raw<TY> (&raw)[4], const bool (&ok)[4]) {
  constexpr int NG = D / kKv4Group;
  uint32_t w[4][2];
  float x[4][8], hi[4], lo[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    kv4_widen<TY>(raw[i], x[i]);
    hi[i] = lo[i] = x[i][0];
#pragma unroll
    for (int j = 1; j < 8; ++j) {
      hi[i] = __builtin_elementwise_maximum(hi[i], x[i][j]);
      lo[i] = __builtin_elementwise_minimum(lo[i], x[i][j]);
    }
    hi[i] = quad_maximum(hi[i]);
    lo[i] = quad_minimum(lo[i]);
  }
  // four lanes share the four tokens' groups: lane j works token j's out
  const int j = L & 3;
  const Group g = group_of(j == 0 ? hi[0] : j == 1 ? hi[1] : j == 2 ? hi[2] : hi[3],
                           j == 0 ? lo[0] : j == 1 ? lo[1] : j == 2 ? lo[2] : lo[3]);
  const float gs[4] = {quad_lane<0>(g.s), quad_lane<1>(g.s), quad_lane<2>(g.s), quad_lane<3>(g.s)};
  const float gm[4] = {quad_lane<0>(g.m), quad_lane<1>(g.m), quad_lane<2>(g.m), quad_lane<3>(g.m)};
  const float gi[4] = {quad_lane<0>(g.inv), quad_lane<1>(g.inv), quad_lane<2>(g.inv), quad_lane<3>(g.inv)};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float c[8];
    codes_of<TY>(x[i], gs[i], gm[i], gi[i], c);
    if constexpr (kKeys) {
      w[i][0] = pack4(c[0], c[2], c[4], c[6]);
      w[i][1] = pack4(c[1], c[3], c[5], c[7]);
    } else {
      w[i][0] = pack4(c[0], c[1], c[2], c[3]);
      w[i][1] = pack4(c[4], c[5], c[6], c[7]);
    }
    if (gs[i] == 0.f) w[i][0] = w[i][1] = 0u;
  }
  const bool whole = ok[0] && ok[1] && ok[2] && ok[3];
  if constexpr (kKeys) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (ok[i]) *(uint32_t*)(tile + (qi * 4 + i) * (D / 2) + L * 4) = w[i][0] | w[i][1] << 16;
  } else {
    // words of lane L: D = 128: row r = L, halves 0 and 1; D = 64: rows 2L
    // and 2L + 1.  Both are 16 consecutive bytes of the quad.
    uint8_t* vp = tile + qi * (2 * D) + L * 16;
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
  if (j == 0 ? ok[0] : j == 1 ? ok[1] : j == 2 ? ok[2] : ok[3])
    *((uint32_t*)(tile + kv4_scales_at(D)) + (qi * NG + L / 4) * 4 + j) = g.pair;
}

// One workgroup per tile of source tokens and head; NW waves, 64 tokens each.
template <int D, int TY, int NW>
__global__ __launch_bounds__(NW * 64) void kv4_append_kernel(AppendArgs a) {
  constexpr int LPR = D / 8;             // lanes per quad
  constexpr int kSlots = NW * 64 / LPR;  // quads per step
  __shared__ uint8_t s_src[NW * 64];
  __shared__ int s_adm[NW], s_before[NW], s_len;
  const int tile = blockIdx.x, bh = blockIdx.y;
  const int b = bh / a.H, h = bh - b * a.H;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int t0 = tile * (NW * 64);
  const uint8_t* mask = a.mask ? a.mask + (int64_t)b * a.m_b + (int64_t)h * a.m_h : nullptr;

  // The head's length, through one thread: the new one may be written over it
  // by the same thread.  Then the admitted tokens in front of the tile.
  int len = 0, before = 0;
  if (NW == 1 || tid == 0) len = NW > 1 && a.ws_len ? a.ws_len[bh] : clamped_len(a, b, h);
  if (NW > 1 && a.ws_len) {
    const int seg = tile / kSegTiles;
    if (wid == 0)
      for (int i = lane; i < seg; i += 64) before += a.ws_seg[(int64_t)bh * a.segments + i];
    if (tid == 0) before += a.ws_tile[(int64_t)bh * a.tiles + tile];
  } else {
    if (NW > 1) {
      if (mask) before = count_flags(mask, 0, t0, tid, NW * 64);
      else if (tid == 0) before = t0;
    }
  }
  bool f = t0 + tid < a.T;
  if (f && mask) f = mask[t0 + tid] != 0;
  const uint64_t bits = __builtin_amdgcn_ballot_w64(f);
  int rank = __builtin_popcountll(bits & ((1ull << lane) - 1));
  int n_adm = __builtin_popcountll(bits);
  if constexpr (NW > 1) {
    before = wave_sum_int(before);
    if (lane == 0) {
      s_adm[wid] = n_adm;
      s_before[wid] = before;
    }
    if (tid == 0) s_len = len;
    __syncthreads();
    len = s_len;
    n_adm = before = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      if (i < wid) rank += s_adm[i];
      n_adm += s_adm[i];
      before += s_before[i];
    }
  }
  if (f) s_src[rank] = (uint8_t)tid;
  if constexpr (NW > 1) __syncthreads();
  else wave_lds_sync();

  // positions [p0, p1) take the tile's admitted tokens
  const int64_t first = (int64_t)len + before, cap = kv4_capacity(a.pg);
  const int p0 = (int)min(first, cap), p1 = (int)min(first + n_adm, cap);
  bool lost = first + n_adm > cap;
  if (tile == max(a.tiles, 1) - 1 && tid == 0) a.new_len[(int64_t)b * a.new_sb + h] = p1;

  const int32_t* bt_row = a.pg.bt + (int64_t)b * a.pg.bt_sb + (int64_t)h * a.pg.bt_sh;
  const int L = tid % LPR, slot = tid / LPR;
  const int64_t kb = (int64_t)b * a.s_b[0] + (int64_t)h * a.s_h[0] + (int64_t)t0 * a.s_t[0] + L * 8;
  const int64_t vb = (int64_t)b * a.s_b[1] + (int64_t)h * a.s_h[1] + (int64_t)t0 * a.s_t[1] + L * 8;
  const uint32_t kst = (uint32_t)a.s_t[0], vst = (uint32_t)a.s_t[1];  // below 2^32 (the host's check)
  const int q0 = p0 >> 2, nq = p1 > p0 ? ((p1 - 1) >> 2) - q0 + 1 : 0;
  // A step takes keys and values of a quad per group of lanes, their eight
  // rows and the page id asked for together.  Few quads (a decode step) give
  // keys and values to neighbouring groups instead.
  const bool apart = 2 * nq <= kSlots;
  const int n_items = apart ? 2 * nq : nq;
  for (int it = slot; it < n_items; it += kSlots) {
    const int quad = q0 + (apart ? it >> 1 : it);
    const bool do_k = !apart || !(it & 1), do_v = !apart || (it & 1);
    Kv4Raw<TY> kr[4], vr[4];
    bool ok[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = quad * 4 + i;
      ok[i] = p >= p0 && p < p1;
      const uint32_t src = s_src[min(max(p - p0, 0), n_adm - 1)];
      if (do_k) kv4_fetch<TY>(a.src[0], kb + (int64_t)((uint64_t)src * kst), kr[i]);
      if (do_v) kv4_fetch<TY>(a.src[1], vb + (int64_t)((uint64_t)src * vst), vr[i]);
    }
    const int64_t at = kv4_tile_at<D>(a.pg, bt_row, quad >> 2);
    if (at < 0) {
      lost = true;
      continue;
    }
    if (do_k) write_quad<D, TY, true>(a.cache[0] + at, quad & 3, L, kr, ok);
    if (do_v) write_quad<D, TY, false>(a.cache[1] + at, quad & 3, L, vr, ok);
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

// A lane's 8 d of four tokens, from the words and pairs of their quad.
template <int D, bool kKeys>
WGKV_DEVICE void quad_values(const uint8_t* tile, int qi, int L, float (&x)[4][8]) {
  constexpr int NG = D / kKv4Group;
  const u32x4_t sm = *(const u32x4_t*)(tile + kv4_scales_at(D) + (qi * NG + L / 4) * 16);
  uint32_t w[4];  // token i's two words
  if constexpr (kKeys) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = *(const uint32_t*)(tile + (qi * 4 + i) * (D / 2) + L * 4);
  } else {
    const u32x4_t v = *(const u32x4_t*)(tile + qi * (2 * D) + L * 16);
    constexpr int kWord = D == 128 ? 1 : 2, kPair = D == 128 ? 2 : 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a = v[(i >> 1) * kPair], b = v[(i >> 1) * kPair + kWord];
      w[i] = i & 1 ? a >> 16 | (b & 0xffff0000u) : (a & 0xffffu) | b << 16;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float s = bf16lo(sm[i]), m = bf16hi(sm[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int sh = kKeys ? 4 * (j >> 1) + 16 * (j & 1) : 4 * j;  // word of d, code in it
      x[i][j] = fmaf(s, (float)(w[i] >> sh & 15u) - 7.5f, m);
    }
  }
}

// One wave per 64 positions of a head's keys or values.
constexpr int kReadTile = 64;

template <int D, int TY, bool kKeys>
WGKV_DEVICE void read_tile(const ReadArgs& a, int b, int h) {
  constexpr int LPR = D / 8, QPW = 64 / LPR;
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
    const int64_t at = p < len ? kv4_tile_at<D>(a.pg, bt_row, (int)(quad >> 2)) : -1;
    if (at >= 0) {
      quad_values<D, kKeys>(a.cache[kKeys ? 0 : 1] + at, (int)(quad & 3), L, x);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool there = at >= 0 && p + i < len;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] = there ? x[i][j] : 0.f;
      const int64_t row = p + i - start;
      if (row >= 0 && row < a.rows) kv4_store8<TY>(a.out[kKeys ? 0 : 1], ob + row * a.o_t, x[i]);
    }
  }
}

template <int D, int TY>
__global__ __launch_bounds__(64) void kv4_read_kernel(ReadArgs a) {
  const int bh = blockIdx.y, b = bh / a.H, h = bh - b * a.H;
  if (blockIdx.z == 0) read_tile<D, TY, true>(a, b, h);
  else read_tile<D, TY, false>(a, b, h);
}

template <int D, int TY>
void launch_append(const AppendArgs& a, hipStream_t st) {
  if (a.T <= kFew) hipLaunchKernelGGL((kv4_append_kernel<D, TY, 1>), dim3(1, a.B * a.H), dim3(64), 0, st, a);
  else hipLaunchKernelGGL((kv4_append_kernel<D, TY, kTile / 64>), dim3(a.tiles, a.B * a.H), dim3(kTile), 0, st, a);
}

template <int D>
void launch_append(const AppendArgs& a, int ty, hipStream_t st) {
  if (ty == kKv4Bf16) launch_append<D, kKv4Bf16>(a, st);
  else if (ty == kKv4F32) launch_append<D, kKv4F32>(a, st);
  else launch_append<D, kKv4F16>(a, st);
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

// Whether two arrays (B, H) with these row strides may share an entry: exact
// for slices of one array, else by their extents.
bool may_meet(const int32_t* x, int64_t sx, const int32_t* y, int64_t sy, int B, int H) {
  const int64_t d = ((intptr_t)y - (intptr_t)x) / (int64_t)sizeof(int32_t);
  if (d >= (B - 1) * sx + H || -d >= (B - 1) * sy + H) return false;
  if (B == 1 || sx != sy || sx <= 0) return true;
  const int64_t r = (d % sx + sx) % sx;
  return r < H || sx - r < H;
}

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
  // Workgroups read a head's length and write another's new one: the same
  // array, or none of its entries.
  const bool in_place = new_lengths == lengths && (batch == 1 || new_stride_b == len_stride_b);
  if (batch > 1 && new_stride_b < num_kv_heads) return WGKV_ERR_ARG;
  if (!in_place && may_meet(lengths, len_stride_b, new_lengths, new_stride_b, batch, num_kv_heads)) return WGKV_ERR_ARG;
  AppendArgs a{};
  const int st = kv4_pages(&a.pg, num_pages, page_size, block_table, bt_stride_b, bt_stride_h, max_pages);
  if (st != WGKV_OK) return st;
  // 16-byte loads of the rows and accesses of the tiles
  const int64_t unit = dtype == kKv4F32 ? 3 : 7;
  if (((uintptr_t)key | (uintptr_t)value | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) return WGKV_ERR_UNSUPPORTED;
  if ((k_stride_b | k_stride_t | k_stride_h | v_stride_b | v_stride_t | v_stride_h) & unit) return WGKV_ERR_UNSUPPORTED;
  if (((uint64_t)k_stride_t | (uint64_t)v_stride_t) >> 32) return WGKV_ERR_UNSUPPORTED;
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
  // Several workgroups read a head's length and one writes the new one: in
  // place, the lengths are copied first too.
  const bool counted = a.tiles > 1 && (in_place || (g_mask && tokens > kCountsItself));
  if (counted && (!workspace || ((uintptr_t)workspace & 3) ||
                  workspace_bytes < wgkv_kv4_append_workspace_bytes(batch, num_kv_heads, tokens)))
    return WGKV_ERR_WORKSPACE;
  // keys and values are written by different lanes
  const int64_t pool = num_pages * (page_size / kKv4Tile) * kv4_tile_bytes(head_dim);
  const intptr_t apart = (intptr_t)v_cache - (intptr_t)k_cache;
  if (apart < pool && -apart < pool) return WGKV_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  if (counted) {
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
  // (both bases are 16-byte aligned, so they are whole elements apart)
  const int64_t apart = ((intptr_t)value - (intptr_t)key) / (dtype == kKv4F32 ? 4 : 2);
  if (kv4_rows_meet({batch, rows, num_kv_heads, 2}, {out_stride_b, out_stride_t, out_stride_h, apart}, head_dim))
    return WGKV_ERR_ARG;
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

extern "C" int wgkv_kv4_append_block(const void* args) {
  int64_t a[32];
  memcpy(a, args, sizeof a);
  if (!kv4_narrow(a, 8, 19, 23, 24, 25, 26, 27)) return WGKV_ERR_UNSUPPORTED;
  return wgkv_kv4_append((const void*)a[0], a[1], a[2], a[3], (const void*)a[4], a[5], a[6], a[7], (int32_t)a[8],
                         (const uint8_t*)a[9], a[10], a[11], (const int32_t*)a[12], a[13], (int32_t*)a[14], a[15],
                         (void*)a[16], (void*)a[17], a[18], (int32_t)a[19], (const int32_t*)a[20], a[21], a[22],
                         (int32_t)a[23], (int32_t)a[24], (int32_t)a[25], (int32_t)a[26], (int32_t)a[27],
                         (int32_t*)a[28], (void*)a[29], (size_t)a[30], (void*)a[31]);
}

extern "C" int wgkv_kv4_read_block(const void* args) {
  int64_t a[23];
  memcpy(a, args, sizeof a);
  if (!kv4_narrow(a, 3, 7, 17, 18, 19, 20, 21)) return WGKV_ERR_UNSUPPORTED;
  return wgkv_kv4_read((const void*)a[0], (const void*)a[1], a[2], (int32_t)a[3], (const int32_t*)a[4], a[5], a[6],
                       (int32_t)a[7], (const int32_t*)a[8], a[9], (const int32_t*)a[10], a[11], (void*)a[12],
                       (void*)a[13], a[14], a[15], a[16], (int32_t)a[17], (int32_t)a[18], (int32_t)a[19],
                       (int32_t)a[20], (int32_t)a[21], (void*)a[22]);
}
