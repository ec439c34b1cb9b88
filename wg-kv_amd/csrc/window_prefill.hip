// Attention of a packed batch of prompts with a sliding window and first
// tokens that stay visible (gfx950).
//
// Sequence b holds the query rows cu_q[b] .. cu_q[b+1] - 1 and the keys
// cu_k[b] .. cu_k[b+1] - 1 of the packed tensors; with nq rows and nk keys its
// row i is at position p = i + nk - nq and sees key j iff
//   j <= p  and  (j > p - window  or  j < sinks),
// under softmax(q . k * scale).  Rows that see nothing (p < 0) give zeros.
// Query head hq uses KV head hq / G.
//
// Work item = (64 rows of a sequence, KV head, group of HPW of its G query
// heads) for a workgroup of 2 * HPW waves; a wave serves 32 rows of one head.
// The item's keys are the `first` tokens below the band and the band
// [lo, last row's position] that the rows' windows reach, counted through as
// one list and cut into tiles of 64, so that a few first tokens cost their
// share of a tile and not one of their own.  Tiles go from memory straight
// into LDS, one tile ahead of the arithmetic (global_load_lds_dwordx4), and
// serve all heads of the group.  S^T = K Q^T on v_mfma_f32_16x16x32_bf16
// leaves each lane 16 scores of a query row, which are the B operand of
// O^T += V^T P^T; V^T comes by LDS transpose reads.  Softmax is in the log2
// domain, fp32, with a running maximum that moves only when a score exceeds it
// by more than 8; probabilities are rounded to bf16 for the products, and
// their sums are taken of the rounded values.  Only the tiles at the two ends
// of a row's window are masked; a wave passes over a tile none of its rows sees.
//
// A masked probability is 0, and 0 times a key's value that is not finite is
// NaN: rows whose result is not finite are worked out once more, key by key
// (exact_rows).
#include <string.h>

#include "kv4.h"

namespace {

constexpr int kBlk = 64;      // query rows per item and keys per tile
constexpr int kMaxSeqs = 2048;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.f;  // log2 units a row maximum may lag its scores

WGKV_DEVICE float fmax_ieee(float x, float y) { return __builtin_elementwise_maximum(x, y); }
WGKV_DEVICE float xor16_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmax_ieee(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
WGKV_DEVICE float xor32_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmax_ieee(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

typedef short v4i16_t __attribute__((ext_vector_type(4)));

// The 16 bytes at g go to LDS at lds + 16 * lane (lds the same in every lane).
WGKV_DEVICE void lds_dma16(const uint16_t* g, uint16_t* lds) { __builtin_amdgcn_global_load_lds(g, lds, 16, 0, 0); }

WGKV_DEVICE v4i16_t lds_read_tr16(const uint16_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4i16_t __attribute__((address_space(3)))*)(p));
}

// Places of a row's 16-byte slices in an unpadded LDS tile: slice c of row r
// is at c ^ swz(r).  16 consecutive rows of a K operand, and the 8 rows of a
// V transpose read, then lie on different banks.
template <int D>
WGKV_DEVICE int swz_k(int row) { return D == 128 ? (row & 15) : ((row >> 1) & 7); }
template <int D>
WGKV_DEVICE int swz_v(int row) { return D == 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3); }

struct WindowArgs {
  const uint16_t* q;
  int64_t q_sn, q_sh;
  const uint16_t* k;
  int64_t k_sn, k_sh;
  const uint16_t* v;
  int64_t v_sn, v_sh;
  uint16_t* out;
  int64_t o_sn, o_sh;
  const int32_t* cu_q;
  const int32_t* cu_k;
  int B, N, Nk, Hkv, G;
  int window, sinks;
  float scale_log2;
  uint32_t q_and, q_xor;
  int clear_rest;  // rows of no sequence get zeros
};

WGKV_DEVICE int clamp_to(int x, int hi) { return min(max(x, 0), hi); }

// The keys of an item as one list: entry x is key x for x < first, else key x + shift.
struct Keys {
  int first, shift, count;
  WGKV_DEVICE int key(int x) const { return x < first ? x : x + shift; }
};

// The rows of one wave, key by key, for results that are not finite.  32
// lanes of a wave would idle in a matrix of one row, so a lane takes D/64
// values of d and the wave one row.
template <int D>
WGKV_DEVICE void exact_row(const WindowArgs& a, const uint16_t* q, const uint16_t* k,
                                                    const uint16_t* v, int p, uint16_t* out, int lane) {
  constexpr int C = D / 64;
  float qf[C], acc[C], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const uint32_t w = ((uint32_t)q[lane * C + c] & (a.q_and & 0xffffu)) ^ (a.q_xor & 0xffffu);
    qf[c] = __uint_as_float(w << 16);
    acc[c] = 0.f;
  }
  const int lo = max(0, p - a.window + 1), first = min(a.sinks, lo);
  for (int x = 0; x < first + p - lo + 1; ++x) {
    const int64_t j = x < first ? x : x - first + lo;
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) s = fmaf(qf[c], __uint_as_float((uint32_t)k[j * a.k_sn + lane * C + c] << 16), s);
    s = wave_sum(s) * a.scale_log2;
    if (s == -INFINITY) continue;
    const float mn = s > m ? s : m;
    const float was = m == -INFINITY ? 0.f : fast_exp2(m - mn), e = fast_exp2(s - mn);
    const float w = round_to_bf16(e);
    l = l * was + w;
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] = acc[c] * was + w * __uint_as_float((uint32_t)v[j * a.v_sn + lane * C + c] << 16);
    m = mn;
    if (l != l) break;  // nothing can change any more
  }
  const float inv = 1.f / l;
#pragma unroll
  for (int c = 0; c < C; ++c) out[lane * C + c] = l == 0.f ? 0 : f32_to_bf16(acc[c] * inv);
}

template <int D, int HPW>
__global__ __launch_bounds__(128 * HPW) void window_prefill_kernel(WindowArgs a) {
  constexpr int NT = 128 * HPW;
  constexpr int KS = D / 32;       // k-steps over head_dim
  constexpr int DT = D / 16;       // 16-wide d tiles
  constexpr int CH = D / 8;        // 16-byte slices per row
  constexpr int NW = 2 * HPW;
  constexpr int RPB = 64 / CH;     // key rows of 1 KB of LDS, one load instruction of a wave
  constexpr int NBLK = kBlk / RPB;
  // with four heads only the older wave of each SIMD loads: it reaches the
  // tile's barrier first
  constexpr int NL = HPW == 4 ? NW / 2 : NW;
  constexpr int KPT = NBLK / NL;
  static_assert(NBLK % NL == 0, "every loading wave loads whole 1 KB blocks");
  // four LDS objects: loads into one buffer then provably leave the other alone
  __shared__ __attribute__((aligned(16))) uint16_t sK0[kBlk * D];
  __shared__ __attribute__((aligned(16))) uint16_t sK1[kBlk * D];
  __shared__ __attribute__((aligned(16))) uint16_t sV0[kBlk * D];
  __shared__ __attribute__((aligned(16))) uint16_t sV1[kBlk * D];
  __shared__ int s_blocks[kMaxSeqs + 1];  // row blocks of the sequences before
  __shared__ int s_wave[NW];

  const int t = threadIdx.x;
  const int lane = t & 63, wid = __builtin_amdgcn_readfirstlane(t >> 6);
  const int n = lane & 15, g = lane >> 4;

  {
    const int per = (a.B + NT - 1) / NT, b0 = min(a.B, t * per), b1 = min(a.B, b0 + per);
    int mine = 0;
    for (int b = b0; b < b1; ++b)
      mine += (max(clamp_to(a.cu_q[b + 1], a.N) - clamp_to(a.cu_q[b], a.N), 0) + kBlk - 1) / kBlk;
    const int incl = wave_incl_scan(mine, lane);
    if (lane == 63) s_wave[wid] = incl;
    __syncthreads();
    int run = incl - mine;
    for (int i = 0; i < NW; ++i) run += i < wid ? s_wave[i] : 0;
    for (int b = b0; b < b1; ++b) {
      s_blocks[b] = run;
      run += (max(clamp_to(a.cu_q[b + 1], a.N) - clamp_to(a.cu_q[b], a.N), 0) + kBlk - 1) / kBlk;
      if (b == a.B - 1) s_blocks[a.B] = run;
    }
    __syncthreads();
  }
  if (a.clear_rest) {
    const int head = clamp_to(a.cu_q[0], a.N), tail = max(clamp_to(a.cu_q[a.B], a.N), head);
    const int64_t pieces = (int64_t)(head + a.N - tail) * a.Hkv * a.G * CH;
    for (int64_t i = (int64_t)blockIdx.x * NT + t; i < pieces; i += (int64_t)gridDim.x * NT) {
      const int64_t r = i / CH, x = r / (a.Hkv * a.G);
      *(u32x4_t*)(a.out + (x < head ? x : x - head + tail) * a.o_sn + (r - x * (a.Hkv * a.G)) * a.o_sh + (i - r * CH) * 8) =
          (u32x4_t){0u, 0u, 0u, 0u};
    }
  }

  // Per-lane LDS element offsets of the operands
  int koff[KS];
#pragma unroll
  for (int j = 0; j < KS; ++j) koff[j] = n * D + ((j * 4 + g) ^ swz_k<D>(n)) * 8;
  const int vrow = 4 * g + (n >> 2);
  int voff[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
    voff[dt] = vrow * D + ((2 * dt + ((n & 3) >> 1)) ^ swz_v<D>(vrow)) * 8 + (n & 1) * 4;

  // Items from the last row block to the first -- later blocks of a sequence
  // see no fewer keys --, heads innermost: workgroups are dealt to the XCDs in
  // turn, so with 8 KV heads each XCD's L2 serves one head's keys.  A
  // workgroup takes items from alternate ends of its rounds.
  const int per_block = a.Hkv * (a.G / HPW);
  const int64_t items = (int64_t)s_blocks[a.B] * per_block;
  for (int round = 0;; ++round) {
    const int64_t item = (int64_t)round * gridDim.x + ((round & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
    if (item >= items) break;
    if (round) __syncthreads();  // every wave is done with the previous item's tiles
    const int blk = s_blocks[a.B] - 1 - (int)(item / per_block), rest = (int)(item % per_block);
    int b = 0;
    for (int hi = a.B - 1; b < hi;) {  // the last sequence that begins at or before the block
      const int mid = (b + hi + 1) >> 1;
      if (s_blocks[mid] <= blk) b = mid; else hi = mid - 1;
    }
    const int h = rest % a.Hkv, hq = h * a.G + (rest / a.Hkv) * HPW + (wid >> 1);
    const int q0 = clamp_to(a.cu_q[b], a.N), nq = max(clamp_to(a.cu_q[b + 1], a.N) - q0, 0);
    const int k0 = clamp_to(a.cu_k[b], a.Nk), nk = max(clamp_to(a.cu_k[b + 1], a.Nk) - k0, 0);
    const int r_blk = (blk - s_blocks[b]) * kBlk;             // the item's rows in the sequence
    const int n_rows = min(kBlk, nq - r_blk);
    const int p_blk = r_blk + nk - nq;                         // the first row's position
    const int r0 = r_blk + (wid & 1) * 32, p0 = p_blk + (wid & 1) * 32;  // the wave's
    const int p_last = p_blk + n_rows - 1;
    Keys ks = {0, 0, 0};
    if (p_last >= 0) {
      const int lo = max(0, p_blk - a.window + 1);
      ks.first = min(a.sinks, lo);
      ks.shift = lo - ks.first;
      ks.count = ks.first + p_last - lo + 1;
    }
    const int ntiles = (ks.count + kBlk - 1) / kBlk;
    const uint16_t* kbase = a.k + (int64_t)k0 * a.k_sn + (int64_t)h * a.k_sh;
    const uint16_t* vbase = a.v + (int64_t)k0 * a.v_sn + (int64_t)h * a.v_sh;

    // queries as the B operand: lane (row n, slice g) of row tile rt, k-step j
    bf16x8_t qb[2][KS];
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
      const int s = min(r0 + rt * 16 + n, nq - 1);
      const uint16_t* qrow = a.q + (int64_t)(q0 + s) * a.q_sn + (int64_t)hq * a.q_sh;
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        const u32x4_t w = *(const u32x4_t*)(qrow + (j * 4 + g) * 8);
        qb[rt][j] = __builtin_bit_cast(bf16x8_t, (w & a.q_and) ^ a.q_xor);
      }
    }
    float m_run[2] = {-INFINITY, -INFINITY};
    f32x4_t lsum[2] = {(f32x4_t){0.f, 0.f, 0.f, 0.f}, (f32x4_t){0.f, 0.f, 0.f, 0.f}};
    const bf16x8_t ones = __builtin_bit_cast(bf16x8_t, (u32x4_t){0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
    f32x4_t o[DT][2];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int rt = 0; rt < 2; ++rt) o[dt][rt] = (f32x4_t){0.f, 0.f, 0.f, 0.f};

    // Loading wave w fills the 1 KB blocks w, w + NL, ...: in block q lane i
    // loads slice (i % CH) ^ swz of list entry q * RPB + i / CH.
    auto tile_load = [&](int tl, uint16_t* dK, uint16_t* dV) __attribute__((always_inline)) {
      if (wid >= NL) return;
#pragma unroll
      for (int i = 0; i < KPT; ++i) {
        const int row = (wid + i * NL) * RPB + lane / CH, blk1k = (wid + i * NL) * 512;
        const int64_t j = ks.key(min(tl * kBlk + row, ks.count - 1));
        lds_dma16(kbase + j * a.k_sn + ((lane % CH) ^ swz_k<D>(row)) * 8, dK + blk1k);
        lds_dma16(vbase + j * a.v_sn + ((lane % CH) ^ swz_v<D>(row)) * 8, dV + blk1k);
      }
    };
    if (ntiles > 0) tile_load(0, sK0, sV0);

    auto step = [&](int tile, const uint16_t* sK, const uint16_t* sV, uint16_t* nK,
                    uint16_t* nV) __attribute__((always_inline)) {
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's loads of the tile have landed
      __syncthreads();
      if (tile + 1 < ntiles) tile_load(tile + 1, nK, nV);
      const int x0 = tile * kBlk, x1 = min(x0 + kBlk, ks.count) - 1;  // the tile's list entries
      // the wave's rows p0 .. p0 + 31 see something of it?  (the list ascends,
      // so its band part is [max(x0, first), x1])
      const bool firsts = x0 < ks.first;
      const int band_lo = max(x0, ks.first) + ks.shift, band_hi = x1 + ks.shift;
      const bool band = x1 >= ks.first && band_lo <= p0 + 31 && p0 - band_hi < a.window;
      if (!firsts && !band) return;
      f32x4_t sc[4][2];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) sc[kt][rt] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
      bf16x8_t kf[2][4];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
        kf[0][kt] = __builtin_bit_cast(bf16x8_t, *(const u32x4_t*)(&sK[kt * 16 * D + koff[0]]));
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        if (j + 1 < KS)
#pragma unroll
          for (int kt = 0; kt < 4; ++kt)
            kf[(j + 1) & 1][kt] = __builtin_bit_cast(bf16x8_t, *(const u32x4_t*)(&sK[kt * 16 * D + koff[j + 1]]));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int rt = 0; rt < 2; ++rt)
            sc[kt][rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[j & 1][kt], qb[rt][j], sc[kt][rt], 0, 0, 0);
      }
      // all 64 keys visible to all 32 rows?
      const bool full = x0 + kBlk <= ks.count && p0 >= 0 &&
                        (x1 < ks.first || (band_hi <= p0 && p0 + 31 - band_lo < a.window));
      float mxs[2];
#pragma unroll
      for (int rt = 0; rt < 2; ++rt) {
        if (!full) {
          const int p = p0 + rt * 16 + n;
#pragma unroll
          for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int x = x0 + kt * 16 + 4 * g + i, j = ks.key(x);
              const bool see = x < ks.count && j <= p && (p - j < a.window || j < a.sinks);
              sc[kt][rt][i] = see ? sc[kt][rt][i] : -INFINITY;
            }
        }
        float mx = sc[0][rt][0];
#pragma unroll
        for (int e = 1; e < 16; ++e) mx = fmax_ieee(mx, sc[e >> 2][rt][e & 3]);
        mxs[rt] = mx * a.scale_log2;
      }
      if (__builtin_amdgcn_ballot_w64(mxs[0] > m_run[0] + kSlack || mxs[1] > m_run[1] + kSlack) != 0) {
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
          const float mx = xor32_max(xor16_max(mxs[rt]));
          const float mnew = mx > m_run[rt] + kSlack ? mx : m_run[rt];
          const float alpha = mnew == m_run[rt] ? 1.f : fast_exp2(m_run[rt] - mnew);
          m_run[rt] = mnew;
          lsum[rt] *= alpha;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) o[dt][rt] *= alpha;
        }
      }
      bf16x8_t pb[2][2];
#pragma unroll
      for (int rt = 0; rt < 2; ++rt) {
        const float mref = m_run[rt] == -INFINITY ? 0.f : m_run[rt];
        uint32_t pw[8];
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int i = 0; i < 4; i += 2)
            pw[kt * 2 + i / 2] = pack_bf16x2(fast_exp2(fmaf(sc[kt][rt][i], a.scale_log2, -mref)),
                                             fast_exp2(fmaf(sc[kt][rt][i + 1], a.scale_log2, -mref)));
#pragma unroll
        for (int s = 0; s < 2; ++s)
          pb[rt][s] = __builtin_bit_cast(bf16x8_t, (u32x4_t){pw[4 * s], pw[4 * s + 1], pw[4 * s + 2], pw[4 * s + 3]});
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const uint16_t* vrd = sV + voff[dt] + s * 32 * D;
          const v4i16_t lo = lds_read_tr16(vrd);
          const v4i16_t hi = lds_read_tr16(vrd + 16 * D);
          const bf16x8_t vf = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
          for (int rt = 0; rt < 2; ++rt)
            o[dt][rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pb[rt][s], o[dt][rt], 0, 0, 0);
        }
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) lsum[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pb[rt][s], lsum[rt], 0, 0, 0);
      }
    };
    for (int tile = 0; tile < ntiles; tile += 2) {
      step(tile, sK0, sV0, sK1, sV1);
      if (tile + 1 < ntiles) step(tile + 1, sK1, sV1, sK0, sV0);
    }

    // lane holds O[row rt*16+n][dt*16 + 4g + i]
    uint32_t again = 0;  // rows with a value that is not finite
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
      float bad = lsum[rt][0] * 0.f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) bad += o[dt][rt][i] * 0.f;
      const uint64_t y = __builtin_amdgcn_ballot_w64(r0 + rt * 16 + n < nq && bad != bad);
      again |= (uint32_t)((y | y >> 16 | y >> 32 | y >> 48) & 0xffff) << (16 * rt);
    }
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
      const float l = lsum[rt][0];
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int s = r0 + rt * 16 + n;
      if (s >= nq || (again >> (rt * 16 + n) & 1)) continue;
      uint16_t* orow = a.out + (int64_t)(q0 + s) * a.o_sn + (int64_t)hq * a.o_sh;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const uint32_t w0 = pack_bf16x2(o[dt][rt][0] * inv, o[dt][rt][1] * inv);
        const uint32_t w1 = pack_bf16x2(o[dt][rt][2] * inv, o[dt][rt][3] * inv);
        *(uint64_t*)(orow + dt * 16 + 4 * g) = (uint64_t)w0 | ((uint64_t)w1 << 32);
      }
    }
    while (again) {
      const int row = r0 + __builtin_ctz(again);
      again &= again - 1;
      const int64_t at = q0 + row;
      exact_row<D>(a, a.q + at * a.q_sn + (int64_t)hq * a.q_sh, kbase, vbase, row + nk - nq,
                   a.out + at * a.o_sn + (int64_t)hq * a.o_sh, lane);
    }
  }
}

// As many workgroups as are resident at once, at most one per item.
template <int D, int HPW>
hipError_t launch(const WindowArgs& a, hipStream_t st) {
  static int per_cu = 0;
  if (per_cu == 0) {
    int nb = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&nb, window_prefill_kernel<D, HPW>, 128 * HPW, 0) != hipSuccess ||
        nb <= 0)
      nb = 1;
    per_cu = nb;
  }
  const int64_t items = ((int64_t)a.N / kBlk + a.B) * a.Hkv * (a.G / HPW);
  const int64_t most = (int64_t)per_cu * cu_count();
  hipLaunchKernelGGL((window_prefill_kernel<D, HPW>), dim3((unsigned)(items < most ? items : most)), dim3(128 * HPW), 0,
                     st, a);
  return hipGetLastError();
}

// Query heads per workgroup: as many of 4, 2, 1 as divide G, halved while the
// smaller workgroups would still get a CU each (a short call's time is its
// longest item's, and a SIMD with one wave runs a tile sooner).
int heads_per_wg(const WindowArgs& a) {
  int h = 4;
  while (a.G % h) h >>= 1;
  while (h > 1 && ((int64_t)a.N / kBlk + a.B) * a.Hkv * (a.G / h) * 2 <= cu_count()) h >>= 1;
  return h;
}

template <int D>
hipError_t launch_heads(const WindowArgs& a, hipStream_t st) {
  const int h = heads_per_wg(a);
  return h == 4 ? launch<D, 4>(a, st) : h == 2 ? launch<D, 2>(a, st) : launch<D, 1>(a, st);
}

}  // namespace

extern "C" int wgkv_sink_window_attn(
    const void* q, int64_t q_stride_n, int64_t q_stride_h,
    const void* k, int64_t k_stride_n, int64_t k_stride_h,
    const void* v, int64_t v_stride_n, int64_t v_stride_h,
    void* out, int64_t out_stride_n, int64_t out_stride_h,
    const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int32_t batch, int32_t num_rows, int32_t num_keys,
    int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t window, int32_t num_sinks, float softmax_scale, int32_t clear_rest, void* stream) {
  if (batch <= 0 || num_rows < 0 || num_keys < 0 || num_kv_heads <= 0 || num_q_heads <= 0) return WGKV_ERR_ARG;
  if (num_q_heads % num_kv_heads || window < 1 || num_sinks < 0) return WGKV_ERR_ARG;
  if (num_rows == 0) return WGKV_OK;
  if (!q || !out || !cu_seqlens_q || !cu_seqlens_k || (num_keys && (!k || !v))) return WGKV_ERR_ARG;
  const int G = num_q_heads / num_kv_heads;
  if (G > 8 || (head_dim != 64 && head_dim != 128) || batch > kMaxSeqs) return WGKV_ERR_UNSUPPORTED;
  if (num_rows > (1 << 30) || num_keys > (1 << 30)) return WGKV_ERR_UNSUPPORTED;  // positions and tiles are 32-bit
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) return WGKV_ERR_UNSUPPORTED;
  if ((q_stride_n | q_stride_h | k_stride_n | k_stride_h | v_stride_n | v_stride_h | out_stride_n | out_stride_h) & 7)
    return WGKV_ERR_UNSUPPORTED;
  if (kv4_rows_meet({num_rows, num_q_heads, 1, 1}, {out_stride_n, out_stride_h, 0, 0}, head_dim)) return WGKV_ERR_ARG;
  WindowArgs a{};
  a.q = (const uint16_t*)q;
  a.q_sn = q_stride_n;
  a.q_sh = q_stride_h;
  a.k = (const uint16_t*)k;
  a.k_sn = k_stride_n;
  a.k_sh = k_stride_h;
  a.v = (const uint16_t*)v;
  a.v_sn = v_stride_n;
  a.v_sh = v_stride_h;
  a.out = (uint16_t*)out;
  a.o_sn = out_stride_n;
  a.o_sh = out_stride_h;
  a.cu_q = cu_seqlens_q;
  a.cu_k = cu_seqlens_k;
  a.B = batch;
  a.N = num_rows;
  a.Nk = num_keys;
  a.Hkv = num_kv_heads;
  a.G = G;
  a.window = window;
  a.sinks = num_sinks;
  // a negative scale negates the queries, and a scale of 0 clears them: masked
  // scores are -inf, and -inf * 0 is not a number
  a.scale_log2 = softmax_scale == 0.f ? 1.f : fabsf(softmax_scale) * kLog2e;
  a.q_and = softmax_scale == 0.f ? 0u : ~0u;
  a.q_xor = softmax_scale < 0.f ? 0x80008000u : 0u;
  a.clear_rest = clear_rest;
  const hipError_t e =
      head_dim == 128 ? launch_heads<128>(a, (hipStream_t)stream) : launch_heads<64>(a, (hipStream_t)stream);
  return e == hipSuccess ? WGKV_OK : WGKV_ERR_HIP;
}

extern "C" int wgkv_sink_window_attn_block(const void* args) {
  int64_t a[25];
  memcpy(a, args, sizeof a);
  if (!kv4_narrow(a, 14, 15, 16, 17, 18, 19, 20, 21, 23)) return WGKV_ERR_UNSUPPORTED;
  double scale;
  memcpy(&scale, &a[22], sizeof scale);
  return wgkv_sink_window_attn((const void*)a[0], a[1], a[2], (const void*)a[3], a[4], a[5], (const void*)a[6], a[7],
                               a[8], (void*)a[9], a[10], a[11], (const int32_t*)a[12], (const int32_t*)a[13],
                               (int32_t)a[14], (int32_t)a[15], (int32_t)a[16], (int32_t)a[17], (int32_t)a[18],
                               (int32_t)a[19], (int32_t)a[20], (int32_t)a[21], (float)scale, (int32_t)a[23],
                               (void*)a[24]);
}
