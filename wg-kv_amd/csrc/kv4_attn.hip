// One token's attention over a paged cache held in 4 bits (gfx950).
//
//   z_t = scale * sum_g [ s_tg sum_{d in g} q_d (c_td - 7.5) + m_tg sum_{d in g} q_d ]
//   out_d = sum_t p_t s_tg (c_td - 7.5) + sum_t p_t m_tg,   p = softmax(z), g = d / 32
//
// Both products run on the matrix core over the codes themselves.  A code c
// becomes the bf16 number 128 + c by one v_and_or (its four bits are the low
// mantissa bits under the exponent of 128), and the offset of 135.5 is taken
// back in fp32.  The steps s differ per group of 32 d, so the 16 columns of
// an MFMA hold (group, query head) pairs -- 4 groups x 4 heads at D = 128,
// 2 x 8 at D = 64:
//   * keys times queries: column (g, h) holds q_h on the d of group g and
//     zeros elsewhere, so that one accumulator chain gives every group's sum
//     apart; a lane scales its own group's, and the groups are added with
//     DPP (tokens are rows, so the sums of a token end in one 16-lane row);
//   * values times probabilities: column (g, h) holds bf16(p_t s_tg), and of
//     its D outputs those of group g are kept.
// Without this the steps would have to be multiplied into every value: D
// more VALU operations per token than the two per column here.
//
// The layouts of kv4.h are these operands: K rows are A operands of 16
// tokens, C of that product (rows = tokens) is the B operand of the second
// one without any exchange between lanes (its k index runs over the same
// tokens 4q..4q+3 of two tiles), and V words are A operands (rows = d) of
// pairs of tokens.  Nothing goes through LDS but the merge of the waves.
//
// Work split: the heads' sequences, in units of 32 tokens, are one line that
// is cut into equal ranges, one per workgroup (so every workgroup has the
// same work whatever the lengths); a range may end one head and begin
// another.  Its waves take units in turn, the next unit's loads in flight.
// A head inside one range is written directly; otherwise the pieces' (max,
// sum, acc) go to the workspace and the head's last workgroup to arrive
// merges them, in the order of the sequence.
#include "kv4.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleSlack = 8.f;  // log2 units a running maximum may lag the scores
constexpr int kMaxBH = 2048;
constexpr int kMaxG = 8;
constexpr int kMaxSlots = 1024;  // workgroups of a launch
constexpr int kFlush = 32;       // units between two corrections of the code offset
constexpr uint32_t kCodeMask = 0x000f000fu, kCodeBase = 0x43004300u;  // 128 + c
constexpr float kOffset = 135.5f;                                     // (128 + c) - (c - 7.5)

struct AttnArgs {
  const uint16_t* q;
  int64_t q_sb, q_sh;
  const uint8_t* kc;
  const uint8_t* vc;
  Kv4Pages pg;
  const int32_t* len;
  int64_t len_sb;
  uint16_t* out;
  int64_t out_sb, out_sh;
  int B, Hkv, G;
  float scale_log2;
  // pieces: two slots per workgroup (the head it ends, the head it begins);
  // slot s, query head i: part_m[s*G+i], part_l[s*G+i], part_acc[(s*G+i)*D..]
  float *part_m, *part_l, *part_acc;
  int* counter;  // arrivals per (b, h), zero between calls
};

WGKV_DEVICE int tokens_of(const AttnArgs& a, int bh) {
  const int b = bh / a.Hkv, h = bh - b * a.Hkv;
  const int64_t cap = kv4_capacity(a.pg);
  const int64_t n = a.len[(int64_t)b * a.len_sb + h];
  return (int)(n < 0 ? 0 : n > cap ? cap : n);
}
WGKV_DEVICE int units_of(int tokens) { return (tokens + 31) >> 5; }

// The heads' units as a line, seen by one wave: lane j knows the units of
// heads [j*per, j*per+per).
struct Line {
  int per;
  int64_t excl;   // units before the lane's heads
  int64_t total;
};

WGKV_DEVICE int64_t wave_incl_scan64(int64_t v, int lane) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t u = __shfl_up(v, off, 64);
    if (lane >= off) v += u;
  }
  return v;
}

WGKV_DEVICE Line make_line(const AttnArgs& a, int lane) {
  const int BH = a.B * a.Hkv;
  Line ln;
  ln.per = (BH + 63) >> 6;
  int64_t n = 0;
  for (int i = 0; i < ln.per; ++i) {
    const int bh = lane * ln.per + i;
    if (bh < BH) n += units_of(tokens_of(a, bh));
  }
  const int64_t incl = wave_incl_scan64(n, lane);
  ln.excl = incl - n;
  ln.total = __shfl(incl, 63, 64);
  return ln;
}

// The head that holds unit `pos` < total of the line.
struct Head {
  int bh, tokens;
  int64_t start;  // its first unit on the line
};

WGKV_DEVICE Head find_head(const AttnArgs& a, const Line& ln, int64_t pos, int lane) {
  const int BH = a.B * a.Hkv;
  // the last lane that starts at or before pos (lanes without units start
  // where the next one does)
  const int o = 63 - __builtin_clzll(__builtin_amdgcn_ballot_w64(ln.excl <= pos));
  const int64_t base = __shfl(ln.excl, o, 64);
  const int bh = o * ln.per + lane;
  const int t = lane < ln.per && bh < BH ? tokens_of(a, bh) : 0;
  const int64_t incl = wave_incl_scan64(units_of(t), lane);
  const int64_t excl = base + incl - units_of(t);
  const int j = 63 - __builtin_clzll(__builtin_amdgcn_ballot_w64(lane < ln.per && bh < BH && excl <= pos));
  Head h;
  h.bh = o * ln.per + j;
  h.tokens = __builtin_amdgcn_readlane(t, j);
  h.start = __shfl(excl, j, 64);
  return h;
}

template <int CTRL>
WGKV_DEVICE float row_ror_add(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + CTRL, 0xf, 0xf, false));
}

// A dword of codes as four operand dwords (pairs of 128 + c).
WGKV_DEVICE void expand(uint32_t w, uint32_t* o) {
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = ((w >> (4 * i)) & kCodeMask) | kCodeBase;
}

template <int D, int NT, int NW>
__global__ __launch_bounds__(NW * 64) void kv4_attn_kernel(AttnArgs a) {
  constexpr int NG = D / kKv4Group;  // groups
  constexpr int HPT = 16 / NG;       // query heads per 16 columns
  constexpr int KS = D / 32;         // k-steps of the first product, dwords of a lane's K and V chunk per tile
  constexpr int MT = D / 16;         // row tiles of the second product
  constexpr int kThreads = NW * 64;
  typedef __attribute__((__vector_size__(KS * sizeof(uint32_t)))) uint32_t chunk_t;
  __shared__ float s_acc[NW][NT * HPT][D];
  __shared__ float s_ml[NW][2][NT * HPT];
  __shared__ int s_last;

  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, quad = lane >> 4;
  const int g = n / HPT, hh = n % HPT;
  const int G = a.G, BH = a.B * a.Hkv;
  const int w = blockIdx.x, n_wg = gridDim.x;

  // heads without tokens
  for (int bh = w; bh < BH; bh += n_wg) {
    if (tokens_of(a, bh) != 0) continue;
    const int b = bh / a.Hkv, h = bh - b * a.Hkv;
    for (int v = threadIdx.x; v < G * D; v += kThreads)
      a.out[(int64_t)b * a.out_sb + (int64_t)(h * G + v / D) * a.out_sh + v % D] = 0;
  }

  const Line ln = make_line(a, lane);
  // units per workgroup: whole rounds of the waves
  int64_t cp = (ln.total + n_wg - 1) / n_wg;
  cp = max((cp + NW - 1) / NW * NW, (int64_t)NW);
  int64_t pos = w * cp;
  const int64_t end = min(ln.total, pos + cp);

  while (pos < end) {
    const Head hd = find_head(a, ln, pos, lane);
    const int b = hd.bh / a.Hkv, h = hd.bh - b * a.Hkv;
    const int T = hd.tokens;
    const int u0 = (int)(pos - hd.start), u1 = (int)min((int64_t)units_of(T), end - hd.start);
    const int32_t* bt_row = a.pg.bt + (int64_t)b * a.pg.bt_sb + (int64_t)h * a.pg.bt_sh;
    const int last_tile = (T - 1) >> 4;

    // queries: column (g, head), k = 8 consecutive d; zeros off the column's group
    bf16x8_t qb[NT][KS];
    f32x4_t c0[NT];
    float qsum[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int qh = nt * HPT + hh;
      const uint16_t* qrow = a.q + (int64_t)b * a.q_sb + (int64_t)(h * G + min(qh, G - 1)) * a.q_sh;
      const bool mine = quad * NG / 4 == g && qh < G;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        u32x4_t v = *(const u32x4_t*)(qrow + quad * (D / 4) + i * 8);
        if (!mine) v = (u32x4_t){0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < 4; ++j) sum += bf16lo(v[j]) + bf16hi(v[j]);
        qb[nt][i] = __builtin_bit_cast(bf16x8_t, v);
      }
      sum += __shfl_xor(sum, 16, 64);  // over the quads: the column's group
      sum += __shfl_xor(sum, 32, 64);
      qsum[nt] = sum;
      const float c = -kOffset * sum;
      c0[nt] = (f32x4_t){c, c, c, c};
    }

    float m_run[NT], l_run[NT], corr[NT];
    f32x4_t acc[NT][MT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m_run[nt] = -INFINITY;
      l_run[nt] = corr[nt] = 0.f;
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[nt][j] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    }

    struct Unit {
      chunk_t k[2], v[2];
      u32x4_t ks[2], vs[2];
    };
    // page ids of the wave's next 32 units, two tiles each, one per lane
    int pages = 0;
    const auto load_pages = [&](int u) {
      const int tile = min(2 * (u + (lane >> 1) * NW) + (lane & 1), last_tile);
      const int pg = bt_row[tile >> a.pg.page_shift];
      pages = pg < 0 ? 0 : pg >= a.pg.num_pages ? (int)(a.pg.num_pages - 1) : pg;
    };
    const auto load_unit = [&](Unit& x, int u, int it) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int tile = min(2 * u + p, last_tile);
        const int pg = __builtin_amdgcn_readlane(pages, 2 * (it & 31) + p);
        const int64_t at = (((int64_t)pg << a.pg.page_shift) + (tile & ((1 << a.pg.page_shift) - 1))) * kv4_tile_bytes(D);
        const uint8_t* kt = a.kc + at;
        const uint8_t* vt = a.vc + at;
        x.k[p] = *(const chunk_t*)(kt + n * (D / 2) + quad * (D / 8));
        x.ks[p] = *(const u32x4_t*)(kt + kv4_scales_at(D) + (quad * NG + g) * 16);
        x.v[p] = *(const chunk_t*)(vt + quad * (2 * D) + n * (D / 8));
        x.vs[p] = *(const u32x4_t*)(vt + kv4_scales_at(D) + (quad * NG + g) * 16);
      }
    };
    // takes the offset's part out of the accumulators: they and the
    // correction grow with the tokens, their difference does not
    const auto flush = [&]() {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float c = corr[nt];
        c += __shfl_xor(c, 16, 64);
        c += __shfl_xor(c, 32, 64);
        corr[nt] = 0.f;
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[nt][j] += c;
      }
    };

    Unit cur;
    int u = u0 + wid, it = 0;
    if (u < u1) {
      load_pages(u);
      load_unit(cur, u, 0);
    }
    for (; u < u1; u += NW, ++it) {
      Unit nxt;
      const int un = u + NW;
      if (un < u1) {
        if (((it + 1) & 31) == 0) load_pages(un);
        load_unit(nxt, un, it + 1);
      }
      if (u * 32 + 32 > T) {  // rows past the end hold anything: step and middle 0
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (u * 32 + p * 16 + quad * 4 + i >= T) cur.ks[p][i] = cur.vs[p][i] = 0u;
      }
      f32x4_t z[NT][2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          u32x4_t o;
          uint32_t e[4];
          expand(cur.k[p][i], e);
          o = (u32x4_t){e[0], e[1], e[2], e[3]};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            z[nt][p] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, o), qb[nt][i],
                                                               i == 0 ? c0[nt] : z[nt][p], 0, 0, 0);
        }
      }
      u32x4_t pb[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float t[2][4];
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float x = fmaf(z[nt][p][i], bf16lo(cur.ks[p][i]), bf16hi(cur.ks[p][i]) * qsum[nt]);
            x = row_ror_add<8>(x);
            if constexpr (NG == 4) x = row_ror_add<4>(x);
            t[p][i] = x * a.scale_log2;
          }
        if (u * 32 + 32 > T) {
#pragma unroll
          for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (u * 32 + p * 16 + quad * 4 + i >= T) t[p][i] = -INFINITY;
        }
        const float top = fmaxf(fmaxf(fmaxf(t[0][0], t[0][1]), fmaxf(t[0][2], t[0][3])),
                                fmaxf(fmaxf(t[1][0], t[1][1]), fmaxf(t[1][2], t[1][3])));
        // The maximum of a column moves only when a score exceeds it by more
        // than the slack (p <= 2^slack); it is the same in the column's four
        // lanes, whose accumulators hold sums over all of them.
        if (__builtin_amdgcn_ballot_w64(top > m_run[nt] + kRescaleSlack)) {
          float mx = fmaxf(top, __shfl_xor(top, 16, 64));
          mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
          const float mn = fmaxf(m_run[nt], mx);
          const float alpha = mn == -INFINITY ? 1.f : fast_exp2(m_run[nt] - mn);
          m_run[nt] = mn;
          l_run[nt] *= alpha;
          corr[nt] *= alpha;
#pragma unroll
          for (int j = 0; j < MT; ++j) acc[nt][j] *= alpha;
        }
        uint32_t pk[4];
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int i0 = 2 * j, i1 = 2 * j + 1;
            const float p0 = fast_exp2(t[p][i0] - m_run[nt]), p1 = fast_exp2(t[p][i1] - m_run[nt]);
            l_run[nt] += p0 + p1;
            const uint32_t s0 = cur.vs[p][i0], s1 = cur.vs[p][i1];
            const uint32_t pr = pack_bf16x2(p0 * bf16lo(s0), p1 * bf16lo(s1));
            pk[2 * p + j] = pr;
            // with the rounded products: the offset must cancel exactly
            float c = fmaf(-kOffset, bf16lo(pr), corr[nt]);
            c = fmaf(-kOffset, bf16hi(pr), c);
            c = fmaf(p0, bf16hi(s0), c);
            corr[nt] = fmaf(p1, bf16hi(s1), c);
          }
        pb[nt] = (u32x4_t){pk[0], pk[1], pk[2], pk[3]};
      }
      // row tile j holds d = MT*r + j: code j%4 of the words of half j/4
#pragma unroll
      for (int hf = 0; hf < KS / 2; ++hf) {
        uint32_t e[4][4];  // (tile, pair), code
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int pr = 0; pr < 2; ++pr) expand(cur.v[p][pr * (KS / 2) + hf], e[2 * p + pr]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const u32x4_t o = (u32x4_t){e[0][c], e[1][c], e[2][c], e[3][c]};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            acc[nt][hf * 4 + c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                __builtin_bit_cast(bf16x8_t, o), __builtin_bit_cast(bf16x8_t, pb[nt]), acc[nt][hf * 4 + c], 0, 0, 0);
        }
      }
      if ((it & (kFlush - 1)) == kFlush - 1) flush();
      cur = nxt;
    }
    flush();

    // ---- merge the waves ---------------------------------------------------
    // lane (quad, g, hh) holds rows 4*quad + i of column (g, hh): d = MT *
    // (4*quad + i) + j, of the column's group where quad*NG/4 == g
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float l = l_run[nt];
      l += __shfl_xor(l, 16, 64);
      l += __shfl_xor(l, 32, 64);
      const int qh = nt * HPT + hh;
      if (quad * NG / 4 == g) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < MT; ++j) s_acc[wid][qh][MT * (4 * quad + i) + j] = acc[nt][j][i];
      }
      if (quad == 0 && g == 0) {
        s_ml[wid][0][qh] = m_run[nt];
        s_ml[wid][1][qh] = l;
      }
    }
    __syncthreads();

    const int64_t f = hd.start / cp;                                    // the head's first and
    const int64_t e = (hd.start + units_of(T) - 1) / cp;                // last workgroup
    const bool single = f == e;
    const int slot = 2 * w + (f == w ? 1 : 0);
    for (int v = threadIdx.x; v < G * D; v += kThreads) {
      const int i = v / D, d = v - i * D;
      float M = -INFINITY;
#pragma unroll
      for (int ww = 0; ww < NW; ++ww) M = fmaxf(M, s_ml[ww][0][i]);
      float L = 0.f, A = 0.f;
#pragma unroll
      for (int ww = 0; ww < NW; ++ww) {
        // a wave without a score has l = acc = 0; NaN scores leave m = -inf
        // and must come through
        const float mw = s_ml[ww][0][i];
        const float sc = mw == -INFINITY ? 1.f : fast_exp2(mw - M);
        L = fmaf(sc, s_ml[ww][1][i], L);
        A = fmaf(sc, s_acc[ww][i][d], A);
      }
      if (single) {
        a.out[(int64_t)b * a.out_sb + (int64_t)(h * G + i) * a.out_sh + d] = f32_to_bf16(A / L);
      } else {
        if (d == 0) {
          store_coherent(&a.part_m[(int64_t)slot * G + i], M);
          store_coherent(&a.part_l[(int64_t)slot * G + i], L);
        }
        store_coherent(&a.part_acc[((int64_t)slot * G + i) * D + d], A);
      }
    }
    if (!single) {
      // The last workgroup of the head to arrive merges.  Its loads see the
      // others' pieces without cache write-backs: the stores above are
      // device-coherent (written through to the point of coherence, where
      // the counter's atomics are performed too), vmcnt(0) waits until they
      // are acknowledged there, the barrier holds the arrival until every
      // wave has waited, and the merge's loads bypass this XCD's L2.
#if defined(__HIP_DEVICE_COMPILE__) && !defined(__gfx950__)
#error "the merge relies on gfx950 store acknowledgement and sc1 ordering"
#endif
      __atomic_signal_fence(__ATOMIC_SEQ_CST);
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
      __atomic_signal_fence(__ATOMIC_SEQ_CST);
      __syncthreads();
      if (threadIdx.x == 0) {
        const int prev = __hip_atomic_fetch_add(&a.counter[hd.bh], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const int last = prev == (int)(e - f);
        if (last) __hip_atomic_store(&a.counter[hd.bh], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_last = last;
      }
      __syncthreads();
      if (s_last) {
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        for (int v = threadIdx.x; v < G * D; v += kThreads) {
          const int i = v / D, d = v - i * D;
          float M = -INFINITY, L = 0.f, A = 0.f;
          for (int64_t x = f; x <= e; ++x) {
            const int64_t s = 2 * x + (x == f ? 1 : 0);
            const float m = load_coherent(&a.part_m[s * G + i]);
            const float l = load_coherent(&a.part_l[s * G + i]);
            const float ac = load_coherent(&a.part_acc[(s * G + i) * D + d]);
            const float mn = fmaxf(M, m);
            const float sa = M == -INFINITY ? 1.f : fast_exp2(M - mn), sb = m == -INFINITY ? 1.f : fast_exp2(m - mn);
            L = L * sa + l * sb;
            A = A * sa + ac * sb;
            M = mn;
          }
          a.out[(int64_t)b * a.out_sb + (int64_t)(h * G + i) * a.out_sh + d] = f32_to_bf16(A / L);
        }
      }
    }
    pos = hd.start + units_of(T);
    __syncthreads();  // LDS is free for the next head
  }
}

size_t part_floats(int G, int D) { return (size_t)2 * kMaxSlots * G * (2 + (size_t)D); }
constexpr size_t kCounterBytes = (size_t)kMaxBH * sizeof(int);

template <int D, int NT>
hipError_t launch(const AttnArgs& a, hipStream_t st) {
  constexpr int NW = 4, kPerCU = 3;
  // no more workgroups than the tables have rounds of units for
  const int64_t most = ((kv4_capacity(a.pg) + 31) / 32 * a.B * a.Hkv + NW - 1) / NW;
  const int slots = min(kMaxSlots, cu_count() * kPerCU);
  hipLaunchKernelGGL((kv4_attn_kernel<D, NT, NW>), dim3((unsigned)(most < slots ? most : slots)), dim3(NW * 64), 0, st, a);
  return hipGetLastError();
}

}  // namespace

extern "C" size_t wgkv_kv4_decode_workspace_bytes(int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim) {
  if (num_kv_heads <= 0 || num_q_heads < num_kv_heads || head_dim <= 0) return 0;
  return kCounterBytes + part_floats(num_q_heads / num_kv_heads, head_dim) * sizeof(float);
}

extern "C" int wgkv_kv4_decode_attn(
    const void* q, int64_t q_stride_b, int64_t q_stride_h,
    const void* k_cache, const void* v_cache, int64_t num_pages, int32_t page_size,
    const int32_t* cache_seqlens, int64_t sl_stride_b,
    const int32_t* block_table, int64_t bt_stride_b, int64_t bt_stride_h, int32_t max_pages,
    void* out, int64_t out_stride_b, int64_t out_stride_h,
    int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    float softmax_scale, void* workspace, size_t workspace_bytes, void* stream) {
  if (!q || !k_cache || !v_cache || !cache_seqlens || !out) return WGKV_ERR_ARG;
  if (batch <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads) return WGKV_ERR_ARG;
  const int G = num_q_heads / num_kv_heads;
  if ((int64_t)batch * num_kv_heads > kMaxBH || G > kMaxG) return WGKV_ERR_UNSUPPORTED;
  if (head_dim != 64 && head_dim != 128) return WGKV_ERR_UNSUPPORTED;
  AttnArgs a{};
  const int st = kv4_pages(&a.pg, num_pages, page_size, block_table, bt_stride_b, bt_stride_h, max_pages);
  if (st != WGKV_OK) return st;
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) return WGKV_ERR_UNSUPPORTED;
  if ((q_stride_b | q_stride_h) & 7) return WGKV_ERR_UNSUPPORTED;
  if (!workspace || ((uintptr_t)workspace & 15) ||
      workspace_bytes < wgkv_kv4_decode_workspace_bytes(num_q_heads, num_kv_heads, head_dim))
    return WGKV_ERR_WORKSPACE;
  a.q = (const uint16_t*)q;
  a.q_sb = q_stride_b;
  a.q_sh = q_stride_h;
  a.kc = (const uint8_t*)k_cache;
  a.vc = (const uint8_t*)v_cache;
  a.len = cache_seqlens;
  a.len_sb = sl_stride_b;
  a.out = (uint16_t*)out;
  a.out_sb = out_stride_b;
  a.out_sh = out_stride_h;
  a.B = batch;
  a.Hkv = num_kv_heads;
  a.G = G;
  a.scale_log2 = softmax_scale * kLog2e;
  a.counter = (int*)workspace;
  const size_t slots = (size_t)2 * kMaxSlots * G;
  a.part_m = (float*)((char*)workspace + kCounterBytes);
  a.part_l = a.part_m + slots;
  a.part_acc = a.part_l + slots;
  hipStream_t s = (hipStream_t)stream;
  const hipError_t e = head_dim == 64 ? launch<64, 1>(a, s) : G <= 4 ? launch<128, 1>(a, s) : launch<128, 2>(a, s);
  return e == hipSuccess ? WGKV_OK : WGKV_ERR_HIP;
}
