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
// Without this the steps would have to be multiplied into every value: 2 D
// VALU operations per token instead of two per column.
//
// The layouts of kv4.h are these operands: K rows are A operands of 16
// tokens, C of that product (rows = tokens) is the B operand of the second
// one without any exchange between lanes (its k index runs over the same
// tokens 4q..4q+3 of two tiles), and V words are A operands (rows = d) of
// pairs of tokens.  Nothing goes through LDS but the merge of the waves.
//
// Work split: the heads' sequences, in units of 64 tokens, are one line that
// is cut into ranges that differ by one unit, one per wave (so all have the
// same work whatever the lengths; 8 waves per CU, in one workgroup); a range
// may end one head and begin another.  Half a unit is worked on while the next half's tiles
// are in flight, and what a new head needs is asked for before that.  A head
// inside one range is written by its wave, one inside a workgroup after its
// waves' pieces (max, sum, acc) met in LDS; otherwise the workgroups' pieces
// go to the workspace and the head's last workgroup to arrive merges them, in
// the order of the sequence, whichever that is.
//
// Bound by reads where the caches are long: 8 sequences of 128K, 2-60 %
// admitted (424 MB), 73 us, 5.8 TB/s (loads of this pattern alone 6.3); 8
// heads of 400K tokens (513 MB) 86 us, 6.0 TB/s, vector instructions half of
// the time.  With 5 to 8 query heads per KV head at D = 128 the first of these
// takes 113 us: two column tiles, half the waves, and one group of threads to
// merge a head's pieces, which also costs lines of one or two heads (one of
// 400K tokens: 31 us, with 8 query heads 76; 10 at the rate of its reads).
// Short ones are latency: 8 heads of ~1300 tokens 12 us in a graph,
// of which 2.4 pass before the first tile, 2 for a unit, 1.5 in the
// workgroup's merge and 4.5 between workgroups.
#include <string.h>

#include "kv4.h"

namespace {

typedef __attribute__((__vector_size__(2 * sizeof(uint32_t)))) uint32_t u32x2_t;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleSlack = 8.f;  // log2 units a running maximum may lag the scores
// Where a running maximum begins.  Finite: a score of -inf (a finite one may
// fall there too, by its sum or its scale) then weighs exp2(-inf) = 0 and a
// piece that saw no other weighs 0 against one that did, without a case of
// their own; from -inf both would be exp2(-inf + inf), not a number.
constexpr float kNoMax = -3.402823466e38f;
constexpr int kMaxBH = 2048;
constexpr int kMaxG = 8;
constexpr int kMaxSlots = 512;  // workgroups of a launch
constexpr int kUnit = 64;        // tokens
constexpr int kFewest = 4;       // units of a workgroup before more workgroups have none
constexpr int kFlush = 16;       // units between two corrections of the code offset
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
  int g_shift;        // G <= 1 << g_shift
  int cap;            // tokens a head's table row has pages for
  uint32_t hkv_inv;   // ceil(2^32 / Hkv), 0 for 1: see sequence_of
  float scale_log2;         // |softmax_scale| * log2(e)
  uint32_t q_and, q_xor;    // its sign (and a scale of 0) is put into the queries
  // pieces: two slots per workgroup (the head it ends, the head it begins);
  // slot s, query head i: (max, sum) at part_ml[(s*G+i)*2], part_acc[(s*G+i)*D..]
  float *part_ml, *part_acc;
  int* counter;  // arrivals per (b, h), zero between calls
};

// bh / Hkv by a multiplication: exact while bh * Hkv < 2^32 (both are at most
// 2048).  A division's code costs more than its time: instructions that run
// once come cold from memory.
WGKV_DEVICE int sequence_of(const AttnArgs& a, int bh) {
  return a.hkv_inv ? (int)__umulhi((uint32_t)bh, a.hkv_inv) : bh;
}

WGKV_DEVICE int tokens_of(const AttnArgs& a, int bh) {
  const int b = sequence_of(a, bh), h = bh - b * a.Hkv;
  return min(max(a.len[(int64_t)b * a.len_sb + h], 0), a.cap);
}
WGKV_DEVICE int units_of(int tokens) { return (tokens + kUnit - 1) / kUnit; }

// Inclusive prefix sum over the wave in DPP steps (no LDS round trips):
// row_shr 1, 2, 4, 8 within 16 lanes, then the rows' ends broadcast onwards.
WGKV_DEVICE int wave_scan_dpp(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast31 into rows 2 and 3
  return v;
}

// The heads' units as a line, seen by one wave: lane j knows the units of
// heads [j*per, j*per+per).  kPer bounds per: 1, 4 (then the lane keeps its
// heads' tokens) or 32 (then they are read again where they are needed).
template <int kPer>
struct Line {
  static constexpr int kKept = kPer <= 4 ? kPer : 1;
  int per;
  int tokens[kKept];  // of the lane's heads, 0 past the last one
  int excl;           // units before the lane's heads
  int total;
};

// Tokens of heads first..first+kN-1, their loads in flight together.
template <int kN>
WGKV_DEVICE void tokens_of_run(const AttnArgs& a, int first, int n, int (&t)[kN]) {
  const int BH = a.B * a.Hkv;
#pragma unroll
  for (int k = 0; k < kN; ++k) t[k] = tokens_of(a, min(first + k, BH - 1));
#pragma unroll
  for (int k = 0; k < kN; ++k)
    if (k >= n || first + k >= BH) t[k] = 0;
}

template <int kPer>
WGKV_DEVICE Line<kPer> make_line(const AttnArgs& a, int lane) {
  Line<kPer> ln;
  ln.per = kPer == 1 ? 1 : (a.B * a.Hkv + 63) >> 6;
  int n = 0;
  if constexpr (kPer <= 4) {
    tokens_of_run(a, lane * ln.per, ln.per, ln.tokens);
#pragma unroll
    for (int k = 0; k < kPer; ++k) n += units_of(ln.tokens[k]);
  } else {
#pragma unroll 1
    for (int i = 0; i < ln.per; i += 4) {
      int t[4];
      tokens_of_run(a, lane * ln.per + i, ln.per - i, t);
#pragma unroll
      for (int k = 0; k < 4; ++k) n += units_of(t[k]);
    }
  }
  const int incl = wave_scan_dpp(n);
  ln.excl = incl - n;
  ln.total = __builtin_amdgcn_readlane(incl, 63);
  return ln;
}

// The head that holds unit `pos` < total of the line (all wave-uniform).
struct Head {
  int bh, tokens;
  int start;  // its first unit on the line
};

template <int kPer>
WGKV_DEVICE Head find_head(const AttnArgs& a, const Line<kPer>& ln, int pos, int lane) {
  Head h;
  // the last lane that starts at or before pos (lanes without units start
  // where the next one does)
  const int o = 63 - __builtin_clzll(__builtin_amdgcn_ballot_w64(ln.excl <= pos));
  const int base = __builtin_amdgcn_readlane(ln.excl, o);
  if constexpr (kPer <= 4) {
    h.bh = o * ln.per;
    h.tokens = __builtin_amdgcn_readlane(ln.tokens[0], o);
    h.start = base;
#pragma unroll
    for (int k = 1; k < kPer; ++k) {
      const int next = h.start + units_of(h.tokens);  // of head o*per + k, where the search has come this far
      if (h.bh == o * ln.per + k - 1 && pos >= next) {
        h.bh = o * ln.per + k;
        h.tokens = __builtin_amdgcn_readlane(ln.tokens[k], o);
        h.start = next;
      }
    }
  } else {
    const int bh = o * ln.per + lane;
    const bool in = lane < ln.per && bh < a.B * a.Hkv;
    const int t = in ? tokens_of(a, bh) : 0;
    const int excl = base + wave_scan_dpp(units_of(t)) - units_of(t);
    const int j = 63 - __builtin_clzll(__builtin_amdgcn_ballot_w64(in && excl <= pos));
    h.bh = o * ln.per + j;
    h.tokens = __builtin_amdgcn_readlane(t, j);
    h.start = __builtin_amdgcn_readlane(excl, j);
  }
  return h;
}

template <int CTRL>
WGKV_DEVICE float row_ror_add(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + CTRL, 0xf, 0xf, false));
}

// Sum and maximum over the four 16-lane rows of a wave, lane by lane
// (v_permlane32_swap, v_permlane16_swap: no LDS round trip).
template <typename Op>
WGKV_DEVICE float over_rows(float x, Op op) {
  uint32_t u = __float_as_uint(x);
  u32x2_t r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  u = __float_as_uint(op(__uint_as_float(r[0]), __uint_as_float(r[1])));
  r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return op(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
WGKV_DEVICE float rows_sum(float x) {
  return over_rows(x, [](float a, float b) { return a + b; });
}
WGKV_DEVICE float rows_max(float x) {
  return over_rows(x, [](float a, float b) { return fmaxf(a, b); });
}

// A dword of codes as four operand dwords (pairs of 128 + c).
// The constants come in registers, one scalar and one vector: as literals
// they would make two instructions of one v_and_or.
WGKV_DEVICE void expand(uint32_t w, uint32_t mask, uint32_t base, uint32_t* o) {
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = ((w >> (4 * i)) & mask) | base;
}

// The weight of a piece with maximum m under the common maximum M >= kNoMax.
// One without a score above it holds zeros, or a NaN that any weight keeps.
WGKV_DEVICE float piece_weight(float m, float M) { return fast_exp2(m - M); }

// 1 / sum of the weights.  The sum is 0 where every score is -inf (else one
// weight is 1): zeros then, as of a head without tokens.
WGKV_DEVICE float inverse_sum(float l) { return l == 0.f ? 0.f : __builtin_amdgcn_rcpf(l); }

// Merges the pieces that workgroups f..e left of head (b, h) and writes its
// G rows.  A thread takes four d of a row over every groups-th piece, four
// pieces' loads in flight, and the groups meet in LDS (kThreads * 6 floats).
template <int D, int kThreads>
WGKV_DEVICE void merge_pieces(const AttnArgs& a, int f, int e, int b, int h, float* lds) {
  constexpr int kBatch = 4, kRow = D / 4;  // threads of a row
  const int G = a.G;
  static_assert(kThreads >= kMaxG * kRow, "a thread for every four d");
  const int t = threadIdx.x, d = t % kRow * 4;
  const int i = t / kRow & ((1 << a.g_shift) - 1), grp = t / kRow >> a.g_shift;
  const int groups = kThreads / kRow >> a.g_shift;
  float* s_m = lds;
  float* s_l = lds + kThreads;
  f32x4_t* s_a = (f32x4_t*)(lds + 2 * kThreads);
  const __amdgpu_buffer_rsrc_t acc = __builtin_amdgcn_make_buffer_rsrc(a.part_acc, (short)0, 0x7fffffff, 0x00020000);
  const int row = min(i, G - 1);
  float M = kNoMax, L = 0.f;
  f32x4_t A = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int x0 = f + grp; x0 <= e; x0 += groups * kBatch) {
    float m[kBatch], l[kBatch];
    f32x4_t ac[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int x = min(x0 + k * groups, e);
      const int s = (2 * x + (x == f ? 1 : 0)) * G + row;
      m[k] = load_coherent(&a.part_ml[s * 2]);
      l[k] = load_coherent(&a.part_ml[s * 2 + 1]);
      ac[k] = load_coherent4(acc, (s * D + d) * (int)sizeof(float));
    }
    float mn = M;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) mn = fmaxf(mn, m[k]);
    const float sa = piece_weight(M, mn);
    L *= sa;
    A *= sa;
    M = mn;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (x0 + k * groups > e) break;
      const float sb = piece_weight(m[k], M);
      L = fmaf(l[k], sb, L);
      A += ac[k] * sb;
    }
  }
  s_m[t] = M;
  s_l[t] = L;
  s_a[t] = A;
  __syncthreads();
  if (grp == 0 && i < G) {
#pragma unroll 1
    for (int x = t + (kRow << a.g_shift); x < kThreads; x += kRow << a.g_shift) {
      const float mn = fmaxf(M, s_m[x]);
      const float sa = piece_weight(M, mn), sb = piece_weight(s_m[x], mn);
      L = fmaf(s_l[x], sb, L * sa);
      A = A * sa + s_a[x] * sb;
      M = mn;
    }
    const float inv = inverse_sum(L);
    uint16_t* o = a.out + (int64_t)b * a.out_sb + (int64_t)(h * G + i) * a.out_sh + d;
    *(uint64_t*)o = (uint64_t)pack_bf16x2(A[2] * inv, A[3] * inv) << 32 | pack_bf16x2(A[0] * inv, A[1] * inv);
  }
}

// unit / per, exact: the quotient is a workgroup's index (below 2^9), so that
// the approximate one is at most 1 off.
WGKV_DEVICE int quotient(int unit, int per) {
  const int q = (int)((float)unit * __builtin_amdgcn_rcpf((float)per));
  const int r = unit - q * per;
  return r < 0 ? q - 1 : r >= per ? q + 1 : q;
}

// The line cut into ranges that differ by a unit: over the workgroups, the
// first `more` of which get units + 1, and so again over a workgroup's waves.
// A unit is 1.7 us of one SIMD's vector instructions, so a line too short for
// all of them goes to workgroups of a unit per SIMD, not per wave (8 heads of
// 1300 tokens in a graph: 13.9 -> 12.0 us; units of 32 tokens 11.9, but 73.9
// -> 77 us at 8 sequences of 128K).
struct Split {
  int used, units, more;
  WGKV_DEVICE int first(int w) const { return min(w, used) * units + min(w, more); }
  WGKV_DEVICE int owner(int unit) const {  // the workgroup that has a unit
    const int cut = more * (units + 1);
    const bool late = unit >= cut;
    return quotient(late ? unit - cut : unit, late ? units : units + 1) + (late ? more : 0);
  }
};

// (The host keeps all of this within 31 bits.)
WGKV_DEVICE Split make_split(int total, int n_wg) {
  Split s;
  s.used = max(min((total + kFewest - 1) / kFewest, n_wg), 1);
  s.units = (int)((unsigned)total / (unsigned)s.used);
  s.more = total - s.units * s.used;
  return s;
}

// What a wave leaves in LDS of a head that it has not seen whole.
struct Piece {
  int bh;            // -1: none
  int start, units;  // of the head on the line
};

template <int D, int NT, int NW, int kPer>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(NW / 4, NW / 4))) void kv4_attn_kernel(AttnArgs a) {
  constexpr int NG = D / kKv4Group;  // groups
  constexpr int HPT = 16 / NG;       // query heads per 16 columns
  constexpr int KS = D / 32;         // k-steps of the first product, dwords of a lane's K and V chunk per tile
  constexpr int MT = D / 16;         // row tiles of the second product
  constexpr int kThreads = NW * 64;
  typedef __attribute__((__vector_size__(KS * sizeof(uint32_t)))) uint32_t chunk_t;
  static_assert(2 * NW * NT * HPT * D >= kThreads * 6, "LDS of the merge");
  __shared__ __attribute__((aligned(16))) float s_acc[2 * NW][NT * HPT][D];
  __shared__ float s_m[2 * NW][NT * HPT], s_l[2 * NW][NT * HPT];
  __shared__ Piece s_piece[2 * NW];
  __shared__ int s_first[2], s_end[2];

  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, quad = lane >> 4;
  const int g = n / HPT, hh = n % HPT;
  const int G = a.G, BH = a.B * a.Hkv;
  const int w = blockIdx.x, n_wg = gridDim.x;

  // a lane's places in a tile: K row n, V row n, the pairs of its group
  const uint32_t koff = n * (D / 2) + quad * (D / 8), voff = quad * (2 * D) + n * (D / 8);
  const uint32_t soff = kv4_scales_at(D) + (quad * NG + g) * 16;
  uint32_t mask = kCodeMask, base = kCodeBase;
  asm("" : "+s"(mask));
  asm("" : "+v"(base));

  const u32x4_t ones = (u32x4_t){0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};  // bf16 1.0

  const Line<kPer> ln = make_line<kPer>(a, lane);
  const Split sp = make_split(ln.total, n_wg);
  const int wg_first = sp.first(w), wg_units = sp.first(w + 1) - wg_first;
  int pos = wg_first + wid * (wg_units / NW) + min(wid, wg_units % NW);
  const int end = pos + wg_units / NW + (wid < wg_units % NW ? 1 : 0);
  if (lane < 2) s_piece[2 * wid + lane].bh = -1;

  // 32 tokens of a head: two tiles of each cache.  Every line is read whole by
  // one load and once: non-temporal (the default policy reads 5.7 TB/s here,
  // these 6.3).
  struct Half {
    chunk_t k[2], v[2];
    u32x4_t ks[2], vs[2];
  };
  // The place the next loads are for.  Page ids of 64 tiles from tile 4*base
  // on, one per lane, clamped to the pool.
  int u = 0, base_u = 0, last_tile = 0, pages = 0;
  const int32_t* bt_row = nullptr;
  const auto load_half = [&](Half& x, int half) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int tile = min(4 * u + 2 * half + p, last_tile);
      const int pg = __builtin_amdgcn_readlane(pages, max(tile - 4 * base_u, 0));
      const int64_t at = (((int64_t)pg << a.pg.page_shift) + (tile & ((1 << a.pg.page_shift) - 1))) * kv4_tile_bytes(D);
      const uint8_t* kt = a.kc + at;
      const uint8_t* vt = a.vc + at;
      x.k[p] = __builtin_nontemporal_load((const chunk_t*)(kt + koff));
      x.ks[p] = __builtin_nontemporal_load((const u32x4_t*)(kt + soff));
      x.v[p] = __builtin_nontemporal_load((const chunk_t*)(vt + voff));
      x.vs[p] = __builtin_nontemporal_load((const u32x4_t*)(vt + soff));
    }
  };
  const auto clamp_page = [&](int pg) { return pg < 0 ? 0 : pg >= a.pg.num_pages ? (int)(a.pg.num_pages - 1) : pg; };
  u32x4_t qraw[NT][KS];
  const auto load_q = [&](int bh) {
    const int b = sequence_of(a, bh), h = bh - b * a.Hkv;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint16_t* qrow = a.q + (int64_t)b * a.q_sb + (int64_t)(h * G + min(nt * HPT + hh, G - 1)) * a.q_sh;
#pragma unroll
      for (int i = 0; i < KS; ++i) qraw[nt][i] = *(const u32x4_t*)(qrow + quad * (D / 4) + i * 8);
    }
  };
  const auto table_row = [&](int bh) {
    const int b = sequence_of(a, bh), h = bh - b * a.Hkv;
    return a.pg.bt + (int64_t)b * a.pg.bt_sb + (int64_t)h * a.pg.bt_sh;
  };

  Half x, y;
  Head hd;
  if (pos < end) {
    hd = find_head<kPer>(a, ln, pos, lane);
    u = base_u = pos - hd.start;
    last_tile = (hd.tokens - 1) >> 4;
    bt_row = table_row(hd.bh);
    const int pg = bt_row[min(4 * u + lane, last_tile) >> a.pg.page_shift];
    load_q(hd.bh);
    pages = clamp_page(pg);
    load_half(x, 0);
    __builtin_amdgcn_sched_barrier(0);  // the loads stay in front of the queries' wait
  }
  // Heads without tokens, while the first tiles are in flight: code after the
  // last tile is time of its own.
  for (int bh = w; bh < BH; bh += n_wg) {
    const int t = kPer > 1 ? tokens_of(a, bh) : __builtin_amdgcn_readlane(ln.tokens[0], bh);
    if (t != 0) continue;
    const int b = sequence_of(a, bh), h = bh - b * a.Hkv;
    for (int v = threadIdx.x; v < G * D; v += kThreads)
      a.out[(int64_t)b * a.out_sb + (int64_t)(h * G + v / D) * a.out_sh + v % D] = 0;
  }

  while (pos < end) {
    const int b = sequence_of(a, hd.bh), h = hd.bh - b * a.Hkv;
    const int T = hd.tokens, units = units_of(T);
    const int u0 = pos - hd.start, cnt = min(units - u0, end - pos);

    // queries: column (g, head), k = 8 consecutive d; zeros off the column's group
    bf16x8_t qb[NT][KS];
    f32x4_t c0[NT];
    float qsum[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool mine = quad * NG / 4 == g && nt * HPT + hh < G;
      const uint32_t keep = mine ? a.q_and : 0u, flip = mine ? a.q_xor : 0u;
      f32x4_t sum = (f32x4_t){0.f, 0.f, 0.f, 0.f};  // of the column, in every row
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const u32x4_t v = (qraw[nt][i] & keep) ^ flip;
        qb[nt][i] = __builtin_bit_cast(bf16x8_t, v);
        sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, ones), qb[nt][i], sum, 0, 0, 0);
      }
      qsum[nt] = sum[0];
      c0[nt] = sum * -kOffset;
    }

    float m_run[NT], l_run[NT], corr[NT];
    f32x4_t acc[NT][MT], usum[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m_run[nt] = kNoMax;
      l_run[nt] = corr[nt] = 0.f;
      usum[nt] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[nt][j] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    }
    // takes the offset's part out of the accumulators and adds the middles':
    // they and the offset's sum grow with the tokens, their difference does not
    const auto flush = [&]() {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float c = fmaf(-kOffset, usum[nt][0], rows_sum(corr[nt]));
        corr[nt] = 0.f;
        usum[nt] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[nt][j] += c;
      }
    };

    // tokens t0..t0+31 of the head
    const auto step = [&](Half& t, int t0) {
      const bool tail = t0 + 32 > T;  // rows past the head's end among them
      if (tail) {                         // those rows hold anything: step and middle 0
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (t0 + p * 16 + quad * 4 + i >= T) t.ks[p][i] = t.vs[p][i] = 0u;
      }
      f32x4_t z[NT][2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          uint32_t e[4];
          expand(t.k[p][i], mask, base, e);
          const u32x4_t o = (u32x4_t){e[0], e[1], e[2], e[3]};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            z[nt][p] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, o), qb[nt][i],
                                                               i == 0 ? c0[nt] : z[nt][p], 0, 0, 0);
        }
      }
      u32x4_t pb[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float s[2][4];
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float v = fmaf(z[nt][p][i], bf16lo(t.ks[p][i]), bf16hi(t.ks[p][i]) * qsum[nt]);
            v = row_ror_add<8>(v);
            if constexpr (NG == 4) v = row_ror_add<4>(v);
            s[p][i] = v;
          }
        if (tail) {
#pragma unroll
          for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              asm volatile("" : "+v"(s[p][i]));  // a branch, not selects in every unit
              if (t0 + p * 16 + quad * 4 + i >= T) s[p][i] = -INFINITY;
            }
        }
        const float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                                fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        // The maximum of a column moves only when a score exceeds it by more
        // than the slack (p <= 2^slack); it is the same in the column's four
        // lanes, whose accumulators hold sums over all of them.
        if (__builtin_amdgcn_ballot_w64(top * a.scale_log2 > m_run[nt] + kRescaleSlack)) {
          const float mn = fmaxf(m_run[nt], rows_max(top) * a.scale_log2);
          const float alpha = fast_exp2(m_run[nt] - mn);
          m_run[nt] = mn;
          l_run[nt] *= alpha;
          corr[nt] *= alpha;
          usum[nt] *= alpha;
#pragma unroll
          for (int j = 0; j < MT; ++j) acc[nt][j] *= alpha;
        }
        uint32_t pk[4];
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t s0 = t.vs[p][2 * j], s1 = t.vs[p][2 * j + 1];
            const float p0 = fast_exp2(fmaf(s[p][2 * j], a.scale_log2, -m_run[nt]));
            const float p1 = fast_exp2(fmaf(s[p][2 * j + 1], a.scale_log2, -m_run[nt]));
            l_run[nt] += p0 + p1;
            corr[nt] = fmaf(p1, bf16hi(s1), fmaf(p0, bf16hi(s0), corr[nt]));
            // Rounded to bf16 for the matrix core, as the bf16 cache's
            // probabilities are: 2^-8 at most of what a code adds, and the
            // middles' part (corr) keeps fp32.  Against 64 bits the outputs
            // are 2.1e-3 to 2.4e-3 off (rms over rms), of which their own
            // rounding is 1.7e-3.
            pk[2 * p + j] = pack_bf16x2(p0 * bf16lo(s0), p1 * bf16lo(s1));
          }
        pb[nt] = (u32x4_t){pk[0], pk[1], pk[2], pk[3]};
        // the sum of the rounded products, for the offset to cancel exactly
        usum[nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, ones),
                                                           __builtin_bit_cast(bf16x8_t, pb[nt]), usum[nt], 0, 0, 0);
      }
      // row tile j holds d = MT*r + j: code j%4 of the words of half j/4
#pragma unroll
      for (int hf = 0; hf < KS / 2; ++hf) {
        uint32_t e[4][4];  // (tile, pair), code
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int pr = 0; pr < 2; ++pr) expand(t.v[p][pr * (KS / 2) + hf], mask, base, e[2 * p + pr]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const u32x4_t o = (u32x4_t){e[0][c], e[1][c], e[2][c], e[3][c]};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            acc[nt][hf * 4 + c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                __builtin_bit_cast(bf16x8_t, o), __builtin_bit_cast(bf16x8_t, pb[nt]), acc[nt][hf * 4 + c], 0, 0, 0);
        }
      }
    };

    Head nx = hd;  // the next unit's head
    for (int it = 0; it < cnt; ++it) {
      // what the next unit needs before its tiles can be asked for -- new
      // page ids, the next head's queries -- is requested ahead of this
      // unit's second half, and so is there when that half is
      // Of a SIMD's two waves the older is served first and was done with its
      // range 15 % before the younger, which then had the memory to itself:
      // the younger goes first for five eighths of it (batch 8 at 128K 76.0 ->
      // 73.8 us, 400K tokens 89.9 -> 87.0; half of it 74.7 and 87.7).
      if constexpr (NW > 4) {
        if (wid >= NW / 2 && it < cnt * 5 / 8) __builtin_amdgcn_s_setprio(1);
        else __builtin_amdgcn_s_setprio(0);
      }
      const int t0 = (u0 + it) * 64;
      const bool cross = it + 1 == cnt && pos + cnt < end;
      const bool refill = cross || u0 + it + 1 - base_u == 16;
      int pg = 0;
      if (refill) {
        if (cross) {
          nx = find_head<kPer>(a, ln, pos + cnt, lane);
          load_q(nx.bh);
        }
        const int first_u = cross ? 0 : u0 + it + 1;
        pg = table_row(nx.bh)[min(4 * first_u + lane, (nx.tokens - 1) >> 4) >> a.pg.page_shift];
      }
      load_half(y, 1);
      step(x, t0);
      if (refill) {
        u = base_u = cross ? 0 : u0 + it + 1;
        last_tile = (nx.tokens - 1) >> 4;
        pages = clamp_page(pg);
      } else {
        ++u;
      }
      load_half(x, 0);  // past the range's end: any of its tiles
      step(y, t0 + 32);
      if ((it & (kFlush - 1)) == kFlush - 1) flush();
    }
    flush();

    // lane (quad, g, hh) holds rows 4*quad + i of column (g, hh): d = MT *
    // (4*quad + i) + j, of the column's group where quad*NG/4 == g
    const bool whole = cnt == units;
    const int slot = 2 * wid + (u0 > 0 ? 0 : 1);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float l = rows_sum(l_run[nt]);
      const int qh = nt * HPT + hh;
      if (quad * NG / 4 == g && qh < G) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = MT * (4 * quad + i);
          if (whole) {
            const float inv = inverse_sum(l);
            uint32_t o[MT / 2];
#pragma unroll
            for (int j = 0; j < MT / 2; ++j) o[j] = pack_bf16x2(acc[nt][2 * j][i] * inv, acc[nt][2 * j + 1][i] * inv);
            uint16_t* dst = a.out + (int64_t)b * a.out_sb + (int64_t)(h * G + qh) * a.out_sh + d;
            if constexpr (MT == 8) *(u32x4_t*)dst = (u32x4_t){o[0], o[1], o[2], o[3]};
            else *(uint64_t*)dst = (uint64_t)o[1] << 32 | o[0];
          } else {
#pragma unroll
            for (int j = 0; j < MT; ++j) s_acc[slot][qh][d + j] = acc[nt][j][i];
          }
        }
      }
      if (!whole && quad == 0 && g == 0) {
        s_m[slot][qh] = m_run[nt];
        s_l[slot][qh] = l;
      }
    }
    if (!whole && lane == 0) s_piece[slot] = Piece{hd.bh, hd.start, units};
    pos += cnt;
    hd = nx;
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the loads past the end
  __syncthreads();

  // ---- the workgroup's heads -----------------------------------------------
  // Waves hold consecutive ranges, so a head's pieces are neighbours in LDS.
  // What the workgroup does not hold whole goes to the workspace: at most the
  // head that it ends and the one that it begins.
  const Piece mine = s_piece[lane & (2 * NW - 1)];
  uint64_t todo = __builtin_amdgcn_ballot_w64(lane < 2 * NW && mine.bh >= 0);
  int n_open = 0, open_bh[2], open_start[2], open_units[2];
  while (todo) {
    const int s0 = __builtin_ctzll(todo);
    const int bh = __builtin_amdgcn_readlane(mine.bh, s0);
    const int start = __builtin_amdgcn_readlane(mine.start, s0), units = __builtin_amdgcn_readlane(mine.units, s0);
    const uint64_t run = __builtin_amdgcn_ballot_w64(lane < 2 * NW && mine.bh == bh);
    todo &= ~run;
    const int b = sequence_of(a, bh), h = bh - b * a.Hkv;
    const bool begins = start >= wg_first, whole = begins && start + units <= wg_first + wg_units;
    const int to = (2 * w + (begins ? 1 : 0)) * G;
    for (int v = threadIdx.x; v < G * D; v += kThreads) {
      const int i = v / D, d = v - i * D;
      float M = kNoMax, L = 0.f, A = 0.f;
      for (uint64_t r = run; r; r &= r - 1) M = fmaxf(M, s_m[__builtin_ctzll(r)][i]);
      for (uint64_t r = run; r; r &= r - 1) {
        const int s = __builtin_ctzll(r);
        const float c = piece_weight(s_m[s][i], M);
        L = fmaf(s_l[s][i], c, L);
        A = fmaf(s_acc[s][i][d], c, A);
      }
      if (whole) {
        a.out[(int64_t)b * a.out_sb + (int64_t)(h * G + i) * a.out_sh + d] = f32_to_bf16(A * inverse_sum(L));
      } else {
        if (d == 0) {
          store_coherent(&a.part_ml[(to + i) * 2], M);
          store_coherent(&a.part_ml[(to + i) * 2 + 1], L);
        }
        store_coherent(&a.part_acc[(to + i) * D + d], A);
      }
    }
    if (!whole) {
      if (n_open == 0) open_bh[0] = bh, open_start[0] = start, open_units[0] = units;
      else open_bh[1] = bh, open_start[1] = start, open_units[1] = units;
      ++n_open;
    }
  }

  if (n_open > 0) {
    // The last workgroup of a head to arrive merges.  Its loads see the
    // others' pieces without cache write-backs: the stores above are
    // device-coherent (written through to the point of coherence, where the
    // counter's atomics are performed too), vmcnt(0) waits until they are
    // acknowledged there, the barrier holds the arrival until every wave has
    // waited, and the merge's loads bypass this XCD's L2.
#if defined(__HIP_DEVICE_COMPILE__) && !defined(__gfx950__)
#error "the merge relies on gfx950 store acknowledgement and sc1 ordering"
#endif
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __syncthreads();
    if ((int)threadIdx.x < n_open) {
      const int t = threadIdx.x;
      const int bh = t ? open_bh[1] : open_bh[0], start = t ? open_start[1] : open_start[0];
      const int prev = __hip_atomic_fetch_add(&a.counter[bh], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const int f = sp.owner(start), e = sp.owner(start + (t ? open_units[1] : open_units[0]) - 1);
      const bool last = prev == e - f;
      if (last) __hip_atomic_store(&a.counter[bh], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      s_first[t] = last ? f : -1;
      s_end[t] = e;
    }
    __syncthreads();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
#pragma unroll 1
    for (int t = 0; t < n_open; ++t) {
      const int f = __builtin_amdgcn_readfirstlane(s_first[t]), e = __builtin_amdgcn_readfirstlane(s_end[t]);
      if (f < 0) continue;
      const int bh = t ? open_bh[1] : open_bh[0], b = sequence_of(a, bh);
      if (t) __syncthreads();  // the first one's LDS
      merge_pieces<D, kThreads>(a, f, e, b, bh - b * a.Hkv, &s_acc[0][0][0]);
    }
  }
}

size_t part_floats(int G, int D) { return (size_t)2 * kMaxSlots * G * (2 + (size_t)D); }
constexpr size_t kCounterBytes = (size_t)kMaxBH * sizeof(int);

// One workgroup per CU: 8 waves, two per SIMD, or with two column tiles, whose
// accumulators and queries take twice the registers, 4.
template <int D, int NT>
hipError_t launch(const AttnArgs& a, hipStream_t st) {
  constexpr int NW = NT == 1 ? 8 : 4;
  // no more workgroups than the tables have units for
  const int64_t most = ((kv4_capacity(a.pg) + kUnit - 1) / kUnit * a.B * a.Hkv + kFewest - 1) / kFewest;
  const int slots = min(kMaxSlots, cu_count());
  const dim3 grid((unsigned)(most < slots ? most : slots));
  const dim3 block(NW * 64);
  const int heads = a.B * a.Hkv;
  if (heads <= 64) hipLaunchKernelGGL((kv4_attn_kernel<D, NT, NW, 1>), grid, block, 0, st, a);
  else if (heads <= 256) hipLaunchKernelGGL((kv4_attn_kernel<D, NT, NW, 4>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((kv4_attn_kernel<D, NT, NW, 32>), grid, block, 0, st, a);
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
  if ((kv4_capacity(a.pg) + kUnit - 1) / kUnit * batch * num_kv_heads > 0x7f000000) return WGKV_ERR_UNSUPPORTED;
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) return WGKV_ERR_UNSUPPORTED;
  if ((q_stride_b | q_stride_h) & 7) return WGKV_ERR_UNSUPPORTED;
  if (((uintptr_t)out & 15) || ((out_stride_b | out_stride_h) & 7)) return WGKV_ERR_UNSUPPORTED;
  if (kv4_rows_meet({batch, num_q_heads, 1, 1}, {out_stride_b, out_stride_h, 0, 0}, head_dim)) return WGKV_ERR_ARG;
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
  a.g_shift = G <= 1 ? 0 : G <= 2 ? 1 : G <= 4 ? 2 : 3;
  a.cap = (int)kv4_capacity(a.pg);
  a.hkv_inv = num_kv_heads == 1 ? 0u : (uint32_t)((0x100000000ull + num_kv_heads - 1) / num_kv_heads);
  // scores in the order of the products: a negative scale negates the
  // queries, and a scale of 0 clears them (masked rows hold -inf, and -inf * 0
  // is not a number)
  a.scale_log2 = softmax_scale == 0.f ? 1.f : fabsf(softmax_scale) * kLog2e;
  a.q_and = softmax_scale == 0.f ? 0u : ~0u;
  a.q_xor = softmax_scale < 0.f ? 0x80008000u : 0u;
  a.counter = (int*)workspace;
  const size_t slots = (size_t)2 * kMaxSlots * G;
  a.part_ml = (float*)((char*)workspace + kCounterBytes);
  a.part_acc = a.part_ml + slots * 2;
  hipStream_t s = (hipStream_t)stream;
  const hipError_t e = head_dim == 64 ? launch<64, 1>(a, s) : G <= 4 ? launch<128, 1>(a, s) : launch<128, 2>(a, s);
  return e == hipSuccess ? WGKV_OK : WGKV_ERR_HIP;
}

extern "C" int wgkv_kv4_decode_attn_block(const void* args) {
  int64_t a[24];
  memcpy(a, args, sizeof a);
  if (!kv4_narrow(a, 6, 12, 16, 17, 18, 19)) return WGKV_ERR_UNSUPPORTED;
  double scale;
  memcpy(&scale, &a[20], sizeof scale);
  return wgkv_kv4_decode_attn((const void*)a[0], a[1], a[2], (const void*)a[3], (const void*)a[4], a[5], (int32_t)a[6],
                              (const int32_t*)a[7], a[8], (const int32_t*)a[9], a[10], a[11], (int32_t)a[12],
                              (void*)a[13], a[14], a[15], (int32_t)a[16], (int32_t)a[17], (int32_t)a[18],
                              (int32_t)a[19], (float)scale, (void*)a[21], (size_t)a[22], (void*)a[23]);
}
