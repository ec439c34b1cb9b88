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
// Work item = (64 rows of a sequence, KV head, group of 4 or 2 of its G query
// heads, or 128 rows and one head) for a workgroup of 8 or 4 waves; a wave
// serves 32 rows of one head.
// The item's keys are the `first` tokens below the band and the band
// [lo, last row's position] that the rows' windows reach, counted through as
// one list and cut into tiles of 64, so that a few first tokens cost their
// share of a tile and not one of their own.  Tiles go from memory straight
// into LDS, one tile ahead of the arithmetic (buffer loads), and
// serve all heads of the group.  S^T = K Q^T on v_mfma_f32_16x16x32_bf16
// leaves each lane 16 scores of a query row, which are the B operand of
// O^T += V^T P^T; V^T comes by LDS transpose reads.  Softmax is in the log2
// domain, fp32, with a running maximum that moves only when a score exceeds it
// by more than 8; probabilities are rounded to bf16 for the products, and
// their sums are taken of the rounded values.  Only the tiles at the two ends
// of a row's window are masked.
//
// Few rows (a last piece of a prompt, drafted tokens behind a long one) do not
// fill the card: the tiles of every item are then cut into equal parts, a
// workgroup each, whose (max, sum, O) a second launch joins.
//
// Measured (32/8 heads, D 128): 32768 rows, window 1024 and 4 first tokens 644
// us, 840 TFLOP/s of the pairs that are seen, 940 of the tiles, where a large
// bf16 product reaches 1395; rows behind earlier keys with a window of 4096 1020;
// the first with D 64 435 us, 624.  Neither unit is full: matrix instructions take
// 41 % of a SIMD's cycles, and a wave, of which a SIMD has two, executes vector
// instructions (these included) in 26 % of its own.  A wave issues 228 that are not
// matrix ones per tile, where the prefill of one prompt (sparse_prefill.hip) takes
// 138; among them are addresses and bounds of the coming tile's loads, which stand
// before the first product, and moves of the 111 scalars that do not fit.  Short prompts
// (7 of 300 to 600 rows, D 64: 15.4 us, of which one row takes 6.6) are a chain of
// tiles' round trips to memory.
//
// A masked probability is 0, and 0 times a key's value that is not finite is
// NaN: of the rows whose result is not finite, those whose tiles held such a value
// that they do not see are worked out once more, one after the other (rows_to_redo,
// exact_row).  Rows that see it keep theirs.  (4096 rows, 8/2 heads, D 128, window
// 1024, 0.06 ms: an infinite value of a first token, which all rows see, 0.07 ms,
// and 12.8 when every such row was redone key by key; of a middle token, which up to
// 63 rows around its block and 63 at the windows' end do not see, 3.8, whatever
// the number of rows; infinities throughout 3.8, and 30 for 32768 rows of 32 heads.)
#include <string.h>

#include "attn_tile.h"
#include "kv4.h"

namespace {

// Query rows per item of that many heads.  (Two waves of one head would load
// each tile for 64 rows alone: 32768 rows, window 1024, three heads a KV head 975
// us, in items of 128 rows 616.)
constexpr int item_rows(int heads) { return heads == 1 ? 128 : 64; }
constexpr int item_waves(int heads) { return heads * item_rows(heads) / 32; }
constexpr int kMaxSeqs = 2048;
constexpr int kLeastTiles = 4;  // of a part: less than about what the join costs

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
  bool far;        // keys may lie 2^31 bytes or more apart
  int parts;       // of an item's tiles; more than 1: (max, sum) and O of (part, row, head) go to
  float* part_ml;
  float* part_o;
};

WGKV_DEVICE int clamp_to(int x, int hi) { return min(max(x, 0), hi); }

// A value that every lane holds, as a scalar.
WGKV_DEVICE int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

typedef const int32_t __attribute__((address_space(4))) ConstInt;

// A sequence's rows and keys (scalar loads where b is a scalar).
struct Seq {
  int q0, nq, k0, nk;
};
WGKV_DEVICE Seq seq_of(const WindowArgs& a, int b) {
  ConstInt *q = (ConstInt*)a.cu_q, *k = (ConstInt*)a.cu_k;
  const int q0 = clamp_to(q[b], a.N), k0 = clamp_to(k[b], a.Nk);
  return {q0, max(clamp_to(q[b + 1], a.N) - q0, 0), k0, max(clamp_to(k[b + 1], a.Nk) - k0, 0)};
}

// The keys of an item as one list: entry x is key x for x < first, else key x + shift.
struct Keys {
  int first, shift, count;
  WGKV_DEVICE int key(int x) const { return x < first ? x : x + shift; }
};

// A row on its own, by a wave: 64 keys at a time, one a lane for the scores; for
// the values D/8 lanes a key, eight values of d each.  What the row does not see
// is not touched.
template <int D>
WGKV_DEVICE void exact_row(const WindowArgs& a, const uint16_t* q, const uint16_t* k, const uint16_t* v, int p,
                           uint16_t* out, int lane) {
  constexpr int CH = D / 8, KPI = 64 / CH;  // 16-byte slices of a row, keys whose values one load of the wave takes
  constexpr int kAhead = 8;                 // loads of values that are asked for together
  const int c = lane % CH;
  float acc[8], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
  const int lo = max(0, p - a.window + 1), first = min(a.sinks, lo), count = first + p - lo + 1;
  const auto key = [&](int x) { return (int64_t)(x < first ? x : x - first + lo); };
  for (int x0 = 0; x0 < count; x0 += 64) {
    const uint16_t* row = k + key(min(x0 + lane, count - 1)) * a.k_sn;
    float s = 0.f;
#pragma unroll(CH / 2)
    for (int j = 0; j < CH; ++j) {
      const u32x4_t kw = *((const u32x4_t*)row + j), qw = (*((const u32x4_t*)q + j) & a.q_and) ^ a.q_xor;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s = fmaf(__uint_as_float(qw[i] << 16), __uint_as_float(kw[i] << 16), s);
        s = fmaf(__uint_as_float(qw[i] & 0xffff0000u), __uint_as_float(kw[i] & 0xffff0000u), s);
      }
    }
    s = x0 + lane < count ? s * a.scale_log2 : -INFINITY;
    if (__builtin_amdgcn_ballot_w64(s != s || s == INFINITY) != 0) {  // so is the row's sum
      l = NAN;
      break;
    }
    const float mn = fmaxf(m, wave_max(s)), by = mn == -INFINITY ? 0.f : mn;  // (a score of -inf: a weight of 0)
    const float was = m == -INFINITY ? 0.f : fast_exp2(m - mn), w = round_to_bf16(fast_exp2(s - by));
    m = mn;
    l = l * was + wave_sum(w);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= was;
    for (int y0 = lane / CH; y0 < 64; y0 += KPI * kAhead) {
      u32x4_t vw[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        vw[j] = *((const u32x4_t*)(v + key(min(x0 + y0 + j * KPI, count - 1)) * a.v_sn) + c);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int y = y0 + j * KPI;
        const float wy = __shfl(w, y, 64);
        const bool on = x0 + y < count;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[2 * i] = on ? fmaf(wy, __uint_as_float(vw[j][i] << 16), acc[2 * i]) : acc[2 * i];
          acc[2 * i + 1] = on ? fmaf(wy, __uint_as_float(vw[j][i] & 0xffff0000u), acc[2 * i + 1]) : acc[2 * i + 1];
        }
      }
    }
    bool nan = true;
#pragma unroll
    for (int e = 0; e < 8; ++e) nan = nan && acc[e] != acc[e];
    uint64_t y = __builtin_amdgcn_ballot_w64(nan);
#pragma unroll
    for (int off = CH; off < 64; off <<= 1) y |= y >> off;
    if ((~y & ((1ull << CH) - 1)) == 0 && l != 0.f) break;  // every value is NaN
  }
#pragma unroll
  for (int off = CH; off < 64; off <<= 1)
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] += __shfl_xor(acc[e], off, 64);
  if (lane >= CH) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  u32x4_t o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = l == 0.f ? 0u : pack_bf16x2(acc[2 * i] * inv, acc[2 * i + 1] * inv);
  *((u32x4_t*)out + c) = o;
}

// Values of d as bits: word d % 4, bit d / 4.
typedef u32x4_t Columns;

// Of up to 32 rows from position p0 on, by a wave, whose sums O are not finite in
// `need` (lane i: row i % 32's; the sum of their weights is finite): those to be
// worked out on their own.  `ks`: the keys that their tiles held.  A row is right as
// it is if keys that it sees have such values in all of these places and others in
// its tiles have none.  It is not if a key that it does not see has some, since a
// masked weight of 0 times its value is NaN, or if no key has: then large values
// have overflowed under a maximum that lags.  A tile that every row sees in full is
// read only while some row lacks such keys.  `twice`: a row's own key may have
// stood in its tiles a second time, masked.
template <int D>
WGKV_DEVICE uint32_t rows_to_redo(const WindowArgs& a, const Keys& ks, const uint16_t* v, int nk, int p0, uint32_t rows,
                                  Columns need, bool twice, int lane) {
  const int p = p0 + (lane & 31);  // the lane's row
  const bool mine = rows >> (lane & 31) & 1;
  bool unseen = false;
  const auto open = [&]() { return mine && !unseen && (need[0] | need[1] | need[2] | need[3]) != 0; };
  for (int x0 = 0; x0 < ks.count; x0 += attn::kKeys) {
    const int x1 = x0 + attn::kKeys - 1, e0 = p0 - ks.shift;
    const bool full = x1 < ks.count && x1 <= e0 && (e0 + 31 - x0 < a.window || x1 < a.sinks);
    if (full && __builtin_amdgcn_ballot_w64(open()) == 0) continue;
    // a key a lane (also behind the rows' keys: the last tile holds them)
    const int j = ks.key(x0 + lane);
    const uint16_t* row = v + (int64_t)min(j, nk - 1) * a.v_sn;
    Columns bad = {0, 0, 0, 0};
#pragma unroll 4
    for (int i = 0; i < D / 8; ++i) {
      const u32x4_t w = *((const u32x4_t*)row + i);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t inf = e & 1 ? 0x7f800000u : 0x7f80u;
        bad[e % 4] |= (uint32_t)((w[e / 2] & inf) == inf) << (2 * i + e / 4);
      }
    }
    const bool some = j < nk && (bad[0] | bad[1] | bad[2] | bad[3]) != 0;
    for (uint64_t left = __builtin_amdgcn_ballot_w64(some); left; left &= left - 1) {
      const int at = __builtin_ctzll(left), jb = ks.key(x0 + at);
      const bool sees = jb <= p && (jb > p - a.window || jb < a.sinks);
      unseen = unseen || !sees || (twice && jb == p);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t has = __builtin_amdgcn_readlane(bad[e], at);
        need[e] = sees ? need[e] & ~has : need[e];
      }
      if (__builtin_amdgcn_ballot_w64(mine && !unseen) == 0) return rows;
      if (full && __builtin_amdgcn_ballot_w64(open()) == 0) break;
    }
  }
  return rows & (uint32_t)__builtin_amdgcn_ballot_w64(unseen || open());
}

struct Item {
  int q0, nq, nk;     // the sequence's first row, rows and keys
  int r_blk, p_blk;   // the item's first row in the sequence, and its position
  int h, hq0;         // KV head, first query head
  Keys keys;
  int part, t0, tiles;  // the part's tiles begin at t0
  const uint16_t *kb, *vb;
};

WGKV_DEVICE Keys keys_of(const WindowArgs& a, int p_blk, int p_last) {
  if (p_last < 0) return {0, 0, 0};
  const int lo = max(0, p_blk - a.window + 1), first = min(a.sinks, lo);
  return {first, lo - first, first + p_last - lo + 1};
}

// The block's sequence; s_blocks: row blocks of the sequences before each.
WGKV_DEVICE int sequence_of(const WindowArgs& a, const int* s_blocks, int blk) {
  int b = 0;
  for (int hi = a.B - 1; b < hi;) {  // the last sequence that begins at or before the block
    const int mid = (b + hi + 1) >> 1;
    if (uniform(s_blocks[mid]) <= blk) b = mid; else hi = mid - 1;
  }
  return b;
}

// A buffer of `bytes` at p (a scalar address), and 16 bytes of it to LDS at lds
// + 16 * lane; beyond its end they are zeros.
WGKV_DEVICE __amdgpu_buffer_rsrc_t rows_buffer(const uint16_t* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, (short)0, bytes, 0x00020000);
}
WGKV_DEVICE void buffer_to_lds(__amdgpu_buffer_rsrc_t r, uint16_t* lds, int off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, lds, 16, off, 0, 0, 0);
}

// FAR: keys that may lie 2^31 bytes or more apart.
template <int D, int HPW, bool FAR>
__global__ __launch_bounds__(64 * item_waves(HPW)) __attribute__((amdgpu_waves_per_eu(2, 2)))
void window_prefill_kernel(WindowArgs a) {
  constexpr int NW = item_waves(HPW), NT = 64 * NW, BLK = item_rows(HPW);
  constexpr int CH = D / 8;        // 16-byte slices per row
  constexpr int RPB = 64 / CH;     // key rows of 1 KB of LDS, one load instruction of a wave
  constexpr int NBLK = attn::kKeys / RPB;
  // with four heads only the older wave of each SIMD loads: it reaches the
  // tile's barrier first
  constexpr int NL = HPW == 4 ? NW / 2 : NW;
  constexpr int KPT = NBLK / NL;
  static_assert(NBLK % NL == 0, "every loading wave loads whole 1 KB blocks");
  // four LDS objects: loads into one buffer then provably leave the other alone
  __shared__ __attribute__((aligned(16))) uint16_t sK0[attn::kKeys * D];
  __shared__ __attribute__((aligned(16))) uint16_t sK1[attn::kKeys * D];
  __shared__ __attribute__((aligned(16))) uint16_t sV0[attn::kKeys * D];
  __shared__ __attribute__((aligned(16))) uint16_t sV1[attn::kKeys * D];
  __shared__ int s_blocks[kMaxSeqs + 1];               // row blocks of the sequences before
  __shared__ int s_wave[NW];

  const int t = threadIdx.x;
  const int lane = t & 63, wid = uniform(t >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int w_row = wid % (BLK / 32) * 32, w_head = wid / (BLK / 32);  // the wave's rows and head of the item

  {
    const int per = (a.B + NT - 1) / NT, b0 = min(a.B, t * per), b1 = min(a.B, b0 + per);
    int mine = 0;
    for (int b = b0; b < b1; ++b) mine += (seq_of(a, b).nq + BLK - 1) / BLK;
    const int incl = wave_incl_scan(mine, lane);
    if (lane == 63) s_wave[wid] = incl;
    __syncthreads();
    int run = incl - mine;
    for (int i = 0; i < NW; ++i) run += i < wid ? s_wave[i] : 0;
    for (int b = b0; b < b1; ++b) {
      s_blocks[b] = run;
      run += per == 1 ? mine : (seq_of(a, b).nq + BLK - 1) / BLK;
      // (all of them where starts ascend; what others would make of it is cut off: items
      // are then no more than the host has counted, within 32 bits)
      if (b == a.B - 1) s_blocks[a.B] = min(run, a.N / BLK + a.B);
    }
    __syncthreads();
  }
  const int blocks = uniform(s_blocks[a.B]);
  const int per_block = a.Hkv * (a.G / HPW);
  if (a.clear_rest) {
    const int head = clamp_to(a.cu_q[0], a.N), tail = max(clamp_to(a.cu_q[a.B], a.N), head);
    const int64_t pieces = (int64_t)(head + a.N - tail) * a.Hkv * a.G * CH;
    for (int64_t i = (int64_t)blockIdx.x * NT + t; i < pieces; i += (int64_t)gridDim.x * NT) {
      const int64_t r = i / CH, x = r / (a.Hkv * a.G);
      *(u32x4_t*)(a.out + (x < head ? x : x - head + tail) * a.o_sn + (r - x * (a.Hkv * a.G)) * a.o_sh + (i - r * CH) * 8) =
          (u32x4_t){0u, 0u, 0u, 0u};
    }
  }
  const attn::Offsets<D> at(n, g);

  // A round's item (part).  Items go from the last row block to the first -- later
  // blocks of a sequence see no fewer keys --, heads innermost: workgroups are
  // dealt to the XCDs in turn, so with 8 KV heads each XCD's L2 serves one
  // head's keys.  A workgroup takes items from alternate ends of its rounds.
  const auto item_at = [&](int round, Item* p) {
    // (32-bit throughout: a 64-bit division is 150 instructions of a short call's start)
    const uint32_t item = round * gridDim.x + ((round & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
    if (item >= (uint32_t)(blocks * a.parts) * per_block) return false;
    const uint32_t of = uniform(item / (uint32_t)per_block), rest = item - of * per_block;
    const uint32_t back = uniform(of / (uint32_t)a.parts);
    const int blk = blocks - 1 - back;
    p->part = of - back * a.parts;
    const int seq = uniform(sequence_of(a, s_blocks, blk));
    const Seq s = seq_of(a, seq);
    p->q0 = uniform(s.q0);
    p->nq = uniform(s.nq);
    p->nk = uniform(s.nk);
    p->r_blk = (blk - uniform(s_blocks[seq])) * BLK;
    p->p_blk = p->r_blk + p->nk - p->nq;
    const Keys k = keys_of(a, p->p_blk, p->p_blk + min(BLK, p->nq - p->r_blk) - 1);
    p->keys = {uniform(k.first), uniform(k.shift), uniform(k.count)};
    const int tiles = (p->keys.count + attn::kKeys - 1) / attn::kKeys;
    const uint32_t each = uniform((uint32_t)tiles / (uint32_t)a.parts), over = tiles - each * a.parts;
    p->t0 = p->part * each + min((uint32_t)p->part, over);
    p->tiles = each + (p->part < (int)over);
    const uint32_t group = uniform(rest / (uint32_t)a.Hkv);
    p->h = rest - group * a.Hkv;
    p->hq0 = p->h * a.G + group * HPW;
    const int k0 = uniform(s.k0);
    p->kb = a.k + (int64_t)k0 * a.k_sn + (int64_t)p->h * a.k_sh;
    p->vb = a.v + (int64_t)k0 * a.v_sn + (int64_t)p->h * a.v_sh;
    return true;
  };

  // Loading wave w fills the 1 KB blocks w, w + NL, ...: in block q lane i
  // loads slice (i % CH) ^ swz of list entry q * RPB + i / CH.  A lane's offset
  // within a tile stays, but for the jump behind the first tokens; entries
  // behind the sequence's keys read as zeros (and are masked).
  const auto tile_load = [&](const Item& p, int tl, bool on, uint16_t* dK, uint16_t* dV) __attribute__((always_inline)) {
    if (wid >= NL) return;
    const Keys& ks = p.keys;
    const int x0 = (p.t0 + tl) * attn::kKeys;
    if constexpr (!FAR) {
      const int j0 = ks.key(x0);
      const int rows = p.nk - j0 - 1;  // (nothing is asked for where there is no tile)
      const auto kr = rows_buffer(p.kb + (int64_t)j0 * a.k_sn, uniform(on ? rows * (int)(a.k_sn * 2) + D * 2 : 0));
      const auto vr = rows_buffer(p.vb + (int64_t)j0 * a.v_sn, uniform(on ? rows * (int)(a.v_sn * 2) + D * 2 : 0));
      const int jump = x0 < ks.first ? ks.shift : 0;
      const int k_jump = jump * (int)(a.k_sn * 2), v_jump = jump * (int)(a.v_sn * 2);
#pragma unroll
      for (int i = 0; i < KPT; ++i) {
        int row = (wid + i * NL) * RPB + lane / CH;
        asm volatile("" : "+v"(row));  // worked out here: over the loop there are no registers to keep it in
        const bool over = x0 + row >= ks.first;
        buffer_to_lds(kr, dK + (wid + i * NL) * 512,
                      row * (int)(a.k_sn * 2) + ((lane % CH) ^ attn::swz_k<D>(row)) * 16 + (over ? k_jump : 0));
        buffer_to_lds(vr, dV + (wid + i * NL) * 512,
                      row * (int)(a.v_sn * 2) + ((lane % CH) ^ attn::swz_v<D>(row)) * 16 + (over ? v_jump : 0));
      }
    } else if (on) {
#pragma unroll
      for (int i = 0; i < KPT; ++i) {
        int row = (wid + i * NL) * RPB + lane / CH;
        asm volatile("" : "+v"(row));
        const int64_t j = ks.key(min(x0 + row, ks.count - 1));
        attn::lds_dma16(p.kb + j * a.k_sn + ((lane % CH) ^ attn::swz_k<D>(row)) * 8, dK + (wid + i * NL) * 512);
        attn::lds_dma16(p.vb + j * a.v_sn + ((lane % CH) ^ attn::swz_v<D>(row)) * 8, dV + (wid + i * NL) * 512);
      }
    }
  };
  const auto ask_rows = [&](const Item& p, attn::Rows32<D>& r) __attribute__((always_inline)) {
    const int r0 = p.r_blk + w_row;
#pragma unroll
    for (int rt = 0; rt < 2; ++rt)
      r.ask_q(rt, a.q + (int64_t)(p.q0 + min(r0 + rt * 16 + n, p.nq - 1)) * a.q_sn + (int64_t)(p.hq0 + w_head) * a.q_sh, g);
  };

  Item cur = {}, nxt = {};
  bool more = item_at(0, &cur);
  attn::Rows32<D> r;
  if (more) {
    tile_load(cur, 0, cur.tiles > 0, sK0, sV0);
    ask_rows(cur, r);
  }
  for (int round = 1; more; ++round) {
    more = item_at(round, &nxt);
    const Keys& ks = cur.keys;
    const int r0 = cur.r_blk + w_row, p0 = cur.p_blk + w_row;  // the wave's rows
    r.take_q(a.q_and, a.q_xor);
    r.clear();
    const auto step = [&](int tile, const uint16_t* sK, const uint16_t* sV, uint16_t* nK, uint16_t* nV,
                          bool second) __attribute__((always_inline)) {
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's loads of the tile have landed
      __syncthreads();
      // the coming tile, of this item or (into the first buffers) the next
      const bool last = tile + 1 >= cur.tiles;
      tile_load(last ? nxt : cur, last ? 0 : tile + 1, !last || (second && more && nxt.tiles > 0), nK, nV);
      // Row p sees the list's entries x <= p - shift, of them those > p -
      // window - shift or < sinks.  (Of the first tokens, below the band, all
      // rows see all.)
      const int x0 = (cur.t0 + tile) * attn::kKeys, x1 = min(x0 + attn::kKeys, ks.count) - 1;
      const int e0 = p0 - ks.shift, e1 = e0 + 31;  // the last entries of the wave's first and last row
      f32x4_t sc[4][2];
      attn::tile_scores<D>(r, sK, at, sc);
      if (last && more) ask_rows(nxt, r);  // the item's own queries have had their last use
      const bool full = x1 - x0 == attn::kKeys - 1 && x1 <= e0 && (e1 - x0 < a.window || x1 < a.sinks);
      if (!full) {
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
          const int top = e0 + rt * 16 + n, hi = min(top, ks.count - 1) - x0 - 4 * g;  // from the lane's first entry
          const int span = min(a.window - 1, INT32_MAX / 2) - max(0, top - (ks.count - 1));
          if (x0 >= a.sinks) {  // hi - span <= entry <= hi
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                sc[kt][rt][i] = (uint32_t)(hi - (kt * 16 + i)) <= (uint32_t)span && span >= 0 ? sc[kt][rt][i] : -INFINITY;
          } else {
            const int f = a.sinks - x0 - 4 * g;
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int x = kt * 16 + i;
                sc[kt][rt][i] = x <= hi && (hi - x <= span || x < f) ? sc[kt][rt][i] : -INFINITY;
              }
          }
        }
      }
      attn::tile_attend<D>(r, sc, sV, at, a.scale_log2);
    };
    for (int tile = 0; tile < cur.tiles; tile += 2) {
      step(tile, sK0, sV0, sK1, sV1, false);
      if (tile + 1 < cur.tiles) step(tile + 1, sK1, sV1, sK0, sV0, true);
    }
    if (cur.tiles == 0 || cur.tiles % 2 != 0) {  // the first buffers were the last in use, or none were
      __syncthreads();
      tile_load(nxt, 0, more && nxt.tiles > 0, sK0, sV0);
      if (cur.tiles == 0 && more) ask_rows(nxt, r);
    }
    const Item done = cur;
    const int hq = done.hq0 + w_head;
    if (a.parts > 1) {
#pragma unroll
      for (int rt = 0; rt < 2; ++rt) {
        const int s = r0 + rt * 16 + n;
        if (s >= done.nq) continue;
        const int64_t at_row = ((int64_t)done.part * a.N + done.q0 + s) * (a.Hkv * a.G) + hq;
        if (g == 0) *(float2*)(a.part_ml + at_row * 2) = make_float2(r.m[rt], r.sum[rt][0]);
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) *(f32x4_t*)(a.part_o + at_row * D + dt * 16 + 4 * g) = r.o[dt][rt];
      }
      cur = nxt;
      continue;
    }
    // Rows with a value that is not finite.  (A sum that is NaN, as its row's scores
    // were, makes every value NaN below.)
    bool bad = false;
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
      float x = 0.f;
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) x += r.o[dt][rt][i] * 0.f;
      bad = bad || (r0 + rt * 16 + n < done.nq && x != x && r.sum[rt][0] == r.sum[rt][0]);
    }
    uint32_t again = 0, none = 0;  // such rows; those of them whose weights are 0
    Columns need = {0, 0, 0, 0};   // lane i: row i % 32's values
    if (__builtin_amdgcn_ballot_w64(bad) != 0) {
#pragma unroll
      for (int rt = 0; rt < 2; ++rt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t w = 0;
#pragma unroll
          for (int dt = 0; dt < D / 16; ++dt) w |= (uint32_t)(r.o[dt][rt][i] * 0.f != 0.f) << (4 * dt);
          w <<= g;
          w |= __shfl_xor(w, 16, 64);
          w |= __shfl_xor(w, 32, 64);
          need[i] = (g & 1) == rt ? w : need[i];
        }
      const float l = g & 1 ? r.sum[1][0] : r.sum[0][0];
      const bool here = r0 + (lane & 31) < done.nq && l == l && (need[0] | need[1] | need[2] | need[3]) != 0;
      again = (uint32_t)__builtin_amdgcn_ballot_w64(here);
      none = (uint32_t)__builtin_amdgcn_ballot_w64(here && l == 0.f);
    }
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
      const float l = r.sum[rt][0];
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int s = r0 + rt * 16 + n;
      if (s >= done.nq) continue;
      uint16_t* orow = a.out + (int64_t)(done.q0 + s) * a.o_sn + (int64_t)hq * a.o_sh;
      // (16.4 -> 15.3 us for 7 prompts of 300 to 600 rows, D 64)
      // a lane has 4 values of d of each dt; lanes g and g ^ 1 (of one row, so both
      // are here) trade so that one has 8 of the even dt and the other of the odd
#pragma unroll
      for (int dt = 0; dt < D / 16; dt += 2) {
        u32x4_t w;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const auto x = __builtin_amdgcn_permlane16_swap(
              pack_bf16x2(r.o[dt][rt][2 * i] * inv, r.o[dt][rt][2 * i + 1] * inv),
              pack_bf16x2(r.o[dt + 1][rt][2 * i] * inv, r.o[dt + 1][rt][2 * i + 1] * inv), false, false);
          w[i] = x[0];
          w[2 + i] = x[1];
        }
        *(u32x4_t*)(orow + (dt + (g & 1)) * 16 + 8 * (g >> 1)) = w;
      }
    }
    // (the wave's own stores to a row keep their order)
    if (again) again = none | rows_to_redo<D>(a, done.keys, done.vb, done.nk, p0, again, need, FAR, lane);
    while (again) {
      const int row = r0 + __builtin_ctz(again);
      again &= again - 1;
      const int64_t to = done.q0 + row;
      exact_row<D>(a, a.q + to * a.q_sn + (int64_t)hq * a.q_sh, done.kb, done.vb, row + done.nk - done.nq,
                   a.out + to * a.o_sn + (int64_t)hq * a.o_sh, lane);
    }
    cur = nxt;
  }
}

// A row of the call, the same in the whole wave: its sequence, and its position.
struct RowOfCall {
  Seq s;
  int p;
};
WGKV_DEVICE RowOfCall row_of_call(const WindowArgs& a, int r) {
  int b = 0;
  for (int hi = a.B - 1; b < hi;) {  // the last sequence that begins at or before the row
    const int mid = (b + hi + 1) >> 1;
    if (a.cu_q[mid] <= r) b = mid; else hi = mid - 1;
  }
  const Seq s = seq_of(a, uniform(b));
  return {s, r - s.q0 + s.nk - s.nq};
}

// The parts of every row, in order: D/4 lanes a row, four values of d each.
template <int D>
__global__ __launch_bounds__(256) void window_join_kernel(WindowArgs a) {
  constexpr int NQ = D / 4, kBatch = 8;
  const int t = threadIdx.x, lane = t & 63, vq = t % NQ, Hq = a.Hkv * a.G;
  const int64_t rows = (int64_t)a.N * Hq, rh = (int64_t)blockIdx.x * (256 / NQ) + t / NQ;
  const int64_t x = min(rh, rows - 1);
  const int row = (int)(x / Hq), hq = (int)(x - (int64_t)row * Hq);
  const bool on = rh < rows && row >= a.cu_q[0] && row < a.cu_q[a.B];
  float m = -INFINITY, l = 0.f;
  f32x4_t o = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  for (int c0 = 0; on && c0 < a.parts; c0 += kBatch) {
    float2 ml[kBatch];
    f32x4_t oc[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int64_t i = min(c0 + k, a.parts - 1) * rows + x;
      ml[k] = *(const float2*)(a.part_ml + i * 2);
      oc[k] = *(const f32x4_t*)(a.part_o + i * D + vq * 4);
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (c0 + k >= a.parts) continue;
      // (a part without keys that weigh has a sum of 0, one of scores that are no numbers a sum of NaN)
      const float mn = fmaxf(m, ml[k].x);
      const float was = m == -INFINITY && l == 0.f ? 0.f : fast_exp2(m - mn);
      const float w = ml[k].x == -INFINITY && ml[k].y == 0.f ? 0.f : fast_exp2(ml[k].x - mn);
      l = l * was + ml[k].y * w;
      o = o * was + oc[k] * w;
      m = mn;
    }
  }
  // (a sum that is NaN makes every value NaN below)
  uint64_t again = 0, left = 0;  // the first lanes of rows to be worked out on their own; rows to be looked at
  uint64_t wrong[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) left |= wrong[e] = __builtin_amdgcn_ballot_w64(on && l == l && o[e] * 0.f != 0.f);
  while (left) {
    const int from = __builtin_ctzll(left) / NQ * NQ;
    left &= ~(((1ull << NQ) - 1) << from);
    const RowOfCall w = row_of_call(a, __builtin_amdgcn_readlane(row, from));
    bool redo = w.p < 0 || __builtin_amdgcn_readlane(__float_as_int(l), from) == 0;
    if (!redo) {  // (at least the keys that its item's tiles held, wherever the item began)
      const Keys ks = keys_of(a, w.p - 127, min(w.p + 127 + attn::kKeys - 1, w.s.nk - 1));
      const int64_t kv = __builtin_amdgcn_readlane(hq, from) / a.G;
      Columns need;
#pragma unroll
      for (int e = 0; e < 4; ++e) need[e] = (uint32_t)(wrong[e] >> from) & (uint32_t)((1ull << NQ) - 1);
      redo = rows_to_redo<D>(a, ks, a.v + w.s.k0 * a.v_sn + kv * a.v_sh, w.s.nk, w.p, 1u, need, a.far, lane) != 0;
    }
    if (redo && w.p < w.s.nk) again |= 1ull << from;  // (behind the sequence's rows: starts that do not ascend)
  }
  if (on && !(again >> (lane / NQ * NQ) & 1)) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *(uint64_t*)(a.out + (int64_t)row * a.o_sn + (int64_t)hq * a.o_sh + vq * 4) =
        (uint64_t)pack_bf16x2(o[0] * inv, o[1] * inv) | (uint64_t)pack_bf16x2(o[2] * inv, o[3] * inv) << 32;
  }
  while (again) {  // a wave per row
    const int from = __builtin_ctzll(again);
    again &= again - 1;
    const int r = __builtin_amdgcn_readlane(row, from), h = __builtin_amdgcn_readlane(hq, from);
    const RowOfCall w = row_of_call(a, r);
    const int64_t kv = h / a.G;
    // (a row at p < 0 sees nothing and gets zeros here: 0 times what other rows of its
    // item see may be NaN)
    exact_row<D>(a, a.q + (int64_t)r * a.q_sn + (int64_t)h * a.q_sh, a.k + w.s.k0 * a.k_sn + kv * a.k_sh,
                 a.v + w.s.k0 * a.v_sn + kv * a.v_sh, w.p, a.out + (int64_t)r * a.o_sn + (int64_t)h * a.o_sh, lane);
  }
}

template <int D, int HPW, bool FAR>
int resident() {
  static int per_cu = 0;
  if (per_cu == 0) {
    int nb = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&nb, window_prefill_kernel<D, HPW, FAR>,
                                                     64 * item_waves(HPW), 0) !=
            hipSuccess ||
        nb <= 0)
      nb = 1;
    per_cu = nb;
  }
  return per_cu * cu_count();
}

// How a call is cut: query heads per workgroup and parts of an item.
struct Cut {
  int heads, parts;
};

int64_t items_of(int64_t N, int64_t B, int Hkv, int G, int heads) {
  return (N / item_rows(heads) + B) * Hkv * (G / heads);
}

// Heads: as many of 4, 2, 1 as divide G.
// Parts: one for each time that the items fit into the card, of kLeastTiles
// tiles at least.
// Below kLongTiles tiles the join of more parts costs what they save, and where
// workgroups of four heads leave half of the CUs without one, those of two
// do better.  Measured (D 128, 8 KV heads of 4; us for 4 heads / 2 heads / 2
// heads in twice as many parts):
//   1000 rows of 1000 keys, window 1024, 2 parts / 1 / 2   43.3 / 34.4 / 41.3
//   40 rows of 1040 keys, window 700, 2 / 2 / 2            20.5 / 18.2 / 18.3
//   1, 5, 9 rows of 3 to 5 thousand, window 2000           20.4 / 22.0 / 22.4
//   256 rows of 6256 keys, window 4096, 6 / 3 / 6          41.8 / 55.2 / 46.8
//   512 rows of 32512 keys, all, 3 / 1 / 3                 307 / 826 / 368
//   64 rows of 32064 keys, all, 16 / 8 / 16                73.7 / 116 / 68.7 (955 in one part of one head)
constexpr int kLongTiles = 32;

Cut cut_of(int N, int Nk, int B, int Hkv, int G, int window, int sinks) {
  Cut c = {4, 1};
  while (G % c.heads) c.heads >>= 1;
  const int64_t reach = (int64_t)window + item_rows(c.heads);
  const int64_t keys = (Nk < reach ? Nk : reach) + (Nk < sinks ? Nk : sinks);
  const int64_t tiles = keys / attn::kKeys, cus = cu_count();
  const bool is_long = tiles >= kLongTiles;
  if (!is_long && c.heads == 4 && items_of(N, B, Hkv, G, 2) <= cus) c.heads = 2;
  // (a long item's workgroups of four waves or fewer come two a CU)
  const int64_t by_room = (is_long && c.heads < 4 ? 2 * cus : cus) / items_of(N, B, Hkv, G, c.heads);
  const int64_t by_tiles = tiles / kLeastTiles, parts = by_room < by_tiles ? by_room : by_tiles;
  if (parts > 1) c.parts = (int)parts;
  return c;
}

size_t aligned(size_t n) { return (n + 255) & ~(size_t)255; }

struct PartsScratch {
  size_t o, bytes;
};
PartsScratch parts_scratch(int parts, int64_t rows, int D) {
  PartsScratch s = {0, 0};
  if (parts == 1) return s;
  s.o = aligned((size_t)parts * rows * 2 * sizeof(float));
  s.bytes = s.o + (size_t)parts * rows * D * sizeof(float);
  return s;
}

// Workgroups: those resident at once, at most one per item.
template <int D, int HPW, bool FAR>
hipError_t launch_items(const WindowArgs& a, hipStream_t st) {
  const int64_t items = items_of(a.N, a.B, a.Hkv, a.G, HPW) * a.parts, most = resident<D, HPW, FAR>();
  hipLaunchKernelGGL((window_prefill_kernel<D, HPW, FAR>), dim3((unsigned)(items < most ? items : most)),
                     dim3(64 * item_waves(HPW)), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.parts == 1) return e;
  const int64_t per = 256 / (D / 4);
  hipLaunchKernelGGL((window_join_kernel<D>), dim3((unsigned)(((int64_t)a.N * a.Hkv * a.G + per - 1) / per)), dim3(256),
                     0, st, a);
  return hipGetLastError();
}

template <int D, int HPW>
hipError_t launch(WindowArgs& a, hipStream_t st) {
  const int64_t bytes = ((int64_t)a.Nk + attn::kKeys) * 2 * (a.k_sn > a.v_sn ? a.k_sn : a.v_sn);
  a.far = a.k_sn < 0 || a.v_sn < 0 || bytes >= 0x7ffff000;
  return a.far ? launch_items<D, HPW, true>(a, st) : launch_items<D, HPW, false>(a, st);
}

template <int D>
hipError_t launch_heads(WindowArgs& a, int heads, hipStream_t st) {
  return heads == 4 ? launch<D, 4>(a, st) : heads == 2 ? launch<D, 2>(a, st) : launch<D, 1>(a, st);
}

bool bad_shape(int B, int N, int Nk, int Hq, int Hkv, int window, int sinks) {
  return B <= 0 || N < 0 || Nk < 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || window < 1 || sinks < 0;
}

}  // namespace

extern "C" size_t wgkv_sink_window_workspace_bytes(int32_t batch, int32_t num_rows, int32_t num_keys, int32_t num_q_heads,
                                                   int32_t num_kv_heads, int32_t head_dim, int32_t window,
                                                   int32_t num_sinks) {
  if (bad_shape(batch, num_rows, num_keys, num_q_heads, num_kv_heads, window, num_sinks) || head_dim <= 0) return 0;
  const Cut c = cut_of(num_rows, num_keys, batch, num_kv_heads, num_q_heads / num_kv_heads, window, num_sinks);
  return parts_scratch(c.parts, (int64_t)num_rows * num_q_heads, head_dim).bytes;
}

extern "C" int wgkv_sink_window_attn(
    const void* q, int64_t q_stride_n, int64_t q_stride_h,
    const void* k, int64_t k_stride_n, int64_t k_stride_h,
    const void* v, int64_t v_stride_n, int64_t v_stride_h,
    void* out, int64_t out_stride_n, int64_t out_stride_h,
    const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int32_t batch, int32_t num_rows, int32_t num_keys,
    int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t window, int32_t num_sinks, float softmax_scale, int32_t clear_rest, void* workspace, size_t workspace_bytes,
    void* stream) {
  if (bad_shape(batch, num_rows, num_keys, num_q_heads, num_kv_heads, window, num_sinks)) return WGKV_ERR_ARG;
  if (num_rows == 0) return WGKV_OK;
  if (!q || !out || !cu_seqlens_q || !cu_seqlens_k || (num_keys && (!k || !v))) return WGKV_ERR_ARG;
  const int G = num_q_heads / num_kv_heads;
  if (G > 8 || (head_dim != 64 && head_dim != 128) || batch > kMaxSeqs) return WGKV_ERR_UNSUPPORTED;
  if (num_rows > (1 << 30) || num_keys > (1 << 30)) return WGKV_ERR_UNSUPPORTED;  // positions and tiles are 32-bit
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) return WGKV_ERR_UNSUPPORTED;
  if ((q_stride_n | q_stride_h | k_stride_n | k_stride_h | v_stride_n | v_stride_h | out_stride_n | out_stride_h) & 7)
    return WGKV_ERR_UNSUPPORTED;
  if (kv4_rows_meet({num_rows, num_q_heads, 1, 1}, {out_stride_n, out_stride_h, 0, 0}, head_dim)) return WGKV_ERR_ARG;
  const Cut cut = cut_of(num_rows, num_keys, batch, num_kv_heads, G, window, num_sinks);
  const PartsScratch sc = parts_scratch(cut.parts, (int64_t)num_rows * num_q_heads, head_dim);
  // row blocks (also where starts do not ascend) and items are counted in 32 bits; workgroups step over the end
  if ((int64_t)batch * (num_rows / 64 + 1) > (1 << 30)) return WGKV_ERR_UNSUPPORTED;
  if (items_of(num_rows, batch, num_kv_heads, G, cut.heads) * cut.parts > 0x7f000000) return WGKV_ERR_UNSUPPORTED;
  if (sc.bytes && (!workspace || workspace_bytes < sc.bytes || ((uintptr_t)workspace & 15))) return WGKV_ERR_WORKSPACE;
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
  // (positions are within 2^30: a larger window shows the same, and its difference to a position stays 32-bit)
  a.window = window < (1 << 30) ? window : 1 << 30;
  a.sinks = num_sinks < (1 << 30) ? num_sinks : 1 << 30;
  // a negative scale negates the queries, and a scale of 0 clears them: masked
  // scores are -inf, and -inf * 0 is not a number
  a.scale_log2 = softmax_scale == 0.f ? 1.f : fabsf(softmax_scale) * attn::kLog2e;
  a.q_and = softmax_scale == 0.f ? 0u : ~0u;
  a.q_xor = softmax_scale < 0.f ? 0x80008000u : 0u;
  a.clear_rest = clear_rest;
  a.parts = cut.parts;
  a.part_ml = (float*)workspace;
  a.part_o = (float*)((char*)workspace + sc.o);
  hipStream_t st = (hipStream_t)stream;
  const hipError_t e = head_dim == 128 ? launch_heads<128>(a, cut.heads, st) : launch_heads<64>(a, cut.heads, st);
  return e == hipSuccess ? WGKV_OK : WGKV_ERR_HIP;
}

extern "C" int wgkv_sink_window_attn_block(const void* args) {
  int64_t a[27];
  memcpy(a, args, sizeof a);
  if (!kv4_narrow(a, 14, 15, 16, 17, 18, 19, 20, 21, 23)) return WGKV_ERR_UNSUPPORTED;
  double scale;
  memcpy(&scale, &a[22], sizeof scale);
  return wgkv_sink_window_attn((const void*)a[0], a[1], a[2], (const void*)a[3], a[4], a[5], (const void*)a[6], a[7],
                               a[8], (void*)a[9], a[10], a[11], (const int32_t*)a[12], (const int32_t*)a[13],
                               (int32_t)a[14], (int32_t)a[15], (int32_t)a[16], (int32_t)a[17], (int32_t)a[18],
                               (int32_t)a[19], (int32_t)a[20], (int32_t)a[21], (float)scale, (int32_t)a[23],
                               (void*)a[24], (size_t)a[25], (void*)a[26]);
}
