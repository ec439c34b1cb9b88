// Decode attention of large batches (gfx950): of sequences that share long
// prefixes, and of sequences that see a window and first tokens.
//
// Shared prefixes: sequences starts[n] .. starts[n+1] - 1 share prefix n: KV head h of each of
// them attends to the first prefix_lens[n, h] tokens of the prefix's pages and
// to the first lens[b, h] tokens of its own, under one softmax.
//
// The prefix is read once for all queries of its group, whose rows (sequence,
// query head of the KV head) form a matrix.
//
// Window: KV head (b, h) of T tokens shows those t with t >= T - window or t <
// first; the sub-pages of 16 tokens that hold some are counted through.
//
// There are two kinds of work:
//
// Few rows (up to 16; a sequence's own tokens have G): reading K and V is all
// that counts, so a wave streams 32 tokens at a time past one operand of rows.
//   * K comes from memory in the layout of the matrix core's A operand, and
//     S^T = K Q^T (v_mfma_f32_16x16x32_bf16) leaves each lane 8 scores of one
//     query row, which after the softmax are the B operand of O^T += V^T P^T.
//   * That A operand wants 8 tokens of one d per lane, while memory holds 8 d
//     of one token: a lane loads the 8 tokens' 16-byte pieces and exchanges
//     halves in its own registers (4 v_perm_b32 per operand), which fixes the
//     order of d over the operands (d = D/16 * m + e for row m of operand e)
//     and needs neither LDS nor other lanes.
//   * Keys are asked for two tiles ahead, values one.  Values are read without
//     being kept (8 x 128K tokens: 119 -> 104 us).
//
// Many rows (a prefix of a larger group): the matrix products count.  A
// workgroup takes 128 rows, 32 per wave, and tiles of 64 tokens that go from
// the pages straight into LDS, one tile ahead (attn_tile.h).
//
// Split: the tiles of all (prefix, head, row tile) and (sequence, head) are
// laid end to end, weighted by what they cost, and the workgroups take equal
// ranges of that line, whatever the lengths.  A workgroup goes through the
// pieces of its range.  Pieces are numbered (workgroup + position of their
// entry), store (max, sum, O) there, and a second launch joins the pieces of
// every query row in a fixed order.
#include <string.h>

#include "attn_tile.h"
#include "kv4.h"
#include "stream_attn.h"

namespace {

using attn::fmax_ieee;
using attn::xor16_max;
using attn::xor32_max;

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kMaxHeads = 2048;     // (sequence, head) pairs; (prefix, head) pairs
constexpr int kMaxG = 8;
constexpr int kWgsPerCu = 2;        // what the registers hold: two waves per SIMD
constexpr int kMaxSlots = 1024;     // workgroups of the split launch at most
constexpr int kFew = 16, kMany = 128;  // rows of a piece
// What a tile costs along the line, in quarters of a streamed tile of 32
// tokens.
constexpr int kStreamed = 4, kTiled = 8;

struct StreamArgs {
  const uint16_t* q;
  int64_t q_sb, q_sh;
  const uint16_t* kc;
  const uint16_t* vc;
  int num_pages, page_shift;  // page_size = 16 << page_shift
  const int32_t* len;
  int64_t len_sb;
  const int32_t* bt;
  int64_t bt_sb, bt_sh;
  int cap;  // tokens a row of the table has room for
  const int32_t* plen;
  int64_t plen_sb;
  const int32_t* pbt;
  int64_t pbt_sb, pbt_sh;
  int pcap;
  const int32_t* starts;
  uint16_t* out;
  int64_t out_sb, out_sh;
  int B, N, H, G;
  int window, sinks;  // windowed calls, which have no prefixes (N = 0)
  float scale_log2;
  uint32_t q_and, q_xor;
  int slots;    // workgroups of the split launch
  // pieces: (max, sum) and O of a prefix piece's rows (kFew or kMany), then of an own piece's G rows
  float* pre_ml;
  float* pre_o;
  float* own_ml;
  float* own_o;
  int* plan;  // cost before each entry, the total, and the cost of a workgroup's range
};

// A value that every lane holds, as a scalar.
WGKV_DEVICE int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

WGKV_DEVICE int clamp_to(int x, int hi) { return min(max(x, 0), hi); }

WGKV_DEVICE int group_start(const StreamArgs& a, int n) { return clamp_to(a.starts[n], a.B); }
WGKV_DEVICE int group_size(const StreamArgs& a, int n) { return max(group_start(a, n + 1) - group_start(a, n), 0); }

// What a call is: prefixes of few or many rows, or a window.
enum Mode { kFewRows, kManyRows, kWindowed };

// Tokens of a head as its tiles count them: sub-page j of the call is sub-page
// j of the head, or j + skip from `cut` on (a window's; cut is beyond the last
// one otherwise).  A window's tokens begin at `lo`, but for those below `first`.
struct Seen {
  int tokens, subs, cut, skip, lo, first;
};

template <Mode KIND>
WGKV_DEVICE Seen seen_of(const StreamArgs& a, int tokens) {
  const int all = (tokens + 15) >> 4;
  Seen x = {tokens, all, INT32_MAX, 0, 0, 0};
  if constexpr (KIND == kWindowed) {
    x.lo = max(0, tokens - a.window);
    x.first = min(tokens, a.sinks);
    const int ns = (x.first + 15) >> 4, w0 = x.lo >> 4;
    if (w0 > ns) {
      x.cut = ns;
      x.skip = w0 - ns;
      x.subs = all - x.skip;
    }
  }
  return x;
}

// Entry e of the line, prefixes first: tokens, tiles (per row tile), row tiles,
// cost of a tile.
struct Entry {
  int tokens, tiles, row_tiles, weight;
  WGKV_DEVICE int cost() const { return tiles * row_tiles * weight; }
};

template <Mode KIND>
constexpr int rows_of() { return KIND == kManyRows ? kMany : kFew; }

template <Mode KIND>
WGKV_DEVICE Entry entry_of(const StreamArgs& a, int e) {
  Entry x;
  const int NH = a.N * a.H;
  if (e < NH) {
    const int n = e / a.H, h = e - n * a.H;
    x.tokens = clamp_to(a.plen[(int64_t)n * a.plen_sb + h], a.pcap);
    x.row_tiles = (group_size(a, n) * a.G + rows_of<KIND>() - 1) / rows_of<KIND>();
    x.weight = KIND == kManyRows ? kTiled : kStreamed;
    x.tiles = KIND == kManyRows ? (x.tokens + 63) >> 6 : (x.tokens + 31) >> 5;
  } else {
    const int b = (e - NH) / a.H, h = e - NH - b * a.H;
    x.tokens = clamp_to(a.len[(int64_t)b * a.len_sb + h], a.cap);
    x.row_tiles = 1;
    x.weight = kStreamed;
    x.tiles = (seen_of<KIND>(a, x.tokens).subs + 1) >> 1;
  }
  return x;
}

// Cost of a workgroup's range: an equal share, but a streamed tile per wave at least.
WGKV_DEVICE int range_cost(int total, int slots) { return max((total + slots - 1) / slots, kWaves * kStreamed); }

// Number of a (prefix, head, row tile) that only grows along the line: groups
// before n have at most starts[n] * G / rows + n row tiles.
template <Mode KIND>
WGKV_DEVICE int64_t piece_of(const StreamArgs& a, int n, int h, int row_tile) {
  constexpr int R = rows_of<KIND>();
  const int row_tiles = (group_size(a, n) * a.G + R - 1) / R;
  return (int64_t)a.H * (group_start(a, n) * a.G / R + n) + h * row_tiles + row_tile;
}

// Pages of a head, and what the call sees of its tokens.
struct Pages {
  const int32_t* bt;
  Seen seen;
  // sub-page j of the call (scalars: see subpage_rows)
  template <Mode KIND>
  WGKV_DEVICE int sub(int j) const {
    return KIND == kWindowed && j >= seen.cut ? j + seen.skip : j;
  }
};
typedef const int32_t __attribute__((address_space(4))) ConstInt;

// Page id of a sub-page of 16 tokens (one scalar load), asked for a tile
// before its rows so that no wait for it holds those up.
WGKV_DEVICE int subpage_id(const StreamArgs& a, const Pages& p, int sp) {
  return ((ConstInt*)p.bt)[min(sp, (p.seen.tokens - 1) >> 4) >> a.page_shift];
}

// Buffer over a sub-page's valid rows: a lane's offset is the same in every
// tile, rows behind the last token read as zeros without a request (V then
// adds 0 for them whatever the pool holds), and a sub-page behind the end asks
// for nothing, so that the loads need no branch.  (A clamp to two bounds is a
// vector instruction, and a descriptor out of vector registers a loop around
// each load: hence uniform.)
template <int D>
WGKV_DEVICE __amdgpu_buffer_rsrc_t subpage_rows(const StreamArgs& a, const Pages& p, const uint16_t* pool, int sp, int id) {
  const int64_t pg = uniform(clamp_to(id, a.num_pages - 1));
  const int64_t row = (pg << (a.page_shift + 4)) + (sp & ((1 << a.page_shift) - 1)) * 16;
  const int valid = uniform(clamp_to(p.seen.tokens - sp * 16, 16));
  return __builtin_amdgcn_make_buffer_rsrc((void*)(pool + row * D), (short)0, valid * D * 2, 0x00020000);
}

// The query rows of a piece: row r is query head h * G + r % G of sequence
// b0 + r / G.
struct Queries {
  int b0, h, first, count;  // rows first .. of `count`
  WGKV_DEVICE const uint16_t* row(const StreamArgs& a, int r) const {
    r = min(first + r, count - 1);
    const int b = r / a.G;
    return a.q + (b0 + b) * a.q_sb + (h * a.G + r - b * a.G) * a.q_sh;
  }
};

// ---- few rows: streamed ------------------------------------------------------
// 32 tokens of a head: K in the A operand's layout (lane (n, g): token
// 16 * kt + n, d = 32 * j + 8 * g ..), V as 8 tokens' pieces of D/16 values
// (lane (n, g), piece s: token 4 * g + s, or 16 + 4 * g + s - 4 from s = 4 on).
template <int D>
struct KTile {
  u32x4_t k[2][D / 32];
};
template <int D>
struct VTile {
  uint32_t v[8][D / 32];
};
struct Ids {
  int pg[2];
};

template <Mode KIND>
WGKV_DEVICE Ids tile_ids(const StreamArgs& a, const Pages& p, int tile) {
  return {{subpage_id(a, p, p.sub<KIND>(2 * tile)), subpage_id(a, p, p.sub<KIND>(2 * tile + 1))}};
}

template <int D, Mode KIND>
WGKV_DEVICE void load_k(const StreamArgs& a, const Pages& p, int tile, const Ids& ids, int koff, KTile<D>& x) {
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) {
    const __amdgpu_buffer_rsrc_t r = subpage_rows<D>(a, p, a.kc, p.sub<KIND>(2 * tile + kt), ids.pg[kt]);
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
      x.k[kt][j] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, koff + j * 64, 0, 0));
  }
}

template <int D, Mode KIND>
WGKV_DEVICE void load_v(const StreamArgs& a, const Pages& p, int tile, const Ids& ids, int voff, VTile<D>& x) {
  constexpr int kNonTemporal = 2;
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) {
    const __amdgpu_buffer_rsrc_t r = subpage_rows<D>(a, p, a.vc, p.sub<KIND>(2 * tile + kt), ids.pg[kt]);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if constexpr (D == 128) {
        const u32x4_t w = __builtin_bit_cast(
            u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, voff + s * D * 2, 0, kNonTemporal));
#pragma unroll
        for (int i = 0; i < 4; ++i) x.v[kt * 4 + s][i] = w[i];
      } else {
        const auto w = __builtin_amdgcn_raw_buffer_load_b64(r, voff + s * D * 2, 0, kNonTemporal);
        x.v[kt * 4 + s][0] = w[0];
        x.v[kt * 4 + s][1] = w[1];
      }
    }
  }
}

// Running state of 16 query rows in a wave: lane (n, g) holds row n, and of O
// the values d = D/16 * (4 * g + i) + e.
template <int D>
struct Rows16 {
  bf16x8_t q[D / 32];
  f32x4_t o[D / 16];
  f32x4_t sum;
  float m;
  f32x4_t s[2];  // scores of the next tile
};

template <int D>
WGKV_DEVICE void scores(Rows16<D>& r, const KTile<D>& x) {
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) r.s[kt] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < D / 32; ++j)
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
      r.s[kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, x.k[kt][j]), r.q[j], r.s[kt], 0, 0, 0);
}

// One tile whose scores are in r.s and whose values are in x.  `reload` runs
// as soon as x is free; `next` holds the keys of the tile after it, whose
// scores replace these.
template <int D, Mode KIND, typename Reload>
WGKV_DEVICE void attend_tile(const StreamArgs& a, Rows16<D>& r, const KTile<D>& next, VTile<D>& x, const Pages& p,
                             int tile, int g, Reload reload) {
  const Seen& sn = p.seen;
  if constexpr (KIND == kWindowed) {
    // tokens of a visible sub-page that are not: no weight, and their values
    // cleared, since 0 times what is not finite is not 0
    const int t0 = p.sub<KIND>(2 * tile) * 16, t1 = p.sub<KIND>(2 * tile + 1) * 16;
    const bool all = t1 + 16 <= sn.tokens && (t0 >= sn.lo || t0 + 16 <= sn.first) && (t1 >= sn.lo || t1 + 16 <= sn.first);
    if (!all) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = (kt ? t1 : t0) + 4 * g + i;
          const bool in = t < sn.tokens && (t >= sn.lo || t < sn.first);
          r.s[kt][i] = in ? r.s[kt][i] : -INFINITY;
#pragma unroll
          for (int c = 0; c < D / 32; ++c) x.v[kt * 4 + i][c] = in ? x.v[kt * 4 + i][c] : 0u;
        }
    }
  } else {
    const int left = sn.tokens - tile * 32;
    if (left < 32) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) r.s[kt][i] = kt * 16 + 4 * g + i < left ? r.s[kt][i] : -INFINITY;
    }
  }
  float mx = r.s[0][0];
#pragma unroll
  for (int i = 1; i < 8; ++i) mx = fmax_ieee(mx, r.s[i >> 2][i & 3]);
  mx *= a.scale_log2;
  if (__builtin_amdgcn_ballot_w64(mx > r.m + attn::kSlack) != 0) {
    const float y = xor32_max(xor16_max(mx));
    const float m = y > r.m + attn::kSlack ? y : r.m;
    const float scale = m == r.m ? 1.f : fast_exp2(r.m - m);
    r.m = m;
    r.sum *= scale;
#pragma unroll
    for (int e = 0; e < D / 16; ++e) r.o[e] *= scale;
  }
  bf16x8_t vf[D / 16];
#pragma unroll
  for (int e = 0; e < D / 16; ++e) {
    u32x4_t w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = __builtin_amdgcn_perm(x.v[2 * i + 1][e / 2], x.v[2 * i][e / 2], e & 1 ? 0x07060302u : 0x05040100u);
    vf[e] = __builtin_bit_cast(bf16x8_t, w);
  }
  __builtin_amdgcn_sched_barrier(0);
  reload();
  const float m = r.m == -INFINITY ? 0.f : r.m;
  u32x4_t w;
#pragma unroll
  for (int i = 0; i < 8; i += 2)
    w[i / 2] = pack_bf16x2(fast_exp2(fmaf(r.s[i >> 2][i & 3], a.scale_log2, -m)),
                           fast_exp2(fmaf(r.s[i >> 2][(i & 3) + 1], a.scale_log2, -m)));
  const bf16x8_t pb = __builtin_bit_cast(bf16x8_t, w);
  __builtin_amdgcn_sched_barrier(0);
  scores<D>(r, next);
  const bf16x8_t ones = __builtin_bit_cast(bf16x8_t, (u32x4_t){0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
  r.sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pb, r.sum, 0, 0, 0);
#pragma unroll
  for (int e = 0; e < D / 16; ++e) r.o[e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[e], pb, r.o[e], 0, 0, 0);
}

template <int D>
constexpr int row_stride() { return D + 4; }  // LDS: rows of one operand on different banks

// A wave's 16 rows in LDS: O, then (max, sum).
template <int D>
constexpr int wave_floats() { return kFew * row_stride<D>() + 2 * kFew; }

// Tiles t0 .. t1 - 1 of a head's tokens for up to 16 rows, the waves taking
// them in turn and meeting in LDS (part[w] is wave w's).  (max, sum) and O of
// rows < rows go to ml and o.
template <int D, Mode KIND>
WGKV_DEVICE void stream_piece(const StreamArgs& a, const Pages& p, int t0, int t1, const Queries& q, int rows, float* ml,
                              float* o, float* const (&part)[kWaves]) {
  constexpr int RS = row_stride<D>();
  const int t = threadIdx.x, lane = t & 63, w = uniform(t >> 6);
  const int n = lane & 15, g = lane >> 4;
  Rows16<D> r;
  const uint16_t* row = q.row(a, n);
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    const u32x4_t x = *(const u32x4_t*)(row + (j * 4 + g) * 8);
    r.q[j] = __builtin_bit_cast(bf16x8_t, (x & a.q_and) ^ a.q_xor);
  }
  r.m = -INFINITY;
  r.sum = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < D / 16; ++e) r.o[e] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  const int koff = (n * D + g * 8) * 2, voff = (4 * g * D + n * (D / 16)) * 2;
  const auto or_none = [&](int tile) { return tile < t1 ? tile : INT32_MAX / 64; };
  int tile = t0 + w;
  if (tile < t1) {
    KTile<D> k0, k1;
    VTile<D> v;
    Ids i0 = tile_ids<KIND>(a, p, tile), i1 = tile_ids<KIND>(a, p, tile + kWaves), i2 = tile_ids<KIND>(a, p, tile + 2 * kWaves);
    load_k<D, KIND>(a, p, tile, i0, koff, k0);
    load_v<D, KIND>(a, p, tile, i0, voff, v);
    load_k<D, KIND>(a, p, or_none(tile + kWaves), i1, koff, k1);
    scores<D>(r, k0);
    // (kc: the next tile's keys, kn: its buffer; i1, i2: page ids one and two tiles on)
    const auto step = [&](KTile<D>& kc, KTile<D>& kn) __attribute__((always_inline)) {
      load_k<D, KIND>(a, p, or_none(tile + 2 * kWaves), i2, koff, kn);
      attend_tile<D, KIND>(a, r, kc, v, p, tile, g, [&] __attribute__((always_inline)) () {
        load_v<D, KIND>(a, p, or_none(tile + kWaves), i1, voff, v);
        i1 = i2;
        i2 = tile_ids<KIND>(a, p, tile + 3 * kWaves);
      });
      tile += kWaves;
    };
    for (;;) {
      step(k1, k0);
      if (tile >= t1) break;
      step(k0, k1);
      if (tile >= t1) break;
    }
  }
  float* mine = w == 0 ? part[0] : w == 1 ? part[1] : w == 2 ? part[2] : part[3];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < D / 16; e += 4)
      *(f32x4_t*)(mine + n * RS + (D / 16) * (4 * g + i) + e) = (f32x4_t){r.o[e][i], r.o[e + 1][i], r.o[e + 2][i], r.o[e + 3][i]};
  if (g == 0) {
    mine[kFew * RS + 2 * n] = r.m;
    mine[kFew * RS + 2 * n + 1] = r.sum[0];
  }
  __syncthreads();
  for (int i = t; i < rows * (D / 4); i += kThreads) {
    const int at = i / (D / 4), d = (i - at * (D / 4)) * 4;
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) m = fmaxf(m, part[k][kFew * RS + 2 * at]);
    f32x4_t sum = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
      const float mk = part[k][kFew * RS + 2 * at], lk = part[k][kFew * RS + 2 * at + 1];
      // a sum of 0 (no token that weighs) has no part; one of NaN (its scores
      // were) has, whatever its maximum
      const float c = mk == -INFINITY && lk == 0.f ? 0.f : fast_exp2(mk - m);
      l += c * lk;
      sum += c * *(const f32x4_t*)(part[k] + at * RS + d);
    }
    *(f32x4_t*)(o + (int64_t)at * D + d) = sum;
    if (d == 0) {
      ml[at * 2] = m;
      ml[at * 2 + 1] = l;
    }
  }
  __syncthreads();
}

// ---- many rows: tiles in LDS ----------------------------------------------------
// 16 bytes of the buffer at `off` (zeros behind its end) go to LDS at lds + 16 * lane.
WGKV_DEVICE void buffer_to_lds(__amdgpu_buffer_rsrc_t r, uint16_t* lds, int off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, lds, 16, off, 0, 0, 0);
}

// Tiles t0 .. t1 - 1 of 64 tokens for `rows` <= 128 rows, 32 per wave.  Wave w
// loads sub-page w of every tile.
template <int D>
WGKV_DEVICE void tile_piece(const StreamArgs& a, const Pages& p, int t0, int t1, const Queries& q, int rows, float* ml,
                            float* o, uint16_t* sK0, uint16_t* sV0, uint16_t* sK1, uint16_t* sV1) {
  constexpr int CH = D / 8, RPB = 64 / CH, NB = 16 / RPB;  // slices of a row, rows of 1 KB, KBs of a sub-page
  const int t = threadIdx.x, lane = t & 63, w = uniform(t >> 6);
  const int n = lane & 15, g = lane >> 4;
  const attn::Offsets<D> at(n, g);
  attn::Rows32<D> r;
  r.clear();
#pragma unroll
  for (int rt = 0; rt < 2; ++rt) r.load_q(rt, q.row(a, w * 32 + rt * 16 + n), g, a.q_and, a.q_xor);
  int koff[NB], voff[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int row = i * RPB + lane / CH;
    koff[i] = row * D * 2 + ((lane % CH) ^ attn::swz_k<D>(row)) * 16;
    voff[i] = row * D * 2 + ((lane % CH) ^ attn::swz_v<D>(row)) * 16;
  }
  const auto load = [&](int tile, int id, uint16_t* sK, uint16_t* sV) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t k = subpage_rows<D>(a, p, a.kc, 4 * tile + w, id);
    const __amdgpu_buffer_rsrc_t v = subpage_rows<D>(a, p, a.vc, 4 * tile + w, id);
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      buffer_to_lds(k, sK + (w * NB + i) * 512, koff[i]);
      buffer_to_lds(v, sV + (w * NB + i) * 512, voff[i]);
    }
  };
  int id = subpage_id(a, p, 4 * t0 + w);
  load(t0, id, sK0, sV0);
  id = subpage_id(a, p, 4 * (t0 + 1) + w);
  const auto step = [&](int tile, const uint16_t* sK, const uint16_t* sV, uint16_t* nK, uint16_t* nV)
      __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's part of the tile has landed
    __syncthreads();                     // every wave's has, and nobody reads the other buffer any more
    if (tile + 1 < t1) {
      load(tile + 1, id, nK, nV);
      id = subpage_id(a, p, 4 * (tile + 2) + w);
    }
    if (w * 32 >= rows) return;
    f32x4_t sc[4][2];
    attn::tile_scores<D>(r, sK, at, sc);
    const int left = p.seen.tokens - tile * 64;
    if (left < 64) {
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = kt * 16 + 4 * g + i < left;
#pragma unroll
          for (int rt = 0; rt < 2; ++rt) sc[kt][rt][i] = in ? sc[kt][rt][i] : -INFINITY;
        }
    }
    attn::tile_attend<D>(r, sc, sV, at, a.scale_log2);
  };
  for (int tile = t0; tile < t1; tile += 2) {
    step(tile, sK0, sV0, sK1, sV1);
    if (tile + 1 < t1) step(tile + 1, sK1, sV1, sK0, sV0);
  }
#pragma unroll
  for (int rt = 0; rt < 2; ++rt) {
    const int row = w * 32 + rt * 16 + n;
    if (row >= rows) continue;
    if (g == 0) {
      ml[row * 2] = r.m[rt];
      ml[row * 2 + 1] = r.sum[rt][0];
    }
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) *(f32x4_t*)(o + (int64_t)row * D + dt * 16 + 4 * g) = r.o[dt][rt];
  }
  __syncthreads();  // the buffers are free
}

template <int D, Mode KIND>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(kWgsPerCu, kWgsPerCu)))
void stream_split_kernel(StreamArgs a) {
  // four objects: loads into one tile buffer then provably leave the others
  // alone; between pieces they hold the waves' rows
  constexpr int kLds = KIND == kManyRows ? attn::kKeys * D * 2 : wave_floats<D>() * 4;
  static_assert(kLds >= wave_floats<D>() * 4, "a wave's rows fit a tile buffer");
  __shared__ __attribute__((aligned(16))) uint16_t s0[kLds / 2];
  __shared__ __attribute__((aligned(16))) uint16_t s1[kLds / 2];
  __shared__ __attribute__((aligned(16))) uint16_t s2[kLds / 2];
  __shared__ __attribute__((aligned(16))) uint16_t s3[kLds / 2];
  // (many rows: at least 17 per prefix, so N * H <= 2048 * 8 / 17)
  __shared__ int s_base[kMaxHeads + (KIND == kManyRows ? 1024 : KIND == kFewRows ? kMaxHeads : 0) + 1];
  __shared__ int s_tmp[4];
  const int t = threadIdx.x, wg = blockIdx.x;
  const int NH = a.N * a.H, E = NH + a.B * a.H;
  // cost before every entry, the same in every workgroup
  const int per_thread = (E + kThreads - 1) / kThreads;
  const int e0 = min(E, t * per_thread), e1 = min(E, e0 + per_thread);
  int mine = 0, total;
  for (int e = e0; e < e1; ++e) mine += entry_of<KIND>(a, e).cost();
  int run = block_exclusive_scan_256(mine, s_tmp, &total);
  for (int e = e0; e < e1; ++e) {
    s_base[e] = run;
    run += entry_of<KIND>(a, e).cost();
  }
  if (t == 0) s_base[E] = total;
  __syncthreads();
  total = uniform(total);
  const int per = uniform(range_cost(total, a.slots));
  if (wg == 0) {
    for (int i = t; i <= E; i += kThreads) a.plan[i] = s_base[i];
    if (t == 0) a.plan[E + 1] = per;
  }
  const int lo = (int)min((int64_t)wg * per, (int64_t)total), hi = (int)min((int64_t)lo + per, (int64_t)total);
  if (lo >= hi) return;
  int first = 0, last = E - 1;  // the last entry that begins at or before lo
  while (first < last) {
    const int mid = (first + last + 1) >> 1;
    if (uniform(s_base[mid]) <= lo) first = mid; else last = mid - 1;
  }
  for (int e = first; e < E; ++e) {
    const int base = uniform(s_base[e]);
    if (base >= hi) break;
    if (uniform(s_base[e + 1]) == base) continue;
    Entry x = entry_of<KIND>(a, e);
    x.tokens = uniform(x.tokens);
    x.tiles = uniform(x.tiles);
    x.row_tiles = uniform(x.row_tiles);
    // the entry's tiles (row tile after row tile) that begin in [lo, hi)
    int u0 = uniform(max(0, (lo - base + x.weight - 1) / x.weight));
    const int u1 = uniform(min(x.tiles * x.row_tiles, (hi - base + x.weight - 1) / x.weight));
    while (u0 < u1) {
      const int row_tile = uniform(u0 / x.tiles), t0 = u0 - row_tile * x.tiles;
      const int t1 = min(x.tiles, t0 + u1 - u0);
      u0 += t1 - t0;
      Queries q;
      Pages p;
      float *ml, *o;
      const bool pre = KIND != kWindowed && e < NH;
      constexpr int R = rows_of<KIND>();
      if (pre) {
        const int n = uniform(e / a.H);
        q.h = e - n * a.H;
        q.b0 = uniform(group_start(a, n));
        q.first = row_tile * R;
        q.count = uniform(group_size(a, n)) * a.G;
        p.bt = a.pbt + n * a.pbt_sb + q.h * a.pbt_sh;
        const int64_t id = wg + piece_of<KIND>(a, n, q.h, row_tile);
        ml = a.pre_ml + id * (R * 2);
        o = a.pre_o + id * (R * D);
      } else {
        const int bh = e - NH;
        q.b0 = uniform(bh / a.H);
        q.h = bh - q.b0 * a.H;
        q.first = 0;
        q.count = a.G;
        p.bt = a.bt + q.b0 * a.bt_sb + q.h * a.bt_sh;
        const int64_t id = wg + bh;
        ml = a.own_ml + id * (a.G * 2);
        o = a.own_o + id * (a.G * D);
      }
      p.seen = seen_of<KIND>(a, x.tokens);
      const int rows = min(R, q.count - q.first);
      if (KIND == kManyRows && pre) {
        tile_piece<D>(a, p, t0, t1, q, rows, ml, o, s0, s1, s2, s3);
      } else {
        float* const part[kWaves] = {(float*)s0, (float*)s1, (float*)s2, (float*)s3};
        stream_piece<D, KIND>(a, p, t0, t1, q, rows, ml, o, part);
      }
    }
  }
}

// The pieces of a query row under one softmax, in the order of the line: one
// workgroup per (sequence, KV head, query head), a thread group of D/4
// threads per piece in turn, then the groups in order.
template <int D, Mode KIND>
__global__ __launch_bounds__(256) void stream_merge_kernel(StreamArgs a) {
  constexpr int NQ = D / 4, GROUPS = 256 / NQ, kBatch = 8, R = rows_of<KIND>();
  __shared__ f32x4_t s_a[256];
  __shared__ float s_m[256], s_l[256];
  const int bh = blockIdx.x, b = bh / a.H, h = bh - b * a.H, gq = blockIdx.y;
  const int t = threadIdx.x, vq = t % NQ, grp = t / NQ;
  const int NH = a.N * a.H;
  const int per = a.plan[NH + a.B * a.H + 1];
  int n_pre = 0;
  const float *pre_ml = nullptr, *pre_o = nullptr;
  if constexpr (KIND != kWindowed) {
    int lo = 0, hi = a.N;  // the last group that starts at or before b
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (group_start(a, mid) <= b) lo = mid; else hi = mid;
    }
    const int at = b - group_start(a, lo);
    if (at >= 0 && at < group_size(a, lo)) {
      const int e = lo * a.H + h;
      const Entry x = entry_of<KIND>(a, e);
      if (x.tiles) {
        const int row = at * a.G + gq, row_tile = row / R;
        const int64_t base = a.plan[e] + (int64_t)row_tile * x.tiles * x.weight;
        const int w0 = (int)(base / per), w1 = (int)((base + (int64_t)(x.tiles - 1) * x.weight) / per);
        n_pre = w1 - w0 + 1;
        const int64_t first = (w0 + piece_of<KIND>(a, lo, h, row_tile)) * R + row - row_tile * R;
        pre_ml = a.pre_ml + first * 2;
        pre_o = a.pre_o + first * D;
      }
    }
  }
  int n_own = 0;
  const float *own_ml = nullptr, *own_o = nullptr;
  const Entry x = entry_of<KIND>(a, NH + bh);
  if (x.tiles) {
    const int base = a.plan[NH + bh];
    const int w0 = base / per, w1 = (base + (x.tiles - 1) * x.weight) / per;
    n_own = w1 - w0 + 1;
    const int64_t first = ((int64_t)w0 + bh) * a.G + gq;
    own_ml = a.own_ml + first * 2;
    own_o = a.own_o + first * D;
  }
  const int pieces = n_pre + n_own;
  float M = -INFINITY, L = 0.f;
  f32x4_t A = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  for (int c0 = grp; c0 < pieces; c0 += GROUPS * kBatch) {
    float mc[kBatch], lc[kBatch];
    f32x4_t ac[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int c = min(c0 + k * GROUPS, pieces - 1);
      const bool pre = c < n_pre;
      const int64_t i = pre ? (int64_t)c * R : (int64_t)(c - n_pre) * a.G;
      const float* ml = (pre ? pre_ml : own_ml) + i * 2;
      mc[k] = ml[0];
      lc[k] = ml[1];
      ac[k] = *(const f32x4_t*)((pre ? pre_o : own_o) + i * D + vq * 4);
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      // (a row whose every score is NaN keeps its maximum at -inf and a sum of NaN)
      if (c0 + k * GROUPS >= pieces || (mc[k] == -INFINITY && lc[k] == 0.f)) continue;
      const float mn = fmaxf(M, mc[k]);
      const float sa = M == -INFINITY && L == 0.f ? 0.f : fast_exp2(M - mn);
      const float sb = fast_exp2(mc[k] - mn);
      L = L * sa + lc[k] * sb;
      A = A * sa + ac[k] * sb;
      M = mn;
    }
  }
  s_m[t] = M;
  s_l[t] = L;
  s_a[t] = A;
  __syncthreads();
  if (t >= NQ) return;
  float Mx = -INFINITY;
  for (int i = 0; i < GROUPS; ++i) Mx = fmaxf(Mx, s_m[i * NQ + t]);
  float Lt = 0.f;
  f32x4_t At = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < GROUPS; ++i) {
    const float m = s_m[i * NQ + t];
    if (m == -INFINITY && s_l[i * NQ + t] == 0.f) continue;
    const float c = fast_exp2(m - Mx);
    Lt += c * s_l[i * NQ + t];
    At += c * s_a[i * NQ + t];
  }
  uint16_t* o = a.out + b * a.out_sb + (int64_t)(h * a.G + gq) * a.out_sh + vq * 4;
  const float inv = 1.f / Lt;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = Lt == 0.f ? 0 : f32_to_bf16(At[e] * inv);
}

// Whether an even share of the batch has more rows than one operand.
bool many_rows(int B, int N, int G) { return (int64_t)B * G > (int64_t)kFew * N; }

struct Scratch {
  int64_t pre, own;  // pieces
  size_t pre_ml, pre_o, own_ml, own_o, bytes;
};

size_t aligned(size_t n) { return (n + 255) & ~(size_t)255; }

constexpr size_t kPlanBytes = ((2 * kMaxHeads + 2) * sizeof(int) + 255) & ~(size_t)255;

Scratch scratch_for(int B, int N, int G, int H, int D) {
  const int R = many_rows(B, N, G) ? kMany : kFew;
  Scratch s;
  s.pre = kMaxSlots + (int64_t)H * ((int64_t)B * G / R + N + 1);
  s.own = kMaxSlots + (int64_t)B * H;
  s.pre_ml = kPlanBytes;
  s.pre_o = s.pre_ml + aligned(s.pre * R * 2 * sizeof(float));
  s.own_ml = s.pre_o + aligned(s.pre * R * D * sizeof(float));
  s.own_o = s.own_ml + aligned(s.own * G * 2 * sizeof(float));
  s.bytes = s.own_o + aligned(s.own * G * D * sizeof(float));
  return s;
}

template <int D, Mode KIND>
hipError_t launch(StreamArgs& a, hipStream_t st) {
  a.slots = min(kMaxSlots, cu_count() * kWgsPerCu);
  hipLaunchKernelGGL((stream_split_kernel<D, KIND>), dim3(a.slots), dim3(kThreads), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((stream_merge_kernel<D, KIND>), dim3(a.B * a.H, a.G), dim3(256), 0, st, a);
  return hipGetLastError();
}

template <int D>
hipError_t launch_rows(StreamArgs& a, bool many, hipStream_t st) {
  return many ? launch<D, kManyRows>(a, st) : launch<D, kFewRows>(a, st);
}

}  // namespace

// Bytes of `scratch` (any contents) for wgkv_stream_window.
size_t wgkv_stream_window_bytes(int B, int H, int G, int D) {
  return kPlanBytes + aligned(((size_t)kMaxSlots + (size_t)B * H) * G * 2 * sizeof(float)) +
         aligned(((size_t)kMaxSlots + (size_t)B * H) * G * D * sizeof(float));
}

// The windowed call for batches of many heads (arguments checked by the caller).
int wgkv_stream_window(const StreamWindow& w, void* scratch, hipStream_t st) {
  StreamArgs a{};
  a.q = w.q;
  a.q_sb = w.q_sb;
  a.q_sh = w.q_sh;
  a.kc = w.kc;
  a.vc = w.vc;
  a.num_pages = (int)(w.num_pages < 0x7fffffff ? w.num_pages : 0x7fffffff);
  a.page_shift = w.page_shift;
  a.len = w.len;
  a.len_sb = w.len_sb;
  a.bt = w.bt;
  a.bt_sb = w.bt_sb;
  a.bt_sh = w.bt_sh;
  a.cap = w.cap;
  a.out = w.out;
  a.out_sb = w.out_sb;
  a.out_sh = w.out_sh;
  a.B = w.B;
  a.H = w.H;
  a.G = w.G;
  a.window = w.window;
  a.sinks = w.sinks;
  a.scale_log2 = w.scale_log2;
  a.q_and = w.q_and;
  a.q_xor = w.q_xor;
  char* s = (char*)scratch;
  a.plan = (int*)s;
  a.own_ml = (float*)(s + kPlanBytes);
  a.own_o = (float*)(s + kPlanBytes + aligned(((size_t)kMaxSlots + (size_t)w.B * w.H) * w.G * 2 * sizeof(float)));
  const hipError_t e = w.D == 128 ? launch<128, kWindowed>(a, st) : launch<64, kWindowed>(a, st);
  return e == hipSuccess ? WGKV_OK : WGKV_ERR_HIP;
}

extern "C" size_t wgkv_shared_decode_workspace_bytes(int32_t batch, int32_t num_groups, int32_t num_q_heads,
                                                     int32_t num_kv_heads, int32_t head_dim) {
  if (batch <= 0 || num_groups <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads || head_dim <= 0) return 0;
  return scratch_for(batch, num_groups, num_q_heads / num_kv_heads, num_kv_heads, head_dim).bytes;
}

extern "C" int wgkv_shared_decode_attn(
    const void* q, int64_t q_stride_b, int64_t q_stride_h,
    const void* k_cache, const void* v_cache, int64_t num_pages, int32_t page_size,
    const int32_t* cache_seqlens, int64_t sl_stride_b,
    const int32_t* block_table, int64_t bt_stride_b, int64_t bt_stride_h, int32_t max_pages,
    const int32_t* prefix_lens, int64_t pl_stride_n,
    const int32_t* prefix_table, int64_t pt_stride_n, int64_t pt_stride_h, int32_t prefix_pages,
    const int32_t* group_starts, int32_t num_groups,
    void* out, int64_t out_stride_b, int64_t out_stride_h,
    int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    float softmax_scale, void* workspace, size_t workspace_bytes, void* stream) {
  if (!q || !k_cache || !v_cache || !cache_seqlens || !block_table || !prefix_lens || !prefix_table || !group_starts ||
      !out)
    return WGKV_ERR_ARG;
  if (batch <= 0 || num_groups <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads)
    return WGKV_ERR_ARG;
  if (num_pages <= 0 || max_pages <= 0 || prefix_pages <= 0) return WGKV_ERR_ARG;
  const int G = num_q_heads / num_kv_heads;
  if (G > kMaxG || (head_dim != 64 && head_dim != 128)) return WGKV_ERR_UNSUPPORTED;
  if (page_size != 16 && page_size != 32 && page_size != 64) return WGKV_ERR_UNSUPPORTED;
  const int64_t own = (int64_t)batch * num_kv_heads, pre = (int64_t)num_groups * num_kv_heads;
  if (own > kMaxHeads || pre > kMaxHeads) return WGKV_ERR_UNSUPPORTED;
  // positions and the line's length are 32-bit
  const int64_t cap = (int64_t)max_pages * page_size, pcap = (int64_t)prefix_pages * page_size;
  if (cap > 0x7fffff00 || pcap > 0x7fffff00) return WGKV_ERR_UNSUPPORTED;
  const bool many = many_rows(batch, num_groups, G);
  const int64_t row_tiles = (int64_t)batch * G / (many ? kMany : kFew) + num_groups;
  if ((cap + 31) / 32 * own * kStreamed + (pcap + 31) / 32 * row_tiles * num_kv_heads * (many ? kTiled : kStreamed) >
      0x70000000)
    return WGKV_ERR_UNSUPPORTED;
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) return WGKV_ERR_UNSUPPORTED;
  if ((q_stride_b | q_stride_h) & 7) return WGKV_ERR_UNSUPPORTED;
  if (kv4_rows_meet({batch, num_q_heads, 1, 1}, {out_stride_b, out_stride_h, 0, 0}, head_dim)) return WGKV_ERR_ARG;
  const Scratch sc = scratch_for(batch, num_groups, G, num_kv_heads, head_dim);
  if (!workspace || workspace_bytes < sc.bytes || ((uintptr_t)workspace & 15)) return WGKV_ERR_WORKSPACE;
  StreamArgs a{};
  a.q = (const uint16_t*)q;
  a.q_sb = q_stride_b;
  a.q_sh = q_stride_h;
  a.kc = (const uint16_t*)k_cache;
  a.vc = (const uint16_t*)v_cache;
  a.num_pages = (int)(num_pages < 0x7fffffff ? num_pages : 0x7fffffff);  // (ids are 32-bit)
  a.page_shift = page_size == 16 ? 0 : page_size == 32 ? 1 : 2;
  a.len = cache_seqlens;
  a.len_sb = sl_stride_b;
  a.bt = block_table;
  a.bt_sb = bt_stride_b;
  a.bt_sh = bt_stride_h;
  a.cap = (int)cap;
  a.plen = prefix_lens;
  a.plen_sb = pl_stride_n;
  a.pbt = prefix_table;
  a.pbt_sb = pt_stride_n;
  a.pbt_sh = pt_stride_h;
  a.pcap = (int)pcap;
  a.starts = group_starts;
  a.out = (uint16_t*)out;
  a.out_sb = out_stride_b;
  a.out_sh = out_stride_h;
  a.B = batch;
  a.N = num_groups;
  a.H = num_kv_heads;
  a.G = G;
  // a negative scale negates the queries, and a scale of 0 clears them (the
  // maximum is taken over the products, and -inf * 0 is not a number)
  a.scale_log2 = softmax_scale == 0.f ? 1.f : fabsf(softmax_scale) * attn::kLog2e;
  a.q_and = softmax_scale == 0.f ? 0u : ~0u;
  a.q_xor = softmax_scale < 0.f ? 0x80008000u : 0u;
  char* ws = (char*)workspace;
  a.plan = (int*)ws;
  a.pre_ml = (float*)(ws + sc.pre_ml);
  a.pre_o = (float*)(ws + sc.pre_o);
  a.own_ml = (float*)(ws + sc.own_ml);
  a.own_o = (float*)(ws + sc.own_o);
  hipStream_t st = (hipStream_t)stream;
  const hipError_t e = head_dim == 128 ? launch_rows<128>(a, many, st) : launch_rows<64>(a, many, st);
  return e == hipSuccess ? WGKV_OK : WGKV_ERR_HIP;
}

extern "C" int wgkv_shared_decode_attn_block(const void* args) {
  int64_t a[32];
  memcpy(a, args, sizeof a);
  if (!kv4_narrow(a, 6, 12, 18, 20, 24, 25, 26, 27)) return WGKV_ERR_UNSUPPORTED;
  double scale;
  memcpy(&scale, &a[28], sizeof scale);
  return wgkv_shared_decode_attn(
      (const void*)a[0], a[1], a[2], (const void*)a[3], (const void*)a[4], a[5], (int32_t)a[6], (const int32_t*)a[7],
      a[8], (const int32_t*)a[9], a[10], a[11], (int32_t)a[12], (const int32_t*)a[13], a[14], (const int32_t*)a[15],
      a[16], a[17], (int32_t)a[18], (const int32_t*)a[19], (int32_t)a[20], (void*)a[21], a[22], a[23], (int32_t)a[24],
      (int32_t)a[25], (int32_t)a[26], (int32_t)a[27], (float)scale, (void*)a[29], (size_t)a[30], (void*)a[31]);
}
