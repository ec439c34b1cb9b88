// Decode attention of large batches (gfx950): of sequences that share long
// prefixes, and of sequences that see a window and first tokens.
//
// Shared prefixes: sequences starts[n] .. starts[n+1] - 1 share prefix n: KV head h of each of
// them attends to the first prefix_lens[n, h] tokens of the prefix's pages and
// to the first lens[b, h] tokens of its own, under one softmax.
//
// The queries of a group are the rows (sequence, query head of the KV head) of a
// matrix; its prefix is read once per 16 rows or once per 256, as one choice for
// the whole call from the average group (many_rows).
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
// workgroup of eight waves takes 256 rows, 32 per wave, and tiles of 64 tokens
// that go from the pages straight into LDS, one tile ahead (attn_tile.h).
//
// Split: the tiles of all (prefix, head, row tile) and (sequence, head) are
// laid end to end and the waves take equal ranges of that line, whatever the
// lengths (half of the waves those of a short line); a wave goes through the
// pieces of its range without draining its loads.  Prefixes of many rows are
// not on the line: they are cut into chunks of equal size, one per workgroup
// where that can be, and the workgroups' waves have their ranges of the line
// besides.  One half of the workgroups begins with the prefix and the other
// with the sequences' own tokens, so that some compute while others read.
// Pieces are numbered (range + position of their entry, or the chunk), store
// (max, sum, O) there, and a second launch joins the pieces of every query row
// in a fixed order.
//
// Measured (us, split + join): 64 windows of 4160 of 8 heads, D 128, 1.09 GB:
// 174 + 6, 6.2 TB/s, more than a copy of the same size reaches (reads only); 128
// sequences, G 4, of 26000 tokens in one prefix of 8 heads: 68, 805 TFLOP/s, of
// which 9 us are the way to the first tile and 10 the join; 4 sequences behind
// 2048 tokens: 11 + 5, a chain of launch, plan, page ids, keys.
#include <string.h>

#include "attn_tile.h"
#include "kv4.h"
#include "stream_attn.h"

namespace {

using attn::fmax_ieee;
using attn::xor16_max;
using attn::xor32_max;

constexpr int kMaxHeads = 2048;     // (sequence, head) pairs; (prefix, head) pairs
constexpr int kMaxG = 8;
constexpr int kWavesPerCu = 8;      // what the registers hold: two per SIMD
constexpr int kMaxWaves = 4096;     // of the split launch
constexpr int kFew = 16, kMany = 256;  // rows of a piece
constexpr int kLeastStreamed = 2, kShortRange = 6;  // tiles of 32 tokens of a wave's range
constexpr int kLeastTiled = 2;  // tiles of 64 tokens of a chunk

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
  // tiles (prefixes of many rows: chunks) before each entry and in all, tiles of
  // a chunk and of a range of the line, groups' first sequences
  int* plan;
};

// A value that every lane holds, as a scalar.
WGKV_DEVICE int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

WGKV_DEVICE int clamp_to(int x, int hi) { return min(max(x, 0), hi); }

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

template <Mode KIND>
constexpr int rows_of() { return KIND == kManyRows ? kMany : kFew; }

// Tokens of entry e of the call, prefixes (prefix, head) first, then (sequence,
// head).
WGKV_DEVICE int entry_tokens(const StreamArgs& a, int e) {
  const int NH = a.N * a.H;
  if (e < NH) {
    const int n = e / a.H, h = e - n * a.H;
    return clamp_to(a.plen[(int64_t)n * a.plen_sb + h], a.pcap);
  }
  const int b = (e - NH) / a.H, h = e - NH - b * a.H;
  return clamp_to(a.len[(int64_t)b * a.len_sb + h], a.cap);
}

// Tiles of an entry's tokens (per row tile), and row tiles of a group.
template <Mode KIND>
WGKV_DEVICE int entry_tiles(const StreamArgs& a, bool pre, int tokens) {
  if (KIND == kManyRows && pre) return (tokens + 63) >> 6;
  return (seen_of<KIND>(a, tokens).subs + 1) >> 1;
}
template <Mode KIND>
WGKV_DEVICE int row_tiles(const StreamArgs& a, int size) { return (size * a.G + rows_of<KIND>() - 1) / rows_of<KIND>(); }

// Tiles of a range of the line: an equal share of all waves, or of half of them
// (one per SIMD) while that is short: then the pieces to join count as much as
// the reads.  (4 sequences behind one prefix, 8 heads, us with shares of all / of
// half: 8192 tokens 24.8 / 20.9, 16384 30.2 / 24.9, 24000 34.4 / 29.6, 32768 40.7 /
// 46.7.)  But kLeastStreamed at least (2048 tokens: 1 15.7, 2 14.5, 3 15.7; 300
// tokens: 11.4, 12.5, 14.6).  Beside prefixes of many rows all workgroups are
// there anyway (32 sequences of 500 tokens behind 3000: 31.3 / 35.4).
template <Mode KIND>
WGKV_DEVICE int range_tiles(int total, int waves) {
  const int of_half = (total + waves / 2 - 1) / (waves / 2);
  return max(KIND != kManyRows && of_half <= kShortRange ? of_half : (total + waves - 1) / waves, kLeastStreamed);
}

// Prefixes of few rows: number of a (prefix, head, row tile) that only grows
// along the line: groups before n have at most starts[n] * G / 16 + n row tiles.
WGKV_DEVICE int piece_of(const StreamArgs& a, int start, int size, int n, int h, int row_tile) {
  return a.H * (start * a.G / kFew + n) + h * row_tiles<kFewRows>(a, size) + row_tile;
}

// Prefixes of many rows: every (prefix, head, row tile) is cut into chunks of
// equal size, so that a workgroup has one where their number allows it (a
// second piece costs it 14 us of 70): at most `slots` chunks while there are
// half as many row tiles.
WGKV_DEVICE int chunk_tiles(int total, int row_tiles, int slots) {
  const int left = max(slots - row_tiles, slots / 2);
  return max((total + left - 1) / left, kLeastTiled);
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

// What the workgroup keeps of the call's plan in LDS.
struct Plan {
  const int* base;   // tiles of the entries before (prefixes of many rows: chunks)
  const int* tokens;
  const int* start;  // groups' first sequences
};

// A tile on its way through a wave: page ids are asked for three tiles before
// it is attended to, keys two, values one.
struct Stage {
  int pos;             // on the line; >= the range's end: none
  int e, row_tile;     // its entry
  int tile, t1;        // within the entry's row tile; the piece's end
  int tokens;
  bool first;          // of its piece
  Ids ids;
};

template <int D, Mode KIND>
struct Stream {
  const StreamArgs& a;
  const Plan& plan;
  int NH, zero, hi, range;
  int n, g;

  WGKV_DEVICE const int32_t* table(int e) const {
    if (KIND != kWindowed && e < NH) {
      const int i = uniform(e / a.H);
      return a.pbt + i * a.pbt_sb + (e - i * a.H) * a.pbt_sh;
    }
    const int b = uniform((e - NH) / a.H);
    return a.bt + b * a.bt_sb + (e - NH - b * a.H) * a.bt_sh;
  }

  // The stage at position pos, which lies in entry e or behind it.
  WGKV_DEVICE Stage at(int pos, int e) const {
    Stage x = {pos, e, 0, 0, 0, 1, true, {{0, 0}}};
    if (pos >= hi) return x;
    int next = uniform(plan.base[e + 1]) - zero;
    while (next <= pos) next = uniform(plan.base[++e + 1]) - zero;
    x.e = e;
    x.tokens = uniform(plan.tokens[e]);
    const int begin = uniform(plan.base[e]) - zero, tiles = uniform(entry_tiles<KIND>(a, e < NH, x.tokens));
    x.row_tile = KIND == kFewRows ? uniform((pos - begin) / tiles) : 0;
    x.tile = pos - begin - x.row_tile * tiles;
    x.t1 = min(tiles, x.tile + hi - pos);
    return x;
  }
  WGKV_DEVICE Stage after(const Stage& s) const {
    if (s.tile + 1 < s.t1) {
      Stage x = s;
      ++x.pos;
      ++x.tile;
      x.first = false;
      return x;
    }
    return at(s.pos + 1, s.e);
  }
  WGKV_DEVICE Pages pages(const Stage& s) const { return {table(s.e), seen_of<KIND>(a, s.tokens)}; }
  WGKV_DEVICE void ask_ids(Stage& s) const {
    if (s.pos < hi) s.ids = tile_ids<KIND>(a, pages(s), s.tile);
  }
  WGKV_DEVICE int tile_or_none(const Stage& s) const { return s.pos < hi ? s.tile : INT32_MAX / 64; }
  WGKV_DEVICE Pages seen_pages(const Stage& s) const { return {nullptr, seen_of<KIND>(a, s.tokens)}; }

  WGKV_DEVICE Queries queries(const Stage& s) const {
    Queries q;
    if (KIND != kWindowed && s.e < NH) {
      const int i = uniform(s.e / a.H);
      q.h = s.e - i * a.H;
      q.b0 = uniform(plan.start[i]);
      q.first = s.row_tile * kFew;
      q.count = (uniform(plan.start[i + 1]) - q.b0) * a.G;
    } else {
      q.b0 = uniform((s.e - NH) / a.H);
      q.h = s.e - NH - q.b0 * a.H;
      q.first = 0;
      q.count = a.G;
    }
    return q;
  }
  WGKV_DEVICE void load_q(const Stage& s, u32x4_t (&q)[D / 32]) const {
    const uint16_t* row = queries(s).row(a, n);
#pragma unroll
    for (int j = 0; j < D / 32; ++j) q[j] = *(const u32x4_t*)(row + (j * 4 + g) * 8);
  }

  // (max, sum) and O of the stage's piece, and the state for the next one.
  WGKV_DEVICE void flush(const Stage& s, Rows16<D>& r) const {
    float *ml, *o;
    int rows;
    if (KIND != kWindowed && s.e < NH) {
      const int i = uniform(s.e / a.H), start = uniform(plan.start[i]), size = uniform(plan.start[i + 1]) - start;
      const int64_t id = range + piece_of(a, start, size, i, s.e - i * a.H, s.row_tile);
      ml = a.pre_ml + id * (kFew * 2);
      o = a.pre_o + id * (kFew * D);
      rows = min(kFew, size * a.G - s.row_tile * kFew);
    } else {
      const int64_t id = range + s.e - NH;
      ml = a.own_ml + id * (a.G * 2);
      o = a.own_o + id * (a.G * D);
      rows = a.G;
    }
    if (n < rows) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < D / 16; e += 4)
          *(f32x4_t*)(o + n * D + (D / 16) * (4 * g + i) + e) =
              (f32x4_t){r.o[e][i], r.o[e + 1][i], r.o[e + 2][i], r.o[e + 3][i]};
      if (g == 0) {
        ml[n * 2] = r.m;
        ml[n * 2 + 1] = r.sum[0];
      }
    }
    clear(r);
  }
  WGKV_DEVICE static void clear(Rows16<D>& r) {
    r.m = -INFINITY;
    r.sum = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < D / 16; ++e) r.o[e] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  }
  WGKV_DEVICE void take_q(Rows16<D>& r, const u32x4_t (&q)[D / 32]) const {
#pragma unroll
    for (int j = 0; j < D / 32; ++j) r.q[j] = __builtin_bit_cast(bf16x8_t, (q[j] & a.q_and) ^ a.q_xor);
  }

  // One wave's range [lo, hi) of the line (not empty); its first entry is at or
  // behind `from`.
  WGKV_DEVICE void run(int lo, int from) const {
    const int koff = (n * D + g * 8) * 2, voff = (4 * g * D + n * (D / 16)) * 2;
    KTile<D> k0, k1;
    VTile<D> v;
    Rows16<D> r;
    u32x4_t q[D / 32];
    Stage s0 = at(lo, from);
    ask_ids(s0);
    load_q(s0, q);
    Stage s1 = after(s0);
    ask_ids(s1);
    Stage s2 = after(s1);
    ask_ids(s2);
    load_k<D, KIND>(a, seen_pages(s0), s0.tile, s0.ids, koff, k0);
    load_v<D, KIND>(a, seen_pages(s0), s0.tile, s0.ids, voff, v);
    load_k<D, KIND>(a, seen_pages(s1), tile_or_none(s1), s1.ids, koff, k1);
    take_q(r, q);
    if (s1.first && s1.pos < hi) load_q(s1, q);
    clear(r);
    scores<D>(r, k0);
    const auto step = [&](KTile<D>& kc, KTile<D>& kn) __attribute__((always_inline)) {
      load_k<D, KIND>(a, seen_pages(s2), tile_or_none(s2), s2.ids, koff, kn);
      if (s1.first) take_q(r, q);  // (its scores come next; s0's are there)
      if (s2.first && s2.pos < hi) load_q(s2, q);
      attend_tile<D, KIND>(a, r, kc, v, seen_pages(s0), s0.tile, g, [&] __attribute__((always_inline)) () {
        load_v<D, KIND>(a, seen_pages(s1), tile_or_none(s1), s1.ids, voff, v);
      });
      if (s0.tile + 1 == s0.t1) flush(s0, r);
      s0 = s1;
      s1 = s2;
      s2 = after(s2);
      ask_ids(s2);
    };
    for (;;) {
      step(k1, k0);
      if (s0.pos >= hi) break;
      step(k0, k1);
      if (s0.pos >= hi) break;
    }
  }
};

// ---- many rows: tiles in LDS ----------------------------------------------------
// 16 bytes of the buffer at `off` (zeros behind its end) go to LDS at lds + 16 * lane.
WGKV_DEVICE void buffer_to_lds(__amdgpu_buffer_rsrc_t r, uint16_t* lds, int off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, lds, 16, off, 0, 0, 0);
}

// Tiles t0 .. t1 - 1 of 64 tokens for `rows` <= 256 rows, 32 per wave of eight.
// Wave w loads sub-page w % 4 of every tile, the keys or the values.
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
  for (int rt = 0; rt < 2; ++rt) r.ask_q(rt, q.row(a, w * 32 + rt * 16 + n), g);
  const int sub = w & 3;
  const bool keys = w < 4;
  const uint16_t* pool = keys ? a.kc : a.vc;
  int off[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int row = i * RPB + lane / CH;
    off[i] = row * D * 2 + ((lane % CH) ^ (keys ? attn::swz_k<D>(row) : attn::swz_v<D>(row))) * 16;
  }
  const auto load = [&](int tile, int id, uint16_t* sK, uint16_t* sV) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t r = subpage_rows<D>(a, p, pool, 4 * tile + sub, id);
    uint16_t* to = (keys ? sK : sV) + sub * NB * 512;
#pragma unroll
    for (int i = 0; i < NB; ++i) buffer_to_lds(r, to + i * 512, off[i]);
  };
  // Page ids of 16 tiles are a lane's each, asked for 16 tiles ahead.  (A
  // scalar load per tile would be waited for by the tile's first LDS read,
  // with which it shares a counter.)
  const auto ids_from = [&](int tile) {
    return p.bt[min(4 * tile + lane, (p.seen.tokens - 1) >> 4) >> a.page_shift];
  };
  int ids = ids_from(t0), ids_next = ids_from(t0 + 16);
  const auto id_of = [&](int tile) { return __builtin_amdgcn_readlane(ids, (tile - t0) % 16 * 4 + sub); };
  load(t0, id_of(t0), sK0, sV0);
  r.take_q(a.q_and, a.q_xor);
  const auto step = [&](int tile, const uint16_t* sK, const uint16_t* sV, uint16_t* nK, uint16_t* nV)
      __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's part of the tile has landed
    __syncthreads();                     // every wave's has, and nobody reads the other buffer any more
    if ((tile + 1 - t0) % 16 == 0) {
      ids = ids_next;
      ids_next = ids_from(tile + 17);
    }
    if (tile + 1 < t1) load(tile + 1, id_of(tile + 1), nK, nV);
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

// (max, sum, O) of a second set of tokens into the first's.  A sum of 0 (no
// token that weighs) has no part; one of NaN (its scores were) has, whatever its
// maximum.
WGKV_DEVICE void join(float& m, float& l, f32x4_t& o, float mb, float lb, f32x4_t ob) {
  const float mn = fmaxf(m, mb);
  const float ca = m == -INFINITY && l == 0.f ? 0.f : fast_exp2(m - mn);
  const float cb = mb == -INFINITY && lb == 0.f ? 0.f : fast_exp2(mb - mn);
  l = l * ca + lb * cb;
  o = o * ca + ob * cb;
  m = mn;
}

// Where the own tokens' line begins among the entries' tiles: prefixes of many
// rows are not on it.
template <Mode KIND>
WGKV_DEVICE int own_zero(const int* base, int NH) { return KIND == kManyRows ? base[NH] : 0; }

template <Mode KIND>
constexpr int waves_of() { return KIND == kManyRows ? 8 : 4; }

// Exclusive sum over the threads of a workgroup of NW waves, and the total.
template <int NW>
WGKV_DEVICE int block_scan(int v, int* s_wave, int* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int incl = wave_incl_scan(v, lane);
  if (lane == 63) s_wave[w] = incl;
  __syncthreads();
  int run = incl - v, all = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    run += i < w ? s_wave[i] : 0;
    all += s_wave[i];
  }
  __syncthreads();
  *total = uniform(all);
  return run;
}

// The greatest value of the threads before (0: none), of values of 0 or more.
template <int NW>
WGKV_DEVICE int block_max_before(int v, int* s_wave) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) {
    const int o = __shfl_up(v, i, 64);
    v = max(v, lane >= i ? o : 0);
  }
  if (lane == 63) s_wave[w] = v;
  const int up = __shfl_up(v, 1, 64);
  __syncthreads();
  int before = lane ? up : 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) before = max(before, i < w ? s_wave[i] : 0);
  __syncthreads();
  return before;
}

template <int D, Mode KIND>
__global__ __launch_bounds__(64 * waves_of<KIND>()) __attribute__((amdgpu_waves_per_eu(2, 2)))
void stream_split_kernel(StreamArgs a) {
  constexpr int NW = waves_of<KIND>(), NT = 64 * NW;
  // tile buffers, as four objects: loads into one provably leave the others alone
  constexpr int kTile = KIND == kManyRows ? attn::kKeys * D : 8;
  __shared__ __attribute__((aligned(16))) uint16_t s_k0[kTile];
  __shared__ __attribute__((aligned(16))) uint16_t s_v0[kTile];
  __shared__ __attribute__((aligned(16))) uint16_t s_k1[kTile];
  __shared__ __attribute__((aligned(16))) uint16_t s_v1[kTile];
  constexpr int kEntries = (KIND == kWindowed ? 1 : 2) * kMaxHeads;
  __shared__ int s_base[kEntries + 1], s_tokens[kEntries], s_start[KIND == kWindowed ? 1 : kMaxHeads + 1];
  __shared__ int s_wave[NW];
  const int t = threadIdx.x, wg = blockIdx.x, wave = uniform(t >> 6);
  const int NH = a.N * a.H, E = NH + a.B * a.H;
  const Plan plan = {s_base, s_tokens, s_start};
  // The plan, the same in every workgroup; each thread has some entries.
  const int each = (E + NT - 1) / NT, e0 = min(E, t * each), e1 = min(E, e0 + each);
  for (int e = e0; e < e1; ++e) s_tokens[e] = entry_tokens(a, e);
  if constexpr (KIND != kWindowed) {
    // starts, made to ascend: what the workspace holds relies on it
    const int n1 = a.N + 1, nt = (n1 + NT - 1) / NT, b0 = min(n1, t * nt), b1 = min(n1, b0 + nt);
    int most = 0;
    for (int n = b0; n < b1; ++n) s_start[n] = most = max(most, clamp_to(a.starts[n], a.B));
    const int before = block_max_before<NW>(most, s_wave);
    for (int n = b0; n < b1; ++n) s_start[n] = max(s_start[n], before);
    __syncthreads();
  }
  const auto rows_tiles = [&](int e) {
    if (KIND == kWindowed || e >= NH) return 1;
    const int n = e / a.H;
    return row_tiles<KIND>(a, s_start[n + 1] - s_start[n]);
  };
  int chunk = 0, total;
  if constexpr (KIND == kManyRows) {
    int tiles = 0, rts = 0, all_tiles, all_rts;
    for (int e = e0; e < min(e1, NH); ++e) {
      const int x = entry_tiles<KIND>(a, true, s_tokens[e]), rt = rows_tiles(e);
      tiles += x * rt;
      rts += x ? rt : 0;
    }
    block_scan<NW>(tiles, s_wave, &all_tiles);
    block_scan<NW>(rts, s_wave, &all_rts);
    chunk = chunk_tiles(all_tiles, all_rts, a.slots);
  }
  {
    int mine = 0;
    for (int e = e0; e < e1; ++e) {
      int x = entry_tiles<KIND>(a, e < NH, s_tokens[e]);
      if (KIND == kManyRows && e < NH) x = (x + chunk - 1) / chunk;
      mine += x * rows_tiles(e);
      s_base[e + 1] = mine;
    }
    const int run = block_scan<NW>(mine, s_wave, &total);
    for (int e = e0; e < e1; ++e) s_base[e + 1] += run;
    if (t == 0) s_base[0] = 0;
    __syncthreads();
  }
  const int zero = uniform(own_zero<KIND>(s_base, NH)), line = total - zero;
  const int per = uniform(range_tiles<KIND>(line, a.slots * NW));
  if (wg == 0) {
    for (int i = t; i <= E; i += NT) a.plan[i] = s_base[i];
    if (t == 0) {
      a.plan[E + 1] = chunk;
      a.plan[E + 2] = per;
    }
    if constexpr (KIND != kWindowed)
      for (int n = t; n <= a.N; n += NT) a.plan[E + 3 + n] = s_start[n];
  }
  const int range = wg * NW + wave;
  const auto stream = [&]() __attribute__((always_inline)) {
    if ((int64_t)range * per >= line) return;
    const int lo = range * per, from = KIND == kManyRows ? NH : 0;
    int first = from, last = E - 1;  // the last entry that begins at or before lo
    while (first < last) {
      const int mid = (first + last + 1) >> 1;
      if (uniform(s_base[mid]) - zero <= lo) first = mid; else last = mid - 1;
    }
    const int lane = t & 63;
    const Stream<D, KIND> s = {a, plan, NH, zero, min(lo + per, line), range, lane & 15, lane >> 4};
    s.run(lo, first);
  };
  if constexpr (KIND != kManyRows) {
    stream();
  } else {
    const bool own_first = wg >= a.slots / 2;
    if (own_first) stream();
    // (from the last workgroup on: the first ones have the ranges of a short line of sequences)
    for (int unit = a.slots - 1 - wg; unit < zero; unit += a.slots) {
      int e = 0, last = NH - 1;  // the last entry that begins at or before the unit
      while (e < last) {
        const int mid = (e + last + 1) >> 1;
        if (uniform(s_base[mid]) <= unit) e = mid; else last = mid - 1;
      }
      const int n = uniform(e / a.H), tiles = uniform(entry_tiles<KIND>(a, true, uniform(s_tokens[e])));
      const int chunks = uniform((tiles + chunk - 1) / chunk), at = unit - uniform(s_base[e]);
      const int row_tile = uniform(at / chunks), c = at - row_tile * chunks;
      Queries q;
      q.h = e - n * a.H;
      q.b0 = uniform(s_start[n]);
      q.first = row_tile * kMany;
      q.count = (uniform(s_start[n + 1]) - q.b0) * a.G;
      const Pages p = {a.pbt + n * a.pbt_sb + q.h * a.pbt_sh, seen_of<KIND>(a, uniform(s_tokens[e]))};
      const int each = uniform(tiles / chunks), over = tiles - each * chunks, from = c * each + min(c, over);
      tile_piece<D>(a, p, from, from + each + (c < over), q, min(kMany, q.count - q.first),
                    a.pre_ml + (int64_t)unit * (kMany * 2), a.pre_o + (int64_t)unit * (kMany * D), s_k0, s_v0, s_k1,
                    s_v1);
    }
    if (!own_first) stream();
  }
}

// The pieces of a query row under one softmax, in the order of the line.  A
// row's pieces are dealt in turn to groups of D/4 lanes, four values of d
// each, of one wave, or (few rows, of which some may have many pieces) of the
// four waves of a workgroup; the groups then meet in order.
template <int D, Mode KIND, bool WIDE>
__global__ __launch_bounds__(256) void stream_merge_kernel(StreamArgs a) {
  constexpr int NQ = D / 4, PER_WAVE = 64 / NQ, GROUPS = WIDE ? 4 * PER_WAVE : PER_WAVE, kBatch = 8, R = rows_of<KIND>();
  __shared__ f32x4_t s_a[WIDE ? 256 : 1];
  __shared__ float s_m[WIDE ? 256 : 1], s_l[WIDE ? 256 : 1];
  const int bh = blockIdx.x, b = uniform(bh / a.H), h = bh - b * a.H;
  const int t = threadIdx.x, wave = uniform(t >> 6), vq = t % NQ;
  const int gq = WIDE ? (int)blockIdx.y : (int)blockIdx.y * 4 + wave;
  if (gq >= a.G) return;  // (whole waves, and no barrier follows)
  const int grp = (WIDE ? t : t & 63) / NQ;
  const int NH = a.N * a.H;
  const int E = NH + a.B * a.H, chunk = a.plan[E + 1], per = a.plan[E + 2];
  int n_pre = 0;
  const float *pre_ml = nullptr, *pre_o = nullptr;
  if constexpr (KIND != kWindowed) {
    const int* starts = a.plan + E + 3;
    int n = 0, hi = a.N;  // the last group that starts at or before b
    while (hi - n > 1) {
      const int mid = (n + hi) >> 1;
      if (starts[mid] <= b) n = mid; else hi = mid;
    }
    const int start = starts[n], size = starts[n + 1] - start, e = n * a.H + h;
    const int tiles = entry_tiles<KIND>(a, true, entry_tokens(a, e));
    if (b >= start && b - start < size && tiles) {
      const int row = (b - start) * a.G + gq, row_tile = row / R;
      int64_t first;
      if constexpr (KIND == kManyRows) {
        n_pre = (tiles + chunk - 1) / chunk;
        first = a.plan[e] + row_tile * n_pre;
      } else {
        const int base = a.plan[e] + row_tile * tiles, w0 = base / per;
        n_pre = (base + tiles - 1) / per - w0 + 1;
        first = w0 + piece_of(a, start, size, n, h, row_tile);
      }
      first = first * R + row - row_tile * R;
      pre_ml = a.pre_ml + first * 2;
      pre_o = a.pre_o + first * D;
    }
  }
  int n_own = 0;
  const float *own_ml = nullptr, *own_o = nullptr;
  const int tiles = entry_tiles<KIND>(a, false, entry_tokens(a, NH + bh));
  if (tiles) {
    const int base = a.plan[NH + bh] - own_zero<KIND>(a.plan, NH), w0 = base / per;
    n_own = (base + tiles - 1) / per - w0 + 1;
    const int64_t first = ((int64_t)w0 + bh) * a.G + gq;
    own_ml = a.own_ml + first * 2;
    own_o = a.own_o + first * D;
  }
  const int pieces = n_pre + n_own;
  float m = -INFINITY, l = 0.f;
  f32x4_t o = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  for (int c0 = grp; c0 < pieces; c0 += GROUPS * kBatch) {
    float mc[kBatch], lc[kBatch];
    f32x4_t oc[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int c = min(c0 + k * GROUPS, pieces - 1);
      const bool pre = c < n_pre;
      const int64_t i = pre ? (int64_t)c * R : (int64_t)(c - n_pre) * a.G;
      const float* ml = (pre ? pre_ml : own_ml) + i * 2;
      mc[k] = ml[0];
      lc[k] = ml[1];
      oc[k] = *(const f32x4_t*)((pre ? pre_o : own_o) + i * D + vq * 4);
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (c0 + k * GROUPS >= pieces) continue;
      join(m, l, o, mc[k], lc[k], oc[k]);
    }
  }
  if constexpr (WIDE) {
    s_m[t] = m;
    s_l[t] = l;
    s_a[t] = o;
    __syncthreads();
    if (t >= NQ) return;
    m = -INFINITY;
    l = 0.f;
    o = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < GROUPS; ++i) join(m, l, o, s_m[i * NQ + t], s_l[i * NQ + t], s_a[i * NQ + t]);
  } else {
#pragma unroll
    for (int i = NQ; i < 64; i <<= 1) {
      const float mo = __shfl_xor(m, i, 64), lo = __shfl_xor(l, i, 64);
      f32x4_t oo;
#pragma unroll
      for (int e = 0; e < 4; ++e) oo[e] = __shfl_xor(o[e], i, 64);
      join(m, l, o, mo, lo, oo);
    }
    if ((t & 63) >= NQ) return;
  }
  uint16_t* out = a.out + b * a.out_sb + (int64_t)(h * a.G + gq) * a.out_sh + vq * 4;
  const float inv = 1.f / l;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = l == 0.f ? 0 : f32_to_bf16(o[e] * inv);
}

// Whether an even share of the batch has more rows than one operand, which
// would otherwise stream a prefix once per 16 rows.  (One prefix, 8 KV heads of
// 4, own 100 tokens; us streamed / in LDS tiles: 5 sequences 15.4 / 17.6 at 2048
// tokens of prefix, 28.9 / 20.6 at 8192, 55.4 / 41.7 at 32K; 16 sequences 23.9 /
// 20.5, 39.5 / 21.9, 92.7 / 45.5; 4 sequences, one operand, 41.0 / 41.3 at 32K.)
// The starts are on the device, so the average decides for all groups.  Where they
// differ much, a large group's prefix may be streamed once per 16 rows all the
// same: of 10 groups one of 31 sequences, 9 of one, 99 us at 8192 tokens and 355 at
// 32K (one more sequence, and tiles: 87 and 273); of 32 groups one of 97, 31 of one,
// 305 at 8192 (tiles: 350, since the small groups' rows then fill a tile each).
bool many_rows(int B, int N, int G) { return (int64_t)B * G > (int64_t)kFew * N; }

struct Scratch {
  int64_t pre, own;  // pieces
  size_t pre_ml, pre_o, own_ml, own_o, bytes;
};

size_t aligned(size_t n) { return (n + 255) & ~(size_t)255; }

constexpr size_t kPlanBytes = ((3 * kMaxHeads + 4) * sizeof(int) + 255) & ~(size_t)255;

// Pieces: one per range, and one more per entry (and row tile).
Scratch scratch_for(int B, int N, int G, int H, int D) {
  const bool many = N && many_rows(B, N, G);
  const int R = many ? kMany : kFew;
  Scratch s;
  s.pre = N ? (many ? kMaxWaves / 8 : kMaxWaves) + (int64_t)H * ((int64_t)B * G / R + N + 1) : 0;
  s.own = kMaxWaves + (int64_t)B * H;
  s.pre_ml = kPlanBytes;
  s.pre_o = s.pre_ml + aligned(s.pre * R * 2 * sizeof(float));
  s.own_ml = s.pre_o + aligned(s.pre * R * D * sizeof(float));
  s.own_o = s.own_ml + aligned(s.own * G * 2 * sizeof(float));
  s.bytes = s.own_o + aligned(s.own * G * D * sizeof(float));
  return s;
}

void use_scratch(StreamArgs& a, const Scratch& s, void* p) {
  char* ws = (char*)p;
  a.plan = (int*)ws;
  a.pre_ml = (float*)(ws + s.pre_ml);
  a.pre_o = (float*)(ws + s.pre_o);
  a.own_ml = (float*)(ws + s.own_ml);
  a.own_o = (float*)(ws + s.own_o);
}

template <int D, Mode KIND>
hipError_t launch(StreamArgs& a, hipStream_t st) {
  constexpr int NW = waves_of<KIND>();
  a.slots = min(kMaxWaves, cu_count() * kWavesPerCu) / NW;
  hipLaunchKernelGGL((stream_split_kernel<D, KIND>), dim3(a.slots), dim3(64 * NW), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  // a wave per row once there are rows for all the CUs' waves (a wave / a
  // workgroup per row: 128 rows of a 65536-token prefix 74 / 62 us, 1024 of
  // 32768 50 / 50, 2048 of 32768 64 / 66)
  if (a.B * a.H * a.G >= 4 * cu_count())
    hipLaunchKernelGGL((stream_merge_kernel<D, KIND, false>), dim3(a.B * a.H, (a.G + 3) / 4), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((stream_merge_kernel<D, KIND, true>), dim3(a.B * a.H, a.G), dim3(256), 0, st, a);
  return hipGetLastError();
}

template <int D>
hipError_t launch_rows(StreamArgs& a, bool many, hipStream_t st) {
  return many ? launch<D, kManyRows>(a, st) : launch<D, kFewRows>(a, st);
}

}  // namespace

// Bytes of `scratch` (any contents) for wgkv_stream_window.
size_t wgkv_stream_window_bytes(int B, int H, int G, int D) { return scratch_for(B, 0, G, H, D).bytes; }

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
  use_scratch(a, scratch_for(w.B, 0, w.G, w.H, w.D), scratch);
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
  if ((cap + 31) / 32 * own + (pcap + 31) / 32 * row_tiles * num_kv_heads > 0x70000000)
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
  use_scratch(a, sc, workspace);
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
