// Decode attention of a batch whose sequences share long prefixes (gfx950).
//
// Sequences starts[n] .. starts[n+1] - 1 share prefix n: KV head h of each of
// them attends to the first prefix_lens[n, h] tokens of the prefix's pages and
// to the first lens[b, h] tokens of its own, under one softmax.
//
// The prefix is read once for all queries of its group.  Its queries are the
// rows (sequence, query head of the KV head) of a matrix, cut into tiles of
// 16 * RT rows; a sequence's own tokens have G rows.  Both are the same work:
//   * a wave takes 32 tokens: K comes from memory in the layout of the matrix
//     core's A operand, and S^T = K Q^T (v_mfma_f32_16x16x32_bf16, the queries
//     held as B operands) leaves each lane 8 scores of one query row;
//   * softmax in the log2 domain with a running maximum per row that moves
//     only when a score exceeds it by more than 8 (so p <= 2^8 and most tiles
//     rescale nothing); probabilities are rounded to bf16 for the products,
//     and their row sums are the matrix core's too (ones . P^T), so that both
//     halves of the quotient see the same rounding; all sums are fp32;
//   * O^T += V^T P^T: a lane's 8 scores are already the B operand.  The A
//     operand wants 8 tokens of one d per lane, while memory holds 8 d of one
//     token: a lane loads the 8 tokens' 16-byte pieces and exchanges halves in
//     its own registers (4 v_perm_b32 per operand), which fixes the order of d
//     over the operands (d = D/16 * m + e for row m of operand e) and needs
//     neither LDS nor other lanes.
// The next tile's K and V are asked for before the current one's arithmetic.
//
// Split: the tiles of all (prefix, head, row tile) and (sequence, head) are
// laid end to end, weighted by what they cost, and the workgroups take equal
// ranges of that line, whatever the lengths.  A workgroup goes through the
// pieces of its range; its four waves take a piece's tiles in turn and meet in
// LDS at its end.  Pieces are numbered (workgroup + position of their entry),
// store (max, sum, O) there, and a second launch joins the pieces of every
// query row in a fixed order.
#include <string.h>

#include "kv4.h"

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kMaxEntries = 4096;   // (prefix, head) and (sequence, head) pairs
constexpr int kMaxG = 8;
constexpr int kMaxSlots = 1024;     // workgroups of the split launch at most
constexpr int kOwnWeight = 4;       // cost of a tile of a sequence's own tokens
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.f;

struct SharedArgs {
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
  const int32_t* plen;
  int64_t plen_sb;
  const int32_t* pbt;
  int64_t pbt_sb, pbt_sh;
  int pcap;
  const int32_t* starts;
  uint16_t* out;
  int64_t out_sb, out_sh;
  int B, N, H, G;
  float scale_log2;
  uint32_t q_and, q_xor;
  int slots;    // workgroups of the split launch
  int weight;   // cost of a tile of a prefix
  // pieces: (max, sum) and O of a prefix piece's 16 * RT rows, then of an own piece's G rows
  float* pre_ml;
  float* pre_o;
  float* own_ml;
  float* own_o;
  int* plan;  // cost before each entry, the total, and the cost of a workgroup's range
};

WGKV_DEVICE int clamp_to(int x, int hi) { return min(max(x, 0), hi); }

WGKV_DEVICE int group_start(const SharedArgs& a, int n) { return clamp_to(a.starts[n], a.B); }
WGKV_DEVICE int group_size(const SharedArgs& a, int n) { return max(group_start(a, n + 1) - group_start(a, n), 0); }

// Tokens, row tiles and cost of entry e: prefixes first.
struct Entry {
  int tokens, tiles, row_tiles, weight;
  WGKV_DEVICE int cost() const { return tiles * row_tiles * weight; }
};

template <int RT>
WGKV_DEVICE Entry entry_of(const SharedArgs& a, int e) {
  Entry x;
  const int NH = a.N * a.H;
  if (e < NH) {
    const int n = e / a.H, h = e - n * a.H;
    x.tokens = clamp_to(a.plen[(int64_t)n * a.plen_sb + h], a.pcap);
    x.row_tiles = (group_size(a, n) * a.G + 16 * RT - 1) / (16 * RT);
    x.weight = a.weight;
  } else {
    const int b = (e - NH) / a.H, h = e - NH - b * a.H;
    x.tokens = clamp_to(a.len[(int64_t)b * a.len_sb + h], a.cap);
    x.row_tiles = 1;
    x.weight = kOwnWeight;
  }
  x.tiles = (x.tokens + 31) >> 5;
  return x;
}

// Cost of a workgroup's range: an equal share, but four tiles (one per wave) at least.
WGKV_DEVICE int range_cost(int total, int slots, int weight) {
  return max((total + slots - 1) / slots, 4 * max(weight, kOwnWeight));
}

// Number of a (prefix, head, row tile) that only grows along the line: groups
// before n have at most starts[n] * G / (16 * RT) + n row tiles.
template <int RT>
WGKV_DEVICE int64_t piece_of(const SharedArgs& a, int n, int h, int row_tile) {
  const int row_tiles = (group_size(a, n) * a.G + 16 * RT - 1) / (16 * RT);
  return (int64_t)a.H * (group_start(a, n) * a.G / (16 * RT) + n) + h * row_tiles + row_tile;
}

WGKV_DEVICE float fmax_ieee(float x, float y) { return __builtin_elementwise_maximum(x, y); }
WGKV_DEVICE float xor16_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmax_ieee(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
WGKV_DEVICE float xor32_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmax_ieee(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// 32 tokens of a head: K in the A operand's layout (lane (n, g): token
// 16 * kt + n, d = 32 * j + 8 * g ..), V as 8 tokens' pieces of D/16 values
// (lane (n, g), piece s: token 4 * g + s, or 16 + 4 * g + s - 4 from s = 4 on).
template <int D>
struct KV {
  u32x4_t k[2][D / 32];
  uint32_t v[8][D / 32];
};

// Pages of a head, and its tokens.
struct Pages {
  const int32_t* bt;
  int tokens;
};

// Page ids of a tile's two sub-pages of 16 tokens, one scalar load each,
// asked for a tile before the rows so that no wait for them holds those up.
struct Ids {
  int pg[2];
};
typedef const int32_t __attribute__((address_space(4))) ConstInt;

WGKV_DEVICE Ids tile_ids(const SharedArgs& a, const Pages& p, int tile) {
  const int last = (p.tokens - 1) >> 4;
  ConstInt* bt = (ConstInt*)p.bt;
  Ids x;
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) x.pg[kt] = bt[min(2 * tile + kt, last) >> a.page_shift];
  return x;
}

// Buffer loads over the sub-page's valid rows: a lane's offset is the same in
// every tile, rows behind the last token read as zeros without a request (V
// then adds 0 for them whatever the pool holds), and a tile behind the end
// asks for nothing, so that the loads need no branch.
template <int D>
WGKV_DEVICE void load_tile(const SharedArgs& a, const Pages& p, int tile, const Ids& ids, int koff, int voff, KV<D>& x) {
  __amdgpu_buffer_rsrc_t kb[2], vb[2];
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) {
    const int sp = 2 * tile + kt;
    const int64_t pg = ids.pg[kt] < 0 ? 0 : (ids.pg[kt] >= a.num_pages ? a.num_pages - 1 : ids.pg[kt]);
    const int64_t row = (pg << (a.page_shift + 4)) + (sp & ((1 << a.page_shift) - 1)) * 16;
    const int valid = clamp_to(p.tokens - sp * 16, 16) * D * 2;
    kb[kt] = __builtin_amdgcn_make_buffer_rsrc((void*)(a.kc + row * D), (short)0, valid, 0x00020000);
    vb[kt] = __builtin_amdgcn_make_buffer_rsrc((void*)(a.vc + row * D), (short)0, valid, 0x00020000);
  }
#pragma unroll
  for (int kt = 0; kt < 2; ++kt)
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
      x.k[kt][j] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(kb[kt], koff + j * 64, 0, 0));
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    if constexpr (D == 128) {
      const u32x4_t w =
          __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(vb[s >> 2], voff + (s & 3) * D * 2, 0, 0));
#pragma unroll
      for (int i = 0; i < 4; ++i) x.v[s][i] = w[i];
    } else {
      const auto w = __builtin_amdgcn_raw_buffer_load_b64(vb[s >> 2], voff + (s & 3) * D * 2, 0, 0);
      x.v[s][0] = w[0];
      x.v[s][1] = w[1];
    }
  }
}

// Running state of 16 * RT query rows in a wave.
template <int D, int RT>
struct Rows {
  bf16x8_t q[RT][D / 32];
  f32x4_t o[D / 16][RT];
  f32x4_t sum[RT];
  float m[RT];
};

template <int D, int RT>
WGKV_DEVICE void attend_tile(const SharedArgs& a, Rows<D, RT>& r, const KV<D>& x, int tokens, int tile, int g) {
  f32x4_t s[2][RT];
#pragma unroll
  for (int kt = 0; kt < 2; ++kt)
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) s[kt][rt] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < D / 32; ++j)
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
        s[kt][rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, x.k[kt][j]), r.q[rt][j],
                                                            s[kt][rt], 0, 0, 0);
  const int left = tokens - tile * 32;
  if (left < 32) {  // tokens behind the last weigh nothing
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in = kt * 16 + 4 * g + i < left;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[kt][rt][i] = in ? s[kt][rt][i] : -INFINITY;
      }
  }
  float mx[RT];
  bool up = false;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    float y = s[0][rt][0];
#pragma unroll
    for (int i = 1; i < 8; ++i) y = fmax_ieee(y, s[i >> 2][rt][i & 3]);
    mx[rt] = y * a.scale_log2;
    up |= mx[rt] > r.m[rt] + kSlack;
  }
  if (__builtin_amdgcn_ballot_w64(up) != 0) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const float y = xor32_max(xor16_max(mx[rt]));
      const float m = y > r.m[rt] + kSlack ? y : r.m[rt];
      const float scale = m == r.m[rt] ? 1.f : fast_exp2(r.m[rt] - m);
      r.m[rt] = m;
      r.sum[rt] *= scale;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) r.o[e][rt] *= scale;
    }
  }
  bf16x8_t pb[RT];
  const bf16x8_t ones = __builtin_bit_cast(bf16x8_t, (u32x4_t){0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float m = r.m[rt] == -INFINITY ? 0.f : r.m[rt];
    u32x4_t w;
#pragma unroll
    for (int i = 0; i < 8; i += 2)
      w[i / 2] = pack_bf16x2(fast_exp2(fmaf(s[i >> 2][rt][i & 3], a.scale_log2, -m)),
                             fast_exp2(fmaf(s[i >> 2][rt][(i & 3) + 1], a.scale_log2, -m)));
    pb[rt] = __builtin_bit_cast(bf16x8_t, w);
    r.sum[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pb[rt], r.sum[rt], 0, 0, 0);
  }
#pragma unroll
  for (int e = 0; e < D / 16; ++e) {
    u32x4_t w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = __builtin_amdgcn_perm(x.v[2 * i + 1][e / 2], x.v[2 * i][e / 2], e & 1 ? 0x07060302u : 0x05040100u);
    const bf16x8_t vf = __builtin_bit_cast(bf16x8_t, w);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) r.o[e][rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pb[rt], r.o[e][rt], 0, 0, 0);
  }
}

// One piece: tiles t0 .. t1 - 1 of a head's tokens for 16 * RT rows; row r's
// query is at query(r) (any valid address for rows >= rows).  (max, sum) and O
// of rows < rows go to ml and o.
template <int D, int RT, typename Query>
WGKV_DEVICE void piece(const SharedArgs& a, const Pages& p, int t0, int t1, int rows, Query query, float* ml, float* o,
                       float* s_o, float* s_ml) {
  constexpr int RS = D + 4;  // LDS row stride: rows of one operand on different banks
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int n = lane & 15, g = lane >> 4;
  Rows<D, RT> r;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const uint16_t* row = query(rt * 16 + n);
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      u32x4_t x = *(const u32x4_t*)(row + (j * 4 + g) * 8);
      r.q[rt][j] = __builtin_bit_cast(bf16x8_t, (x & a.q_and) ^ a.q_xor);
    }
    r.m[rt] = -INFINITY;
    r.sum[rt] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < D / 16; ++e) r.o[e][rt] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  }
  const int koff = (n * D + g * 8) * 2, voff = (4 * g * D + n * (D / 16)) * 2;
  KV<D> x0, x1;
  int tile = t0 + w;
  Ids id = tile_ids(a, p, tile);
  load_tile<D>(a, p, tile < t1 ? tile : INT32_MAX / 64, id, koff, voff, x0);
  id = tile_ids(a, p, tile + kWaves);
  for (; tile < t1; tile += 2 * kWaves) {
    load_tile<D>(a, p, tile + kWaves < t1 ? tile + kWaves : INT32_MAX / 64, id, koff, voff, x1);
    id = tile_ids(a, p, tile + 2 * kWaves);
    attend_tile<D, RT>(a, r, x0, p.tokens, tile, g);
    load_tile<D>(a, p, tile + 2 * kWaves < t1 ? tile + 2 * kWaves : INT32_MAX / 64, id, koff, voff, x0);
    id = tile_ids(a, p, tile + 3 * kWaves);
    if (tile + kWaves < t1) attend_tile<D, RT>(a, r, x1, p.tokens, tile + kWaves, g);
  }
  // the waves meet: lane (n, g) holds d = D/16 * (4 * g + i) + e of row 16 * rt + n
  constexpr int R = 16 * RT;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = rt * 16 + n;
    if (g == 0) {
      s_ml[(w * R + row) * 2] = r.m[rt];
      s_ml[(w * R + row) * 2 + 1] = r.sum[rt][0];
    }
    float* to = s_o + (w * R + row) * RS;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < D / 16; e += 4)
        *(f32x4_t*)(to + (D / 16) * (4 * g + i) + e) =
            (f32x4_t){r.o[e][rt][i], r.o[e + 1][rt][i], r.o[e + 2][rt][i], r.o[e + 3][rt][i]};
  }
  __syncthreads();
  for (int i = t; i < rows * (D / 4); i += kThreads) {
    const int row = i / (D / 4), d = (i - row * (D / 4)) * 4;
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) m = fmaxf(m, s_ml[(k * R + row) * 2]);
    f32x4_t sum = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
      const float mk = s_ml[(k * R + row) * 2], lk = s_ml[(k * R + row) * 2 + 1];
      if (mk == -INFINITY && lk == 0.f) continue;  // a wave without a token that weighs
      const float c = fast_exp2(mk - m);
      l += c * lk;
      sum += c * *(const f32x4_t*)(s_o + (k * R + row) * RS + d);
    }
    *(f32x4_t*)(o + (int64_t)row * D + d) = sum;
    if (d == 0) {
      ml[row * 2] = m;
      ml[row * 2 + 1] = l;
    }
  }
  __syncthreads();
}

template <int D, int RT>
constexpr int lds_floats() { return kWaves * 16 * RT * (D + 4); }

// Resident workgroups per CU: with one row tile two waves fit a SIMD.
constexpr int wgs_per_cu(int RT) { return RT == 1 ? 2 : 1; }

template <int D, int RT>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(wgs_per_cu(RT), wgs_per_cu(RT))))
void shared_split_kernel(SharedArgs a) {
  __shared__ __attribute__((aligned(16))) float s_o[lds_floats<D, RT>()];
  __shared__ float s_ml[kWaves * 16 * RT * 2];
  __shared__ int s_base[kMaxEntries + 1];
  __shared__ int s_tmp[4];
  const int t = threadIdx.x, wg = blockIdx.x;
  const int NH = a.N * a.H, E = NH + a.B * a.H;
  // cost before every entry, the same in every workgroup
  const int per_thread = (E + kThreads - 1) / kThreads;
  const int e0 = min(E, t * per_thread), e1 = min(E, e0 + per_thread);
  int mine = 0, total;
  for (int e = e0; e < e1; ++e) mine += entry_of<RT>(a, e).cost();
  int run = block_exclusive_scan_256(mine, s_tmp, &total);
  for (int e = e0; e < e1; ++e) {
    s_base[e] = run;
    run += entry_of<RT>(a, e).cost();
  }
  if (t == 0) s_base[E] = total;
  __syncthreads();
  const int per = range_cost(total, a.slots, a.weight);
  if (wg == 0) {
    for (int i = t; i <= E; i += kThreads) a.plan[i] = s_base[i];
    if (t == 0) a.plan[E + 1] = per;
  }
  const int lo = (int)min((int64_t)wg * per, (int64_t)total), hi = (int)min((int64_t)lo + per, (int64_t)total);
  if (lo >= hi) return;
  int first = 0, last = E - 1;  // the last entry that begins at or before lo
  while (first < last) {
    const int mid = (first + last + 1) >> 1;
    if (s_base[mid] <= lo) first = mid; else last = mid - 1;
  }
  for (int e = first; e < E && s_base[e] < hi; ++e) {
    const int base = s_base[e];
    if (s_base[e + 1] == base) continue;
    const Entry x = entry_of<RT>(a, e);
    // the entry's tiles (row tile after row tile) that begin in [lo, hi)
    int u0 = max(0, (lo - base + x.weight - 1) / x.weight);
    const int u1 = min(x.tiles * x.row_tiles, (hi - base + x.weight - 1) / x.weight);
    while (u0 < u1) {
      const int row_tile = u0 / x.tiles, t0 = u0 - row_tile * x.tiles;
      const int t1 = min(x.tiles, t0 + u1 - u0);
      u0 += t1 - t0;
      if (e < NH) {
        const int n = e / a.H, h = e - n * a.H, r0 = row_tile * 16 * RT;
        const int b0 = group_start(a, n), rows = group_size(a, n) * a.G;
        const int64_t id = wg + piece_of<RT>(a, n, h, row_tile);
        piece<D, RT>(a, {a.pbt + n * a.pbt_sb + h * a.pbt_sh, x.tokens}, t0, t1, min(16 * RT, rows - r0),
                     [&](int r) {
                       const int row = min(r0 + r, rows - 1), b = row / a.G;
                       return a.q + (b0 + b) * a.q_sb + (h * a.G + row - b * a.G) * a.q_sh;
                     },
                     a.pre_ml + id * (16 * RT * 2), a.pre_o + id * (16 * RT * D), s_o, s_ml);
      } else {
        const int bh = e - NH, b = bh / a.H, h = bh - b * a.H;
        const int64_t id = wg + bh;
        piece<D, 1>(a, {a.bt + b * a.bt_sb + h * a.bt_sh, x.tokens}, t0, t1, a.G,
                    [&](int r) { return a.q + b * a.q_sb + (h * a.G + min(r, a.G - 1)) * a.q_sh; },
                    a.own_ml + id * (a.G * 2), a.own_o + id * (a.G * D), s_o, s_ml);
      }
    }
  }
}

// The pieces of a query row under one softmax, in the order of the line: one
// workgroup per (sequence, KV head, query head), a thread group of D/4
// threads per piece in turn, then the groups in order.
template <int D, int RT>
__global__ __launch_bounds__(256) void shared_merge_kernel(SharedArgs a) {
  constexpr int NQ = D / 4, GROUPS = 256 / NQ, kBatch = 8;
  __shared__ f32x4_t s_a[256];
  __shared__ float s_m[256], s_l[256];
  const int bh = blockIdx.x, b = bh / a.H, h = bh - b * a.H, gq = blockIdx.y;
  const int t = threadIdx.x, vq = t % NQ, grp = t / NQ;
  const int NH = a.N * a.H;
  const int per = a.plan[NH + a.B * a.H + 1];
  int n_pre = 0;
  const float *pre_ml = nullptr, *pre_o = nullptr;
  int lo = 0, hi = a.N;  // the last group that starts at or before b
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (group_start(a, mid) <= b) lo = mid; else hi = mid;
  }
  const int at = b - group_start(a, lo);
  if (at >= 0 && at < group_size(a, lo)) {
    const int e = lo * a.H + h;
    const Entry x = entry_of<RT>(a, e);
    if (x.tiles) {
      const int row = at * a.G + gq, row_tile = row / (16 * RT);
      const int64_t base = a.plan[e] + (int64_t)row_tile * x.tiles * x.weight;
      const int w0 = (int)(base / per), w1 = (int)((base + (int64_t)(x.tiles - 1) * x.weight) / per);
      n_pre = w1 - w0 + 1;
      const int64_t first = (w0 + piece_of<RT>(a, lo, h, row_tile)) * (16 * RT) + row - row_tile * 16 * RT;
      pre_ml = a.pre_ml + first * 2;
      pre_o = a.pre_o + first * D;
    }
  }
  int n_own = 0;
  const float *own_ml = nullptr, *own_o = nullptr;
  const Entry x = entry_of<RT>(a, NH + bh);
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
      const int64_t i = pre ? (int64_t)c * (16 * RT) : (int64_t)(c - n_pre) * a.G;
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

// Rows of a prefix's matrix per wave: as many row tiles as an even share of
// the batch fills (a tile's K and V then serve more rows per read), four at
// most, which is what the registers of a lane hold.
int row_tiles_for(int B, int N, int G) {
  const int rows = (B + N - 1) / N * G;
  return rows > 32 ? 4 : rows > 16 ? 2 : 1;
}

struct Scratch {
  int64_t pre, own;  // pieces
  size_t pre_ml, pre_o, own_ml, own_o, bytes;
};

size_t aligned(size_t n) { return (n + 255) & ~(size_t)255; }

constexpr size_t kPlanBytes = ((kMaxEntries + 2) * sizeof(int) + 255) & ~(size_t)255;

Scratch scratch_for(int B, int N, int G, int H, int D) {
  const int RT = row_tiles_for(B, N, G);
  Scratch s;
  s.pre = kMaxSlots + (int64_t)H * ((int64_t)B * G / (16 * RT) + N + 1);
  s.own = kMaxSlots + (int64_t)B * H;
  s.pre_ml = kPlanBytes;
  s.pre_o = s.pre_ml + aligned(s.pre * 16 * RT * 2 * sizeof(float));
  s.own_ml = s.pre_o + aligned(s.pre * 16 * RT * D * sizeof(float));
  s.own_o = s.own_ml + aligned(s.own * G * 2 * sizeof(float));
  s.bytes = s.own_o + aligned(s.own * G * D * sizeof(float));
  return s;
}

template <int D, int RT>
hipError_t launch(SharedArgs& a, hipStream_t st) {
  a.slots = min(kMaxSlots, cu_count() * wgs_per_cu(RT));
  a.weight = kOwnWeight;
  hipLaunchKernelGGL((shared_split_kernel<D, RT>), dim3(a.slots), dim3(kThreads), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((shared_merge_kernel<D, RT>), dim3(a.B * a.H, a.G), dim3(256), 0, st, a);
  return hipGetLastError();
}

template <int D>
hipError_t launch_rows(SharedArgs& a, int RT, hipStream_t st) {
  return RT == 1 ? launch<D, 1>(a, st) : RT == 2 ? launch<D, 2>(a, st) : launch<D, 4>(a, st);
}

}  // namespace

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
  if (own > kMaxEntries / 2 || pre > kMaxEntries / 2) return WGKV_ERR_UNSUPPORTED;
  // positions and the line's length are 32-bit
  const int64_t cap = (int64_t)max_pages * page_size, pcap = (int64_t)prefix_pages * page_size;
  if (cap > 0x7fffff00 || pcap > 0x7fffff00) return WGKV_ERR_UNSUPPORTED;
  const int RT = row_tiles_for(batch, num_groups, G);
  const int64_t row_tiles = (int64_t)batch * G / (16 * RT) + num_groups;
  if (((cap + 31) / 32 * own + (pcap + 31) / 32 * row_tiles * num_kv_heads) * kOwnWeight > 0x70000000)
    return WGKV_ERR_UNSUPPORTED;
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) return WGKV_ERR_UNSUPPORTED;
  if ((q_stride_b | q_stride_h) & 7) return WGKV_ERR_UNSUPPORTED;
  if (kv4_rows_meet({batch, num_q_heads, 1, 1}, {out_stride_b, out_stride_h, 0, 0}, head_dim)) return WGKV_ERR_ARG;
  const Scratch sc = scratch_for(batch, num_groups, G, num_kv_heads, head_dim);
  if (!workspace || workspace_bytes < sc.bytes || ((uintptr_t)workspace & 15)) return WGKV_ERR_WORKSPACE;
  SharedArgs a{};
  a.q = (const uint16_t*)q;
  a.q_sb = q_stride_b;
  a.q_sh = q_stride_h;
  a.kc = (const uint16_t*)k_cache;
  a.vc = (const uint16_t*)v_cache;
  a.num_pages = num_pages;
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
  a.scale_log2 = softmax_scale == 0.f ? 1.f : fabsf(softmax_scale) * kLog2e;
  a.q_and = softmax_scale == 0.f ? 0u : ~0u;
  a.q_xor = softmax_scale < 0.f ? 0x80008000u : 0u;
  char* ws = (char*)workspace;
  a.plan = (int*)ws;
  a.pre_ml = (float*)(ws + sc.pre_ml);
  a.pre_o = (float*)(ws + sc.pre_o);
  a.own_ml = (float*)(ws + sc.own_ml);
  a.own_o = (float*)(ws + sc.own_o);
  hipStream_t st = (hipStream_t)stream;
  const hipError_t e = head_dim == 128 ? launch_rows<128>(a, RT, st) : launch_rows<64>(a, RT, st);
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
