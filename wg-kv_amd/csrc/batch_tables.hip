// Page tables and cache rows of a packed batch's tokens, and the copy of its
// keys and values to those rows (gfx950).
//
// A packed batch holds the new tokens of B requests behind each other, rows
// cu[b] .. cu[b+1] - 1 of N for request b.  Head (b, h) holds len tokens
// already and keeps c of the new ones (all, or those its mask admits).  With
// pages of P tokens it needs ceil((len + c)/P) - ceil(len/P) new pages; the
// new pages of all heads are numbered by an exclusive sum in row-major (b, h)
// order, and number i is
//   free_ids[held - take + i]   for i < take = min(pages needed, held)
//   next + i - take             from there on
// (the free list's last entries in list order, then the bump pointer: the
// dual cache's rule).  The r-th kept token of a head goes to position len + r,
// row table[b, h, pos / P] * P + pos % P of the pools.  A page's first token
// writes the page's table entry, so no launch goes over pages.
//
// All of it is latency: 0.5 MB of mask and 2 MB of rows of 16K tokens and 8
// heads take under a microsecond of bandwidth.  So launches are few and loads
// do not wait for one another: a step of up to 256 tokens (a decode step) is one
// launch of one workgroup.  A longer one has a workgroup per 256 tokens, each
// of which makes the whole plan in LDS for itself; its kept tokens are counted
// by a launch before that if there is a mask.  Where the plan does not fit into
// LDS it is a launch of one workgroup between the two.
#include <string.h>

#include "kv4.h"

namespace {

constexpr int kTile = 256;       // tokens per tile
constexpr int kHeadGroup = 16;   // heads whose rows are gathered in LDS for one coalesced write
constexpr int kPlanThreads = 1024;
constexpr int kLdsHeads = 4096;    // (request, head) pairs that a workgroup plans in LDS, (tile, head) pairs too

struct TablesArgs {
  const int32_t* len;
  int64_t len_sb;
  const int32_t* cu;
  int N;
  const uint8_t* mask;  // (H, N) or NULL: every token is kept
  int64_t mask_sh;
  int32_t* bt;
  int64_t bt_sb, bt_sh;
  int max_pages;
  const int32_t* state;  // next unused page, entries of the free list
  int32_t* state_out;
  const int32_t* free_ids;
  int free_cap;
  int64_t num_pages;
  int page_log2;
  int32_t* out;  // new lengths
  int64_t out_sb;
  int32_t* slots;  // (N, H)
  int B, H;
  int32_t* status;
  // scratch of the steps that take more than one launch
  int tiles;
  int* tile_count;   // (H, tiles): kept tokens of a tile; of the tiles before it once there is a plan
  int* start_count;  // (B + 1, H): kept tokens of cu[b]'s tile before cu[b]
  int4* plan;        // (B * H)
  int4* head;        // one entry
  // lengths and page state as they were, for the workgroups that read them while
  // one replaces them
  int* len_copy;
  int* state_copy;
};

// What the rows of a head need: tokens held, kept tokens of the whole batch
// before the request's first, first new page's number.
struct HeadPlan {
  int len, before, page;
};
// The step's page state: entries taken off the free list, the bump pointer,
// entries held, and whether everything fits.
struct StepPlan {
  int take, next, held, fits;
};

WGKV_DEVICE int clamped_cu(const TablesArgs& a, int b) { return min(max(a.cu[b], 0), a.N); }

WGKV_DEVICE int clamped_len(const TablesArgs& a, int e) {
  const int b = e / a.H, h = e - b * a.H;
  return min(max(a.len[(int64_t)b * a.len_sb + h], 0), a.max_pages << a.page_log2);
}

// The last of B requests that starts at or before token n, or -1 where n lies
// in none (before the first or behind the last).
WGKV_DEVICE int request_of(const int* cu, int B, int n) {
  int lo = 0, hi = B;  // cu[lo] <= n < cu[hi]
  if (n < cu[0] || n >= cu[B]) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= n) lo = mid; else hi = mid;
  }
  return lo;
}

// First b with cu[b] >= n (B + 1: none).
WGKV_DEVICE int first_start(const TablesArgs& a, int n) {
  int lo = 0, hi = a.B + 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (clamped_cu(a, mid) < n) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// Lane's four tokens of a tile (4 * lane ...): bit i set where token i of
// them is kept by head h.
WGKV_DEVICE int kept_bits(const TablesArgs& a, int h, int tile, int lane) {
  const int n0 = tile * kTile + 4 * lane;
  int bits = 0;
  const uint8_t* m = a.mask + (int64_t)h * a.mask_sh;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n0 + i < a.N && m[n0 + i]) bits |= 1 << i;
  return bits;
}

// One wave: head h's kept tokens of a tile, and of the tile before each
// request start in it (starts b0 .. b1 - 1) to start_count.
WGKV_DEVICE int count_tile(const TablesArgs& a, int h, int tile, int b0, int b1, int lane, int* start_count) {
  const int bits = kept_bits(a, h, tile, lane);
  const int mine = __builtin_popcount(bits);
  const int incl = wave_incl_scan(mine, lane);
  for (int base = b0; base < b1; base += 64) {  // every lane takes part in the exchange
    const int b = base + lane;
    const int x = b < b1 ? clamped_cu(a, b) - tile * kTile : 0;
    const int from = min(max(x >> 2, 0), 63);
    const int before = __shfl(incl - mine, from, 64);
    const int there = __shfl(bits, from, 64);
    if (b < b1) start_count[(int64_t)b * a.H + h] = before + __builtin_popcount(there & ((1 << (x & 3)) - 1));
  }
  return __builtin_amdgcn_readlane(incl, 63);
}

// Exclusive sum over the threads of a workgroup of kThreads, and the total.
template <int kThreads>
WGKV_DEVICE int block_exclusive_scan(int v, int* s_wave, int* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int incl = wave_incl_scan(v, lane);
  if (lane == 63) s_wave[w] = incl;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) {
    before += i < w ? s_wave[i] : 0;
    all += s_wave[i];
  }
  __syncthreads();
  *total = all;
  return before + incl - v;
}

// Page state as a plan starts from it.
struct PageState {
  int next, held, held_given;
};
WGKV_DEVICE PageState page_state(const TablesArgs& a) {
  const int given = a.state[1];
  return {max(a.state[0], 0), a.free_ids ? min(max(given, 0), a.free_cap) : 0, given};
}

// New pages of a head that keeps `kept` tokens more; *over: it outgrows its table.
WGKV_DEVICE int pages_needed(const TablesArgs& a, int len, int kept, int* over) {
  const int up = (1 << a.page_log2) - 1;
  if ((int64_t)len + kept > (int64_t)a.max_pages << a.page_log2) {
    *over = 1;
    return 0;
  }
  return ((len + kept + up) >> a.page_log2) - ((len + up) >> a.page_log2);
}

// The step's plan from the pages that it needs in all.
WGKV_DEVICE StepPlan step_plan(const TablesArgs& a, const PageState& st, int total, bool over) {
  StepPlan s;
  s.held = st.held;
  s.next = st.next;
  s.take = min(total, s.held);
  s.fits = !over && (int64_t)s.next + total - s.take <= a.num_pages;
  return s;
}

// New page state and status, by one thread.
WGKV_DEVICE void put_state(const TablesArgs& a, const PageState& st, const StepPlan& s, int total) {
  a.state_out[0] = s.next + (s.fits ? total - s.take : 0);
  a.state_out[1] = a.free_ids ? s.held - (s.fits ? s.take : 0) : st.held_given;
  if (!s.fits && a.status) *a.status = WGKV_ERR_CAPACITY;
}

// Rows of a tile's tokens for all heads, by a workgroup of NW waves: a wave
// takes a head and 64 of the tokens, whose requests are in s_req; the rows of
// kHeadGroup heads meet in LDS and are written as they lie in memory.
// tile_before(h): kept tokens of the tiles before this one.
template <int NW, typename Plan, typename Before>
WGKV_DEVICE void tile_rows(const TablesArgs& a, int tile, const StepPlan& s, const int* s_req, int* s_row, Plan plan,
                           Before tile_before) {
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int mask = (1 << a.page_log2) - 1;
  const int n_tok = min(kTile, a.N - tile * kTile);
  for (int h0 = 0; h0 < a.H; h0 += kHeadGroup) {
    const int hg = min(kHeadGroup, a.H - h0);
    for (int u = w; u < hg * (kTile / 64); u += NW) {
      const int hh = u / (kTile / 64), part = u % (kTile / 64), h = h0 + hh, x = part * 64 + lane;
      bool kept = x < n_tok;
      int before = tile * kTile + x;  // kept tokens of the batch before this one
      if (a.mask) {
        const uint8_t* m = a.mask + (int64_t)h * a.mask_sh + tile * kTile;
        uint8_t on[kTile / 64];
#pragma unroll
        for (int i = 0; i < kTile / 64; ++i) on[i] = i <= part && i * 64 + lane < n_tok ? m[i * 64 + lane] : 0;
        before = tile_before(h);
#pragma unroll
        for (int i = 0; i < kTile / 64; ++i) {
          const uint64_t set = __ballot(on[i] != 0);
          if (i < part) before += __popcll(set);
          if (i == part) {
            before += __popcll(set & ((1ull << lane) - 1));
            kept = on[i] != 0;
          }
        }
      }
      const int b = s_req[x];
      int row = -1;
      if (b >= 0 && kept && s.fits) {
        const HeadPlan p = plan(b * a.H + h);
        const int pos = p.len + before - p.before;
        const int j = pos >> a.page_log2, p0 = (p.len + mask) >> a.page_log2;
        // (a negative or too large position: cu does not ascend)
        if (pos >= p.len && j < a.max_pages) {
          int32_t* entry = a.bt + (int64_t)b * a.bt_sb + (int64_t)h * a.bt_sh + j;
          const int k = p.page + j - p0;  // of the new pages
          int id = k < 0 ? -1 : s.next + k - s.take;
          const int32_t* held = j < p0 ? entry : k >= 0 && k < s.take ? a.free_ids + (s.held - s.take + k) : nullptr;
          if (held) id = *held;
          if (j >= p0 && k >= 0 && (pos & mask) == 0) *entry = id;
          if (id >= 0 && id < a.num_pages) row = (id << a.page_log2) + (pos & mask);
          else if (a.status) *a.status = WGKV_ERR_CAPACITY;
        }
      }
      s_row[x * hg + hh] = row;
    }
    __syncthreads();
    for (int i = t; i < n_tok * hg; i += NW * 64) {
      const int x = i / hg;
      a.slots[(int64_t)(tile * kTile + x) * a.H + h0 + i - x * hg] = s_row[i];
    }
    __syncthreads();
  }
}

// Steps whose plan fits into LDS.  (256 requests x 8 heads x 1 token 6.9 us; 8
// requests of 2 to 4 thousand gated tokens 8.7 behind 4.3 of counting; 64K tokens
// of one request 6.9.)  ONE: of up to kTile tokens, one workgroup,
// which counts the mask itself; otherwise a workgroup per tile, of which the
// first writes the lengths and the state.
template <bool ONE>
__global__ __launch_bounds__(kPlanThreads) void tables_step_kernel(TablesArgs a) {
  constexpr int NW = kPlanThreads / 64, PER = kLdsHeads / kPlanThreads;
  __shared__ int s_cu[kLdsHeads], s_len[kLdsHeads], s_before[kLdsHeads], s_page[kLdsHeads];
  __shared__ int s_kept[kLdsHeads + kTile];  // ONE: kept tokens before each start; else before each tile
  __shared__ int s_row[kTile * kHeadGroup];
  __shared__ int s_req[kTile], s_wave[NW], s_over;
  const int t = threadIdx.x, lane = t & 63, w = t >> 6, tile = blockIdx.x, BH = a.B * a.H;
  const int per = (BH + kPlanThreads - 1) / kPlanThreads;
  const int lo = min(BH, t * per), n_mine = min(BH, lo + per) - lo;
  // What does not depend on anything is asked for at once.
  const PageState st = page_state(a);
  int len[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) len[k] = k < n_mine ? clamped_len(a, lo + k) : 0;
  for (int b = t; b <= a.B; b += kPlanThreads) s_cu[b] = clamped_cu(a, b);
  if (t == 0) s_over = 0;
  if (a.mask) {
    for (int h = w; h < a.H; h += NW) {
      if constexpr (ONE) {
        const int all = count_tile(a, h, 0, 0, a.B + 1, lane, s_kept);
        // (a start at kTile lies behind the tile's last lane)
        for (int b = lane; b <= a.B; b += 64)
          if (clamped_cu(a, b) >= kTile) s_kept[b * a.H + h] = all;
      } else {
        const int* c = a.tile_count + (int64_t)h * a.tiles;
        int run = 0;
        for (int i0 = 0; i0 <= a.tiles; i0 += 64) {  // entry `tiles` is the total
          const int n = i0 + lane < a.tiles ? c[i0 + lane] : 0;
          const int incl = wave_incl_scan(n, lane);
          if (i0 + lane <= a.tiles) s_kept[h * (a.tiles + 1) + i0 + lane] = run + incl - n;
          run += __builtin_amdgcn_readlane(incl, 63);
        }
      }
    }
  }
  __syncthreads();
  if (t < kTile) s_req[t] = tile * kTile + t < a.N ? request_of(s_cu, a.B, tile * kTile + t) : -1;
  const auto kept_before = [&](int b, int h) {
    if (!a.mask) return s_cu[b];
    if (ONE) return s_kept[b * a.H + h];
    const int n = s_cu[b], in_tile = n < a.N ? a.start_count[(int64_t)b * a.H + h] : 0;
    return s_kept[h * (a.tiles + 1) + (n < a.N ? n / kTile : a.tiles)] + in_tile;
  };
  int need[PER], kept[PER], mine = 0, over = 0, total;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    need[k] = kept[k] = 0;
    if (k >= n_mine) continue;
    const int e = lo + k, b = e / a.H, h = e - b * a.H, before = kept_before(b, h);
    kept[k] = max(kept_before(b + 1, h) - before, 0);
    need[k] = pages_needed(a, len[k], kept[k], &over);
    s_len[e] = len[k];
    s_before[e] = before;
    mine += need[k];
  }
  if (over) s_over = 1;
  int page = block_exclusive_scan<kPlanThreads>(mine, s_wave, &total);
  const StepPlan s = step_plan(a, st, total, s_over);
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    if (k >= n_mine) continue;
    const int e = lo + k, b = e / a.H;
    s_page[e] = page;
    page += need[k];
    // (in place, ONE only: this thread alone has read this length)
    if (ONE || tile == 0) a.out[(int64_t)b * a.out_sb + e - b * a.H] = len[k] + (s.fits ? kept[k] : 0);
  }
  if ((ONE || tile == 0) && t == 0) put_state(a, st, s, total);  // (every thread has read it: it has passed barriers)
  __syncthreads();
  if (a.N)
    tile_rows<NW>(a, tile, s, s_req, s_row, [&](int e) { return HeadPlan{s_len[e], s_before[e], s_page[e]}; },
                  [&](int h) { return ONE ? 0 : s_kept[h * (a.tiles + 1) + tile]; });
}

// Kept tokens of every tile and head, and of a tile before the request starts
// in it; copies of what is replaced in place.
__global__ __launch_bounds__(256) void tables_count_kernel(TablesArgs a) {
  const int tile = blockIdx.x, lane = threadIdx.x & 63;
  if (tile == 0 && a.len_copy) {
    for (int e = threadIdx.x; e < a.B * a.H; e += 256) a.len_copy[e] = clamped_len(a, e);
    if (threadIdx.x < 2) a.state_copy[threadIdx.x] = a.state[threadIdx.x];
  }
  if (!a.mask) return;
  const int b0 = first_start(a, tile * kTile), b1 = first_start(a, (tile + 1) * kTile);
  for (int h = threadIdx.x >> 6; h < a.H; h += 4) {
    const int n = count_tile(a, h, tile, b0, b1, lane, a.start_count);
    if (lane == 0) a.tile_count[(int64_t)h * a.tiles + tile] = n;
  }
}

// The plan over all heads, by one workgroup whose threads take consecutive
// entries.
__global__ __launch_bounds__(kPlanThreads) void tables_plan_kernel(TablesArgs a) {
  __shared__ int s_wave[kPlanThreads / 64], s_over;
  const int t = threadIdx.x, lane = t & 63, BH = a.B * a.H;
  if (a.mask) {  // tile counts become sums of the tiles before; entry `tiles` is the total
    for (int h = t >> 6; h < a.H; h += kPlanThreads / 64) {
      int* c = a.tile_count + (int64_t)h * a.tiles;
      int run = 0;
      for (int i0 = 0; i0 < a.tiles; i0 += 64) {
        const int n = i0 + lane < a.tiles ? c[i0 + lane] : 0;
        const int incl = wave_incl_scan(n, lane);
        if (i0 + lane < a.tiles) c[i0 + lane] = run + incl - n;
        run += __builtin_amdgcn_readlane(incl, 63);
      }
      if (lane == 0) a.tile_count[(int64_t)a.H * a.tiles + h] = run;
    }
    __threadfence_block();
  }
  if (t == 0) s_over = 0;
  __syncthreads();
  const auto kept_before = [&](int b, int h) {
    const int n = clamped_cu(a, b);
    if (!a.mask) return n;
    if (n >= a.N) return a.tile_count[(int64_t)a.H * a.tiles + h];
    return a.tile_count[(int64_t)h * a.tiles + n / kTile] + a.start_count[(int64_t)b * a.H + h];
  };
  const PageState st = page_state(a);
  const int per = (BH + kPlanThreads - 1) / kPlanThreads, lo = min(BH, t * per), hi = min(BH, lo + per);
  int mine = 0, over = 0, total;
  for (int e = lo; e < hi; ++e) {
    const int b = e / a.H, h = e - b * a.H, before = kept_before(b, h);
    mine += pages_needed(a, clamped_len(a, e), max(kept_before(b + 1, h) - before, 0), &over);
  }
  if (over) s_over = 1;
  int page = block_exclusive_scan<kPlanThreads>(mine, s_wave, &total);
  const StepPlan s = step_plan(a, st, total, s_over);
  for (int e = lo; e < hi; ++e) {
    const int b = e / a.H, h = e - b * a.H, len = clamped_len(a, e), before = kept_before(b, h);
    const int kept = max(kept_before(b + 1, h) - before, 0);
    a.plan[e] = make_int4(len, before, page, 0);
    page += pages_needed(a, len, kept, &over);
    // (in place: only this thread reads this length, before)
    a.out[(int64_t)b * a.out_sb + h] = len + (s.fits ? kept : 0);
  }
  if (t == 0) {
    put_state(a, st, s, total);  // (every thread has read it: it has passed barriers)
    *a.head = make_int4(s.take, s.next, s.held, s.fits);
  }
}

__global__ __launch_bounds__(256) void tables_rows_kernel(TablesArgs a) {
  __shared__ int s_row[kTile * kHeadGroup];
  __shared__ int s_req[kTile];
  const int4 hd = *a.head;
  const StepPlan s = {hd.x, hd.y, hd.z, hd.w};
  const int t = threadIdx.x, tile = blockIdx.x;
  s_req[t] = tile * kTile + t < a.N ? request_of(a.cu, a.B, tile * kTile + t) : -1;
  __syncthreads();
  tile_rows<4>(a, tile, s, s_req, s_row,
               [&](int e) {
                 const int4 p = a.plan[e];
                 return HeadPlan{p.x, p.y, p.z};
               },
               [&](int h) { return a.tile_count[(int64_t)h * a.tiles + tile]; });
}

struct AppendArgs {
  const uint16_t* src[2];
  int64_t s_n[2], s_h[2];
  uint16_t* dst[2];
  const int32_t* slots;
  int64_t rows;  // N * H
  int64_t cache_rows;
  int H, chunks;  // 16-byte pieces of a row
};

// Rows to their places, 16 bytes per thread and step, keys and values
// together: pure bandwidth.  Four pieces of each are asked for before the
// first is written.  Nothing orders two tokens with one slot: a row may come to
// hold pieces of both.  64K tokens x 8 heads, D 128: 537 MB in 109 us, 4.9 TB/s (a
// plain copy 5.0).
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a) {
  constexpr int U = 4;
  // the workgroup's first piece; what is behind it stays in 32 bits
  const int64_t e0 = (int64_t)blockIdx.x * (256 * U);
  const uint32_t r0 = (uint32_t)(e0 / a.chunks), c0 = (uint32_t)(e0 - (int64_t)r0 * a.chunks);
  u32x4_t x[2][U];
  int64_t at[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t e = c0 + threadIdx.x + u * 256, up = e / (uint32_t)a.chunks, r = r0 + up;
    const int c = (int)(e - up * a.chunks);
    at[u] = -1;
    if (r >= a.rows) continue;
    const int64_t row = a.slots[r];
    if (row < 0 || row >= a.cache_rows) continue;
    const int64_t n = r / (uint32_t)a.H;
    const int h = (int)(r - (uint32_t)n * a.H);
    at[u] = row * a.chunks + c;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      x[i][u] = __builtin_nontemporal_load((const u32x4_t*)(a.src[i] + n * a.s_n[i] + h * a.s_h[i]) + c);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (at[u] < 0) continue;
#pragma unroll
    for (int i = 0; i < 2; ++i) *((u32x4_t*)a.dst[i] + at[u]) = x[i][u];
  }
}

int page_log2_of(int page_size) { return page_size == 16 ? 4 : page_size == 32 ? 5 : page_size == 64 ? 6 : -1; }

// Whether the plan fits into LDS, with the sums over its tiles.
bool lds_step(int B, int H, int N) {
  return (int64_t)(B + 1) * H <= kLdsHeads && ((int64_t)N / kTile + 2) * H <= kLdsHeads;
}
bool small_step(int B, int H, int N) { return N <= kTile && (int64_t)(B + 1) * H <= kLdsHeads; }

size_t aligned(size_t n) { return (n + 255) & ~(size_t)255; }

struct TablesScratch {
  size_t count, start, plan, head, bytes;
};

TablesScratch tables_scratch(int B, int H, int N) {
  TablesScratch s;
  const size_t tiles = ((size_t)N + kTile - 1) / kTile;
  s.count = 0;
  s.start = aligned((size_t)H * (tiles + 1) * sizeof(int));
  s.plan = s.start + aligned((size_t)(B + 1) * H * sizeof(int));
  s.head = s.plan + aligned((size_t)B * H * sizeof(int4));
  s.bytes = s.head + 256;
  return s;
}

}  // namespace

extern "C" size_t wgkv_block_tables_workspace_bytes(int32_t batch, int32_t num_kv_heads, int32_t num_tokens) {
  if (batch <= 0 || num_kv_heads <= 0 || num_tokens < 0 || small_step(batch, num_kv_heads, num_tokens)) return 0;
  return tables_scratch(batch, num_kv_heads, num_tokens).bytes;
}

extern "C" int wgkv_build_block_tables(
    const int32_t* lengths, int64_t len_stride_b, const int32_t* cu_seqlens, int32_t num_tokens,
    const uint8_t* g_mask, int64_t gm_stride_h,
    int32_t* block_table, int64_t bt_stride_b, int64_t bt_stride_h, int32_t max_pages,
    const int32_t* page_state, int32_t* state_out, const int32_t* free_ids, int32_t free_capacity,
    int64_t num_pages, int32_t page_size,
    int32_t* new_lengths, int64_t new_stride_b, int32_t* slots,
    int32_t batch, int32_t num_kv_heads, int32_t* status,
    void* workspace, size_t workspace_bytes, void* stream) {
  if (!lengths || !cu_seqlens || !block_table || !page_state || !state_out || !new_lengths) return WGKV_ERR_ARG;
  if (batch <= 0 || num_kv_heads <= 0 || num_tokens < 0 || max_pages <= 0 || num_pages <= 0) return WGKV_ERR_ARG;
  if ((num_tokens && !slots) || free_capacity < 0 || (!free_ids && free_capacity)) return WGKV_ERR_ARG;
  const int log2 = page_log2_of(page_size);
  if (log2 < 0) return WGKV_ERR_UNSUPPORTED;
  // positions, rows and heads are counted in 32 bits
  constexpr int64_t kMax = 0x7fffffff;
  if (num_pages > (kMax >> log2) || max_pages > (kMax >> log2) - 1 || num_tokens > kMax - 2 * kTile ||
      ((int64_t)batch + 1) * num_kv_heads > (1 << 24) || (int64_t)num_tokens * num_kv_heads > kMax)
    return WGKV_ERR_UNSUPPORTED;
  // rows that are written apart
  if (kv4_rows_meet({batch, num_kv_heads, 1, 1}, {bt_stride_b, bt_stride_h, 0, 0}, max_pages) ||
      kv4_rows_meet({batch, 1, 1, 1}, {new_stride_b, 0, 0, 0}, num_kv_heads))
    return WGKV_ERR_ARG;
  const TablesScratch sc = tables_scratch(batch, num_kv_heads, num_tokens);
  const bool small = small_step(batch, num_kv_heads, num_tokens);
  const bool lds = lds_step(batch, num_kv_heads, num_tokens);
  const bool copies = !small && lds && (new_lengths == lengths || state_out == page_state);
  const bool scratch = !small && (g_mask || copies || !lds);
  if (scratch && (!workspace || workspace_bytes < sc.bytes || ((uintptr_t)workspace & 15))) return WGKV_ERR_WORKSPACE;
  TablesArgs a{};
  a.len = lengths;
  a.len_sb = len_stride_b;
  a.cu = cu_seqlens;
  a.N = num_tokens;
  a.mask = g_mask;
  a.mask_sh = gm_stride_h;
  a.bt = block_table;
  a.bt_sb = bt_stride_b;
  a.bt_sh = bt_stride_h;
  a.max_pages = max_pages;
  a.state = page_state;
  a.state_out = state_out;
  a.free_ids = free_ids;
  a.free_cap = free_capacity;
  a.num_pages = num_pages;
  a.page_log2 = log2;
  a.out = new_lengths;
  a.out_sb = new_stride_b;
  a.slots = slots;
  a.B = batch;
  a.H = num_kv_heads;
  a.status = status;
  hipStream_t st = (hipStream_t)stream;
  if (small) {
    hipLaunchKernelGGL(tables_step_kernel<true>, dim3(1), dim3(kPlanThreads), 0, st, a);
    return hipGetLastError() == hipSuccess ? WGKV_OK : WGKV_ERR_HIP;
  }
  a.tiles = (num_tokens + kTile - 1) / kTile;
  if (scratch) {
    char* ws = (char*)workspace;
    a.tile_count = (int*)(ws + sc.count);
    a.start_count = (int*)(ws + sc.start);
    a.plan = (int4*)(ws + sc.plan);
    a.head = (int4*)(ws + sc.head);
  }
  if (copies) {
    a.len_copy = (int*)a.plan;
    a.state_copy = (int*)a.head;
  }
  if ((g_mask && a.tiles) || copies) {
    hipLaunchKernelGGL(tables_count_kernel, dim3(g_mask ? a.tiles : 1), dim3(256), 0, st, a);
    WGKV_HIP_CHECK(hipGetLastError());
  }
  if (lds) {
    if (copies) {
      a.len = a.len_copy;
      a.len_sb = num_kv_heads;
      a.state = a.state_copy;
    }
    hipLaunchKernelGGL(tables_step_kernel<false>, dim3(a.tiles), dim3(kPlanThreads), 0, st, a);
    return hipGetLastError() == hipSuccess ? WGKV_OK : WGKV_ERR_HIP;
  }
  hipLaunchKernelGGL(tables_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, a);
  WGKV_HIP_CHECK(hipGetLastError());
  if (a.tiles) {
    hipLaunchKernelGGL(tables_rows_kernel, dim3(a.tiles), dim3(256), 0, st, a);
    WGKV_HIP_CHECK(hipGetLastError());
  }
  return WGKV_OK;
}

extern "C" int wgkv_paged_append(
    const void* key, int64_t k_stride_n, int64_t k_stride_h, const void* value, int64_t v_stride_n, int64_t v_stride_h,
    void* k_cache, void* v_cache, int64_t cache_rows, const int32_t* slots,
    int32_t num_tokens, int32_t num_kv_heads, int32_t head_dim, void* stream) {
  if (num_tokens < 0 || num_kv_heads <= 0 || head_dim <= 0 || cache_rows < 0) return WGKV_ERR_ARG;
  if (num_tokens == 0) return WGKV_OK;
  if (!key || !value || !k_cache || !v_cache || !slots) return WGKV_ERR_ARG;
  if (head_dim % 8 || cache_rows > 0x7fffffff || (int64_t)num_tokens * num_kv_heads > 0x7fffffff)
    return WGKV_ERR_UNSUPPORTED;
  if (((uintptr_t)key | (uintptr_t)value | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) return WGKV_ERR_UNSUPPORTED;
  if ((k_stride_n | k_stride_h | v_stride_n | v_stride_h) & 7) return WGKV_ERR_UNSUPPORTED;
  const int64_t bytes = cache_rows * head_dim * 2;
  const char *k0 = (const char*)k_cache, *v0 = (const char*)v_cache;
  if (k0 < v0 + bytes && v0 < k0 + bytes) return WGKV_ERR_ARG;  // the pools share bytes
  AppendArgs a{};
  a.src[0] = (const uint16_t*)key;
  a.src[1] = (const uint16_t*)value;
  a.s_n[0] = k_stride_n;
  a.s_n[1] = v_stride_n;
  a.s_h[0] = k_stride_h;
  a.s_h[1] = v_stride_h;
  a.dst[0] = (uint16_t*)k_cache;
  a.dst[1] = (uint16_t*)v_cache;
  a.slots = slots;
  a.rows = (int64_t)num_tokens * num_kv_heads;
  a.cache_rows = cache_rows;
  a.H = num_kv_heads;
  a.chunks = head_dim / 8;
  const int64_t blocks = (a.rows * a.chunks + 1023) / 1024;
  if (blocks > 0x7fffffff) return WGKV_ERR_UNSUPPORTED;
  hipLaunchKernelGGL(paged_append_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a);
  return hipGetLastError() == hipSuccess ? WGKV_OK : WGKV_ERR_HIP;
}

extern "C" int wgkv_build_block_tables_block(const void* args) {
  int64_t a[25];
  memcpy(a, args, sizeof a);
  if (!kv4_narrow(a, 3, 9, 13, 15, 19, 20)) return WGKV_ERR_UNSUPPORTED;
  return wgkv_build_block_tables((const int32_t*)a[0], a[1], (const int32_t*)a[2], (int32_t)a[3], (const uint8_t*)a[4],
                                 a[5], (int32_t*)a[6], a[7], a[8], (int32_t)a[9], (const int32_t*)a[10],
                                 (int32_t*)a[11], (const int32_t*)a[12], (int32_t)a[13], a[14], (int32_t)a[15],
                                 (int32_t*)a[16], a[17], (int32_t*)a[18], (int32_t)a[19], (int32_t)a[20],
                                 (int32_t*)a[21], (void*)a[22], (size_t)a[23], (void*)a[24]);
}

extern "C" int wgkv_paged_append_block(const void* args) {
  int64_t a[14];
  memcpy(a, args, sizeof a);
  if (!kv4_narrow(a, 10, 11, 12)) return WGKV_ERR_UNSUPPORTED;
  return wgkv_paged_append((const void*)a[0], a[1], a[2], (const void*)a[3], a[4], a[5], (void*)a[6], (void*)a[7], a[8],
                           (const int32_t*)a[9], (int32_t)a[10], (int32_t)a[11], (int32_t)a[12], (void*)a[13]);
}
