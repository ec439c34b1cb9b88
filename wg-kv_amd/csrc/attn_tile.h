// Softmax attention of 32 query rows per wave over a tile of 64 keys in LDS,
// on bf16 MFMA (gfx950).
//
// S^T = K Q^T on v_mfma_f32_16x16x32_bf16 (K from LDS as the A operand, the
// wave's queries held as the B operand) leaves each lane 16 scores of one
// query row, which after the softmax are already the B operand of
// O^T = V^T P^T; the V^T operand comes by LDS transpose reads of the row-major
// V tile.  Softmax runs in the log2 domain in fp32 with a running maximum that
// moves only when a score exceeds it by more than 8 (so p <= 2^8 and few
// tiles rescale anything).  Probabilities are rounded to bf16 for the
// products, and their sums are the matrix core's too (ones . P^T), so that
// both halves of the quotient see the same rounding.
//
// Tiles are stored unpadded, D * 2 bytes per key, with the 16-byte slices of
// a row permuted so that operand reads spread over the banks: slice c of row r
// sits at c ^ swz_k(r) in K and at c ^ swz_v(r) in V.
#pragma once

#include "wgkv_common.h"

namespace attn {

constexpr int kKeys = 64;      // keys per tile
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.f;  // log2 units a row maximum may lag its scores

// IEEE-754-2019 maximum (v_maximum3_f32): no canonicalisation, and -inf
// (masked scores) is ordered.
WGKV_DEVICE float fmax_ieee(float x, float y) { return __builtin_elementwise_maximum(x, y); }

// max of x over lanes i and i^16 / i^32
WGKV_DEVICE float xor16_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmax_ieee(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
WGKV_DEVICE float xor32_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmax_ieee(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

typedef short v4i16_t __attribute__((ext_vector_type(4)));

WGKV_DEVICE v4i16_t lds_read_tr16(const uint16_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4i16_t __attribute__((address_space(3)))*)(p));
}

// The 16 bytes at g go to LDS at lds + 16 * lane (lds the same in every lane).
WGKV_DEVICE void lds_dma16(const void* g, uint16_t* lds) { __builtin_amdgcn_global_load_lds(g, lds, 16, 0, 0); }

// 16 consecutive rows of a K operand, and the 8 rows of a V transpose read,
// lie on different banks.
template <int D>
WGKV_DEVICE int swz_k(int row) { return D == 128 ? (row & 15) : ((row >> 1) & 7); }
template <int D>
WGKV_DEVICE int swz_v(int row) { return D == 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3); }

// Per-lane LDS element offsets of the operands: K row kt * 16 + n, slice
// j * 4 + g; the transpose read of lane n in group g covers V row 4g + n/4
// (+ 16u + 32s), d 16 * dt + 4 * (n % 4).
template <int D>
struct Offsets {
  int k[D / 32], v[D / 16];
  WGKV_DEVICE Offsets(int n, int g) {
#pragma unroll
    for (int j = 0; j < D / 32; ++j) k[j] = n * D + ((j * 4 + g) ^ swz_k<D>(n)) * 8;
    const int row = 4 * g + (n >> 2);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
      v[dt] = row * D + ((2 * dt + ((n & 3) >> 1)) ^ swz_v<D>(row)) * 8 + (n & 1) * 4;
  }
};

// 32 query rows of a wave: lane (n, g) holds rows n and 16 + n, and of O the
// values d = 16 * dt + 4 * g + i.
template <int D>
struct Rows32 {
  bf16x8_t q[2][D / 32];
  f32x4_t o[D / 16][2];
  f32x4_t sum[2];  // every entry: the row's sum
  float m[2];

  WGKV_DEVICE void clear() {
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
      m[rt] = -INFINITY;
      sum[rt] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) o[dt][rt] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    }
  }
  // asks for the lane's row of row tile rt at p
  WGKV_DEVICE void ask_q(int rt, const uint16_t* p, int g) {
#pragma unroll
    for (int j = 0; j < D / 32; ++j) q[rt][j] = __builtin_bit_cast(bf16x8_t, *(const u32x4_t*)(p + (j * 4 + g) * 8));
  }
  // the rows have come: the bits' masks apply the scale's sign
  WGKV_DEVICE void take_q(uint32_t q_and, uint32_t q_xor) {
#pragma unroll
    for (int rt = 0; rt < 2; ++rt)
#pragma unroll
      for (int j = 0; j < D / 32; ++j)
        q[rt][j] = __builtin_bit_cast(bf16x8_t, (__builtin_bit_cast(u32x4_t, q[rt][j]) & q_and) ^ q_xor);
  }
};

// sc[kt][rt][i]: key kt * 16 + 4g + i of row rt * 16 + n.  The k-step's operand
// reads run under the k-step before, and the eight chains are independent.
template <int D>
WGKV_DEVICE void tile_scores(const Rows32<D>& r, const uint16_t* sK, const Offsets<D>& at, f32x4_t (&sc)[4][2]) {
#pragma unroll
  for (int kt = 0; kt < 4; ++kt)
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) sc[kt][rt] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  bf16x8_t kf[2][4];
#pragma unroll
  for (int kt = 0; kt < 4; ++kt) kf[0][kt] = __builtin_bit_cast(bf16x8_t, *(const u32x4_t*)(&sK[kt * 16 * D + at.k[0]]));
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    if (j + 1 < D / 32)
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
        kf[(j + 1) & 1][kt] = __builtin_bit_cast(bf16x8_t, *(const u32x4_t*)(&sK[kt * 16 * D + at.k[j + 1]]));
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int rt = 0; rt < 2; ++rt)
        sc[kt][rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[j & 1][kt], r.q[rt][j], sc[kt][rt], 0, 0, 0);
  }
}

// The softmax step over masked scores and the tile's part of O.
template <int D>
WGKV_DEVICE void tile_attend(Rows32<D>& r, f32x4_t (&sc)[4][2], const uint16_t* sV, const Offsets<D>& at,
                             float scale_log2) {
  float mx[2];
#pragma unroll
  for (int rt = 0; rt < 2; ++rt) {
    float x = sc[0][rt][0];
#pragma unroll
    for (int e = 1; e < 15; e += 2)
      x = fmax_ieee(fmax_ieee(x, sc[e >> 2][rt][e & 3]), sc[(e + 1) >> 2][rt][(e + 1) & 3]);
    mx[rt] = fmax_ieee(x, sc[3][rt][3]) * scale_log2;  // this lane's 16 keys of the row
  }
  // only where a lane's maximum exceeds the running one are the row's lanes compared
  if (__builtin_amdgcn_ballot_w64(mx[0] > r.m[0] + kSlack || mx[1] > r.m[1] + kSlack) != 0) {
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
      const float x = xor32_max(xor16_max(mx[rt]));
      const float m = x > r.m[rt] + kSlack ? x : r.m[rt];
      const float scale = m == r.m[rt] ? 1.f : fast_exp2(r.m[rt] - m);
      r.m[rt] = m;
      r.sum[rt] *= scale;
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) r.o[dt][rt] *= scale;
    }
  }
  bf16x8_t pb[2][2];  // [rt][32 keys]
#pragma unroll
  for (int rt = 0; rt < 2; ++rt) {
    const float m = r.m[rt] == -INFINITY ? 0.f : r.m[rt];  // rows with nothing visible keep p = 0
    uint32_t w[8];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int i = 0; i < 4; i += 2)
        w[kt * 2 + i / 2] = pack_bf16x2(fast_exp2(fmaf(sc[kt][rt][i], scale_log2, -m)),
                                        fast_exp2(fmaf(sc[kt][rt][i + 1], scale_log2, -m)));
#pragma unroll
    for (int s = 0; s < 2; ++s)
      pb[rt][s] = __builtin_bit_cast(bf16x8_t, (u32x4_t){w[4 * s], w[4 * s + 1], w[4 * s + 2], w[4 * s + 3]});
  }
  const bf16x8_t ones = __builtin_bit_cast(bf16x8_t, (u32x4_t){0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
#pragma unroll
  for (int s = 0; s < 2; ++s) {
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
      const uint16_t* p = sV + at.v[dt] + s * 32 * D;
      const v4i16_t lo = lds_read_tr16(p), hi = lds_read_tr16(p + 16 * D);
      const bf16x8_t vf = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
      for (int rt = 0; rt < 2; ++rt)
        r.o[dt][rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pb[rt][s], r.o[dt][rt], 0, 0, 0);
    }
#pragma unroll
    for (int rt = 0; rt < 2; ++rt)
      r.sum[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pb[rt][s], r.sum[rt], 0, 0, 0);
  }
}

}  // namespace attn
