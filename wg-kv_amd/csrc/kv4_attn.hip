// One token's attention over a paged cache held in 4 bits (gfx950).
//
//   z_t = scale * sum_d q_d (m_tg + s_tg (c_td - 7.5)),  p = softmax(z),
//   out_d = sum_t p_t (m_tg + s_tg (c_td - 7.5)),  g = d / 32
//
// One workgroup per (sequence, query head).  D/8 lanes share a quad of 4
// tokens (kv4.h: a lane takes 8 consecutive d of the quad), keep a running
// maximum and sum of their own quads, and the groups are merged through LDS.
#include "kv4.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f;

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
  int B, Hq, Hkv;
  float scale_log2;
};

template <int D>
__global__ __launch_bounds__(256) void kv4_attn_kernel(AttnArgs a) {
  constexpr int LPR = D / 8, QPW = 64 / LPR, NG = D / kKv4Group, GROUPS = 256 / LPR;
  __shared__ float s_acc[GROUPS][D];
  __shared__ float s_m[GROUPS], s_l[GROUPS];
  const int b = blockIdx.y, hq = blockIdx.x;
  const int h = hq / (a.Hq / a.Hkv);
  const int64_t cap = kv4_capacity(a.pg);
  int64_t len = a.len[(int64_t)b * a.len_sb + h];
  len = len < 0 ? 0 : len > cap ? cap : len;
  const int32_t* bt_row = a.pg.bt + (int64_t)b * a.pg.bt_sb + (int64_t)h * a.pg.bt_sh;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int L = lane % LPR, grp = wid * QPW + lane / LPR;

  float q[8];
  kv4_load8<kKv4Bf16>(a.q, (int64_t)b * a.q_sb + (int64_t)hq * a.q_sh + L * 8, q);

  float m_run = -INFINITY, l_run = 0.f, acc[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = 0.f;

  const int nq = (int)((len + 3) >> 2);
  for (int quad = grp; quad < nq; quad += GROUPS) {
    const int64_t at = kv4_tile_clamped<D>(a.pg, bt_row, quad >> 2);
    const int qi = quad & 3;
    const int soff = kv4_scales_at(D) + (qi * NG + L / 4) * 16;
    const u32x4_t ks = *(const u32x4_t*)(a.kc + at + soff), vs = *(const u32x4_t*)(a.vc + at + soff);
    const u32x4_t v = *(const u32x4_t*)(a.vc + at + qi * (2 * D) + L * 16);
    float z[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = *(const uint32_t*)(a.kc + at + (qi * 4 + i) * (D / 2) + L * 4);
      const float s = bf16lo(ks[i]), m = bf16hi(ks[i]);
      float x = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x = fmaf(q[2 * j], fmaf(s, (float)(w >> (4 * j) & 15u) - 7.5f, m), x);
        x = fmaf(q[2 * j + 1], fmaf(s, (float)(w >> (16 + 4 * j) & 15u) - 7.5f, m), x);
      }
#pragma unroll
      for (int o = 1; o < LPR; o <<= 1) x += __shfl_xor(x, o, 64);
      z[i] = quad * 4 + i < len ? x * a.scale_log2 : -INFINITY;
    }
    const float mn = fmaxf(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])), m_run);
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float alpha = fast_exp2(m_run - mu);
    m_run = mn;
    l_run *= alpha;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] *= alpha;
    constexpr int kWord = D == 128 ? 1 : 2, kPair = D == 128 ? 2 : 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (quad * 4 + i >= len) continue;  // rows past the end hold anything
      const float p = fast_exp2(z[i] - mu);
      const float s = bf16lo(vs[i]), m = bf16hi(vs[i]);
      l_run += p;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t w = v[(i >> 1) * kPair + (j >> 2) * kWord] >> (16 * (i & 1));
        acc[j] = fmaf(p, fmaf(s, (float)(w >> (4 * (j & 3)) & 15u) - 7.5f, m), acc[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) s_acc[grp][L * 8 + j] = acc[j];
  if (L == 0) {
    s_m[grp] = m_run;
    s_l[grp] = l_run;
  }
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += 256) {
    float M = -INFINITY, S = 0.f, A = 0.f;
    for (int g = 0; g < GROUPS; ++g) M = fmaxf(M, s_m[g]);
    if (M == -INFINITY) M = 0.f;
    for (int g = 0; g < GROUPS; ++g) {
      const float sc = fast_exp2(s_m[g] - M);
      S = fmaf(sc, s_l[g], S);
      A = fmaf(sc, s_acc[g][d], A);
    }
    a.out[(int64_t)b * a.out_sb + (int64_t)hq * a.out_sh + d] = f32_to_bf16(len > 0 ? A / S : 0.f);
  }
}

}  // namespace

extern "C" int wgkv_kv4_decode_attn(
    const void* q, int64_t q_stride_b, int64_t q_stride_h,
    const void* k_cache, const void* v_cache, int64_t num_pages, int32_t page_size,
    const int32_t* cache_seqlens, int64_t sl_stride_b,
    const int32_t* block_table, int64_t bt_stride_b, int64_t bt_stride_h, int32_t max_pages,
    void* out, int64_t out_stride_b, int64_t out_stride_h,
    int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    float softmax_scale, void* stream) {
  if (!q || !k_cache || !v_cache || !cache_seqlens || !out) return WGKV_ERR_ARG;
  if (batch <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads) return WGKV_ERR_ARG;
  if ((int64_t)batch * num_kv_heads > 2048 || num_q_heads / num_kv_heads > 8) return WGKV_ERR_UNSUPPORTED;
  if (head_dim != 64 && head_dim != 128) return WGKV_ERR_UNSUPPORTED;
  AttnArgs a{};
  const int st = kv4_pages(&a.pg, num_pages, page_size, block_table, bt_stride_b, bt_stride_h, max_pages);
  if (st != WGKV_OK) return st;
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) return WGKV_ERR_UNSUPPORTED;
  if ((q_stride_b | q_stride_h) & 7) return WGKV_ERR_UNSUPPORTED;
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
  a.Hq = num_q_heads;
  a.Hkv = num_kv_heads;
  a.scale_log2 = softmax_scale * kLog2e;
  const dim3 g(num_q_heads, batch);
  hipStream_t s = (hipStream_t)stream;
  if (head_dim == 128) hipLaunchKernelGGL((kv4_attn_kernel<128>), g, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((kv4_attn_kernel<64>), g, dim3(256), 0, s, a);
  return hipGetLastError() == hipSuccess ? WGKV_OK : WGKV_ERR_HIP;
}
