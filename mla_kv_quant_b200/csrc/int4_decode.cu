// Absorbed attention over the 4-bit latent cache.
//
// One CTA per query row (query token and head) and request; its warps take the request's tokens in
// turn.  A lane holds D/32 latent columns (one group's) and Dr/32 rotary ones; the running maximum
// and sum of the softmax stay in registers, the warps' results are joined at the end.
#include "int4.cuh"

namespace rolaq {
namespace i4 {
namespace {

constexpr int kWarps = 8;

template <int D, int DR>
__global__ void __launch_bounds__(kWarps * 32) decode_kernel(DecodeArgs a) {
  constexpr int E = D / 32, R = DR / 32;  // columns of a lane: E * lane .. and D + R * lane ..
  __shared__ float part_o[kWarps][D], part_m[kWarps], part_l[kWarps];
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int t = blockIdx.x / a.heads, h = blockIdx.x % a.heads, b = blockIdx.y;
  int len = a.seq_lens[b];
  if (len > a.max_pages * kPage) {
    if (threadIdx.x == 0) report(a.err, ROLAQ_DEV_BAD_REQ);
    len = a.max_pages * kPage;
  }
  const int seen = len - a.q_len + t + 1;
  const uint16_t* qrow = a.q + b * a.q_sb + t * a.q_st + h * a.q_sh;
  float q[E], q_pe[R], o[E] = {};
#pragma unroll
  for (int i = 0; i < E; ++i) q[i] = bf16_lo(qrow[E * lane + i]);
#pragma unroll
  for (int i = 0; i < R; ++i) q_pe[i] = bf16_lo(qrow[D + R * lane + i]);
  float m = -INFINITY, l = 0.f;
  for (int tok = warp; tok < seen; tok += kWarps) {
    const int64_t page = a.page_table[b * a.pt_stride + tok / kPage];
    if (page < 0 || page >= a.cache.num_slots / kPage) {
      if (lane == 0) report(a.err, ROLAQ_DEV_BAD_PAGE);
      continue;
    }
    const int64_t slot = page * kPage + tok % kPage;
    const float2 p = reinterpret_cast<const float2*>(a.cache.params)[slot * (D / kGroup) + lane * E / kGroup];
    float v[E], s = 0.f;
#pragma unroll
    for (int k = 0; k < E / 8; ++k) {
      const uint32_t w = reinterpret_cast<const uint32_t*>(a.cache.codes)[slot * (D / 8) + lane * (E / 8) + k];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[8 * k + i] = value((w >> (4 * i)) & 15u, p.x, p.y);
        s += q[8 * k + i] * v[8 * k + i];
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) s += q_pe[i] * bf16_lo(a.cache.rope[slot * DR + R * lane + i]);
#pragma unroll
    for (int k = 16; k >= 1; k /= 2) s += __shfl_xor_sync(0xFFFFFFFFu, s, k);
    s *= a.sm_scale;
    const float m_new = fmaxf(m, s);
    const float keep = m == -INFINITY ? 0.f : expf(m - m_new), e = expf(s - m_new);
    l = l * keep + e;
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = o[i] * keep + e * v[i];
    m = m_new;
  }
#pragma unroll
  for (int i = 0; i < E; ++i) part_o[warp][E * lane + i] = o[i];
  if (lane == 0) part_m[warp] = m, part_l[warp] = l;
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
  for (int k = 0; k < kWarps; ++k) top = fmaxf(top, part_m[k]);
  float share[kWarps];
#pragma unroll
  for (int k = 0; k < kWarps; ++k) {
    share[k] = part_m[k] == -INFINITY ? 0.f : expf(part_m[k] - top);
    sum += share[k] * part_l[k];
  }
  uint16_t* out = a.out + b * a.o_sb + t * a.o_st + h * a.o_sh;
  for (int c = threadIdx.x; c < D; c += kWarps * 32) {
    float x = 0.f;
    for (int k = 0; k < kWarps; ++k) x += share[k] * part_o[k][c];
    out[c] = __bfloat16_as_ushort(__float2bfloat16_rn(sum == 0.f ? 0.f : x / sum));
  }
  if (threadIdx.x == 0 && a.lse)
    a.lse[(static_cast<int64_t>(b) * a.q_len + t) * a.heads + h] = sum == 0.f ? -INFINITY : top + logf(sum);
}

}  // namespace

int64_t decode_workspace(int batch, int q_len, int heads, int d) { return kHeaderBytes; }

int launch_decode(const DecodeArgs& a, cudaStream_t s) {
  const dim3 grid(a.q_len * a.heads, a.batch);
  if (a.cache.latent_dim == 512 && a.cache.rope_dim == 64)
    decode_kernel<512, 64><<<grid, kWarps * 32, 0, s>>>(a);
  else if (a.cache.latent_dim == 512)
    decode_kernel<512, 32><<<grid, kWarps * 32, 0, s>>>(a);
  else if (a.cache.rope_dim == 64)
    decode_kernel<256, 64><<<grid, kWarps * 32, 0, s>>>(a);
  else
    decode_kernel<256, 32><<<grid, kWarps * 32, 0, s>>>(a);
  return cudaGetLastError() == cudaSuccess ? ROLAQ_OK : ROLAQ_ECUDA;
}

}  // namespace i4
}  // namespace rolaq
