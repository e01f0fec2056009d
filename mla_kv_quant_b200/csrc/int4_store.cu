// The 4-bit latent cache's memory-bound kernels: quantising rows as they are written, reading rows
// back, and the page boxes.
//
// Codec (the uniform min/max codec of mla_quant/oscar.py:91-101 with 16 levels): per 128 elements
// scale = (hi - lo) / 15, code = round((x - lo) / scale), zero = -lo / scale, value = (code - zero) scale.
#include "int4.cuh"

namespace rolaq {
namespace i4 {
namespace {

// 16 consecutive elements of a row as FP32.
__device__ __forceinline__ void load16(const float* p, float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 v = reinterpret_cast<const float4*>(p)[i];
    x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
  }
}
__device__ __forceinline__ void load16(const uint16_t* p, float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint4 v = reinterpret_cast<const uint4*>(p)[i];
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) x[8 * i + 2 * k] = bf16_lo(w[k]), x[8 * i + 2 * k + 1] = bf16_hi(w[k]);
  }
}

// Eight threads per unit: a unit is one 128-element group of a row (16 elements a thread, min and max
// over the eight by shuffles) or the row's k_pe.
template <typename T>
__global__ void write_kernel(const T* __restrict__ c, int64_t ld_c, const uint16_t* __restrict__ k_pe, int64_t ld_pe,
                             const void* slots, int slots64, int64_t n, rolaq_int4_cache cache, int32_t* err) {
  const int ng = cache.latent_dim / kGroup;
  const int64_t unit = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / 8;
  const int part = threadIdx.x & 7;
  const int64_t row = unit / (ng + 1);
  const int g = static_cast<int>(unit % (ng + 1));
  if (row >= n) return;  // whole groups of eight threads leave together
  const int64_t slot = load_index(slots, slots64, row);
  if (slot < 0 || slot >= cache.num_slots) {
    if (part == 0) report(err, ROLAQ_DEV_BAD_SLOT);
    return;
  }
  if (g == ng) {
    if (part * 8 < cache.rope_dim)
      *reinterpret_cast<uint4*>(cache.rope + slot * cache.rope_dim + part * 8) =
          *reinterpret_cast<const uint4*>(k_pe + row * ld_pe + part * 8);
    return;
  }
  float x[16];
  load16(c + row * ld_c + g * kGroup + part * 16, x);
  float lo = x[0], hi = x[0], bad = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    bad += x[i] * 0.f;  // NaN as soon as one element is no finite number
  }
  const uint32_t lanes = 0xFFu << (threadIdx.x & 24);
#pragma unroll
  for (int o = 1; o < 8; o *= 2) {
    lo = fminf(lo, __shfl_xor_sync(lanes, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(lanes, hi, o));
    bad += __shfl_xor_sync(lanes, bad, o);
  }
  const float range = __fsub_rn(hi, lo);
  float scale = fabsf(range) <= 1e-8f ? 1.f : __fdiv_rn(range, kTop);
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float code = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[i], lo), scale)), 0.f), kTop);
    w[i / 8] |= static_cast<uint32_t>(code) << (4 * (i % 8));
  }
  if (bad != 0.f) scale = __int_as_float(0x7FC00000);
  *reinterpret_cast<uint2*>(cache.codes + slot * (cache.latent_dim / 2) + g * 64 + part * 8) = make_uint2(w[0], w[1]);
  if (part == 0) reinterpret_cast<float2*>(cache.params)[slot * ng + g] = make_float2(scale, __fdiv_rn(-lo, scale));
}

__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(uint16_t* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

// One thread per 8 elements of a row (a word of codes), and per 8 elements of its rotary part.
template <typename T>
__global__ void read_kernel(rolaq_int4_cache cache, const void* slots, int slots64, int64_t n, T* __restrict__ out,
                            int64_t ld_out, uint16_t* __restrict__ out_pe, int64_t ld_pe, int32_t* err) {
  const int words = cache.latent_dim / 8, all = words + (out_pe ? cache.rope_dim / 8 : 0);
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t row = unit / all;
  const int k = static_cast<int>(unit % all);
  if (row >= n) return;
  const int64_t slot = load_index(slots, slots64, row);
  const bool ok = slot >= 0 && slot < cache.num_slots;
  if (!ok && k == 0) report(err, ROLAQ_DEV_BAD_SLOT);
  if (k >= words) {
    const int j = 8 * (k - words);
    *reinterpret_cast<uint4*>(out_pe + row * ld_pe + j) =
        ok ? *reinterpret_cast<const uint4*>(cache.rope + slot * cache.rope_dim + j) : make_uint4(0, 0, 0, 0);
    return;
  }
  float v[8] = {};
  if (ok) {
    const uint32_t w = reinterpret_cast<const uint32_t*>(cache.codes)[slot * words + k];
    const float2 p = reinterpret_cast<const float2*>(cache.params)[slot * (cache.latent_dim / kGroup) + k / 16];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = value((w >> (4 * i)) & 15u, p.x, p.y);
  }
  store8(out + row * ld_out + 8 * k, v);
}

// One CTA per page, a column at a time per thread.
__global__ void boxes_kernel(rolaq_int4_cache cache, const int32_t* __restrict__ pages,
                             const int32_t* __restrict__ counts, int32_t* err) {
  __shared__ float tops[2][32];
  const int d = cache.latent_dim, w = d + cache.rope_dim, ng = d / kGroup;
  const int64_t page = pages[blockIdx.x];
  const int count = counts[blockIdx.x];
  if (page < 0 || page >= cache.num_slots / kPage || count < 1 || count > kPage) {
    if (threadIdx.x == 0) report(err, ROLAQ_DEV_BAD_PAGE);
    return;
  }
  float lo[3], hi[3], top[2] = {0.f, 0.f};
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const int col = threadIdx.x + 256 * k;
    lo[k] = INFINITY;
    hi[k] = -INFINITY;
    if (col >= w) continue;
    for (int t = 0; t < count; ++t) {
      const int64_t slot = page * kPage + t;
      float v;
      if (col < d) {
        const float2 p = reinterpret_cast<const float2*>(cache.params)[slot * ng + col / kGroup];
        v = value((cache.codes[slot * (d / 2) + col / 2] >> (4 * (col & 1))) & 15u, p.x, p.y);
      } else {
        v = bf16_lo(cache.rope[slot * cache.rope_dim + col - d]);
      }
      lo[k] = fminf(lo[k], v);
      hi[k] = fmaxf(hi[k], v);
    }
    top[col >= d] = fmaxf(top[col >= d], fmaxf(fabsf(lo[k]), fabsf(hi[k])));
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    top[i] = warp_max_f32(top[i]);
    if ((threadIdx.x & 31) == 0) tops[i][threadIdx.x / 32] = top[i];
  }
  __syncthreads();
  int e[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float m = 0.f;
    for (int k = 0; k < 8; ++k) m = fmaxf(m, tops[i][k]);
    e[i] = unit_exponent(m);
    if (threadIdx.x == 0) cache.box_exps[page * 2 + i] = e[i];
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const int col = threadIdx.x + 256 * k;
    if (col >= w) continue;
    const float inv = pow2(-e[col >= d]);
    const float center = rintf(__fmul_rn(__fmul_rn(__fadd_rn(lo[k], hi[k]), 0.5f), inv));
    const float radius = ceilf(fmaxf(__fsub_rn(__fmul_rn(hi[k], inv), center), __fsub_rn(center, __fmul_rn(lo[k], inv))));
    cache.box_center[page * w + col] = static_cast<int8_t>(static_cast<int>(fminf(fmaxf(center, -127.f), 127.f)));
    cache.box_radius[page * w + col] = static_cast<uint8_t>(static_cast<int>(fminf(fmaxf(radius, 0.f), 255.f)));
  }
}

__global__ void read_boxes_kernel(rolaq_int4_cache cache, const int32_t* __restrict__ pages, int64_t n,
                                  float* __restrict__ lo, float* __restrict__ hi, int64_t ld, int32_t* err) {
  const int d = cache.latent_dim, w = d + cache.rope_dim;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t i = unit / (w / 4);
  const int col = static_cast<int>(unit % (w / 4)) * 4;
  if (i >= n) return;
  const int64_t page = pages[i];
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
  if (page >= 0 && page < cache.num_slots / kPage) {
    const float unit_size = pow2(cache.box_exps[page * 2 + (col >= d)]);
    const char4 c = *reinterpret_cast<const char4*>(cache.box_center + page * w + col);
    const uchar4 r = *reinterpret_cast<const uchar4*>(cache.box_radius + page * w + col);
    a = make_float4((c.x - r.x) * unit_size, (c.y - r.y) * unit_size, (c.z - r.z) * unit_size, (c.w - r.w) * unit_size);
    b = make_float4((c.x + r.x) * unit_size, (c.y + r.y) * unit_size, (c.z + r.z) * unit_size, (c.w + r.w) * unit_size);
  } else if (col == 0) {
    report(err, ROLAQ_DEV_BAD_PAGE);
  }
  *reinterpret_cast<float4*>(lo + i * ld + col) = a;
  *reinterpret_cast<float4*>(hi + i * ld + col) = b;
}

unsigned blocks_for(int64_t threads_wanted, int threads) {
  return static_cast<unsigned>((threads_wanted + threads - 1) / threads);
}

int status() { return cudaGetLastError() == cudaSuccess ? ROLAQ_OK : ROLAQ_ECUDA; }

}  // namespace

int launch_write(const void* c, bool f32, int64_t ld_c, const uint16_t* k_pe, int64_t ld_pe, const void* slots,
                 int slots64, int64_t n, const rolaq_int4_cache& cache, int32_t* err, cudaStream_t s) {
  const unsigned grid = blocks_for(n * (cache.latent_dim / kGroup + 1) * 8, 256);
  if (f32)
    write_kernel<<<grid, 256, 0, s>>>(static_cast<const float*>(c), ld_c, k_pe, ld_pe, slots, slots64, n, cache, err);
  else
    write_kernel<<<grid, 256, 0, s>>>(static_cast<const uint16_t*>(c), ld_c, k_pe, ld_pe, slots, slots64, n, cache, err);
  return status();
}

int launch_read(const rolaq_int4_cache& cache, const void* slots, int slots64, int64_t n, void* out, bool f32,
                int64_t ld_out, uint16_t* out_pe, int64_t ld_pe, int32_t* err, cudaStream_t s) {
  const unsigned grid = blocks_for(n * (cache.latent_dim / 8 + (out_pe ? cache.rope_dim / 8 : 0)), 256);
  if (f32)
    read_kernel<<<grid, 256, 0, s>>>(cache, slots, slots64, n, static_cast<float*>(out), ld_out, out_pe, ld_pe, err);
  else
    read_kernel<<<grid, 256, 0, s>>>(cache, slots, slots64, n, static_cast<uint16_t*>(out), ld_out, out_pe, ld_pe, err);
  return status();
}

int launch_update_boxes(const rolaq_int4_cache& cache, const int32_t* pages, const int32_t* counts, int64_t n,
                        int32_t* err, cudaStream_t s) {
  boxes_kernel<<<static_cast<unsigned>(n), 256, 0, s>>>(cache, pages, counts, err);
  return status();
}

int launch_read_boxes(const rolaq_int4_cache& cache, const int32_t* pages, int64_t n, float* lo, float* hi, int64_t ld,
                      int32_t* err, cudaStream_t s) {
  read_boxes_kernel<<<blocks_for(n * (cache.latent_dim + cache.rope_dim) / 4, 256), 256, 0, s>>>(cache, pages, n, lo,
                                                                                              hi, ld, err);
  return status();
}

}  // namespace i4
}  // namespace rolaq
