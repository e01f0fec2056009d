// The 4-bit latent cache's memory-bound kernels: quantising rows as they are written, reading rows
// back, and the page boxes.
//
// Codec (the uniform min/max codec of mla_quant/oscar.py:91-101 with 16 levels): per 128 elements
// scale = (hi - lo) / 15, code = round((x - lo) / scale), zero = -lo / scale, value = (code - zero) scale.
#include <algorithm>
#include <type_traits>

#include "int4.cuh"

namespace rolaq {
namespace i4 {
namespace {

// Every fourth 8 of 128 elements of a row as FP32.
__device__ __forceinline__ void load32(const float* p, float (&x)[32]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float4 v = reinterpret_cast<const float4*>(p)[8 * (i / 2) + i % 2];
    x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
  }
}
__device__ __forceinline__ void load32(const uint16_t* p, float (&x)[32]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint4 v = reinterpret_cast<const uint4*>(p)[4 * i];
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) x[8 * i + 2 * k] = bf16_lo(w[k]), x[8 * i + 2 * k + 1] = bf16_hi(w[k]);
  }
}

// The least and greatest of three, NaN where one is.
__device__ __forceinline__ float min3_nan(float a, float b, float c) {
  float d;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Four threads per 128-element group of a row, min and max over the four by shuffles; the last blocks copy k_pe.  A thread
// loads words of 8 elements 4 apart (whole sectors a load) and changes its words of codes with the other three, so that
// it stores 16 bytes in a row.
// Divisions: with y = 1 / b rounded and q within one unit of a / b's last place, the residual a - b q is exact and
// q + (a - b q) y rounds to the rounded quotient (Markstein, IBM J. Res. Dev. 34, 1990); the first such step brings the
// product a y, which is within 1.5 units, within one, the second to the quotient.  All is far from the ends of the range:
// 6e-10 < scale < 3e37.  That is without branches, where a check of the product for nearness to a half and a division then
// met the many exact halves of BF16 rows (62 us against 55).
// Measured: 131072 rows of 512 + 64 in BF16 (206 MB) 54 us, 3.8 TB/s, in FP32 (340 MB) 61 us, 5.6
// TB/s; in BF16 bound by instructions (61% of the issue slots) and their latency at 32 warps; 76 with a thread's elements side by side and k_pe among the groups.
template <typename T, int NG>
__global__ void __launch_bounds__(256, 4) write_kernel(const T* __restrict__ c, int64_t ld_c,
                                                       const uint16_t* __restrict__ k_pe, int64_t ld_pe, const void* slots,
                                                       int slots64, int64_t n, unsigned group_blocks, rolaq_int4_cache cache,
                                                       int32_t* err) {
  if (blockIdx.x >= group_blocks) {
    const uint32_t unit = (blockIdx.x - group_blocks) * 256u + threadIdx.x, chunks = cache.rope_dim / 8;
    const int64_t row = unit / chunks;
    const int col = 8 * (unit % chunks);
    if (row >= n) return;
    const int64_t slot = load_index(slots, slots64, row);
    if (slot >= 0 && slot < cache.num_slots)
      *reinterpret_cast<uint4*>(cache.rope + slot * cache.rope_dim + col) = *reinterpret_cast<const uint4*>(k_pe + row * ld_pe + col);
    else if (col == 0)
      report(err, ROLAQ_DEV_BAD_SLOT);
    return;
  }
  const uint32_t unit = (blockIdx.x * 256u + threadIdx.x) / 4;
  const int part = threadIdx.x & 3;
  const int64_t row = unit / NG;
  const int g = unit % NG;
  if (row >= n) return;  // whole groups of four threads leave together
  const int64_t slot = load_index(slots, slots64, row);
  float x[32];  // on its way together with the slot
  load32(c + row * ld_c + g * kGroup + part * 8, x);
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 0; i < 32; i += 2) lo = min3_nan(lo, x[i], x[i + 1]), hi = max3_nan(hi, x[i], x[i + 1]);
  const uint32_t lanes = 0xFu << (threadIdx.x & 28);
#pragma unroll
  for (int o = 1; o < 4; o *= 2) {
    const float l = __shfl_xor_sync(lanes, lo, o), h = __shfl_xor_sync(lanes, hi, o);
    lo = min3_nan(lo, lo, l);
    hi = max3_nan(hi, hi, h);
  }
  const float range = __fsub_rn(hi, lo);
  float scale = fabsf(range) <= 1e-8f ? 1.f : __fdiv_rn(range, kTop);
  const float inv = __frcp_rn(scale);
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {  // a word of 8 codes
    float code[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = __fsub_rn(x[8 * k + i], lo);
      float q = __fmul_rn(d, inv);
      q = __fmaf_rn(__fmaf_rn(-q, scale, d), inv, q);
      q = __fmaf_rn(__fmaf_rn(-q, scale, d), inv, q);
      code[i] = __fsub_rn(__fadd_rn(q, 12582912.f), 12582912.f);  // the nearest whole number, halves to even
    }
    float half[2];  // four codes as one whole number below 2^16 (0 <= code <= 15: lo and hi are the group's own)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      half[h] = fmaf(fmaf(fmaf(code[4 * h + 3], 16.f, code[4 * h + 2]), 16.f, code[4 * h + 1]), 16.f, code[4 * h]);
    // under 2^23 a whole number is the float's low bits
    w[k] = (__float_as_uint(half[0] + 8388608.f) & 0xFFFFu) | __float_as_uint(half[1] + 8388608.f) << 16;
  }
  // words part + 4 i to words 4 part + i: a transpose among the four
#pragma unroll
  for (int o = 1; o < 4; o *= 2) {
    const bool up = part & o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i & o) continue;
      const uint32_t got = __shfl_xor_sync(lanes, up ? w[i] : w[i | o], o);
      if (up) w[i] = got;
      else w[i | o] = got;
    }
  }
  if (!(range < INFINITY)) scale = __int_as_float(0x7FC00000);  // as soon as an element is no finite number
  if (slot < 0 || slot >= cache.num_slots) return;  // reported with its k_pe
  *reinterpret_cast<uint4*>(cache.codes + slot * (NG * 64) + g * 64 + part * 16) = make_uint4(w[0], w[1], w[2], w[3]);
  if (part == 0) reinterpret_cast<float2*>(cache.params)[slot * NG + g] = make_float2(scale, __fdiv_rn(-lo, scale));
}

__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(uint16_t* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

// Eight threads per unit, a unit being a group of a row or its k_pe, and two rows a thread, `apart` rows from each other, so that
// twice as much is under way: a thread reads the words of 8 elements at 8 part and at 64 + 8 part of its group, so
// that a warp's stores are whole lines.  Bound by memory: the rows above back in BF16 41 us, 5.0 TB/s, in FP32 67 us, 5.1 TB/s.
template <typename T, int NG>
__global__ void __launch_bounds__(256) read_kernel(rolaq_int4_cache cache, const void* slots, int slots64, int64_t n,
                                                   int64_t apart, T* __restrict__ out, int64_t ld_out,
                                                   uint16_t* __restrict__ out_pe, int64_t ld_pe, int32_t* err) {
  const uint32_t unit = (blockIdx.x * 256u + threadIdx.x) / 8;
  const int part = threadIdx.x & 7;
  const int g = unit % (NG + 1);
  if (unit / (NG + 1) >= apart) return;
  int64_t row[2], slot[2];
  bool ok[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    row[i] = unit / (NG + 1) + i * apart;
    slot[i] = row[i] < n ? load_index(slots, slots64, row[i]) : 0;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    ok[i] = row[i] < n && slot[i] >= 0 && slot[i] < cache.num_slots;
    if (row[i] < n && !ok[i] && g == 0 && part == 0) report(err, ROLAQ_DEV_BAD_SLOT);
  }
  if (g == NG) {
    if (out_pe == nullptr || part * 8 >= cache.rope_dim) return;
    uint4 v[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      v[i] = ok[i] ? *reinterpret_cast<const uint4*>(cache.rope + slot[i] * cache.rope_dim + part * 8) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (row[i] < n) *reinterpret_cast<uint4*>(out_pe + row[i] * ld_pe + part * 8) = v[i];
    return;
  }
  uint32_t w[2][2];
  float2 p[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (!ok[i]) continue;
    const uint32_t* src = reinterpret_cast<const uint32_t*>(cache.codes + slot[i] * (NG * 64) + g * 64) + part;
    w[i][0] = src[0], w[i][1] = src[8];
    p[i] = reinterpret_cast<const float2*>(cache.params)[slot[i] * NG + g];
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (row[i] < n) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = ok[i] ? value((w[i][h] >> (4 * k)) & 15u, p[i].x, p[i].y) : 0.f;
        store8(out + row[i] * ld_out + g * kGroup + 64 * h + 8 * part, v);
      }
    }
}

// The least and greatest of three; a NaN is passed over.
__device__ __forceinline__ float min3(float a, float b, float c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Two BF16 columns at a time; a NaN is passed over.
__device__ __forceinline__ uint32_t min_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("min.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Two tokens' words of 8 codes each widen the minima and maxima of the columns, in 32-bit steps that are value()'s: codes
// become floats by one OR under 2^23 (their place in the word a power of 16) and one exact FMA.
__device__ __forceinline__ void widen(const uint32_t (&w)[2], const float2 (&p)[2], float (&lo)[8], float (&hi)[8]) {
  const uint32_t high[2] = {w[0] >> 12, w[1] >> 12};  // codes 5, 6 and 7 at places 2, 3 and 4
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int place = i < 5 ? i : i - 3;
    const float at = 1.f / static_cast<float>(1 << (4 * place));
    float v[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float code = fmaf(__uint_as_float(((i < 5 ? w[k] : high[k]) & (15u << (4 * place))) | 0x4B000000u), at, -8388608.f * at);
      v[k] = __fmul_rn(__fsub_rn(code, p[k].y), p[k].x);
    }
    lo[i] = min3(lo[i], v[0], v[1]);
    hi[i] = max3(hi[i], v[0], v[1]);
  }
}

// One CTA per page: a thread takes a word (8 columns) of every (512 * 8 / W)-th token, the CTA joins them through
// shared memory.  The operations on an element bound it (the logic pipe, which the minima and maxima need, is 58% full),
// not memory: 2048 whole pages of 512 + 64 (57 MB) 30 us, 1.9 TB/s; 37 with addresses for pages that may end early, and
// with a token a step and the rotary part in FP32.
template <int D, int DR>
__global__ void __launch_bounds__(256, 4) boxes_kernel(rolaq_int4_cache cache, const int32_t* __restrict__ pages,
                                                    const int32_t* __restrict__ counts, int32_t* err) {
  constexpr int W = D + DR, NG = D / kGroup, WORDS = D / 8, SHARES = 256 / WORDS, EACH = kPage / SHARES;
  constexpr int RWORDS = DR / 8, RSHARES = 256 / RWORDS, REACH = kPage / RSHARES;  // the rotary part: 8 columns of 16 bits
  __shared__ __align__(16) float box[2][SHARES][D], rope_box[2][8][DR];  // low and high; the rotary part by warps
  __shared__ float tops[2][8];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
  const int64_t page = pages[blockIdx.x];
  const int count = counts[blockIdx.x];
  if (page < 0 || page >= cache.num_slots / kPage || count < 1 || count > kPage) {
    if (tid == 0) report(err, ROLAQ_DEV_BAD_PAGE);
    return;
  }
  {
    const int word = tid % WORDS, share = tid / WORDS;
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(cache.codes) + (page * kPage + share) * WORDS + word;
    const float2* params = reinterpret_cast<const float2*>(cache.params) + (page * kPage + share) * NG + word / 16;
    float lo[8], hi[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] = INFINITY, hi[i] = -INFINITY;
    constexpr int AT_ONCE = EACH < 8 ? EACH : 8;
    // Tokens past the count are the share's first one again (or, where that is past it too, nothing).
    auto walk = [&](auto whole) {
#pragma unroll 1
      for (int k0 = 0; k0 < EACH; k0 += AT_ONCE) {
        uint32_t w[AT_ONCE / 2][2];
        float2 p[AT_ONCE / 2][2];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
          const int at = whole || share + (k0 + k) * SHARES < count ? k0 + k : 0;
          w[k / 2][k % 2] = codes[at * SHARES * WORDS], p[k / 2][k % 2] = params[at * SHARES * NG];
        }
#pragma unroll
        for (int k = 0; k < AT_ONCE / 2; ++k) widen(w[k], p[k], lo, hi);
      }
    };
    if (count == kPage) walk(std::true_type());
    else if (share < count) walk(std::false_type());
    store8(&box[0][share][8 * word], lo);
    store8(&box[1][share][8 * word], hi);
  }
  {
    const int word = tid % RWORDS, share = tid / RWORDS;
    uint32_t lo[4], hi[4];  // two columns each
#pragma unroll
    for (int i = 0; i < 4; ++i) lo[i] = 0x7F807F80u, hi[i] = 0xFF80FF80u;
#pragma unroll
    for (int k = 0; k < REACH; ++k) {
      const int t = share + k * RSHARES;
      if (t >= count) continue;
      const uint4 v = *reinterpret_cast<const uint4*>(cache.rope + (page * kPage + t) * DR + 8 * word);
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) lo[i] = min_bf16x2(lo[i], u[i]), hi[i] = max_bf16x2(hi[i], u[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // over the warp's tokens
#pragma unroll
      for (int o = RWORDS; o < 32; o *= 2) {
        lo[i] = min_bf16x2(lo[i], __shfl_xor_sync(0xFFFFFFFFu, lo[i], o));
        hi[i] = max_bf16x2(hi[i], __shfl_xor_sync(0xFFFFFFFFu, hi[i], o));
      }
      if (lane < RWORDS) {
        *reinterpret_cast<float2*>(&rope_box[0][warp][8 * word + 2 * i]) = make_float2(bf16_lo(lo[i]), bf16_hi(lo[i]));
        *reinterpret_cast<float2*>(&rope_box[1][warp][8 * word + 2 * i]) = make_float2(bf16_lo(hi[i]), bf16_hi(hi[i]));
      }
    }
  }
  __syncthreads();
  constexpr int COLS = (W + 255) / 256;
  float lo[COLS], hi[COLS], top[2] = {0.f, 0.f};
#pragma unroll
  for (int k = 0; k < COLS; ++k) {
    const int col = tid + 256 * k;
    lo[k] = INFINITY;
    hi[k] = -INFINITY;
    if (col < D) {
#pragma unroll
      for (int s = 0; s < SHARES; ++s) lo[k] = fminf(lo[k], box[0][s][col]), hi[k] = fmaxf(hi[k], box[1][s][col]);
    } else if (col < W) {
#pragma unroll
      for (int s = 0; s < 8; ++s) lo[k] = fminf(lo[k], rope_box[0][s][col - D]), hi[k] = fmaxf(hi[k], rope_box[1][s][col - D]);
    } else {
      continue;
    }
    // no number among the tokens, or an infinity: no box (0 -+ 0), no part in the unit
    if (!(fabsf(lo[k]) < INFINITY && fabsf(hi[k]) < INFINITY)) lo[k] = hi[k] = 0.f;
    top[col >= D] = fmaxf(top[col >= D], fmaxf(fabsf(lo[k]), fabsf(hi[k])));
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    top[i] = warp_max_f32(top[i]);
    if (lane == 0) tops[i][warp] = top[i];
  }
  __syncthreads();
  int e[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float m = 0.f;
    for (int k = 0; k < 8; ++k) m = fmaxf(m, tops[i][k]);
    e[i] = unit_exponent(m);
    if (tid == 0) cache.box_exps[page * 2 + i] = e[i];
  }
#pragma unroll
  for (int k = 0; k < COLS; ++k) {
    const int col = tid + 256 * k;
    if (col >= W) continue;
    const float inv = pow2(-e[col >= D]);
    const float a = __fmul_rn(lo[k], inv), b = __fmul_rn(hi[k], inv);  // in units, at most 127: their sum cannot overflow
    const float center = rintf(__fmul_rn(__fadd_rn(a, b), 0.5f));
    const float radius = ceilf(fmaxf(__fsub_rn(b, center), __fsub_rn(center, a)));
    cache.box_center[page * W + col] = static_cast<int8_t>(static_cast<int>(fminf(fmaxf(center, -127.f), 127.f)));
    cache.box_radius[page * W + col] = static_cast<uint8_t>(static_cast<int>(fminf(fmaxf(radius, 0.f), 255.f)));
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
  const int ng = cache.latent_dim / kGroup;
  // 32 bits of units a launch
  const int64_t most = (int64_t(1) << 31) / (4 * (ng + 1)) / 256 * 256;
  for (int64_t at = 0; at < n; at += most) {
    const int64_t rows = std::min(n - at, most);
    const unsigned groups = blocks_for(rows * ng * 4, 256), grid = groups + blocks_for(rows * (cache.rope_dim / 8), 256);
    const void* sl = static_cast<const char*>(slots) + at * (slots64 ? 8 : 4);
    auto go = [&](auto kernel, auto* src) {
      kernel<<<grid, 256, 0, s>>>(src + at * ld_c, ld_c, k_pe + at * ld_pe, ld_pe, sl, slots64, rows, groups, cache, err);
    };
    if (f32 && ng == 4) go(write_kernel<float, 4>, static_cast<const float*>(c));
    else if (f32) go(write_kernel<float, 2>, static_cast<const float*>(c));
    else if (ng == 4) go(write_kernel<uint16_t, 4>, static_cast<const uint16_t*>(c));
    else go(write_kernel<uint16_t, 2>, static_cast<const uint16_t*>(c));
  }
  return status();
}

int launch_read(const rolaq_int4_cache& cache, const void* slots, int slots64, int64_t n, void* out, bool f32,
                int64_t ld_out, uint16_t* out_pe, int64_t ld_pe, int32_t* err, cudaStream_t s) {
  const int ng = cache.latent_dim / kGroup;
  const int64_t most = (int64_t(1) << 31) / (8 * (ng + 1)) / 256 * 256;
  for (int64_t at = 0; at < n; at += most) {
    const int64_t rows = std::min(n - at, most);
    const int64_t apart = (rows + 1) / 2;
    const unsigned grid = blocks_for(apart * (ng + 1) * 8, 256);
    const void* sl = static_cast<const char*>(slots) + at * (slots64 ? 8 : 4);
    uint16_t* pe = out_pe ? out_pe + at * ld_pe : nullptr;
    auto go = [&](auto kernel, auto* dst) {
      kernel<<<grid, 256, 0, s>>>(cache, sl, slots64, rows, apart, dst + at * ld_out, ld_out, pe, ld_pe, err);
    };
    if (f32 && ng == 4) go(read_kernel<float, 4>, static_cast<float*>(out));
    else if (f32) go(read_kernel<float, 2>, static_cast<float*>(out));
    else if (ng == 4) go(read_kernel<uint16_t, 4>, static_cast<uint16_t*>(out));
    else go(read_kernel<uint16_t, 2>, static_cast<uint16_t*>(out));
  }
  return status();
}

int launch_update_boxes(const rolaq_int4_cache& cache, const int32_t* pages, const int32_t* counts, int64_t n,
                        int32_t* err, cudaStream_t s) {
  const auto kernel = cache.latent_dim == 512 ? (cache.rope_dim == 64 ? boxes_kernel<512, 64> : boxes_kernel<512, 32>)
                                              : (cache.rope_dim == 64 ? boxes_kernel<256, 64> : boxes_kernel<256, 32>);
  kernel<<<static_cast<unsigned>(n), 256, 0, s>>>(cache, pages, counts, err);
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
