// Argument blocks, launchers and device helpers of the 4-bit latent cache (int4_*.cu).
#pragma once

#include "common.cuh"

namespace rolaq {
namespace i4 {

constexpr int kPage = 64;    // tokens of a page
constexpr int kGroup = 128;  // elements that share a scale and a zero
constexpr float kTop = 15.f;

// The scratch: a header of counters that are zero between calls, the decode's partials, and at its
// end the page scores of a selection.
constexpr int64_t kHeaderBytes = 65536;

struct DecodeArgs {
  const uint16_t* q;
  int64_t q_sb, q_st, q_sh;
  int32_t batch, q_len, heads;
  rolaq_int4_cache cache;
  const int32_t* page_table;
  int64_t pt_stride;
  int32_t max_pages;
  const int32_t* seq_lens;
  float sm_scale;
  void* workspace;
  uint16_t* out;
  int64_t o_sb, o_st, o_sh;
  float* lse;
  int32_t* err;
};

struct SelectArgs {
  const uint16_t* q;
  int64_t q_sb, q_sh;
  int32_t batch, heads;
  rolaq_int4_cache cache;
  const int32_t* page_table;
  int64_t pt_stride;
  int32_t max_pages;
  const int32_t* seq_lens;
  int32_t budget, keep_first, keep_last;
  float* scores;      // [batch, max_pages]
  int32_t* counters;  // the scratch's header
  int32_t* sel_table;
  int64_t sel_stride;
  int32_t* sel_lens;
  int32_t* err;
};

int launch_write(const void* c, bool f32, int64_t ld_c, const uint16_t* k_pe, int64_t ld_pe, const void* slots,
                 int slots64, int64_t n, const rolaq_int4_cache& cache, int32_t* err, cudaStream_t s);
int launch_read(const rolaq_int4_cache& cache, const void* slots, int slots64, int64_t n, void* out, bool f32,
                int64_t ld_out, uint16_t* out_pe, int64_t ld_pe, int32_t* err, cudaStream_t s);
int launch_update_boxes(const rolaq_int4_cache& cache, const int32_t* pages, const int32_t* counts, int64_t n,
                        int32_t* err, cudaStream_t s);
int launch_read_boxes(const rolaq_int4_cache& cache, const int32_t* pages, int64_t n, float* lo, float* hi, int64_t ld,
                      int32_t* err, cudaStream_t s);
int64_t decode_workspace(int batch, int q_len, int heads, int d);
int launch_decode(const DecodeArgs& a, cudaStream_t s);
int64_t select_workspace(int batch, int max_pages);
int launch_select(const SelectArgs& a, cudaStream_t s);

// The least e >= -100 with top <= 127 * 2^e; 0 for top = 0 (and for a top that is no number).
__device__ __forceinline__ int unit_exponent(float top) {
  if (!(top > 0.f)) return 0;
  top = fminf(top, 3.402823466e38f);
  int x;
  const float m = frexpf(top, &x);  // top = m * 2^x with m in [1/2, 1)
  return max(m > 127.f / 128.f ? x - 6 : x - 7, -100);
}
// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// The value a code stands for, as the plain form rounds it: one subtraction, one product.
__device__ __forceinline__ float value(uint32_t code, float scale, float zero) {
  return __fmul_rn(__fsub_rn(static_cast<float>(code), zero), scale);
}

}  // namespace i4
}  // namespace rolaq
