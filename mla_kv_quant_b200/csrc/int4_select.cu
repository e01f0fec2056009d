// Page selection: scores of the pages of a request against its query, and the pages that are kept.
//
// score(page) = max over the heads of sum over both parts of 2^(e_q + e_page) (sum q8 center + sum |q8| radius).
// The sums are whole numbers below 2^24 (127 * 127 * 512 for the centers, 127 * 128 * 512 for the radii),
// so their order does not matter; each part is one conversion and one exact product, the two parts one addition.
#include "int4.cuh"

namespace rolaq {
namespace i4 {
namespace {

constexpr int kThreads = 256;

// A score's place in an order of unsigned whole numbers.
__device__ __forceinline__ uint32_t rank_key(float s) {
  const uint32_t u = __float_as_uint(s);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One CTA per request.  The query is quantised into shared memory (values, and their sizes), warps
// score pages, and a page is kept when fewer than the free places lie before it.
__global__ void __launch_bounds__(kThreads) select_kernel(SelectArgs a) {
  extern __shared__ int8_t sm[];
  const int d = a.cache.latent_dim, w = d + a.cache.rope_dim, words = w / 4, d_words = d / 4;
  const int b = blockIdx.x, tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
  int* q8 = reinterpret_cast<int*>(sm);  // [heads][words]
  int* q8_abs = q8 + a.heads * words;
  __shared__ float tops[2][kThreads / 32];
  __shared__ int base;
  int len = a.seq_lens[b];
  if (len > a.max_pages * kPage) {
    if (tid == 0) report(a.err, ROLAQ_DEV_BAD_REQ);
    len = a.max_pages * kPage;
  }
  len = max(len, 0);
  const int held = (len + kPage - 1) / kPage, most = min(held, a.budget);
  int32_t* sel = a.sel_table + b * a.sel_stride;
  const int32_t* table = a.page_table + b * a.pt_stride;
  for (int i = most + tid; i < a.budget; i += kThreads) sel[i] = -1;
  if (tid == 0) a.sel_lens[b] = held == 0 ? 0 : (most - 1) * kPage + len - (held - 1) * kPage;
  if (held <= a.budget) {
    for (int i = tid; i < held; i += kThreads) sel[i] = table[i];
    return;
  }
  const uint16_t* q = a.q + b * a.q_sb;
  float top[2] = {0.f, 0.f};
  for (int i = tid; i < a.heads * w; i += kThreads) {
    const int col = i % w;
    top[col >= d] = fmaxf(top[col >= d], fabsf(bf16_lo(q[(i / w) * a.q_sh + col])));
  }
  for (int k = 0; k < 2; ++k) {
    top[k] = warp_max_f32(top[k]);
    if (lane == 0) tops[k][warp] = top[k];
  }
  __syncthreads();
  int e[2];
  for (int k = 0; k < 2; ++k) {
    float m = 0.f;
    for (int i = 0; i < kThreads / 32; ++i) m = fmaxf(m, tops[k][i]);
    e[k] = unit_exponent(m);
  }
  for (int i = tid; i < a.heads * w; i += kThreads) {
    const int col = i % w;
    const float x = rintf(bf16_lo(q[(i / w) * a.q_sh + col]) * pow2(-e[col >= d]));
    const int v = static_cast<int>(fminf(fmaxf(x, -127.f), 127.f));
    sm[i] = static_cast<int8_t>(v);
    sm[a.heads * w + i] = static_cast<int8_t>(abs(v));
  }
  __syncthreads();
  float* scores = a.scores + static_cast<int64_t>(b) * a.max_pages;
  const int64_t pool_pages = a.cache.num_slots / kPage;
  for (int p = warp; p < held; p += kThreads / 32) {
    const int64_t page = table[p];
    float best = -INFINITY;
    if (page >= 0 && page < pool_pages) {
      const int* c = reinterpret_cast<const int*>(a.cache.box_center + page * w);
      const int* r = reinterpret_cast<const int*>(a.cache.box_radius + page * w);
      const float u0 = pow2(e[0]) * pow2(a.cache.box_exps[page * 2]);
      const float u1 = pow2(e[1]) * pow2(a.cache.box_exps[page * 2 + 1]);
      for (int h = 0; h < a.heads; ++h) {
        int s[2] = {0, 0};
        for (int i = lane; i < words; i += 32) {
          int& acc = s[i >= d_words];
          acc = __dp4a(q8[h * words + i], c[i], acc);
          acc = static_cast<int>(__dp4a(static_cast<unsigned>(q8_abs[h * words + i]), static_cast<unsigned>(r[i]),
                                        static_cast<unsigned>(acc)));
        }
        s[0] = __reduce_add_sync(0xFFFFFFFFu, s[0]);
        s[1] = __reduce_add_sync(0xFFFFFFFFu, s[1]);
        best = fmaxf(best, __fadd_rn(__fmul_rn(static_cast<float>(s[0]), u0), __fmul_rn(static_cast<float>(s[1]), u1)));
      }
    } else if (lane == 0) {
      report(a.err, ROLAQ_DEV_BAD_PAGE);
    }
    if (p < a.keep_first || p >= held - a.keep_last) best = INFINITY;
    if (lane == 0) scores[p] = best;
  }
  if (tid == 0) base = 0;
  __syncthreads();
  for (int p0 = 0; p0 < held; p0 += kThreads) {
    const int p = p0 + tid;
    bool kept = false;
    if (p < held) {
      const uint32_t mine = rank_key(scores[p]);
      int before = 0;
      for (int i = 0; i < held; ++i) {
        const uint32_t other = rank_key(scores[i]);
        before += other > mine || (other == mine && i < p);
      }
      kept = before < a.budget;
    }
    for (int k = 0; k < kThreads / 32; ++k) {  // the warps in turn append what they keep
      if (warp == k) {
        const uint32_t votes = __ballot_sync(0xFFFFFFFFu, kept);
        const int at = base;
        __syncwarp();
        if (kept) sel[at + __popc(votes & ((1u << lane) - 1))] = table[p];
        if (lane == 0) base = at + __popc(votes);
      }
      __syncthreads();
    }
  }
}

}  // namespace

int64_t select_workspace(int batch, int max_pages) { return (int64_t(batch) * max_pages * 4 + 15) / 16 * 16 + 16; }

int launch_select(const SelectArgs& a, cudaStream_t s) {
  const int smem = 2 * a.heads * (a.cache.latent_dim + a.cache.rope_dim);
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return ROLAQ_ECUDA;
  select_kernel<<<a.batch, kThreads, smem, s>>>(a);
  return cudaGetLastError() == cudaSuccess ? ROLAQ_OK : ROLAQ_ECUDA;
}

}  // namespace i4
}  // namespace rolaq
