// Page selection: scores of the pages of a request against its query, and the pages that are kept.
//
// score(page) = max over the heads of sum over both parts of 2^(e_q + e_page) (sum q8 center + sum |q8| radius).
// The sums are whole numbers below 2^24 (127 * 127 * 512 for the centers, 127 * 128 * 512 for the radii),
// so their order does not matter; each part is one conversion and one exact product, the two parts one addition.  Only
// the order of a request's scores counts, so they are taken over 2^20 times the query's larger unit: with units of 2^-100
// to 2^122 in the boxes none then overflows, and infinity is left to the pages that are kept whatever they score.
//
// The boxes are read once (bandwidth is the bound): a warp takes 8 pages at a time, a lane 16 bytes of a page
// per 64 columns, which are the operands of two m16n8k32 integer products as they are - centers times q8 and radii
// times |q8| into the same sums - with the 16 heads of a tile as rows; q8 lies in shared memory in operand order.
// A request's pages are shared by a few CTAs; the one that scores last keeps the pages: the budget-th largest
// score by an 8-bit radix search, then, in the pages' order, all above it and the first of its equals.
// Measured: 64 requests of 256 pages, 16 heads (19 MB of boxes) 17 us, of which memory needs 3: a CTA's one pass over its
// pages and the search are chains of dependent steps.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "int4.cuh"
#include "kernels.cuh"

namespace rolaq {
namespace i4 {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kTile = 8;        // pages of a warp's products
constexpr int kCached = 4096;   // scores that the radix search holds in shared memory

// A score's place in an order of unsigned whole numbers.
__device__ __forceinline__ uint32_t rank_key(float s) {
  const uint32_t u = __float_as_uint(s);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// 2^e for e <= 127, rounded to a subnormal or 0 below 2^-126.
__device__ __forceinline__ float any_pow2(int e) {
  const float x = pow2(max(e, -126));
  return e >= -126 ? x : x * pow2(max(e + 126, -126));
}

__device__ __forceinline__ void mma_s8s8(int (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8u8(int (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// Which pages of a request with `held` pages are kept, in order: the table's ids to sel.  All threads of the CTA.
__device__ void keep_pages(const float* __restrict__ scores, const int32_t* __restrict__ table, int held, int budget,
                           int32_t* __restrict__ sel, uint32_t* cached) {
  __shared__ int hist[256], warp_sum[kWarps];
  __shared__ uint32_t found_digit;
  __shared__ int found_left;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
  const bool fits = held <= kCached;
  if (fits)
    for (int i = tid; i < held; i += kThreads) cached[i] = rank_key(__ldcg(scores + i));
  auto key_at = [&](int i) { return fits ? cached[i] : rank_key(__ldcg(scores + i)); };
  // the budget-th largest key, 8 bits at a time: `prefix` so far, `left` of it and above still to be found
  uint32_t prefix = 0, mask = 0;
  int left = budget;
  for (int shift = 24; shift >= 0; shift -= 8) {
    hist[tid] = 0;
    __syncthreads();
    for (int i0 = 0; i0 < held; i0 += kThreads) {
      const int i = i0 + tid;
      const uint32_t key = i < held ? key_at(i) : 0;
      const bool counts = i < held && (key & mask) == prefix;
      const int digit = counts ? static_cast<int>((key >> shift) & 255u) : 256;
      const uint32_t same = __match_any_sync(0xFFFFFFFFu, digit);  // one add a value and warp
      if (counts && lane == __ffs(same) - 1) atomicAdd(&hist[digit], __popc(same));
    }
    __syncthreads();
    // keys with a larger digit: a suffix sum over the 256 counters, thread t the one of digit 255 - t
    const int mine = hist[255 - tid];
    int x = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int y = __shfl_up_sync(0xFFFFFFFFu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_sum[warp] = x;
    __syncthreads();
    for (int w = 0; w < warp; ++w) x += warp_sum[w];
    if (x - mine < left && left <= x) found_digit = 255 - tid, found_left = left - (x - mine);
    __syncthreads();
    prefix |= found_digit << shift;
    mask |= 255u << shift;
    left = found_left;
  }
  // in order: all above the key, and the first `left` equal to it
  int placed = 0, equals = 0;
  for (int p0 = 0; p0 < held; p0 += kThreads) {
    const int p = p0 + tid;
    const uint32_t key = p < held ? key_at(p) : 0;
    const bool above = p < held && key > prefix, equal = p < held && key == prefix;
    const uint32_t v_above = __ballot_sync(0xFFFFFFFFu, above), v_equal = __ballot_sync(0xFFFFFFFFu, equal);
    if (lane == 0) warp_sum[warp] = __popc(v_above) | __popc(v_equal) << 16;
    __syncthreads();
    int before = 0, total = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += warp_sum[w];
      total += warp_sum[w];
    }
    const uint32_t lower = (1u << lane) - 1;
    const int eq = equals + (before >> 16) + __popc(v_equal & lower);  // equal keys before this one
    const int ab = (before & 0xFFFF) + __popc(v_above & lower);        // keys above, before it in this chunk
    if (above || (equal && eq < left)) {
      const int eq_kept = min(eq, left) - min(equals, left);  // equals of this chunk kept before it
      sel[placed + ab + eq_kept] = table[p];
    }
    placed += (total & 0xFFFF) + min(equals + (total >> 16), left) - min(equals, left);
    equals += total >> 16;
    __syncthreads();
  }
}

// chunk_pages pages of a request per CTA (a multiple of kTile * kWarps).
template <int D, int DR>
__global__ void __launch_bounds__(kThreads) select_kernel(const SelectArgs a, const int chunk_pages) {
  constexpr int W = D + DR, STEPS = (D + DR) / 32;  // 32-column steps
  extern __shared__ __align__(16) uint8_t dynamic[];
  uint4* q8 = reinterpret_cast<uint4*>(dynamic);  // [tile][step][q8, |q8|][lane]
  __shared__ float tops[2][kWarps];
  __shared__ bool last;
  const int b = blockIdx.y, tid = threadIdx.x, warp = tid / 32, lane = tid & 31, g = lane >> 2, j = lane & 3;
  grid_launch_dependents();
  grid_dependency_wait();
  int len = a.seq_lens[b];
  if (len > a.max_pages * static_cast<int64_t>(kPage)) {
    if (tid == 0 && blockIdx.x == 0) report(a.err, ROLAQ_DEV_BAD_REQ);
    len = a.max_pages * kPage;
  }
  len = max(len, 0);
  const int held = (len + kPage - 1) / kPage, most = min(held, a.budget);
  int32_t* sel = a.sel_table + b * a.sel_stride;
  const int32_t* table = a.page_table + b * a.pt_stride;
  if (blockIdx.x == 0) {
    for (int i = most + tid; i < a.budget; i += kThreads) sel[i] = -1;
    if (tid == 0) a.sel_lens[b] = held == 0 ? 0 : (most - 1) * kPage + len - (held - 1) * kPage;
    if (held <= a.budget)
      for (int i = tid; i < held; i += kThreads) sel[i] = table[i];
  }
  const int p_begin = blockIdx.x * chunk_pages, p_end = min(held, p_begin + chunk_pages);
  if (held <= a.budget || p_begin >= p_end) return;

  // The boxes of the warp's next 8 pages, the lane's part as operands.  The first are on their way while the query
  // is quantised.
  const int pool_pages = static_cast<int>(a.cache.num_slots / kPage);
  uint4 c[STEPS / 2], r[STEPS / 2];
  uint2 c_end, r_end;
  int2 e_page;
  bool ok;
  auto load_boxes = [&](int p0) {
    const int id = p0 + g < p_end ? table[p0 + g] : 0;
    ok = id >= 0 && id < pool_pages;
    if (!ok && j == 0) report(a.err, ROLAQ_DEV_BAD_PAGE);
    const int64_t page = ok ? id : 0, at = page * W;
#pragma unroll
    for (int s = 0; s < STEPS / 2; ++s) {
      c[s] = *reinterpret_cast<const uint4*>(a.cache.box_center + at + 64 * s + 16 * j);
      r[s] = *reinterpret_cast<const uint4*>(a.cache.box_radius + at + 64 * s + 16 * j);
    }
    if (DR == 32) {
      c_end = *reinterpret_cast<const uint2*>(a.cache.box_center + at + D + 8 * j);
      r_end = *reinterpret_cast<const uint2*>(a.cache.box_radius + at + D + 8 * j);
    }
    e_page = *reinterpret_cast<const int2*>(a.cache.box_exps + 2 * page);
  };
  const int first = p_begin + warp * kTile;
  if (first < p_end) load_boxes(first);

  // ---- the query in 8 bits, in operand order ----
  const uint16_t* q = a.q + b * a.q_sb;
  // The parts' largest elements; elements that are no finite numbers are looked for only where an infinity shows.
  float m[2];
  auto find_tops = [&](auto finite) {
    float top[2] = {0.f, 0.f};
    for (int i = tid; i < a.heads * (W / 8); i += kThreads) {
      const int col = 8 * (i % (W / 8));
      const uint4 w = *reinterpret_cast<const uint4*>(q + (i / (W / 8)) * a.q_sh + col);
      const uint32_t v[4] = {w.x, w.y, w.z, w.w};
      float most = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float size = fabsf(h ? bf16_hi(v[k]) : bf16_lo(v[k]));
          if (!finite || size < INFINITY) most = fmaxf(most, size);  // fmaxf passes a NaN over
        }
      top[col >= D] = fmaxf(top[col >= D], most);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      top[k] = warp_max_f32(top[k]);
      if (lane == 0) tops[k][warp] = top[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      m[k] = 0.f;
      for (int i = 0; i < kWarps; ++i) m[k] = fmaxf(m[k], tops[k][i]);
    }
  };
  find_tops(std::false_type());
  if (!(m[0] < INFINITY && m[1] < INFINITY)) {
    __syncthreads();
    find_tops(std::true_type());
  }
  const int e[2] = {unit_exponent(m[0]), unit_exponent(m[1])};
  const int e_top = m[0] > 0.f ? (m[1] > 0.f ? max(e[0], e[1]) : e[0]) : e[1];  // of the parts that hold anything
  const int rel[2] = {m[0] > 0.f ? e[0] - e_top - 20 : -20, m[1] > 0.f ? e[1] - e_top - 20 : -20};
  // Operand register r of lane (g, j), step s: row g + 8 (r & 1), columns that the boxes' 16-byte pieces put there:
  // block s / 2, bytes 16 j + 8 (s & 1) + 4 (r >> 1) of it; a half block at the end (DR = 32) has 8-byte pieces.
  const int tiles = (a.heads + 15) / 16;
  for (int i = tid; i < tiles * STEPS * 128; i += kThreads) {  // a register each
    const int r = i & 3, l = (i >> 2) & 31, s = (i >> 7) % STEPS, tile = i / (STEPS * 128);
    const int head = tile * 16 + (l >> 2) + 8 * (r & 1);
    const int col = DR == 32 && s == STEPS - 1 ? D + 8 * (l & 3) + 4 * (r >> 1)
                                               : 64 * (s >> 1) + 16 * (l & 3) + 8 * (s & 1) + 4 * (r >> 1);
    uint32_t v = 0, u = 0;
    if (head < a.heads) {
      const uint2 w = *reinterpret_cast<const uint2*>(q + head * a.q_sh + col);
      const float inv = pow2(-e[col >= D]);
      const float x[4] = {bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y)};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float t = rintf(x[k] * inv);
        const int c = fabsf(x[k]) < INFINITY ? static_cast<int>(fminf(fmaxf(t, -127.f), 127.f)) : 0;
        v |= static_cast<uint32_t>(c & 255) << (8 * k);
        u |= static_cast<uint32_t>(abs(c)) << (8 * k);
      }
    }
    uint32_t* at = reinterpret_cast<uint32_t*>(q8 + ((tile * STEPS + s) * 2) * 32 + l) + r;
    at[0] = v;
    at[128] = u;
  }
  __syncthreads();

  // ---- the scores ----
  float* scores = a.scores + static_cast<int64_t>(b) * a.max_pages;
  for (int p0 = first; p0 < p_end; p0 += kTile * kWarps) {
    if (p0 != first) load_boxes(p0);
    // pages 2 j and 2 j + 1 of the tile are the lane's as results
    float unit[2][2];
    bool there[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int from = (2 * j + x) * 4;
      unit[x][0] = any_pow2(rel[0] + __shfl_sync(0xFFFFFFFFu, e_page.x, from));
      unit[x][1] = any_pow2(rel[1] + __shfl_sync(0xFFFFFFFFu, e_page.y, from));
      there[x] = __shfl_sync(0xFFFFFFFFu, ok, from);
    }
    float best[2] = {-INFINITY, -INFINITY};
#pragma unroll 1
    for (int tile = 0; tile < tiles; ++tile) {
      int lat[4] = {0, 0, 0, 0}, rot[4] = {0, 0, 0, 0};
      const uint4* qs = q8 + tile * STEPS * 64 + lane;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const uint4 qv = qs[(2 * s) * 32], qa = qs[(2 * s + 1) * 32];
        uint32_t cb[2], rb[2];
        if (DR == 32 && s == STEPS - 1) {
          cb[0] = c_end.x, cb[1] = c_end.y, rb[0] = r_end.x, rb[1] = r_end.y;
        } else if (s & 1) {
          cb[0] = c[s / 2].z, cb[1] = c[s / 2].w, rb[0] = r[s / 2].z, rb[1] = r[s / 2].w;
        } else {
          cb[0] = c[s / 2].x, cb[1] = c[s / 2].y, rb[0] = r[s / 2].x, rb[1] = r[s / 2].y;
        }
        mma_s8s8(s < D / 32 ? lat : rot, qv, cb[0], cb[1]);
        mma_s8u8(s < D / 32 ? lat : rot, qa, rb[0], rb[1]);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float s = __fadd_rn(__fmul_rn(static_cast<float>(lat[x]), unit[x & 1][0]),
                                  __fmul_rn(static_cast<float>(rot[x]), unit[x & 1][1]));
        if (tile * 16 + g + 8 * (x >> 1) < a.heads) best[x & 1] = fmaxf(best[x & 1], s);
      }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int o = 4; o < 32; o *= 2) best[x] = fmaxf(best[x], __shfl_xor_sync(0xFFFFFFFFu, best[x], o));
      const int page = p0 + 2 * j + x;
      if (g == 0 && page < p_end) {
        const bool kept = page < a.keep_first || page >= held - a.keep_last;
        __stcg(scores + page, kept ? INFINITY : there[x] ? best[x] : -INFINITY);
      }
    }
  }

  // ---- the CTA that scores last keeps the pages ----
  const int chunks = (held + chunk_pages - 1) / chunk_pages;
  __syncthreads();
  if (chunks > 1) {
    if (tid == 0) {
      __threadfence();
      const int before = atomicAdd(&a.counters[b], 1);
      last = before == chunks - 1;
      if (last) a.counters[b] = 0;
      __threadfence();
    }
    __syncthreads();
    if (!last) return;
  }
  keep_pages(scores, table, held, a.budget, sel, reinterpret_cast<uint32_t*>(dynamic));
}

template <int D, int DR>
int launch(const SelectArgs& a, cudaStream_t s) {
  const int q_bytes = (a.heads + 15) / 16 * ((D + DR) / 32) * 1024, smem = std::max(q_bytes, kCached * 4);
  static std::atomic<uint64_t> prepared{0};  // devices whose limit is raised
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return ROLAQ_ECUDA;
  if (smem > 46 * 1024 && !(prepared.load() >> (device & 63) & 1)) {
    if (cudaFuncSetAttribute(select_kernel<D, DR>, cudaFuncAttributeMaxDynamicSharedMemorySize, 8 * ((D + DR) / 32) * 1024) !=
        cudaSuccess)
      return ROLAQ_ECUDA;
    prepared |= uint64_t(1) << (device & 63);
  }
  // CTAs of one pass over their pages each, as long as two a multiprocessor are enough for it: few requests are spread
  // over the machine (one of 2048 pages), many get one CTA each, which then needs no join of the scores
  constexpr int pass = kTile * kWarps;
  const int passes = (a.max_pages + pass - 1) / pass;
  const int per_request = std::max(1, 2 * sm_count() / a.batch);
  const int chunks = a.batch > static_cast<int>(kHeaderBytes / 4) ? 1 : std::max(1, std::min(passes, per_request));
  const int chunk_pages = (passes + chunks - 1) / chunks * pass;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(std::max(1, (a.max_pages + chunk_pages - 1) / std::max(1, chunk_pages)), a.batch);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, select_kernel<D, DR>, a, chunk_pages) == cudaSuccess ? ROLAQ_OK : ROLAQ_ECUDA;
}

}  // namespace

int64_t select_workspace(int batch, int max_pages) { return (int64_t(batch) * max_pages * 4 + 15) / 16 * 16 + 16; }

int launch_select(const SelectArgs& a, cudaStream_t s) {
  if (a.cache.latent_dim == 512) return a.cache.rope_dim == 64 ? launch<512, 64>(a, s) : launch<512, 32>(a, s);
  return a.cache.rope_dim == 64 ? launch<256, 64>(a, s) : launch<256, 32>(a, s);
}

}  // namespace i4
}  // namespace rolaq
