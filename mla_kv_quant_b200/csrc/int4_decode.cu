// Absorbed attention over the 4-bit latent cache.
//
// With value (c - z) s of a 4-bit code c, per 128-element group g of a token t:
//   q . k_t = sum_g s_gt (q_g . c_gt - z_gt sum q_g) + q_pe . k_pe_t
//   sum_t P_t v_t = sum_t (P_t s_gt) c_gt - sum_t (P_t s_gt) z_gt
// so both contractions run on the raw codes, which tensor cores take after one AND per register:
// the FP16 patterns 0..15 and 16 * (0..15) are c 2^-24 and 16 c 2^-24 exactly.  The factor 16 of odd
// elements is taken out of the query before and out of the result after.  The query is FP16 under a
// power of two of its row (exact for BF16 within 2^26 of the row's largest element), P s is FP16 (11
// bits), the rotary part stays BF16; all are m16n8k16 products with FP32 sums.
//
// Codes are the 16-high side of the products, the query rows (query tokens x heads) the 8-wide side: a CTA holds
// NH tiles of 8 rows (one or two for D = 512, up to five for D = 256, where 40 heads then are one pass) and
// walks the pages of one or more requests; a page (64 tokens) is one pipeline stage (TMA, 128-byte swizzle,
// so that ldmatrix reads without conflicts).
// The 8 working warps form pairs: a pair scores 16 of a page's tokens, each warp of it over half of the
// latent columns (the query's operand registers would not fit otherwise), and swaps partial scores, so
// that a tick later each warp weighs 8 tokens: against a reference maximum that moves only when weights
// pass it by 2^10, P s of each group going to shared memory.  Another tick later each warp adds D/8
// latent columns of the page up.  So three pages are under way in a tick, with nothing to wait for between
// their parts, and one barrier ends it: it publishes the swap and the weights, carries the vote on
// moving the references, and joins two helping warps: one waits for the next page's arrival before it,
// one refills the stage that became free after it (either would cost a working warp hundreds of cycles).
//
// The pages of all requests are dealt to the CTAs in one equal run each (a run may begin or end inside
// a request); what is cut is joined by merge_kernel by log-sum-exp.
#include <algorithm>
#include <atomic>

#include "int4.cuh"
#include "kernels.cuh"

namespace rolaq {
namespace i4 {
namespace {

// Eight working warps and a warpgroup of which two warps load.  Of the 168 registers a thread that a block of
// 384 is launched with, the loaders hand most to the workers: 2 * 224 + 56 = 2 * 232 + 40 = 3 * 168.
constexpr int kWarps = 8, kWorkers = kWarps * 32, kThreads = kWorkers + 128;
constexpr int kMinPages = 2;  // least run of pages worth a CTA of its own
constexpr float kSlack = 1024.f, kScaleSlack = 32.f;  // how far weights and scales may pass their references (P s <= 2^15)
constexpr float kNoMax = -1e30f, kNoUnit = 1.329227995784916e36f;  // references not yet set: the first token passes them
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <int D, int DR, int NH>
struct Cfg {
  static constexpr int NG = D / kGroup;             // groups of a token
  static constexpr int CODES = kPage * D / 2, ROPE = kPage * DR * 2, PARAMS = kPage * NG * 8;
  static constexpr int STAGE = CODES + ROPE + PARAMS;
  static constexpr int QROW = (D + DR) * 2 + 16;    // bytes of a query row in shared memory (16: no bank conflicts)
  static constexpr int STAGES = D == 512 ? 6 : DR == 64 ? 8 : 10;
  static constexpr int PTILE = kPage * 16;          // P s of a page, a group and 8 rows: [token][row] FP16
  static constexpr int PBUF = NG * NH * PTILE;
  static constexpr int SMEM = 1024 + STAGES * STAGE + 2 * PBUF + 8 * NH * QROW;
  static constexpr int HG = NG / 2;                 // groups that a warp scores
  static constexpr int CH = D / kWarps / 32;        // 32-column chunks that a warp adds up
  static constexpr int ROWS = 8 * NH;
  static constexpr int WORKER_REGS = NH < 4 ? 224 : 232, LOADER_REGS = NH < 4 ? 56 : 40;
};

template <int NG, int NH>
struct Shared {
  float2 swap[2][kWarps][NH][32];
  float red_m[kWarps][8 * NH], red_s[kWarps][NG], red_l[kWarps][8 * NH], red_z[kWarps][NG][8 * NH];
  float q_top[2][8 * NH], q_sum[NG][8 * NH], row_scale[8 * NH];
  float l_all[8 * NH], z_all[NG][8 * NH], max[8 * NH];
};

// Named barriers: the end of a tick (working and loading warps), and the working warps'.
constexpr int kBarTick = 1, kBarWork = 2;
__device__ __forceinline__ void work_sync() { named_bar_sync(kBarWork, kWorkers); }
__device__ __forceinline__ bool tick(bool vote) {
  int any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %3, 0;\n\tbar.red.or.pred q, %1, %2, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "n"(kBarTick), "n"(kWorkers + 64), "r"(static_cast<int>(vote))
      : "memory");
  return any != 0;
}

__device__ __forceinline__ int pages_of(const DecodeArgs& a, int b) {
  const int64_t len = min(static_cast<int64_t>(a.seq_lens[b]), static_cast<int64_t>(a.max_pages) * kPage);
  return len <= 0 ? 0 : static_cast<int>((len + kPage - 1) / kPage);
}

// Runs are equal shares of the `total` pages: run r of n begins at page total * r / n.
struct Runs {
  int64_t total;
  int n;
  __device__ Runs(int64_t total_, int groups)
      : total(total_), n(static_cast<int>(min(static_cast<int64_t>(groups), max(int64_t(1), (total_ + kMinPages - 1) / kMinPages)))) {}
  __device__ int64_t begin(int r) const {
    const uint64_t x = static_cast<uint64_t>(total) * r;
    return x >> 32 ? static_cast<int64_t>(x / n) : static_cast<uint32_t>(x) / static_cast<uint32_t>(n);  // 32 bits where they do
  }
  __device__ int holding(int64_t page) const {  // the run that holds a page
    const uint64_t x = static_cast<uint64_t>(page) * n;
    int r = static_cast<int>(x >> 32 || total >> 32 ? x / total : static_cast<uint32_t>(x) / static_cast<uint32_t>(total));
    while (begin(r + 1) <= page) ++r;
    return r;
  }
};

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// D (16 x 8, FP32) += A (16 x 16) B (16 x 8).  Not volatile: the compiler may interleave them.
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Bytes 1 and 3 as 16-bit halves.
__device__ __forceinline__ uint32_t odd_bytes(uint32_t w) { return prmt(w, 0u, 0x4341u); }
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The shared-memory offset of 16-byte chunk `chunk` of row `row` under TMA's swizzles.
__device__ __forceinline__ uint32_t sw128(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }
__device__ __forceinline__ uint32_t sw64(int row, int chunk) { return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4); }

// Sum over a quad's four lanes / maximum over them, and over the eight lanes of the same place in their quads.
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xFFFFFFFFu, v, 1);
  return v + __shfl_xor_sync(0xFFFFFFFFu, v, 2);
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 2));
}

__device__ __forceinline__ float oct_sum(float v) {
#pragma unroll
  for (int o = 4; o < 32; o *= 2) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
__device__ __forceinline__ float oct_max(float v) {
#pragma unroll
  for (int o = 4; o < 32; o *= 2) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}

// Exclusive prefix over the CTA's threads of v; the total in `total`.
template <int WARPS>
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t& total, int64_t* sm) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int64_t y = __shfl_up_sync(0xFFFFFFFFu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) sm[warp] = x;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int k = 0; k < WARPS; ++k) {
    if (k < warp) before += sm[k];
    total += sm[k];
  }
  return before + x - v;
}

struct Partials {
  float* o;    // [2 * groups * row blocks][rows of a CTA][D], normalised
  float* lse;  // [2 * groups * row blocks][rows of a CTA], natural log
  int4* cut;   // [batch]: a request's first run, its runs, whether the first begins in an earlier request
  int rows;    // of a CTA
};

template <int D, int DR, int NH>
__global__ void __launch_bounds__(kThreads, 1)
    decode_kernel(const __grid_constant__ CUtensorMap map_codes, const __grid_constant__ CUtensorMap map_rope,
                  const DecodeArgs a, const Partials part, const int groups, const int blocks) {
  using C = Cfg<D, DR, NH>;
  constexpr int NG = C::NG, HG = C::HG, CH = C::CH, STAGES = C::STAGES, ROWS = C::ROWS;
  constexpr bool HELD_MAX = NH < 4;  // references in registers
  constexpr int KR = DR / 32;  // 16-column steps of the rotary part that a warp scores
  extern __shared__ char raw[];
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  char* pbuf = smem + STAGES * C::STAGE;
  char* qbuf = pbuf + 2 * C::PBUF;
  __shared__ uint64_t full[STAGES], q_full;
  __shared__ int bad_page[STAGES];
  __shared__ int64_t scan[kThreads / 32];
  __shared__ int start[2];
  __shared__ int64_t run_total, run_begin;  // read again where a request ends (registers are short in between)
  __shared__ Shared<NG, NH> sh;

  const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31, g = lane >> 2, j = lane & 3;
  const int block = blockIdx.x % blocks, group = blockIdx.x / blocks;
  const int rows = a.q_len * a.heads, row0 = block * ROWS;
  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) mbar_init(&full[s], 1);
    mbar_init(&q_full, 1);
    fence_mbar_init();
    prefetch_tensormap(&map_codes);
    prefetch_tensormap(&map_rope);
  }
  grid_launch_dependents();
  grid_dependency_wait();

  // ---- this CTA's run of pages ----
  const int per = (a.batch + kThreads - 1) / kThreads;
  int64_t mine = 0, total;
  for (int b = tid * per; b < min(a.batch, (tid + 1) * per); ++b) mine += pages_of(a, b);
  int64_t before = block_scan<kThreads / 32>(mine, total, scan);
  for (int b = group; b < a.batch; b += groups) {  // requests without a token
    if (pages_of(a, b) != 0) continue;
    if (tid == 0 && block == 0) part.cut[b] = make_int4(0, 0, 0, 0);
    for (int i = tid; i < min(ROWS, rows - row0) * (D / 8); i += kThreads) {
      const int row = row0 + i / (D / 8), t = row / a.heads, h = row % a.heads;
      *reinterpret_cast<uint4*>(a.out + b * a.o_sb + t * a.o_st + h * a.o_sh + 8 * (i % (D / 8))) = make_uint4(0, 0, 0, 0);
      if (a.lse && i % (D / 8) == 0) a.lse[static_cast<int64_t>(b) * rows + row] = -INFINITY;
    }
  }
  const Runs runs(total, groups);
  if (group >= runs.n || total == 0) return;
  const int64_t u0 = runs.begin(group);
  const int n_units = static_cast<int>(runs.begin(group + 1) - u0);
  if (tid == 0) run_total = total, run_begin = u0;
  if (before <= u0 && u0 < before + mine) {
    int b = tid * per;
    for (int n; before + (n = pages_of(a, b)) <= u0; ++b) before += n;
    start[0] = b;
    start[1] = static_cast<int>(u0 - before);
  }
  __syncthreads();
  int seg_b = start[0], seg_p = start[1];

  if (warp >= kWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::LOADER_REGS));
    if (warp > kWarps + 1) return;
    const bool loader = warp == kWarps;
    // ================= the loading warp: stage k holds page k of the run =================
    // Lane l holds the id of page `base` + l of the run; the next 32 are requested 32 pages ahead of their use.
    const int pool_pages = static_cast<int>(a.cache.num_slots / kPage);
    int id_b = seg_b, id_p = seg_p + lane, ids = -1, next_ids = -1, loaded = 0, load_stage = 0;
    auto fetch_ids = [&](int first) {
      int id = -1;
      if (first + lane < n_units) {
        for (int n; id_p >= (n = pages_of(a, id_b)); ++id_b) id_p -= n;
        id = a.page_table[id_b * a.pt_stride + id_p];
      }
      id_p += 32;
      return id;
    };
    auto load = [&]() {
      if (loaded == n_units) return;
      if ((loaded & 31) == 0) {
        ids = next_ids;
        next_ids = fetch_ids(loaded + 32);
      }
      const int id = __shfl_sync(0xFFFFFFFFu, ids, loaded & 31);
      ++loaded;
      const bool ok = id >= 0 && id < pool_pages;
      const int page = ok ? id : 0;
      if (lane == 0) {
        char* dst = smem + load_stage * C::STAGE;
        uint64_t* bar = &full[load_stage];
        bad_page[load_stage] = !ok;
        mbar_expect_tx(bar, C::STAGE);
#pragma unroll
        for (int k = 0; k < D / 256; ++k) tma_load_2d(dst + k * 8192, &map_codes, bar, k * 128, page * kPage);
        tma_load_2d(dst + C::CODES, &map_rope, bar, 0, page * kPage);
        bulk_load(dst + C::CODES + C::ROPE, a.cache.params + static_cast<int64_t>(page) * (kPage * NG * 2), C::PARAMS, bar);
        if (!ok) report(a.err, ROLAQ_DEV_BAD_PAGE);
      }
      __syncwarp();
      if (++load_stage == STAGES) load_stage = 0;
    };
    auto load_query = [&](int b) {
      const int live = min(ROWS, rows - row0);
      if (lane == 0) mbar_expect_tx(&q_full, live * ((D + DR) * 2));
      __syncwarp();
      for (int r = lane; r < live; r += 32) {
        const int t = (row0 + r) / a.heads, h = (row0 + r) % a.heads;
        bulk_load(qbuf + r * C::QROW, a.q + b * a.q_sb + t * a.q_st + h * a.q_sh, (D + DR) * 2, &q_full);
      }
    };
    // ================= the awaiting warp =================
    int stage = 0, lap = 0, arrived = 0, queries = 0;
    bool healthy = true;
    auto await = [&]() {  // the next page of the run; after one that did not come in time the rest is not awaited
      if (arrived == n_units) return;
      if (healthy) healthy = mbar_wait(&full[stage], lap & 1, a.err);
      __syncwarp();
      ++arrived;
      if (++stage == STAGES) stage = 0, ++lap;
    };
    auto await_query = [&]() {
      if (healthy) healthy = mbar_wait(&q_full, queries & 1, a.err);
      __syncwarp();
      ++queries;
    };
    if (loader) {
      next_ids = fetch_ids(0);
      load_query(seg_b);
      for (int i = 0; i < STAGES; ++i) load();
    } else {
      await_query();
      await();
    }
    tick(false);
    for (int done = 0; done < n_units;) {
      const int count = min(pages_of(a, seg_b) - seg_p, n_units - done);
      done += count;
      do ++seg_b;  // the request after this one, where the run has one
      while (done < n_units && pages_of(a, seg_b) == 0);
      seg_p = 0;
      for (int t = 0; t < count + 2; ++t) {
        if (!loader && t + 1 < count) await();  // the page that the next tick scores
        if (!loader && t == count + 1 && done < n_units) {
          await_query();
          await();
        }
        tick(false);
        if (loader && t == 0 && done < n_units) load_query(seg_b);  // this request's query has been taken
        if (loader && t >= 2) load();                               // page t - 2 has been added up
      }
    }
    return;
  }

  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::WORKER_REGS));
  const int half = warp & 1, quarter = warp >> 1;  // half of the latent columns, 16 of the page's tokens
  const int own = warp * NG / kWarps;              // the group of the columns that the warp adds up
  // Offsets of the lane's ldmatrix rows from a 1024-byte boundary.  Chunk c of a row lies at c ^ row % 8, so
  // chunk c ^ x is at the address ^ 16 x.  Of the pair's 16 tokens the warp's own eight come first.
  const uint32_t stages = smem_u32(smem), pbufs = smem_u32(pbuf);
  const int tok_row = 16 * quarter + ((8 * half + (lane & 15)) & 15);
  const uint32_t code_off = D == 512 ? half * 8192 + sw128(tok_row, lane >> 4) : sw128(tok_row, 4 * half + (lane >> 4));
  const uint32_t rope_off = C::CODES + (DR == 64 ? sw128(tok_row, 4 * half + (lane >> 4)) : sw64(tok_row, 2 * half + (lane >> 4)));
  const uint32_t add_off = (warp * CH / 8) * 8192 + sw128(lane, (warp * CH) & 7);
  const uint32_t p_off = own * (NH * C::PTILE) + lane * 16;
  const uint32_t p_dst = (8 * warp + g) * 16 + 4 * j;
  const float qk_scale = a.sm_scale * kLog2e;
  int done = 0, stage = 0;  // pages of the run; the stage of the page scored next
  tick(false);              // the first query and page are there

  while (done < n_units) {
    const int seg_pages = pages_of(a, seg_b);
    if (seg_pages == 0) {
      ++seg_b;
      continue;
    }
    const bool first = done == 0;
    const int count = min(seg_pages - seg_p, n_units - done);
    const int len = min(static_cast<int64_t>(a.seq_lens[seg_b]), static_cast<int64_t>(a.max_pages) * kPage);
    if (tid == 0 && len != a.seq_lens[seg_b]) report(a.err, ROLAQ_DEV_BAD_REQ);
    const int lim_min = len - a.q_len + 1;

    // ---- the query: brought to operand form in place, 8 elements at a time, then row g of each tile to registers ----
    constexpr int QC = D / 8;  // 16-byte pieces of a row's latent part
    const int live = min(ROWS, rows - row0);
#pragma unroll 1
    for (int i = tid; i < ROWS * QC; i += kWorkers) {
      const int r = i / QC;
      float top = 0.f, odd = 0.f;
      if (r < live) {
        const uint4 w = *reinterpret_cast<const uint4*>(qbuf + r * C::QROW + 16 * (i % QC));
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          top = fmaxf(top, fmaxf(fabsf(bf16_lo(v[k])), fabsf(bf16_hi(v[k]))));
          odd = fmaf(bf16_lo(v[k]), 0.f, fmaf(bf16_hi(v[k]), 0.f, odd));  // NaN where an element is no finite number
        }
      }
      top = warp_max_f32(odd != 0.f ? INFINITY : top);
      if (lane == 0) sh.q_top[D == 512 ? (i / 32) & 1 : 0][r] = top;
    }
    work_sync();
    auto row_top = [&](int r) { return D == 512 ? fmaxf(sh.q_top[0][r], sh.q_top[1][r]) : sh.q_top[0][r]; };
    auto row_unit = [&](float top) {  // 2^k with top 2^k in [2^13, 2^14)
      return top > 0.f ? pow2(min(max(13 - (static_cast<int>(__float_as_uint(top) >> 23) - 127), -100), 100)) : 1.f;
    };
#pragma unroll 1
    for (int i = tid; i < ROWS * QC; i += kWorkers) {
      const int r = i / QC, c = i % QC;
      const float top = row_top(r), up = row_unit(top);
      uint4* at = reinterpret_cast<uint4*>(qbuf + r * C::QROW + 16 * c);
      const uint4 w = r < live ? *at : make_uint4(0, 0, 0, 0);
      const uint32_t v[4] = {w.x, w.y, w.z, w.w};
      float x[8], sum = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] = bf16_lo(v[e]) * up, x[2 * e + 1] = bf16_hi(v[e]) * up;
        sum += x[2 * e] + x[2 * e + 1];
      }
      // a word of codes gives elements (0, 4), 16 (1, 5), (2, 6) and 16 (3, 7)
      *at = make_uint4(pack_half2(x[0], x[4]), pack_half2(x[1] * 0.0625f, x[5] * 0.0625f), pack_half2(x[2], x[6]),
                       pack_half2(x[3] * 0.0625f, x[7] * 0.0625f));
#pragma unroll
      for (int o = 1; o < 16; o *= 2) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
      if (c % 16 == 0) sh.q_sum[c / 16][r] = sum * (1.f / 16777216.f);
      if (c == 0) sh.row_scale[r] = top == INFINITY ? __int_as_float(0x7FC00000) : qk_scale * (16777216.f / up);
    }
    // the rotary part under the same power of two (exact), so that both parts add up
#pragma unroll 1
    for (int i = tid; i < ROWS * (DR / 2); i += kWorkers) {
      const int r = i / (DR / 2);
      const float down = row_unit(row_top(r)) * (1.f / 16777216.f);
      uint32_t* at = reinterpret_cast<uint32_t*>(qbuf + r * C::QROW + 2 * D) + i % (DR / 2);
      *at = r < live ? pack_bf16x2(bf16_lo(*at) * down, bf16_hi(*at) * down) : 0u;
    }
    work_sync();
    uint32_t q[NH][8 * HG][2], q_pe[NH][KR][2];
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      const char* src = qbuf + (8 * n + g) * C::QROW;
#pragma unroll
      for (int c = 0; c < 4 * HG; ++c) {
        const uint4 w = *reinterpret_cast<const uint4*>(src + half * D + 64 * c + 16 * j);
        q[n][2 * c][0] = w.x, q[n][2 * c][1] = w.y, q[n][2 * c + 1][0] = w.z, q[n][2 * c + 1][1] = w.w;
      }
#pragma unroll
      for (int c = 0; c < KR; ++c)
#pragma unroll
        for (int e = 0; e < 2; ++e) q_pe[n][c][e] = *reinterpret_cast<const uint32_t*>(src + 2 * (D + 16 * (half * KR + c) + 8 * e + 2 * j));
    }
    // the rows' factors: held where few, read again each page where many
    float2 held_sum[NH <= 2 ? HG : 1][NH <= 2 ? NH : 1], held_scale[NH <= 2 ? NH : 1];
    auto q_sum_of = [&](int k, int n) { return *reinterpret_cast<const float2*>(&sh.q_sum[half * HG + k][8 * n + 2 * j]); };
    auto scale_of = [&](int n) { return *reinterpret_cast<const float2*>(&sh.row_scale[8 * n + 2 * j]); };
    if constexpr (NH <= 2) {
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        held_scale[n] = scale_of(n);
#pragma unroll
        for (int k = 0; k < HG; ++k) held_sum[k][n] = q_sum_of(k, n);
      }
    }

    // accumulators: tile 2 c + h of chunk c holds columns 4 g + 2 h (and that + 16 times the next one) x rows 2 j, + 1
    float acc[2 * CH][NH][4], zsum[NH][2][NG], unit[NG], l_sum[NH][2];
    float2 held_max[HELD_MAX ? NH : 1];  // references: the largest scores so far, kNoMax before the first
#pragma unroll
    for (int n = 0; n < NH; ++n) {
#pragma unroll
      for (int c = 0; c < 2 * CH; ++c) acc[c][n][0] = acc[c][n][1] = acc[c][n][2] = acc[c][n][3] = 0.f;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        l_sum[n][x] = 0.f;
#pragma unroll
        for (int k = 0; k < NG; ++k) zsum[n][x][k] = 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < NG; ++k) unit[k] = kNoUnit;
    auto max_of = [&](int n) {
      if constexpr (HELD_MAX) return held_max[n];
      else return *reinterpret_cast<const float2*>(&sh.max[8 * n + 2 * j]);
    };
    auto set_max = [&](int n, float2 m) {
      if constexpr (HELD_MAX) held_max[n] = m;
      else if (warp == 0 && g == 0) *reinterpret_cast<float2*>(&sh.max[8 * n + 2 * j]) = m;
    };
#pragma unroll
    for (int n = 0; n < NH; ++n) set_max(n, make_float2(kNoMax, kNoMax));

    // Partial scores of the pair's 16 tokens: the warp's own eight in mine_s, the partner's to the swap.
    float mine_s[NH][2] = {};
    auto score = [&](int st_at, int pb) {
      const uint32_t st = stages + st_at * C::STAGE;
      float c_acc[HG][NH][4], r_acc[NH][4];
      uint32_t w[HG][2][4], w_pe[KR][4];
#pragma unroll
      for (int k = 0; k < HG; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i) ldsm_x4((st + code_off) ^ (k << 6) ^ (i << 5), w[k][i]);
#pragma unroll
      for (int c = 0; c < KR; ++c) ldsm_x4((st + rope_off) ^ (c << 5), w_pe[c]);
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          r_acc[n][x] = 0.f;
#pragma unroll
          for (int k = 0; k < HG; ++k) c_acc[k][n][x] = 0.f;
        }
      // the accumulators in turn, so that no product waits for the one before it
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int k = 0; k < HG; ++k) {
              const uint32_t lo = e ? odd_bytes(w[k][i][2 * c]) : w[k][i][2 * c], hi = e ? odd_bytes(w[k][i][2 * c + 1]) : w[k][i][2 * c + 1];
              const uint32_t lo0 = lo & 0x000F000Fu, hi0 = hi & 0x000F000Fu;
              const uint32_t codes[4] = {lo0, hi0, e ? lo - lo0 : lo & 0x00F000F0u, e ? hi - hi0 : hi & 0x00F000F0u};
#pragma unroll
              for (int n = 0; n < NH; ++n) mma_f16(c_acc[k][n], codes, q[n][8 * k + 4 * i + 2 * c + e][0], q[n][8 * k + 4 * i + 2 * c + e][1]);
            }
#pragma unroll
      for (int c = 0; c < KR; ++c)
#pragma unroll
        for (int n = 0; n < NH; ++n) mma_bf16(r_acc[n], w_pe[c], q_pe[n][c][0], q_pe[n][c][1]);
      // tokens g (own) and g + 8 (the partner's)
      float s[2][HG], z[2][HG];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const char* par = smem + st_at * C::STAGE + C::CODES + C::ROPE + ((8 * (warp ^ t)) + g) * (NG * 8) + half * (HG * 8);
        if constexpr (HG == 2) {
          const float4 v = *reinterpret_cast<const float4*>(par);
          s[t][0] = v.x, z[t][0] = v.y, s[t][1] = v.z, z[t][1] = v.w;
        } else {
          const float2 v = *reinterpret_cast<const float2*>(par);
          s[t][0] = v.x, z[t][0] = v.y;
        }
      }
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        float sum[4] = {r_acc[n][0], r_acc[n][1], r_acc[n][2], r_acc[n][3]};
#pragma unroll
        for (int k = 0; k < HG; ++k) {
          float2 qs;
          if constexpr (NH <= 2) qs = held_sum[k][n];
          else qs = q_sum_of(k, n);
#pragma unroll
          for (int x = 0; x < 4; ++x)
            sum[x] = fmaf(s[x >> 1][k], fmaf(-z[x >> 1][k], x & 1 ? qs.y : qs.x, c_acc[k][n][x]), sum[x]);
        }
        mine_s[n][0] = sum[0], mine_s[n][1] = sum[1];
        sh.swap[pb][warp][n][lane] = make_float2(sum[2], sum[3]);
      }
    };

    // A page's weights.  s_val: the whole scores of the warp's 8 tokens (the thread's: token g) in log2 units.
    float s_val[NH][2], s_tok[NG], z_tok[NG], p_val[NH][2];
    auto join = [&](int st_at, int pb, int p, const float (&own_s)[NH][2]) {
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        const float2 theirs = sh.swap[pb][warp ^ 1][n][lane];
        float2 scale;
        if constexpr (NH <= 2) scale = held_scale[n];
        else scale = scale_of(n);
        s_val[n][0] = (own_s[n][0] + theirs.x) * scale.x;
        s_val[n][1] = (own_s[n][1] + theirs.y) * scale.y;
      }
      const float4* par = reinterpret_cast<const float4*>(smem + st_at * C::STAGE + C::CODES + C::ROPE) + (8 * warp + g) * (NG / 2);
#pragma unroll
      for (int k = 0; k < NG; k += 2) {
        const float4 v = par[k / 2];
        s_tok[k] = v.x, z_tok[k] = v.y, s_tok[k + 1] = v.z, z_tok[k + 1] = v.w;
      }
      const int bad = bad_page[st_at];
      if ((p + 1) * kPage > lim_min || bad) {  // the request's end, or a page that is not there
        const int tok = p * kPage + 8 * warp + g;
        if (tok >= len || bad)
#pragma unroll
          for (int k = 0; k < NG; ++k) s_tok[k] = z_tok[k] = 0.f;
#pragma unroll
        for (int n = 0; n < NH; ++n)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            if (bad || tok >= lim_min + (row0 + 8 * n + 2 * j + x) / a.heads) s_val[n][x] = -INFINITY;
      }
    };

    // Weights against the present references, times each group's scale, to shared memory; true where a
    // weight or a scale has left its reference behind (their sums: moving early does no harm), or is NaN.
    auto weigh = [&](int pb) {
      float weights = 0.f, sizes = 0.f;
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        const float2 m = max_of(n);
        p_val[n][0] = ex2_approx(s_val[n][0] - m.x);
        p_val[n][1] = ex2_approx(s_val[n][1] - m.y);
        weights += p_val[n][0] + p_val[n][1];
      }
      char* dst = pbuf + pb * C::PBUF + p_dst;
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        const float s = s_tok[k] * unit[k];
        sizes += fabsf(s);
#pragma unroll
        for (int n = 0; n < NH; ++n)
          *reinterpret_cast<uint32_t*>(dst + (k * NH + n) * C::PTILE) = pack_half2(p_val[n][0] * s, p_val[n][1] * s);
      }
      return !(weights <= kSlack) || !(sizes <= kScaleSlack);
    };

    // New references: the page's maxima; the sums so far are brought to them.
    auto move_references = [&](int pb) {
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float m = oct_max(s_val[n][x]);
          if (g == 0) sh.red_m[warp][8 * n + 2 * j + x] = m;
        }
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        const float s = oct_max(fabsf(s_tok[k]));
        if (lane == 0) sh.red_s[warp][k] = s;
      }
      work_sync();
      float keep_unit[NG], keep_own = 1.f;
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        float s = 0.f;
        for (int w = 0; w < kWarps; ++w) s = fmaxf(s, sh.red_s[w][k]);
        keep_unit[k] = 1.f;
        if (s * unit[k] > 2.f) {  // bring the largest scale into [1, 2)
          const float u = pow2(min(max(127 - static_cast<int>(__float_as_uint(s) >> 23), -100), 100));
          keep_unit[k] = u / unit[k];
          unit[k] = u;
        }
        if (k == own) keep_own = keep_unit[k];
      }
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        const float2 old = max_of(n);
        float2 m = old;
        for (int w = 0; w < kWarps; ++w) {
          const float2 v = *reinterpret_cast<const float2*>(&sh.red_m[w][8 * n + 2 * j]);
          m.x = fmaxf(m.x, v.x), m.y = fmaxf(m.y, v.y);
        }
        if constexpr (!HELD_MAX) work_sync();  // all have read the old ones
        set_max(n, m);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float keep = ex2_approx(x ? old.y - m.y : old.x - m.x);
          l_sum[n][x] *= keep;
#pragma unroll
          for (int k = 0; k < NG; ++k) zsum[n][x][k] *= keep * keep_unit[k];
#pragma unroll
          for (int c = 0; c < 2 * CH; ++c) acc[c][n][x] *= keep * keep_own, acc[c][n][x + 2] *= keep * keep_own;
        }
      }
      if constexpr (!HELD_MAX) work_sync();
      weigh(pb);
      work_sync();
    };

    // After the references stand: the denominators and the zeros' share.
    auto add_weights = [&]() {
#pragma unroll
      for (int n = 0; n < NH; ++n) l_sum[n][0] += p_val[n][0], l_sum[n][1] += p_val[n][1];
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        const float f = s_tok[k] * unit[k] * z_tok[k];
#pragma unroll
        for (int n = 0; n < NH; ++n)
          zsum[n][0][k] = fmaf(p_val[n][0], f, zsum[n][0][k]), zsum[n][1][k] = fmaf(p_val[n][1], f, zsum[n][1][k]);
      }
    };

    // acc += c^T (P s) over tokens 32 h .. 32 h + 31 of a page, the warp's columns.
    auto gather = [&](int st_at, int pb, int h) {
      const uint32_t st = stages + st_at * C::STAGE + add_off, ps = pbufs + pb * C::PBUF + p_off;
      uint32_t pb_[NH][4], x[CH][4];
#pragma unroll
      for (int c = 0; c < CH; ++c) ldsm_x4_t((st + h * 4096) ^ (c << 4), x[c]);
#pragma unroll
      for (int n = 0; n < NH; ++n) ldsm_x4_t(ps + n * C::PTILE + h * 512, pb_[n]);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          // of four elements e: e0 over e0 + 16 e1, e2 over e2 + 16 e3
          const uint32_t u = x[c][2 * i], v = x[c][2 * i + 1], u8 = odd_bytes(u), v8 = odd_bytes(v);
          const uint32_t even[4] = {u & 0x000F000Fu, u & 0x00FF00FFu, v & 0x000F000Fu, v & 0x00FF00FFu};
          const uint32_t odd[4] = {u8 & 0x000F000Fu, u8, v8 & 0x000F000Fu, v8};
#pragma unroll
          for (int n = 0; n < NH; ++n) mma_f16(acc[2 * c][n], even, pb_[n][2 * i], pb_[n][2 * i + 1]);
#pragma unroll
          for (int n = 0; n < NH; ++n) mma_f16(acc[2 * c + 1][n], odd, pb_[n][2 * i], pb_[n][2 * i + 1]);
        }
    };

    // ---- the pages: tick t scores page t, weighs page t - 1 and adds page t - 2 up ----
    auto after = [](int s, int n) { return s + n >= STAGES ? s + n - STAGES : s + n; };
    int st_score = stage, st_weigh = stage, st_add = stage;
    // A tick of whatever parts it has: the first two and the last.
    auto any_tick = [&](int t) {
      const int pb = t & 1;
      float own_s[NH][2];
#pragma unroll
      for (int n = 0; n < NH; ++n) own_s[n][0] = mine_s[n][0], own_s[n][1] = mine_s[n][1];
      if (t < count) {
        score(st_score, pb);
        st_score = after(st_score, 1);
      }
      if (t >= 2) {
        gather(st_add, pb, 0);
        gather(st_add, pb, 1);
        st_add = after(st_add, 1);
      }
      bool vote = false;
      if (t >= 1) {
        join(st_weigh, pb ^ 1, seg_p + t - 1, own_s);
        st_weigh = after(st_weigh, 1);
        vote = weigh(pb ^ 1);
      }
      if (tick(vote)) move_references(pb ^ 1);
      if (t >= 1) add_weights();
    };
#pragma unroll 1
    for (int t = 0; t <= count; ++t) {
      if (t < 2 || t == count) {
        any_tick(t);
        continue;
      }
      const int pb = t & 1;
      float own_s[NH][2];
#pragma unroll
      for (int n = 0; n < NH; ++n) own_s[n][0] = mine_s[n][0], own_s[n][1] = mine_s[n][1];
      score(st_score, pb);
      gather(st_add, pb, 0);
      gather(st_add, pb, 1);
      join(st_weigh, pb ^ 1, seg_p + t - 1, own_s);
      const bool vote = weigh(pb ^ 1);
      st_score = after(st_score, 1), st_weigh = after(st_weigh, 1), st_add = after(st_add, 1);
      if (tick(vote)) move_references(pb ^ 1);
      add_weights();
    }
    gather(st_add, (count - 1) & 1, 0);
    gather(st_add, (count - 1) & 1, 1);
    stage = st_score;
    done += count;
    // ---- the rows' results ----
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float l = oct_sum(l_sum[n][x]);
        if (g == 0) sh.red_l[warp][8 * n + 2 * j + x] = l;
#pragma unroll
        for (int k = 0; k < NG; ++k) {
          const float z = oct_sum(zsum[n][x][k]);
          if (g == 0) sh.red_z[warp][k][8 * n + 2 * j + x] = z;
        }
      }
    tick(false);
    for (int i = tid; i < ROWS * (NG + 1); i += kWorkers) {
      const int at = i % ROWS, k = i / ROWS - 1;
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) s += k < 0 ? sh.red_l[w][at] : sh.red_z[w][max(k, 0)][at];
      if (k < 0) sh.l_all[at] = s;
      else sh.z_all[k][at] = s;
    }
    work_sync();
    const bool whole = seg_p == 0 && count == seg_pages;
    if (tid == 0 && block == 0 && seg_p == 0) {  // the run that begins a request says how it is cut
      const Runs again(run_total, groups);
      const int64_t page0 = run_begin + (done - count);
      part.cut[seg_b] = whole ? make_int4(0, 0, 0, 0)
                              : make_int4(group, again.holding(page0 + seg_pages - 1) - group + 1, run_begin < page0, 0);
    }
    float u = unit[0];
#pragma unroll
    for (int k = 1; k < NG; ++k) u = own == k ? unit[k] : u;
    const float inv_u = 1.f / u;
    // a cut request's partial: slot 0 where the run begins in (or with) this request, else 1
    const int64_t slot = (static_cast<int64_t>(2 * group + (first ? 0 : 1)) * blocks + block) * ROWS;
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int at = 8 * n + 2 * j + x, row = row0 + at;
        const float l = sh.l_all[at], z = sh.z_all[own][at];
        const float inv = l == 0.f ? 0.f : inv_u / l;
        const float lse = l == 0.f ? -INFINITY : ((x ? max_of(n).y : max_of(n).x) + log2f(l)) * kLn2;
        const bool live = row < rows;
        const int t = live ? row / a.heads : 0, h = live ? row % a.heads : 0;
        uint16_t* out = a.out + seg_b * a.o_sb + t * a.o_st + h * a.o_sh;
        float* out_part = part.o + (slot + at) * D;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const int col = 32 * (warp * CH + c) + 4 * g;
          float v[4];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float even = acc[2 * c + i][n][x], both = acc[2 * c + i][n][x + 2];
            v[2 * i] = fmaf(even, 16777216.f, -z) * inv;
            v[2 * i + 1] = fmaf(both - even, 1048576.f, -z) * inv;
          }
          if (!whole) *reinterpret_cast<float4*>(out_part + col) = make_float4(v[0], v[1], v[2], v[3]);
          else if (live) *reinterpret_cast<uint2*>(out + col) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
        }
        if (warp == 0 && g == 0) {
          if (!whole) part.lse[slot + at] = lse;
          else if (live && a.lse) a.lse[static_cast<int64_t>(seg_b) * rows + row] = lse;
        }
      }

    ++seg_b;
    seg_p = 0;
  }
}

constexpr int kMergeWarps = 8, kMergeThreads = kMergeWarps * 32;

// Joins the partials of the requests that more than one run holds, in the runs' order.  WARPS warps share the
// partials of 128 columns of one row.
template <int D, int WARPS>
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(const DecodeArgs a, const Partials part, const int blocks) {
  constexpr int CHUNKS = D / 128, TASKS = kMergeWarps / WARPS;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, b = blockIdx.y;
  const int task = blockIdx.x * TASKS + warp / WARPS, share = warp % WARPS;
  const int row = task / CHUNKS, col = (task % CHUNKS) * 128 + 4 * lane;
  const bool live = row < a.q_len * a.heads;
  grid_dependency_wait();
  const int4 cut = part.cut[b];
  const int n = cut.y;
  if (n == 0) return;
  auto slot = [&](int i) {
    return (static_cast<int64_t>(2 * (cut.x + i) + (i == 0 ? cut.z : 0)) * blocks + row / part.rows) * part.rows + row % part.rows;
  };
  float top = -INFINITY, den = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (live) {
    bool odd = false;
    for (int i = lane; i < n; i += 32) {
      const float l = part.lse[slot(i)];
      odd |= l != l;
      top = fmaxf(top, l);
    }
    top = warp_max_f32(top);
    if (__any_sync(0xFFFFFFFFu, odd)) top = __int_as_float(0x7FC00000);
#pragma unroll 8
    for (int i = share; i < n; i += WARPS) {
      const float l = part.lse[slot(i)];
      const float4 v = *reinterpret_cast<const float4*>(part.o + slot(i) * D + col);
      const float w = l == -INFINITY ? 0.f : ex2_approx((l - top) * kLog2e);
      den += w;
      acc.x = fmaf(w, v.x, acc.x), acc.y = fmaf(w, v.y, acc.y), acc.z = fmaf(w, v.z, acc.z), acc.w = fmaf(w, v.w, acc.w);
    }
  }
  if constexpr (WARPS > 1) {
    __shared__ float4 red[kMergeWarps][32];
    __shared__ float dens[kMergeWarps];
    red[warp][lane] = acc;
    if (lane == 0) dens[warp] = den;
    __syncthreads();
    if (share != 0) return;
    for (int k = 1; k < WARPS; ++k) {
      const float4 v = red[warp + k][lane];
      acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
      den += dens[warp + k];
    }
  }
  if (!live) return;
  const float inv = den == 0.f ? 0.f : 1.f / den;
  const int t = row / a.heads, h = row % a.heads;
  *reinterpret_cast<uint2*>(a.out + b * a.o_sb + t * a.o_st + h * a.o_sh + col) =
      make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
  if (a.lse && col == 0)
    a.lse[(static_cast<int64_t>(b) * a.q_len + t) * a.heads + h] = den == 0.f ? -INFINITY : top + logf(den);
}

// A CTA's tiles of 8 query rows: as few CTAs as hold them all, evenly filled.
struct Shape {
  int tiles, blocks, groups;  // tiles of a CTA, CTAs for all rows, runs of pages (a CTA each and row block)
};
Shape shape_of(int d, int q_len, int heads) {
  const int tiles = (q_len * heads + 7) / 8, most = d == 512 ? 2 : 5;
  const int blocks = (tiles + most - 1) / most;
  return {(tiles + blocks - 1) / blocks, blocks, std::max(1, sm_count() / blocks)};
}

bool encode(CUtensorMap* map, const void* base, CUtensorMapDataType type, uint64_t width, uint64_t rows,
            uint64_t row_bytes, uint32_t box_width, CUtensorMapSwizzle swizzle) {
  const EncodeTiledFn fn = encode_fn();
  const cuuint64_t dims[2] = {width, rows}, strides[1] = {row_bytes};
  const cuuint32_t box[2] = {box_width, kPage}, step[2] = {1, 1};
  return fn != nullptr && fn(map, type, 2, const_cast<void*>(base), dims, strides, box, step,
                             CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int DR, int NH>
int launch(const DecodeArgs& a, const Shape& shape, cudaStream_t s) {
  using C = Cfg<D, DR, NH>;
  CUtensorMap codes, rope;
  if (!encode(&codes, a.cache.codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, D / 2, a.cache.num_slots, D / 2, 128,
              CU_TENSOR_MAP_SWIZZLE_128B) ||
      !encode(&rope, a.cache.rope, CU_TENSOR_MAP_DATA_TYPE_UINT16, DR, a.cache.num_slots, DR * 2, DR,
              DR == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B))
    return ROLAQ_ECUDA;
  const int blocks = shape.blocks, groups = shape.groups;
  Partials part;
  part.cut = reinterpret_cast<int4*>(static_cast<char*>(a.workspace) + kHeaderBytes);
  part.o = reinterpret_cast<float*>(part.cut + a.batch);
  part.lse = part.o + int64_t(2) * groups * blocks * C::ROWS * D;
  part.rows = C::ROWS;
  static std::atomic<uint64_t> prepared{0};  // devices whose shared-memory limit is raised
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return ROLAQ_ECUDA;
  if (!(prepared.load() >> (device & 63) & 1)) {
    if (cudaFuncSetAttribute(decode_kernel<D, DR, NH>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess)
      return ROLAQ_ECUDA;
    prepared |= uint64_t(1) << (device & 63);
  }
  // Both kernels may start before the one ahead of them in the stream has ended; they wait for it where they
  // first read or write what it may have to do with.
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(groups * blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, decode_kernel<D, DR, NH>, codes, rope, a, part, groups, blocks) != cudaSuccess) return ROLAQ_ECUDA;

  // Few requests are cut into many partials: all warps of a CTA share a row's then.
  const bool wide = groups >= 8 * a.batch;
  const int tasks = a.q_len * a.heads * (D / 128), per_cta = wide ? 1 : kMergeWarps;
  cfg.gridDim = dim3((tasks + per_cta - 1) / per_cta, a.batch);
  cfg.blockDim = dim3(kMergeThreads);
  cfg.dynamicSmemBytes = 0;
  const auto kernel = wide ? merge_kernel<D, kMergeWarps> : merge_kernel<D, 1>;
  return cudaLaunchKernelEx(&cfg, kernel, a, part, blocks) == cudaSuccess ? ROLAQ_OK : ROLAQ_ECUDA;
}

template <int D, int DR>
int launch_tiles(const DecodeArgs& a, cudaStream_t s) {
  const Shape shape = shape_of(D, a.q_len, a.heads);
  if (shape.tiles == 1) return launch<D, DR, 1>(a, shape, s);
  if (shape.tiles == 2) return launch<D, DR, 2>(a, shape, s);
  if constexpr (D == 256) {
    if (shape.tiles == 3) return launch<D, DR, 3>(a, shape, s);
    if (shape.tiles == 4) return launch<D, DR, 4>(a, shape, s);
    return launch<D, DR, 5>(a, shape, s);
  }
  return ROLAQ_EUNSUPPORTED;
}

}  // namespace

int64_t decode_workspace(int batch, int q_len, int heads, int d) {
  const Shape s = shape_of(d, q_len, heads);  // groups * blocks <= sm_count() + blocks; that does not shrink as calls grow
  return kHeaderBytes + int64_t(16) * batch + int64_t(2) * (sm_count() + s.blocks) * s.tiles * 8 * (d + 1) * 4;
}

int launch_decode(const DecodeArgs& a, cudaStream_t s) {
  if (a.cache.latent_dim == 512) return a.cache.rope_dim == 64 ? launch_tiles<512, 64>(a, s) : launch_tiles<512, 32>(a, s);
  return a.cache.rope_dim == 64 ? launch_tiles<256, 64>(a, s) : launch_tiles<256, 32>(a, s);
}

}  // namespace i4
}  // namespace rolaq
