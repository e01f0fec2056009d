// Absorbed attention over the 4-bit latent cache.
//
// With value (c - z) s of a 4-bit code c, per 128-element group g of a token t:
//   q . k_t = sum_g s_gt (q_g . c_gt - z_gt sum q_g) + q_pe . k_pe_t
//   sum_t P_t v_t = sum_t (P_t s_gt) c_gt - sum_t (P_t s_gt) z_gt
// so both contractions run on the raw codes, which become operands by ANDs:
//   - scores: the E4M3 patterns 0..15 are c 2^-9 exactly.  tcgen05.mma of 128 tokens (codes in TMEM) by the query rows
//     in two E4M3 terms each (hi + lo: with the row's largest element in [2^7, 2^8) and steps of 2^-9 at the lower end, BF16
//     within 2^9 of that element is exact, what lies below is off by up to 2^-17 of it), one FP32 sum a group; the rotary
//     part BF16 by BF16.  Asynchronous: no warp's issue slots go into it.
//   - sums: the FP16 patterns 0..255 are that many 2^-24 exactly.  mma.sync m16n8k16 with the codes as rows (c of an
//     even element, and c + 16 c' of it and the next: c' comes out at the end) and P s in FP16 as columns.
// All sums are FP32, and so is the zeros' share.
//
// FP16 holds P s to 11 bits from 2^-14 to 2^16 only, so it is held relative to the largest P s that a row has met in a group:
// a group's unit follows the largest scale, which is enough while each row gives weight to tokens of about that scale.
// Where the references move, and the scales do not already say that each row has met a P s unit of 2 in each group, the
// rows' largest are taken too, and a row that has not met that much in a group (its tokens' scales are far below
// others') gets a power of two of its own there; while one is in use, each tile goes that way.  Equal elements are stored
// with scale 1 and codes 0: they add nothing but their zero's share, and their scale is not taken for a size.
//
// A CTA holds NH tiles of 8 query rows (query tokens x heads; up to two for D = 512, five for D = 256) and walks the
// pages of one or more requests, two (a tile of 128 tokens) at a time:
//   - two loading warps bring codes with params, and rotary parts, by TMA (128-byte swizzle);
//   - eight token warps, two threads a token: codes to TMEM (a tile ahead), scores from TMEM, the softmax against
//     references that move only when weights pass them by 2^10, P s of each group to shared memory.  A vote a tile
//     moves the references; a move leaves the factors for the sums beside the weights;
//   - one warp issues the tcgen05 products of a tile as soon as its codes are there;
//   - eight adding warps hold D/8 latent columns of the result each.
// The roles meet in mbarriers only.  The pages of all requests are dealt to the CTAs in one equal run each (a run may
// begin or end inside a request); what is cut is joined by merge_kernel by log-sum-exp.
//
// Measured, 16 heads of 512 + 64, 64 requests of about 16K tokens (417 MB): 137 to 142 us, 3.0 TB/s, 45 to 47% of a copy's
// rate (290 while a row of each request has a factor of its own, 340 with a row of zeros among small latents in each tile).  What
// bounds it is the schedulers: a tile costs each of them about 2000 instructions and 128 mma.sync, and an mma.sync holds
// back all else for 8 cycles (HMMA + n logic + m FP32 instructions measured 8 + 0.9 n + 1.2 m cycles), 2900 of the 3900
// cycles a tile takes; memory alone would take 2050.  With the scores on mma.sync too it was 160 us.  Slower, where this
// took 135: four warps more that only bring codes (179), the adding warps bringing them (166), sharing that (152); one
// thread of a divergent branch issuing (167: 2000 cycles for 20 products, against 300 by an elected lane of a warp whose
// operands are the same in all lanes).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "int4.cuh"
#include "kernels.cuh"

namespace rolaq {
namespace i4 {
namespace {

// Warps 0..7 are the token warps, 8..15 the adding ones, 16 and 17 load, 18 issues.  Of the 96 registers a thread that a
// block of 640 is launched with, the others hand some to the token warps.
constexpr int kTokenWarps = 8, kAddWarps = 8;
constexpr int kTokens = kTokenWarps * 32, kAdders = kAddWarps * 32, kThreads = kTokens + kAdders + 128;
constexpr int kAhead = 4;         // pages ahead of their loads that they are called to L2 (24: 157 us against 144, single calls)
// The least run of pages worth a CTA of its own (a tile), unless the requests are shorter: 31 of 20 tokens, 4 query tokens of
// 40 heads of 256, are 10 us faster with a request a CTA than with two (40 us against 50, single calls).
constexpr int kMinPages = 2;
// Scales are brought into [2^3, 2^4); weights and scales may pass their references until P s is 2^15.
constexpr float kSlack = 1024.f, kScaleTop = 16.f, kScaleSlack = 32.f;
constexpr float kLeast = 2.f;       // the least of a row's largest P s unit that needs no factor of the row's own
constexpr float kZeroShare = 9.094947017729282e-13f;  // 2^-40: a scale below this share of its value's size counts as that much
constexpr float kNoMax = -3.402823466e38f, kNoUnit = 1.329227995784916e36f;  // references not yet set: the first token passes them
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <int D, int DR, int NH>
struct Cfg {
  static constexpr int NG = D / kGroup;             // groups of a token
  static constexpr int CODES = kPage * D / 2, ROPE = kPage * DR * 2, PARAMS = kPage * NG * 8;  // of a page
  static constexpr int PAGES = D == 512 ? 8 : 12;   // a ring of pages' codes and params
  static constexpr int TILES = 2;                   // one of tiles' rotary parts, which only the scores need
  static constexpr int WEIGHTS = 3;                 // and one of pages' P s: a tile's first is written while the last one's second is in use
  static constexpr int ROWS = 8 * NH;
  static constexpr int NQ = (ROWS + 15) / 16 * 16;  // columns of the scores' products
  static constexpr int QB_GROUP = NQ * 128, QB = 2 * NG * QB_GROUP, QPE = NQ * DR * 2;  // hi of all groups, lo of all groups
  static constexpr int PTILE = kPage * 16;          // P s of a page, a group and 8 rows: [token][row] FP16
  static constexpr int PBUF = NG * NH * PTILE;
  // swizzled tiles first, on 1024-byte boundaries; the pages' params apart
  static constexpr int OFF_ROPE = PAGES * CODES, OFF_QB = OFF_ROPE + TILES * 2 * ROPE, OFF_QPE = OFF_QB + QB;
  static constexpr int OFF_P = OFF_QPE + QPE, OFF_PARAMS = OFF_P + WEIGHTS * PBUF;
  static constexpr int SMEM = 1024 + OFF_PARAMS + PAGES * PARAMS;
  static constexpr int CH = D / kAddWarps / 32;     // 32-column chunks that an adding warp holds
  static constexpr int HT = (NH + 1) / 2;           // tiles of 8 rows of a token thread
  // TMEM columns: two tiles' codes; two tiles' scores (the groups' sums, the rotary part's)
  static constexpr int T_CODES = D / 4, T_SUM = 2 * T_CODES, T_ROPE = NG * NQ, T_TILE = (NG + 1) * NQ;
  static constexpr int TOKEN_REGS = NH < 5 ? 136 : 144, ADD_REGS = 80, LOAD_REGS = NH < 5 ? 48 : 32;
  static_assert(T_SUM + 2 * T_TILE <= 512 && 2 * TOKEN_REGS + 2 * ADD_REGS + LOAD_REGS <= 5 * 96, "TMEM, registers");
};

template <int NG, int NH>
struct alignas(16) Shared {  // rows are read two at a time
  float red_m[4][8 * NH], red_s[4][NG], red_w[4][NG * 8 * NH];  // by quarters of the tile's tokens
  float keep[3][NG][8 * NH];                              // factors for the sums before tile i (at i % 3), where moved[i % 3]
  float keep_row[8 * NH], keep_unit[NG];                  // the parts of the last ones
  float max[8 * NH], q_sum[NG][8 * NH], row_scale[8 * NH];
  float met[NG * 8 * NH], factor[NG][8 * NH];             // a row's largest P s unit in a group, as of the last move; its own factor
  float l[4][8 * NH], z[4][NG][8 * NH], max_out[8 * NH], unit_out[NG], factor_out[NG * 8 * NH];  // of a finished request (1 / factor)
  int moved[3];
};

// Named barriers: the token warps; a request's sums are written / have been taken.
constexpr int kBarToken = 1, kBarSums = 2, kBarTaken = 3;
__device__ __forceinline__ void token_sync() { named_bar_sync(kBarToken, kTokens); }
__device__ __forceinline__ bool token_any(bool vote) {
  int any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %3, 0;\n\tbar.red.or.pred q, %1, %2, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "n"(kBarToken), "n"(kTokens), "r"(static_cast<int>(vote))
      : "memory");
  return any != 0;
}
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ void bar_arrive(int id, int threads) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Two FP32 operations an instruction, each rounded like the plain one.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(d)
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)), "l"(*reinterpret_cast<uint64_t*>(&c)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
// Eight values summed over the warp: lane l gets the sum of value l % 8.
__device__ __forceinline__ float warp_sums(const float2 (&pairs)[4]) {
  const int lane = threadIdx.x & 31;
  float v[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[2 * i] = pairs[i].x, v[2 * i + 1] = pairs[i].y;
#pragma unroll
  for (int h = 4; h >= 1; h /= 2) {
    const bool up = lane & h;
#pragma unroll
    for (int i = 0; i < h; ++i) v[i] = (up ? v[i + h] : v[i]) + __shfl_xor_sync(0xFFFFFFFFu, up ? v[i] : v[i + h], h);
  }
  v[0] += __shfl_xor_sync(0xFFFFFFFFu, v[0], 8);
  return v[0] + __shfl_xor_sync(0xFFFFFFFFu, v[0], 16);
}

__device__ __forceinline__ int pages_of(const DecodeArgs& a, int b) {
  const int64_t len = min(static_cast<int64_t>(a.seq_lens[b]), static_cast<int64_t>(a.max_pages) * kPage);
  return len <= 0 ? 0 : static_cast<int>((len + kPage - 1) / kPage);
}

// Runs are equal shares of the `total` pages: run r of n begins at page total * r / n.
struct Runs {
  int64_t total;
  int n;
  __device__ Runs(int64_t total_, int batch, int groups) : total(total_) {
    const int64_t most = max((total + kMinPages - 1) / kMinPages, min(total, static_cast<int64_t>(batch)));
    n = static_cast<int>(min(static_cast<int64_t>(groups), max(int64_t(1), most)));
  }
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
// Bytes 1 and 3 as 16-bit halves.
__device__ __forceinline__ uint32_t odd_bytes(uint32_t w) { return prmt(w, 0u, 0x4341u); }
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The shared-memory offset of 16-byte chunk `chunk` of row `row` under TMA's swizzles.
__device__ __forceinline__ uint32_t sw128(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }
__device__ __forceinline__ uint32_t sw64(int row, int chunk) { return row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4); }

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
  constexpr int NG = C::NG, CH = C::CH, PAGES = C::PAGES, TILES = C::TILES, ROWS = C::ROWS, HT = C::HT;
  extern __shared__ char raw[];
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  // a page's codes loaded / added; a tile's rotary part loaded / used; its codes in TMEM, its scores there, they are taken,
  // its weights in shared memory; the request's query there
  __shared__ uint64_t full[PAGES], page_free[PAGES], rope_full[TILES], rope_free[TILES], coded[2], scored[2], taken[2], weighed[3], q_ready;
  __shared__ int bad_page[PAGES];
  __shared__ int64_t scan[kThreads / 32];
  __shared__ int start[2];
  __shared__ uint32_t tmem_slot;
  __shared__ Shared<NG, NH> sh;

  const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid / 32, 0), lane = tid & 31;
  const int block = blockIdx.x % blocks, group = blockIdx.x / blocks;
  const int rows = a.q_len * a.heads, row0 = block * ROWS;
  if (tid == 0) {
    for (int s = 0; s < PAGES; ++s) mbar_init(&full[s], 1), mbar_init(&page_free[s], kAddWarps);
    for (int s = 0; s < TILES; ++s) mbar_init(&rope_full[s], 1), mbar_init(&rope_free[s], 1);
    for (int s = 0; s < 2; ++s) mbar_init(&coded[s], kTokenWarps), mbar_init(&scored[s], 1), mbar_init(&taken[s], kTokenWarps);
    for (int s = 0; s < 3; ++s) mbar_init(&weighed[s], 1);
    mbar_init(&q_ready, 1);
    fence_mbar_init();
    prefetch_tensormap(&map_codes);
    prefetch_tensormap(&map_rope);
  }
  if (warp == 0) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
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
  const Runs runs(total, a.batch, groups);
  if (group >= runs.n || total == 0) {
    if (warp == 0) tmem_dealloc(tmem_slot, 512);
    return;
  }
  const int64_t u0 = runs.begin(group);
  const int n_units = static_cast<int>(runs.begin(group + 1) - u0);
  if (before <= u0 && u0 < before + mine) {
    int b = tid * per;
    for (int n; before + (n = pages_of(a, b)) <= u0; ++b) before += n;
    start[0] = b;
    start[1] = static_cast<int>(u0 - before);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, tmem_slot, 0);
  int seg_b = start[0], seg_p = start[1];
  // A wait that ran out of time is reported; the role goes on without waiting, so that all barriers are met.
  bool healthy = true;
  auto wait_for = [&](uint64_t* bar, int phase) {
    if (healthy) healthy = mbar_wait(bar, phase & 1, a.err);
  };

  if (tid >= kTokens + kAdders) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::LOAD_REGS));
    constexpr int first_warp = kTokenWarps + kAddWarps;
    if (warp <= first_warp + 1) {
      // ================= the loading warps: codes and params by pages; rotary parts by tiles =================
      // Lane l holds the id of page l of 32; the next 32 are requested 32 pages ahead of their use.
      const bool codes = warp == first_warp;
      const int pool_pages = static_cast<int>(a.cache.num_slots / kPage);
      int id_b = seg_b, id_p = seg_p + lane, ids = -1, next_ids = -1;
      auto fetch_ids = [&](int first) {
        int id = -1;
        if (first + lane < n_units) {
          for (int n; id_p >= (n = pages_of(a, id_b)); ++id_b) id_p -= n;
          id = a.page_table[id_b * a.pt_stride + id_p];
        }
        id_p += 32;
        return id;
      };
      next_ids = fetch_ids(0);
      int slot = 0, lap = 0, left = 0, in_tile = 0;  // pages left of the present request, and its page modulo 2
      for (int i = 0; i < n_units; ++i) {
        if ((i & 31) == 0) {
          ids = next_ids;
          next_ids = fetch_ids(i + 32);
        }
        const int id = __shfl_sync(0xFFFFFFFFu, ids, i & 31);
        const bool ok = id >= 0 && id < pool_pages;
        const int page = ok ? id : 0;
        // The rings are short of covering the way from memory: pages come to L2 ahead of them.
        const int ahead_id = __shfl_sync(0xFFFFFFFFu, (i & 31) + kAhead < 32 ? ids : next_ids, (i + kAhead) & 31);
        if (lane == 1 && i + kAhead < n_units && ahead_id >= 0 && ahead_id < pool_pages) {
          const int64_t token = static_cast<int64_t>(ahead_id) * kPage;
          if (codes) {
            prefetch_l2(a.cache.codes + token * (D / 2), C::CODES);
            prefetch_l2(a.cache.params + token * (NG * 2), C::PARAMS);
          } else {
            prefetch_l2(a.cache.rope + token * DR, C::ROPE);
          }
        }
        if (codes) {
          if (lap > 0) wait_for(&page_free[slot], lap - 1);
          if (lane == 0) {
            uint64_t* bar = &full[slot];
            bad_page[slot] = !ok;
            if (!ok) report(a.err, ROLAQ_DEV_BAD_PAGE);
            mbar_expect_tx(bar, C::CODES + C::PARAMS);
#pragma unroll
            for (int k = 0; k < D / 256; ++k)
              tma_load_2d(smem + slot * C::CODES + k * 8192, &map_codes, bar, k * 128, page * kPage);
            bulk_load(smem + C::OFF_PARAMS + slot * C::PARAMS, a.cache.params + static_cast<int64_t>(page) * (kPage * NG * 2),
                      C::PARAMS, bar);
          }
          if (++slot == PAGES) slot = 0, ++lap;
        } else {
          if (left == 0) {
            for (; pages_of(a, seg_b) - seg_p <= 0; seg_p = 0) ++seg_b;
            left = min(pages_of(a, seg_b) - seg_p, n_units - i);
            ++seg_b;
            seg_p = 0;
            in_tile = 0;
          }
          if (in_tile == 0) {
            if (lap > 0) wait_for(&rope_free[slot], lap - 1);
            if (lane == 0) mbar_expect_tx(&rope_full[slot], (left > 1 ? 2 : 1) * C::ROPE);
          }
          if (lane == 0) tma_load_2d(smem + C::OFF_ROPE + (2 * slot + in_tile) * C::ROPE, &map_rope, &rope_full[slot], 0, page * kPage);
          in_tile ^= 1, --left;
          if (in_tile == 0 || left == 0)
            if (++slot == TILES) slot = 0, ++lap;
        }
      }
    } else if (warp == first_warp + 2) {
      // ================= the issuing warp: scores of tile i = codes (TMEM) x query, rope x query =================
      // One lane issues; the others go along, so that all its operands are known to be the same in all lanes.
      constexpr uint32_t id_qk = idesc_e4m3(128, C::NQ, 0, 0), id_pe = idesc_bf16(128, C::NQ);
      const uint64_t d_q = sw128_kmajor_desc(smem_u32(smem + C::OFF_QB));
      const uint64_t d_qp = DR == 64 ? sw128_kmajor_desc(smem_u32(smem + C::OFF_QPE)) : sw64_kmajor_desc(smem_u32(smem + C::OFF_QPE));
      int tile = 0, queries = 0;
      for (int done = 0; done < n_units; ++seg_b, seg_p = 0) {
        const int count = min(pages_of(a, seg_b) - seg_p, n_units - done);
        if (count <= 0) continue;
        wait_for(&q_ready, queries++);
        for (int p = 0; p < count; p += 2, ++tile) {
          wait_for(&rope_full[tile & 1], tile >> 1);
          wait_for(&coded[tile & 1], tile >> 1);
          if (tile >= 2) wait_for(&taken[tile & 1], (tile >> 1) - 1);
          __syncwarp();
          tc_fence_after();
          const uint32_t codes = tmem + (tile & 1) * C::T_CODES, sums = tmem + C::T_SUM + (tile & 1) * C::T_TILE;
          const uint32_t rope = smem_u32(smem + C::OFF_ROPE + (tile & 1) * 2 * C::ROPE);
          const uint64_t d_k = DR == 64 ? sw128_kmajor_desc(rope) : sw64_kmajor_desc(rope);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < NG; ++k)
#pragma unroll
              for (int m = 0; m < 8; ++m)  // hi, then lo
                umma_f8_ts(sums + k * C::NQ, codes + 32 * k + 8 * (m & 3),
                           d_q + static_cast<uint64_t>((C::QB_GROUP >> 4) * (k + (m >> 2) * NG) + 2 * (m & 3)), id_qk, m > 0);
#pragma unroll
            for (int m = 0; m < DR / 16; ++m) umma_bf16_ss(sums + C::T_ROPE, d_k + 2 * m, d_qp + 2 * m, id_pe, m > 0);
            umma_commit(&scored[tile & 1]);
            umma_commit(&rope_free[tile & 1]);
          }
          __syncwarp();
        }
        done += count;
      }
    } else if (block == 0) {
      // ================= the run that begins a request says how it is cut =================
      for (int done = 0; done < n_units; ++seg_b, seg_p = 0) {
        const int pages = pages_of(a, seg_b), count = min(pages - seg_p, n_units - done);
        if (count <= 0) continue;
        const int64_t page0 = u0 + done;
        if (seg_p == 0 && lane == 0)
          part.cut[seg_b] = count == pages ? make_int4(0, 0, 0, 0)
                                           : make_int4(group, runs.holding(page0 + pages - 1) - group + 1, u0 < page0, 0);
        done += count;
      }
    }
    if (!healthy) __nanosleep(1000000);  // what is under way to shared memory arrives before the CTA's end
    __syncwarp();
  } else if (tid >= kTokens) {
    // ================= adding warps: D / 8 latent columns each =================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::ADD_REGS));
    const int w = warp - kTokenWarps, g = lane >> 2, j = lane & 3;
    const int own = w * NG / kAddWarps;  // the group of the warp's columns
    // Offsets of the lane's ldmatrix rows from a 1024-byte boundary.  Chunk c of a row lies at c ^ row % 8, so
    // chunk c ^ x is at the address ^ 16 x.
    const uint32_t add_off = (w * CH / 8) * 8192 + sw128(lane, (w * CH) & 7);
    const uint32_t base = smem_u32(smem), p_base = base + C::OFF_P + own * (NH * C::PTILE) + lane * 16;
    int done = 0, turn = 0, lap = 0, slot = 0, p_slot = 0;  // tiles % 3, / 3; pages % PAGES, % 3
    while (done < n_units) {
      const int seg_pages = pages_of(a, seg_b);
      if (seg_pages == 0) {
        ++seg_b;
        continue;
      }
      const bool first = done == 0;
      const int count = min(seg_pages - seg_p, n_units - done);
      // accumulators: tile 2 c + h of chunk c holds columns 4 g + 2 h (and that + 16 times the next one) x rows 2 j, + 1
      float acc[2 * CH][NH][4];
#pragma unroll
      for (int c = 0; c < 2 * CH; ++c)
#pragma unroll
        for (int n = 0; n < NH; ++n) acc[c][n][0] = acc[c][n][1] = acc[c][n][2] = acc[c][n][3] = 0.f;
      for (int p = 0; p < count; p += 2) {
        wait_for(&weighed[turn], lap);
        __syncwarp();
        if (sh.moved[turn]) {
#pragma unroll
          for (int n = 0; n < NH; ++n) {
            const float2 k = *reinterpret_cast<const float2*>(&sh.keep[turn][own][8 * n + 2 * j]);
#pragma unroll
            for (int c = 0; c < 2 * CH; ++c) {
              acc[c][n][0] *= k.x, acc[c][n][2] *= k.x;
              acc[c][n][1] *= k.y, acc[c][n][3] *= k.y;
            }
          }
        }
#pragma unroll 1
        for (int i = 0; i < min(2, count - p); ++i) {
          const uint32_t st = base + slot * C::CODES + add_off, ps = p_base + p_slot * C::PBUF;
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // 32 tokens
            uint32_t x[CH][4], pf[NH][4];
#pragma unroll
            for (int c = 0; c < CH; ++c) ldsm_x4_t((st + h * 4096) ^ (c << 4), x[c]);
#pragma unroll
            for (int n = 0; n < NH; ++n) ldsm_x4_t(ps + n * C::PTILE + h * 512, pf[n]);
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
              for (int c = 0; c < CH; ++c) {
                // of four elements e: e0 over e0 + 16 e1, e2 over e2 + 16 e3
                const uint32_t u = x[c][2 * k], v = x[c][2 * k + 1], u8 = odd_bytes(u), v8 = odd_bytes(v);
                const uint32_t even[4] = {u & 0x000F000Fu, u & 0x00FF00FFu, v & 0x000F000Fu, v & 0x00FF00FFu};
                const uint32_t odd[4] = {u8 & 0x000F000Fu, u8, v8 & 0x000F000Fu, v8};
#pragma unroll
                for (int n = 0; n < NH; ++n) mma_f16(acc[2 * c][n], even, pf[n][2 * k], pf[n][2 * k + 1]);
#pragma unroll
                for (int n = 0; n < NH; ++n) mma_f16(acc[2 * c + 1][n], odd, pf[n][2 * k], pf[n][2 * k + 1]);
              }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&page_free[slot]);
          if (++slot == PAGES) slot = 0;
          if (++p_slot == C::WEIGHTS) p_slot = 0;
        }
        if (++turn == 3) turn = 0, ++lap;
      }
      done += count;
      // ---- the rows' results ----
      named_bar_sync(kBarSums, kTokens + kAdders);
      const bool whole = seg_p == 0 && count == seg_pages;
      const float inv_u = 1.f / sh.unit_out[own];
      // a cut request's partial: slot 0 where the run begins in (or with) this request, else 1
      const int64_t slot = (static_cast<int64_t>(2 * group + (first ? 0 : 1)) * blocks + block) * ROWS;
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int at = 8 * n + 2 * j + x, row = row0 + at;
          float l = 0.f, z = 0.f;
#pragma unroll
          for (int k = 0; k < 4; ++k) l += sh.l[k][at], z += sh.z[k][own][at];
          const float inv = l == 0.f ? 0.f : inv_u / l, inv_f = sh.factor_out[own * ROWS + at];
          const float lse = l == 0.f ? -INFINITY : (sh.max_out[at] + log2f(l)) * kLn2;
          const bool live = row < rows;
          const int t = live ? row / a.heads : 0, h = live ? row % a.heads : 0;
          uint16_t* out = a.out + seg_b * a.o_sb + t * a.o_st + h * a.o_sh;
          float* out_part = part.o + (slot + at) * D;
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            const int col = 32 * (w * CH + c) + 4 * g;
            float v[4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float even = acc[2 * c + i][n][x], sum = acc[2 * c + i][n][x + 2];
              v[2 * i] = fmaf(even, 16777216.f * inv_f, -z) * inv;
              v[2 * i + 1] = fmaf(sum - even, 1048576.f * inv_f, -z) * inv;
            }
            if (!whole) *reinterpret_cast<float4*>(out_part + col) = make_float4(v[0], v[1], v[2], v[3]);
            else if (live) *reinterpret_cast<uint2*>(out + col) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
          }
          if (w == 0 && g == 0) {
            if (!whole) part.lse[slot + at] = lse;
            else if (live && a.lse) a.lse[static_cast<int64_t>(seg_b) * rows + row] = lse;
          }
        }
      bar_arrive(kBarTaken, kTokens + kAdders);
      ++seg_b;
      seg_p = 0;
    }
  } else {
    // ================= token warps: thread (token of the tile, half of the columns and of the rows) =================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::TOKEN_REGS));
    const int quarter = warp & 3, half = warp >> 2, token = 32 * quarter + lane;
    const int n0 = half * HT, my_tiles = half == 0 ? HT : NH - HT;  // tiles of 8 rows
    const uint32_t lanes = static_cast<uint32_t>(32 * quarter) << 16;
    const float qk_scale = a.sm_scale * kLog2e;
    const char* token_params = smem + C::OFF_PARAMS + (token & 63) * (NG * 8);
    int done = 0, tile = 0, turn = 0;  // turn: tiles % 3
    bool begun = false;

    // The codes of tile `to` as E4M3 bytes to TMEM: of each word of 8 the even elements, then the odd ones; the thread has
    // half the columns of a token.  `page`: its page, counted over the run.
    const char* token_codes = smem + (D == 512 ? half * 8192 : 0) + (token & 63) * 128;
    auto bring_codes = [&](int to, int page) {
      const int at = page % PAGES;
      wait_for(&full[at], page / PAGES);
      __syncwarp();
      const uint32_t dst = tmem + lanes + (to & 1) * C::T_CODES + half * (D / 8);
      const char* src = token_codes + at * C::CODES;
#pragma unroll
      for (int c0 = 0; c0 < D / 64; c0 += 4) {
        uint4 v[4];
#pragma unroll
        for (int c = 0; c < 4; ++c)
          v[c] = *reinterpret_cast<const uint4*>(src + ((((D == 512 ? 0 : 4 * half) + c0 + c) ^ (token & 7)) << 4));
#pragma unroll
        for (int c = 0; c < 4; c += 2) {
          const uint32_t x[8] = {v[c].x, v[c].y, v[c].z, v[c].w, v[c + 1].x, v[c + 1].y, v[c + 1].z, v[c + 1].w};
          uint32_t r[16];
#pragma unroll
          for (int k = 0; k < 8; ++k) r[2 * k] = x[k] & 0x0F0F0F0Fu, r[2 * k + 1] = (x[k] >> 4) & 0x0F0F0F0Fu;
          tmem_st16(dst + 8 * (c0 + c), r);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&coded[to & 1]);
    };
    // The page of the thread's token of a tile that begins with `page` and has n (where there is no second, the first).
    auto own_page = [&](int page, int n) { return page + (token >= kPage && n > 1); };

    while (done < n_units) {
      const int seg_pages = pages_of(a, seg_b);
      if (seg_pages == 0) {
        ++seg_b;
        continue;
      }
      const int count = min(seg_pages - seg_p, n_units - done);
      const int len = min(static_cast<int64_t>(a.seq_lens[seg_b]), static_cast<int64_t>(a.max_pages) * kPage);
      if (tid == 0 && len != a.seq_lens[seg_b]) report(a.err, ROLAQ_DEV_BAD_REQ);
      const int lim_min = len - a.q_len + 1;

      // ---- the query: a row a warp at a time; the last tile's products are done with the one before ----
#pragma unroll 1
      for (int r = warp; r < C::NQ; r += kTokenWarps) {
        const int row = row0 + r;
        const bool live = r < ROWS && row < rows;
        const int t = live ? row / a.heads : 0, h = live ? row % a.heads : 0;
        const uint16_t* src = a.q + seg_b * a.q_sb + t * a.q_st + h * a.q_sh;
        // lane: words (8 elements) lane and, for D = 512, lane + 32
        uint4 w[D / 256], pe = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < D / 256; ++i) w[i] = live ? *reinterpret_cast<const uint4*>(src + 8 * (lane + 32 * i)) : pe;
        if (live && lane < DR / 8) pe = *reinterpret_cast<const uint4*>(src + D + 8 * lane);
        if (lane < DR / 8) {
          const uint32_t off = DR == 64 ? (r >> 3) * 1024 + sw128(r & 7, lane) : (r >> 3) * 512 + sw64(r & 7, lane);
          *reinterpret_cast<uint4*>(smem + C::OFF_QPE + off) = pe;
        }
        if (r >= ROWS) continue;
        float top = 0.f, odd = 0.f;
#pragma unroll
        for (int i = 0; i < D / 256; ++i) {
          const uint32_t v[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            top = fmaxf(top, fmaxf(fabsf(bf16_lo(v[k])), fabsf(bf16_hi(v[k]))));
            odd = fmaf(bf16_lo(v[k]), 0.f, fmaf(bf16_hi(v[k]), 0.f, odd));  // NaN where an element is no finite number
          }
        }
        // The rotary part (0 in the lanes that have none of it): its products alone could be all -inf, a row that sees nothing.
        uint32_t odd_pe = 0;
        for (const uint32_t v : {pe.x, pe.y, pe.z, pe.w}) asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(odd_pe) : "r"(v), "r"(0u));
        const bool no_row = __any_sync(0xFFFFFFFFu, (odd_pe & 0x7FFF7FFFu) != 0);
        top = warp_max_f32(odd != 0.f ? INFINITY : top);
        // 2^k with top 2^k in [2^7, 2^8), at most 2^100: scores of smaller rows stay normal numbers in row_scale
        const float up = top > 0.f ? pow2(min(max(7 - (static_cast<int>(__float_as_uint(top) >> 23) - 127), -120), 100)) : 1.f;
        if (lane == 0) sh.row_scale[r] = top == INFINITY || no_row ? __int_as_float(0x7FC00000) : (qk_scale * 512.f) / up;
#pragma unroll
        for (int i = 0; i < D / 256; ++i) {
          const uint32_t v[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
          uint32_t hi[2], lo[2];  // even elements, odd elements
          float sum = 0.f;
          float x[8];
#pragma unroll
          for (int k = 0; k < 4; ++k) x[2 * k] = bf16_lo(v[k]) * up, x[2 * k + 1] = bf16_hi(v[k]) * up;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t h0 = f32x2_to_e4m3x2(x[e], x[e + 2]), h1 = f32x2_to_e4m3x2(x[e + 4], x[e + 6]);
            const float2 f0 = __half22float2(e4m3x2_to_half2(h0)), f1 = __half22float2(e4m3x2_to_half2(h1));
            const uint32_t l0 = f32x2_to_e4m3x2(x[e] - f0.x, x[e + 2] - f0.y), l1 = f32x2_to_e4m3x2(x[e + 4] - f1.x, x[e + 6] - f1.y);
            const float2 s0 = __half22float2(e4m3x2_to_half2(l0)), s1 = __half22float2(e4m3x2_to_half2(l1));
            sum += ((f0.x + s0.x) + (f0.y + s0.y)) + ((f1.x + s1.x) + (f1.y + s1.y));
            hi[e] = h0 | h1 << 16, lo[e] = l0 | l1 << 16;
          }
          const int word = lane + 32 * i, k = word / 16, at = word % 16;  // 8 bytes of the group's 128
          char* dst = smem + C::OFF_QB + k * C::QB_GROUP + (r >> 3) * 1024 + sw128(r & 7, at >> 1) + 8 * (at & 1);
          *reinterpret_cast<uint2*>(dst) = make_uint2(hi[0], hi[1]);
          *reinterpret_cast<uint2*>(dst + NG * C::QB_GROUP) = make_uint2(lo[0], lo[1]);
#pragma unroll
          for (int o = 1; o < 16; o *= 2) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
          if ((lane & 15) == 0) sh.q_sum[k][r] = sum * (1.f / 512.f);
        }
      }
      if (tid < ROWS) sh.max[tid] = kNoMax;
      if (tid < NG * ROWS) sh.met[tid] = 0.f, sh.factor[0][tid] = 1.f;
      fence_proxy_async();
      token_sync();
      if (tid == 0) mbar_arrive(&q_ready);

      float2 l_sum[HT][4], zsum[NG][HT][4];
      float unit[NG];
#pragma unroll
      for (int n = 0; n < HT; ++n)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          l_sum[n][x] = both(0.f);
#pragma unroll
          for (int k = 0; k < NG; ++k) zsum[k][n][x] = both(0.f);
        }
#pragma unroll
      for (int k = 0; k < NG; ++k) unit[k] = kNoUnit;
      bool factors = false;  // a row has a factor of its own, or has met nothing yet
      const int tiles = (count + 1) / 2;
      bring_codes(tile, own_page(done, count));
      for (int i = 0; i < tiles; ++i, ++tile) {
        const int n_pages = min(2, count - 2 * i), page = own_page(done + 2 * i, n_pages), at = page % PAGES;
        const bool here = (token >> 6) < n_pages;
        if (i + 1 < tiles) bring_codes(tile + 1, own_page(done + 2 * i + 2, count - 2 * i - 2));
        float s_tok[NG], z_tok[NG];
        {
          const float4* par = reinterpret_cast<const float4*>(token_params + at * C::PARAMS);
#pragma unroll
          for (int k = 0; k < NG; k += 2) {
            const float4 v = par[k / 2];
            s_tok[k] = v.x, z_tok[k] = v.y, s_tok[k + 1] = v.z, z_tok[k + 1] = v.w;
          }
        }
        // ---- scores of the thread's rows, in log2 units ----
        wait_for(&scored[tile & 1], tile >> 1);
        __syncwarp();
        tc_fence_after();
        float2 s_val[HT][4];
        const uint32_t sums = tmem + lanes + C::T_SUM + (tile & 1) * C::T_TILE + 8 * n0;
#pragma unroll
        for (int n = 0; n < HT; ++n)
          if (n < my_tiles) {
            uint32_t pe[8];
            float2 sum[4] = {both(0.f), both(0.f), both(0.f), both(0.f)};
#pragma unroll
            for (int k0 = 0; k0 < NG; k0 += 2) {
              uint32_t d[2][8];
              tmem_ld8(sums + k0 * C::NQ + 8 * n, d[0]);
              tmem_ld8(sums + (k0 + 1) * C::NQ + 8 * n, d[1]);
              if (k0 == 0) tmem_ld8(sums + C::T_ROPE + 8 * n, pe);
              tmem_wait_ld();
              reg_fence(d[0]);
              reg_fence(d[1]);
              if (k0 == 0) reg_fence(pe);
#pragma unroll
              for (int k = k0; k < k0 + 2; ++k)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                  const float2 dot = make_float2(__uint_as_float(d[k - k0][2 * x]), __uint_as_float(d[k - k0][2 * x + 1]));
                  const float2 qs = *reinterpret_cast<const float2*>(&sh.q_sum[k][8 * (n0 + n) + 2 * x]);
                  sum[x] = fma2(both(s_tok[k]), fma2(both(-z_tok[k]), qs, dot), sum[x]);
                }
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const float2 scale = *reinterpret_cast<const float2*>(&sh.row_scale[8 * (n0 + n) + 2 * x]);
              const float2 rope = make_float2(__uint_as_float(pe[2 * x]), __uint_as_float(pe[2 * x + 1]));
              s_val[n][x] = fma2(rope, both(qk_scale), mul2(sum[x], scale));
            }
          }
        const int pos = (seg_p + 2 * i) * kPage + token;
        const bool bad = bad_page[at] != 0;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&taken[tile & 1]);
        // From here on z_tok is what the zero takes from each value: z s.
#pragma unroll
        for (int k = 0; k < NG; ++k) z_tok[k] *= s_tok[k];
        if (__any_sync(0xFFFFFFFFu, pos >= lim_min || bad || !here)) {
          // the request's or the run's end, or a page that is not there
          const bool none = bad || !here || pos >= len;
          // A group that is no number: rows that see the token have a weight of NaN by their score, and for those that do
          // not a weight of 0 has to stay 0 in its products.
#pragma unroll
          for (int k = 0; k < NG; ++k)
            if (none || !(fabsf(s_tok[k]) < INFINITY && fabsf(z_tok[k]) < INFINITY)) s_tok[k] = z_tok[k] = 0.f;
#pragma unroll
          for (int n = 0; n < HT; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int row = row0 + 8 * (n0 + n) + 2 * x;
              if (none || pos >= lim_min + row / a.heads) s_val[n][x].x = -INFINITY;
              if (none || pos >= lim_min + (row + 1) / a.heads) s_val[n][x].y = -INFINITY;
            }
        }
        if (here && page >= C::WEIGHTS) wait_for(&page_free[(page - C::WEIGHTS) % PAGES], (page - C::WEIGHTS) / PAGES);
        __syncwarp();

        // Equal elements, which the store gives scale 1 and codes 0: no scale.  Looked for where a scale of 1 matters.
        auto drop_equal = [&]() {
#pragma unroll
          for (int k = 0; k < NG; ++k) {
            if (s_tok[k] != 1.f) continue;
            const char* row = smem + at * C::CODES + (D == 512 ? k / 2 * 8192 : 0) + (token & 63) * 128;
            uint32_t any = 0;
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              const uint4 v = *reinterpret_cast<const uint4*>(row + (((D == 512 ? k % 2 : k) * 4 + c) ^ (token & 7)) * 16);
              any |= v.x | v.y | v.z | v.w;
            }
            if (any == 0) s_tok[k] = 0.f;
          }
        };
        // Weights against the present references, times each group's scale, to shared memory; true where a
        // weight or a scale has left its reference behind (their sums: moving early does no harm), or is NaN.
        float2 p_val[HT][4];
        auto weigh = [&]() {
          char* weights_at = smem + C::OFF_P + (page % C::WEIGHTS) * C::PBUF + n0 * C::PTILE + (token & 63) * 16;
          float2 weights = both(0.f);
          float sizes = 0.f;
#pragma unroll
          for (int n = 0; n < HT; ++n)
            if (n < my_tiles) {
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const float2 m = *reinterpret_cast<const float2*>(&sh.max[8 * (n0 + n) + 2 * x]);
                const float2 d = add2(s_val[n][x], make_float2(-m.x, -m.y));
                p_val[n][x] = make_float2(ex2_approx(d.x), ex2_approx(d.y));
                weights = add2(weights, p_val[n][x]);
              }
            }
#pragma unroll
          for (int k = 0; k < NG; ++k) {
            const float s = s_tok[k] * unit[k];
            sizes = fmaxf(sizes, fmaf(fabsf(z_tok[k] * unit[k]), kZeroShare, fabsf(s)));
#pragma unroll
            for (int n = 0; n < HT; ++n)
              if (n < my_tiles) {
                uint32_t h[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                  const float2 v = mul2(p_val[n][x], both(s));
                  h[x] = pack_half2(v.x, v.y);
                }
                if (here) *reinterpret_cast<uint4*>(weights_at + (k * NH + n) * C::PTILE) = make_uint4(h[0], h[1], h[2], h[3]);
              }
          }
          return !(weights.x + weights.y <= kSlack) || !(sizes <= kScaleSlack);
        };
        // A request's first tile brings the first references; while a row has a factor of its own, each tile moves them.
        const bool move = token_any(weigh() || factors);
        if (move) {  // new references: the tile's maxima; the sums so far are brought to them
          drop_equal();
#pragma unroll
          for (int n = 0; n < HT; ++n)
            if (n < my_tiles) {
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const float m0 = warp_max_f32(s_val[n][x].x), m1 = warp_max_f32(s_val[n][x].y);
                if (lane == 0) *reinterpret_cast<float2*>(&sh.red_m[quarter][8 * (n0 + n) + 2 * x]) = make_float2(m0, m1);
              }
            }
#pragma unroll
          for (int k = 0; k < NG; ++k) {
            const float s = warp_max_f32(fmaf(fabsf(z_tok[k]), kZeroShare, fabsf(s_tok[k])));
            if (lane == 0 && half == 0) sh.red_s[quarter][k] = s;
          }
          token_sync();
          float keep_unit[NG];
          bool doubt = factors;  // that each row has met P s unit of kLeast in each group
          float seen = -INFINITY;
#pragma unroll
          for (int n = 0; n < HT; ++n)
            if (n < my_tiles)
#pragma unroll
              for (int x = 0; x < 4; ++x) seen = fmaxf(seen, fmaxf(s_val[n][x].x, s_val[n][x].y));
#pragma unroll
          for (int k = 0; k < NG; ++k) {
            const float s = fmaxf(fmaxf(sh.red_s[0][k], sh.red_s[1][k]), fmaxf(sh.red_s[2][k], sh.red_s[3][k]));
            keep_unit[k] = 1.f;
            if (s * unit[k] > kScaleTop) {  // bring the largest scale into [kScaleTop / 2, kScaleTop)
              const float u = pow2(min(max(130 - static_cast<int>(__float_as_uint(s) >> 23), -126), 100));
              keep_unit[k] = u / unit[k];
              unit[k] = u;
            }
            if (tid == 0) sh.keep_unit[k] = keep_unit[k];
            doubt |= seen > -INFINITY && !(s_tok[k] * unit[k] >= kLeast);
          }
          if (tid < ROWS) {
            const float old = sh.max[tid];
            const float m = fmaxf(fmaxf(sh.red_m[0][tid], sh.red_m[1][tid]), fmaxf(sh.red_m[2][tid], sh.red_m[3][tid]));
            sh.keep_row[tid] = ex2_approx(old - fmaxf(old, m));
            sh.max[tid] = fmaxf(old, m);
            // Else the row's largest weight, 1, is in this tile; or it has seen nothing yet, and its first token moves again.
            if (m < old && old > kNoMax)
#pragma unroll
              for (int k = 0; k < NG; ++k) doubt |= !(sh.met[k * ROWS + tid] * keep_unit[k] >= kLeast);
          }
          __syncwarp();
          doubt = token_any(doubt);
          weigh();
#pragma unroll
          for (int n = 0; n < HT; ++n)
            if (n < my_tiles) {
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const float2 keep = *reinterpret_cast<const float2*>(&sh.keep_row[8 * (n0 + n) + 2 * x]);
                l_sum[n][x] = mul2(l_sum[n][x], keep);
#pragma unroll
                for (int k = 0; k < NG; ++k) zsum[k][n][x] = mul2(zsum[k][n][x], mul2(keep, both(keep_unit[k])));
              }
            }
          if (!doubt) {
            if (tid < ROWS) {
#pragma unroll
              for (int k = 0; k < NG; ++k) {
                sh.keep[turn][k][tid] = sh.keep_row[tid] * keep_unit[k];
                sh.met[k * ROWS + tid] = kLeast;
              }
            }
          } else {  // each row's largest P s unit of the tile, and factors for those that have met too little
            float su[NG];
#pragma unroll
            for (int k = 0; k < NG; ++k) su[k] = s_tok[k] * unit[k];
#pragma unroll 1
            for (int k = 0; k < NG; ++k)
#pragma unroll
              for (int n = 0; n < HT; ++n)
                if (n < my_tiles) {
#pragma unroll
                  for (int x = 0; x < 4; ++x) {
                    const float2 w = mul2(p_val[n][x], both(fabsf(su[k])));
                    const float w0 = warp_max_f32(w.x), w1 = warp_max_f32(w.y);
                    float* at_row = &sh.red_w[quarter][k * ROWS + 8 * (n0 + n) + 2 * x];
                    if (lane == 0) *reinterpret_cast<float2*>(at_row) = make_float2(w0, w1);
                  }
                }
            token_sync();
            // Weights that came between two moves are not in `met`: a factor may be larger for that, which loses nothing.
            bool odd = false;
            if (tid < NG * ROWS) {
              const float kept = sh.keep_row[tid % ROWS] * sh.keep_unit[tid / ROWS];
              const float here_w = fmaxf(fmaxf(sh.red_w[0][tid], sh.red_w[1][tid]), fmaxf(sh.red_w[2][tid], sh.red_w[3][tid]));
              const float w = fmaxf(sh.met[tid] * kept, here_w);
              odd = !(w >= kLeast) && sh.max[tid % ROWS] > kNoMax;  // of a row that has seen something
              const float f = odd && w > 0.f ? pow2(min(130 - static_cast<int>(__float_as_uint(w) >> 23), 100)) : 1.f;
              sh.met[tid] = w;
              sh.keep[turn][0][tid] = kept * (f / sh.factor[0][tid]);
              sh.factor[0][tid] = f;
            }
            __syncwarp();
            factors = token_any(odd);
            char* weights_at = smem + C::OFF_P + (page % C::WEIGHTS) * C::PBUF + n0 * C::PTILE + (token & 63) * 16;
            if (factors && here)
#pragma unroll 1
              for (int k = 0; k < NG; ++k)
#pragma unroll
                for (int n = 0; n < HT; ++n)
                  if (n < my_tiles) {
                    uint32_t h[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                      const float2 f = *reinterpret_cast<const float2*>(&sh.factor[k][8 * (n0 + n) + 2 * x]);
                      const float2 v = mul2(mul2(p_val[n][x], both(su[k])), f);
                      h[x] = pack_half2(v.x, v.y);
                    }
                    *reinterpret_cast<uint4*>(weights_at + (k * NH + n) * C::PTILE) = make_uint4(h[0], h[1], h[2], h[3]);
                  }
          }
          token_sync();
        }
        if (tid == 0) {
          sh.moved[turn] = move;
          mbar_arrive(&weighed[turn]);
        }
        if (++turn == 3) turn = 0;
        // ---- the denominators and the zeros' share ----
#pragma unroll
        for (int n = 0; n < HT; ++n)
          if (n < my_tiles) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              l_sum[n][x] = add2(l_sum[n][x], p_val[n][x]);
#pragma unroll
              for (int k = 0; k < NG; ++k) zsum[k][n][x] = fma2(p_val[n][x], both(z_tok[k] * unit[k]), zsum[k][n][x]);
            }
          }
      }
      done += count;
      // ---- the request's sums, for the adding warps ----
      if (begun) named_bar_sync(kBarTaken, kTokens + kAdders);  // they have taken the last request's
      begun = true;
#pragma unroll
      for (int n = 0; n < HT; ++n)
        if (n < my_tiles) {
          const int row = 8 * (n0 + n) + (lane & 7);
          const float l = warp_sums(l_sum[n]);
          if (lane < 8) sh.l[quarter][row] = l;
#pragma unroll
          for (int k = 0; k < NG; ++k) {
            const float z = warp_sums(zsum[k][n]);
            if (lane < 8) sh.z[quarter][k][row] = z;
          }
        }
      if (tid < ROWS) sh.max_out[tid] = sh.max[tid];
      if (tid < NG * ROWS) sh.factor_out[tid] = 1.f / sh.factor[0][tid];
      if (tid == 0)
#pragma unroll
        for (int k = 0; k < NG; ++k) sh.unit_out[k] = unit[k];
      bar_arrive(kBarSums, kTokens + kAdders);
      ++seg_b;
      seg_p = 0;
    }
    if (begun) named_bar_sync(kBarTaken, kTokens + kAdders);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, 512);
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

// A CTA's tiles of 8 query rows: as few CTAs as hold them all, evenly filled.  A page is read once for each, so five
// tiles (40 rows) in one CTA beat three in each of two even though its registers spill a little: 128 requests of 8K,
// 40 heads of 256 + 32: 190 us against 241, single calls.
struct Shape {
  int tiles, blocks, groups;  // tiles of a CTA, CTAs for all rows, runs of pages (a CTA each and row block)
};
int most_tiles(int d) { return d == 512 ? 2 : 5; }
Shape shape_of(int d, int q_len, int heads) {
  const int tiles = (q_len * heads + 7) / 8, most = most_tiles(d);
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

  // Few requests are cut into many partials: all warps of a CTA share 128 columns of a row then (one request of 128K: 42 us
  // in all); with less than 8 partials a request a warp each is enough and needs no join.
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

// The partials of the largest of all calls of up to this many rows: a CTA's tiles may fall as rows are added (41 rows of
// D = 256 take two CTAs of 3 tiles, 40 one of 5), so tiles and CTAs are counted apart, each at its most.
int64_t decode_workspace(int batch, int q_len, int heads, int d) {
  const int tiles = (q_len * heads + 7) / 8, most = most_tiles(d), blocks = (tiles + most - 1) / most;
  // groups * blocks <= sm_count() + blocks
  return kHeaderBytes + int64_t(16) * batch + int64_t(2) * (sm_count() + blocks) * std::min(tiles, most) * 8 * (d + 1) * 4;
}

int launch_decode(const DecodeArgs& a, cudaStream_t s) {
  if (a.cache.latent_dim == 512) return a.cache.rope_dim == 64 ? launch_tiles<512, 64>(a, s) : launch_tiles<512, 32>(a, s);
  return a.cache.rope_dim == 64 ? launch_tiles<256, 64>(a, s) : launch_tiles<256, 32>(a, s);
}

}  // namespace i4
}  // namespace rolaq
