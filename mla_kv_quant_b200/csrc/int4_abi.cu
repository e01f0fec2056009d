// extern "C" entry points of the 4-bit latent cache (declared in include/rolaq_b200.h).  Every
// function validates its arguments on the host before launching, returns a status code, and
// records a message for rolaq_last_error() on failure.
#include "abi.cuh"
#include "int4.cuh"

using namespace rolaq;

namespace {

int check_cache(const rolaq_int4_cache* c) {
  if (c == nullptr) return fail(ROLAQ_EINVAL, "cache is NULL");
  if (c->latent_dim != 256 && c->latent_dim != 512)
    return fail(ROLAQ_EUNSUPPORTED, "latent_dim %d unsupported (256 or 512)", c->latent_dim);
  if (c->rope_dim != 32 && c->rope_dim != 64)
    return fail(ROLAQ_EUNSUPPORTED, "rope_dim %d unsupported (32 or 64)", c->rope_dim);
  if (!c->codes || !c->params || !c->rope) return fail(ROLAQ_EINVAL, "cache codes/params/rope must be non-NULL");
  if (!aligned16(c->codes) || !aligned16(c->params) || !aligned16(c->rope))
    return fail(ROLAQ_EINVAL, "cache codes/params/rope must be 16-byte aligned");
  if (c->num_slots <= 0 || c->num_slots % i4::kPage || c->num_slots >= (int64_t(1) << 31))
    return fail(ROLAQ_EINVAL, "num_slots %lld must be a positive multiple of 64 below 2^31", (long long)c->num_slots);
  return ROLAQ_OK;
}

int check_boxes(const rolaq_int4_cache* c) {
  if (int rc = check_cache(c)) return rc;
  if (!c->box_center || !c->box_radius || !c->box_exps) return fail(ROLAQ_EINVAL, "the cache has no page boxes");
  if (!aligned16(c->box_center) || !aligned16(c->box_radius) || !aligned16(c->box_exps))
    return fail(ROLAQ_EINVAL, "page boxes must be 16-byte aligned");
  return ROLAQ_OK;
}

// Rows of `width` elements at a stride of ld, loaded or stored 16 bytes at a time.
bool row_ok(const void* p, int64_t ld, int64_t width) { return aligned16(p) && ld >= width && ld % 8 == 0; }

// Where the page scores of a selection start in the scratch: after the decode's part.
int64_t select_offset(int64_t decode_bytes) { return (decode_bytes + 255) / 256 * 256; }

bool sizes_ok(int32_t batch, int32_t q_len, int32_t heads, int32_t max_pages) {
  return batch >= 0 && batch <= 65535 && q_len >= 1 && q_len <= 64 && heads >= 1 && heads <= 128 && max_pages >= 0 &&
         max_pages < (1 << 25);
}

}  // namespace

extern "C" {

int rolaq_int4_write(const void* c, int c_is_f32, int64_t ld_c, const uint16_t* k_pe, int64_t ld_pe,
                     const void* slots, int slots_are_int64, int64_t n, const rolaq_int4_cache* cache, int32_t* err,
                     cudaStream_t stream) {
  if (n < 0) return fail(ROLAQ_EINVAL, "n < 0");
  if (int rc = check_cache(cache)) return rc;
  if (n == 0) return ROLAQ_OK;
  if (!c || !k_pe || !slots) return fail(ROLAQ_EINVAL, "NULL pointer");
  if (!row_ok(c, ld_c, cache->latent_dim) || !row_ok(k_pe, ld_pe, cache->rope_dim))
    return fail(ROLAQ_EINVAL, "c and k_pe must be 16-byte aligned, row strides >= the width and multiples of 8");
  if (n >= (int64_t(1) << 31)) return fail(ROLAQ_EINVAL, "n too large");
  return cuda_rc(i4::launch_write(c, c_is_f32 != 0, ld_c, k_pe, ld_pe, slots, slots_are_int64, n, *cache, err,
                                    stream),
                 "int4_write");
}

int rolaq_int4_read(const rolaq_int4_cache* cache, const void* slots, int slots_are_int64, int64_t n, void* out,
                    int out_is_f32, int64_t ld_out, uint16_t* out_pe, int64_t ld_pe, int32_t* err,
                    cudaStream_t stream) {
  if (n < 0) return fail(ROLAQ_EINVAL, "n < 0");
  if (int rc = check_cache(cache)) return rc;
  if (n == 0) return ROLAQ_OK;
  if (!out || !slots) return fail(ROLAQ_EINVAL, "NULL pointer");
  if (!row_ok(out, ld_out, cache->latent_dim) || (out_pe && !row_ok(out_pe, ld_pe, cache->rope_dim)))
    return fail(ROLAQ_EINVAL, "outputs must be 16-byte aligned, row strides >= the width and multiples of 8");
  if (n >= (int64_t(1) << 31)) return fail(ROLAQ_EINVAL, "n too large");
  return cuda_rc(i4::launch_read(*cache, slots, slots_are_int64, n, out, out_is_f32 != 0, ld_out, out_pe, ld_pe, err,
                                   stream),
                 "int4_read");
}

int rolaq_int4_update_boxes(const rolaq_int4_cache* cache, const int32_t* pages, const int32_t* counts, int64_t n,
                            int32_t* err, cudaStream_t stream) {
  if (n < 0) return fail(ROLAQ_EINVAL, "n < 0");
  if (int rc = check_boxes(cache)) return rc;
  if (n == 0) return ROLAQ_OK;
  if (!pages || !counts) return fail(ROLAQ_EINVAL, "NULL pointer");
  if (n >= (int64_t(1) << 31)) return fail(ROLAQ_EINVAL, "n too large");
  return cuda_rc(i4::launch_update_boxes(*cache, pages, counts, n, err, stream), "int4_update_boxes");
}

int rolaq_int4_read_boxes(const rolaq_int4_cache* cache, const int32_t* pages, int64_t n, float* lo, float* hi,
                          int64_t ld, int32_t* err, cudaStream_t stream) {
  if (n < 0) return fail(ROLAQ_EINVAL, "n < 0");
  if (int rc = check_boxes(cache)) return rc;
  if (n == 0) return ROLAQ_OK;
  if (!pages || !lo || !hi) return fail(ROLAQ_EINVAL, "NULL pointer");
  if (!aligned16(lo) || !aligned16(hi) || ld % 4 || ld < cache->latent_dim + cache->rope_dim)
    return fail(ROLAQ_EINVAL, "lo and hi must be 16-byte aligned, ld >= D + Dr and a multiple of 4");
  if (n >= (int64_t(1) << 31)) return fail(ROLAQ_EINVAL, "n too large");
  return cuda_rc(i4::launch_read_boxes(*cache, pages, n, lo, hi, ld, err, stream), "int4_read_boxes");
}

int64_t rolaq_int4_workspace_bytes(int32_t batch, int32_t q_len, int32_t heads, int32_t latent_dim,
                                   int32_t max_pages) {
  if (!sizes_ok(batch, q_len, heads, max_pages) || (latent_dim != 256 && latent_dim != 512)) return -1;
  return select_offset(i4::decode_workspace(batch, q_len, heads, latent_dim)) +
         i4::select_workspace(batch, max_pages);
}

int rolaq_int4_decode(const uint16_t* q, int64_t q_stride_b, int64_t q_stride_t, int64_t q_stride_h, int32_t batch,
                      int32_t q_len, int32_t heads, const rolaq_int4_cache* cache, const int32_t* page_table,
                      int64_t pt_stride, int32_t max_pages, const int32_t* seq_lens, float sm_scale, void* workspace,
                      int64_t workspace_bytes, uint16_t* out, int64_t out_stride_b, int64_t out_stride_t,
                      int64_t out_stride_h, float* lse, int32_t* err, cudaStream_t stream) {
  if (!sizes_ok(batch, q_len, heads, max_pages))
    return fail(ROLAQ_EINVAL, "batch in [0, 65535], q_len in [1, 64], heads in [1, 128], max_pages in [0, 2^25)");
  if (int rc = check_cache(cache)) return rc;
  if (!(sm_scale > 0.f) || !(sm_scale < 1e30f)) return fail(ROLAQ_EINVAL, "sm_scale must be finite and > 0");
  if (batch == 0) return ROLAQ_OK;
  const int d = cache->latent_dim, w = d + cache->rope_dim;
  if (!q || !seq_lens || !out || !workspace || (max_pages > 0 && !page_table)) return fail(ROLAQ_EINVAL, "NULL pointer");
  if (pt_stride < max_pages) return fail(ROLAQ_EINVAL, "page table rows are shorter than max_pages");
  if (!row_ok(q, q_stride_h, w) || q_stride_t % 8 || q_stride_b % 8 || q_stride_t < 0 || q_stride_b < 0)
    return fail(ROLAQ_EINVAL, "q must be 16-byte aligned with strides that are multiples of 8, rows of D + Dr");
  if (!row_ok(out, out_stride_h, d) || out_stride_t % 8 || out_stride_b % 8 || out_stride_t < 0 || out_stride_b < 0)
    return fail(ROLAQ_EINVAL, "out must be 16-byte aligned with strides that are multiples of 8, rows of D");
  if (!aligned16(workspace) || workspace_bytes < i4::decode_workspace(batch, q_len, heads, d))
    return fail(ROLAQ_EINVAL, "workspace of %lld bytes is too small (%lld) or not 16-byte aligned",
                (long long)workspace_bytes, (long long)i4::decode_workspace(batch, q_len, heads, d));
  i4::DecodeArgs a{q, q_stride_b, q_stride_t, q_stride_h, batch, q_len, heads, *cache, page_table, pt_stride,
                     max_pages, seq_lens, sm_scale, workspace, out, out_stride_b, out_stride_t, out_stride_h, lse, err};
  return cuda_rc(i4::launch_decode(a, stream), "int4_decode");
}

int rolaq_int4_select_pages(const uint16_t* q, int64_t q_stride_b, int64_t q_stride_h, int32_t batch, int32_t heads,
                            const rolaq_int4_cache* cache, const int32_t* page_table, int64_t pt_stride,
                            int32_t max_pages, const int32_t* seq_lens, int32_t budget, int32_t keep_first,
                            int32_t keep_last, void* workspace, int64_t workspace_bytes, int32_t* sel_table,
                            int64_t sel_stride, int32_t* sel_lens, int32_t* err, cudaStream_t stream) {
  if (!sizes_ok(batch, 1, heads, max_pages))
    return fail(ROLAQ_EINVAL, "batch in [0, 65535], heads in [1, 128], max_pages in [0, 2^25)");
  if (int rc = check_boxes(cache)) return rc;
  if (keep_first < 0 || keep_last < 1 || budget < 1 || int64_t(keep_first) + keep_last > budget || budget >= (1 << 25))
    return fail(ROLAQ_EINVAL, "needs 0 <= keep_first, 1 <= keep_last, keep_first + keep_last <= budget < 2^25");
  if (batch == 0) return ROLAQ_OK;
  if (!q || !seq_lens || !workspace || !sel_table || !sel_lens || (max_pages > 0 && !page_table))
    return fail(ROLAQ_EINVAL, "NULL pointer");
  if (pt_stride < max_pages || sel_stride < budget) return fail(ROLAQ_EINVAL, "page table or sel_table rows too short");
  if (!row_ok(q, q_stride_h, cache->latent_dim + cache->rope_dim) || q_stride_b % 8 || q_stride_b < 0)
    return fail(ROLAQ_EINVAL, "q must be 16-byte aligned with strides that are multiples of 8, rows of D + Dr");
  // The scores lie at the end of the scratch, behind the part that a decode of any size uses.
  const int64_t need = i4::select_workspace(batch, max_pages);  // behind the header
  if (!aligned16(workspace) || workspace_bytes < i4::kHeaderBytes + need)
    return fail(ROLAQ_EINVAL, "workspace of %lld bytes is too small (%lld) or not 16-byte aligned",
                (long long)workspace_bytes, (long long)(i4::kHeaderBytes + need));
  char* scores = static_cast<char*>(workspace) + (workspace_bytes - need) / 16 * 16;
  i4::SelectArgs a{q, q_stride_b, q_stride_h, batch, heads, *cache, page_table, pt_stride, max_pages, seq_lens,
                     budget, keep_first, keep_last, reinterpret_cast<float*>(scores), static_cast<int32_t*>(workspace), sel_table, sel_stride, sel_lens, err};
  return cuda_rc(i4::launch_select(a, stream), "int4_select_pages");
}

}  // extern "C"
