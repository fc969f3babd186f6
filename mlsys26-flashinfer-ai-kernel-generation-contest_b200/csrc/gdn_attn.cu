// C-ABI entry points of the softmax-attention operators: argument checks and the choice
// of the kernel.
#include <cmath>

#include "gdn_attn_sched.cuh"

namespace gdn {
namespace {

inline bool misaligned(const void* p, uintptr_t n) {
  return (reinterpret_cast<uintptr_t>(p) % n) != 0;
}

int check_heads(int hq, int hkv, int head_size) {
  if (hq <= 0 || hkv <= 0) return GDN_ERR_INVALID_ARGUMENT;
  if (head_size != kHeadDim || hq % hkv != 0 || hq / hkv > 64) return GDN_ERR_UNSUPPORTED;
  return GDN_OK;
}

// rows of `width` elements, 16-byte aligned, that do not overlap
bool bad_rows(const void* p, long long stride, long long width) {
  return !p || misaligned(p, 16) || stride < width || stride % 8 != 0;
}

// CTAs of a launch: one per SM of the current device (without one: what a size needs at most).
constexpr int kMaxParts = 160;
int parts() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0 ||
      n > kMaxParts)
    n = kMaxParts;
  return n;
}

size_t workspace_size() { return attn_partial_bytes(attn_tc_rows(), kMaxParts); }

int launch(AttnArgs& p, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  if (!workspace || workspace_bytes < workspace_size()) return GDN_ERR_WORKSPACE;
  if (misaligned(workspace, 16)) return GDN_ERR_INVALID_ARGUMENT;
  p.scale_log2 = default_scale(scale) * 1.4426950408889634f;
  return launch_attn_tc(p, parts(), static_cast<float*>(workspace),
                        static_cast<cudaStream_t>(stream)) == cudaSuccess
             ? GDN_OK
             : GDN_ERR_LAUNCH;
}

}  // namespace
}  // namespace gdn

extern "C" size_t gdn_attn_workspace_size(int total_q, int num_seqs, int num_q_heads,
                                          int num_kv_heads) {
  (void)total_q;
  (void)num_seqs;
  (void)num_q_heads;
  (void)num_kv_heads;
  return gdn::workspace_size();
}

extern "C" int gdn_attn_prefill_launch(const void* q, const void* k, const void* v,
                                       const void* cu_seqlens, int cu_seqlens_int64, float scale,
                                       void* output, int total_tokens, int num_seqs,
                                       int num_q_heads, int num_kv_heads, int head_size,
                                       long long q_stride, long long k_stride, long long v_stride,
                                       long long output_stride, void* workspace,
                                       size_t workspace_bytes, void* stream) {
  using namespace gdn;
  if (total_tokens < 0 || num_seqs < 0) return GDN_ERR_INVALID_ARGUMENT;
  if (const int e = check_heads(num_q_heads, num_kv_heads, head_size)) return e;
  if (total_tokens == 0 || num_seqs == 0) return GDN_OK;
  const long long qw = (long long)num_q_heads * kHeadDim, kw = (long long)num_kv_heads * kHeadDim;
  if (!cu_seqlens || misaligned(cu_seqlens, cu_seqlens_int64 ? 8 : 4) ||
      bad_rows(q, q_stride, qw) || bad_rows(k, k_stride, kw) || bad_rows(v, v_stride, kw) ||
      bad_rows(output, output_stride, qw))
    return GDN_ERR_INVALID_ARGUMENT;
  AttnArgs p{};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.out = static_cast<__nv_bfloat16*>(output);
  p.cu = cu_seqlens;
  p.cu64 = cu_seqlens_int64 != 0;
  p.q_stride = q_stride;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.o_stride = output_stride;
  p.total_q = total_tokens;
  p.num_seqs = num_seqs;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  return launch(p, scale, workspace, workspace_bytes, stream);
}

extern "C" int gdn_attn_paged_launch(
    const void* q, const void* k_cache, const void* v_cache, const int* block_table,
    long long block_table_stride, const void* kv_lens, int kv_lens_int64, const void* cu_seqlens,
    int cu_seqlens_int64, float scale, void* output, int total_q, int num_seqs, int table_width,
    int num_pages, int page_size, long long k_page_stride, long long v_page_stride,
    int num_q_heads, int num_kv_heads, int head_size, long long q_stride, long long output_stride,
    void* workspace, size_t workspace_bytes, void* stream) {
  using namespace gdn;
  if (total_q < 0 || num_seqs < 0 || table_width < 0 || num_pages < 0 || page_size <= 0)
    return GDN_ERR_INVALID_ARGUMENT;
  if (const int e = check_heads(num_q_heads, num_kv_heads, head_size)) return e;
  if (page_size % 8 != 0) return GDN_ERR_UNSUPPORTED;
  if (total_q == 0 || num_seqs == 0) return GDN_OK;
  const long long qw = (long long)num_q_heads * kHeadDim, kw = (long long)num_kv_heads * kHeadDim;
  if (!kv_lens || misaligned(kv_lens, kv_lens_int64 ? 8 : 4) || (!block_table && table_width > 0) ||
      misaligned(block_table, 4) || block_table_stride < table_width ||
      (cu_seqlens && misaligned(cu_seqlens, cu_seqlens_int64 ? 8 : 4)) ||
      (!cu_seqlens && total_q % num_seqs != 0) || bad_rows(q, q_stride, qw) ||
      bad_rows(output, output_stride, qw) || bad_rows(k_cache, k_page_stride, page_size * kw) ||
      bad_rows(v_cache, v_page_stride, page_size * kw) ||
      (long long)table_width * page_size > 0x7fffff00LL)
    return GDN_ERR_INVALID_ARGUMENT;
  AttnArgs p{};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k_cache);
  p.v = static_cast<const __nv_bfloat16*>(v_cache);
  p.out = static_cast<__nv_bfloat16*>(output);
  p.cu = cu_seqlens;
  p.cu64 = cu_seqlens_int64 != 0;
  p.paged = true;
  p.block_table = block_table;
  p.table_stride = block_table_stride;
  p.table_width = table_width;
  p.page_size = page_size;
  p.num_pages = num_pages;
  p.k_page_stride = k_page_stride;
  p.v_page_stride = v_page_stride;
  p.kv_lens = kv_lens;
  p.kv64 = kv_lens_int64 != 0;
  p.q_stride = q_stride;
  p.o_stride = output_stride;
  p.total_q = total_q;
  p.num_seqs = num_seqs;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  return launch(p, scale, workspace, workspace_bytes, stream);
}
