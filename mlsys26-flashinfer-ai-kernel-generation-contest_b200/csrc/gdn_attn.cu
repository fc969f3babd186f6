// C-ABI entry points of the softmax-attention operators: argument checks and the choice
// of the kernel.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <atomic>
#include <chrono>

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
int parts() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0 ||
      n > kAttnMaxParts)
    n = kAttnMaxParts;
  return n;
}

// Rows of an item for the few-rows kernel, or 0 where the tensor-core kernel runs.  Up to 32
// rows on average the former's padding and hand-overs are the smaller (64 single tokens of 4096
// keys, 16 / 2 heads: 55 us, the other 92; 32 x 4: 53 and 58).  The host does not see how
// ragged a packed batch is.  One chunk among single tokens would be read by many small items,
// so past 32 items in the longest sequence that is possible the tensor cores take it (255
// single tokens and a chunk of 512 over 16384 keys, 8 / 8 heads: 329 us, few rows 604; below,
// 63 and a chunk of 256 over 8192: few rows 219, the other 295).  Possible with a token in every
// sequence: empty ones void that bound (16 / 2 heads: a prompt of 1000 tokens with 999 empty
// sequences 188 us, alone 31; a chunk of 1000 over 8192 keys 619 and 85).  Without counting on
// those tokens every packed batch of more than 32 single tokens, 16 / 2 heads, would go to the
// tensor cores.
int few_rows(long long total_q, int num_seqs, int hq, int hkv, bool uniform) {
  const int grp = hq / hkv;
  const long long mean = (total_q + num_seqs - 1) / num_seqs * grp;
  const int rows = mean <= 8 ? 8 : mean <= 16 ? 16 : mean <= 32 ? 32 : 0;
  return !uniform && (total_q - num_seqs) * grp > 32 * rows ? 0 : rows;
}

// (It does not depend on how the tokens come: of the larger of the two choices.)
size_t workspace_size(long long total_q, int num_seqs, int hq, int hkv) {
  const int few = few_rows(total_q, num_seqs, hq, hkv, false);
  return attn_workspace_bytes(few ? few : attn_tc_rows(), kAttnMaxParts);
}

// A call's tag (48 bits, not 0), which memory that was not written by it holds by a chance
// of 2^-48: a counter mixed by the finaliser of the splitmix64 generator.
unsigned long long next_tag() {
  static std::atomic<unsigned long long> count{
      (unsigned long long)std::chrono::steady_clock::now().time_since_epoch().count()};
  unsigned long long z = (count.fetch_add(1, std::memory_order_relaxed) + 1) * 0x9e3779b97f4a7c15ull;
  z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ull;
  z = (z ^ (z >> 27)) * 0x94d049bb133111ebull;
  z = (z ^ (z >> 31)) >> 16;
  return z != 0 ? z : 1;
}

int launch(AttnArgs& p, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  if (!workspace || workspace_bytes < workspace_size(p.total_q, p.num_seqs, p.hq, p.hkv))
    return GDN_ERR_WORKSPACE;
  if (misaligned(workspace, 16)) return GDN_ERR_INVALID_ARGUMENT;
  p.scale_log2 = default_scale(scale) * 1.4426950408889634f;
  const int few = few_rows(p.total_q, p.num_seqs, p.hq, p.hkv, p.cu == nullptr);
  const unsigned long long tag = next_tag();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = few ? launch_attn_rows(p, few, parts(), workspace, tag, st)
                            : launch_attn_tc(p, parts(), workspace, tag, st);
  return e == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }();
  return fn;
}

}  // namespace

bool attn_map(CUtensorMap* m, const void* base, int rank, const long long* dims,
              const long long* strides, const int* box) {
  auto fn = encoder();
  if (!fn || rank > 5) return false;
  cuuint64_t d[5], st[4];
  cuuint32_t b[5], one[5];
  for (int i = 0; i < rank; ++i) {
    d[i] = (cuuint64_t)dims[i];
    b[i] = (cuuint32_t)box[i];
    one[i] = 1;
    if (i > 0) st[i - 1] = (cuuint64_t)strides[i - 1] * 2;
  }
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, const_cast<void*>(base), d, st, b,
            one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int attn_key_box(const AttnArgs& p, int most) {
  int box = most;
  while (p.paged && p.page_size % box != 0) box /= 2;
  return box;
}

bool attn_key_maps(CUtensorMap* mk, CUtensorMap* mv, const AttnArgs& p, int box) {
  const long long w = (long long)p.hkv * kHeadDim;
  if (p.paged) {
    // 64 columns, 8 rows, halves of the heads, groups of 8 rows of a page, pages
    const long long dims[5] = {64, 8, 2 * p.hkv, p.page_size / 8, p.num_pages};
    const long long ks[4] = {w, 64, 8 * w, p.k_page_stride}, vs[4] = {w, 64, 8 * w, p.v_page_stride};
    const int b[5] = {64, 8, 2, box / 8, 1};
    return attn_map(mk, p.k, 5, dims, ks, b) && attn_map(mv, p.v, 5, dims, vs, b);
  }
  const long long dims[2] = {w, p.total_q};
  const int b[2] = {64, box};
  return attn_map(mk, p.k, 2, dims, &p.k_stride, b) && attn_map(mv, p.v, 2, dims, &p.v_stride, b);
}

unsigned read_attn_device_error(bool clear) {
  return read_attn_tc_error(clear) | read_attn_rows_error(clear);
}
bool count_attn_report() { return count_attn_tc_report() && count_attn_rows_report(); }

}  // namespace gdn

extern "C" size_t gdn_attn_workspace_size(int total_q, int num_seqs, int num_q_heads,
                                          int num_kv_heads) {
  if (total_q <= 0 || num_seqs <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads) return 0;
  return gdn::workspace_size(total_q, num_seqs, num_q_heads, num_kv_heads);
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
