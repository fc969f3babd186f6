// Internal interface of the softmax-attention kernels (packed prompts, paged cache).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>

#include "gdn_common.cuh"

namespace gdn {

// One call: the newest q_len tokens of each sequence against its kv_len tokens (those
// included), causal.  Packed prompts: kv rows are the token rows themselves; paged: row j
// of sequence s is row j % page_size of page block_table[s][j / page_size].
struct AttnArgs {
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16* out;
  const void* cu;  // [num_seqs + 1] (null: every sequence has total_q / num_seqs tokens)
  bool cu64;
  bool paged;
  const int* block_table;
  const void* kv_lens;
  bool kv64;
  long long table_stride;  // entries between the rows of block_table
  int table_width;         // pages a sequence can have
  int page_size;
  long long num_pages;
  long long k_page_stride, v_page_stride;  // elements
  long long q_stride, k_stride, v_stride, o_stride;
  long long total_q;
  int num_seqs, hq, hkv;
  float scale_log2;  // scale * log2(e)
};

__device__ __forceinline__ long long attn_index(const void* p, bool is64, long long i) {
  return is64 ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int*>(p)[i];
}

// A sequence's rows, kept inside the buffers whatever cu_seqlens and kv_lens hold.
struct AttnSeq {
  long long q0;  // first query row
  int q_len, kv_len;
};
__device__ __forceinline__ AttnSeq attn_seq(const AttnArgs& p, int s) {
  AttnSeq r;
  long long a, b;
  if (p.cu != nullptr) {
    a = attn_index(p.cu, p.cu64, s);
    b = attn_index(p.cu, p.cu64, s + 1);
  } else {
    const long long per = p.total_q / p.num_seqs;
    a = s * per;
    b = a + per;
  }
  a = a < 0 ? 0 : (a > p.total_q ? p.total_q : a);
  b = b < a ? a : (b > p.total_q ? p.total_q : b);
  r.q0 = a;
  r.q_len = (int)(b - a);
  if (!p.paged) {
    r.kv_len = r.q_len;
  } else {
    const long long most = (long long)p.table_width * p.page_size;
    long long n = attn_index(p.kv_lens, p.kv64, s);
    r.kv_len = (int)(n < 0 ? 0 : (n > most ? most : n));
  }
  return r;
}

// TMA map of a bf16 tensor (strides of dimensions 1 .. in elements), 128-byte swizzle; the
// maps of K and V, `box` key rows high: rows of the packed prompts by halves of 64 columns, or
// of a page, both halves for 8 rows after 8 rows (a head's 256 bytes of a row are asked for
// together).
bool attn_map(CUtensorMap* m, const void* base, int rank, const long long* dims,
              const long long* strides, const int* box);
bool attn_key_maps(CUtensorMap* mk, CUtensorMap* mv, const AttnArgs& p, int box);
// The highest box (a power of two, at most `most`) that does not cross a page's end.
int attn_key_box(const AttnArgs& p, int most);

// Tensor-core kernel on `sms` CTAs (workspace: attn_workspace_bytes(attn_tc_rows(), sms));
// `tag`: 48 bits, not 0, another one for every call (a graph's replays repeat its call's).
int attn_tc_rows();
cudaError_t launch_attn_tc(const AttnArgs& p, int sms, void* workspace, unsigned long long tag,
                           cudaStream_t st);
unsigned read_attn_tc_error(bool clear);

// Kernel for few rows: an item has at most `rows` (8, 16 or 32) of them.
cudaError_t launch_attn_rows(const AttnArgs& p, int rows, int sms, void* workspace,
                             unsigned long long tag, cudaStream_t st);
unsigned read_attn_rows_error(bool clear);

// After a failure was read and cleared, with nothing running: what launches that failed left in
// their scratch counts for no later launch, replays of the same graph among them.
bool count_attn_tc_report();
bool count_attn_rows_report();

}  // namespace gdn
