// Softmax attention, one warp per (query token, head): the definition with a running
// maximum and sum, one key at a time.
//   m' = max(m, s_j);  l' = l 2^(m - m') + 2^(s_j - m');  o' = o 2^(m - m') + 2^(s_j - m') v_j
#include "gdn_attn.cuh"

namespace gdn {
namespace {

__global__ void __launch_bounds__(128) attn_simple_kernel(const AttnArgs p) {
  const int lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (item >= p.total_q * p.hq) return;
  const long long row = item / p.hq;
  const int h = (int)(item - row * p.hq);
  const int hk = h / (p.hq / p.hkv);
  AttnSeq s{0, 0, 0};
  int n = 0;
  for (; n < p.num_seqs; ++n) {
    s = attn_seq(p, n);
    if (row >= s.q0 && row < s.q0 + s.q_len) break;
  }
  if (n == p.num_seqs) return;  // behind the last sequence: left as it was
  const long long end = (long long)s.kv_len - s.q_len + (row - s.q0) + 1;
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f};
  const __nv_bfloat16* qp = p.q + row * p.q_stride + (long long)h * kHeadDim + 4 * lane;
#pragma unroll
  for (int e = 0; e < 4; ++e) q[e] = bf2f(qp[e]) * p.scale_log2;
  float m = -INFINITY, l = 0.f;
  for (long long j = 0; j < end; ++j) {
    long long kr, vr;
    bool there = true;
    if (!p.paged) {
      kr = (s.q0 + j) * p.k_stride;
      vr = (s.q0 + j) * p.v_stride;
    } else {
      const long long page = p.block_table[n * p.table_stride + j / p.page_size];
      there = page >= 0 && page < p.num_pages;
      const long long off = (j % p.page_size) * (long long)p.hkv * kHeadDim;
      kr = page * p.k_page_stride + off;
      vr = page * p.v_page_stride + off;
    }
    const long long c = (long long)hk * kHeadDim + 4 * lane;
    float d = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) d = fmaf(q[e], there ? bf2f(p.k[kr + c + e]) : 0.f, d);
#pragma unroll
    for (int w = 1; w < 32; w *= 2) d += __shfl_xor_sync(0xffffffffu, d, w);
    const float m2 = fmaxf(m, d);
    const float a = exp2f(m - m2), b = exp2f(d - m2);
    l = l * a + b;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = o[e] * a + b * (there ? bf2f(p.v[vr + c + e]) : 0.f);
    m = m2;
  }
  __nv_bfloat16* op = p.out + row * p.o_stride + (long long)h * kHeadDim + 4 * lane;
  const float inv = end > 0 ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) op[e] = __float2bfloat16_rn(o[e] * inv);
}

}  // namespace

cudaError_t launch_attn_simple(const AttnArgs& p, cudaStream_t st) {
  const long long items = p.total_q * p.hq;
  attn_simple_kernel<<<(unsigned)((items + 3) / 4), 128, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace gdn
