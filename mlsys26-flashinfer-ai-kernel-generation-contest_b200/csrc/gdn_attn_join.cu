// Joins the partial results of attention items whose keys were split between CTAs.
//
// Piece i of a row has its maximum m_i (log2 units), sum l_i and unnormalised output o_i:
//   M = max m_i,  out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i,
// added in the order of the keys.  Block (c, y) looks at the cut between CTAs c and c + 1:
// if it is the first one inside an item that has more than one piece, the block joins its
// share of that item's rows; otherwise it has nothing to do.  A warp takes a row.
#include "gdn_attn_sched.cuh"

namespace gdn {
namespace {

constexpr int kJoinThreads = 128;

__global__ void __launch_bounds__(kJoinThreads)
    attn_join_kernel(const AttnArgs p, const AttnGrid g, int rows, int parts,
                     float* __restrict__ ws) {
  __shared__ AttnShare share;
  // the lengths are inputs of the whole call: they may be read before the partial results
  const int c = blockIdx.x + 1;
  attn_share<kJoinThreads>(p, g, c, parts, &share);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long total = share.total, u = share.u0;
  if (u >= total) return;
  AttnCursor cur;
  cur.seek(p, g, share.seq, share.seq_start, u);
  const int e = cur.keys(g);
  const int n = (e + g.tile - 1) / g.tile;
  const long long end = cur.start + cur.cost(g);
  if (cur.start >= u || attn_cut(total, c - 1, parts) > cur.start) return;  // not the first cut
  // the pieces: CTA c - 1 .. last
  int last = c;
  while (last + 1 < parts && attn_cut(total, last + 1, parts) < end) ++last;
  if (attn_tile_at(g, e, n, u - cur.start) == n ||
      (last == c && attn_tile_at(g, e, n, u - cur.start) == 0))
    return;  // all tiles on one side of the cut
  int pieces = 0;
  for (int i = c - 1; i <= last; ++i) {
    const long long lo = attn_cut(total, i, parts) - cur.start;
    const long long hi = attn_cut(total, i + 1, parts) - cur.start;
    pieces += attn_tile_at(g, e, n, lo > 0 ? lo : 0) < attn_tile_at(g, e, n, hi);
  }
  if (pieces <= 1) return;

  const int grp = p.hq / p.hkv;
  const int tok0 = cur.b * g.block;
  int toks = cur.seq.q_len - tok0;
  if (toks > g.block) toks = g.block;
  const int lane = threadIdx.x & 31;
  for (int r = blockIdx.y * (kJoinThreads / 32) + (threadIdx.x >> 5); r < toks * grp;
       r += gridDim.y * (kJoinThreads / 32)) {
    const int tok = r / grp;
    const int row = tok / g.sub * g.sub_rows + (tok % g.sub) * grp + r % grp;
    float M = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = c - 1; i <= last; ++i) {
      const long long lo = attn_cut(total, i, parts) - cur.start;
      const long long hi = attn_cut(total, i + 1, parts) - cur.start;
      if (attn_tile_at(g, e, n, lo > 0 ? lo : 0) >= attn_tile_at(g, e, n, hi)) continue;
      const float* part = attn_partial(ws, rows, i, lo > 0 ? 0 : 1);
      const float2 ml =
          *reinterpret_cast<const float2*>(part + (long long)rows * kHeadDim + 2 * row);
      const float4 x = *reinterpret_cast<const float4*>(part + (long long)row * kHeadDim + 4 * lane);
      if (ml.x == -INFINITY) continue;  // the row saw nothing of this piece
      const float m2 = fmaxf(M, ml.x);
      const float a = exp2f(M - m2), b = exp2f(ml.x - m2);
      l = l * a + ml.y * b;
      o.x = o.x * a + x.x * b;
      o.y = o.y * a + x.y * b;
      o.z = o.z * a + x.z * b;
      o.w = o.w * a + x.w * b;
      M = m2;
    }
    const float inv = M == -INFINITY ? 0.f : 1.f / l;
    __nv_bfloat162 b0 = __floats2bfloat162_rn(o.x * inv, o.y * inv);
    __nv_bfloat162 b1 = __floats2bfloat162_rn(o.z * inv, o.w * inv);
    uint2 w;
    w.x = *reinterpret_cast<uint32_t*>(&b0);
    w.y = *reinterpret_cast<uint32_t*>(&b1);
    __nv_bfloat16* op = p.out + (cur.seq.q0 + tok0 + tok) * p.o_stride +
                        ((long long)cur.h * grp + r % grp) * kHeadDim + 4 * lane;
    *reinterpret_cast<uint2*>(op) = w;
  }
}

}  // namespace

cudaError_t launch_attn_join(const AttnArgs& p, const AttnGrid& g, int rows, int parts,
                             float* workspace, cudaStream_t st) {
  if (parts < 2) return cudaSuccess;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(parts - 1), (unsigned)(rows > 64 ? 8 : 2));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, attn_join_kernel, p, g, rows, parts, workspace);
}

}  // namespace gdn
