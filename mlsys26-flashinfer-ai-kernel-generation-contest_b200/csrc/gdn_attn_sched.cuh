// How the attention kernels share out their work, on the device, from the lengths alone.
//
// An item is one key/value head of one sequence with a block of `block` query tokens (all
// heads of its group): it reads the first e = kv_len - q_len + (tokens up to the block's
// last) keys.  Its cost is e plus a constant for its start and end.  The costs of all items,
// in the order (sequence, head, block), lie on one line that is cut into one equal range
// per CTA: ragged batches, causal blocks and one long sequence come out balanced alike,
// and no list is made.  A cut inside an item splits its keys, at a tile; both sides write
// partial results, and a second kernel joins the pieces in the order of the keys (so the
// result does not depend on timing).  An item of few tiles is not split: it goes to the
// CTA that holds its middle.
#pragma once

#include "gdn_attn.cuh"

namespace gdn {

// a CTA has at most two partial pieces: of the item its range begins inside (slot 0) and
// of the one its range ends inside (slot 1)
constexpr int kAttnSlots = 2;

struct AttnGrid {
  int block;     // query tokens per item
  int sub;       // query tokens per tile of rows: row (tok / sub) * sub_rows + (tok % sub) *
  int sub_rows;  // heads of the group + head
  int tile;      // keys per tile
  int overhead;  // cost of an item's start and end, in keys
  int whole;     // items of at most this many tiles are not split
};

// Keys that block b of a sequence reads.
__device__ __forceinline__ int attn_block_keys(const AttnSeq& s, int block, int b) {
  const long long last = (long long)(b + 1) * block;
  const long long e = (long long)s.kv_len - s.q_len + (last < s.q_len ? last : s.q_len);
  return e > 0 ? (int)e : 0;
}
__device__ __forceinline__ int attn_blocks(const AttnSeq& s, int block) {
  return (s.q_len + block - 1) / block;
}
// Cost of the first n blocks of one head of a sequence, in closed form.
__device__ __forceinline__ long long attn_cost_before(const AttnSeq& s, const AttnGrid& g, int n) {
  if (n <= 0) return 0;
  const int nb = attn_blocks(s, g.block);
  const long long a = (long long)s.kv_len - s.q_len;
  const long long m = n < nb ? n : nb - 1;              // blocks of full size
  long long b0 = a < 0 ? -a / g.block : 0;              // leading blocks that see nothing
  if (b0 > m) b0 = m;
  long long c = (m - b0) * a + (long long)g.block * ((m * (m + 1) - b0 * (b0 + 1)) / 2);
  if (n == nb) c += s.kv_len;
  return c + (long long)n * g.overhead;
}
__device__ __forceinline__ long long attn_head_cost(const AttnSeq& s, const AttnGrid& g) {
  return attn_cost_before(s, g, attn_blocks(s, g.block));
}
// Tile of an item (e keys, n tiles) at cost offset x.
__device__ __forceinline__ int attn_tile_at(const AttnGrid& g, int e, int n, long long x) {
  const long long cost = (long long)e + g.overhead;
  if (x >= cost) return n;
  if (n <= g.whole) return 2 * x > cost ? n : 0;
  const long long y = x - g.overhead;
  return y <= 0 ? 0 : (int)(y / g.tile);
}

struct AttnCursor {
  long long start;  // cost before the item
  AttnSeq seq;
  int s, h, b, nb;  // sequence, head, block, blocks of the sequence

  __device__ __forceinline__ void open(const AttnArgs& p, const AttnGrid& g, int seq_index) {
    s = seq_index;
    seq = attn_seq(p, s);
    nb = attn_blocks(seq, g.block);
    h = 0;
    b = 0;
  }
  // To the item that holds cost u, in sequence s whose cost begins at `at`.
  __device__ __forceinline__ void seek(const AttnArgs& p, const AttnGrid& g, int seq_index,
                                       long long at, long long u) {
    open(p, g, seq_index);
    const long long per = attn_head_cost(seq, g);
    h = (int)((u - at) / per);
    const long long r = u - at - h * per;
    int lo = 0, hi = nb - 1;  // the last block whose cost begins at or before r
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (attn_cost_before(seq, g, mid) <= r) lo = mid; else hi = mid - 1;
    }
    b = lo;
    start = at + h * per + attn_cost_before(seq, g, b);
  }
  __device__ __forceinline__ int keys(const AttnGrid& g) const {
    return attn_block_keys(seq, g.block, b);
  }
  __device__ __forceinline__ long long cost(const AttnGrid& g) const {
    return (long long)keys(g) + g.overhead;
  }
  // To the next item; false behind the last one.
  __device__ __forceinline__ bool next(const AttnArgs& p, const AttnGrid& g) {
    start += cost(g);
    if (++b < nb) return true;
    b = 0;
    if (++h < p.hkv) return true;
    do {
      if (s + 1 >= p.num_seqs) return false;
      open(p, g, s + 1);
    } while (nb == 0);
    return true;
  }
};

__device__ __forceinline__ long long attn_cut(long long total, int c, int parts) {
  return total / parts * c + total % parts * c / parts;
}

// The block's share of the line: range [u0, u1) and the sequence that u0 lies in.
struct AttnShare {
  long long total, u0, seq_start;
  int seq;
};

// Collective over a block of NT threads (a multiple of 32): the total cost, and the
// sequence that holds the `c`-th of `parts` cuts.
template <int NT>
__device__ __forceinline__ void attn_share(const AttnArgs& p, const AttnGrid& g, int c, int parts,
                                           AttnShare* out) {
  __shared__ long long warp_sum[NT / 32];
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  long long mine = 0, own = 0;  // own: the cost of the last sequence looked at
  for (int s = tid; s < p.num_seqs; s += NT) {
    own = attn_head_cost(attn_seq(p, s), g) * p.hkv;
    mine += own;
  }
  for (int w = 16; w > 0; w >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, w);
  if (lane == 0) warp_sum[warp] = mine;
  if (tid == 0) found = 0;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) total += warp_sum[w];
  const long long u = attn_cut(total, c, parts);
  if (tid == 0) {
    out->total = total;
    out->u0 = u;
    out->seq = p.num_seqs;
    out->seq_start = total;
  }
  __syncthreads();
  long long base = 0;
  for (int s0 = 0; s0 < p.num_seqs && u < total; s0 += NT) {
    const int s = s0 + tid;
    long long x = 0;
    if (s < p.num_seqs)
      x = p.num_seqs <= NT ? own : attn_head_cost(attn_seq(p, s), g) * p.hkv;
    long long sum = x;
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, sum, w);
      if (lane >= w) sum += y;
    }
    if (lane == 31) warp_sum[warp] = sum;
    __syncthreads();
    long long all = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
      if (w < warp) sum += warp_sum[w];
      all += warp_sum[w];
    }
    sum += base;
    if (x > 0 && sum - x <= u && u < sum) {
      out->seq = s;
      out->seq_start = sum - x;
      found = 1;
    }
    base += all;
    __syncthreads();
    if (found) break;
  }
  __syncthreads();
}

// Partial results of a piece: rows of 128 fp32 sums, then (maximum in log2 units, sum) per row.
__host__ __device__ inline size_t attn_partial_bytes(int rows, int parts) {
  return (size_t)parts * kAttnSlots * rows * (kHeadDim + 2) * sizeof(float);
}
__device__ __forceinline__ float* attn_partial(float* ws, int rows, int cta, int slot) {
  return ws + ((long long)cta * kAttnSlots + slot) * rows * (kHeadDim + 2);
}

// Joins the pieces of split items (of `rows` rows); `parts` CTAs shared the work on `g`.
cudaError_t launch_attn_join(const AttnArgs& p, const AttnGrid& g, int rows, int parts,
                             float* workspace, cudaStream_t st);

}  // namespace gdn
