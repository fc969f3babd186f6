// How the attention kernels share out their work, on the device, from the lengths alone.
//
// An item is one key/value head of one sequence with a block of `block` query tokens (all
// heads of its group): it reads the first e = kv_len - q_len + (tokens up to the block's
// last) keys.  Its cost is e plus a constant for its start and end.  The costs of all items,
// in the order (sequence, head, block), lie on one line that is cut into one equal range
// per CTA: ragged batches, causal blocks and one long sequence come out balanced alike,
// and no list is made.  A cut inside an item splits its keys, at a tile; both sides write
// partial results, and the CTA that finishes last joins the pieces in the order of the keys
// (so the result does not depend on timing).  An item of few tiles is not split: it goes to
// the CTA that holds its middle.
#pragma once

#include "gdn_attn.cuh"

namespace gdn {

// a CTA has at most two partial pieces: of the item its range begins inside (slot 0) and
// of the one its range ends inside (slot 1)
constexpr int kAttnSlots = 2;
constexpr int kAttnTile = 128;      // keys per tile
constexpr int kAttnMaxParts = 152;  // CTAs that share the work (one per SM)
constexpr int kAttnFan = 16;        // pieces that one CTA joins; more are joined in two levels

struct AttnGrid {
  int block;     // query tokens per item
  int sub;       // query tokens per tile of rows
  int overhead;  // cost of an item's start and end, in keys
  int whole;     // items of at most this many tiles are not split
  int snap;      // a cut nearer to an item's end than this many tiles goes to the end
  int least;     // cost below which a CTA's share is not worth a split
  int each;      // pieces of an item that are, all the same, where there are few items
};

// Quotients of costs: 32 bits where they do (a 64-bit division is some 100 instructions).
__device__ __forceinline__ long long attn_div(long long x, long long y) {
  if (((x | y) >> 32) == 0) return (unsigned)x / (unsigned)y;
  return x / y;
}

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
  if (nb == 1) return (long long)s.kv_len + g.overhead;  // as the rest would give
  const long long a = (long long)s.kv_len - s.q_len;
  const long long m = n < nb ? n : nb - 1;              // blocks of full size
  long long b0 = a < 0 ? (unsigned)-a / (unsigned)g.block : 0;              // leading blocks that see nothing
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
  const int t = y <= 0 ? 0 : (int)((unsigned long long)y / kAttnTile);
  return t < g.snap ? 0 : n - t < g.snap ? n : t;
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
  // To the item that holds cost u, in sequence s whose cost begins at `at` (by a whole warp).
  __device__ __forceinline__ void seek(const AttnArgs& p, const AttnGrid& g, int seq_index,
                                       long long at, long long u) {
    open(p, g, seq_index);
    const long long per = attn_head_cost(seq, g);
    h = (int)attn_div(u - at, per);
    const long long r = u - at - h * per;
    int lo = 0, hi = nb;  // the last block whose cost begins at or before r: in [lo, hi)
    while (hi - lo > 1) {  // 32 places at a time
      const int step = (hi - lo + 31) / 32, n = lo + (int)(threadIdx.x & 31) * step;
      const bool before = n < hi && attn_cost_before(seq, g, n) <= r;
      lo += (__popc(__ballot_sync(0xffffffffu, before)) - 1) * step;
      hi = min(hi, lo + step);
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

// The line of all costs, cut into `parts`.
struct AttnLine {
  long long total, per;
  int rest, parts;
  __device__ __forceinline__ long long cut(int c) const {
    return per * c + (unsigned)(rest * c) / (unsigned)parts;  // total * c / parts, rounded down
  }
};

// What a CTA starts from: its range [u0, u1) and the sequence that u0 lies in.
struct AttnShare {
  AttnLine line;
  long long u0, u1, seq_start;
  int seq;
};

// By one warp: the share of CTA c of `parts`.
__device__ __forceinline__ AttnShare attn_share(const AttnArgs& p, const AttnGrid& g, int c,
                                                int parts) {
  const int lane = threadIdx.x & 31;
  AttnShare r;
  long long cost = 0, mine = 0;  // of the lane's last sequence, of all of them
  int items = 0;
#pragma unroll 4
  for (int s = lane; s < p.num_seqs; s += 32) {
    const AttnSeq seq = attn_seq(p, s);
    cost = attn_head_cost(seq, g) * p.hkv;
    mine += cost;
    items = min(items + (int)min((long long)attn_blocks(seq, g.block) * p.hkv, (long long)parts),
                parts);  // (only below `parts` counts)
  }
#pragma unroll
  for (int w = 1; w < 32; w <<= 1) {
    mine += __shfl_xor_sync(0xffffffffu, mine, w);
    items = min(items + __shfl_xor_sync(0xffffffffu, items, w), parts);
  }
  // Little work is not cut into as many pieces as there are CTAs, whose join would cost more than
  // it saves: shares of `least` at least, but `each` for each item (so items that are not split
  // find a CTA each).
  if (g.each * items < parts) {
    const long long some = attn_div(mine, g.least);
    parts = some < g.each * items ? g.each * items : some < parts ? (int)some : parts;
    if (parts < 1) parts = 1;
  }
  r.line.total = mine;
  r.line.per = attn_div(mine, parts);
  r.line.rest = (int)(mine - r.line.per * parts);
  r.line.parts = parts;
  r.u0 = r.line.cut(c);
  r.u1 = r.line.cut(c + 1);
  r.seq = 0;
  r.seq_start = 0;
  if (c >= parts) r.u1 = r.u0;
  if (r.u0 >= r.u1) return r;  // no work
  long long base = 0;
  for (int s0 = 0; s0 < p.num_seqs; s0 += 32) {
    if (p.num_seqs > 32) {
      cost = s0 + lane < p.num_seqs ? attn_head_cost(attn_seq(p, s0 + lane), g) * p.hkv : 0;
    }
    long long sum = base + cost;
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, sum - base, w);
      if (lane >= w) sum += y;
    }
    const unsigned past = __ballot_sync(0xffffffffu, sum > r.u0);
    base = __shfl_sync(0xffffffffu, sum, 31);
    if (past != 0) {  // the first sequence that ends behind u0
      const int at = __ffs(past) - 1;
      r.seq = s0 + at;
      r.seq_start = __shfl_sync(0xffffffffu, sum - cost, at);
      break;
    }
  }
  return r;
}

// ---------------------------------------------------------------- partial results
// Workspace: arrival counters, then for every CTA and slot the rows of 128 fp32 sums and
// (maximum in log2 units, sum) of each row.
struct AttnCounters {
  unsigned long long arrived[kAttnMaxParts * kAttnSlots][2][2];  // [first piece][level][row tile]
};
__host__ __device__ inline size_t attn_workspace_bytes(int rows, int parts) {
  return sizeof(AttnCounters) +
         (size_t)parts * kAttnSlots * rows * (kHeadDim + 2) * sizeof(float);
}
struct AttnPartials {
  AttnCounters* counters;
  float* base;
  unsigned long long tag;  // of this launch: 48 bits, not 0 (attn_launch_tag)
  int rows;
  __device__ __forceinline__ float* sums(int piece) const {  // piece = 2 CTA + slot
    return base + (long long)piece * rows * (kHeadDim + 2);
  }
  __device__ __forceinline__ float* stats(int piece) const {
    return sums(piece) + (long long)rows * kHeadDim;
  }
};
inline AttnPartials attn_partials(void* workspace, int rows, unsigned long long tag) {
  return AttnPartials{static_cast<AttnCounters*>(workspace),
                      reinterpret_cast<float*>(static_cast<AttnCounters*>(workspace) + 1), tag,
                      rows};
}
// The tag of a launch: the host's, another one for every call, and how many failures have been
// reported on this device.  A captured graph replays its call's tag; its words are cleared by
// each replay's last arrivals, but not where a bounded wait ran out: such a replay leaves words
// of partial counts behind, which the replays after the report are not to take for their own.
__device__ __forceinline__ unsigned long long attn_launch_tag(unsigned long long tag,
                                                              unsigned reported) {
  tag = (tag + reported) & 0xffffffffffffull;
  return tag != 0 ? tag : 1;
}
// A counter's memory may hold anything before the launch: only a word with this launch's tag
// counts.  Each CTA of an item sees to the tag well before it arrives (attn_pieces), so that an
// arrival is one addition (a loop of compare-and-swaps by 16 CTAs that finish together took
// 8 us).  The last of n arrivals (true) clears the word; no CTA tags it after that, since each
// does so before its own arrival.
__device__ __forceinline__ void attn_tag(unsigned long long* word, unsigned long long tag) {
  const unsigned long long was = atomicCAS(word, 0ull, tag << 16);  // cleared by an earlier launch?
  if (was != 0 && (was >> 16) != tag) atomicCAS(word, was, tag << 16);  // (or another CTA was first)
}
__device__ __forceinline__ bool attn_arrive(unsigned long long* word, int n) {
  const bool last = (int)(atomicAdd(word, 1ull) & 0xffffu) + 1 == n;
  if (last) atomicExch(word, 0ull);
  return last;
}
__device__ __forceinline__ void attn_fence() { asm volatile("fence.acq_rel.gpu;" ::: "memory"); }

// The pieces of one item, in the order of the keys, as every one of its CTAs finds them.
struct AttnPieces {
  short list[kAttnMaxParts];  // 2 CTA + slot
  int count, mine;            // mine: this CTA's place in the list
};
// By one warp, for the item at cost `start` (e keys, n tiles) and CTA `cta`; tags the counters
// that this CTA may arrive at, for `tiles` row tiles.
__device__ __forceinline__ void attn_pieces(const AttnGrid& g, const AttnLine& line,
                                            const AttnPartials& ws, long long start, int e, int n,
                                            int cta, int tiles, AttnPieces* out) {
  const int lane = threadIdx.x & 31;
  const long long end = start + e + g.overhead;
  int count = 0;
  // (the CTA of cost `start` is not before this one: a range is at most per + 1 long)
  for (int c0 = (int)attn_div(start, line.per + 1); c0 < line.parts && line.cut(c0) < end; c0 += 32) {
    const int c = c0 + lane;
    bool has = false;
    long long lo = 0;
    if (c < line.parts) {
      lo = line.cut(c);
      const long long hi = line.cut(c + 1);
      has = hi > start && lo < end &&
            attn_tile_at(g, e, n, lo > start ? lo - start : 0) < attn_tile_at(g, e, n, hi - start);
    }
    const unsigned some = __ballot_sync(0xffffffffu, has);
    if (has) {
      const int at = count + __popc(some & ((1u << lane) - 1));
      out->list[at] = (short)(2 * c + (lo > start ? 0 : 1));
      if (c == cta) out->mine = at;
    }
    count += __popc(some);
  }
  if (lane == 0) out->count = count;
  __syncwarp();
  const int level = lane >> 1, tile = lane & 1;
  if (level < (count > kAttnFan ? 2 : 1) && tile < tiles) {
    const int first = level == 0 ? out->mine / kAttnFan * kAttnFan : 0;
    attn_tag(&ws.counters->arrived[out->list[first]][level][tile], ws.tag);
  }
}

// Joins `count` <= kAttnFan pieces list[0], list[step], .. of the rows [row0, row0 + rows),
// by kWarps warps together (rows <= 32 kWarps).  First a thread takes a row's statistics and
// leaves the pieces' weights in `weights` (shared memory, attn_weight_bytes(rows)) with the
// row's place, then a warp takes R rows and U pieces at a time, all their loads in flight.
// stat(row, maximum, sum) gives what the row's weights are multiplied with, place(row) where
// it goes, out(place, lane's four columns) gets the weighted sums.
__host__ __device__ constexpr int attn_weight_bytes(int rows) {
  return rows * (kAttnFan * (int)sizeof(float) + (int)sizeof(long long));
}
template <int kWarps, int R, int U, typename Sync, typename Stat, typename Place, typename Out>
__device__ __forceinline__ void attn_merge(const AttnPartials& ws, const short* list, int step,
                                           int count, int row0, int rows, int warp,
                                           void* weights_smem, Sync&& sync, Stat&& stat, Place&& place,
                                           Out&& out) {
  long long* places = static_cast<long long*>(weights_smem);
  float* weights = reinterpret_cast<float*>(places + rows);
  const int lane = threadIdx.x & 31, r = warp * 32 + lane;
  if (r < rows) {
    float2 ml[kAttnFan];
    float M = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < kAttnFan; ++i)
      ml[i] = i < count
                  ? __ldcg(reinterpret_cast<const float2*>(ws.stats(list[i * step])) + row0 + r)
                  : make_float2(-INFINITY, 0.f);
#pragma unroll
    for (int i = 0; i < kAttnFan; ++i)
      if (ml[i].y != 0.f) M = fmaxf(M, ml[i].x);  // sum 0: the row saw nothing of the piece
#pragma unroll
    for (int i = 0; i < kAttnFan; ++i) {
      ml[i].x = ml[i].y == 0.f ? 0.f : exp2f(ml[i].x - M);
      l += ml[i].y == 0.f ? 0.f : ml[i].x * ml[i].y;
    }
    const float f = stat(row0 + r, M, l);
    places[r] = place(row0 + r);
#pragma unroll
    for (int i = 0; i < kAttnFan; ++i)
      if (i < count) weights[i * rows + r] = ml[i].y == 0.f ? 0.f : ml[i].x * f;
  }
  sync();
  for (int r0 = warp * R; r0 < rows; r0 += kWarps * R) {
    float4 o[R];
#pragma unroll
    for (int j = 0; j < R; ++j) o[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < count; i0 += U) {
      float4 x[U][R];
      float w[U][R];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const bool there = i0 + i < count;
        const float* src = ws.sums(list[(there ? i0 + i : 0) * step]) +
                           (long long)(row0 + r0) * kHeadDim + 4 * lane;
#pragma unroll
        for (int j = 0; j < R; ++j) {
          w[i][j] = there && r0 + j < rows ? weights[(i0 + i) * rows + r0 + j] : 0.f;
          x[i][j] = w[i][j] != 0.f ? __ldcg(reinterpret_cast<const float4*>(src + j * kHeadDim))
                                   : make_float4(0.f, 0.f, 0.f, 0.f);
        }
      }
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int j = 0; j < R; ++j) {
          o[j].x = fmaf(w[i][j], x[i][j].x, o[j].x);
          o[j].y = fmaf(w[i][j], x[i][j].y, o[j].y);
          o[j].z = fmaf(w[i][j], x[i][j].z, o[j].z);
          o[j].w = fmaf(w[i][j], x[i][j].w, o[j].w);
        }
    }
#pragma unroll
    for (int j = 0; j < R; ++j)
      if (r0 + j < rows) out(places[r0 + j], o[j]);
  }
}

// After a piece's partial result is written: by the kWarps warps that wrote the rows [row0,
// row0 + rows) (row tile `tile`) together, `sync` their barrier, `flag` an int of theirs in
// shared memory, `weights` attn_weight_bytes(rows) of theirs, 8-byte aligned.  The last CTA of
// an item to come here writes its output through store(place(row), four columns).
template <int kWarps, int R, int U, typename Sync, typename Place, typename Store>
__device__ __forceinline__ void attn_join(const AttnPartials& ws, const AttnPieces& pieces,
                                          int tile, int row0, int rows, int warp, volatile int* flag,
                                          void* weights, Sync&& sync, Place&& place, Store&& store) {
  const int lane = threadIdx.x & 31;
  auto arrive = [&](int first, int level, int n) {  // true in the last CTA to arrive
    sync();  // the others' rows before this thread's fence
    if (warp == 0 && lane == 0) {
      attn_fence();
      *flag = attn_arrive(&ws.counters->arrived[pieces.list[first]][level][tile], n);
      attn_fence();
    }
    sync();
    return *flag != 0;
  };
  auto whole = [](int, float, float l) { return l == 0.f ? 0.f : 1.f / l; };
  int n = pieces.count, step = 1, first = 0;
  if (n > kAttnFan) {
    first = pieces.mine / kAttnFan * kAttnFan;
    const int some = min(kAttnFan, n - first);
    if (!arrive(first, 0, some)) return;
    const int head = pieces.list[first];  // the group's result replaces its first piece
    attn_merge<kWarps, R, U>(
        ws, pieces.list + first, 1, some, row0, rows, warp, weights, sync,
        [&](int row, float M, float l) {
          reinterpret_cast<float2*>(ws.stats(head))[row] = make_float2(M, l);
          return 1.f;
        },
        [&](int row) { return (long long)row * kHeadDim; },
        [&](long long at, float4 o) {
          *reinterpret_cast<float4*>(ws.sums(head) + at + 4 * lane) = o;
        });
    n = (n + kAttnFan - 1) / kAttnFan;
    step = kAttnFan;
    if (!arrive(0, 1, n)) return;
  } else if (!arrive(0, 0, n)) {
    return;
  }
  attn_merge<kWarps, R, U>(ws, pieces.list, step, n, row0, rows, warp, weights, sync, whole, place,
                           store);
}

}  // namespace gdn
