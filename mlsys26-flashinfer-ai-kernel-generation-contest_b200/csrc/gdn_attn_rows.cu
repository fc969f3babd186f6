// Causal softmax attention for few query rows: decode steps and draft tokens over a paged
// cache (or very short prompts).  Bound by the HBM traffic of K and V.
//
// An item has up to R = 16, 32 or 64 rows: the query heads of one key/value head for as
// many tokens as fit.  Every SM runs one CTA whose eight consumer warps split the keys:
// with R = 16 MT, MT warps (16 rows each) share a chunk of 16 MT keys and there are 8 / MT
// such groups, each with a ring of three chunks in shared memory (192 KB in all, what keeps
// about 28 MB of loads in flight over the card) that one loader warp fills by TMA, a lane
// per group.  16 rows per mma.sync m16n8k16: the tensor work is 2 % of the time that the
// keys take to arrive, and a 128-row tcgen05 tile would be mostly padding and a longer chain
// (it measured 378 us for 128 sequences of up to 8192 tokens).
//
// Each warp keeps its own running maximum, sum and output in registers (raised lazily, as in
// the tensor-core kernel); the groups are joined through shared memory at the end of a piece,
// in the stage that each consumed last.  How the keys are shared out among the CTAs, and the
// join of split items, is in gdn_attn_sched.cuh.
#include "gdn_attn_dev.cuh"
#include "gdn_attn_sched.cuh"

namespace gdn {
namespace {

using namespace sm100;

constexpr int kWarps = 8;    // consumers
constexpr int kRing = 3;     // chunks per group
constexpr int kTile = kAttnTile;  // keys that all groups take together
constexpr int kWorks = 2;
constexpr int kThreads = (kWarps + 2) * 32;
constexpr size_t kSmemBytes = 1024 + (size_t)kRing * kTile * 2 * kHeadDim * 2;

__device__ unsigned int g_rows_error = 0;

struct RowsArgs {
  AttnArgs a;
  AttnGrid g;
  AttnPartials ws;
  int box;
};
struct Work {
  long long row0;   // query row of the block's first token
  int seq, head, toks;
  int kv0, kv_len;  // first key row (packed prompts), keys of the sequence
  int lim0;         // keys that the block's first token sees (may be negative); one more each
  int k0, k1;       // keys of the piece
  int slot;         // partial results' slot, -1: the piece is the whole item
  bool live;        // false: behind the last one
  AttnPieces pieces;  // of the item, where it has more than this one
};

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int MT>
__global__ void __launch_bounds__(kThreads, 1)
    attn_rows_kernel(const __grid_constant__ CUtensorMap mk,
                     const __grid_constant__ CUtensorMap mv, const RowsArgs p) {
  constexpr int kGroups = kWarps / MT;
  constexpr int kChunk = 16 * MT;              // keys
  constexpr int kHalf = kChunk * 128;          // 64 columns of a chunk's K or V
  constexpr int kStage = 4 * kHalf;            // K, V; also the size of a group's fp32 output
  constexpr int kRowsItem = 16 * MT;
  static_assert(kRowsItem * kHeadDim * 4 == kStage, "the join goes through a stage");
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[kGroups][kRing], empty[kGroups][kRing];
  __shared__ uint64_t work_full[kWorks], work_empty[kWorks];
  __shared__ Work works[kWorks];
  __shared__ AttnShare share;
  __shared__ float2 stat[kGroups][kRowsItem];  // (maximum, sum) of each group's rows
  __shared__ uint32_t kept[kGroups];           // the stage that holds a group's output
  __shared__ int failed_flag, joining;
  const uint32_t ring0 = smem_u32(raw) + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const AttnArgs& a = p.a;
  const AttnGrid& g = p.g;
  const int grp = a.hq / a.hkv;
  volatile int* failed = &failed_flag;

  if (tid == 0) {
    for (int i = 0; i < kGroups; ++i)
      for (int j = 0; j < kRing; ++j) {
        mbar_init(&full[i][j], 1);
        mbar_init(&empty[i][j], MT);
      }
    for (int i = 0; i < kWorks; ++i) {
      mbar_init(&work_full[i], 1);
      mbar_init(&work_empty[i], 1 + kWarps);
    }
    fence_mbar_init();
    failed_flag = 0;
    tma_prefetch_desc(&mk);
    tma_prefetch_desc(&mv);
  }
  attn_share<kThreads>(a, g, blockIdx.x, gridDim.x, &share);  // ends with __syncthreads

  if (warp == kWarps + 1) {
    // ------------------------------------------------------------------ the pieces
    const long long u0 = share.u0, u1 = share.u1;
    AttnCursor cur;
    bool more = u0 < u1;
    if (more) cur.seek(a, g, share.seq, share.seq_start, u0);
    for (uint32_t n = 0;; ++n) {
      if (n >= kWorks && !__all_sync(0xffffffffu, mbar_wait(&work_empty[n % kWorks],
                                                            (n / kWorks - 1) & 1)))
        break;
      if (__any_sync(0xffffffffu, *failed)) break;
      Work* w = &works[n % kWorks];
      bool found = false;
      while (more && !found) {
        const int e = cur.keys(g), tiles = (e + kTile - 1) / kTile;
        const int t0 = attn_tile_at(g, e, tiles, u0 > cur.start ? u0 - cur.start : 0);
        const int t1 = attn_tile_at(g, e, tiles, u1 - cur.start);
        // an item without keys belongs to the CTA that it starts in (its rows are zeroed)
        found = t1 > t0 || (tiles == 0 && cur.start >= u0);
        if (found) {
          const int slot = (t0 == 0 && t1 == tiles) ? -1 : (u0 > cur.start ? 0 : 1);
          if (slot >= 0) attn_pieces(g, share.line, cur.start, e, tiles, blockIdx.x, &w->pieces);
          if (lane == 0) {
            const int first = cur.b * g.block;
            w->row0 = cur.seq.q0 + first;
            w->seq = cur.s;
            w->head = cur.h;
            w->toks = min(g.block, cur.seq.q_len - first);
            w->kv0 = (int)cur.seq.q0;
            w->kv_len = cur.seq.kv_len;
            w->lim0 = cur.seq.kv_len - cur.seq.q_len + first + 1;
            w->k0 = t0 * kTile;
            w->k1 = min(t1 * kTile, e);
            w->slot = slot;
          }
        }
        more = cur.next(a, g) && cur.start < u1;
      }
      if (lane == 0) w->live = found;
      __syncwarp();
      if (lane == 0) mbar_arrive(&work_full[n % kWorks]);
      if (!found) break;
    }
  } else if (warp == kWarps) {
    // ------------------------------------------------------------------ loads
    uint32_t done = 0;  // chunks of this lane's group
    bool ok = true;
    for (uint32_t n = 0;; ++n) {
      ok = mbar_wait(&work_full[n % kWorks], n / kWorks & 1);
      const Work& w = works[n % kWorks];  // handed back when its loads are issued
      ok = __all_sync(0xffffffffu, ok && !*failed);
      if (!ok || !w.live) break;
      const int* table = a.paged ? a.block_table + w.seq * a.table_stride : nullptr;
      const int x = w.head * kHeadDim;
      if (lane < kGroups) {
        for (int key0 = w.k0 + lane * kChunk; key0 < w.k1; key0 += kTile) {
          const uint32_t st = done % kRing;
          if (done >= kRing) ok = mbar_wait(&empty[lane][st], (done / kRing - 1) & 1);
          ok = ok && !*failed;
          if (!ok) break;
          mbar_arrive_expect_tx(&full[lane][st], kStage);
          const uint32_t dst = ring0 + (lane * kRing + st) * kStage;
          for (int i = 0; i < kChunk; i += p.box) {
            const int key = key0 + i;
            int row, page;
            if (table == nullptr) {
              row = w.kv0 + key;
              page = 0;
            } else {
              row = key % a.page_size;
              page = key < w.kv_len ? __ldg(table + key / a.page_size) : -1;  // -1: not used
              if (page < 0 || page >= a.num_pages) page = -1;  // no such page: zeros
            }
            for (int h = 0; h < 2; ++h) {
              tma_load_3d(dst + h * kHalf + i * 128, &mk, &full[lane][st], x + 64 * h, row, page);
              tma_load_3d(dst + (2 + h) * kHalf + i * 128, &mv, &full[lane][st], x + 64 * h, row,
                          page);
            }
          }
          ++done;
        }
      }
      __syncwarp();
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane == 0) mbar_arrive(&work_empty[n % kWorks]);
    }
    if (!ok) {
      *failed = 1;
      if (lane == 0) atomicOr(&g_rows_error, kErrLoad);
    }
    if (!ok && lane < kGroups) {
      // copies in flight write into this block's memory: wait for them before it ends
      for (uint32_t i = done > kRing ? done - kRing : 0; i < done; ++i)
        mbar_wait(&full[lane][i % kRing], i / kRing & 1, 1u << 20);
    }
  } else {
    // ------------------------------------------------------------------ consumers
    const int group = warp / MT;
    const int mrow = (warp % MT) * 16;             // first row of the warp's tile
    const int qr = lane >> 2, qc = lane & 3;       // rows qr, qr + 8; column pair of a fragment
    uint32_t done = 0;
    bool ok = true;
    for (uint32_t n = 0;; ++n) {
      ok = __all_sync(0xffffffffu, mbar_wait(&work_full[n % kWorks], n / kWorks & 1));
      if (group_or(1, kWarps * 32, !ok)) {  // all warps leave together
        ok = false;
        break;
      }
      const Work& w = works[n % kWorks];
      if (!w.live) break;
      // rows r0, r1: keys that they see, queries as the A operand
      const int r0 = mrow + qr, r1 = r0 + 8;
      const int tok0 = r0 / grp, tok1 = r1 / grp;
      const bool in0 = r0 < g.sub * grp && tok0 < w.toks, in1 = r1 < g.sub * grp && tok1 < w.toks;
      const int lim0 = in0 ? max(w.lim0 + tok0, 0) : 0, lim1 = in1 ? max(w.lim0 + tok1, 0) : 0;
      const __nv_bfloat16* q0 = a.q + (w.row0 + tok0) * a.q_stride +
                                ((long long)w.head * grp + r0 % grp) * kHeadDim + 2 * qc;
      const __nv_bfloat16* q1 = a.q + (w.row0 + tok1) * a.q_stride +
                                ((long long)w.head * grp + r1 % grp) * kHeadDim + 2 * qc;
      uint32_t qf[8][4];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        qf[i][0] = in0 ? __ldg(reinterpret_cast<const uint32_t*>(q0 + 16 * i)) : 0u;
        qf[i][1] = in1 ? __ldg(reinterpret_cast<const uint32_t*>(q1 + 16 * i)) : 0u;
        qf[i][2] = in0 ? __ldg(reinterpret_cast<const uint32_t*>(q0 + 16 * i + 8)) : 0u;
        qf[i][3] = in1 ? __ldg(reinterpret_cast<const uint32_t*>(q1 + 16 * i + 8)) : 0u;
      }
      float o[16][4];
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
      float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
      const int first = w.k0 + group * kChunk;
      const uint32_t begun = done;
      for (int key0 = first; key0 < w.k1; key0 += kTile) {
        if (done > begun) {  // the stage before is free (the last one is kept for the join)
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty[group][(done - 1) % kRing]);
        }
        const uint32_t st = done % kRing;
        ok = __all_sync(0xffffffffu, mbar_wait(&full[group][st], done / kRing & 1));
        if (!ok) break;
        ++done;
        const uint32_t kb = ring0 + (group * kRing + st) * kStage, vb = kb + 2 * kHalf;
        float s[2 * MT][4];
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
          for (int c = 0; c < MT; ++c) {  // 16 keys
            uint32_t kf[4];
            const uint32_t key = 16 * c + (lane >> 4) * 8 + (lane & 7);
            ldmatrix4(kb + (i >> 2) * kHalf + sw128(key, 2 * (i & 3) + ((lane >> 3) & 1)), kf);
            mma16816(s[2 * c], qf[i], kf[0], kf[1]);
            mma16816(s[2 * c + 1], qf[i], kf[2], kf[3]);
          }
        }
        const int c0 = key0 + 2 * qc;  // key of s[0][0]
        if (__any_sync(0xffffffffu, key0 + kChunk > lim0 || key0 + kChunk > lim1)) {
#pragma unroll
          for (int i = 0; i < 2 * MT; ++i) {
            s[i][0] = c0 + 8 * i < lim0 ? s[i][0] : -INFINITY;
            s[i][1] = c0 + 8 * i + 1 < lim0 ? s[i][1] : -INFINITY;
            s[i][2] = c0 + 8 * i < lim1 ? s[i][2] : -INFINITY;
            s[i][3] = c0 + 8 * i + 1 < lim1 ? s[i][3] : -INFINITY;
          }
        }
        float x0 = fmaxf(s[0][0], s[0][1]), x1 = fmaxf(s[0][2], s[0][3]);
#pragma unroll
        for (int i = 1; i < 2 * MT; ++i) {
          x0 = fmaxf(x0, fmaxf(s[i][0], s[i][1]));
          x1 = fmaxf(x1, fmaxf(s[i][2], s[i][3]));
        }
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2)) * a.scale_log2;
        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2)) * a.scale_log2;
        const bool up0 = x0 > m0 + kRaise, up1 = x1 > m1 + kRaise;
        if (__any_sync(0xffffffffu, up0 || up1)) {
          const float f0 = up0 ? (m0 == -INFINITY ? 0.f : ex2(m0 - x0)) : 1.f;
          const float f1 = up1 ? (m1 == -INFINITY ? 0.f : ex2(m1 - x1)) : 1.f;
          if (up0) m0 = x0;
          if (up1) m1 = x1;
          l0 *= f0;
          l1 *= f1;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            o[i][0] *= f0;
            o[i][1] *= f0;
            o[i][2] *= f1;
            o[i][3] *= f1;
          }
        }
        const float b0 = m0 == -INFINITY ? 0.f : m0, b1 = m1 == -INFINITY ? 0.f : m1;
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) {
          s[i][0] = ex2(fmaf(s[i][0], a.scale_log2, -b0));
          s[i][1] = ex2(fmaf(s[i][1], a.scale_log2, -b0));
          s[i][2] = ex2(fmaf(s[i][2], a.scale_log2, -b1));
          s[i][3] = ex2(fmaf(s[i][3], a.scale_log2, -b1));
          l0 += s[i][0] + s[i][1];
          l1 += s[i][2] + s[i][3];
        }
        const bool tail = key0 + kChunk > w.kv_len;  // rows of V behind the last key: zeroed
#pragma unroll
        for (int c = 0; c < MT; ++c) {
          const uint32_t pf[4] = {pack_bf16(s[2 * c][0], s[2 * c][1]),
                                  pack_bf16(s[2 * c][2], s[2 * c][3]),
                                  pack_bf16(s[2 * c + 1][0], s[2 * c + 1][1]),
                                  pack_bf16(s[2 * c + 1][2], s[2 * c + 1][3])};
          uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
          if (tail) {
            const int k = c0 + 16 * c;
            keep0 = (k < w.kv_len ? 0xffffu : 0u) | (k + 1 < w.kv_len ? 0xffff0000u : 0u);
            keep1 = (k + 8 < w.kv_len ? 0xffffu : 0u) | (k + 9 < w.kv_len ? 0xffff0000u : 0u);
          }
#pragma unroll
          for (int d = 0; d < 8; ++d) {  // 16 columns of V
            uint32_t vf[4];
            const uint32_t key = 16 * c + ((lane >> 3) & 1) * 8 + (lane & 7);
            ldmatrix4_trans(vb + (d >> 2) * kHalf + sw128(key, 2 * (d & 3) + (lane >> 4)), vf);
            mma16816(o[2 * d], pf, vf[0] & keep0, vf[1] & keep1);
            mma16816(o[2 * d + 1], pf, vf[2] & keep0, vf[3] & keep1);
          }
        }
      }
      // the group's result into the stage that it consumed last: row r's column pair c at
      // pair c ^ 4 (r % 4) (two rows of lanes to a bank otherwise)
      const bool has = done > begun;
      const uint32_t last = (done - 1) % kRing;
      l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
      l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
      l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
      l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
      if (lane == 0) kept[group] = last;  // the same from each of the group's warps
      if (qc == 0) {
        stat[group][r0] = make_float2(has ? m0 : -INFINITY, l0);
        stat[group][r1] = make_float2(has ? m1 : -INFINITY, l1);
      }
      if constexpr (MT > 1) group_sync(2 + group, MT * 32);  // the others have read V
      if (has) {
        const uint32_t base = ring0 + (group * kRing + last) * kStage;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint32_t c = 4 * (i ^ (qr & 3)) + qc;
          asm volatile("st.shared.v2.f32 [%0], {%1,%2};" ::"r"(base + r0 * 512 + 8 * c),
                       "f"(o[i][0]), "f"(o[i][1])
                       : "memory");
          asm volatile("st.shared.v2.f32 [%0], {%1,%2};" ::"r"(base + r1 * 512 + 8 * c),
                       "f"(o[i][2]), "f"(o[i][3])
                       : "memory");
        }
      }
      if (group_or(1, kWarps * 32, !ok)) {
        ok = false;
        break;
      }
      // join: 16 threads per row, 8 columns each
#pragma unroll 1
      for (int it = 0; it < MT; ++it) {
        const int r = it * 16 + tid / 16, nt = tid % 16;
        float M = -INFINITY;
#pragma unroll
        for (int k = 0; k < kGroups; ++k) M = fmaxf(M, stat[k][r].x);
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, l = 0.f;
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
          const float2 ml = stat[k][r];
          if (ml.y == 0.f) continue;  // saw nothing
          const float f = ex2(ml.x - M);
          const uint32_t src = ring0 + (k * kRing + kept[k]) * kStage + r * 512 +
                               32 * (nt ^ (r & 3));
          const uint4 u = ld_shared_v4(src), v = ld_shared_v4(src + 16);
          l = fmaf(f, ml.y, l);
          x[0] = fmaf(f, __uint_as_float(u.x), x[0]);
          x[1] = fmaf(f, __uint_as_float(u.y), x[1]);
          x[2] = fmaf(f, __uint_as_float(u.z), x[2]);
          x[3] = fmaf(f, __uint_as_float(u.w), x[3]);
          x[4] = fmaf(f, __uint_as_float(v.x), x[4]);
          x[5] = fmaf(f, __uint_as_float(v.y), x[5]);
          x[6] = fmaf(f, __uint_as_float(v.z), x[6]);
          x[7] = fmaf(f, __uint_as_float(v.w), x[7]);
        }
        const int tok = r / grp;
        if (w.slot < 0) {
          if (r < g.sub * grp && tok < w.toks) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            *reinterpret_cast<uint4*>(a.out + (w.row0 + tok) * a.o_stride +
                                      ((long long)w.head * grp + r % grp) * kHeadDim + 8 * nt) =
                make_uint4(pack_bf16(x[0] * inv, x[1] * inv), pack_bf16(x[2] * inv, x[3] * inv),
                           pack_bf16(x[4] * inv, x[5] * inv), pack_bf16(x[6] * inv, x[7] * inv));
          }
        } else {
          const int piece = 2 * blockIdx.x + w.slot;
          float4* po = reinterpret_cast<float4*>(p.ws.sums(piece) + r * kHeadDim + 8 * nt);
          po[0] = make_float4(x[0], x[1], x[2], x[3]);
          po[1] = make_float4(x[4], x[5], x[6], x[7]);
          if (nt == 0)
            reinterpret_cast<float2*>(p.ws.stats(piece))[r] = make_float2(M, l);
        }
      }
      fence_proxy_async();                 // the stages are next written by TMA
      group_sync(1, kWarps * 32);          // everyone has read stages, statistics and the piece
      if (lane == 0 && has) mbar_arrive(&empty[group][last]);
      if (w.slot >= 0) {
        const int head0 = w.head * grp;
        attn_join<kWarps, 2>(
            p.ws, w.pieces, 0, 0, w.toks * grp, warp, &joining,
            [] { group_sync(1, kWarps * 32); },
            [&](int row, float4 x) {
              *reinterpret_cast<uint2*>(a.out + (w.row0 + row / grp) * a.o_stride +
                                        ((long long)head0 + row % grp) * kHeadDim + 4 * lane) =
                  make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
            });
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&work_empty[n % kWorks]);
    }
    if (!ok) {
      *failed = 1;
      if (lane == 0) atomicOr(&g_rows_error, kErrLoad);
    }
  }
}

template <int MT>
cudaError_t launch(const AttnArgs& a, int sms, void* workspace, unsigned long long tag,
                   cudaStream_t st) {
  const int grp = a.hq / a.hkv;
  RowsArgs p{};
  p.a = a;
  p.g.sub = 16 * MT / grp;
  p.g.block = p.g.sub;
  p.g.sub_rows = 16 * MT;
  p.g.overhead = 128;
  p.g.whole = 4;
  p.ws = attn_partials(workspace, 16 * MT, tag);
  p.box = attn_key_box(a, 16 * MT);
  CUtensorMap mk, mv;
  if (!attn_key_maps(&mk, &mv, a, p.box)) return cudaErrorInvalidValue;
  static thread_local int set_for = -1;  // the attribute belongs to the device's context
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (set_for != dev) {
    e = cudaFuncSetAttribute(attn_rows_kernel<MT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)kSmemBytes);
    if (e != cudaSuccess) return e;
    set_for = dev;
  }
  attn_rows_kernel<MT><<<sms, kThreads, kSmemBytes, st>>>(mk, mv, p);
  return cudaGetLastError();
}

}  // namespace

unsigned read_attn_rows_error(bool clear) {
  unsigned v = 0;
  if (cudaMemcpyFromSymbol(&v, g_rows_error, sizeof(v)) != cudaSuccess) return ~0u;
  if (clear && v != 0) {
    const unsigned zero = 0;
    if (cudaMemcpyToSymbol(g_rows_error, &zero, sizeof(zero)) != cudaSuccess) return ~0u;
  }
  return v;
}

cudaError_t launch_attn_rows(const AttnArgs& p, int rows, int sms, void* workspace,
                             unsigned long long tag, cudaStream_t st) {
  return rows == 16   ? launch<1>(p, sms, workspace, tag, st)
         : rows == 32 ? launch<2>(p, sms, workspace, tag, st)
                      : launch<4>(p, sms, workspace, tag, st);
}

}  // namespace gdn
