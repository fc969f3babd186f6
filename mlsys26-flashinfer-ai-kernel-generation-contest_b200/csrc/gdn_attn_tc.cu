// Causal softmax attention on the tensor cores: packed prompts and chunks over a paged cache.
//
//   S = scale Q K^T,  P = 2^(S - m),  l = sum P,  O = P V / l
// over tiles of 128 keys with a running maximum m per row.  A tile of 128 rows holds the
// query heads of one key/value head for 128 / group tokens (all of them read the same keys),
// and a CTA works on two such tiles: while one's scores go through the exponential (16 per
// clock and SM), the tensor cores multiply for the other.  A row's scores are taken 64 keys at
// a time, into two buffers, so that a tile's next product never waits for its own softmax.  A
// block of one tile of rows ("twin") gives its key tiles to both halves of the CTA in turn,
// whose results are merged at the end.
//
// Warps 0-3 and 4-7: softmax of tile 0 and 1, one row per thread, scores read from TMEM and
// P written back over them as the bf16 A operand of the second product.  Warps 8 and 11: issue
// the products of tile 0 and 1.  Warp 9: loads K and V tiles by TMA into a ring of four (K and
// V in turn), Q once per item.  Warp 10: finds the pieces of work, two ahead.  TMEM: S0 S1 O0
// O1, 128 columns each.
//
// Bound by the chain of each row tile, scores -> TMEM read -> maximum -> exponentials -> P ->
// product, of which two are in flight: for 128 keys of both tiles the products take 2048 clocks
// and the exponentials 2048 (16 a clock; 1536 with a quarter of them on the FMA pipe), and the
// pipes are 55 % and 45 % busy.  One prompt of 16384 tokens (16 / 2 heads): 0.91 to 0.96 ms in
// bursts, 1.15 to 1.21 PFLOP/s (cuBLAS 1.68), and 1.04 to 1.09 call after call, 1.01 to 1.06
// (cuBLAS 1.39): the power limit leaves 1650 of 1965 MHz.
//
// The maximum that a row's sums are relative to is raised only when the new one exceeds it
// by 2^8: P then stays below 2^8 and the sums in fp32 lose nothing, and the rescaling of O
// (a round trip through the registers) is rare.  The sum l adds the fp32 values of P; the
// product takes them rounded to bf16 (relative 2^-8, as the output's own rounding).
//
// Key rows behind kv_len in a sequence's last tile can hold anything: their scores are
// replaced, and their rows of V are zeroed in shared memory (0 * inf is not 0).
#include "gdn_attn_dev.cuh"
#include "gdn_attn_sched.cuh"
#include "gdn_prefill.cuh"

namespace gdn {
namespace {

using namespace sm100;

constexpr int kRows = 128;             // rows of a tile
constexpr int kTile = kAttnTile;       // keys of a tile
constexpr int kPart = 64;              // keys that a row's scores are taken for at once
constexpr int kStages = 4;             // K / V ring
constexpr int kHalfBytes = 128 * 128;  // 64 columns of 128 rows, 128-byte swizzle
constexpr int kTileBytes = 2 * kHalfBytes;
constexpr int kThreads = 384;          // 168 registers a thread at launch: 64512
// the softmax warps hold a row of scores: 256 x 216 + 128 x 72 registers = 64512
constexpr int kSoftmaxRegs = 216, kOtherRegs = 72;

__device__ unsigned int g_attn_error = 0;
__device__ unsigned int g_attn_reports = 0;  // of failures, so far (attn_launch_tag)

constexpr int kWorks = 2;  // items handed out ahead
struct Bars {
  uint64_t q_full[2], q_empty;
  uint64_t kv_full[kStages], kv_empty[kStages];
  uint64_t s_full[2][2], p_ready[2][2], pv_done[2], o_full[2];
  uint64_t work_full[kWorks], pieces_full[kWorks], work_empty[kWorks];
  uint64_t twin_ready, twin_done;
  uint64_t drain[2];
};
// One piece of an item, for all roles.
struct Work {
  long long row0;  // query row of the block's first token
  int seq, head;
  int toks;        // tokens of the block
  int kv0, kv_len;  // first key row (packed prompts), keys of the sequence
  int lim0;        // keys that the block's first token sees (may be negative); one more each
  int t0, t1;      // key tiles of the piece
  int end[2];      // of which row tile 0 / 1 needs those below
  int slot;        // partial results' slot, -1: the piece is the whole item
  bool twin;       // one row tile: both halves of the CTA work on it, on key tiles in turn
  bool live;       // false: behind the last one
  AttnPieces pieces;  // of the item, where it has more than this one
};
struct Shared {
  Bars bars;
  Work work[kWorks];
  uint32_t tmem;
  int failed, joining[2];
  float2 twin[kRows];  // (maximum, sum) of the second half's rows
};
constexpr int kStageOut = 4096;         // a softmax warp's buffer on the way out
static_assert(attn_weight_bytes(kRows) <= 4 * kStageOut, "the join uses the buffers");
constexpr size_t kSmemBytes = 1024 + 2 * kTileBytes + kStages * kTileBytes + 8 * kStageOut;

struct TcArgs {
  AttnArgs a;
  AttnGrid g;
  AttnPartials ws;
  int box;  // key rows per TMA box
};

// The piece of item `cur` inside [u0, u1), written by lane 0 of a whole warp.
enum PieceOf { kNone, kWhole, kPartial };
__device__ __forceinline__ PieceOf piece_of(const AttnCursor& cur, const AttnGrid& g,
                                         const AttnShare& share, Work* w) {
  const long long u0 = share.u0, u1 = share.u1;
  const int e = cur.keys(g);
  const int n = (e + kTile - 1) / kTile;
  const int t0 = attn_tile_at(g, e, n, u0 > cur.start ? u0 - cur.start : 0);
  const int t1 = attn_tile_at(g, e, n, u1 - cur.start);
  // an item without keys belongs to the CTA that it starts in (its rows are zeroed)
  if (t1 <= t0 && !(n == 0 && cur.start >= u0)) return kNone;
  const int slot = (t0 == 0 && t1 == n) ? -1 : (u0 > cur.start ? 0 : 1);
  const PieceOf found = slot < 0 ? kWhole : kPartial;
  if ((threadIdx.x & 31) != 0) return found;
  const int first = cur.b * g.block;
  w->row0 = cur.seq.q0 + first;
  w->seq = cur.s;
  w->head = cur.h;
  w->toks = min(g.block, cur.seq.q_len - first);
  w->kv0 = (int)cur.seq.q0;
  w->kv_len = cur.seq.kv_len;
  w->lim0 = cur.seq.kv_len - cur.seq.q_len + first + 1;
  w->t0 = t0;
  w->t1 = t1;
#pragma unroll
  for (int t = 0; t < 2; ++t) {  // a row tile sees what its last token sees
    const int toks = min(w->toks - t * g.sub, g.sub);
    const int sees = toks > 0 ? w->lim0 + t * g.sub + toks - 1 : 0;
    w->end[t] = min(t1, sees > 0 ? (sees + kTile - 1) / kTile : 0);
  }
  w->slot = slot;
  w->twin = w->toks <= g.sub;
  w->live = true;
  return found;
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// One lane of a converged warp, the same each time.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}
// mbar_wait that also gives up when another role has.
__device__ __forceinline__ bool mbar_wait_or(uint64_t* bar, uint32_t parity, volatile int* failed) {
  for (uint32_t i = 0; i < (1u << 24); ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255u) == 255u && *failed) return false;
  }
  return false;
}

__device__ __forceinline__ float max3_nan(float x, float y, float z) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
__device__ __forceinline__ float max_of(const float (&s)[2][32]) {  // NaN if any is
  float m[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {  // four chains
    const float(&x)[32] = s[k >> 1];
    const int o = 16 * (k & 1);
    m[k] = max3_nan(x[o], x[o + 1], x[o + 2]);
#pragma unroll
    for (int i = 3; i < 15; i += 2) m[k] = max3_nan(m[k], x[o + i], x[o + i + 1]);
    m[k] = max3_nan(m[k], x[o + 15], x[o + 15]);
  }
  return max3_nan(max3_nan(m[0], m[1], m[2]), m[3], m[3]);
}

// 2^x of a finite pair, below 2^9 (from 2^-126 up; less gives 2^-126), on the FMA pipe: the
// nearest integer n comes out of the sum with 1.5 2^23, and 2^(x - n) on [-1/2, 1/2] is a
// cubic, fitted by reweighted least squares to a relative error of 7.5e-5 at most, a
// fiftieth of the rounding to bf16 that follows.
__device__ __forceinline__ uint64_t exp2_pair(uint64_t x) {
  const float2 v = unpair(x);
  const uint64_t y = pair(fmaxf(v.x, -126.f), fmaxf(v.y, -126.f));
  const uint64_t big = pair(12582912.f, 12582912.f), less = pair(-12582912.f, -12582912.f);
  const uint64_t n = add2(y, big);
  const uint64_t f = fma2(add2(n, less), pair(-1.f, -1.f), y);
  uint64_t r = fma2(f, pair(0.0551716685f, 0.0551716685f), pair(0.242611125f, 0.242611125f));
  r = fma2(r, f, pair(0.693260968f, 0.693260968f));
  r = fma2(r, f, pair(0.999928057f, 0.999928057f));
  const float2 p = unpair(r), k = unpair(n);
  return pair(__int_as_float(__float_as_int(p.x) + (__float_as_int(k.x) << 23)),
              __int_as_float(__float_as_int(p.y) + (__float_as_int(k.y) << 23)));
}

// P = 2^(scale s + shift) of a row's part into TMEM (bf16, over the scores); returns the sum.
// With kMixed a quarter of the exponentials go to the FMA pipe: 16 a clock is what the
// special-function units of an SM give, which is just what the products take.  (A quarter or
// none of them: the 16384-token prompt 986 or 1042 us on average of 12 runs in turn, chunks over
// pages 330 or 322, and 343 with half.)
constexpr int kMixEvery = 4;  // pairs
template <bool kMixed>
__device__ __forceinline__ float exponentials(const float (&s)[2][32], float scale, float shift,
                                              uint32_t ts) {
  const uint64_t scale2 = pair(scale, scale), shift2 = pair(shift, shift);
  uint64_t sum[2] = {0, 0};
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t pk[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint64_t x = fma2(pair(s[c][2 * i], s[c][2 * i + 1]), scale2, shift2);
      uint64_t y;
      if (kMixed && i % kMixEvery == kMixEvery - 1) {
        y = exp2_pair(x);
      } else {
        const float2 v = unpair(x);
        y = pair(ex2(v.x), ex2(v.y));
      }
      sum[i & 1] = add2(sum[i & 1], y);
      const float2 v = unpair(y);
      pk[i] = pack_bf16(v.x, v.y);
    }
    tmem_st16(ts + 16 * c, pk);
  }
  const float2 v = unpair(add2(sum[0], sum[1]));
  return v.x + v.y;
}

// Where a K or V tile's 128 keys lie in a stage (8-row groups of 64 columns, 1024 bytes each):
// packed prompts one half of the columns after the other, pages both halves of a group.
template <bool kPaged>
struct TileLayout {
  static constexpr uint32_t kHalf = kPaged ? 1024 : kHalfBytes;  // to the other 64 columns
  static constexpr uint32_t kGroup = kPaged ? 2048 : 1024;       // to the next 8 keys
  __device__ static __forceinline__ uint32_t row(uint32_t r) {
    return (r >> 3) * kGroup + (r & 7) * 128;
  }
};

template <bool kPaged>
__global__ void __launch_bounds__(kThreads, 1)
    attn_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                   const __grid_constant__ CUtensorMap mv, const TcArgs p) {
  extern __shared__ uint8_t raw[];
  __shared__ Shared sh;
  uint8_t* tiles = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  const uint32_t sq = smem_u32(tiles);
  const uint32_t skv = sq + 2 * kTileBytes, sout = skv + kStages * kTileBytes;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const AttnArgs& a = p.a;
  const AttnGrid& g = p.g;
  const int grp = a.hq / a.hkv;
  using Layout = TileLayout<kPaged>;

  if (tid == 0) {
    Bars& b = sh.bars;
    for (int t = 0; t < 2; ++t) {
      mbar_init(&b.q_full[t], 1);
      for (int h = 0; h < 2; ++h) {
        mbar_init(&b.s_full[t][h], 1);
        mbar_init(&b.p_ready[t][h], 4);  // a warp arrives as one
      }
      mbar_init(&b.pv_done[t], 1);
      mbar_init(&b.drain[t], 1);
      mbar_init(&b.o_full[t], 1);
    }
    mbar_init(&b.q_empty, 2);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&b.kv_full[i], 1);
      mbar_init(&b.kv_empty[i], 2);  // the two issuing warps
    }
    for (int i = 0; i < kWorks; ++i) {
      mbar_init(&b.work_full[i], 1);
      mbar_init(&b.pieces_full[i], 1);
      mbar_init(&b.work_empty[i], 11);  // loader, two issuers, eight softmax warps
    }
    mbar_init(&b.twin_ready, 4);
    mbar_init(&b.twin_done, 4);
    fence_mbar_init();
    sh.failed = 0;
    tma_prefetch_desc(&mq);
    tma_prefetch_desc(&mk);
    tma_prefetch_desc(&mv);
  }
  if (warp == 8) {
    tmem_alloc(&sh.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  volatile int* failed = &sh.failed;
  Bars& bars = sh.bars;

  // Every role takes the same pieces in the same order.  K tile i of the CTA is ring entry
  // 2 i, its V entry 2 i + 1.
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 10) {
      // ------------------------------------------------------------------ the pieces
      AttnPartials ws = p.ws;
      ws.tag = attn_launch_tag(ws.tag, g_attn_reports);
      const AttnShare share = attn_share(a, g, blockIdx.x, gridDim.x);
      AttnCursor cur;
      bool more = share.u0 < share.u1;
      if (more) cur.seek(a, g, share.seq, share.seq_start, share.u0);
      for (uint32_t n = 0;; ++n) {
        if (n >= kWorks && !__all_sync(0xffffffffu, mbar_wait(&bars.work_empty[n % kWorks],
                                                              (n / kWorks - 1) & 1)))
          break;
        if (__any_sync(0xffffffffu, *failed)) break;
        Work* w = &sh.work[n % kWorks];
        PieceOf found = kNone;
        long long start = 0;
        int keys = 0, toks = 0;
        while (more && found == kNone) {
          found = piece_of(cur, g, share, w);
          start = cur.start;
          keys = cur.keys(g);
          toks = cur.seq.q_len - cur.b * g.block;
          more = cur.next(a, g) && cur.start < share.u1;
        }
        if (lane == 0 && found == kNone) w->live = false;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.work_full[n % kWorks]);
        if (found == kNone) break;
        // needed at the piece's end only
        if (found == kPartial)
          attn_pieces(g, share.line, ws, start, keys, (keys + kTile - 1) / kTile, blockIdx.x,
                      toks > g.sub ? 2 : 1, &w->pieces);
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.pieces_full[n % kWorks]);
      }
    } else if (warp == 9) {
      // ------------------------------------------------------------------ loads
      uint32_t ring = 0, items = 0;
      bool ok = true;
      for (uint32_t n = 0;; ++n) {
        ok = mbar_wait(&bars.work_full[n % kWorks], n / kWorks & 1);
        const Work& w = sh.work[n % kWorks];  // handed back when its loads are issued
        ok = __all_sync(0xffffffffu, ok && !*failed);
        if (!ok || !w.live) break;
        if (w.t1 <= w.t0) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.work_empty[n % kWorks]);
          continue;
        }
        if (items > 0)
          ok = __all_sync(0xffffffffu, mbar_wait(&bars.q_empty, (items - 1) & 1));
        if (!ok) break;
        if (lane == 0) {
          for (int t = 0; t < 2; ++t) {
            if (w.end[t] <= w.t0) continue;  // the row tile has nothing to do
            mbar_arrive_expect_tx(&bars.q_full[t], 2 * g.sub * grp * 128);
            for (int h = 0; h < 2; ++h)
              tma_load_3d(sq + t * kTileBytes + h * kHalfBytes, &mq, &bars.q_full[t], 64 * h,
                          w.head * grp, (int)w.row0 + t * g.sub);
          }
        }
        ++items;
        const int* table = kPaged ? a.block_table + w.seq * a.table_stride : nullptr;
        const int x = w.head * kHeadDim;
        // lane i: the page of the tile's box i, asked for a tile ahead
        const int kv_len = w.kv_len, boxes = kTile / p.box;
        auto page_of = [&](int j) {
          const int key = j * kTile + lane * p.box;
          if (!kPaged || lane >= boxes || key >= kv_len) return -1;  // -1: not used
          return __ldg(table + key / a.page_size);
        };
        int page = page_of(w.t0);
        for (int j = w.t0; j < w.t1 && ok; ++j) {
          const int next = j + 1 < w.t1 ? page_of(j + 1) : -1;
          for (int kv = 0; kv < 2; ++kv) {
            const uint32_t st = ring % kStages;
            if (ring >= kStages) ok = mbar_wait(&bars.kv_empty[st], (ring / kStages - 1) & 1);
            ok = ok && !*failed;
            if (!__all_sync(0xffffffffu, ok)) {
              ok = false;
              break;
            }
            if (lane == 0) mbar_arrive_expect_tx(&bars.kv_full[st], kTileBytes);
            __syncwarp();
            const uint32_t dst = skv + st * kTileBytes;
            const CUtensorMap* m = kv ? &mv : &mk;
            if constexpr (kPaged) {
              if (lane < boxes) {
                const int key = j * kTile + lane * p.box;
                tma_load_5d(dst + lane * p.box * 256, m, &bars.kv_full[st], 0, 0, 2 * w.head,
                            key % a.page_size / 8,
                            (unsigned)page < (unsigned)a.num_pages ? page : -1);  // none: zeros
              }
            } else if (lane < 2) {
              tma_load_2d(tiles + (dst - sq) + lane * kHalfBytes, m, &bars.kv_full[st],
                          x + 64 * lane, w.kv0 + j * kTile);
            }
            ++ring;
          }
          page = next;
        }
        if (!ok) break;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.work_empty[n % kWorks]);
      }
      if (!ok) {
        *failed = 1;
        if (lane == 0) atomicOr(&g_attn_error, kErrLoad);
      }
      if (!ok) {
        // copies in flight write into this block's memory: wait for them before it ends
        for (uint32_t i = ring > kStages ? ring - kStages : 0; i < ring; ++i)
          mbar_wait(&bars.kv_full[i % kStages], (i / kStages) & 1, 1u << 20);
      }
    } else if (warp == 8 || warp == 11) {
      // ------------------------------------------------------------------ products
      // A warp for each row tile (or, for twins, each half of the key tiles).  The whole warp
      // walks the tiles, so that addresses and descriptors stay in uniform registers; one
      // elected lane issues.  (A single lane that did both took 100 cycles for each product,
      // which last 64.)
      const int t = warp == 8 ? 0 : 1;
      constexpr uint32_t idesc_s = umma_idesc_bf16(128, kPart, false, false);
      constexpr uint32_t idesc_o = umma_idesc_bf16(128, 128, false, true);
      const uint64_t qdesc = umma_desc_k(sq), kdesc = umma_desc_sw128(skv, 16, Layout::kGroup);
      const uint64_t vdesc = umma_desc_sw128(skv, Layout::kHalf, Layout::kGroup);
      constexpr uint32_t kStep = kTileBytes >> 4;  // of a descriptor, to the next tile
      const uint32_t td = __shfl_sync(0xffffffffu, tmem, 0) + 128 * t;
      uint32_t tile0 = 0;         // K / V tiles before this piece
      uint32_t np = 0;            // p_ready phases used
      uint32_t nq0 = 0, nq1 = 0;  // q_full phases used
      bool ok = true;
      unsigned why = 0;
      auto wait = [&](uint64_t* bar, uint32_t phase, unsigned err) {
        if (!ok) return;
        ok = __all_sync(0xffffffffu, mbar_wait_or(bar, phase & 1, failed));
        if (!ok) why = err;
      };
      auto commit = [&](uint64_t* bar) {
        if (elect_one()) umma_commit(bar);
      };
      auto wait_kv = [&](uint32_t entry) {
        wait(&bars.kv_full[entry % kStages], entry / kStages, kErrLoad);
      };
      // this warp has no use for a ring entry (arrived only when it is there: in step)
      auto skip_kv = [&](uint32_t entry) {
        wait_kv(entry);
        if (ok && elect_one()) mbar_arrive(&bars.kv_empty[entry % kStages]);
      };
      auto scores = [&](uint64_t q, uint32_t entry, int h) {  // S_h = Q K^T, keys 64 h ..
        const uint64_t k = kdesc + entry % kStages * kStep + h * (kPart / 8 * Layout::kGroup >> 4);
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            umma_bf16(td + kPart * h, q + (((i >> 2) * kHalfBytes + (i & 3) * 32) >> 4),
                      k + (((i >> 2) * Layout::kHalf + (i & 3) * 32) >> 4), idesc_s, i > 0);
          }
          umma_commit(&bars.s_full[t][h]);
        }
      };
      auto values = [&](uint32_t entry, int h, bool first) {  // O += P_h V, keys 64 h ..
        const uint64_t v = vdesc + entry % kStages * kStep + h * (kPart / 8 * Layout::kGroup >> 4);
        wait(&bars.p_ready[t][h], np, kErrTensor);
        tc_fence_after();
        if (ok && elect_one()) {
#pragma unroll
          for (int i = 0; i < kPart / 16; ++i)
            umma_bf16_tmem_a(td + 256, td + kPart * h + 8 * i, v + i * (2 * Layout::kGroup >> 4),
                             idesc_o,
                             !first || i > 0);
          umma_commit(&bars.pv_done[t]);
        }
      };
      for (uint32_t n = 0; ok; ++n) {
        wait(&bars.work_full[n % kWorks], n / kWorks, kErrLoad);
        const Work& w = sh.work[n % kWorks];
        if (!ok || !w.live) break;
        const int t0 = __shfl_sync(0xffffffffu, w.t0, 0), t1 = __shfl_sync(0xffffffffu, w.t1, 0);
        const int end0 = __shfl_sync(0xffffffffu, w.end[0], 0);
        const int end1 = __shfl_sync(0xffffffffu, w.end[1], 0);
        const bool twin = __shfl_sync(0xffffffffu, (int)w.twin, 0) != 0;
        if (lane == 0) mbar_arrive(&bars.work_empty[n % kWorks]);
        if (t1 <= t0) continue;
        if (end0 > t0) wait(&bars.q_full[0], nq0++, kErrLoad);
        if (end1 > t0) wait(&bars.q_full[1], nq1++, kErrLoad);
        // this warp's key tiles: first, first + step, .. below end
        const int first = t0 + (twin ? t : 0), step = twin ? 2 : 1;
        const int end = twin ? t1 : (t ? end1 : end0);
        const uint64_t q = qdesc + (twin ? 0 : t) * kStep;
        auto entry_of = [&](int j) { return 2 * (tile0 + j - t0); };
        int at = t0;  // ring entries of tiles before `at` are used or skipped
        auto skip_to = [&](int j) {
          for (; at < j && ok; ++at) {
            skip_kv(entry_of(at));
            skip_kv(entry_of(at) + 1);
          }
        };
        if (first < end) {
          skip_to(first);
          uint32_t k = entry_of(first);
          wait_kv(k);
          if (!ok) break;
          scores(q, k, 0);
          scores(q, k, 1);
          commit(&bars.kv_empty[k % kStages]);
          if (first + step >= end) commit(&bars.q_empty);
          for (int j = first; j < end && ok; j += step) {
            const uint32_t v = k + 1;
            const bool more = j + step < end;
            wait_kv(v);
            values(v, 0, j == first);
            if (more) {
              at = j + 1;
              skip_to(j + step);
              k = entry_of(j + step);
              wait_kv(k);
              if (!ok) break;
              scores(q, k, 0);
            }
            values(v, 1, false);
            ++np;
            if (!ok) break;
            commit(&bars.kv_empty[v % kStages]);
            if (more) {
              scores(q, k, 1);
              commit(&bars.kv_empty[k % kStages]);
              if (j + 2 * step >= end) commit(&bars.q_empty);
            } else {
              commit(&bars.o_full[t]);
            }
            at = j + 1;
          }
        } else if (ok) {
          commit(&bars.q_empty);
        }
        skip_to(t1);
        tile0 += t1 - t0;
      }
      if (!ok) {
        *failed = 1;
        if (why && lane == 0) atomicOr(&g_attn_error, why);
      }
      commit(&bars.drain[t]);  // nothing is in flight when the block ends
      mbar_wait(&bars.drain[t], 0);
    }
  } else {
    // ------------------------------------------------------------------ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int t = warp >> 2;        // tile of rows
    const int r = tid & 127;        // row
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // TMEM lane field: 32 (warp % 4)
    const uint32_t ts = tmem + 128 * t + lanes, to = tmem + 256 + 128 * t + lanes;
    uint32_t ns = 0, no = 0, nt = 0, npv = 0, tile0 = 0;
    bool ok = true;
    for (uint32_t n = 0;; ++n) {
      if (!__all_sync(0xffffffffu, mbar_wait(&bars.work_full[n % kWorks], n / kWorks & 1))) ok = false;
      if (group_or(1 + t, 128, !ok)) {  // the four warps leave together
        ok = false;
        break;
      }
      const Work& w = sh.work[n % kWorks];
      if (!w.live) break;
      const bool twin = w.twin;
      const int rt = twin ? 0 : t;            // row tile
      const int rtok = rt * g.sub + r / grp;  // token of the block
      const bool mine = r < g.sub * grp && rtok < w.toks;
      const int lim = mine ? max(w.lim0 + rtok, 0) : 0;  // keys that the row sees
      const int kv_len = w.kv_len, t0 = w.t0, t1 = w.end[rt];
      const int jb = twin ? t0 + t : t0, step = twin ? 2 : 1;  // this half's key tiles
      float m = -INFINITY, l = 0.f;  // m in log2 units
      uint32_t parts = 0;            // of the piece so far
      for (int j = jb; j < t1 && ok; j += step) {
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          ok = ok && __all_sync(0xffffffffu, mbar_wait(&bars.s_full[t][h], ns & 1));
          if (!ok) break;
          if (h == 0 && (j + 1) * kTile > kv_len) {
            // Rows of V behind the last key.  These scores were issued after the values of this
            // half's tile before, so the stage's earlier tile has long arrived and the wait
            // below is for this one (before that, its parity would be the one before last's).
            const uint32_t entry = 2 * (tile0 + j - t0) + 1;
            ok = __all_sync(0xffffffffu,
                            mbar_wait(&bars.kv_full[entry % kStages], entry / kStages & 1));
            if (ok && j * kTile + r >= kv_len) {
              const uint32_t row = skv + entry % kStages * kTileBytes + Layout::row(r);
#pragma unroll
              for (int c = 0; c < 8; ++c) {
                st_shared_v4(row + 16 * c, 0, 0, 0, 0);
                st_shared_v4(row + Layout::kHalf + 16 * c, 0, 0, 0, 0);
              }
            }
            fence_proxy_async();
            if (!ok) break;
          }
          tc_fence_after();
          const uint32_t tp = ts + kPart * h;
          float s[2][32];
          tmem_ld32(tp, s[0]);
          tmem_ld32(tp + 32, s[1]);
          tmem_wait_ld();
          const int vis = lim - j * kTile - h * kPart;  // visible columns
          const bool masked = __any_sync(0xffffffffu, vis < kPart);
          if (masked) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              s[0][i] = i < vis ? s[0][i] : -INFINITY;
              s[1][i] = 32 + i < vis ? s[1][i] : -INFINITY;
            }
          }
          const float mx = max_of(s) * a.scale_log2;  // scale > 0
          const bool raise = mx > m + kRaise;         // always for the first finite score
          if (__any_sync(0xffffffffu, raise)) {
            const float m2 = raise ? mx : m;
            const float f = m == -INFINITY ? 0.f : ex2(m - m2);
            l *= f;
            if (parts > 0) {  // O holds earlier parts: once their product is complete
              ok = __all_sync(0xffffffffu, mbar_wait(&bars.pv_done[t], (npv + parts - 1) & 1));
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < 8; ++c) {  // 16 columns at a time: few registers, rare
                uint32_t o[16];
                tmem_ld16(to + 16 * c, o);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                tmem_st16(to + 16 * c, o);
              }
            }
            m = m2;
          }
          const float mm = m == -INFINITY ? 0.f : m;
          if (masked || __any_sync(0xffffffffu, !(fabsf(mx) < INFINITY)))
            l += exponentials<false>(s, a.scale_log2, -mm, tp);
          else
            l += exponentials<true>(s, a.scale_log2, -mm, tp);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.p_ready[t][h]);
          ++parts;
        }
        ++ns;
      }
      npv += parts;
      if (t1 > jb && ok)
        ok = __all_sync(0xffffffffu, mbar_wait(&bars.o_full[t], no++ & 1));
      if (group_or(1 + t, 128, !ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int slot = w.slot;
      const bool has = t1 > jb;  // O_t holds something
      if (twin && t == 1) {      // the first half reads this half's rows and finishes them
        sh.twin[r] = has ? make_float2(m, l) : make_float2(-INFINITY, 0.f);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.twin_ready);
        if (!__all_sync(0xffffffffu, mbar_wait(&bars.twin_done, nt++ & 1))) ok = false;
      } else {
        float f0 = 1.f, f1 = 0.f;  // weights of O_t and, for twins, of O_1
        if (twin) {
          if (!__all_sync(0xffffffffu, mbar_wait(&bars.twin_ready, nt++ & 1))) ok = false;
          tc_fence_after();
          const float2 x = sh.twin[r];
          const float top = fmaxf(l == 0.f ? -INFINITY : m, x.y == 0.f ? -INFINITY : x.x);
          f0 = l == 0.f ? 0.f : ex2(m - top);
          f1 = x.y == 0.f ? 0.f : ex2(x.x - top);
          l = f0 * l + f1 * x.y;
          m = top;
        }
        const bool both = twin && t1 > t0 + 1;      // O_1 holds something
        // some key of the piece; of one whose scores are all -inf the sum is 0: zeros too
        const bool saw = mine && lim > t0 * kTile && l != 0.f;
        auto load = [&](int c, float(&o)[32]) {     // 32 columns of the row's sums, asked for
          if (has) tmem_ld32(to + 32 * c, o);
        };
        auto with_twin = [&](int c, float(&o)[32]) {
          if (both) {
            float o1[32];
            tmem_ld32(to + 128 + 32 * c, o1);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = f0 * o[i] + f1 * o1[i];
          }
        };
        // Out through the warp's buffer, 128 bytes of its 32 rows at a time: a row a thread, then
        // a row to eight lanes (a store of 32 rows takes 32 turns, one of 4 rows 4).
        const uint32_t buf = sout + warp * kStageOut;
        const int wr = (warp & 3) * 32;                                // the warp's first row
        const int rows = min(w.toks - rt * g.sub, g.sub) * grp - wr;  // that are there, if > 0
        if (rows <= 0) {
          // nothing of this warp's
        } else if (slot < 0) {
          const float inv = 1.f / l;
          const long long mine_at = (w.row0 + rtok) * a.o_stride +
                                    ((long long)w.head * grp + r % grp) * kHeadDim;
          __nv_bfloat16* at[8];  // where the lane's rows go
#pragma unroll
          for (int i = 0; i < 8; ++i)
            at[i] = a.out + __shfl_sync(0xffffffffu, mine_at, 4 * i + (lane >> 3)) + 8 * (lane & 7);
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {  // 64 columns of bf16
            float o[2][32];
            load(2 * c, o[0]);
            load(2 * c + 1, o[1]);
            tmem_wait_ld();
#pragma unroll
            for (int d = 0; d < 2; ++d) {
              with_twin(2 * c + d, o[d]);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                uint32_t pk[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  pk[k] = saw ? pack_bf16(o[d][8 * i + 2 * k] * inv, o[d][8 * i + 2 * k + 1] * inv)
                              : 0u;
                st_shared_v4(buf + sw128(lane, 4 * d + i), pk[0], pk[1], pk[2], pk[3]);
              }
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int x = 4 * i + (lane >> 3);
              const uint4 v = ld_shared_v4(buf + sw128(x, lane & 7));
              if (x < rows) *reinterpret_cast<uint4*>(at[i] + 64 * c) = v;
            }
            __syncwarp();
          }
        } else {
          // a row that saw nothing of the piece: (-inf, 0), its sums are not read
          const int piece = 2 * blockIdx.x + slot;
          float* po = p.ws.sums(piece) + (t * kRows + wr) * kHeadDim;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {  // 32 columns of fp32
            float o[32];
            load(c, o);
            tmem_wait_ld();
            with_twin(c, o);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              st_shared_v4(buf + sw128(lane, i), __float_as_uint(o[4 * i]),
                           __float_as_uint(o[4 * i + 1]), __float_as_uint(o[4 * i + 2]),
                           __float_as_uint(o[4 * i + 3]));
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int x = 4 * i + (lane >> 3);
              const uint4 v = ld_shared_v4(buf + sw128(x, lane & 7));
              if (x < rows)
                *reinterpret_cast<uint4*>(po + x * kHeadDim + 32 * c + 4 * (lane & 7)) = v;
            }
            __syncwarp();
          }
          reinterpret_cast<float2*>(p.ws.stats(piece))[t * kRows + r] =
              saw ? make_float2(m, l) : make_float2(-INFINITY, 0.f);
        }
        if (twin) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.twin_done);
        }
        const int toks = min(w.toks - t * g.sub, g.sub);
        if (slot >= 0 && toks > 0) {
          // (the entry is not used again before this warp hands it back, so the wait is for
          // this piece's phase, whatever others it left out)
          if (!__all_sync(0xffffffffu, mbar_wait(&bars.pieces_full[n % kWorks], n / kWorks & 1)))
            ok = false;
          if (group_or(1 + t, 128, !ok)) {
            ok = false;
            break;
          }
          const long long out0 = w.row0 + t * g.sub;
          attn_join<4, 8, 2>(
              p.ws, w.pieces, t, t * kRows, toks * grp, warp & 3, &sh.joining[t],
              tiles + (sout - sq) + 4 * t * kStageOut,
              [&] { group_sync(1 + t, 128); },
              [&](int row) {
                const int i = row - t * kRows;
                return (out0 + i / grp) * a.o_stride +
                       ((long long)w.head * grp + i % grp) * kHeadDim;
              },
              [&](long long at, float4 x) {
                *reinterpret_cast<uint2*>(a.out + at + 4 * lane) =
                    make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
              });
        }
      }
      tc_fence_before();
      tile0 += w.t1 - t0;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.work_empty[n % kWorks]);
    }
    if (!ok) {
      *failed = 1;
      if (lane == 0) atomicOr(&g_attn_error, kErrTensor);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(tmem, 512);
}

}  // namespace

bool count_attn_tc_report() {
  unsigned v = 0;
  if (cudaMemcpyFromSymbol(&v, g_attn_reports, sizeof(v)) != cudaSuccess) return false;
  ++v;
  return cudaMemcpyToSymbol(g_attn_reports, &v, sizeof(v)) == cudaSuccess;
}

unsigned read_attn_tc_error(bool clear) {
  unsigned v = 0;
  if (cudaMemcpyFromSymbol(&v, g_attn_error, sizeof(v)) != cudaSuccess) return ~0u;
  if (clear && v != 0) {
    const unsigned zero = 0;
    if (cudaMemcpyToSymbol(g_attn_error, &zero, sizeof(zero)) != cudaSuccess) return ~0u;
  }
  return v;
}

int attn_tc_rows() { return 2 * kRows; }

cudaError_t launch_attn_tc(const AttnArgs& a, int sms, void* workspace, unsigned long long tag,
                           cudaStream_t st) {
  const int grp = a.hq / a.hkv;
  TcArgs p{};
  p.a = a;
  p.g.sub = kRows / grp;
  p.g.block = 2 * p.g.sub;
  // Packed prompts of 16384 tokens take 288 us, with an overhead of 16 keys 418 and of 1024 318;
  // those of 8191 tokens and 8 heads 54.1, 56.0 where no cut is moved and 55.3 where every item
  // may be split.  Three chunks of up to 64 tokens over 3000: 37 us with at least 4 pieces of an
  // item, 40.3 with 2, 44.6 with 16.
  p.g.overhead = 320;
  p.g.whole = 4;
  p.g.snap = 3;
  p.g.least = 1024;
  p.g.each = 4;
  p.ws = attn_partials(workspace, 2 * kRows, tag);
  CUtensorMap mq, mk, mv;
  const long long qd[3] = {kHeadDim, a.hq, a.total_q}, qs[2] = {kHeadDim, a.q_stride};
  const int qb[3] = {64, grp, p.g.sub};
  bool ok = attn_map(&mq, a.q, 3, qd, qs, qb);
  p.box = attn_key_box(a, kTile);
  ok = ok && attn_key_maps(&mk, &mv, a, p.box);
  if (!ok) return cudaErrorInvalidValue;
  auto* kernel = a.paged ? attn_tc_kernel<true> : attn_tc_kernel<false>;
  static thread_local int set_for[2] = {-1, -1};  // the attribute belongs to the device's context
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (set_for[a.paged] != dev) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes);
    if (e != cudaSuccess) return e;
    set_for[a.paged] = dev;
  }
  kernel<<<sms, kThreads, kSmemBytes, st>>>(mq, mk, mv, p);
  return cudaGetLastError();
}

}  // namespace gdn
