// Causal softmax attention for few query rows: decode steps and draft tokens over a paged
// cache (or very short prompts).  Bound by the HBM traffic of K and V.
//
// An item has up to R = 8, 16 or 32 rows: the query heads of one key/value head for as many
// tokens as fit.  Every SM runs one CTA whose twelve consumer warps split the keys: a group of
// W = R / 8 warps shares a chunk of 16 W keys, each warp for 8 of the rows.  Each group has two chunks in shared memory (192 KB a CTA) that its own lanes fill by
// cp.async, the next one while they work, across the ends of pieces; a box of 16 keys is too
// small for TMA, whose issue then bounds the loads (2 KB boxes measured 5.2 TB/s from eight
// lanes and 2.0 TB/s from one).
//
// The products are taken transposed, S^T = K Q^T and O^T = V^T P^T, in mma.sync m16n8k16: the
// keys (then the columns of V) fill the 16 and the rows the 8, so that a decode step's eight
// heads of a group waste nothing, and a row's maximum, sum and scale stay in one thread's
// columns.  P^T needs a transposed fragment, one movmatrix per 8 keys.  The warps are bound by
// latency (the tensor pipe is 13 % busy): what counts is instructions per chunk and warps.
// A 128-row tcgen05 tile would be mostly padding and a longer chain of hand-overs.
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

constexpr int kTile = kAttnTile;
constexpr int kWorks = 4;   // pieces handed out ahead
constexpr int kWarps = 12;  // that consume
constexpr int kRing = 2;    // chunks of a group in shared memory
constexpr size_t smem_bytes(int rows) {  // ring, queries (later the join's weights)
  static_assert(attn_weight_bytes(1) <= kHeadDim * 2, "the weights take the queries' place");
  return 1024 + (size_t)kRing * 16 * kWarps * 2 * kHeadDim * 2 + (size_t)rows * kHeadDim * 2;
}

__device__ unsigned int g_rows_error = 0;
__device__ unsigned int g_rows_reports = 0;  // of failures, so far (attn_launch_tag)

struct RowsArgs {
  AttnArgs a;
  AttnGrid g;
  AttnPartials ws;
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
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// An 8 x 8 matrix of bf16 (a row's column pair in each thread), transposed.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <int W>
__global__ void __launch_bounds__((kWarps + 1) * 32, 1)
    attn_rows_kernel(const __grid_constant__ RowsArgs p) {
  constexpr int kGroups = kWarps / W;
  constexpr int kRound = 16 * kWarps;          // keys that all groups take together
  constexpr int kChunk = 16 * W;               // keys
  constexpr int kHalf = kChunk * 128;          // 64 columns of a chunk's K or V
  constexpr int kStage = 4 * kHalf;            // K, V
  constexpr int kRowsItem = 8 * W;
  static_assert(kRowsItem * kHeadDim * 4 <= kStage, "the join goes through a stage");
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t work_full[kWorks], pieces_full[kWorks], work_empty[kWorks];
  __shared__ Work works[kWorks];
  __shared__ float2 stat[kGroups][kRowsItem];  // (maximum, sum) of each group's rows
  __shared__ uint32_t kept[kGroups];           // the stage that holds a group's output
  __shared__ int failed_flag, joining;
  const uint32_t ring0 = smem_u32(raw) + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  const uint32_t sq = ring0 + kRing * kRound * 2 * kHeadDim * 2;  // the item's queries
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const AttnArgs& a = p.a;
  const AttnGrid& g = p.g;
  const int grp = a.hq / a.hkv;
  volatile int* failed = &failed_flag;

  if (tid == 0) {
    for (int i = 0; i < kWorks; ++i) {
      mbar_init(&work_full[i], 1);
      mbar_init(&pieces_full[i], 1);
      mbar_init(&work_empty[i], kWarps);
    }
    fence_mbar_init();
    failed_flag = 0;
  }
  __syncthreads();

  if (warp == kWarps) {
    // ------------------------------------------------------------------ the pieces
    AttnPartials ws = p.ws;
    ws.tag = attn_launch_tag(ws.tag, g_rows_reports);
    const AttnShare share = attn_share(a, g, blockIdx.x, gridDim.x);
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
      bool found = false, split = false;
      long long start = 0;
      int keys = 0;
      while (more && !found) {
        const int e = cur.keys(g), tiles = (e + kTile - 1) / kTile;
        const int t0 = attn_tile_at(g, e, tiles, u0 > cur.start ? u0 - cur.start : 0);
        const int t1 = attn_tile_at(g, e, tiles, u1 - cur.start);
        // an item without keys belongs to the CTA that it starts in (its rows are zeroed)
        found = t1 > t0 || (tiles == 0 && cur.start >= u0);
        if (found) {
          const int slot = (t0 == 0 && t1 == tiles) ? -1 : (u0 > cur.start ? 0 : 1);
          split = slot >= 0;
          start = cur.start;
          keys = e;
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
      // needed at the piece's end only
      if (split)
        attn_pieces(g, share.line, ws, start, keys, (keys + kTile - 1) / kTile, blockIdx.x, 1,
                    &w->pieces);
      __syncwarp();
      if (lane == 0) mbar_arrive(&pieces_full[n % kWorks]);
    }
  } else {
    // ------------------------------------------------------------------ consumers
    const int group = warp / W;
    const int mkey = (warp % W) * 16;              // the chunk's keys that the warp loads
    const int mrow = (warp % W) * 8;               // its first row
    const int fr = lane >> 2, fc = 2 * (lane & 3);  // row and column pair of a fragment
    const uint32_t stages = ring0 + group * kRing * kStage;
    uint32_t done = 0;  // chunks consumed
    bool ok = true;

    // The loads run ahead of the pieces, up to the last one handed out.  Lane l < 16 knows the
    // page of key l of the warp's 16 in the next chunk, lane 16 + l too (the first half makes
    // K's addresses, the other V's).
    uint32_t issued = 0, ln = 0;
    bool opened = false, more = true;  // piece ln has a next chunk; pieces left
    int lkey = 0, lk1 = 0, lend = 0, lkv0 = 0, page = 0;
    int lrow = 0, lidx = 0;  // of the lane's key: row of its page, place of the page in the table
    const int* ltable = nullptr;
    const __nv_bfloat16* lbase = nullptr;
    const long long page_stride = !a.paged ? 0 : lane < 16 ? a.k_page_stride : a.v_page_stride;
    const long long row_stride = a.paged ? (long long)a.hkv * kHeadDim
                                         : (lane < 16 ? a.k_stride : a.v_stride);
    const bool runs = !a.paged || a.page_size % 16 == 0;  // a warp's 16 keys are in one page
    uint32_t at_sw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      at_sw[i] = (uint32_t)((lane & 7) ^ ((2 * i + (lane >> 4)) & 7)) << 4;
    const int step_pages = a.paged ? kRound / a.page_size : 0;
    const int step_rows = kRound - step_pages * (a.paged ? a.page_size : 0);
    auto find_page = [&] {  // asked for a chunk ahead of its use
      if (a.paged) page = lkey + mkey + (lane & 15) < lend ? __ldg(ltable + lidx) : -1;
    };
    // To the next chunk; `n` is the piece at hand (a wait for one kWorks later would not end,
    // and the place of one before it may hold another by now: a group without chunks in
    // several pieces on end comes late).
    auto open = [&](uint32_t n) {
      if (ln < n) ln = n;
      while (!opened && more && ln < n + kWorks) {
        if (!__all_sync(0xffffffffu, mbar_wait(&work_full[ln % kWorks], ln / kWorks & 1))) {
          ok = more = false;
          break;
        }
        const Work& w = works[ln % kWorks];
        more = w.live;
        lkey = w.k0 + group * kChunk;
        lk1 = w.k1;
        if (more && lkey < lk1) {
          opened = true;
          lend = w.kv_len;
          lkv0 = w.kv0;
          const int key = lkey + mkey + (lane & 15);
          lidx = a.paged ? key / a.page_size : 0;
          lrow = a.paged ? key - lidx * a.page_size : lkv0 + key;
          lbase = (lane < 16 ? a.k : a.v) + (long long)w.head * kHeadDim;
          ltable = a.paged ? a.block_table + w.seq * a.table_stride : nullptr;
          find_page();
        } else {
          ++ln;
        }
      }
      return opened;
    };
    auto issue = [&] {  // its loads: keys behind the last one and missing pages become zeros
      const bool there = lkey + mkey + (lane & 15) < lend &&
                         (!a.paged || (page >= 0 && page < a.num_pages));
      const unsigned long long from = reinterpret_cast<unsigned long long>(
          there ? lbase + page * page_stride + lrow * row_stride : a.k);
      const uint32_t valid = __ballot_sync(0xffffffffu, there);
      // lane: 16 bytes of a row, two rows at a time; `at_sw`: their swizzled places
      const int c = lane & 15, hi = lane >> 4;
      const uint32_t dst = stages + issued % kRing * kStage + (c >> 3) * kHalf + (mkey + hi) * 128;
      if (runs && valid == 0xffffffffu) {  // 16 rows one after the other
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const long long step = __shfl_sync(0xffffffffu, row_stride, 16 * kv) * 2;
          unsigned long long at = __shfl_sync(0xffffffffu, from, 16 * kv) + hi * step + 16 * c;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16;" ::"r"(
                             dst + 2 * kv * kHalf + 256 * i + at_sw[i & 3]),
                         "l"(at)
                         : "memory");
            at += 2 * step;
          }
        }
      } else {
#pragma unroll
        for (int kv = 0; kv < 2; ++kv)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int src = 16 * kv + 2 * i + hi;
            const unsigned long long at = __shfl_sync(0xffffffffu, from, src) + 16 * c;
            asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(
                             dst + 2 * kv * kHalf + 256 * i + at_sw[i & 3]),
                         "l"(at), "r"((valid >> src & 1) ? 16 : 0)
                         : "memory");
          }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      ++issued;
      lkey += kRound;
      if (lkey < lk1) {
        lidx += step_pages;
        lrow += step_rows;
        if (a.paged && lrow >= a.page_size) {
          lrow -= a.page_size;
          ++lidx;
        }
        find_page();
      } else {
        opened = false;
        ++ln;
      }
    };
    while (issued < kRing - 1 && open(0)) issue();
    for (uint32_t n = 0;; ++n) {
      if (!__all_sync(0xffffffffu, mbar_wait(&work_full[n % kWorks], n / kWorks & 1))) ok = false;
      if (group_or(1, kWarps * 32, !ok)) {  // all warps leave together
        ok = false;
        break;
      }
      const Work& w = works[n % kWorks];
      if (!w.live) break;
      while (issued < done + kRing - 1 && open(n)) issue();
      // the item's queries, as K and V: 64 columns of all rows, 128-byte swizzle
      for (int i = tid; i < kRowsItem * 16; i += kWarps * 32) {
        const int r = i >> 4, c = i & 15, tok = r / grp;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (r < g.sub * grp && tok < w.toks)
          x = __ldg(reinterpret_cast<const uint4*>(a.q + (w.row0 + tok) * a.q_stride +
                                                   ((long long)w.head * grp + r % grp) * kHeadDim) +
                    c);
        st_shared_v4(sq + (c >> 3) * kRowsItem * 128 + sw128(r, c & 7), x.x, x.y, x.z, x.w);
      }
      group_sync(1, kWarps * 32);
      // the thread's rows (columns of the transposed products) are mrow + fc and the next one:
      // keys that they see.  The queries, the B operand, stay in registers.
      int lim[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int r = mrow + fc + k, tok = r / grp;
        lim[k] = r < g.sub * grp && tok < w.toks ? max(w.lim0 + tok, 0) : 0;
      }
      uint32_t qk[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i)  // two steps of 16 columns
        ldmatrix4(sq + (i >> 1) * kRowsItem * 128 +
                      sw128(mrow + (lane & 7), 4 * (i & 1) + (lane >> 3)),
                  qk[i]);
      float o[8][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
      const int first = w.k0 + group * kChunk;
      const uint32_t begun = done;
      for (int key0 = first; key0 < w.k1; key0 += kRound) {
        // this chunk has arrived, the only one on its way
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        if constexpr (W > 1) group_sync(2 + group, W * 32);
        else __syncwarp();
        if (open(n)) issue();  // into the stage of the chunk before, which everyone has left
        const uint32_t kb = stages + done % kRing * kStage, vb = kb + 2 * kHalf;
        ++done;
        // 16 keys, or twice 16 at a time: one vote, and chains that overlap (128 sequences of up
        // to 8000 tokens, 4 draft tokens each: 155 -> 144 us)
        constexpr int G = W == 1 ? 1 : 2;
#pragma unroll
        for (int c = 0; c < W; c += G) {
          float s[G][4] = {}, s2[G][4] = {};  // chains of four products
#pragma unroll
          for (int i = 0; i < 8; ++i) {
#pragma unroll
            for (int x = 0; x < G; ++x) {
              uint32_t kf[4];
              ldmatrix4(kb + (i >> 2) * kHalf +
                            sw128(16 * (c + x) + (lane & 15), 2 * (i & 3) + (lane >> 4)),
                        kf);
              mma16816((i & 1) ? s2[x] : s[x], kf, qk[i >> 1][2 * (i & 1)],
                       qk[i >> 1][2 * (i & 1) + 1]);
            }
          }
          const int k0 = key0 + 16 * c + fr;  // key of s[0][0], s[0][1]; k0 + 8 of the others
          float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int x = 0; x < G; ++x)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              s[x][k] = (s[x][k] + s2[x][k]) * a.scale_log2;
              if (k0 + 16 * x + (k & 2) * 4 >= lim[k & 1]) s[x][k] = -INFINITY;
              top[k & 1] = fmaxf(top[k & 1], s[x][k]);
            }
          const bool up = top[0] > m[0] + kRaise || top[1] > m[1] + kRaise;
          if (__any_sync(0xffffffffu, up)) {  // some row's maximum has to be raised
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              float x = top[k];
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
              x = fmaxf(x, m[k]);
              const float f = m[k] == -INFINITY ? 0.f : ex2(m[k] - x);
              m[k] = x;
              l[k] *= f;
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                o[i][k] *= f;
                o[i][k + 2] *= f;
              }
            }
          }
          uint32_t pt[G][2];
#pragma unroll
          for (int x = 0; x < G; ++x) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              s[x][k] = ex2(s[x][k] - (m[k & 1] == -INFINITY ? 0.f : m[k & 1]));
              l[k & 1] += s[x][k];
            }
            pt[x][0] = transpose8x8(pack_bf16(s[x][0], s[x][1]));
            pt[x][1] = transpose8x8(pack_bf16(s[x][2], s[x][3]));
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {  // 16 columns of V
#pragma unroll
            for (int x = 0; x < G; ++x) {
              uint32_t vf[4];
              ldmatrix4_trans(vb + (i >> 2) * kHalf +
                                  sw128(16 * (c + x) + (lane >> 4) * 8 + (lane & 7),
                                        2 * (i & 3) + ((lane >> 3) & 1)),
                              vf);
              mma16816(o[i], vf, pt[x][0], pt[x][1]);
            }
          }
        }
      }
      // the group's result into the stage that it consumed last: column d of row r at
      // d ^ 8 (r / 2 % 4), so that a store's rows fall on different banks
      const bool has = done > begun;
      const uint32_t last = (done - 1) % kRing;
      if (lane == 0) kept[group] = last;  // the same from each of the group's warps
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float x = l[k];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        if (fr == 0) stat[group][mrow + fc + k] = make_float2(m[k], x);
      }
      if constexpr (W > 1) group_sync(2 + group, W * 32);  // the others have read V
      if (has) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int r = mrow + fc + (k & 1), d = 16 * i + fr + (k & 2) * 4;
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(stages + last * kStage + r * 512 +
                                                         4 * (d ^ ((r >> 1 & 3) << 3))),
                         "f"(o[i][k])
                         : "memory");
          }
      }
      if (group_or(1, kWarps * 32, !ok)) {
        ok = false;
        break;
      }
      // join: 16 threads per row, 8 columns each
#pragma unroll 1
      for (int r = tid / 16; r < kRowsItem; r += kWarps * 2) {
        const int nt = tid % 16;
        float M = -INFINITY;
#pragma unroll
        for (int k = 0; k < kGroups; ++k) M = fmaxf(M, stat[k][r].x);
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, l = 0.f;
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
          const float2 ml = stat[k][r];
          const uint32_t src = ring0 + (k * kRing + kept[k]) * kStage + r * 512 +
                               32 * (nt ^ (r >> 1 & 3));
          const uint4 u = ld_shared_v4(src), v = ld_shared_v4(src + 16);
          if (ml.y == 0.f) continue;  // saw nothing: no sums of its there
          const float f = ex2(ml.x - M);
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
      // (every thread waits for every piece: the phases stay in step)
      if (!__all_sync(0xffffffffu, mbar_wait(&pieces_full[n % kWorks], n / kWorks & 1))) ok = false;
      if (group_or(1, kWarps * 32, !ok)) {  // everyone has read the stages and statistics
        ok = false;
        break;
      }
      if (w.slot >= 0) {
        const int head0 = w.head * grp;
        attn_join<kWarps, 1, 16>(
            p.ws, w.pieces, 0, 0, w.toks * grp, warp, &joining,
            raw + (sq - smem_u32(raw)),  // the queries are done with
            [] { group_sync(1, kWarps * 32); },
            [&](int row) {
              return (w.row0 + row / grp) * a.o_stride +
                     ((long long)head0 + row % grp) * kHeadDim;
            },
            [&](long long at, float4 x) {
              *reinterpret_cast<uint2*>(a.out + at + 4 * lane) =
                  make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
            });
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&work_empty[n % kWorks]);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (!ok) {
      *failed = 1;
      if (lane == 0) atomicOr(&g_rows_error, kErrLoad);
    }
  }
}

template <int W>
cudaError_t launch(const AttnArgs& a, int sms, void* workspace, unsigned long long tag,
                   cudaStream_t st) {
  const int grp = a.hq / a.hkv;
  RowsArgs p{};
  p.a = a;
  constexpr int rows = 8 * W;
  p.g.sub = rows / grp;
  p.g.block = p.g.sub;
  // Over 176 batches of 1 to 150 sequences of up to 8000 keys, 1 and 4 tokens each, an overhead
  // of 128 takes 2.1 % more time and of 768 0.8 % more, cuts moved over 5 tiles 1.9 % more; 32 x 4
  // draft tokens take 48 us, 52.5 where no cut is moved, 51 where every item may be split.  16
  // pieces of an item are what one level joins: one sequence of 4096 keys 15.3 us, with 4 17.2.
  p.g.overhead = 512;
  p.g.whole = 8;
  p.g.snap = 3;
  p.g.least = 768;
  p.g.each = 16;
  p.ws = attn_partials(workspace, rows, tag);
  static thread_local int set_for = -1;  // the attribute belongs to the device's context
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (set_for != dev) {
    e = cudaFuncSetAttribute(attn_rows_kernel<W>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)smem_bytes(rows));
    if (e != cudaSuccess) return e;
    set_for = dev;
  }
  attn_rows_kernel<W><<<sms, (kWarps + 1) * 32, smem_bytes(rows), st>>>(p);
  return cudaGetLastError();
}

}  // namespace

bool count_attn_rows_report() {
  unsigned v = 0;
  if (cudaMemcpyFromSymbol(&v, g_rows_reports, sizeof(v)) != cudaSuccess) return false;
  ++v;
  return cudaMemcpyToSymbol(g_rows_reports, &v, sizeof(v)) == cudaSuccess;
}

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
  return rows == 8    ? launch<1>(p, sms, workspace, tag, st)
         : rows == 16 ? launch<2>(p, sms, workspace, tag, st)
                      : launch<4>(p, sms, workspace, tag, st);
}

}  // namespace gdn
