// Per-head RMSNorm of queries and keys, the position rotation, and the write of keys and
// values to the paged cache, in one pass (the softmax-attention layers that stand between
// Gated DeltaNet layers; no counterpart in the reference).
//
// For a row x of 128 values (one token, one head), weights w and the table row (c, s) of
// the token's position:
//   y = x * rsqrt(mean(x^2) + eps) * w              (without weights: y = x)
//   (y_a, y_b) -> (y_a c_i - y_b s_i, y_b c_i + y_a s_i)   for the rd / 2 pairs
// with pairs (i, i + rd/2) or, interleaved, (2i, 2i + 1); values from rd on pass through.
// Everything is fp32 and rounded once, to bf16, at the end; a row whose squares leave fp32's
// range is taken times a power of two for its norm.  The angles come from a table
// because a position times a frequency loses the angle in 32 bits at far positions (a
// 2^-24 relative error of 10^6 radians is 0.06); the caller computes it once in 64 bits.
//
// Bound by HBM: 256 bytes in and out per row, one table row per token.  16 lanes own a row
// (16-byte accesses); the sum of squares is four shuffles, the partner of a value in the
// half layout one shuffle when rd / 2 is a multiple of 8, else a pass through shared memory.
#include "gdn_attn_dev.cuh"

namespace gdn {
namespace {

struct RopeArgs {
  const __nv_bfloat16 *q, *k, *v;
  const void* positions;
  const float* table;
  const float *q_weight, *k_weight;  // null: no normalisation
  __nv_bfloat16 *q_out, *k_out;
  const void* slots;
  __nv_bfloat16 *k_cache, *v_cache;  // null: k_out is written instead
  long long q_stride, k_stride, v_stride, qo_stride, ko_stride;
  long long k_page_stride, v_page_stride, num_slots, table_rows;
  unsigned groups;  // tokens * groups of heads
  float eps;
  int hq, hkv, rd, page_size, groups_per_token;
  int batches;  // of HPG heads in a group
  bool pos64, slot64, wide;  // wide: a lane's table values are whole 16-byte pieces
};

__device__ __forceinline__ long long load_index(const void* p, bool is64, long long i) {
  return is64 ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int*>(p)[i];
}

__device__ __forceinline__ float sum16(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 1);
  x += __shfl_xor_sync(0xffffffffu, x, 2);
  x += __shfl_xor_sync(0xffffffffu, x, 4);
  x += __shfl_xor_sync(0xffffffffu, x, 8);
  return x;
}

// 1 / sqrt(mean(x^2) + eps) of a row, of which each of 16 lanes has eight values.
__device__ __forceinline__ float inverse_rms(const uint4& v, float eps) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 x = bf2x2_to_f2(w[e]);
    ss = fmaf(x.x, x.x, ss);
    ss = fmaf(x.y, x.y, ss);
  }
  return rsqrtf(sum16(ss) * (1.f / kHeadDim) + eps);
}

// A row times a power of two, which is exact, and the norm of that: of a finite row times 2^-70
// the squares sum to less than 2^123; of a small one times 2^100 they are above 2^-66, as its
// values are multiples of 2^-133, and sum to less than 2^115.  Not inlined: rare.
struct Scaled {
  uint4 v;
  float norm;
};
__device__ __forceinline__ bool in_range(float norm) { return norm > 0.f && norm <= 0x1p46f; }
__device__ __noinline__ Scaled scaled_row(uint4 v, float norm, float eps) {
  const float f = in_range(norm) ? 1.f : norm > 0x1p46f ? 0x1p100f : 0x1p-70f;
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 x = bf2x2_to_f2(w[e]);
    const __nv_bfloat162 y = __floats2bfloat162_rn(x.x * f, x.y * f);
    w[e] = *reinterpret_cast<const uint32_t*>(&y);
  }
  return {v, inverse_rms(v, eps * f * f)};
}

enum RopeLayout { kInterleaved = 0, kHalfAligned = 1, kHalfAny = 2 };

// One half-warp per group of heads of one token, HPG at a time: the table row is read once
// for the group, a batch's loads are in flight together, and with the batch before's work.
template <int HPG, int LAYOUT, bool kNorm>
__global__ void __launch_bounds__(256, HPG > 1 ? 3 : 1) rope_kernel(const RopeArgs p) {
  __shared__ float stage[LAYOUT == kHalfAny ? 16 : 1][kHeadDim];
  const int lane = threadIdx.x & 15;
  const unsigned group = blockIdx.x * 16 + (threadIdx.x >> 4);
  const bool live = group < p.groups;
  // lanes of a dead half-warp go along with the shuffles on group 0's values
  const unsigned g = live ? group : 0, token = g / (unsigned)p.groups_per_token;
  const long long t = token;
  int h0 = (int)(g - token * p.groups_per_token) * p.batches * HPG;
  const int heads = p.hq + p.hkv + (p.k_cache != nullptr ? p.hkv : 0);

  uint4 raw[HPG];
  auto load = [&](int from) {
#pragma unroll
    for (int i = 0; i < HPG; ++i) {
      const int h = from + i;
      const __nv_bfloat16* src =
          h < p.hq ? p.q + t * p.q_stride + (long long)h * kHeadDim
          : h < p.hq + p.hkv
              ? p.k + t * p.k_stride + (long long)(h - p.hq) * kHeadDim
              : p.v + t * p.v_stride + (long long)(h - p.hq - p.hkv) * kHeadDim;
      raw[i] = h < heads ? *reinterpret_cast<const uint4*>(src + 8 * lane) : make_uint4(0, 0, 0, 0);
    }
  };
  load(h0);

  const long long pos = load_index(p.positions, p.pos64, t);
  const bool known = pos >= 0 && pos < p.table_rows;  // else: a padding token
  long long slot = -1;
  if (p.k_cache != nullptr && known) {
    slot = load_index(p.slots, p.slot64, t);
    if (slot >= p.num_slots) slot = -1;
  }
  const long long page = slot < 0            ? 0
                         : slot >> 32 == 0 ? (unsigned)slot / (unsigned)p.page_size
                                           : slot / p.page_size;
  const long long off = slot >= 0 ? slot - page * p.page_size : 0;

  // cos / sin of the lane's 8 values (1, 0 where nothing turns)
  const int half = p.rd >> 1;
  float c[8], s[8];
  const float* row = p.table + (known ? pos : 0) * (long long)p.rd;  // not read unless known
  if (p.wide) {  // the lane's 8 values turn, or none does
    const bool turns = known && 8 * lane < p.rd;
    if constexpr (LAYOUT == kInterleaved) {
      const float4 one = make_float4(1.f, 1.f, 1.f, 1.f), none = make_float4(0.f, 0.f, 0.f, 0.f);
      const float4 x = turns ? __ldg(reinterpret_cast<const float4*>(row) + lane) : one;
      const float4 y = turns ? __ldg(reinterpret_cast<const float4*>(row + half) + lane) : none;
      c[0] = c[1] = x.x; c[2] = c[3] = x.y; c[4] = c[5] = x.z; c[6] = c[7] = x.w;
      s[1] = y.x; s[3] = y.y; s[5] = y.z; s[7] = y.w;
      s[0] = -y.x; s[2] = -y.y; s[4] = -y.z; s[6] = -y.w;
    } else {
      const bool front = 8 * lane < half;  // the first of a pair takes -s of the second
      const int i = front ? 8 * lane : 8 * lane - half;
      const float4 one = make_float4(1.f, 1.f, 1.f, 1.f), none = make_float4(0.f, 0.f, 0.f, 0.f);
      const float4* pc = reinterpret_cast<const float4*>(row + (turns ? i : 0));
      const float4* ps = reinterpret_cast<const float4*>(row + half + (turns ? i : 0));
      const float4 x = turns ? __ldg(pc) : one, x2 = turns ? __ldg(pc + 1) : one;
      const float4 y = turns ? __ldg(ps) : none, y2 = turns ? __ldg(ps + 1) : none;
      const float sign = front ? -1.f : 1.f;
      c[0] = x.x; c[1] = x.y; c[2] = x.z; c[3] = x.w;
      c[4] = x2.x; c[5] = x2.y; c[6] = x2.z; c[7] = x2.w;
      s[0] = sign * y.x; s[1] = sign * y.y; s[2] = sign * y.z; s[3] = sign * y.w;
      s[4] = sign * y2.x; s[5] = sign * y2.y; s[6] = sign * y2.z; s[7] = sign * y2.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = 8 * lane + e;
      const int i = LAYOUT == kInterleaved ? d >> 1 : (d < half ? d : d - half);
      const bool turns = known && d < p.rd;
      c[e] = turns ? __ldg(row + i) : 1.f;
      s[e] = turns ? __ldg(row + half + i) : 0.f;
      // the first of a pair takes -s of the second
      if (LAYOUT == kInterleaved ? (d & 1) == 0 : d < half) s[e] = -s[e];
    }
  }
  // half layout: the lane that holds the partners
  const int step = half >> 3;
  const int partner = 8 * lane < half ? lane + step : (8 * lane < p.rd ? lane - step : lane);

  for (int b = 0;; h0 += HPG) {
    uint4 now[HPG];
#pragma unroll
    for (int i = 0; i < HPG; ++i) now[i] = raw[i];
    const bool last = ++b == p.batches;
    if (!last) load(h0 + HPG);
    // 1 / the root mean squares, and where the squares leave fp32's range, or fall below it next
    // to an eps that does not hide them (their mean is below 2^-92 then), of the row times a
    // power of two.  One vote for a batch: a branch in each head keeps the heads from overlapping
    // (32768 tokens 74 us, with this 65.9; products in pairs, without which it is 70.7).
    float norm[HPG];
    if constexpr (kNorm) {
      bool odd = false;
#pragma unroll
      for (int i = 0; i < HPG; ++i) {
        norm[i] = inverse_rms(now[i], p.eps);
        odd |= !in_range(norm[i]);
      }
      if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
        for (int i = 0; i < HPG; ++i) {
          const int h = h0 + i;
          const bool normed = h < p.hq          ? p.q_weight != nullptr
                              : h < p.hq + p.hkv ? p.k_weight != nullptr
                                                 : false;
          const Scaled z = scaled_row(now[i], normed ? norm[i] : 1.f, p.eps);
          now[i] = z.v;
          norm[i] = z.norm;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < HPG; ++i) {
      const int h = h0 + i;
      const bool is_v = h >= p.hq + p.hkv;
      float x[8];
      {
        const uint32_t w[4] = {now[i].x, now[i].y, now[i].z, now[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = bf2x2_to_f2(w[e]);
          x[2 * e] = f.x;
          x[2 * e + 1] = f.y;
        }
      }
      const float* weight = h < p.hq ? p.q_weight : p.k_weight;
      if (kNorm && weight != nullptr && !is_v) {
        const float r = norm[i];
        const float4 w0 = __ldg(reinterpret_cast<const float4*>(weight) + 2 * lane);
        const float4 w1 = __ldg(reinterpret_cast<const float4*>(weight) + 2 * lane + 1);
        const uint64_t r2 = pair(r, r);
        const uint64_t ww[4] = {pair(w0.x, w0.y), pair(w0.z, w0.w), pair(w1.x, w1.y),
                                pair(w1.z, w1.w)};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 z = unpair(mul2(pair(x[2 * e], x[2 * e + 1]), mul2(r2, ww[e])));
          x[2 * e] = z.x;
          x[2 * e + 1] = z.y;
        }
      }
      float y[8];
      if constexpr (LAYOUT == kInterleaved) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = x[e ^ 1];
      } else if constexpr (LAYOUT == kHalfAligned) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = __shfl_sync(0xffffffffu, x[e], partner, 16);
      } else {
        float* st = stage[threadIdx.x >> 4];
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 8; ++e) st[8 * lane + e] = x[e];
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int d = 8 * lane + e;
          y[e] = d < p.rd ? st[d < half ? d + half : d - half] : 0.f;
        }
      }
      uint4 o;
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = 8 * lane + 2 * e;  // rd is even: both values turn or neither does
        const float a = d < p.rd ? fmaf(x[2 * e], c[2 * e], y[2 * e] * s[2 * e]) : x[2 * e];
        const float b = d < p.rd ? fmaf(x[2 * e + 1], c[2 * e + 1], y[2 * e + 1] * s[2 * e + 1])
                                 : x[2 * e + 1];
        const __nv_bfloat162 b2 = __floats2bfloat162_rn(a, b);
        w[e] = *reinterpret_cast<const uint32_t*>(&b2);
      }
      o = is_v ? now[i] : known ? make_uint4(w[0], w[1], w[2], w[3]) : make_uint4(0, 0, 0, 0);
      if (!live || h >= heads) continue;
      __nv_bfloat16* dst;
      if (h < p.hq) {
        dst = p.q_out + t * p.qo_stride + (long long)h * kHeadDim;
      } else if (p.k_cache == nullptr) {
        dst = p.k_out + t * p.ko_stride + (long long)(h - p.hq) * kHeadDim;
      } else {
        if (slot < 0) continue;
        dst = is_v ? p.v_cache + page * p.v_page_stride +
                         (off * p.hkv + (h - p.hq - p.hkv)) * (long long)kHeadDim
                   : p.k_cache + page * p.k_page_stride +
                         (off * p.hkv + (h - p.hq)) * (long long)kHeadDim;
      }
      *reinterpret_cast<uint4*>(dst + 8 * lane) = o;
    }
    if (last) break;
  }
}

template <int HPG, bool kNorm>
cudaError_t launch_rope(const RopeArgs& p, int layout, cudaStream_t st) {
  const unsigned grid = (unsigned)((p.groups + 15) / 16);
  if (layout == kInterleaved)
    rope_kernel<HPG, kInterleaved, kNorm><<<grid, 256, 0, st>>>(p);
  else if (layout == kHalfAligned)
    rope_kernel<HPG, kHalfAligned, kNorm><<<grid, 256, 0, st>>>(p);
  else
    rope_kernel<HPG, kHalfAny, kNorm><<<grid, 256, 0, st>>>(p);
  return cudaGetLastError();
}

inline bool misaligned(const void* p, uintptr_t n) {
  return (reinterpret_cast<uintptr_t>(p) % n) != 0;
}

}  // namespace
}  // namespace gdn

extern "C" int gdn_attn_qk_norm_rope_launch(
    const void* q, const void* k, const void* v, const void* positions, int positions_int64,
    const float* rope_table, long long table_rows, const float* q_weight, const float* k_weight,
    float eps, int interleaved, void* q_out, void* k_out, const void* slots, int slots_int64,
    void* k_cache, void* v_cache, long long num_pages, int page_size, long long k_page_stride,
    long long v_page_stride, int num_tokens, int num_q_heads, int num_kv_heads, int head_size,
    int rotary_dim, long long q_stride, long long k_stride, long long v_stride,
    long long q_out_stride, long long k_out_stride, void* stream) {
  using namespace gdn;
  const long long D = kHeadDim;
  if (num_tokens < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || table_rows < 0 || !(eps >= 0.f))
    return GDN_ERR_INVALID_ARGUMENT;
  if (head_size != kHeadDim || num_q_heads % num_kv_heads != 0 || rotary_dim < 2 ||
      rotary_dim > kHeadDim || (rotary_dim & 1) != 0)
    return GDN_ERR_UNSUPPORTED;
  if (num_q_heads > (1 << 16)) return GDN_ERR_UNSUPPORTED;
  if (num_tokens == 0) return GDN_OK;
  const bool cached = k_cache != nullptr;
  if (!q || !k || !positions || (!rope_table && table_rows > 0) || !q_out)
    return GDN_ERR_INVALID_ARGUMENT;
  if (cached ? (!v || !v_cache || !slots) : !k_out) return GDN_ERR_INVALID_ARGUMENT;
  const long long qw = num_q_heads * D, kw = num_kv_heads * D;
  auto bad_rows = [](const void* p, long long stride, long long width) {
    return misaligned(p, 16) || stride < width || stride % 8 != 0;
  };
  if (bad_rows(q, q_stride, qw) || bad_rows(k, k_stride, kw) || bad_rows(q_out, q_out_stride, qw) ||
      misaligned(positions, positions_int64 ? 8 : 4) || misaligned(rope_table, 4) ||
      misaligned(q_weight, 16) || misaligned(k_weight, 16))
    return GDN_ERR_INVALID_ARGUMENT;
  if (cached) {
    if (num_pages < 0 || page_size <= 0 || bad_rows(v, v_stride, kw) ||
        bad_rows(k_cache, k_page_stride, page_size * kw) ||
        bad_rows(v_cache, v_page_stride, page_size * kw) || misaligned(slots, slots_int64 ? 8 : 4))
      return GDN_ERR_INVALID_ARGUMENT;
  } else if (bad_rows(k_out, k_out_stride, kw)) {
    return GDN_ERR_INVALID_ARGUMENT;
  }
  using B16 = __nv_bfloat16;
  RopeArgs p{};
  p.q = static_cast<const B16*>(q);
  p.k = static_cast<const B16*>(k);
  p.v = static_cast<const B16*>(v);
  p.positions = positions;
  p.table = rope_table;
  p.q_weight = q_weight;
  p.k_weight = k_weight;
  p.q_out = static_cast<B16*>(q_out);
  p.k_out = static_cast<B16*>(k_out);
  p.slots = slots;
  p.k_cache = static_cast<B16*>(k_cache);
  p.v_cache = static_cast<B16*>(v_cache);
  p.q_stride = q_stride;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.qo_stride = q_out_stride;
  p.ko_stride = k_out_stride;
  p.k_page_stride = k_page_stride;
  p.v_page_stride = v_page_stride;
  p.num_slots = cached ? num_pages * page_size : 0;
  p.table_rows = table_rows;
  p.eps = eps;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  p.rd = rotary_dim;
  p.page_size = cached ? page_size : 1;
  p.pos64 = positions_int64 != 0;
  p.slot64 = slots_int64 != 0;
  const int heads = num_q_heads + num_kv_heads * (cached ? 2 : 1);
  const int layout =
      interleaved ? kInterleaved : (rotary_dim % 16 == 0 ? kHalfAligned : kHalfAny);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  p.wide = misaligned(rope_table, 16) == 0 &&
           (interleaved ? rotary_dim % 8 == 0 : layout == kHalfAligned && rotary_dim % 16 == 0);
  // A half-warp takes all heads of a token, four at a time, where there are tokens enough to
  // fill the card (32768 tokens of 20 heads: 66.6 us, four heads a half-warp 101; 4095: 12.5 and
  // 13.1; 1777: 9.8 and 8.2), four heads where not, and one where even that leaves SMs idle (7
  // tokens: 2.5 us, four 3.5; 600: 4.9 and 4.3).
  const int hpg = (long long)num_tokens * heads <= 16 * 148 ? 1 : 4;
  p.batches = num_tokens >= 4096 ? (heads + hpg - 1) / hpg : 1;
  p.groups_per_token = (heads + hpg * p.batches - 1) / (hpg * p.batches);
  const long long groups = (long long)num_tokens * p.groups_per_token;
  if (groups > 0x7fffffffLL) return GDN_ERR_INVALID_ARGUMENT;
  p.groups = (unsigned)groups;
  const bool norm = q_weight != nullptr || k_weight != nullptr;
  const cudaError_t err = hpg == 1 ? (norm ? launch_rope<1, true>(p, layout, st)
                                           : launch_rope<1, false>(p, layout, st))
                                   : (norm ? launch_rope<4, true>(p, layout, st)
                                           : launch_rope<4, false>(p, layout, st));
  return err == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH;
}
