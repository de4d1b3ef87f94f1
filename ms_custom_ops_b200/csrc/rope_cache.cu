// rope_and_cache: per-head norm, position rotation and cache write of a serving step in one pass.
//
//   n = x * w / sqrt(mean(x^2) + eps)  (only with a weight),  (a, b) -> (a c - b s, b c + a s)  per pair,
//   query rows -> query_out, key rows -> their cache slot, value rows copied; int8 caches quantised on the way.
//
// HBM-bound: every row is read once and written once, about ten float operations per element.
#include <algorithm>

#include "msco_common.cuh"

namespace msco {
namespace {

struct RopeArgs {
  const void *q, *k, *v;
  void *q_out, *k_cache, *v_cache;
  const int32_t *slots, *positions;
  const float *cos_sin;
  const void *q_weight, *k_weight;
  const float *k_descale, *v_descale;
  const int32_t *k_offset, *v_offset;
  int32_t *oob;
  int64_t tokens, slots_total, max_positions, q_stride, k_stride, v_stride;
  int q_heads, kv_heads, head_dim, rotary, block_size, layout, interleaved;
  float eps;
};

// first element of head `h` of slot `s` in a cache
__device__ __forceinline__ int64_t cache_row(const RopeArgs &a, int64_t s, int h) {
  if (a.layout == 1) return ((s / a.block_size * a.kv_heads + h) * a.block_size + s % a.block_size) * a.head_dim;
  return (s * a.kv_heads + h) * a.head_dim;
}

// rint(x / descale) - offset, saturated; NaN becomes 0 (the rule of reshape_and_cache_quant)
__device__ __forceinline__ int8_t quantise(float x, float descale, float offset) {
  const float z = rintf(__fdiv_rn(x, descale)) - offset;
  return z == z ? (int8_t)fminf(fmaxf(z, -128.f), 127.f) : (int8_t)0;
}

// Any head_dim, rotary_dim, stride and alignment: one warp per head row, elements one at a time.
template <typename T, bool I8>
__global__ void __launch_bounds__(256) rope_cache_any_kernel(RopeArgs a) {
  const int rows = a.q_heads + 2 * a.kv_heads;
  const int lane = threadIdx.x & 31;
  const int64_t total = a.tokens * rows;
  for (int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); w < total; w += (int64_t)gridDim.x * 8) {
    const int64_t t = w / rows;
    const int r = (int)(w - t * rows);
    const int kind = r < a.q_heads ? 0 : (r < a.q_heads + a.kv_heads ? 1 : 2);
    const int h = kind == 0 ? r : (kind == 1 ? r - a.q_heads : r - a.q_heads - a.kv_heads);
    const int D = a.head_dim;
    const int32_t pos = a.positions[t];
    const bool pos_ok = pos >= 0 && pos < a.max_positions;
    const int64_t slot = a.slots[t];
    const bool store = slot >= 0 && slot < a.slots_total && pos_ok;
    if (r == 0 && lane == 0 && a.oob != nullptr && (!pos_ok || slot >= a.slots_total)) atomicAdd(a.oob, 1);
    if (kind != 0 && !store) continue;
    const T *src = kind == 0 ? static_cast<const T *>(a.q) + t * a.q_stride
                             : (kind == 1 ? static_cast<const T *>(a.k) + t * a.k_stride
                                          : static_cast<const T *>(a.v) + t * a.v_stride);
    src += (int64_t)h * D;
    const T *weight = static_cast<const T *>(kind == 0 ? a.q_weight : (kind == 1 ? a.k_weight : nullptr));
    float inv = 1.f;
    if (weight != nullptr) {
      float ss = 0.f;
      for (int d = lane; d < D; d += 32) {
        const float x = to_f32(src[d]);
        ss = fmaf(x, x, ss);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      inv = 1.f / sqrtf(ss / (float)D + a.eps);
    }
    const int half = a.rotary / 2;
    const float *cs = a.cos_sin + (int64_t)(pos_ok ? pos : 0) * a.rotary;
    for (int d = lane; d < D; d += 32) {
      float y = to_f32(src[d]);
      if (weight != nullptr) y = y * inv * to_f32(weight[d]);
      if (kind != 2 && d < a.rotary) {
        const bool first = a.interleaved ? (d & 1) == 0 : d < half;
        const int i = a.interleaved ? d >> 1 : (first ? d : d - half);
        const int od = a.interleaved ? d ^ 1 : (first ? d + half : d - half);
        float other = to_f32(src[od]);
        if (weight != nullptr) other = other * inv * to_f32(weight[od]);
        const float c = cs[i], s = cs[half + i];
        y = first ? y * c - other * s : y * c + other * s;
      }
      if (kind == 0) {
        static_cast<T *>(a.q_out)[(t * a.q_heads + h) * D + d] = from_f32<T>(pos_ok ? y : 0.f);
      } else {
        const int64_t at = cache_row(a, slot, h) + d;
        void *cache = kind == 1 ? a.k_cache : a.v_cache;
        if (I8) {
          const float *ds = kind == 1 ? a.k_descale : a.v_descale;
          const int32_t *of = kind == 1 ? a.k_offset : a.v_offset;
          const int c = h * D + d;
          static_cast<int8_t *>(cache)[at] = quantise(y, ds[c], of != nullptr ? (float)of[c] : 0.f);
        } else {
          static_cast<T *>(cache)[at] = from_f32<T>(y);
        }
      }
    }
  }
}

// eight consecutive 16-bit values
template <typename T>
__device__ __forceinline__ void unpack8(const uint4 &v, float (&x)[8]) {
  const T *e = reinterpret_cast<const T *>(&v);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_f32(e[i]);
}
// head_dim 64 / 128 / 256, 16-byte rows.  D / 8 lanes own a head row; such a group takes ROWS consecutive head rows of one
// token, all queries, all keys or all values (ROWS divides both head counts), so that the cosines, sines and weights are
// fetched once for them and all loads are in flight before the first is used.  A lane has eight consecutive elements
// (interleaved: both of each pair); when whole heads are rotated by halves (SPLIT) it has four of each half instead, so
// that no pair lies in two lanes -- otherwise the other element comes from rotary / 16 lanes on.
// Bound by issue slots and shuffles before memory: with eight consecutive elements, one shuffle per element and a choice
// of source per row the prefill step of 16384 tokens took 110 to 130 us.
template <typename T, int D, bool I8, bool INTER, bool NORM, bool SPLIT, int ROWS>
__global__ void __launch_bounds__(256) rope_cache_vec_kernel(RopeArgs a) {
  constexpr int L = D / 8;
  const int lane = threadIdx.x & 31, sub = threadIdx.x & (L - 1);
  const unsigned mask = L == 32 ? 0xffffffffu : ((1u << (L & 31)) - 1) << (lane & ~(L - 1));
  const int q_chunks = a.q_heads / ROWS, kv_chunks = a.kv_heads / ROWS, chunks = q_chunks + 2 * kv_chunks;
  const uint32_t group = blockIdx.x * (256 / L) + threadIdx.x / L;  // (fewer than 2^32: the launch checks)
  const uint32_t t = group / (uint32_t)chunks;
  if (t >= a.tokens) return;  // whole groups: the shuffles below stay inside one
  const int ch = (int)(group - t * chunks);
  const int kind = ch < q_chunks ? 0 : (ch < q_chunks + kv_chunks ? 1 : 2);
  const int h0 = (kind == 0 ? ch : (kind == 1 ? ch - q_chunks : ch - q_chunks - kv_chunks)) * ROWS;
  const int d0 = SPLIT ? sub * 4 : sub * 8, d1 = SPLIT ? D / 2 + sub * 4 : d0 + 4;  // first of the lane's two quads
  const T *src = static_cast<const T *>(kind == 0 ? a.q : (kind == 1 ? a.k : a.v)) +
                 (int64_t)t * (kind == 0 ? a.q_stride : (kind == 1 ? a.k_stride : a.v_stride)) + h0 * D;
  uint4 raw[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    if (SPLIT) {
      const uint2 lo = __ldg(reinterpret_cast<const uint2 *>(src + i * D + d0));
      const uint2 hi = __ldg(reinterpret_cast<const uint2 *>(src + i * D + d1));
      raw[i] = make_uint4(lo.x, lo.y, hi.x, hi.y);
    } else {
      raw[i] = __ldg(reinterpret_cast<const uint4 *>(src + i * D + d0));
    }
  }
  const int32_t pos = __ldg(a.positions + t), slot = __ldg(a.slots + t);
  const bool pos_ok = pos >= 0 && pos < a.max_positions;
  const bool store = slot >= 0 && slot < a.slots_total && pos_ok;
  if (ch == 0 && sub == 0 && a.oob != nullptr && (!pos_ok || slot >= a.slots_total)) atomicAdd(a.oob, 1);
  if (kind != 0 && !store) return;
  // where the rows go: consecutive rows lie `step` elements apart
  int64_t at, step = D;
  if (kind == 0) {
    at = ((int64_t)t * a.q_heads + h0) * D;
  } else if (a.layout == 1) {
    const uint32_t blk = (uint32_t)slot / (uint32_t)a.block_size, off = (uint32_t)slot - blk * a.block_size;
    at = (((int64_t)blk * a.kv_heads + h0) * a.block_size + off) * D;
    step = (int64_t)a.block_size * D;
  } else {
    at = ((int64_t)slot * a.kv_heads + h0) * D;
  }
  T *dst16 = static_cast<T *>(kind == 0 ? a.q_out : (kind == 1 ? a.k_cache : a.v_cache)) + at;
  int8_t *dst8 = static_cast<int8_t *>(kind == 1 ? a.k_cache : a.v_cache) + at;
  const float *ds = kind == 1 ? a.k_descale : a.v_descale;
  const int32_t *of = kind == 1 ? a.k_offset : a.v_offset;
  auto put8 = [&](int i, const float (&y)[8]) {  // quantised row i
    const int c = (h0 + i) * D;
    uint32_t q8[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int d = c + (n == 0 ? d0 : d1);
      const float4 s4 = __ldg(reinterpret_cast<const float4 *>(ds + d));
      const int4 o4 = of != nullptr ? __ldg(reinterpret_cast<const int4 *>(of + d)) : make_int4(0, 0, 0, 0);
      q8[n] = (uint32_t)(uint8_t)quantise(y[4 * n], s4.x, (float)o4.x) |
              (uint32_t)(uint8_t)quantise(y[4 * n + 1], s4.y, (float)o4.y) << 8 |
              (uint32_t)(uint8_t)quantise(y[4 * n + 2], s4.z, (float)o4.z) << 16 |
              (uint32_t)(uint8_t)quantise(y[4 * n + 3], s4.w, (float)o4.w) << 24;
    }
    *reinterpret_cast<uint32_t *>(dst8 + i * step + d0) = q8[0];
    *reinterpret_cast<uint32_t *>(dst8 + i * step + d1) = q8[1];
  };
  auto put16 = [&](int i, const uint4 &v) {
    if (SPLIT) {
      *reinterpret_cast<uint2 *>(dst16 + i * step + d0) = make_uint2(v.x, v.y);
      *reinterpret_cast<uint2 *>(dst16 + i * step + d1) = make_uint2(v.z, v.w);
    } else {
      *reinterpret_cast<uint4 *>(dst16 + i * step + d0) = v;
    }
  };
  if (kind == 2) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      if (I8) {
        float x[8];
        unpack8<T>(raw[i], x);
        put8(i, x);
      } else {
        put16(i, raw[i]);
      }
    }
    return;
  }
  if (kind == 0 && !pos_ok) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i) put16(i, make_uint4(0, 0, 0, 0));
    return;
  }
  const int half = a.rotary >> 1;
  const bool turns = SPLIT || d0 < a.rotary, first = d0 < half;
  constexpr int kN = INTER || SPLIT ? 4 : 8;  // pairs that this lane has a part in
  float c[kN], sn[kN];
  const float *cs = a.cos_sin + (int64_t)pos * a.rotary + (INTER ? d0 >> 1 : (SPLIT || first ? d0 : d0 - half));
#pragma unroll
  for (int i = 0; i < kN; i += 4) {
    const float4 cc = turns ? __ldg(reinterpret_cast<const float4 *>(cs + i)) : make_float4(1, 1, 1, 1);
    const float4 ss = turns ? __ldg(reinterpret_cast<const float4 *>(cs + half + i)) : make_float4(0, 0, 0, 0);
    c[i] = cc.x; c[i + 1] = cc.y; c[i + 2] = cc.z; c[i + 3] = cc.w;
    sn[i] = ss.x; sn[i + 1] = ss.y; sn[i + 2] = ss.z; sn[i + 3] = ss.w;
  }
  const int other = turns ? (first ? lane + half / 8 : lane - half / 8) : lane;
  const T *weight = static_cast<const T *>(kind == 0 ? a.q_weight : a.k_weight);
  const bool norms = NORM && weight != nullptr;
  float w[8];
  if (norms) {
    const uint2 lo = __ldg(reinterpret_cast<const uint2 *>(weight + d0)), hi = __ldg(reinterpret_cast<const uint2 *>(weight + d1));
    unpack8<T>(make_uint4(lo.x, lo.y, hi.x, hi.y), w);
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    float x[8], y[8];
    unpack8<T>(raw[i], x);
    if (norms) {
      float ss = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) ss = fmaf(x[k], x[k], ss);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
      const float inv = __frsqrt_rn(ss * (1.f / D) + a.eps);
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = x[k] * inv * w[k];
    }
    if (SPLIT) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        y[k] = x[k] * c[k] - x[k + 4] * sn[k];
        y[k + 4] = x[k + 4] * c[k] + x[k] * sn[k];
      }
    } else if (INTER) {
#pragma unroll
      for (int k = 0; k < 8; k += 2) {
        y[k] = x[k] * c[k / 2] - x[k + 1] * sn[k / 2];
        y[k + 1] = x[k + 1] * c[k / 2] + x[k] * sn[k / 2];
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float o = __shfl_sync(mask, x[k], other);
        y[k] = first ? x[k] * c[k % kN] - o * sn[k % kN] : x[k] * c[k % kN] + o * sn[k % kN];
      }
    }
    if (I8 && kind == 1) {
      put8(i, y);
    } else {
      put16(i, make_uint4(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]), pack2<T>(y[4], y[5]), pack2<T>(y[6], y[7])));
    }
  }
}

template <typename T, int D, bool I8, bool INTER, bool NORM, bool SPLIT>
int launch_vec(const RopeArgs &a, cudaStream_t st) {
  constexpr int L = D / 8;
  const int rows = a.q_heads + 2 * a.kv_heads;
  auto blocks_of = [&](int per) { return (a.tokens * (rows / per) * L + 255) / 256; };
  if (blocks_of(1) > (int64_t)(0xffffffffu / (256 / L))) return fail(MSCO_ERR_INVALID_ARG, "rope_and_cache: too many rows");
  // several rows per group once that still fills the GPU several times over, one row where latency counts
  const int by = (a.q_heads | a.kv_heads) & 3;
  if (by == 0 && blocks_of(4) >= 148 * 8)
    rope_cache_vec_kernel<T, D, I8, INTER, NORM, SPLIT, 4><<<(unsigned)blocks_of(4), 256, 0, st>>>(a);
  else if ((by & 1) == 0 && blocks_of(2) >= 148 * 8)
    rope_cache_vec_kernel<T, D, I8, INTER, NORM, SPLIT, 2><<<(unsigned)blocks_of(2), 256, 0, st>>>(a);
  else
    rope_cache_vec_kernel<T, D, I8, INTER, NORM, SPLIT, 1><<<(unsigned)blocks_of(1), 256, 0, st>>>(a);
  MSCO_CUDA_CHECK(cudaGetLastError());
  return MSCO_OK;
}

template <typename T, bool I8>
int launch_any(const RopeArgs &a, cudaStream_t st) {
  const int64_t warps = a.tokens * (a.q_heads + 2 * a.kv_heads);
  const int64_t blocks = std::min<int64_t>((warps + 7) / 8, 148 * 8 * 4);
  rope_cache_any_kernel<T, I8><<<(unsigned)blocks, 256, 0, st>>>(a);
  MSCO_CUDA_CHECK(cudaGetLastError());
  return MSCO_OK;
}

template <typename T, int D, bool I8>
int launch_vec_of(const RopeArgs &a, cudaStream_t st) {
  const bool norm = a.q_weight != nullptr || a.k_weight != nullptr;
  if (a.interleaved) return norm ? launch_vec<T, D, I8, true, true, false>(a, st) : launch_vec<T, D, I8, true, false, false>(a, st);
  if (a.rotary == D) return norm ? launch_vec<T, D, I8, false, true, true>(a, st) : launch_vec<T, D, I8, false, false, true>(a, st);
  return norm ? launch_vec<T, D, I8, false, true, false>(a, st) : launch_vec<T, D, I8, false, false, false>(a, st);
}

// 16-byte pieces: every row address, and pairs that stay inside a lane or lie whole lanes apart
template <typename T, bool I8>
int launch_rope(const RopeArgs &a, cudaStream_t st) {
  const uintptr_t all = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                        reinterpret_cast<uintptr_t>(a.q_out) | reinterpret_cast<uintptr_t>(a.k_cache) |
                        reinterpret_cast<uintptr_t>(a.v_cache) | reinterpret_cast<uintptr_t>(a.cos_sin) |
                        reinterpret_cast<uintptr_t>(a.q_weight) | reinterpret_cast<uintptr_t>(a.k_weight) |
                        reinterpret_cast<uintptr_t>(a.k_descale) | reinterpret_cast<uintptr_t>(a.v_descale) |
                        reinterpret_cast<uintptr_t>(a.k_offset) | reinterpret_cast<uintptr_t>(a.v_offset);
  const bool strides = a.tokens == 1 || ((a.q_stride | a.k_stride | a.v_stride) & 7) == 0;
  const bool vec = (all & 15) == 0 && strides && a.rotary % (a.interleaved ? 8 : 16) == 0;
  if (vec && a.head_dim == 128) return launch_vec_of<T, 128, I8>(a, st);
  if (vec && a.head_dim == 64) return launch_vec_of<T, 64, I8>(a, st);
  if (vec && a.head_dim == 256) return launch_vec_of<T, 256, I8>(a, st);
  return launch_any<T, I8>(a, st);
}

}  // namespace
}  // namespace msco

using namespace msco;

extern "C" int msco_rope_and_cache(const MscoRopeDesc *desc, const void *query, const void *key, const void *value,
                                   void *query_out, void *key_cache, void *value_cache, const int32_t *slot_mapping,
                                   const int32_t *positions, const float *cos_sin, const void *q_weight,
                                   const void *k_weight, const float *k_descale, const int32_t *k_offset,
                                   const float *v_descale, const int32_t *v_offset, int32_t *oob_count, void *stream) {
  if (desc == nullptr) return fail(MSCO_ERR_INVALID_ARG, "rope_and_cache: NULL argument");
  const MscoRopeDesc &d = *desc;
  if (d.dtype != MSCO_DTYPE_F16 && d.dtype != MSCO_DTYPE_BF16)
    return fail(MSCO_ERR_INVALID_ARG, "rope_and_cache: query / key / value must be float16 or bfloat16");
  const bool i8 = d.cache_dtype == MSCO_DTYPE_I8;
  if (!i8 && d.cache_dtype != d.dtype)
    return fail(MSCO_ERR_INVALID_ARG, "rope_and_cache: the caches must have the type of key / value or be int8");
  if (d.num_q_heads < 0 || d.num_kv_heads <= 0 || d.num_q_heads > (1 << 20) || d.num_kv_heads > (1 << 20))
    return fail(MSCO_ERR_INVALID_ARG, "rope_and_cache: bad head counts (%d, %d)", d.num_q_heads, d.num_kv_heads);
  if (d.head_dim <= 0 || d.head_dim > 512)
    return fail(MSCO_ERR_INVALID_ARG, "rope_and_cache: head_dim must be in (0, 512], got %d", d.head_dim);
  if (d.rotary_dim < 0 || d.rotary_dim > d.head_dim || d.rotary_dim % 2 != 0)
    return fail(MSCO_ERR_INVALID_ARG, "rope_and_cache: rotary_dim must be even and at most head_dim, got %d", d.rotary_dim);
  if (d.block_size <= 0 || d.num_blocks <= 0 || d.num_blocks > ((int64_t)1 << 40) / d.block_size)
    return fail(MSCO_ERR_INVALID_ARG, "rope_and_cache: bad cache geometry");
  if (d.cache_layout != 0 && d.cache_layout != 1)
    return fail(MSCO_ERR_INVALID_ARG, "rope_and_cache: cache_layout must be 0 (block_size major) or 1 (head major)");
  if (d.num_tokens < 0 || d.num_tokens > 0x7fffffffLL || d.max_positions < 0)
    return fail(MSCO_ERR_INVALID_ARG, "rope_and_cache: bad token or position count");
  if (!(d.eps >= 0.f)) return fail(MSCO_ERR_INVALID_ARG, "rope_and_cache: eps must not be negative");
  if (d.num_tokens == 0) return MSCO_OK;
  const int64_t q_row = (int64_t)d.num_q_heads * d.head_dim, kv_row = (int64_t)d.num_kv_heads * d.head_dim;
  if (d.num_tokens > 1 && (d.q_stride < q_row || d.k_stride < kv_row || d.v_stride < kv_row))
    return fail(MSCO_ERR_INVALID_ARG, "rope_and_cache: the token strides must be at least one row");
  if (key == nullptr || value == nullptr || key_cache == nullptr || value_cache == nullptr || slot_mapping == nullptr ||
      positions == nullptr || (cos_sin == nullptr && d.rotary_dim > 0 && d.max_positions > 0) ||
      (d.num_q_heads > 0 && (query == nullptr || query_out == nullptr)))
    return fail(MSCO_ERR_INVALID_ARG, "rope_and_cache: NULL tensor");
  if (i8 && (k_descale == nullptr || v_descale == nullptr))
    return fail(MSCO_ERR_INVALID_ARG, "rope_and_cache: int8 caches need k_descale and v_descale");
  RopeArgs a = {};
  a.q = query; a.k = key; a.v = value; a.q_out = query_out; a.k_cache = key_cache; a.v_cache = value_cache;
  a.slots = slot_mapping; a.positions = positions; a.cos_sin = cos_sin; a.q_weight = q_weight; a.k_weight = k_weight;
  a.k_descale = k_descale; a.v_descale = v_descale; a.k_offset = k_offset; a.v_offset = v_offset; a.oob = oob_count;
  a.tokens = d.num_tokens; a.slots_total = d.num_blocks * d.block_size; a.max_positions = d.max_positions;
  a.q_stride = d.q_stride; a.k_stride = d.k_stride; a.v_stride = d.v_stride;
  a.q_heads = d.num_q_heads; a.kv_heads = d.num_kv_heads; a.head_dim = d.head_dim; a.rotary = d.rotary_dim;
  a.block_size = d.block_size; a.layout = d.cache_layout; a.interleaved = d.interleaved != 0; a.eps = d.eps;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool f16 = d.dtype == MSCO_DTYPE_F16;
  if (i8) return f16 ? launch_rope<__half, true>(a, st) : launch_rope<__nv_bfloat16, true>(a, st);
  return f16 ? launch_rope<__half, false>(a, st) : launch_rope<__nv_bfloat16, false>(a, st);
}
