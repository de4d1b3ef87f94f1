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

template <typename T, bool I8>
int launch_any(const RopeArgs &a, cudaStream_t st) {
  const int64_t warps = a.tokens * (a.q_heads + 2 * a.kv_heads);
  const int64_t blocks = std::min<int64_t>((warps + 7) / 8, 148 * 8 * 4);
  rope_cache_any_kernel<T, I8><<<(unsigned)blocks, 256, 0, st>>>(a);
  MSCO_CUDA_CHECK(cudaGetLastError());
  return MSCO_OK;
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
  if (i8) return f16 ? launch_any<__half, true>(a, st) : launch_any<__nv_bfloat16, true>(a, st);
  return f16 ? launch_any<__half, false>(a, st) : launch_any<__nv_bfloat16, false>(a, st);
}
