// Argument checks shared by the operators that are extensions of the plugin.
#ifndef MS_CUSTOM_OPS_B200_FRAMEWORK_CHECKS_H_
#define MS_CUSTOM_OPS_B200_FRAMEWORK_CHECKS_H_

#include <string>

#include "ops/framework/tensor.h"

namespace ms_custom_ops {

inline void CheckProvided(const Tensor &t, const char *op, const char *name) {
  if (!t.defined()) MS_VALUE_ERROR << "For " << op << ", " << name << " must be provided.";
}

inline void CheckDType(const Tensor &t, const char *op, const char *name, int32_t dt) {
  if (t.defined() && t.dtype() != dt)
    MS_TYPE_ERROR << "For " << op << ", " << name << " must be " << DTypeName(dt) << ", but got " << DTypeName(t.dtype())
                  << ".";
}

inline void CheckRank(const Tensor &t, const char *op, const char *name, size_t rank) {
  if (t.defined() && t.rank() != rank)
    MS_VALUE_ERROR << "For " << op << ", " << name << " must have rank " << rank << ", but got " << t.rank() << ".";
}

// Required vector (or matrix) of `n` elements.
inline void CheckNumel(const Tensor &t, const char *op, const char *name, int64_t n) {
  if (t.defined() && t.numel() != n)
    MS_VALUE_ERROR << "For " << op << ", " << name << " must have " << n << " elements, but got " << t.numel() << ".";
}

inline void CheckOnDevice(const Tensor &t, const char *op, const char *name) {
  if (t.defined() && t.on_host() && t.numel() != 0)
    MS_RUNTIME_ERROR << "For " << op << ", " << name << " must be a device tensor.";
}

// An output that other blocks of the same launch still read as an input would be a race.
inline void CheckApart(const Tensor &out, const Tensor &in, const char *op, const char *out_name, const char *in_name) {
  if (!out.defined() || !in.defined() || out.numel() == 0 || in.numel() == 0) return;
  int64_t last = 0;  // offset of the input's last element
  for (size_t i = 0; i < in.rank(); ++i) last += (in.dim(i) - 1) * in.desc()->strides[i];
  const uintptr_t o = reinterpret_cast<uintptr_t>(out.data()), o_end = o + out.numel() * DTypeSize(out.dtype());
  const uintptr_t a = reinterpret_cast<uintptr_t>(in.data()), a_end = a + (last + 1) * DTypeSize(in.dtype());
  if (o < a_end && a < o_end)
    MS_VALUE_ERROR << "For " << op << ", " << out_name << " must not share memory with " << in_name << ".";
}

// Scales and offsets of int8 caches: all or nothing, per channel.
inline void CheckQuantVectors(const char *op, bool int8_cache, int64_t channels, const Tensor &k_descale,
                              const Tensor &k_offset, const Tensor &v_descale, const Tensor &v_offset) {
  const struct { const Tensor *t; const char *name; int32_t dt; bool required; } all[] = {
      {&k_descale, "k_descale", MSCO_DTYPE_F32, true}, {&v_descale, "v_descale", MSCO_DTYPE_F32, true},
      {&k_offset, "k_offset", MSCO_DTYPE_I32, false}, {&v_offset, "v_offset", MSCO_DTYPE_I32, false}};
  for (const auto &v : all) {
    if (!int8_cache) {
      if (v.t->defined()) MS_VALUE_ERROR << "For " << op << ", " << v.name << " is only taken with Int8 caches.";
      continue;
    }
    if (v.required) CheckProvided(*v.t, op, v.name);
    CheckDType(*v.t, op, v.name, v.dt);
    CheckNumel(*v.t, op, v.name, channels);
    CheckContiguous(*v.t, op, v.name);
    CheckOnDevice(*v.t, op, v.name);
  }
}

// Geometry of a pair of 16-bit or int8 caches in either block layout.
struct CachePair {
  int64_t num_blocks = 0, block_size = 0, kv_heads = 0, head_dim = 0;
  bool int8 = false;
};
inline CachePair CheckCachePair(const char *op, const Tensor &key_cache, const Tensor &value_cache, int64_t input_layout) {
  CachePair c;
  if (input_layout != 0 && input_layout != 1)
    MS_VALUE_ERROR << "For " << op << ", input_layout must be 0 (BSND) or 1 (BNSD), but got " << input_layout << ".";
  CheckProvided(key_cache, op, "key_cache");
  CheckProvided(value_cache, op, "value_cache");
  CheckRank(key_cache, op, "key_cache", 4);
  CheckRank(value_cache, op, "value_cache", 4);
  if (key_cache.shape() != value_cache.shape())
    MS_VALUE_ERROR << "For " << op << ", key_cache and value_cache must have the same shape.";
  if (key_cache.dtype() != value_cache.dtype())
    MS_TYPE_ERROR << "For " << op << ", key_cache and value_cache must have the same dtype, but got "
                  << DTypeName(key_cache.dtype()) << " and " << DTypeName(value_cache.dtype()) << ".";
  c.num_blocks = key_cache.dim(0);
  c.block_size = key_cache.dim(input_layout == 1 ? 2 : 1);
  c.kv_heads = key_cache.dim(input_layout == 1 ? 1 : 2);
  c.head_dim = key_cache.dim(3);
  c.int8 = key_cache.dtype() == MSCO_DTYPE_I8;
  if (key_cache.has_zero_dim()) MS_VALUE_ERROR << "For " << op << ", the caches must not be empty.";
  if (c.num_blocks > 0x7fffffffLL || c.block_size > 0x7fffffffLL || c.kv_heads > (1 << 20) || c.head_dim > (1 << 20))
    MS_VALUE_ERROR << "For " << op << ", the caches are too large.";
  CheckContiguous(key_cache, op, "key_cache");
  CheckContiguous(value_cache, op, "value_cache");
  return c;
}

}  // namespace ms_custom_ops
#endif  // MS_CUSTOM_OPS_B200_FRAMEWORK_CHECKS_H_
