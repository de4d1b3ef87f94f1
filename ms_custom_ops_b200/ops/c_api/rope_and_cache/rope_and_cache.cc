// rope_and_cache: operator glue.  An extension of the plugin (no reference counterpart on this path): per-head
// norm, position rotation and cache write in one launch, next to reshape_and_cache, whose slot and cache rules it
// keeps.  The device work is msco_rope_and_cache (libmsco_b200.so).
#include "ms_custom_ops_c.h"
#include "ops/framework/checks.h"
#include "ops/framework/module.h"
#include "ops/framework/tensor.h"

namespace ms_custom_ops {
namespace {

constexpr const char *kOpName = "RopeAndCache";

struct Inputs {
  Tensor query, key, value, key_cache, value_cache, slot_mapping, positions, cos_sin, q_weight, k_weight, k_descale,
      k_offset, v_descale, v_offset, oob_count;
  double eps;
  int32_t interleaved;
  int64_t input_layout;
};

// Rows (tokens, heads, head_dim) whose heads are adjacent; the token stride is free.
int64_t CheckRows(const Tensor &t, const char *name, int64_t tokens, int64_t head_dim) {
  CheckProvided(t, kOpName, name);
  CheckRank(t, kOpName, name, 3);
  if (t.dim(0) != tokens || t.dim(2) != head_dim)
    MS_VALUE_ERROR << "For " << kOpName << ", " << name << " must be (" << tokens << ", heads, " << head_dim << "), but got ("
                   << t.dim(0) << ", " << t.dim(1) << ", " << t.dim(2) << ").";
  const MsTensorDesc *d = t.desc();
  const int64_t row = t.dim(1) * head_dim;
  if (tokens == 0 || row == 0) return row;
  if ((head_dim > 1 && d->strides[2] != 1) || (t.dim(1) > 1 && d->strides[1] != head_dim) ||
      (tokens > 1 && d->strides[0] < row))
    MS_RUNTIME_ERROR << "For " << kOpName << ", the heads of a token of " << name << " must be adjacent, and its tokens must not "
                     << "overlap.";
  return tokens > 1 ? d->strides[0] : row;
}

MscoRopeDesc Check(const Inputs &in) {
  MscoRopeDesc d = {};
  const CachePair c = CheckCachePair(kOpName, in.key_cache, in.value_cache, in.input_layout);
  CheckProvided(in.key, kOpName, "key");
  CheckRank(in.key, kOpName, "key", 3);
  const int64_t tokens = in.key.dim(0);
  CheckProvided(in.query, kOpName, "query");
  d.k_stride = CheckRows(in.key, "key", tokens, c.head_dim);
  d.v_stride = CheckRows(in.value, "value", tokens, c.head_dim);
  d.q_stride = CheckRows(in.query, "query", tokens, c.head_dim);
  if (in.key.dim(1) != c.kv_heads || in.value.dim(1) != c.kv_heads)
    MS_VALUE_ERROR << "For " << kOpName << ", key and value must have the caches' " << c.kv_heads << " heads, but got "
                   << in.key.dim(1) << " and " << in.value.dim(1) << ".";
  if (in.query.dim(1) > (1 << 20)) MS_VALUE_ERROR << "For " << kOpName << ", too many query heads.";
  if (in.key.dtype() != MSCO_DTYPE_F16 && in.key.dtype() != MSCO_DTYPE_BF16)
    MS_TYPE_ERROR << "For " << kOpName << ", key must be Float16/BFloat16, but got " << DTypeName(in.key.dtype()) << ".";
  CheckDType(in.value, kOpName, "value", in.key.dtype());
  CheckDType(in.query, kOpName, "query", in.key.dtype());
  if (!c.int8 && in.key_cache.dtype() != in.key.dtype())
    MS_TYPE_ERROR << "For " << kOpName << ", the caches must be Int8 or have key's dtype, but got "
                  << DTypeName(in.key_cache.dtype()) << " and " << DTypeName(in.key.dtype()) << ".";
  for (const auto &v : {std::pair<const Tensor *, const char *>{&in.slot_mapping, "slot_mapping"}, {&in.positions, "positions"}}) {
    CheckProvided(*v.first, kOpName, v.second);
    CheckDType(*v.first, kOpName, v.second, MSCO_DTYPE_I32);
    CheckNumel(*v.first, kOpName, v.second, tokens);
    CheckContiguous(*v.first, kOpName, v.second);
  }
  CheckProvided(in.cos_sin, kOpName, "cos_sin");
  CheckDType(in.cos_sin, kOpName, "cos_sin", MSCO_DTYPE_F32);
  CheckRank(in.cos_sin, kOpName, "cos_sin", 2);
  CheckContiguous(in.cos_sin, kOpName, "cos_sin");
  if (in.cos_sin.dim(1) > c.head_dim || in.cos_sin.dim(1) % 2 != 0)
    MS_VALUE_ERROR << "For " << kOpName << ", cos_sin must be (max_positions, rotary_dim) with rotary_dim even and at most "
                   << "head_dim " << c.head_dim << ", but rotary_dim is " << in.cos_sin.dim(1) << ".";
  for (const auto &v : {std::pair<const Tensor *, const char *>{&in.q_weight, "q_weight"}, {&in.k_weight, "k_weight"}}) {
    CheckDType(*v.first, kOpName, v.second, in.key.dtype());
    CheckNumel(*v.first, kOpName, v.second, c.head_dim);
    CheckContiguous(*v.first, kOpName, v.second);
  }
  if (!(in.eps >= 0)) MS_VALUE_ERROR << "For " << kOpName << ", eps must not be negative, but got " << in.eps << ".";
  CheckQuantVectors(kOpName, c.int8, c.kv_heads * c.head_dim, in.k_descale, in.k_offset, in.v_descale, in.v_offset);
  CheckDType(in.oob_count, kOpName, "oob_count", MSCO_DTYPE_I32);
  CheckNumel(in.oob_count, kOpName, "oob_count", 1);
  d.dtype = in.key.dtype();
  d.cache_dtype = in.key_cache.dtype();
  d.num_q_heads = static_cast<int32_t>(in.query.dim(1));
  d.num_kv_heads = static_cast<int32_t>(c.kv_heads);
  d.head_dim = static_cast<int32_t>(c.head_dim);
  d.rotary_dim = static_cast<int32_t>(in.cos_sin.dim(1));
  d.block_size = static_cast<int32_t>(c.block_size);
  d.cache_layout = static_cast<int32_t>(in.input_layout);
  d.num_blocks = c.num_blocks;
  d.num_tokens = tokens;
  d.max_positions = in.cos_sin.dim(0);
  d.eps = static_cast<float>(in.eps);
  d.interleaved = in.interleaved;
  return d;
}

int Launch(const Inputs &in, const Tensor &query_out, void *stream) {
  const MscoRopeDesc d = Check(in);
  CheckProvided(query_out, kOpName, "query_out");
  CheckDType(query_out, kOpName, "query_out", in.query.dtype());
  if (query_out.shape() != in.query.shape())
    MS_VALUE_ERROR << "For " << kOpName << ", query_out must have query's shape.";
  CheckContiguous(query_out, kOpName, "query_out");
  const struct { const Tensor *t; const char *name; } dev[] = {
      {&in.query, "query"}, {&in.key, "key"}, {&in.value, "value"}, {&in.key_cache, "key_cache"},
      {&in.value_cache, "value_cache"}, {&in.slot_mapping, "slot_mapping"}, {&in.positions, "positions"},
      {&in.cos_sin, "cos_sin"}, {&in.q_weight, "q_weight"}, {&in.k_weight, "k_weight"}, {&in.oob_count, "oob_count"},
      {&query_out, "query_out"}};
  for (const auto &v : dev) CheckOnDevice(*v.t, kOpName, v.name);
  for (const Tensor *t : {&in.query, &in.key, &in.value}) CheckApart(query_out, *t, kOpName, "query_out", "the inputs");
  return msco_rope_and_cache(
      &d, in.query.data(), in.key.data(), in.value.data(), query_out.data(), in.key_cache.data(), in.value_cache.data(),
      static_cast<const int32_t *>(in.slot_mapping.data()), static_cast<const int32_t *>(in.positions.data()),
      static_cast<const float *>(in.cos_sin.data()), in.q_weight.data(), in.k_weight.data(),
      static_cast<const float *>(in.k_descale.data()), static_cast<const int32_t *>(in.k_offset.data()),
      static_cast<const float *>(in.v_descale.data()), static_cast<const int32_t *>(in.v_offset.data()),
      static_cast<int32_t *>(in.oob_count.data()), stream);
}

}  // namespace
}  // namespace ms_custom_ops

MS_CUSTOM_OPS_REGISTER_OP(rope_and_cache,
                          "rope_and_cache(query, key, value, key_cache, value_cache, slot_mapping, positions, cos_sin, "
                          "q_weight=None, k_weight=None, eps=1e-06, interleaved=False, input_layout=0, k_descale=None, "
                          "k_offset=None, v_descale=None, v_offset=None, oob_count=None)")

extern "C" int ms_custom_ops_rope_and_cache_infer(
    const MsTensorDesc *query, const MsTensorDesc *key, const MsTensorDesc *value, const MsTensorDesc *key_cache,
    const MsTensorDesc *value_cache, const MsTensorDesc *slot_mapping, const MsTensorDesc *positions,
    const MsTensorDesc *cos_sin, const MsTensorDesc *q_weight, const MsTensorDesc *k_weight, double eps,
    int32_t interleaved, int64_t input_layout, const MsTensorDesc *k_descale, const MsTensorDesc *k_offset,
    const MsTensorDesc *v_descale, const MsTensorDesc *v_offset, const MsTensorDesc *oob_count, int32_t *out_dtype,
    int32_t *out_ndim, int64_t *out_shape) {
  using namespace ms_custom_ops;
  return GuardedCall(kOpName, [&] {
    const Inputs in = {Tensor(query), Tensor(key), Tensor(value), Tensor(key_cache), Tensor(value_cache),
                       Tensor(slot_mapping), Tensor(positions), Tensor(cos_sin), Tensor(q_weight), Tensor(k_weight),
                       Tensor(k_descale), Tensor(k_offset), Tensor(v_descale), Tensor(v_offset), Tensor(oob_count),
                       eps, interleaved, input_layout};
    (void)Check(in);
    if (out_dtype != nullptr) *out_dtype = in.query.dtype();
    if (out_ndim != nullptr) *out_ndim = 3;
    if (out_shape != nullptr)
      for (size_t i = 0; i < 3; ++i) out_shape[i] = in.query.dim(i);
    return MSCO_OK;
  });
}

extern "C" int ms_custom_ops_rope_and_cache(
    const MsTensorDesc *query, const MsTensorDesc *key, const MsTensorDesc *value, const MsTensorDesc *key_cache,
    const MsTensorDesc *value_cache, const MsTensorDesc *slot_mapping, const MsTensorDesc *positions,
    const MsTensorDesc *cos_sin, const MsTensorDesc *q_weight, const MsTensorDesc *k_weight, double eps,
    int32_t interleaved, int64_t input_layout, const MsTensorDesc *k_descale, const MsTensorDesc *k_offset,
    const MsTensorDesc *v_descale, const MsTensorDesc *v_offset, const MsTensorDesc *oob_count,
    const MsTensorDesc *query_out, void *stream) {
  using namespace ms_custom_ops;
  return GuardedCall(kOpName, [&] {
    const Inputs in = {Tensor(query), Tensor(key), Tensor(value), Tensor(key_cache), Tensor(value_cache),
                       Tensor(slot_mapping), Tensor(positions), Tensor(cos_sin), Tensor(q_weight), Tensor(k_weight),
                       Tensor(k_descale), Tensor(k_offset), Tensor(v_descale), Tensor(v_offset), Tensor(oob_count),
                       eps, interleaved, input_layout};
    return Launch(in, Tensor(query_out), stream);
  });
}
