// chunk_attention: operator glue.  An extension of the plugin (no reference counterpart on this path): causal
// attention of a ragged batch of new tokens over the paged cache, next to paged_attention, whose cache layouts,
// scales and host-side lengths it keeps.  The device work is msco_chunk_attention (libmsco_b200.so).
#include "ms_custom_ops_c.h"
#include "ops/framework/checks.h"
#include "ops/framework/module.h"
#include "ops/framework/tensor.h"

namespace ms_custom_ops {
namespace {

constexpr const char *kOpName = "ChunkAttention";

struct Call {
  MscoChunkDesc desc = {};
  const int32_t *q_lens = nullptr, *ctx = nullptr;
  int32_t batch = 0;
};

const int32_t *HostVector(const Tensor &t, const char *name, int64_t n) {
  CheckProvided(t, kOpName, name);
  CheckDType(t, kOpName, name, MSCO_DTYPE_I32);
  if (!t.on_host() && t.numel() != 0)
    MS_RUNTIME_ERROR << "For " << kOpName << ", " << name << " must be a CPU tensor (move it to CPU before the call): its values "
                     << "are read on the host.";
  CheckRank(t, kOpName, name, 1);
  CheckNumel(t, kOpName, name, n);
  CheckContiguous(t, kOpName, name);
  if (n > 0 && t.data() == nullptr)
    MS_RUNTIME_ERROR << "For " << kOpName << ", the data ptr of " << name << " can not be nullptr.";
  return static_cast<const int32_t *>(t.data());
}

Call Check(const MsChunkAttentionArgs &a) {
  Call call;
  MscoChunkDesc &d = call.desc;
  const Tensor query(a.query), key_cache(a.key_cache), value_cache(a.value_cache), tables(a.block_tables);
  CheckProvided(query, kOpName, "query");
  CheckRank(query, kOpName, "query", 3);
  const CachePair c = CheckCachePair(kOpName, key_cache, value_cache, a.input_layout);
  if (query.dtype() != MSCO_DTYPE_F16 && query.dtype() != MSCO_DTYPE_BF16)
    MS_TYPE_ERROR << "For " << kOpName << ", query must be Float16/BFloat16, but got " << DTypeName(query.dtype()) << ".";
  if (!c.int8 && key_cache.dtype() != query.dtype())
    MS_TYPE_ERROR << "For " << kOpName << ", the caches must be Int8 or have query's dtype, but got "
                  << DTypeName(key_cache.dtype()) << " and " << DTypeName(query.dtype()) << ".";
  if (query.dim(2) != c.head_dim)
    MS_VALUE_ERROR << "For " << kOpName << ", query's head_dim " << query.dim(2) << " must equal the caches' " << c.head_dim << ".";
  if (query.dim(1) <= 0 || query.dim(1) > (1 << 20) || query.dim(1) % c.kv_heads != 0)
    MS_VALUE_ERROR << "For " << kOpName << ", the number of query heads (" << query.dim(1) << ") must be a positive multiple of "
                   << "the caches' " << c.kv_heads << " heads.";
  if (c.head_dim > 256)
    MS_VALUE_ERROR << "For " << kOpName << ", head_dim must be at most 256, but got " << c.head_dim << ".";
  CheckContiguous(query, kOpName, "query");
  CheckProvided(tables, kOpName, "block_tables");
  CheckDType(tables, kOpName, "block_tables", MSCO_DTYPE_I32);
  CheckRank(tables, kOpName, "block_tables", 2);
  CheckContiguous(tables, kOpName, "block_tables");
  if (tables.dim(0) > (1 << 24) || tables.dim(1) > 0x7fffffffLL / c.block_size)
    MS_VALUE_ERROR << "For " << kOpName << ", block_tables is too large.";
  call.batch = static_cast<int32_t>(tables.dim(0));
  call.q_lens = HostVector(Tensor(a.q_seq_lens), "q_seq_lens", call.batch);
  call.ctx = HostVector(Tensor(a.context_lens), "context_lens", call.batch);
  int64_t rows = 0;
  for (int32_t b = 0; b < call.batch; ++b) rows += call.q_lens[b] > 0 ? call.q_lens[b] : 0;
  if (rows > query.dim(0))
    MS_VALUE_ERROR << "For " << kOpName << ", q_seq_lens add up to " << rows << " tokens, but query holds " << query.dim(0) << ".";
  if (a.window_size < 0 || a.window_size > 0x7fffffffLL)
    MS_VALUE_ERROR << "For " << kOpName << ", window_size must not be negative, but got " << a.window_size << ".";
  CheckQuantVectors(kOpName, c.int8, c.kv_heads * c.head_dim, Tensor(a.k_descale), Tensor(a.k_offset),
                    Tensor(a.v_descale), Tensor(a.v_offset));
  CheckDType(Tensor(a.oob_count), kOpName, "oob_count", MSCO_DTYPE_I32);
  CheckNumel(Tensor(a.oob_count), kOpName, "oob_count", 1);
  d.q_dtype = query.dtype();
  d.kv_dtype = key_cache.dtype();
  d.num_q_heads = static_cast<int32_t>(query.dim(1));
  d.num_kv_heads = static_cast<int32_t>(c.kv_heads);
  d.head_dim = static_cast<int32_t>(c.head_dim);
  d.block_size = static_cast<int32_t>(c.block_size);
  d.num_blocks = c.num_blocks;
  d.max_blocks_per_seq = static_cast<int32_t>(tables.dim(1));
  d.cache_layout = static_cast<int32_t>(a.input_layout);
  d.qk_scale = static_cast<float>(a.qk_scale);
  d.window = static_cast<int32_t>(a.window_size);
  return call;
}

int Launch(const MsChunkAttentionArgs &a, const Tensor &out, const Tensor &lse, void *workspace, size_t workspace_bytes,
           void *stream) {
  const Call call = Check(a);
  const Tensor query(a.query);
  CheckProvided(out, kOpName, "out");
  CheckDType(out, kOpName, "out", query.dtype());
  if (out.shape() != query.shape()) MS_VALUE_ERROR << "For " << kOpName << ", out must have query's shape.";
  CheckContiguous(out, kOpName, "out");
  CheckDType(lse, kOpName, "lse", MSCO_DTYPE_F32);
  CheckRank(lse, kOpName, "lse", 2);
  if (lse.defined() && (lse.dim(0) != query.dim(0) || lse.dim(1) != query.dim(1)))
    MS_VALUE_ERROR << "For " << kOpName << ", lse must be (" << query.dim(0) << ", " << query.dim(1) << ").";
  CheckContiguous(lse, kOpName, "lse");
  const Tensor tables(a.block_tables), kc(a.key_cache), vc(a.value_cache), oob(a.oob_count);
  const struct { const Tensor *t; const char *name; } dev[] = {{&query, "query"}, {&kc, "key_cache"}, {&vc, "value_cache"},
                                                              {&tables, "block_tables"}, {&out, "out"}, {&lse, "lse"},
                                                              {&oob, "oob_count"}};
  for (const auto &v : dev) CheckOnDevice(*v.t, kOpName, v.name);
  CheckApart(out, query, kOpName, "out", "query");
  CheckApart(out, kc, kOpName, "out", "key_cache");
  CheckApart(out, vc, kOpName, "out", "value_cache");
  return msco_chunk_attention(
      &call.desc, call.q_lens, call.ctx, call.batch, query.data(), kc.data(), vc.data(),
      static_cast<const int32_t *>(tables.data()), static_cast<const float *>(Tensor(a.k_descale).data()),
      static_cast<const int32_t *>(Tensor(a.k_offset).data()), static_cast<const float *>(Tensor(a.v_descale).data()),
      static_cast<const int32_t *>(Tensor(a.v_offset).data()), out.data(), static_cast<float *>(lse.data()), workspace,
      workspace_bytes, static_cast<int32_t *>(oob.data()), stream);
}

}  // namespace
}  // namespace ms_custom_ops

MS_CUSTOM_OPS_REGISTER_OP(chunk_attention,
                          "chunk_attention(query, key_cache, value_cache, block_tables, q_seq_lens, context_lens, "
                          "qk_scale=1.0, window_size=0, input_layout=0, k_descale=None, k_offset=None, v_descale=None, "
                          "v_offset=None, out=None, return_lse=False, oob_count=None)")

extern "C" int ms_custom_ops_chunk_attention_infer(const MsChunkAttentionArgs *args, int32_t *out_dtype,
                                                   int32_t *out_ndim, int64_t *out_shape) {
  using namespace ms_custom_ops;
  return GuardedCall(kOpName, [&] {
    if (args == nullptr) MS_VALUE_ERROR << "For " << kOpName << ", args must be provided.";
    const Call call = Check(*args);
    size_t bytes = 0;  // the checks of the lengths
    const int rc = msco_chunk_attention_workspace(&call.desc, call.q_lens, call.ctx, call.batch, &bytes);
    if (rc != MSCO_OK) return rc;
    const Tensor q(args->query);
    if (out_dtype != nullptr) *out_dtype = q.dtype();
    if (out_ndim != nullptr) *out_ndim = 3;
    if (out_shape != nullptr)
      for (size_t i = 0; i < 3; ++i) out_shape[i] = q.dim(i);
    return static_cast<int>(MSCO_OK);
  });
}

extern "C" int ms_custom_ops_chunk_attention_workspace_size(const MsChunkAttentionArgs *args, size_t *bytes) {
  using namespace ms_custom_ops;
  return GuardedCall(kOpName, [&] {
    if (args == nullptr || bytes == nullptr) MS_VALUE_ERROR << "For " << kOpName << ", args must be provided.";
    const Call call = Check(*args);
    return msco_chunk_attention_workspace(&call.desc, call.q_lens, call.ctx, call.batch, bytes);
  });
}

extern "C" int ms_custom_ops_chunk_attention(const MsChunkAttentionArgs *args, const MsTensorDesc *out,
                                             const MsTensorDesc *lse, void *workspace, size_t workspace_bytes,
                                             void *stream) {
  using namespace ms_custom_ops;
  return GuardedCall(kOpName, [&] {
    if (args == nullptr) MS_VALUE_ERROR << "For " << kOpName << ", args must be provided.";
    return Launch(*args, Tensor(out), Tensor(lse), workspace, workspace_bytes, stream);
  });
}
