// Chunk attention: checks, work list and launch (C ABI).
#include <algorithm>
#include <cmath>
#include <exception>
#include <utility>
#include <vector>

#include "chunk_params.h"
#include "msco_common.cuh"

namespace msco {
namespace {

int check_desc(const MscoChunkDesc &d) {
  if (d.q_dtype != MSCO_DTYPE_F16 && d.q_dtype != MSCO_DTYPE_BF16)
    return fail(MSCO_ERR_INVALID_ARG, "chunk_attention: query must be float16 or bfloat16");
  if (d.kv_dtype != d.q_dtype && d.kv_dtype != MSCO_DTYPE_I8)
    return fail(MSCO_ERR_INVALID_ARG, "chunk_attention: the caches must have the query's type or be int8");
  if (d.num_q_heads <= 0 || d.num_kv_heads <= 0 || d.num_q_heads % d.num_kv_heads != 0)
    return fail(MSCO_ERR_INVALID_ARG, "chunk_attention: q heads (%d) must be a positive multiple of kv heads (%d)",
                d.num_q_heads, d.num_kv_heads);
  if (d.head_dim <= 0 || d.head_dim > 256)
    return fail(MSCO_ERR_INVALID_ARG, "chunk_attention: head_dim must be in (0, 256], got %d", d.head_dim);
  if (d.block_size <= 0 || d.num_blocks <= 0 || d.max_blocks_per_seq < 0)
    return fail(MSCO_ERR_INVALID_ARG, "chunk_attention: bad cache geometry");
  if (d.cache_layout != 0 && d.cache_layout != 1)
    return fail(MSCO_ERR_INVALID_ARG, "chunk_attention: cache_layout must be 0 (block_size major) or 1 (head major)");
  if (d.window < 0) return fail(MSCO_ERR_INVALID_ARG, "chunk_attention: window must not be negative, got %d", d.window);
  if (!std::isfinite(d.qk_scale)) return fail(MSCO_ERR_INVALID_ARG, "chunk_attention: qk_scale must be finite");
  if (d.kernel != 0 && d.kernel != kChunkKernelGeneric)
    return fail(MSCO_ERR_INVALID_ARG, "chunk_attention: kernel must be 0 or 1");
  return MSCO_OK;
}

// The sequences with new tokens.
int collect(const MscoChunkDesc &d, const int32_t *q_lens, const int32_t *ctx, int32_t batch,
            std::vector<ChunkSeq> *out) {
  if (batch < 0 || (batch > 0 && (q_lens == nullptr || ctx == nullptr)))
    return fail(MSCO_ERR_INVALID_ARG, "chunk_attention: NULL lengths");
  const int64_t cap = (int64_t)d.max_blocks_per_seq * d.block_size;
  int64_t rows = 0;
  out->clear();
  for (int b = 0; b < batch; ++b) {
    if (q_lens[b] < 0 || ctx[b] < 0)
      return fail(MSCO_ERR_INVALID_ARG, "chunk_attention: q_seq_lens[%d] = %d and context_lens[%d] = %d must not be "
                  "negative", b, q_lens[b], b, ctx[b]);
    if (ctx[b] > cap)
      return fail(MSCO_ERR_INVALID_ARG, "chunk_attention: context_lens[%d] = %d exceeds the block table (%d blocks of "
                  "%d)", b, ctx[b], d.max_blocks_per_seq, d.block_size);
    if (rows + q_lens[b] > 0x7fffffffLL) return fail(MSCO_ERR_INVALID_ARG, "chunk_attention: too many query tokens");
    if (q_lens[b] > 0) out->push_back({0, (int32_t)rows, q_lens[b], ctx[b], b, 1, 0x7fffffff, 0});
    rows += q_lens[b];
  }
  return MSCO_OK;
}

bool use_tc(const MscoChunkDesc &d) { return d.kernel != kChunkKernelGeneric && chunk_tc_supported(d); }
int item_tokens_of(const MscoChunkDesc &d) { return 2 * (kChunkKvTile / (d.num_q_heads / d.num_kv_heads)); }

// KV splits of the tensor-core kernel.  A function of the sequence's own lengths and of the head counts, so that the
// result of a sequence does not depend on the others of the call.
void split_rule(const MscoChunkDesc &d, ChunkSeq *e, int64_t *cost) {
  const int group = d.num_q_heads / d.num_kv_heads, it = item_tokens_of(d);
  const int64_t alone = (int64_t)((e->q_len + it - 1) / it) * d.num_kv_heads;  // items without splits
  // KV tiles of the longest item
  const int last0 = (e->q_len - 1) / it * it;
  const int hi = e->ctx, lo = d.window > 0 ? std::max(0, e->ctx - e->q_len + last0 - d.window + 1) : 0;
  const int tiles = hi > lo ? (hi + kChunkKvTile - 1) / kChunkKvTile - lo / kChunkKvTile : 0;
  const int rows = std::min(e->q_len, it) * group;
  const bool dual = rows > kChunkKvTile;
  // The count that ends first when the sequence has the GPU (148 SMs) to itself: rounds of items times an item's tiles and
  // what an item costs besides, in tiles (its rows' partial results are written and read again; few rows: little).
  // Measured with 6 / 3 for two streams of rows: 512 tokens over 32k 253 / 285 us, a windowed batch 136 / 150 us; with at
  // least 8 / 4 tiles a split: a mixed batch 156 / 184 us, and for single tokens 4 / 8: one over 4096 19 / 26 us.
  const int fixed = rows <= 32 ? 2 : (dual ? 6 : 4), most = std::max(1, tiles / (rows <= 32 ? 4 : 8));
  int nsplit = 1;
  int64_t best = INT64_MAX;
  for (int ns = 1; ns <= most && alone * ns <= 148 * 4; ++ns) {
    const int64_t cost = (alone * ns + 147) / 148 * ((tiles + ns - 1) / ns + (ns > 1 ? fixed : fixed / 2));
    if (cost < best) {
      best = cost;
      nsplit = ns;
    }
  }
  e->chunk = nsplit > 1 ? (tiles + nsplit - 1) / nsplit : 0x3fffffff;
  e->nsplit = nsplit > 1 ? (tiles + e->chunk - 1) / e->chunk : 1;
  // windows: an earlier item may touch one tile more than the last one
  if (e->nsplit > 1 && d.window > 0) e->nsplit += 1;
  // what the longest item takes, for the order: streams share the tiles of a single item
  *cost = (int64_t)std::min(tiles, e->chunk) * (dual ? 2 : 1);
}

struct Plan {
  std::vector<ChunkSeq> seqs;
  std::vector<int64_t> items;  // of every launch (group of kChunkSeqsMax sequences)
  int64_t part_rows = 0, q_rows = 0;
};

int make_plan(const MscoChunkDesc &d, const int32_t *q_lens, const int32_t *ctx, int32_t batch, Plan *pl) {
  if (int rc = collect(d, q_lens, ctx, batch, &pl->seqs)) return rc;
  for (const ChunkSeq &e : pl->seqs) pl->q_rows += e.q_len;
  if (!use_tc(d)) return MSCO_OK;
  const int it = item_tokens_of(d), group = d.num_q_heads / d.num_kv_heads;
  std::vector<std::pair<int64_t, ChunkSeq>> order;
  order.reserve(pl->seqs.size());
  for (ChunkSeq &e : pl->seqs) {
    int64_t cost = 0;
    split_rule(d, &e, &cost);
    order.push_back({cost, e});
  }
  // the longest items first: the blocks take them in this order
  std::stable_sort(order.begin(), order.end(),
                   [](const auto &a, const auto &b) { return a.first > b.first; });
  for (size_t i = 0; i < order.size(); ++i) pl->seqs[i] = order[i].second;
  for (size_t i = 0; i < pl->seqs.size(); ++i) {
    if (i % kChunkSeqsMax == 0) pl->items.push_back(0);
    ChunkSeq &e = pl->seqs[i];
    const int64_t tiles = ((int64_t)e.q_len + it - 1) / it * e.nsplit * d.num_kv_heads;
    e.item_base = (int32_t)pl->items.back();
    pl->items.back() += tiles;
    if (e.nsplit > 1) {
      e.part_base = (int32_t)pl->part_rows;
      pl->part_rows += tiles * std::min(e.q_len, it) * group;
    }
    if (pl->items.back() > 0x3fffffffLL || pl->part_rows > 0x7fffffffLL)
      return fail(MSCO_ERR_INVALID_ARG, "chunk_attention: too many work items");
  }
  return MSCO_OK;
}

size_t part_ml_offset(const MscoChunkDesc &d, const Plan &pl) {
  return ((size_t)pl.part_rows * d.head_dim * 4 + 255) / 256 * 256;
}
size_t bytes_of(const MscoChunkDesc &d, const Plan &pl) {
  return pl.part_rows == 0 ? 0 : part_ml_offset(d, pl) + (size_t)pl.part_rows * 8;
}

int workspace_bytes_of(const MscoChunkDesc *desc, const int32_t *q_lens, const int32_t *ctx, int32_t batch, size_t *bytes) {
  if (desc == nullptr || bytes == nullptr) return fail(MSCO_ERR_INVALID_ARG, "chunk_attention: NULL argument");
  *bytes = 0;
  if (int rc = check_desc(*desc)) return rc;
  Plan pl;
  if (int rc = make_plan(*desc, q_lens, ctx, batch, &pl)) return rc;
  *bytes = bytes_of(*desc, pl);
  return MSCO_OK;
}

int launch(const MscoChunkDesc *desc, const int32_t *q_lens, const int32_t *ctx, int32_t batch, const void *query,
           const void *key_cache, const void *value_cache, const int32_t *block_tables, const float *k_descale,
           const int32_t *k_offset, const float *v_descale, const int32_t *v_offset, void *out, float *lse,
           void *workspace, size_t workspace_bytes, int32_t *oob_count, void *stream) {
  if (desc == nullptr) return fail(MSCO_ERR_INVALID_ARG, "chunk_attention: NULL argument");
  const MscoChunkDesc &d = *desc;
  if (int rc = check_desc(d)) return rc;
  Plan pl;
  if (int rc = make_plan(d, q_lens, ctx, batch, &pl)) return rc;
  if (pl.seqs.empty()) return MSCO_OK;
  if (query == nullptr || key_cache == nullptr || value_cache == nullptr || out == nullptr ||
      (block_tables == nullptr && d.max_blocks_per_seq > 0))
    return fail(MSCO_ERR_INVALID_ARG, "chunk_attention: query, caches, block_tables and out must not be NULL");
  if (d.kv_dtype == MSCO_DTYPE_I8 && (k_descale == nullptr || v_descale == nullptr))
    return fail(MSCO_ERR_INVALID_ARG, "chunk_attention: int8 caches need k_descale and v_descale");
  const size_t need = bytes_of(d, pl);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255) != 0))
    return fail(MSCO_ERR_INVALID_ARG, "chunk_attention: the workspace must be 256-byte aligned and hold %zu bytes, got %zu",
                need, workspace_bytes);
  ChunkParams p = {};
  p.q = query; p.key_cache = key_cache; p.value_cache = value_cache; p.block_tables = block_tables;
  p.k_descale = k_descale; p.k_offset = k_offset; p.v_descale = v_descale; p.v_offset = v_offset;
  p.out = out; p.lse = lse; p.oob_count = oob_count;
  p.num_blocks = d.num_blocks;
  p.num_q_heads = d.num_q_heads; p.num_kv_heads = d.num_kv_heads; p.head_dim = d.head_dim;
  p.block_size = d.block_size; p.max_blocks_per_seq = d.max_blocks_per_seq; p.cache_layout = d.cache_layout;
  p.group = d.num_q_heads / d.num_kv_heads;
  p.window = d.window;
  p.scale_log2e = (float)((double)d.qk_scale * 1.4426950408889634);
  bool tc = use_tc(d);
  if (tc) {
    p.item_tokens = item_tokens_of(d);
    p.part_o = static_cast<float *>(workspace);
    p.part_ml = reinterpret_cast<float *>(static_cast<char *>(workspace) + part_ml_offset(d, pl));
    if (((reinterpret_cast<uintptr_t>(query) | reinterpret_cast<uintptr_t>(key_cache) |
          reinterpret_cast<uintptr_t>(value_cache)) & 15) != 0 || (reinterpret_cast<uintptr_t>(out) & 31) != 0)
      tc = false;  // rows that the copies cannot start on: the general kernel takes them
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (size_t at = 0; at < pl.seqs.size(); at += kChunkSeqsMax) {
    p.nseq = (int)std::min<size_t>(kChunkSeqsMax, pl.seqs.size() - at);
    if (tc) p.items = (int)pl.items[at / kChunkSeqsMax];
    if (int rc = tc ? launch_chunk_tc(d, p, pl.seqs.data() + at, pl.q_rows, st)
                    : launch_chunk_generic(d, p, pl.seqs.data() + at, st))
      return rc;
  }
  return MSCO_OK;
}

}  // namespace
}  // namespace msco

using namespace msco;

// Exceptions of the host containers end here: the callers are C.
extern "C" int msco_chunk_attention_workspace(const MscoChunkDesc *desc, const int32_t *host_q_seq_lens,
                                              const int32_t *host_context_lens, int32_t batch, size_t *bytes) try {
  return workspace_bytes_of(desc, host_q_seq_lens, host_context_lens, batch, bytes);
} catch (const std::exception &e) {
  return fail(MSCO_ERR_INTERNAL, "chunk_attention: %s", e.what());
}

extern "C" int msco_chunk_attention(const MscoChunkDesc *desc, const int32_t *host_q_seq_lens,
                                    const int32_t *host_context_lens, int32_t batch, const void *query,
                                    const void *key_cache, const void *value_cache, const int32_t *block_tables,
                                    const float *k_descale, const int32_t *k_offset, const float *v_descale,
                                    const int32_t *v_offset, void *out, float *lse, void *workspace,
                                    size_t workspace_bytes, int32_t *oob_count, void *stream) try {
  return launch(desc, host_q_seq_lens, host_context_lens, batch, query, key_cache, value_cache, block_tables, k_descale,
                k_offset, v_descale, v_offset, out, lse, workspace, workspace_bytes, oob_count, stream);
} catch (const std::exception &e) {
  return fail(MSCO_ERR_INTERNAL, "chunk_attention: %s", e.what());
}

extern "C" int msco_chunk_attention_status(void) {
  const int rc = chunk_tc_status();
  if (rc == MSCO_ERR_TIMEOUT)
    return fail(rc, "chunk_attention: a bounded device-side wait ran out on this device; results of that launch are not valid");
  if (rc != MSCO_OK) return fail(rc, "chunk_attention: the error word of the device cannot be read");
  return MSCO_OK;
}
