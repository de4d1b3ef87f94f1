// Plan and kernel parameters of chunk attention (a chunk of new tokens per sequence over the paged cache).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "msco_b200.h"

namespace msco {

constexpr int kChunkKernelGeneric = 1;
constexpr int kChunkKernelTc = 2;
constexpr int kChunkKvTile = 128;  // cached tokens per tile: KV splits start and end at multiples of it

// One sequence with new tokens.  Its items are numbered from item_base: query tile (the last one, which sees
// the most, first), then KV split, then kv head.
struct ChunkSeq {
  int32_t item_base;
  int32_t q_start;    // row of the sequence's first new token in query / out
  int32_t q_len;      // new tokens
  int32_t ctx;        // cached tokens, the new ones included
  int32_t row;        // block-table row
  int32_t nsplit;     // KV splits of every query tile
  int32_t chunk;      // KV tiles per split
  int32_t part_base;  // first partial row (nsplit > 1); its tiles are numbered (query tile * nsplit + split) * kv_heads + kv head
};

struct ChunkParams {
  const void *q;
  const void *key_cache;
  const void *value_cache;
  const int32_t *block_tables;
  const float *k_descale;
  const int32_t *k_offset;
  const float *v_descale;
  const int32_t *v_offset;
  void *out;
  float *lse;          // optional [tokens, num_q_heads], natural logarithm
  float *part_o;       // [partial row, head_dim] un-normalised partial outputs
  float *part_ml;      // [partial row, 2] running max (log2 domain) and sum
  int32_t *oob_count;  // optional: block ids outside the cache
  int64_t num_blocks;
  int num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, cache_layout;
  int group;           // q heads per kv head
  int item_tokens;     // new tokens of one item (two streams of item_tokens / 2)
  int window;          // 0: none
  float scale_log2e;   // qk_scale * log2(e)
  int nseq, items;
};

// The sequences of a launch travel as a kernel parameter: nothing to upload and nothing that a captured graph
// could find changed.  Batches of more sequences than fit are launched in several parts.
constexpr int kChunkSeqsSmall = 64;
constexpr int kChunkSeqsMax = 960;
template <int N>
struct ChunkSeqs {
  ChunkSeq s[N];
};

#ifdef __CUDACC__
// What one item computes: query tokens [tok0, tok1) of sequence `seq` for kv head `kvh` against the KV tiles
// [tile0, tile1) of its split.
struct ChunkItem {
  int seq, kvh, split, qtile;
  int tok0, tok1;
  int tile0, tile1;
  int kv_hi;  // cached tokens from here on are seen by no row of the item (a token, not a tile)
};

template <int N>
__device__ __forceinline__ ChunkItem chunk_item(const ChunkSeqs<N> &seqs, const ChunkParams &p, int t) {
  int lo = 0, hi = p.nseq;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (seqs.s[mid].item_base <= t) lo = mid; else hi = mid;
  }
  const ChunkSeq &e = seqs.s[lo];
  ChunkItem w;
  w.seq = lo;
  int r = t - e.item_base;
  w.kvh = r % p.num_kv_heads;
  r /= p.num_kv_heads;
  w.split = r % e.nsplit;
  const int ntile = (e.q_len + p.item_tokens - 1) / p.item_tokens;
  w.qtile = ntile - 1 - r / e.nsplit;
  w.tok0 = w.qtile * p.item_tokens;
  w.tok1 = min(e.q_len, w.tok0 + p.item_tokens);
  const int pos0 = e.ctx - e.q_len;  // position of the sequence's first new token
  w.kv_hi = max(0, pos0 + w.tok1);
  const int kv_lo = p.window > 0 ? max(0, pos0 + w.tok0 - p.window + 1) : 0;
  const int first = kv_lo / kChunkKvTile, end = (w.kv_hi + kChunkKvTile - 1) / kChunkKvTile;
  w.tile0 = first + w.split * e.chunk;
  w.tile1 = min(end, w.tile0 + e.chunk);
  return w;
}
#endif  // __CUDACC__

// launchers (defined next to the kernels)
bool chunk_tc_supported(const MscoChunkDesc &d);
int launch_chunk_tc(const MscoChunkDesc &d, const ChunkParams &p, const ChunkSeq *seqs, int64_t q_rows,
                    cudaStream_t stream);
int chunk_tc_status();  // MSCO_OK, or MSCO_ERR_TIMEOUT once a bounded wait ran out on the current device (synchronises)
int launch_chunk_generic(const MscoChunkDesc &d, const ChunkParams &p, const ChunkSeq *seqs, cudaStream_t stream);

}  // namespace msco
