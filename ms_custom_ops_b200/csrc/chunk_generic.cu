// Chunk attention, general kernel: every head_dim up to 256, block size, group and cache type.
//
// One CTA per (row block, kv head): up to kRows packed rows (token-major, the q heads of one kv head adjacent)
// against all cached tokens that the block sees, 32 at a time in shared memory as float32.  A warp owns
// kRows / 4 rows: a lane is a cached token for the scores and a set of columns for the product with V; running
// maximum and sum per row.  Bound by the FMA pipe and shared-memory reads (4 + 4 bytes per two FMAs): the
// shapes that the tensor-core kernel does not take.
#include <math_constants.h>

#include "chunk_params.h"
#include "msco_common.cuh"

namespace msco {
namespace {

constexpr int kThreads = 128;
constexpr int kRows = 16;
constexpr int kWarpRows = kRows / 4;
constexpr int kTok = 32;
constexpr int kMaxCols = 8;  // columns per lane: head_dim <= 256

template <typename TQ, typename TKV, int N>
__global__ void __launch_bounds__(kThreads)
chunk_generic_kernel(ChunkParams p, const __grid_constant__ ChunkSeqs<N> seqs) {
  extern __shared__ float sm[];
  const int D = p.head_dim, DP = D + 1;  // odd stride: lanes that read a column of K each hit their own bank
  float *qs = sm;                        // [kRows][D]
  float *ks = qs + kRows * D;            // [kTok][DP]
  float *vs = ks + kTok * DP;            // [kTok][D]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = p.group;
  // row blocks are numbered through the sequences: item_base counts them here
  int lo = 0, hi = p.nseq;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (seqs.s[mid].item_base <= (int)blockIdx.x) lo = mid; else hi = mid;
  }
  const ChunkSeq e = seqs.s[lo];
  const int kvh = blockIdx.y;
  const int64_t row0 = (int64_t)(blockIdx.x - e.item_base) * kRows;
  const int nrows = (int)min((int64_t)kRows, (int64_t)e.q_len * g - row0);
  const int pos0 = e.ctx - e.q_len;
  const int tok_first = (int)(row0 / g), tok_last = (int)((row0 + nrows - 1) / g);
  const int kv_hi = max(0, pos0 + tok_last + 1);
  const int kv_lo = p.window > 0 ? max(0, pos0 + tok_first - p.window + 1) : 0;
  const TQ *q = static_cast<const TQ *>(p.q);
  for (int i = threadIdx.x; i < kRows * D; i += kThreads) {
    const int r = i / D, d = i - r * D;
    float v = 0.f;
    if (r < nrows) {
      const int64_t row = row0 + r;
      const int64_t tok = e.q_start + row / g;
      v = to_f32(q[(tok * p.num_q_heads + kvh * g + row % g) * D + d]);
    }
    qs[i] = v;
  }
  float m[kWarpRows], l[kWarpRows], acc[kWarpRows][kMaxCols];
  int pos[kWarpRows];
#pragma unroll
  for (int r = 0; r < kWarpRows; ++r) {
    m[r] = -CUDART_INF_F;
    l[r] = 0.f;
    const int row = warp * kWarpRows + r;
    pos[r] = row < nrows ? pos0 + (int)((row0 + row) / g) : -1;
#pragma unroll
    for (int c = 0; c < kMaxCols; ++c) acc[r][c] = 0.f;
  }
  const int32_t *table = p.block_tables + (int64_t)e.row * p.max_blocks_per_seq;
  for (int t0 = kv_lo; t0 < kv_hi; t0 += kTok) {
    const int nt = min(kTok, kv_hi - t0);
    __syncthreads();  // the rows of the tile before are done with (and qs is written)
    for (int j = warp; j < kTok; j += 4) {
      if (j < nt) {
        const int tok = t0 + j;
        int64_t blk = table[tok / p.block_size];
        if (blk < 0 || blk >= p.num_blocks) {
          if (lane == 0 && p.oob_count != nullptr && tok % p.block_size == 0) atomicAdd(p.oob_count, 1);
          blk = 0;
        }
        const int off = tok % p.block_size;
        const int64_t base = (p.cache_layout == 1 ? (blk * p.num_kv_heads + kvh) * p.block_size + off
                                                  : (blk * p.block_size + off) * p.num_kv_heads + kvh) * D;
        const TKV *kr = static_cast<const TKV *>(p.key_cache) + base;
        const TKV *vr = static_cast<const TKV *>(p.value_cache) + base;
        for (int d = lane; d < D; d += 32) {
          float k = to_f32(kr[d]), v = to_f32(vr[d]);
          if (sizeof(TKV) == 1) {
            const int c = kvh * D + d;
            k = (k + (p.k_offset ? (float)p.k_offset[c] : 0.f)) * p.k_descale[c];
            v = (v + (p.v_offset ? (float)p.v_offset[c] : 0.f)) * p.v_descale[c];
          }
          ks[j * DP + d] = k;
          vs[j * D + d] = v;
        }
      } else {
        for (int d = lane; d < D; d += 32) ks[j * DP + d] = vs[j * D + d] = 0.f;
      }
    }
    __syncthreads();
    const int tok = t0 + lane;
#pragma unroll
    for (int r = 0; r < kWarpRows; ++r) {
      const float *qr = qs + (warp * kWarpRows + r) * D;
      float s = 0.f;
      for (int d = 0; d < D; ++d) s = fmaf(qr[d], ks[lane * DP + d], s);
      s *= p.scale_log2e;
      const bool seen = tok < kv_hi && tok <= pos[r] && (p.window == 0 || tok > pos[r] - p.window);
      if (!__any_sync(0xffffffffu, seen)) continue;
      s = seen ? s : -CUDART_INF_F;
      float mx = s;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float mn = fmaxf(m[r], mx);
      const float base = mn == -CUDART_INF_F ? 0.f : mn;
      const float w = exp2f(m[r] - base), pr = exp2f(s - base);
      float sum = pr;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      l[r] = l[r] * w + sum;
      m[r] = mn;
#pragma unroll
      for (int c = 0; c < kMaxCols; ++c) acc[r][c] *= w;
      for (int j = 0; j < nt; ++j) {
        const float pj = __shfl_sync(0xffffffffu, pr, j);
        // a token that this row does not see adds nothing, whatever its row of V holds
        if (pj != 0.f) {
#pragma unroll
          for (int c = 0; c < kMaxCols; ++c)
            if (lane + 32 * c < D) acc[r][c] = fmaf(pj, vs[j * D + lane + 32 * c], acc[r][c]);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < kWarpRows; ++r) {
    const int row = warp * kWarpRows + r;
    if (row >= nrows) continue;
    const int64_t tok = e.q_start + (row0 + row) / g;
    const int64_t orow = tok * p.num_q_heads + kvh * g + (int)((row0 + row) % g);
    const float inv = l[r] > 0.f ? 1.f / l[r] : (l[r] == 0.f ? 0.f : l[r]);
#pragma unroll
    for (int c = 0; c < kMaxCols; ++c)
      if (lane + 32 * c < D) static_cast<TQ *>(p.out)[orow * D + lane + 32 * c] = from_f32<TQ>(acc[r][c] * inv);
    if (lane == 0 && p.lse != nullptr)
      p.lse[orow] = l[r] == 0.f ? -CUDART_INF_F : (m[r] + log2f(l[r])) * 0.6931471805599453f;
  }
}

template <typename TQ, typename TKV, int N>
int launch_sized(const ChunkParams &p, const ChunkSeq *src, cudaStream_t stream) {
  ChunkSeqs<N> seqs;
  int64_t blocks = 0;
  for (int i = 0; i < p.nseq; ++i) {
    seqs.s[i] = src[i];
    seqs.s[i].item_base = (int32_t)blocks;
    blocks += ((int64_t)src[i].q_len * p.group + kRows - 1) / kRows;
  }
  if (blocks > 0x7fffffffLL) return fail(MSCO_ERR_INVALID_ARG, "chunk_attention: too many query rows");
  if (p.num_kv_heads > 65535) return fail(MSCO_ERR_UNSUPPORTED, "chunk_attention: more than 65535 kv heads");
  const int D = p.head_dim;
  const size_t smem = (size_t)(kRows * D + kTok * (D + 1) + kTok * D) * 4;
  auto kfn = chunk_generic_kernel<TQ, TKV, N>;
  // 82 KB at head_dim 256: above the default limit.  Set per call: the attribute belongs to a device.
  MSCO_CUDA_CHECK(cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  kfn<<<dim3((unsigned)blocks, (unsigned)p.num_kv_heads), kThreads, smem, stream>>>(p, seqs);
  MSCO_CUDA_CHECK(cudaGetLastError());
  return MSCO_OK;
}

template <typename TQ, typename TKV>
int launch_typed(const ChunkParams &p, const ChunkSeq *src, cudaStream_t stream) {
  if (p.nseq <= kChunkSeqsSmall) return launch_sized<TQ, TKV, kChunkSeqsSmall>(p, src, stream);
  return launch_sized<TQ, TKV, kChunkSeqsMax>(p, src, stream);
}

}  // namespace

int launch_chunk_generic(const MscoChunkDesc &d, const ChunkParams &p, const ChunkSeq *seqs, cudaStream_t stream) {
  const bool f16 = d.q_dtype == MSCO_DTYPE_F16;
  if (d.kv_dtype == MSCO_DTYPE_I8)
    return f16 ? launch_typed<__half, int8_t>(p, seqs, stream) : launch_typed<__nv_bfloat16, int8_t>(p, seqs, stream);
  return f16 ? launch_typed<__half, __half>(p, seqs, stream)
             : launch_typed<__nv_bfloat16, __nv_bfloat16>(p, seqs, stream);
}

}  // namespace msco
