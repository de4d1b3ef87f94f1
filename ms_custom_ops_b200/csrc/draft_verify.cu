// verify_draft_tokens: rejection sampling of drafted tokens against the target's probabilities.
//
//   accept draft i while u_i q_i(d_i) < p_i(d_i); at the first that is not, draw from max(p_n - q_n, 0), after the
//   last from p_n: the lowest t with cumsum(weights)[t] > u_K * sum(weights).
//
// One thread-block cluster per sequence; a CTA owns a contiguous slice of the vocabulary, a warp a contiguous part
// of it, and one pass leaves every warp's sum of weights in shared memory.  All CTAs read all sums through
// distributed shared memory, so each knows the total and in whose part the drawn token lies; that warp alone
// goes over its part once more.  Sums are 64-bit: the order in which they are taken moves the result by
// 1e-16 of the total, far below the distance of two neighbouring borders (1e-8 for 32-bit probabilities).
// HBM- or latency-bound: one or two rows of the vocabulary per sequence.
#include <cooperative_groups.h>

#include <algorithm>

#include "msco_common.cuh"

namespace msco {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;

struct VerifyArgs {
  const void *target, *draft;
  const int32_t *draft_tokens, *draft_lens;
  const float *uniform;
  int32_t *tokens, *accepted;
  int batch, drafts, vocab;
};

// weight of one vocabulary entry (NaN and negative differences count as nothing)
__device__ __forceinline__ double weight_of(float p, float q) {
  const double w = (double)p - (double)q;
  return w > 0.0 ? w : 0.0;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) verify_kernel(VerifyArgs a) {
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
  const int b = blockIdx.x / ranks;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ double sums[kWarps];
  __shared__ int s_taken;
  const T *target = static_cast<const T *>(a.target) + (int64_t)b * (a.drafts + 1) * a.vocab;
  const T *draft = static_cast<const T *>(a.draft);
  if (draft != nullptr) draft += (int64_t)b * a.drafts * a.vocab;
  const int32_t *dtok = a.draft_tokens + (int64_t)b * a.drafts;
  const float *u = a.uniform + (int64_t)b * (a.drafts + 1);
  const int len = a.draft_lens != nullptr ? min(max(a.draft_lens[b], 0), a.drafts) : a.drafts;
  if (warp == 0) {
    int taken = 0;
    for (int i0 = 0; i0 < len; i0 += 32) {
      const int i = i0 + lane;
      bool ok = false;
      if (i < len) {
        const int t = dtok[i];
        if (t >= 0 && t < a.vocab) {
          const double q = draft != nullptr ? (double)to_f32(draft[(int64_t)i * a.vocab + t]) : 1.0;
          ok = (double)u[i] * q < (double)to_f32(target[(int64_t)i * a.vocab + t]);
        }
      }
      const unsigned no = __ballot_sync(0xffffffffu, !ok);
      taken += no != 0 ? __ffs(no) - 1 : 32;
      if (no != 0) break;
    }
    if (lane == 0) s_taken = min(taken, len);
  }
  __syncthreads();
  const int n = s_taken;
  const T *p = target + (int64_t)n * a.vocab;
  const bool rest = n < len;
  const T *q = rest && draft != nullptr ? draft + (int64_t)n * a.vocab : nullptr;
  const int certain = rest && draft == nullptr ? dtok[n] : -1;  // a draft without probabilities was certain
  // this warp's part of the vocabulary
  const int per = (a.vocab + ranks * kWarps - 1) / (ranks * kWarps);
  const int id = rank * kWarps + warp;
  const int lo = (int)min((int64_t)a.vocab, (int64_t)id * per), hi = min(a.vocab, lo + per);
  int drawn = -1;
  bool here = false, found = false;
  for (int mode = 0; mode < 2; ++mode) {  // mode 1: the rest was nowhere positive, draw from the target itself
    const bool less = mode == 0 && rest;
    auto weight = [&](int t) -> double {
      const float pt = to_f32(p[t]);
      if (!less) return weight_of(pt, 0.f);
      if (q != nullptr) return weight_of(pt, to_f32(q[t]));
      return t == certain ? 0.0 : weight_of(pt, 0.f);
    };
    double s = 0.0;
    for (int t = lo + lane; t < hi; t += 32) s += weight(t);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) sums[warp] = s;
    cluster.sync();
    double total = 0.0, before = 0.0;
    for (int r = 0; r < ranks; ++r) {
      const double *rs = cluster.map_shared_rank(sums, r);
      for (int w = 0; w < kWarps; ++w) {
        if (r * kWarps + w == id) before = total;
        total += rs[w];
      }
    }
    // every warp adds the sums in the same order, so all agree on the total and on whose part holds the border
    const double goal = (double)u[a.drafts] * total;
    found = goal >= 0.0 && goal < total;  // not for a row that is nowhere positive, nor for uniform outside [0, 1)
    here = found && before <= goal && before + s > goal;
    cluster.sync();  // the sums have been read
    if (total > 0.0) {
      if (here) {
        double run = before;
        int last = -1;
        for (int t0 = lo; t0 < hi && drawn < 0; t0 += 32) {
          const int t = t0 + lane;
          const double w = t < hi ? weight(t) : 0.0;
          double c = w;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double up = __shfl_up_sync(0xffffffffu, c, o);
            if (lane >= o) c += up;
          }
          const unsigned over = __ballot_sync(0xffffffffu, run + c > goal);
          const unsigned pos = __ballot_sync(0xffffffffu, w > 0.0);
          if (over != 0) drawn = t0 + __ffs(over) - 1;
          if (pos != 0) last = t0 + 31 - __clz(pos);
          run += __shfl_sync(0xffffffffu, c, 31);
        }
        // the part's sum and the scan round differently in the last place: the last entry that counts then
        if (drawn < 0) drawn = last;
      }
      break;
    }
  }
  int32_t *out = a.tokens + (int64_t)b * (a.drafts + 1);
  if (here && lane == 0) out[n] = drawn;
  if (rank == 0 && warp == 0) {
    if (lane == 0) a.accepted[b] = n;
    for (int i = lane; i <= a.drafts; i += 32)
      if (i != n || !found) out[i] = i < n ? dtok[i] : -1;
  }
}

template <typename T>
int launch_verify(const VerifyArgs &a, cudaStream_t st) {
  // parts of at least 2048 entries per CTA
  const int cluster = std::max(1, std::min(kMaxCluster, a.vocab / 2048));
  int c = 1;
  while (c * 2 <= cluster) c *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.batch * c));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)c;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  MSCO_CUDA_CHECK(cudaLaunchKernelEx(&cfg, verify_kernel<T>, a));
  return MSCO_OK;
}

}  // namespace
}  // namespace msco

using namespace msco;

extern "C" int msco_verify_draft_tokens(const void *target_probs, const void *draft_probs, int32_t dtype,
                                        const int32_t *draft_tokens, const int32_t *draft_lens, const float *uniform,
                                        int32_t *tokens, int32_t *accepted, int32_t batch, int32_t drafts,
                                        int32_t vocab, void *stream) {
  if (dtype != MSCO_DTYPE_F32 && dtype != MSCO_DTYPE_F16 && dtype != MSCO_DTYPE_BF16)
    return fail(MSCO_ERR_INVALID_ARG, "verify_draft_tokens: probabilities must be float32, float16 or bfloat16");
  if (batch < 0 || drafts < 0 || vocab <= 0 || batch > (1 << 24) || drafts > (1 << 20) || vocab > (1 << 30))
    return fail(MSCO_ERR_INVALID_ARG, "verify_draft_tokens: bad sizes (batch %d, drafts %d, vocab %d)", batch, drafts, vocab);
  if (batch == 0) return MSCO_OK;
  if (target_probs == nullptr || (drafts > 0 && draft_tokens == nullptr) || uniform == nullptr || tokens == nullptr ||
      accepted == nullptr)
    return fail(MSCO_ERR_INVALID_ARG, "verify_draft_tokens: NULL tensor");
  const VerifyArgs a = {target_probs, draft_probs, draft_tokens, draft_lens, uniform, tokens, accepted,
                        batch, drafts, vocab};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == MSCO_DTYPE_F32) return launch_verify<float>(a, st);
  if (dtype == MSCO_DTYPE_F16) return launch_verify<__half>(a, st);
  return launch_verify<__nv_bfloat16>(a, st);
}
