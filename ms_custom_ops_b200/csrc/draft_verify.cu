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
constexpr int kMaxCluster = 8;  // (at most 64 warps: two sums per lane)

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

constexpr int kLane = 8;             // vocabulary entries per lane and chunk
constexpr int kChunk = 32 * kLane;   // entries of a chunk

// Entries t0 .. t0 + 255 of a row, 8 per lane, 0 behind the end.  VEC: rows are 16-byte aligned (and t0 is a multiple of
// 256), so a lane's entries come in 16-byte pieces, piece i of all lanes adjacent; otherwise one entry at a time.
// The entry `skip` reads as 0.
template <typename T, bool VEC>
__device__ __forceinline__ void load_chunk(const T *row, int t0, int end, int lane, int skip, float (&x)[kLane]) {
  if (VEC && t0 + kChunk <= end) {
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < kLane / kPer; ++i) {
      const uint4 v = __ldg(reinterpret_cast<const uint4 *>(row + t0) + i * 32 + lane);
      const T *e = reinterpret_cast<const T *>(&v);
#pragma unroll
      for (int k = 0; k < kPer; ++k) x[i * kPer + k] = to_f32(e[k]);
    }
    if (skip >= t0 && skip < t0 + kChunk) {
#pragma unroll
      for (int i = 0; i < kLane; ++i)
        if (t0 + (i / kPer * 32 + lane) * kPer + i % kPer == skip) x[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kLane; ++i) {
      const int t = t0 + i * 32 + lane;
      x[i] = t < end && t != skip ? to_f32(row[t]) : 0.f;
    }
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads, 4) verify_kernel(VerifyArgs a) {
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
  const int b = blockIdx.x / ranks;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ double all_sums[2][kWarps];  // per mode
  const T *target = static_cast<const T *>(a.target) + (int64_t)b * (a.drafts + 1) * a.vocab;
  const T *draft = static_cast<const T *>(a.draft);
  if (draft != nullptr) draft += (int64_t)b * a.drafts * a.vocab;
  const int32_t *dtok = a.draft_tokens + (int64_t)b * a.drafts;
  const float *u = a.uniform + (int64_t)b * (a.drafts + 1);
  const int len = a.draft_lens != nullptr ? min(max(__ldg(a.draft_lens + b), 0), a.drafts) : a.drafts;
  // every warp finds the first draft that is turned down for itself: no exchange
  int n = 0;
  for (int i0 = 0; i0 < len; i0 += 32) {
    const int i = i0 + lane;
    bool ok = false;
    if (i < len) {
      const int t = __ldg(dtok + i);
      if (t >= 0 && t < a.vocab) {
        const double q = draft != nullptr ? (double)to_f32(draft[(int64_t)i * a.vocab + t]) : 1.0;
        ok = (double)__ldg(u + i) * q < (double)to_f32(target[(int64_t)i * a.vocab + t]);
      }
    }
    const unsigned no = __ballot_sync(0xffffffffu, !ok);
    n += no != 0 ? __ffs(no) - 1 : 32;
    if (no != 0) break;
  }
  n = min(n, len);
  const T *p = target + (int64_t)n * a.vocab;
  const bool rest = n < len;
  const T *q = rest && draft != nullptr ? draft + (int64_t)n * a.vocab : nullptr;
  const int certain = rest && draft == nullptr ? __ldg(dtok + n) : -1;  // a draft without probabilities was certain
  // this warp's part of the vocabulary: up to 32 chunks of `span` entries, lane k keeps the sum of chunk k
  const int warps = ranks * kWarps, id = rank * kWarps + warp;
  const int blocks = (a.vocab + kChunk - 1) / kChunk, per = (blocks + warps - 1) / warps;  // in units of kChunk
  const int span = (per + 31) / 32 * kChunk;
  const int lo = (int)min((int64_t)a.vocab, (int64_t)id * per * kChunk);
  const int hi = (int)min((int64_t)a.vocab, (int64_t)lo + (int64_t)per * kChunk);
  int drawn = -1;
  bool here = false, found = false;
  for (int mode = 0; mode < 2; ++mode) {  // mode 1: the rest was nowhere positive, draw from the target itself
    const bool less = mode == 0 && q != nullptr;
    const int skip = mode == 0 ? certain : -1;
    double mine = 0.0, s = 0.0;
    for (int k = 0, c0 = lo; c0 < hi; ++k, c0 += span) {
      double sum = 0.0;
      for (int t0 = c0; t0 < min(hi, c0 + span); t0 += kChunk) {
        float x[kLane], y[kLane];
        load_chunk<T, VEC>(p, t0, hi, lane, skip, x);
        if (less) {
          load_chunk<T, VEC>(q, t0, hi, lane, -1, y);
        } else {
#pragma unroll
          for (int i = 0; i < kLane; ++i) y[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < kLane; ++i) sum += weight_of(x[i], y[i]);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == k) mine = sum;
      s += sum;
    }
    double *sums = all_sums[mode];
    if (lane == 0) sums[warp] = s;
    cluster.sync();
    // every warp scans all sums in the same way, so all agree on the total and on whose part holds the border
    double part[2], own[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int w = k * 32 + lane;
      own[k] = part[k] = w < warps ? cluster.map_shared_rank(sums, w / kWarps)[w % kWarps] : 0.0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, part[k], o);
        if (lane >= o) part[k] += up;
      }
    }
    part[1] += __shfl_sync(0xffffffffu, part[0], 31);
    const double total = __shfl_sync(0xffffffffu, part[1], 31);
    const double goal = (double)__ldg(u + a.drafts) * total;
    found = goal >= 0.0 && goal < total;  // not for a row that is nowhere positive, nor for uniform outside [0, 1)
    // the first part that counts whose running sum passes the goal (should the last place of the sums leave none, the last
    // part that counts)
    const uint64_t counts = (uint64_t)__ballot_sync(0xffffffffu, own[1] > 0.0) << 32 | __ballot_sync(0xffffffffu, own[0] > 0.0);
    const uint64_t over = counts & ((uint64_t)__ballot_sync(0xffffffffu, part[1] > goal) << 32 |
                                    __ballot_sync(0xffffffffu, part[0] > goal));
    const int owner = over != 0 ? __ffsll((long long)over) - 1 : 63 - __clzll((long long)counts);
    here = found && owner == id;
    const int prev = max(owner - 1, 0);
    const double prev0 = __shfl_sync(0xffffffffu, part[0], prev & 31), prev1 = __shfl_sync(0xffffffffu, part[1], prev & 31);
    const double before = owner == 0 ? 0.0 : (prev < 32 ? prev0 : prev1);
    if (!(total > 0.0)) continue;
    if (here) {
      // the chunk in which the running sum passes the goal, then the entry
      double c = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, c, o);
        if (lane >= o) c += up;
      }
      const unsigned some = __ballot_sync(0xffffffffu, mine > 0.0);
      const unsigned over = some & __ballot_sync(0xffffffffu, before + c > goal);
      const int k = over != 0 ? __ffs(over) - 1 : 31 - __clz(some);
      double run = before + (__shfl_sync(0xffffffffu, c, k) - __shfl_sync(0xffffffffu, mine, k));
      int last = -1;
      const int c0 = lo + k * span, c1 = min(hi, c0 + span);
      for (int t0 = c0; t0 < c1 && drawn < 0; t0 += kChunk) {
        double w[kLane], sum = 0.0;  // this lane's entries, consecutive ones
        const int t = t0 + lane * kLane;
#pragma unroll
        for (int i = 0; i < kLane; ++i) {
          const bool in = t + i < c1 && t + i != skip;
          const float x = in ? to_f32(p[t + i]) : 0.f, y = in && less ? to_f32(q[t + i]) : 0.f;
          w[i] = weight_of(x, y);
          sum += w[i];
        }
        double d = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double up = __shfl_up_sync(0xffffffffu, d, o);
          if (lane >= o) d += up;
        }
        double at = run + (d - sum);
        int hit = -1, end = -1;
#pragma unroll
        for (int i = 0; i < kLane; ++i) {
          at += w[i];
          if (hit < 0 && w[i] > 0.0 && at > goal) hit = t + i;
          if (w[i] > 0.0) end = t + i;
        }
        const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), ends = __ballot_sync(0xffffffffu, end >= 0);
        if (hits != 0) drawn = __shfl_sync(0xffffffffu, hit, __ffs(hits) - 1);
        if (ends != 0) last = __shfl_sync(0xffffffffu, end, 31 - __clz(ends));
        run += __shfl_sync(0xffffffffu, d, 31);
      }
      if (drawn < 0) drawn = last;
    }
    break;
  }
  cluster.barrier_arrive();  // this block reads no other's sums any more
  int32_t *out = a.tokens + (int64_t)b * (a.drafts + 1);
  if (here && lane == 0) out[n] = drawn;
  if (rank == 0 && warp == 0) {
    if (lane == 0) a.accepted[b] = n;
    for (int i = lane; i <= a.drafts; i += 32)
      if (i != n || !found) out[i] = i < n ? __ldg(dtok + i) : -1;
  }
  cluster.barrier_wait();    // and none reads this block's
}

template <typename T>
int launch_verify(const VerifyArgs &a, cudaStream_t st) {
  // as many CTAs as have a chunk for each of their warps
  int c = 1;
  while (c < kMaxCluster && (int64_t)c * kWarps * kChunk < a.vocab) c *= 2;
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
  const uintptr_t rows = reinterpret_cast<uintptr_t>(a.target) | reinterpret_cast<uintptr_t>(a.draft) |
                         (uintptr_t)((int64_t)a.vocab * sizeof(T));
  if ((rows & 15) == 0)
    MSCO_CUDA_CHECK(cudaLaunchKernelEx(&cfg, verify_kernel<T, true>, a));
  else
    MSCO_CUDA_CHECK(cudaLaunchKernelEx(&cfg, verify_kernel<T, false>, a));
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
