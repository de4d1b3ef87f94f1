// Chunk attention on the 5th-generation tensor cores: head_dim 64 / 128, 16-bit and int8 caches.
//
// An item is up to 256 packed rows of one kv head (token-major, the q heads of the group adjacent) against the
// cached tokens that they see, or a split of them, 128 at a time.  Two streams keep the tensor cores busy:
// while one stream's 128 rows are in their softmax, the other's products run.
//   rows > 128   ("dual")   stream s owns rows 128 s .. 128 s + 127, both go over all KV tiles
//   rows <= 128  ("single") both streams own the same rows, stream s the KV tiles s, s + 2, ...; their states
//                           are merged at the end
// Per tile and stream:  S = Q K^T (shared x shared -> TMEM),  P = 2^(S scale - m) (registers, half a row per thread, back
// to TMEM in 16 bits over S),  O += P V (TMEM x shared -> TMEM).  The running maximum only moves when it grows by
// more than kSlack (a factor 256): until then P is up to 256 instead of 1, which costs no precision in a floating
// format, and O stays where it is; it is rescaled in TMEM by the softmax warps in the rare tiles where it must.
//
// Warps: 0 loads (TMA, 128-byte swizzle), 1 matrix instructions, 2 nothing (registers are handed out by groups of four
// warps), 3 the next items; int8 caches: four that convert; then eight of softmax for stream 0, eight for stream 1.
// The matrix instructions are issued O_0 += P_0 V, S_0 = Q_0 K', O_1 += P_1 V, S_1 = Q_1 K' (K' the next tile); they execute in
// that order, so a completed S' means that the product that read P, which lies over it, is complete too.
//
// What bounds it, head_dim 128, prompt of 8192 tokens, 32 / 8 heads (460 us, 1190 TFLOP/s of a measured 1653): the products
// themselves take 390 us of that with the softmax left out, since the tensor cores idle while the issuing warp waits for
// a barrier between two of them (150 clocks each).  head_dim 64: the exponentials (as many per product as at 128, for half
// the product).  Single tokens (282 us, 5.4 TB/s at contexts of 20k to 64k): the ring holds five tiles of 32 KB, and
// V waits for its tile's softmax; shorter splits lose more to their ends.  int8: the conversion's share of issue slots and
// shared memory (830 TFLOP/s on the same prompt).
#include <cuda.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "chunk_params.h"
#include "msco_common.cuh"
#include "tc05.cuh"

namespace msco {
namespace {

constexpr int kRows = 128;        // rows of one stream
constexpr int kTile = kChunkKvTile;
constexpr int kSoftWarps = 8;     // per stream
constexpr float kSlack = 8.f;     // log2 of how far a probability may exceed 1
constexpr float kLn2 = 0.6931471805599453f;
// polls before a wait gives up: over a second, while the longest legitimate wait is two items (2 us per tile of 128 tokens)
constexpr uint32_t kWaitLimit = 1u << 26;

__device__ int g_chunk_error;  // MSCO_ERR_TIMEOUT once a bounded wait has run out

template <int D, bool KV8>
struct Cfg {
  static_assert(D == 64 || D == 128, "head_dim 64 or 128");
  // four warps of loads and matrix instructions, four that convert int8 tiles, sixteen of softmax
  static constexpr int kFirstSoft = KV8 ? 8 : 4;
  static constexpr int kThreads = (kFirstSoft + 16) * 32;
  static constexpr int kBoxes = D / 64;                 // 128-byte wide sub-tiles of a row
  static constexpr int kSub = kTile * 128;              // bytes of one sub-tile
  static constexpr int kStageBytes = kTile * D * 2;
  static constexpr int kQBytes = kRows * D * 2;
  // ring of 16-bit tiles; int8 caches: four of them (what the matrix instructions look ahead) behind a ring of raw tiles
  static constexpr int kStages = KV8 ? 4 : (D == 128 ? 5 : 10);
  static constexpr int kRawBytes = kTile * D;
  static constexpr int kRaw = KV8 ? (D == 128 ? 2 : 8) : 0;
  static constexpr int kOffKv = 2 * kQBytes;
  static constexpr int kOffRaw = kOffKv + kStages * kStageBytes;
  static constexpr int kOffBar = kOffRaw + kRaw * kRawBytes;
  static constexpr int kNumBars = 2 * kStages + 2 * kRaw + 18;
  static constexpr int kOffResp = (kOffBar + kNumBars * 8 + 16 + 15) / 16 * 16;  // answers of the launch control
  static constexpr int kOffPair = kOffResp + 32;               // [8] items of the softmax pairs
  static constexpr int kOffXch = kOffPair + 32;  // [stream][half][row]: what the two threads of a row exchange
  static constexpr int kSmem = kOffXch + 2 * 2 * kRows * 4 + (KV8 ? (kRows + 32) * 4 : 0);
  // Of eight pairs of probabilities, those whose exponentials the FMA pipe computes.  At head_dim 128 the special-function
  // unit alone (1024 clocks a tile and stream) is as long as the two products: 2 of 8 took the prompt of 8192 tokens from
  // 503 to 460 us, 3 of 8 gave 475; at 64, where issue slots are short, any made it slower (316 us without, 355 with 2).
  static constexpr int kPolyOf8 = D == 128 ? 2 : 0;
  static constexpr int kColO = 2 * kTile;               // TMEM columns: S_0, S_1, O_0, O_1
};

// A bounded wait on an mbarrier.  Should one run out (a lost arrival), the block's flag is set, every wait of the block
// returns at once from then on, and all roles leave after their item, without waiting: whatever they do
// stays inside their buffers, the result is worthless and the device's error word says so.
__device__ __forceinline__ bool mbar_try_wait_at(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void mbar_arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
struct Waiter {
  volatile int *abort;
  __device__ __forceinline__ void operator()(uint64_t *bar, uint32_t parity) const { (*this)(smem_u32(bar), parity); }
  __device__ __forceinline__ void operator()(uint32_t bar, uint32_t parity) const {  // by a whole warp
    for (uint32_t i = 0; !mbar_try_wait_at(bar, parity); ++i) {
      if ((i & 255) != 255) continue;
      if (*abort) break;
      if (i >= kWaitLimit) {
        *abort = 1;
        atomicExch(&g_chunk_error, MSCO_ERR_TIMEOUT);
      }
    }
    __syncwarp();
  }
};

// Everything about an item that the roles share.
struct Work {
  ChunkItem it;
  int n;        // KV tiles
  int dual;
  int t1;       // first token of stream 1's rows (dual)
  int j0[2], j1[2];  // tiles of each stream, absolute
  int step;     // 1 (dual) or 2
};

// int8 cache: value of channel `c` from the mean x of its raw values (inv 0: nothing seen, stays 0)
__device__ __forceinline__ float dequant_out(const ChunkParams &p, int c, float x, float inv) {
  if (p.v_offset != nullptr && inv != 0.f) x += (float)__ldg(p.v_offset + c);
  return x * __ldg(p.v_descale + c);
}

// 32 aligned bytes: a whole sector in one store
__device__ __forceinline__ void store_32b(void *p, const uint32_t *r) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

template <int N>
__device__ __forceinline__ Work make_work(const ChunkSeqs<N> &seqs, const ChunkParams &p, int item) {
  Work w;
  w.it = chunk_item(seqs, p, item);
  const ChunkSeq &e = seqs.s[w.it.seq];
  const int half = p.item_tokens >> 1;
  w.n = max(0, w.it.tile1 - w.it.tile0);
  w.dual = w.it.tok1 - w.it.tok0 > half;
  w.t1 = w.it.tok0 + half;
  w.step = w.dual ? 1 : 2;
  if (w.dual) {
    // tiles that no row of the stream sees are left out: behind the last token of stream 0's rows, in front of
    // the window of stream 1's first
    const int pos0 = e.ctx - e.q_len;
    const int end0 = (max(0, pos0 + w.t1) + kTile - 1) / kTile;
    const int beg1 = p.window > 0 ? max(0, pos0 + w.t1 - p.window + 1) / kTile : 0;
    w.j0[0] = w.it.tile0;
    w.j1[0] = max(w.it.tile0, min(w.it.tile1, end0));
    w.j0[1] = min(max(w.it.tile0, beg1), max(w.it.tile0, w.it.tile1));
    w.j1[1] = max(w.it.tile0, w.it.tile1);
  } else {
    w.j0[0] = w.it.tile0;
    w.j0[1] = w.it.tile0 + 1;
    w.j1[0] = w.j1[1] = max(w.it.tile0, w.it.tile1);
  }
  return w;
}

// The grid has a block per item, longest first; a running block takes further items by cancelling blocks that have not
// started (cluster launch control), so that whoever is free takes the next longest.  One warp asks, two answers ahead at
// most; every other working warp reads each answer and says so.
struct Items {
  uint32_t resp, full, empty;  // shared addresses: 16-byte answers [2], mbarriers [2] each
  int item;
  uint32_t n;                  // answers read so far
  template <typename W>
  __device__ __forceinline__ bool next(const W &wait, int lane) {
    const uint32_t slot = n & 1;
    wait(full + slot * 8, (n >> 1) & 1);
    if (*wait.abort) return false;
    ++n;
    uint32_t ok, x;
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b128 h;\n\tld.shared.b128 h, [%2];\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\tselp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, _, _, _}, h;\n\t}"
        : "=r"(ok), "=r"(x)
        : "r"(resp + slot * 16)
        : "memory");
    fence_proxy_async();  // the answer's place is written next by the asynchronous proxy
    __syncwarp();
    if (lane == 0) mbar_arrive_at(empty + slot * 8);
    item = (int)x;
    return ok != 0;
  }
};

template <typename T, int D, bool KV8, int N>
__global__ void __launch_bounds__(Cfg<D, KV8>::kThreads, 1)
chunk_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ ChunkParams p,
                const __grid_constant__ ChunkSeqs<N> seqs) {
  using C = Cfg<D, KV8>;
  // int8 caches: all operands fp16, in which every int8 is exact
  using M = typename std::conditional<KV8, __half, T>::type;
  constexpr bool kBf16 = !std::is_same<M, __half>::value;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::kOffBar);
  uint64_t *kv_full = bars, *kv_empty = bars + C::kStages;
  uint64_t *q_full = bars + 2 * C::kStages, *q_empty = q_full + 1, *s_full = q_full + 2, *p_full = q_full + 4,
           *o_full = q_full + 6, *tail = q_full + 8, *fin = q_full + 9, *clc_full = q_full + 10, *clc_empty = q_full + 12,
           *m_free = q_full + 14, *merge_bar = q_full + 16, *q_full2 = q_full + 17, *raw_full = q_full + 18, *raw_empty = raw_full + C::kRaw;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + C::kNumBars);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  float *xch = reinterpret_cast<float *>(smem + C::kOffXch);
  float *q_scale = xch + 2 * 2 * kRows;  // int8, single: what stream 0 found for the rows, and for the first 32
  float *q_shift = q_scale + kRows;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&kv_full[i], KV8 ? 4 : 1);  // the copy, or the four converting warps
      mbar_init(&kv_empty[i], 1);
    }
    mbar_init(q_full, KV8 ? 2 * kSoftWarps : 1);   // even items
    mbar_init(q_full2, KV8 ? 2 * kSoftWarps : 1);  // odd items
    for (int i = 0; i < C::kRaw; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], 4);
    }
    mbar_init(q_empty, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], kSoftWarps);
      mbar_init(&o_full[s], 1);
    }
    mbar_init(tail, 1);
    mbar_init(merge_bar, 2 * kSoftWarps);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&clc_full[i], 1);
      mbar_init(&clc_empty[i], 2 + kSoftWarps + (KV8 ? 4 : 0));  // loads, matrix instructions, a warp of each softmax pair, conversion
      mbar_init(&m_free[i], 1);
    }
    mbar_init(fin, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const Waiter wait{abort_flag};
  const int half = p.item_tokens >> 1;
  const Items items = {smem_u32(smem + C::kOffResp), smem_u32(clc_full), smem_u32(clc_empty), (int)blockIdx.x, 0};

  // Registers: 640 x 96 at launch = 512 x 104 (softmax) + 128 x 64, with the converting warps 768 x 80 = 512 x 96 + 256 x 48
  if (warp < C::kFirstSoft) {
    if (KV8) asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
  }
  if (warp == 0) {
    // ------------------------------------------------------------------ loads
    if (lane == 0) {
      prefetch_tmap(&tm_q);
      prefetch_tmap(&tm_k);
      prefetch_tmap(&tm_v);
    }
    const int bs = p.block_size;
    const int box_rows = min(bs, kTile), boxes = kTile / box_rows;
    uint32_t c = 0, q_round = 0, tails = 0;  // ring position, items so far, waits on `tail` so far
    for (Items it = items; it.item >= 0; it.item = it.next(wait, lane) ? it.item : -1) {
      const Work w = make_work(seqs, p, it.item);
      if (w.n == 0) continue;
      const ChunkSeq &e = seqs.s[w.it.seq];
      // cached tokens that some new token of the sequence sees: the rest of the table may hold anything
      const int alive0 = p.window > 0 ? max(0, e.ctx - e.q_len - p.window + 1) : 0, alive1 = e.ctx;
      const int32_t *table = p.block_tables + (int64_t)e.row * p.max_blocks_per_seq;
      // The item's query rows.  Their space is free when the last products on them are complete; its second tile also holds
      // the merge of the two streams of a single item, so a dual item waits for the one in front to be through with that.
      const uint32_t k_item = q_round++;
      auto load_q = [&]() {
        if (KV8) return;  // the softmax warps fold the scales into them
        if (k_item >= 1) wait(q_empty, (k_item - 1) & 1);
        if (k_item >= 2) wait(&m_free[k_item & 1], ((k_item - 2) >> 1) & 1);
        if (w.dual && k_item >= 1) wait(&m_free[(k_item - 1) & 1], ((k_item - 1) >> 1) & 1);
        uint64_t *bar = k_item & 1 ? q_full2 : q_full;
        if (lane == 0) {
          const int tiles = w.dual ? 2 : 1;
          mbar_arrive_expect_tx(bar, (uint32_t)(tiles * C::kBoxes * half * p.group * 128));
          for (int s = 0; s < tiles; ++s)
            for (int x = 0; x < C::kBoxes; ++x)
              tma_load_3d(smem + s * C::kQBytes + x * (kRows * 128), &tm_q, x * 64, w.it.kvh * p.group,
                          e.q_start + (s == 0 ? w.it.tok0 : w.t1), bar);
        }
        __syncwarp();
      };
      int win = -1;        // first block-table column of the 32 ids that the lanes hold
      int32_t id = 0;
      // one tile of K or V into the next stage of the ring
      auto load = [&](const CUtensorMap *tm, int j, bool is_v) {
        constexpr int kRing = KV8 ? C::kRaw : C::kStages;
        const uint32_t st = c % kRing, use = c / kRing;
        ++c;
        if (use > 0) wait(KV8 ? &raw_empty[st] : &kv_empty[st], (use - 1) & 1);
        uint8_t *dst = smem + (KV8 ? C::kOffRaw + st * C::kRawBytes : C::kOffKv + st * C::kStageBytes);
        const int tok = j * kTile;
        const int a = max(0, alive0 - tok), b = min(kTile, alive1 - tok);  // rows of the tile that are alive
        const int b0 = a / box_rows, b1 = (b + box_rows - 1) / box_rows;   // boxes that hold some of them
        // a V row that is not alive is zeroed: its probability is 0, but what it holds may not be finite
        // (int8: the converting warps see to it)
        const bool patch = !KV8 && is_v && (a > 0 || b < kTile);
        uint64_t *bar = KV8 ? &raw_full[st] : (patch ? tail : &kv_full[st]);
        const int col = (tok + lane * box_rows) / bs;  // this lane's block-table column (boxes <= 16)
        const int first = tok / bs;
        if (win < 0 || first < win || (tok + kTile - 1) / bs >= win + 32) {
          win = first;
          const int wc = win + lane;
          id = wc < p.max_blocks_per_seq && (int64_t)wc * bs < alive1 ? __ldg(table + wc) : 0;
        }
        const bool mine = lane >= b0 && lane < b1 && lane < boxes;
        int32_t blk = __shfl_sync(0xffffffffu, id, mine ? col - win : 0);
        if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)((b1 - b0) * box_rows * (KV8 ? D : 2 * D)));
        __syncwarp();
        if (mine) {
          if (blk < 0 || blk >= p.num_blocks) {
            if (p.oob_count != nullptr && !is_v) atomicAdd(p.oob_count, 1);
            blk = 0;
          }
          const int off = (tok + lane * box_rows) % bs;
          const int y = p.cache_layout == 1 ? off : w.it.kvh;
          const int z = p.cache_layout == 1 ? blk * p.num_kv_heads + w.it.kvh : blk * bs + off;
          if (KV8) {
            tma_load_3d(dst + lane * box_rows * D, tm, 0, y, z, bar);
          } else {
#pragma unroll
            for (int x = 0; x < C::kBoxes; ++x) tma_load_3d(dst + x * C::kSub + lane * box_rows * 128, tm, x * 64, y, z, bar);
          }
        }
        if (patch) {
          wait(tail, tails & 1);
          ++tails;
          for (int i = lane; i < kTile * 8 * C::kBoxes; i += 32) {  // 16-byte pieces; a row is 128 bytes of a sub-tile
            const int x = i / (kTile * 8), row = (i / 8) % kTile;
            if (row < a || row >= b)
              *reinterpret_cast<uint4 *>(dst + x * C::kSub + row * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&kv_full[st]);
        }
      };
      // The order in which the tiles are used: V of a tile right in front of the K that follows it on its stream.  The query
      // rows come behind the first four tiles, which do not wait for the item in front to end.
      const int ahead = w.step, total = 2 * w.n;
      int issued = 0;
      auto step = [&](const CUtensorMap *tm, int j, bool is_v) {
        if (issued == min(4, total - 1)) load_q();
        ++issued;
        load(tm, j, is_v);
      };
      for (int i = 0; i < min(ahead, w.n); ++i) step(&tm_k, w.it.tile0 + i, false);
      for (int i = 0; i < w.n; ++i) {
        step(&tm_v, w.it.tile0 + i, true);
        if (i + ahead < w.n) step(&tm_k, w.it.tile0 + i + ahead, false);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ matrix instructions
    // This warp is the block's pace: the queue of matrix instructions is a few deep, so whatever it does between them the
    // tensor cores wait for.  The whole warp goes through the loop (addresses and descriptors stay in uniform registers),
    // one elected lane issues, and everything between two waits is issued in one go.
    constexpr uint32_t kIdQk = mma_idesc<kBf16, kRows, kTile, false>();
    constexpr uint32_t kIdPv = mma_idesc<kBf16, kRows, D, true>();
    constexpr uint32_t kStep = C::kStageBytes >> 4;
    const uint64_t dq = smem_desc(smem_u32(smem));
    const uint64_t dk = smem_desc(smem_u32(smem + C::kOffKv)), dv = smem_desc(smem_u32(smem + C::kOffKv), C::kSub);
    const uint32_t b_full = smem_u32(kv_full), b_empty = smem_u32(kv_empty), b_s = smem_u32(s_full), b_p = smem_u32(p_full),
                   b_o = smem_u32(o_full), b_q = smem_u32(q_empty);
    uint32_t st = 0, st_par = 0, k_item = 0, p_par0 = 0, p_par1 = 0;
    auto take = [&]() {  // the next stage of the ring, filled
      const uint32_t now = st;
      wait(b_full + now * 8, st_par);
      if (++st == C::kStages) {
        st = 0;
        st_par ^= 1;
      }
      return now;
    };
    auto pv = [&](int s, uint64_t b, bool acc) {  // the halves' P lie 64 columns apart
#pragma unroll
      for (int k = 0; k < kTile / 16; ++k)
        mma_ts(tmem + C::kColO + s * D, tmem + s * kTile + (k >> 2) * 64 + (k & 3) * 8, b + (k * 2048 >> 4), kIdPv, acc || k > 0);
    };
    auto qk = [&](int s, uint64_t a, uint64_t b) {
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t off = ((k / 4) * (kRows * 128) + (k % 4) * 32) >> 4;
        mma_ss(tmem + s * kTile, a + off, b + off, kIdQk, k > 0);
      }
      tc_commit_at(b_s + s * 8);
    };
    auto wait_p = [&](int s) {
      uint32_t &par = s == 0 ? p_par0 : p_par1;
      wait(b_p + s * 8, par);
      par ^= 1;
      tc_fence_after();
    };
    for (Items it = items; it.item >= 0; it.item = it.next(wait, lane) ? it.item : -1) {
      const Work w = make_work(seqs, p, it.item);
      if (w.n == 0) continue;
      wait(k_item & 1 ? q_full2 : q_full, (k_item >> 1) & 1);
      ++k_item;
      if (w.dual) {
        // V of tile j, then K of tile j + 1; the streams alternate.  The next pair of stages is waited for behind stream 0's
        // products, while they run.
        uint32_t sv = 0, sk = take();
        for (int j = w.it.tile0 - 1; j < w.it.tile1; ++j) {
          const bool has_v = j >= w.it.tile0, has_k = j + 1 < w.it.tile1;
          const bool av0 = has_v && j < w.j1[0], av1 = has_v && j >= w.j0[1];
          const bool ak0 = has_k && j + 1 < w.j1[0], ak1 = has_k && j + 1 >= w.j0[1];
          tc_fence_after();
          if (av0) wait_p(0);
          if (elect_one()) {
            if (av0) {
              pv(0, dv + sv * kStep, j > w.j0[0]);
              if (j + 1 == w.j1[0]) tc_commit_at(b_o);
            }
            if (ak0) qk(0, dq, dk + sk * kStep);
          }
          __syncwarp();
          uint32_t nv = 0, nk = 0;
          if (has_k) nv = take();
          if (j + 2 < w.it.tile1) nk = take();
          if (av1) wait_p(1);
          if (elect_one()) {
            if (av1) {
              pv(1, dv + sv * kStep, j > w.j0[1]);
              if (j + 1 == w.j1[1]) tc_commit_at(b_o + 8);
            }
            if (has_v) tc_commit_at(b_empty + sv * 8);
            if (ak1) qk(1, dq + (C::kQBytes >> 4), dk + sk * kStep);
            if (has_k) {
              tc_commit_at(b_empty + sk * 8);
              if (j + 2 >= w.it.tile1) tc_commit_at(b_q);
            }
          }
          __syncwarp();
          sv = nv;
          sk = nk;
        }
      } else {
        // V of tile i, then K of tile i + 2, both on stream i & 1
        for (int i = -2; i < w.n; ++i) {
          const bool has_v = i >= 0, has_k = i + 2 < w.n;
          const uint32_t sv = has_v ? take() : 0, sk = has_k ? take() : 0;
          tc_fence_after();
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if ((i & 1) != s) continue;
            if (has_v) wait_p(s);
            if (elect_one()) {
              if (has_v) {
                pv(s, dv + sv * kStep, i > 1);
                if (i + 2 >= w.n) tc_commit_at(b_o + s * 8);
                tc_commit_at(b_empty + sv * 8);
              }
              if (has_k) {
                qk(s, dq, dk + sk * kStep);
                tc_commit_at(b_empty + sk * 8);
                if (i + 3 == w.n) tc_commit_at(b_q);
              }
            }
            __syncwarp();
          }
        }
      }
    }
    if (elect_one()) tc_commit(fin);  // every arrival that the instructions still owe has happened before the block ends
    __syncwarp();
    wait(fin, 0);
  } else if (warp == 3) {
    // ------------------------------------------------------------------ the next items
    for (uint32_t n = 0;; ++n) {
      const uint32_t slot = n & 1;
      if (n >= 2) wait(&clc_empty[slot], ((n >> 1) - 1) & 1);
      if (*abort_flag) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&clc_full[slot], 16);
        asm volatile(
            "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                items.resp + slot * 16),
            "r"(smem_u32(&clc_full[slot]))
            : "memory");
      }
      wait(&clc_full[slot], (n >> 1) & 1);
      uint32_t ok;
      asm volatile(
          "{\n\t.reg .pred p;\n\t.reg .b128 h;\n\tld.shared.b128 h, [%1];\n\t"
          "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\tselp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(ok)
          : "r"(items.resp + slot * 16)
          : "memory");
      if (ok == 0) break;  // nothing left (asking again would not be allowed)
    }
  } else if (warp < C::kFirstSoft) {
    if constexpr (KV8) {
      if (warp >= 4) {
      // ------------------------------------------------------------------ int8 tiles to fp16, a quarter of a tile per warp
      // A byte u = x + 128 under 0x64 is the fp16 1024 + u, exactly; 1152 taken off gives x.
      uint32_t c = 0;
      const int r_first = (warp - 4) * (kTile / 4);
      for (Items it = items; it.item >= 0; it.item = it.next(wait, lane) ? it.item : -1) {
        const Work w = make_work(seqs, p, it.item);
        if (w.n == 0) continue;
        const ChunkSeq &e = seqs.s[w.it.seq];
        const int alive0 = p.window > 0 ? max(0, e.ctx - e.q_len - p.window + 1) : 0, alive1 = e.ctx;
        auto convert = [&](int j) {
          const uint32_t rs = c % C::kRaw, st = c % C::kStages, raw_use = c / C::kRaw, use = c / C::kStages;
          ++c;
          wait(&raw_full[rs], raw_use & 1);
          if (use > 0) wait(&kv_empty[st], (use - 1) & 1);
          const uint8_t *src = smem + C::kOffRaw + rs * C::kRawBytes;
          uint8_t *dst = smem + C::kOffKv + st * C::kStageBytes;
          const int tok = j * kTile;
          const int a = max(0, alive0 - tok), b = min(kTile, alive1 - tok);  // rows that are alive; the others become zero
          constexpr int kPieces = D / 16;  // 16-byte pieces of a raw row
            constexpr int kBatch = D / 32;  // pieces of a lane that are read before the first is converted
#pragma unroll 1
          for (int i0 = lane; i0 < kTile / 4 * kPieces; i0 += 32 * kBatch) {
            uint4 v[kBatch];
#pragma unroll
            for (int n = 0; n < kBatch; ++n) {
              const int i = i0 + n * 32, row = r_first + i / kPieces;
              v[n] = *reinterpret_cast<const uint4 *>(src + row * D + i % kPieces * 16);
              if (row < a || row >= b) v[n] = make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int n = 0; n < kBatch; ++n) {
              const int i = i0 + n * 32, row = r_first + i / kPieces, pc = i % kPieces;
              uint32_t o[8];
              const uint32_t in[4] = {v[n].x, v[n].y, v[n].z, v[n].w};
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint32_t u = in[k] ^ 0x80808080u;
                const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1152
                uint32_t lo = __byte_perm(u, 0x64646464u, 0x4140), hi = __byte_perm(u, 0x64646464u, 0x4342);
                __half2 l2 = __hsub2(*reinterpret_cast<__half2 *>(&lo), bias), h2 = __hsub2(*reinterpret_cast<__half2 *>(&hi), bias);
                o[2 * k] = *reinterpret_cast<uint32_t *>(&l2);
                o[2 * k + 1] = *reinterpret_cast<uint32_t *>(&h2);
              }
              // two 16-byte chunks of the swizzled row; lanes of the second sub-tile write theirs in the other order, so
              // that the eight lanes of a row hit eight different chunks
              uint8_t *base = dst + (pc / 4) * C::kSub + row * 128;
              const int ch = (pc % 4) * 2, odd = (pc / 4) & 1;
              const uint4 c0 = make_uint4(o[0], o[1], o[2], o[3]), c1 = make_uint4(o[4], o[5], o[6], o[7]);
              *reinterpret_cast<uint4 *>(base + (((ch + odd) ^ (row & 7)) << 4)) = odd ? c1 : c0;
              *reinterpret_cast<uint4 *>(base + (((ch + 1 - odd) ^ (row & 7)) << 4)) = odd ? c0 : c1;
            }
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&kv_full[st]);
            mbar_arrive(&raw_empty[rs]);
          }
        };
        const int ahead = w.step;
        for (int i = 0; i < min(ahead, w.n); ++i) convert(w.it.tile0 + i);
        for (int i = 0; i < w.n; ++i) {
          convert(w.it.tile0 + i);
          if (i + ahead < w.n) convert(w.it.tile0 + i + ahead);
        }
      }
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax, two threads per row
    // The threads of a row are in two warps, one for each half of a tile's columns (and of O's): with four softmax warps
    // on each scheduler the latencies of one hide behind the others.  They exchange their halves' maxima.
    if (KV8) asm volatile("setmaxnreg.inc.sync.aligned.u32 96;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    const int s = (warp - C::kFirstSoft) >> 3, hf = ((warp >> 2) & 1) ^ 1;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)(warp & 3) * 32 << 16;
    const uint32_t t_s = tmem + lanes + s * kTile + hf * 64, t_o = tmem + lanes + C::kColO + s * D + hf * (D / 2);
    // Named barrier of the two warps of these rows.  One of them takes the items for both, so that neither leaves (when a
    // wait has run out, too) while the other still comes to this barrier.  The barrier of all softmax warps, once in an item
    // that merges, is a bounded wait like the others: pairs may leave on their own.
    const int pair = 1 + s * 4 + (warp & 3);
    volatile int *pair_item = reinterpret_cast<volatile int *>(smem + C::kOffPair) + s * 4 + (warp & 3);
    const uint32_t b_merge = smem_u32(merge_bar);
    uint32_t merge_par = 0;
    auto pair_sync = [&]() { named_bar_sync(pair, 64); };
    auto merge_sync = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive_at(b_merge);
      wait(b_merge, merge_par);
      merge_par ^= 1;
    };
    float *x_mine = xch + (s * 2 + hf) * kRows + row, *x_other = xch + (s * 2 + (hf ^ 1)) * kRows + row;
    const int g = p.group;
    const int tok_in = row / g, head_in = row - tok_in * g;
    const bool speaker = s == 1 && hf == 0 && (warp & 3) == 0;  // the warp that speaks for its stream
    uint32_t s_round = 0, o_round = 0, k_items = 0;
    Items it = items;
    for (int item = it.item; item >= 0;) {
      const Work w = make_work(seqs, p, item);
      const ChunkSeq &e = seqs.s[w.it.seq];
      const int tok0 = w.dual && s == 1 ? w.t1 : w.it.tok0;
      const int ntok = min(half, w.it.tok1 - tok0);
      const bool live = tok_in < ntok;  // this thread has a row
      const bool warp_live = __any_sync(0xffffffffu, live);
      const int pos0 = e.ctx - e.q_len + tok0;
      const int pos = live ? pos0 + tok_in : -1;
      const int j_beg = s == 0 ? w.j0[0] : w.j0[1], j_end = s == 0 ? w.j1[0] : w.j1[1];
      const uint32_t k_item = k_items;
      if (w.n > 0) ++k_items;
      float m = -INFINITY, l = 0.f;
      float sc = p.scale_log2e;  // score -> log2 domain
      float shift = 0.f;         // int8 with offsets: the part of a row's scores that all tokens share (for the lse)
      if (KV8 && w.n > 0) {
        // Q' = q * k_descale, scaled by a power of two to a largest magnitude of 2^13 .. 2^14 and rounded to fp16 (2^-11 of
        // each, whatever the scales), into this stream's tile (single: stream 0's).  The tile is free: this stream's products
        // of the item in front are complete, and those of the other on the same tile by the merge.
        if (w.dual || s == 0) {
          float top = 0.f, off = 0.f;
          const T *src = static_cast<const T *>(p.q) +
                         (((int64_t)e.q_start + tok0 + tok_in) * p.num_q_heads + w.it.kvh * g + head_in) * D + hf * (D / 2);
          const float *ds = p.k_descale + w.it.kvh * D + hf * (D / 2);
          const int32_t *of = p.k_offset == nullptr ? nullptr : p.k_offset + w.it.kvh * D + hf * (D / 2);
          float q[D / 2];
#pragma unroll
          for (int c = 0; c < D / 2; c += 8) {
            uint4 v = live ? __ldg(reinterpret_cast<const uint4 *>(src + c)) : make_uint4(0, 0, 0, 0);
            const T *qe = reinterpret_cast<const T *>(&v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              q[c + i] = to_f32(qe[i]) * __ldg(ds + c + i);
              top = fmaxf(top, fabsf(q[c + i]));
              if (of != nullptr) off = fmaf(q[c + i], (float)__ldg(of + c + i), off);
            }
          }
          *x_mine = top;
          pair_sync();
          top = fmaxf(top, *x_other);
          pair_sync();
          if (of != nullptr) {
            *x_mine = off;
            pair_sync();
            off += *x_other;
            pair_sync();
          }
          const int ex = min(max((int)(__float_as_uint(top) >> 23) - 127, -113), 128);  // exponent of the largest
          const float up = top > 0.f ? __uint_as_float((uint32_t)(127 + 13 - ex) << 23) : 1.f;
          uint8_t *dst = smem + (w.dual ? s * C::kQBytes : 0) + row * 128;
#pragma unroll
          for (int c = 0; c < D / 2; c += 8) {
            const int col = hf * (D / 2) + c;
            const uint4 v = make_uint4(pack2<M>(q[c] * up, q[c + 1] * up), pack2<M>(q[c + 2] * up, q[c + 3] * up),
                                       pack2<M>(q[c + 4] * up, q[c + 5] * up), pack2<M>(q[c + 6] * up, q[c + 7] * up));
            *reinterpret_cast<uint4 *>(dst + (col / 64) * (kRows * 128) + ((((col % 64) / 8) ^ (row & 7)) << 4)) = v;
          }
          sc = p.scale_log2e / up;
          shift = off * p.scale_log2e;
          if (!w.dual && hf == 0) q_scale[row] = sc;
          if (!w.dual && hf == 0 && row < 32) q_shift[row] = shift;
          fence_proxy_async();
        }
        __syncwarp();
        uint64_t *bar = k_item & 1 ? q_full2 : q_full;
        if (lane == 0) mbar_arrive(bar);
        wait(bar, (k_item >> 1) & 1);  // (single: stream 1 takes its rows' scales from stream 0; and nobody runs ahead)
        if (!w.dual && s == 1) sc = q_scale[row];
      }
      if (!KV8 && speaker && w.n > 0) {
        // Stream 1 says when the second tile of Q's space is not (dual), or not any more (single: behind the merge), a merge
        // buffer.  It does so behind the arrival of the item's rows, so never before the item in front is done with.
        wait(k_item & 1 ? q_full2 : q_full, (k_item >> 1) & 1);
        if (w.dual && lane == 0) mbar_arrive(&m_free[k_item & 1]);
      }
      for (int j = j_beg; j < j_end; j += w.step) {
        wait(&s_full[s], s_round & 1);
        ++s_round;
        tc_fence_after();
        if (warp_live) {
          uint32_t x[64];
          tmem_ld32(t_s, x);
          tmem_ld32(t_s + 32, x + 32);
          tmem_wait_ld32(x);
          tmem_wait_ld32(x + 32);
          const int col0 = j * kTile + hf * 64;
          if (pos0 < col0 + 63 || (p.window > 0 && pos0 + ntok - p.window > col0)) {
            const int hi = pos - col0;                                    // columns 0 .. hi are seen
            const int lo = p.window > 0 ? pos - p.window + 1 - col0 : 0;  // from column lo on
#pragma unroll
            for (int c = 0; c < 64; ++c) x[c] = c <= hi && c >= lo ? x[c] : 0xff800000u;  // -inf
          }
          // four chains of three-way maxima: one chain would be 64 dependent steps
          float mx4[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) mx4[i] = __uint_as_float(x[i]);
#pragma unroll
          for (int c = 4; c < 60; c += 8)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              mx4[i] = fmaxf(mx4[i], fmaxf(__uint_as_float(x[c + i]), __uint_as_float(x[c + 4 + i])));
#pragma unroll
          for (int i = 0; i < 4; ++i) mx4[i] = fmaxf(mx4[i], __uint_as_float(x[60 + i]));
          float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
          // (the next tile's exchange comes behind that tile's s_full, which both warps' p_full of this one precede)
          *x_mine = mx;
          pair_sync();
          mx = fmaxf(mx, *x_other) * sc;
          const bool first = j == j_beg;
          const bool grow = mx > m + kSlack;  // also for the first value: m is -inf
          if (__any_sync(0xffffffffu, grow)) {
            const float w_old = grow ? fast_exp2(m - mx) : 1.f;
            m = grow ? mx : m;
            l *= w_old;
            if (!first) {
#pragma unroll 1
              for (int c = 0; c < D / 2; c += 16) {
                uint32_t o[16];
                tmem_ld16(t_o + c, o);
                tmem_wait_ld16(o);
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * w_old);
                tmem_st16(t_o + c, o);
              }
            }
          }
          const float base = m == -INFINITY ? 0.f : m;
          const uint64_t scale2 = pack_f32x2(sc, sc), base2 = pack_f32x2(-base, -base);
          uint64_t sum2[2] = {0, 0};
#pragma unroll
          for (int c0 = 0; c0 < 64; c0 += 32) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const uint64_t v = fma_f32x2(pack_f32x2(__uint_as_float(x[c0 + i]), __uint_as_float(x[c0 + i + 1])), scale2, base2);
              float a, b;
              unpack_f32x2(v, a, b);
              if ((i >> 1) % 8 < C::kPolyOf8) {
                exp2_poly2(v, a, b);
              } else {
                a = fast_exp2(a);
                b = fast_exp2(b);
              }
              sum2[(i >> 1) & 1] = add_f32x2(sum2[(i >> 1) & 1], pack_f32x2(a, b));
              pk[i / 2] = pack2<M>(a, b);
            }
            tmem_st16(t_s + c0 / 2, pk);
          }
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[s]);
          float s0, s1;
          unpack_f32x2(add_f32x2(sum2[0], sum2[1]), s0, s1);
          l += s0 + s1;
          if (m == -INFINITY) l = 0.f;  // nothing seen so far: the polynomial's 2^-126 does not count
        } else if (lane == 0) {
          mbar_arrive(&p_full[s]);
        }
      }
      // ---- the item's result
      const bool has = j_beg < j_end;
      if (has) {
        wait(&o_full[s], o_round & 1);
        ++o_round;
        tc_fence_after();
      }
      // the row's sum (o_full: both warps are through with the exchanges of the tiles)
      if (warp_live) {
        *x_mine = l;
        pair_sync();
        l += *x_other;
      }
      const bool two = !w.dual && w.n > 1;  // two states of the same rows
      const bool split = e.nsplit > 1;
      const int tile_rows = min(p.item_tokens, e.q_len) * g;
      const int64_t part_row0 = (int64_t)e.part_base +
                                ((int64_t)(w.it.qtile * e.nsplit + w.it.split) * p.num_kv_heads + w.it.kvh) * tile_rows;
      if (two && ntok * g <= 32) {
        // Up to 32 rows (one warp of each half has them): both streams lay all their columns down, [stream][column][row], and
        // all 512 threads add and write eight columns of a row each.  Row by row, as below, this took 7000 clocks of an
        // item that reads its four tiles in 11000.
        float *buf = reinterpret_cast<float *>(smem + C::kQBytes);
        if (warp_live) {
          pair_sync();  // the sums have been read
          *x_mine = hf == 0 ? m : l;
#pragma unroll 1
          for (int c = 0; c < D / 2; c += 32) {
            uint32_t o[32];
            tmem_ld32(t_o + c, o);
            tmem_wait_ld32(o);
            float *dst = buf + (s * D + hf * (D / 2) + c) * 32 + lane;
#pragma unroll
            for (int i = 0; i < 32; ++i) dst[i * 32] = __uint_as_float(o[i]);
          }
        }
        tc_fence_before();
        merge_sync();
        const int rows = ntok * g, n = (int)threadIdx.x - C::kFirstSoft * 32;
        const int rr = n % rows, c0 = n / rows * 8;
        if (c0 < D) {
          const float m0 = xch[rr], l0 = xch[kRows + rr], m1 = xch[2 * kRows + rr], l1 = xch[3 * kRows + rr];
          const float mm = fmaxf(m0, m1), b = mm == -INFINITY ? 0.f : mm;
          const float f0 = fast_exp2(m0 - b), f1 = fast_exp2(m1 - b), ll = l0 * f0 + l1 * f1;
          uint32_t o[8];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            o[i] = __float_as_uint(buf[(c0 + i) * 32 + rr] * f0 + buf[(D + c0 + i) * 32 + rr] * f1);
          const int64_t orow2 = ((int64_t)e.q_start + tok0 + rr / g) * p.num_q_heads + w.it.kvh * g + rr % g;
          const float m_row = mm + (KV8 ? q_shift[rr] : 0.f);
          if (split) {
            store_32b(p.part_o + (part_row0 + rr) * D + c0, o);
            if (c0 == 0) *reinterpret_cast<float2 *>(p.part_ml + (part_row0 + rr) * 2) = make_float2(m_row, ll);
          } else {
            const float inv2 = ll > 0.f ? 1.f / ll : 0.f;
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              f[i] = __uint_as_float(o[i]) * inv2;
              if (KV8) f[i] = dequant_out(p, w.it.kvh * D + c0 + i, f[i], inv2);
            }
            *reinterpret_cast<uint4 *>(static_cast<T *>(p.out) + orow2 * D + c0) =
                make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
            if (c0 == 0 && p.lse != nullptr) p.lse[orow2] = ll > 0.f ? (m_row + log2f(ll)) * kLn2 : -INFINITY;
          }
        }
        fence_proxy_async();  // the buffer's next use is by the loads
        merge_sync();
      } else {
      float scale0 = 1.f, scale1 = 0.f, m_out = m, l_out = l;
      if (two) {
        if (s == 1) {
          if (warp_live) pair_sync();  // the sums have been read
          *x_mine = hf == 0 ? m : l;
        }
        merge_sync();
        if (s == 0) {
          const float m1 = xch[2 * kRows + row], l1 = xch[3 * kRows + row];
          m_out = fmaxf(m, m1);
          const float b = m_out == -INFINITY ? 0.f : m_out;
          scale0 = fast_exp2(m - b);
          scale1 = fast_exp2(m1 - b);
          l_out = l * scale0 + l1 * scale1;
        }
      }
      const int64_t tok = (int64_t)e.q_start + tok0 + tok_in;
      const int64_t orow = tok * p.num_q_heads + w.it.kvh * g + head_in;
      const int64_t prow = part_row0 + (tok0 - w.it.tok0) * g + row;
      const float inv = split ? 1.f : (l_out > 0.f ? 1.f / l_out : 0.f);
      const bool writes = live && (w.dual || s == 0);
      // This half's columns that go through the merge buffer (the space of Q's second tile) at a time: with up to 64 rows
      // all of them.
      const bool few = ntok * g <= 64;
      const int part = few ? D / 2 : D / 4, stride = few ? 64 : kRows;
      float *buf = reinterpret_cast<float *>(smem + C::kQBytes) + hf * (part * stride) + row;
#pragma unroll 1
      for (int c0 = 0; c0 < D / 2; c0 += part) {
#pragma unroll 1
        for (int c = 0; c < part; c += 16) {
          uint32_t o[16];
          if (warp_live && has) {
            tmem_ld16(t_o + c0 + c, o);
            tmem_wait_ld16(o);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = 0;
          }
          if (two) {
            // stream 1 lays its columns down one by one (consecutive rows: no bank conflicts), stream 0 adds them in
            if (s == 1) {
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (warp_live) buf[(c + i) * stride] = __uint_as_float(o[i]);
              if (c + 16 < part) continue;
            }
            if (c == (s == 1 ? part - 16 : 0)) merge_sync();
            if (s == 1) continue;
#pragma unroll
            for (int i = 0; i < 16; ++i)
              o[i] = __float_as_uint(__uint_as_float(o[i]) * scale0 + (warp_live ? buf[(c + i) * stride] : 0.f) * scale1);
          }
          if (writes) {
            const int col = hf * (D / 2) + c0 + c;
            if (split) {
              float *dst = p.part_o + prow * D + col;
              store_32b(dst, o);
              store_32b(dst + 8, o + 8);
            } else {
              uint32_t pk[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                float a = __uint_as_float(o[2 * i]) * inv, b = __uint_as_float(o[2 * i + 1]) * inv;
                if (KV8) {
                  a = dequant_out(p, w.it.kvh * D + col + 2 * i, a, inv);
                  b = dequant_out(p, w.it.kvh * D + col + 2 * i + 1, b, inv);
                }
                pk[i] = pack2<T>(a, b);
              }
              store_32b(static_cast<T *>(p.out) + orow * D + col, pk);
            }
          }
        }
        if (two) {
          fence_proxy_async();  // the buffer's next use is by the loads
          merge_sync();
        }
      }
      if (writes && hf == 0) {
        m_out += shift;
        if (split) *reinterpret_cast<float2 *>(p.part_ml + prow * 2) = make_float2(m_out, l_out);
        else if (p.lse != nullptr) p.lse[orow] = l_out > 0.f ? (m_out + log2f(l_out)) * kLn2 : -INFINITY;
      }
      }
      // the merge buffer lies over Q's second tile: only now may the next item's rows come in
      if (!KV8 && speaker && w.n > 0 && !w.dual && lane == 0) mbar_arrive(&m_free[k_item & 1]);
      tc_fence_before();  // the reads of O are ordered before the next item's products (which wait for its P)
      if (hf == 0) {
        const bool more = it.next(wait, lane);
        if (lane == 0) *pair_item = more ? it.item : -1;
      }
      pair_sync();
      item = *pair_item;
      pair_sync();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) __nanosleep(1000000);  // copies that nothing has waited for land before the block's memory is given back
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// One warp per (token, q head) of the sequences that were split: the log-sum-exp merge in split order.
template <typename T, int D, int N>
__global__ void __launch_bounds__(256) chunk_merge_kernel(const __grid_constant__ ChunkParams p,
                                                         const __grid_constant__ ChunkSeqs<N> seqs) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const ChunkSeq &e = seqs.s[blockIdx.y];
  if (e.nsplit <= 1) return;
  const int lane = threadIdx.x & 31;
  const int64_t rows = (int64_t)e.q_len * p.num_q_heads;
  constexpr int kCols = D / 32;
  for (int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); w < rows; w += (int64_t)gridDim.x * 8) {
    const int tok = (int)(w / p.num_q_heads), hq = (int)(w - (int64_t)tok * p.num_q_heads);
    const int kvh = hq / p.group, h = hq - kvh * p.group;
    const int qtile = tok / p.item_tokens;
    const int tile_rows = min(p.item_tokens, e.q_len) * p.group;
    const int64_t prow0 = (int64_t)e.part_base + ((int64_t)qtile * e.nsplit * p.num_kv_heads + kvh) * tile_rows +
                          (tok - qtile * p.item_tokens) * p.group + h;
    const int64_t step = (int64_t)p.num_kv_heads * tile_rows;
    float m = -INFINITY;
    for (int s = lane; s < e.nsplit; s += 32) m = fmaxf(m, __ldcg(p.part_ml + (prow0 + s * step) * 2));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f, acc[kCols];
#pragma unroll
    for (int c = 0; c < kCols; ++c) acc[c] = 0.f;
    for (int s = 0; s < e.nsplit; ++s) {
      const int64_t pr = prow0 + s * step;
      const float2 v = __ldcg(reinterpret_cast<const float2 *>(p.part_ml + pr * 2));
      const float f = fast_exp2(v.x - base);
      l = fmaf(f, v.y, l);
      const float *src = p.part_o + pr * D + lane * kCols;
      if (kCols == 4) {
        const float4 t = __ldcg(reinterpret_cast<const float4 *>(src));
        acc[0] = fmaf(f, t.x, acc[0]); acc[1] = fmaf(f, t.y, acc[1]);
        acc[2] = fmaf(f, t.z, acc[2]); acc[kCols - 1] = fmaf(f, t.w, acc[kCols - 1]);
      } else {
        const float2 t = __ldcg(reinterpret_cast<const float2 *>(src));
        acc[0] = fmaf(f, t.x, acc[0]); acc[1] = fmaf(f, t.y, acc[1]);
      }
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    const int64_t orow = ((int64_t)e.q_start + tok) * p.num_q_heads + hq;
    uint32_t *dst = reinterpret_cast<uint32_t *>(static_cast<T *>(p.out) + orow * D + lane * kCols);
#pragma unroll
    for (int c = 0; c < kCols; c += 2) {
      float a = acc[c] * inv, b = acc[c + 1] * inv;
      if (p.v_descale != nullptr) {
        a = dequant_out(p, kvh * D + lane * kCols + c, a, inv);
        b = dequant_out(p, kvh * D + lane * kCols + c + 1, b, inv);
      }
      dst[c / 2] = pack2<T>(a, b);
    }
    if (lane == 0 && p.lse != nullptr) p.lse[orow] = l > 0.f ? (m + log2f(l)) * kLn2 : -INFINITY;
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void *ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
  });
  return fn;
}

int encode(CUtensorMap *tm, const void *base, int32_t dtype, bool swizzle, const cuuint64_t (&dims)[3], const cuuint64_t (&strides)[2],
           const cuuint32_t (&box)[3]) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return fail(MSCO_ERR_CUDA, "chunk_attention: cuTensorMapEncodeTiled is not available");
  const cuuint32_t one[3] = {1, 1, 1};
  const CUtensorMapDataType dt = dtype == MSCO_DTYPE_I8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                 : dtype == MSCO_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUresult r = fn(tm, dt, 3, const_cast<void *>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MSCO_ERR_CUDA, "chunk_attention: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return MSCO_OK;
}

template <typename T, int D, bool KV8, int N>
int launch_sized(const MscoChunkDesc &d, const ChunkParams &p, const ChunkSeq *src, int64_t q_rows,
                 cudaStream_t stream) {
  using C = Cfg<D, KV8>;
  static_assert(C::kSmem <= 232448, "shared memory of one SM exceeded");
  const cuuint64_t h = (cuuint64_t)d.num_kv_heads, bs = (cuuint64_t)d.block_size, nb = (cuuint64_t)d.num_blocks;
  const cuuint64_t row = (cuuint64_t)D * (KV8 ? 1 : 2);  // bytes of one token of one head
  const cuuint32_t rows = (cuuint32_t)std::min(d.block_size, kTile), cols = KV8 ? (cuuint32_t)D : 64u;
  CUtensorMap tq, tk, tv;
  int rc = encode(&tq, p.q, d.q_dtype, true, {(cuuint64_t)D, (cuuint64_t)d.num_q_heads, (cuuint64_t)q_rows},
                  {(cuuint64_t)D * 2, (cuuint64_t)d.num_q_heads * D * 2},
                  {64u, (cuuint32_t)p.group, (cuuint32_t)(p.item_tokens / 2)});
  if (rc != MSCO_OK) return rc;
  for (int i = 0; i < 2; ++i) {
    const void *cache = i == 0 ? p.key_cache : p.value_cache;
    CUtensorMap *tm = i == 0 ? &tk : &tv;
    rc = d.cache_layout == 1
             ? encode(tm, cache, d.kv_dtype, !KV8, {(cuuint64_t)D, bs, nb * h}, {row, bs * row}, {cols, rows, 1u})
             : encode(tm, cache, d.kv_dtype, !KV8, {(cuuint64_t)D, h, nb * bs}, {row, h * row}, {cols, 1u, rows});
    if (rc != MSCO_OK) return rc;
  }
  ChunkSeqs<N> seqs;
  bool split = false;
  int64_t max_rows = 0;
  for (int i = 0; i < p.nseq; ++i) {
    seqs.s[i] = src[i];
    if (src[i].nsplit > 1) {
      split = true;
      max_rows = std::max<int64_t>(max_rows, (int64_t)src[i].q_len * p.num_q_heads);
    }
  }
  auto kfn = chunk_tc_kernel<T, D, KV8, N>;
  // set per call: the attribute belongs to a device
  MSCO_CUDA_CHECK(cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
  kfn<<<p.items, C::kThreads, C::kSmem, stream>>>(tq, tk, tv, p, seqs);
  MSCO_CUDA_CHECK(cudaGetLastError());
  if (split) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)std::min<int64_t>((max_rows + 7) / 8, 1024), (unsigned)p.nseq);
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    MSCO_CUDA_CHECK(cudaLaunchKernelEx(&cfg, chunk_merge_kernel<T, D, N>, p, seqs));
  }
  return MSCO_OK;
}

template <typename T, int D, bool KV8>
int launch_typed(const MscoChunkDesc &d, const ChunkParams &p, const ChunkSeq *src, int64_t q_rows,
                 cudaStream_t stream) {
  if (p.nseq <= kChunkSeqsSmall) return launch_sized<T, D, KV8, kChunkSeqsSmall>(d, p, src, q_rows, stream);
  return launch_sized<T, D, KV8, kChunkSeqsMax>(d, p, src, q_rows, stream);
}

template <typename T>
int launch_of(const MscoChunkDesc &d, const ChunkParams &p, const ChunkSeq *src, int64_t q_rows, cudaStream_t stream) {
  const bool i8 = d.kv_dtype == MSCO_DTYPE_I8;
  if (d.head_dim == 64)
    return i8 ? launch_typed<T, 64, true>(d, p, src, q_rows, stream)
              : launch_typed<T, 64, false>(d, p, src, q_rows, stream);
  return i8 ? launch_typed<T, 128, true>(d, p, src, q_rows, stream)
            : launch_typed<T, 128, false>(d, p, src, q_rows, stream);
}

}  // namespace

// Pages have to tile a KV tile (or be tiled by it) in pieces of whole 8-row swizzle groups.
bool chunk_tc_supported(const MscoChunkDesc &d) {
  const int bs = d.block_size;
  const bool bs_ok = bs % kTile == 0 || bs == 8 || bs == 16 || bs == 32 || bs == 64;
  const int group = d.num_q_heads / d.num_kv_heads;
  return (d.head_dim == 64 || d.head_dim == 128) && bs_ok && group <= kRows && d.qk_scale > 0 &&
         d.num_blocks * (int64_t)bs < (1ll << 31) && d.num_blocks * (int64_t)d.num_kv_heads < (1ll << 31);
}

int launch_chunk_tc(const MscoChunkDesc &d, const ChunkParams &p, const ChunkSeq *seqs, int64_t q_rows,
                    cudaStream_t stream) {
  return d.q_dtype == MSCO_DTYPE_F16 ? launch_of<__half>(d, p, seqs, q_rows, stream)
                                     : launch_of<__nv_bfloat16>(d, p, seqs, q_rows, stream);
}

int chunk_tc_status() {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_chunk_error, sizeof(v)) != cudaSuccess) {
    (void)cudaGetLastError();
    return MSCO_ERR_CUDA;
  }
  return v;
}

}  // namespace msco
