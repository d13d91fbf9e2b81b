// One step of a beam search: selection over beams and vocabulary, and the reordering of the beams'
// recurrent states.
//
//   c[k, v] = score[k] + (logit[k, v] - lse[k]),   lse[k] = log sum_v exp(logit[k, v])
//
// and the K candidates of K x V that come first in the order (c descending, flat index k V + v
// ascending).  c is formed in float32 with those two roundings, and the order is total, so the
// selection is the same on every run.  A beam that has finished has one candidate: the end token at its
// own score.  A NaN (a NaN or +inf logit, a row of -inf) counts as -inf: such candidates come last, in
// index order.
//
// Bound by latency and, for large batches, by reading the logits.  One cluster of CTAs (16 for few sequences,
// else 8) takes one sequence, so that the whole step is one launch: the K rows (cut into parts where K is less
// than the cluster) go to the CTAs; pass 1 takes the maximum and sum of exponentials of each part and the
// largest logit of each group of lanes; the parts' statistics meet through distributed shared memory; pass 2
// forms c and keeps what is not below c at the K-th largest group maximum, a bound that at least K candidates
// reach: a short list, ranked by counting.  A part of 64 to 208 KB is copied once into shared memory (bulk copies,
// worked on as they arrive) and read from there in both passes (16 rows x 8 beams x 50257 in bf16: 16.6 us, 23
// with two readings); shorter ones are read twice, the second time from L1 and L2 (4 beams x 50257 in float32 over
// 16 CTAs: 9.2 us, 10.2 through shared memory), and so are longer ones.  The loops stay short on purpose: a part unrolled into
// registers ran slower (29 us at the first of these sizes), fetching instructions that run once.  The parts' best K keys meet the same way in one
// CTA, which ranks them and writes the step's outputs.  What a CTA waits for is mostly the others, at its own and the
// cluster's barriers; DRAM is at 8% at the first of these sizes.  A key is the order-preserving image of c above
// the complement of the flat index, so one 64-bit comparison is the whole order.  A list that does not
// fit (rows of equal logits) falls back to K passes of a plain maximum.
#include "tc_common.cuh"

#include <cooperative_groups.h>

#include <atomic>

namespace pgf {
namespace beam {

namespace cg = cooperative_groups;

constexpr int THREADS = 512;
constexpr int MAX_K = 32;
constexpr int LIST = 1024;
constexpr int CHUNKS = 4;          // a held part is copied in this many
constexpr int HELD_LEAST = 64 * 1024, HELD_MOST = 208 * 1024;   // bytes of a part that is held

struct Args {
  const void* logits;        // (B, K, V)
  const float* scores;       // (B, K)
  const uint8_t* finished;   // (B, K) or NULL
  float* out_scores;         // (B, K)
  int64_t* out_rows;         // (B, K): flat row b K + k of the beam that goes on
  int64_t* out_tokens;       // (B, K)
  uint8_t* out_finished;     // (B, K)
  int K, V, end, parts;
};

// A row's columns [lo, hi) for the CTA's threads: single elements up to a 16-byte boundary, 16-byte pieces, single
// elements behind them (a row of an odd vocabulary starts anywhere).
template <class T>
struct Span {
  static constexpr int W = 16 / int(sizeof(T));
  const T* row;
  int lo, hi, a0, nv;
  __device__ __forceinline__ Span(const T* row, int lo, int hi) : row(row), lo(lo), hi(hi) {
    const int mis = int((reinterpret_cast<uintptr_t>(row + lo) & 15) / sizeof(T));
    a0 = min(hi, mis ? lo + W - mis : lo);
    nv = (hi - a0) / W;
  }
  __device__ __forceinline__ const uint4* pieces() const { return reinterpret_cast<const uint4*>(row + a0); }
  // this thread's single elements in front (0) and behind (1): the column, or -1
  __device__ __forceinline__ int single(int which) const {
    const int c = which ? a0 + nv * W + int(threadIdx.x) : lo + int(threadIdx.x);
    return c < (which ? hi : a0) ? c : -1;
  }
};

__device__ __forceinline__ float candidate(float x, float lse, float score) {
  const float c = __fadd_rn(score, __fsub_rn(x, lse));
  return c == c ? c : -INFINITY;
}
__device__ __forceinline__ uint64_t key_of(float c, uint32_t flat) {
  const uint32_t u = __float_as_uint(c + 0.f);  // -0 as +0: they are equal
  return uint64_t(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (0xFFFFFFFFu - flat);
}
__device__ __forceinline__ float score_of(uint64_t key) {
  const uint32_t u = uint32_t(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}

__device__ __forceinline__ void unpack(const uint4& t, float (&f)[4]) {
  f[0] = __uint_as_float(t.x); f[1] = __uint_as_float(t.y); f[2] = __uint_as_float(t.z); f[3] = __uint_as_float(t.w);
}
__device__ __forceinline__ void unpack(const uint4& t, float (&f)[8]) {
  const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f[2 * k] = __uint_as_float(w[k] << 16);
    f[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
  }
}

// body(values, at): an array of consecutive elements from column `at`, for this thread's share of the span.
// HELD: the pieces lie in shared memory from `at_smem` on; chunk c of them is there once bars[c] has completed.
template <bool HELD, class T, class Body>
__device__ __forceinline__ bool scan(const Span<T>& sp, uint32_t at_smem, uint64_t* bars, Body body) {
  constexpr int W = Span<T>::W;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int c = sp.single(e);
    if (c >= 0) {
      const float one[1] = {ld(sp.row, c)};
      body(one, c);
    }
  }
  if (HELD) {
    const int per = (sp.nv + CHUNKS - 1) / CHUNKS;
    for (int c = 0; c < CHUNKS; ++c) {
      if (bars && !mbar_wait_warp(&bars[c], 0)) return false;
      const int end = min(sp.nv, (c + 1) * per);
#pragma unroll 2
      for (int i = c * per + threadIdx.x; i < end; i += THREADS) {
        uint4 t;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(t.x), "=r"(t.y), "=r"(t.z), "=r"(t.w)
                     : "r"(at_smem + uint32_t(i) * 16));
        float f[W];
        unpack(t, f);
        body(f, sp.a0 + i * W);
      }
    }
  } else {
#pragma unroll 4
    for (int i = threadIdx.x; i < sp.nv; i += THREADS) {
      float f[W];
      unpack(__ldg(sp.pieces() + i), f);
      body(f, sp.a0 + i * W);
    }
  }
  return true;
}

// HOLD: every CTA has one unit at most, and it fits shared memory.
template <class T, int CS, bool HOLD>
__global__ void __cluster_dims__(CS, 1, 1) __launch_bounds__(THREADS, 1) select_kernel(const Args a) {
  constexpr int UNITS = MAX_K / CS;                  // (row, part) units of one CTA at most
  constexpr int WARPS = THREADS / 32;
  __shared__ float s_max[UNITS], s_sum[UNITS];       // a unit's maximum and sum, read by the cluster
  __shared__ float s_tau[UNITS];                     // the logit that at least K of the unit reach
  __shared__ uint64_t s_best[UNITS][MAX_K];          // a unit's first K keys, read by the cluster
  __shared__ uint64_t s_list[LIST];
  __shared__ float s_wm[WARPS], s_ws[WARPS], s_g[2 * WARPS];
  __shared__ int s_n;
  __shared__ float s_lse;
  __shared__ uint64_t s_bars[CHUNKS];
  __shared__ float s_score[UNITS];
  __shared__ bool s_done[UNITS], s_fixed[UNITS];
  __shared__ uint64_t s_wk[WARPS];
  __shared__ bool s_failed;                          // a wait for the held part ran out
  cg::cluster_group cl = cg::this_cluster();
  const int rank = int(cl.block_rank());
  const int64_t b = blockIdx.x / CS;
  const int K = a.K, V = a.V, P = a.parts, U = K * P;
  const int len = (V + P - 1) / P;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr float L2E = 1.4426950408889634f;

  // s_fixed: a unit without candidates of its own scan, as its row has finished or cannot go on at all
  for (int u = rank + CS * int(threadIdx.x); u < U; u += CS * THREADS) {
    const int n = u / CS, k = u / P;
    const float score = a.scores[b * K + k];
    const bool done = a.finished && a.finished[b * K + k];
    s_score[n] = score;
    s_done[n] = done;
    s_fixed[n] = done || score == -INFINITY;
  }
  auto span = [&](int u) {
    const int lo = min(V, (u % P) * len);
    return Span<T>(static_cast<const T*>(a.logits) + (b * K + u / P) * V, lo, min(V, lo + len));
  };
  uint32_t held = 0;
  if constexpr (HOLD) {
    extern __shared__ __align__(128) uint8_t smem[];
    held = smem_u32(smem);
    if (threadIdx.x == 0) {
      s_failed = false;
      for (int c = 0; c < CHUNKS; ++c) mbar_init(&s_bars[c], 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      // every copy that begins is waited for in pass 1, so a unit that pass 1 does not read copies nothing (thread 0
      // has just formed s_fixed[0])
      if (rank < U && !s_fixed[0]) {
        const Span<T> sp = span(rank);
        const int per = (sp.nv + CHUNKS - 1) / CHUNKS;
        for (int c = 0; c < CHUNKS; ++c) {
          const int i = min(sp.nv, c * per), n = min(sp.nv, i + per) - i;
          mbar_expect_tx(&s_bars[c], uint32_t(n) * 16);
          if (n > 0)
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                         ::"r"(held + uint32_t(i) * 16), "l"(sp.pieces() + i), "r"(uint32_t(n) * 16),
                           "r"(smem_u32(&s_bars[c])) : "memory");
        }
      }
    }
  }
  __syncthreads();

  // ---- pass 1: maximum, sum of exponentials, group maxima
  for (int u = rank, n = 0; u < U; u += CS, ++n) {
    float m = -INFINITY, s = 0.f;
    if (!s_fixed[n]) {
      const bool ok = scan<HOLD>(span(u), held, s_bars, [&](const auto& f, int) {
        constexpr int n = int(sizeof(f) / sizeof(float));
        float mm = f[0];
#pragma unroll
        for (int e = 1; e < n; ++e) mm = fmaxf(mm, f[e]);
        if (mm > m) {
          s *= ex2f((m - mm) * L2E);
          m = mm;
        }
        // nothing but -inf so far: terms of zero, and a NaN enters the sum wherever it stands
        const float ref = m == -INFINITY ? 0.f : m;
        float q = 0.f;
#pragma unroll
        for (int e = 0; e < n; ++e) q += ex2f((f[e] - ref) * L2E);
        s += q;
      });
      if (HOLD && !ok) {
        // a wait ran out: the step writes no outputs, and no copy is in flight when the block leaves
        if (lane == 0) s_failed = true;
        for (int c = 0; c < CHUNKS; ++c) mbar_wait_warp(&s_bars[c], 0);
      }
    }
    // the K-th largest of the maxima of 16 warps (K <= 16) or 32 half warps: that many candidates reach it
    float gm = m;
    for (int o = 8; o > 0; o >>= 1) gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, o));
    if (K <= WARPS) gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, 16));
    const int groups = K <= WARPS ? WARPS : 2 * WARPS;
    if (K <= WARPS ? lane == 0 : (lane & 15) == 0) s_g[K <= WARPS ? warp : threadIdx.x >> 4] = gm;
    const float wm = warp_max(m);
    s = wm == -INFINITY ? s : s * ex2f((m - wm) * L2E);
    s = warp_sum(s);
    if (lane == 0) { s_wm[warp] = wm; s_ws[warp] = s; }
    __syncthreads();
    if (threadIdx.x < groups) {
      const float mine = s_g[threadIdx.x];
      int before = 0;
      for (int g = 0; g < groups; ++g) before += s_g[g] > mine || (s_g[g] == mine && g < int(threadIdx.x));
      if (before == K - 1) s_tau[n] = mine;
    }
    if (warp == 1) {  // (the first warps' threads find the group's bound)
      const float pm = lane < WARPS ? s_wm[lane] : -INFINITY, ps = lane < WARPS ? s_ws[lane] : 0.f;
      const float tm = warp_max(pm);
      const float ts = warp_sum(pm == -INFINITY ? ps : ps * ex2f((pm - tm) * L2E));
      if (lane == 0) {
        s_max[n] = tm;
        s_sum[n] = ts;
      }
    }
    __syncthreads();
  }
  cl.sync();

  // ---- pass 2: the unit's first K keys
  for (int u = rank, n = 0; u < U; u += CS, ++n) {
    const int k = u / P;
    const float score = s_score[n];
    const uint32_t flat0 = uint32_t(k) * uint32_t(V);
    if (threadIdx.x < MAX_K) s_best[n][threadIdx.x] = 0;  // below every key
    if (threadIdx.x == 0) s_n = 0;
    __syncthreads();
    if (s_fixed[n]) {
      // the end token at the score (if it has finished), then -inf from the lowest index
      const bool done = s_done[n] && score > -INFINITY;
      const int j = threadIdx.x;
      if (u % P == 0 && j < K) {
        if (done && j == 0) {
          s_best[n][0] = key_of(score, flat0 + a.end);
        } else {
          int v = done ? j - 1 : j;
          if (done && v >= a.end) ++v;
          if (v < V) s_best[n][j] = key_of(-INFINITY, flat0 + v);
        }
      }
      __syncthreads();
      continue;
    }
    if (warp == 0) {  // the row's log sum from its parts' (at most CS of them)
      const int v = k * P + lane;
      const float pm = lane < P ? cl.map_shared_rank(s_max, v % CS)[v / CS] : -INFINITY;
      const float ps = lane < P ? cl.map_shared_rank(s_sum, v % CS)[v / CS] : 0.f;
      const float m = warp_max(pm);
      const float s = warp_sum(pm == -INFINITY ? ps : ps * ex2f((pm - m) * L2E));
      if (lane == 0) s_lse = m + logf(s);
    }
    __syncthreads();
    const float lse = s_lse;
    const float bound = candidate(s_tau[n], lse, score);
    const Span<T> sp = span(u);
    auto keep = [&](const auto& f, int at) {
      constexpr int n = int(sizeof(f) / sizeof(float));
      float top = f[0];                       // c grows with the logit: the largest speaks for its piece
#pragma unroll
      for (int e = 1; e < n; ++e) top = fmaxf(top, f[e]);
      if (candidate(top, lse, score) >= bound) {
        for (int e = 0; e < n; ++e) {
          const float c = candidate(f[e], lse, score);
          if (c >= bound) {
            const int i = atomicAdd(&s_n, 1);
            if (i < LIST) s_list[i] = key_of(c, flat0 + at + e);
          }
        }
      }
    };
    scan<HOLD>(sp, held, nullptr, keep);
    __syncthreads();
    const int cnt = s_n;
    if (cnt <= LIST) {
      for (int i = threadIdx.x; i < cnt; i += THREADS) {
        const uint64_t mine = s_list[i];
        int before = 0;
        for (int j = 0; j < cnt; ++j) before += s_list[j] > mine;
        if (before < K) s_best[n][before] = mine;
      }
    } else {
      uint64_t last = ~uint64_t(0);
      for (int j = 0; j < K; ++j) {
        uint64_t top = 0;
        scan<HOLD>(sp, held, nullptr, [&](const auto& f, int at) {
#pragma unroll
          for (int e = 0; e < int(sizeof(f) / sizeof(float)); ++e) {
            const uint64_t key = key_of(candidate(f[e], lse, score), flat0 + at + e);
            if (key < last && key > top) top = key;
          }
        });
        for (int o = 16; o > 0; o >>= 1) {
          const uint64_t other = __shfl_xor_sync(0xffffffffu, top, o);
          top = other > top ? other : top;
        }
        if (lane == 0) s_wk[warp] = top;
        __syncthreads();
        for (int w = 0; w < WARPS; ++w) top = s_wk[w] > top ? s_wk[w] : top;
        last = top;
        if (threadIdx.x == 0) s_best[n][j] = top;
        __syncthreads();
      }
    }
    __syncthreads();
  }
  cl.sync();

  // ---- the sequence's K: all units' keys ranked by counting
  if (rank == 0) {
    static_assert(MAX_K * MAX_K <= LIST && CS * MAX_K <= LIST, "the units' keys fit the list");
    for (int i = threadIdx.x; i < U * K; i += THREADS) {
      const int u = i / K;
      s_list[i] = cl.map_shared_rank(&s_best[0][0], u % CS)[(u / CS) * MAX_K + i % K];
    }
    const bool failed = HOLD && threadIdx.x < CS && *cl.map_shared_rank(&s_failed, int(threadIdx.x));
    const bool skip = __syncthreads_or(failed);
    for (int i = threadIdx.x; i < U * K && !skip; i += THREADS) {
      const uint64_t mine = s_list[i];
      if (mine == 0) continue;
      int before = 0;
      for (int j = 0; j < U * K; ++j) before += s_list[j] > mine;
      if (before >= K) continue;
      const uint32_t flat = 0xFFFFFFFFu - uint32_t(mine);
      const int k = int(flat / uint32_t(V)), v = int(flat % uint32_t(V));
      const int64_t o = b * K + before;
      a.out_scores[o] = score_of(mine);
      a.out_rows[o] = b * K + k;
      a.out_tokens[o] = v;
      if (a.out_finished) a.out_finished[o] = (a.finished && a.finished[b * K + k]) || v == a.end;
    }
  }
  cl.sync();  // the others' shared memory stays until it has been read
}

template <class T, int CS>
static int select_as(Args a, int64_t Bsz, cudaStream_t s) {
  constexpr int W = Span<T>::W;
  a.parts = a.K < CS ? CS / a.K : 1;
  const int len = (a.V + a.parts - 1) / a.parts;
  const size_t bytes = size_t(len) / W * 16;
  const unsigned grid = unsigned(Bsz * CS);
  if (a.K * a.parts <= CS && bytes >= HELD_LEAST && bytes <= HELD_MOST) {
    static int limit = 0;
    PGF_CUDA(ensure_dynamic_smem(select_kernel<T, CS, true>, bytes, limit));
    select_kernel<T, CS, true><<<grid, THREADS, bytes, s>>>(a);
  } else {
    select_kernel<T, CS, false><<<grid, THREADS, 0, s>>>(a);
  }
  PGF_LAUNCH_CHECK();
  return PGF_OK;
}

// Few sequences (up to 4) take clusters of 16, more of them 8 (one sequence of 4 x 50257: 9 us against 12; 16 of
// them fill the GPU either way).  Clusters of 16 are beyond the portable size: asked for once on each device, and used
// if that can place one, also when each CTA fills an SM.
template <class T>
static bool ask_wide() {
  for (auto* k : {select_kernel<T, 16, true>, select_kernel<T, 16, false>})
    if (cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return false;
  if (cudaFuncSetAttribute(select_kernel<T, 16, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, HELD_MOST) != cudaSuccess)
    return false;
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(16);
  c.blockDim = dim3(THREADS);
  c.dynamicSmemBytes = HELD_MOST;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = 16;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  c.attrs = &at;
  c.numAttrs = 1;
  int n = 0;
  return cudaOccupancyMaxActiveClusters(&n, select_kernel<T, 16, true>, &c) == cudaSuccess && n >= 1;
}
template <class T>
static bool wide_clusters() {
  constexpr int DEVICES = 64;                              // (further ones go without)
  static std::atomic<signed char> answer[DEVICES];         // 0: not asked
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= DEVICES) {
    cudaGetLastError();
    return false;
  }
  if (answer[dev] == 0) {
    const bool ok = ask_wide<T>();
    if (!ok) cudaGetLastError();                           // a refusal is an answer, not the launch's error
    answer[dev] = ok ? 1 : -1;
  }
  return answer[dev] > 0;
}

// 16 CTAs a sequence while all of them run at once (a GPC holds one such cluster).
template <class T>
static int select(const Args& a, int64_t Bsz, cudaStream_t s) {
  return Bsz <= 4 && wide_clusters<T>() ? select_as<T, 16>(a, Bsz, s) : select_as<T, 8>(a, Bsz, s);
}

constexpr int MAX_T = 64;           // tensors of one reorder launch
constexpr int PIECE = 16384;        // bytes of a row that one CTA copies

struct Table {
  const uint8_t* src[MAX_T];
  uint8_t* dst[MAX_T];
  int64_t bytes[MAX_T];             // of one row
  int64_t first[MAX_T + 1];         // first CTA of the tensor
  int count;
};

template <class W>
__device__ __forceinline__ void copy_piece(uint8_t* d, const uint8_t* s, int64_t n) {
  const int m = int(n / int64_t(sizeof(W)));
#pragma unroll 4
  for (int i = threadIdx.x; i < m; i += 256) {
    W w = {};
    if (s) w = __ldg(reinterpret_cast<const W*>(s) + i);
    reinterpret_cast<W*>(d)[i] = w;
  }
}

// dst[i] = src[rows[i]] of every tensor; a row out of range gives zeros (the call does not
// synchronise to report it).
__global__ void __launch_bounds__(256) reorder_kernel(const __grid_constant__ Table t, const int64_t* __restrict__ rows,
                                                      int64_t n_src) {
  int z = 0;
  while (z + 1 < t.count && int64_t(blockIdx.x) >= t.first[z + 1]) ++z;
  const int64_t bytes = t.bytes[z];
  const int64_t pieces = (bytes + PIECE - 1) / PIECE, i = int64_t(blockIdx.x) - t.first[z];
  const int64_t row = i / pieces, off = (i % pieces) * PIECE;
  const int64_t n = min(int64_t(PIECE), bytes - off), from = rows[row];
  const uint8_t* s = from >= 0 && from < n_src ? t.src[z] + from * bytes + off : nullptr;
  uint8_t* d = t.dst[z] + row * bytes + off;
  const uintptr_t al = reinterpret_cast<uintptr_t>(t.src[z]) | reinterpret_cast<uintptr_t>(t.dst[z]) | uintptr_t(bytes);
  if (al % 16 == 0) copy_piece<uint4>(d, s, n);
  else if (al % 4 == 0) copy_piece<uint32_t>(d, s, n);
  else copy_piece<uint8_t>(d, s, n);
}

}  // namespace beam

int beam_fault() { return take_tc_fault(); }

}  // namespace pgf

using namespace pgf;

extern "C" int pgf_beam_select(const void* logits, const float* scores, const uint8_t* finished, float* out_scores,
                               int64_t* out_rows, int64_t* out_tokens, uint8_t* out_finished, int64_t Bsz, int64_t K,
                               int64_t V, int64_t end_id, int dtype, pgf_stream_t stream) {
  clear_error();
  PGF_CHECK_ARG(Bsz >= 0 && Bsz < (int64_t(1) << 27) && K >= 1 && K <= beam::MAX_K && V >= 1 &&
                    K * V < (int64_t(1) << 31),
                "beam_select: bad shape B=%lld K=%lld (1 to %d) V=%lld", (long long)Bsz, (long long)K, beam::MAX_K,
                (long long)V);
  PGF_CHECK_ARG(end_id >= -1 && end_id < V, "beam_select: end token %lld of %lld", (long long)end_id, (long long)V);
  PGF_CHECK_ARG(!finished || end_id >= 0, "beam_select: finished beams need an end token");
  PGF_CHECK_ARG(dtype == PGF_DTYPE_F32 || dtype == PGF_DTYPE_BF16, "beam_select: dtype %d", dtype);
  if (Bsz == 0) return PGF_OK;
  PGF_CHECK_ARG(logits && scores && out_scores && out_rows && out_tokens, "beam_select: null pointer");
  PGF_CHECK_ARG(aligned(logits, dtype == PGF_DTYPE_BF16 ? 2 : 4), "beam_select: misaligned logits");
  beam::Args a = {logits, scores, finished, out_scores, out_rows, out_tokens, out_finished,
                  int(K), int(V), int(end_id), 1};
  if (dtype == PGF_DTYPE_BF16) return beam::select<__nv_bfloat16>(a, Bsz, as_stream(stream));
  return beam::select<float>(a, Bsz, as_stream(stream));
}

extern "C" int pgf_beam_reorder(const void* const* src, void* const* dst, const int64_t* row_bytes, int count,
                                const int64_t* rows, int64_t n_rows, int64_t n_src, pgf_stream_t stream) {
  clear_error();
  PGF_CHECK_ARG(count >= 0 && n_rows >= 0 && n_src >= 0, "beam_reorder: bad shape");
  if (count == 0 || n_rows == 0) return PGF_OK;
  PGF_CHECK_ARG(src && dst && row_bytes && rows, "beam_reorder: null pointer");
  for (int i = 0; i < count; ++i) {
    PGF_CHECK_ARG(row_bytes[i] >= 0, "beam_reorder: row of %lld bytes", (long long)row_bytes[i]);
    if (row_bytes[i] == 0) continue;
    PGF_CHECK_ARG(dst[i] && (src[i] || n_src == 0), "beam_reorder: null pointer");
    // the tensors are copied side by side: no output may lie over any state, nor over another output
    const char *d0 = static_cast<const char*>(dst[i]), *d1 = d0 + n_rows * row_bytes[i];
    const char *r0 = reinterpret_cast<const char*>(rows), *r1 = r0 + n_rows * int64_t(sizeof(int64_t));
    PGF_CHECK_ARG(d1 <= r0 || r1 <= d0, "beam_reorder: tensor %d would overwrite the order", i);
    for (int j = 0; j < count; ++j) {
      if (row_bytes[j] <= 0) continue;
      const char *s0 = static_cast<const char*>(src[j]), *s1 = s0 + n_src * row_bytes[j];
      PGF_CHECK_ARG(d1 <= s0 || s1 <= d0, "beam_reorder: tensor %d would overwrite rows that tensor %d reads", i, j);
      if (j >= i) continue;
      const char *o0 = static_cast<const char*>(dst[j]), *o1 = o0 + n_rows * row_bytes[j];
      PGF_CHECK_ARG(d1 <= o0 || o1 <= d0, "beam_reorder: tensor %d would overwrite the output of tensor %d", i, j);
    }
  }
  for (int i = 0; i < count;) {
    beam::Table t;
    t.count = 0;
    int64_t ctas = 0;
    for (; i < count && t.count < beam::MAX_T; ++i) {
      if (row_bytes[i] == 0) continue;
      const int64_t need = n_rows * ((row_bytes[i] + beam::PIECE - 1) / beam::PIECE);
      PGF_CHECK_ARG(need < 0x7fffffff, "beam_reorder: tensor %d is too large", i);
      if (ctas + need >= 0x7fffffff) break;
      t.src[t.count] = static_cast<const uint8_t*>(src[i]);
      t.dst[t.count] = static_cast<uint8_t*>(dst[i]);
      t.bytes[t.count] = row_bytes[i];
      t.first[t.count++] = ctas;
      ctas += need;
    }
    if (!ctas) continue;
    t.first[t.count] = ctas;
    beam::reorder_kernel<<<unsigned(ctas), 256, 0, as_stream(stream)>>>(t, rows, n_src);
    PGF_LAUNCH_CHECK();
  }
  return PGF_OK;
}
