// The tensor-core engine of the decay attention: its entry points and what its kernels share.
#pragma once
#include "decay_attn.cuh"
#include "f32x2.cuh"
#include "tc_common.cuh"

namespace pgf {
namespace da {

constexpr int TC_CHUNK = 128;
constexpr uint32_t BLK = 16384;   // a tile of 128 rows x 64 bf16 columns, 128B swizzle

// Whether a bf16 tensor can be read by the engine's TMA loads: 16-byte aligned base, pitches and width, at
// most 128 wide.
bool tc_fits(const Tensor& t, int64_t B, int64_t L);
// One F call.  job.seg_len: a multiple of TC_CHUNK.
int tc_walk(const Job& job, const Link& link, cudaStream_t s);
// The pieces' own end states from zero, into job.start.
int tc_pieces(const Job& job, const Link& link, cudaStream_t s);

// grad ln a: partial sums (H, B, segs, blocks), blocks = tc_tangent_blocks(Dk, Dv).  start: the state that enters
// each piece, behind: the adjoint (scaled) of the state behind it; NULL: zeros.
struct TangentJob {
  Tensor q, k, v, g;
  const float* log_decay;
  const int32_t* lengths;
  const float *start, *behind;
  int64_t start_stride, behind_stride;
  float* part;
  float scale;
  int64_t B, L, seg_len;
  int H, segs;
};
static inline int tc_tangent_blocks(int64_t dk, int64_t dv) { return ceil_div(dk, 64) * ceil_div(dv, 64); }
int tc_tangent(const TangentJob& job, const Link& link, cudaStream_t s);

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%1, %2, %3, %4}], [%5];"
               ::"l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(src)
               : "memory");
}
__device__ __forceinline__ void tmem_ld16_nowait(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void lds128(uint32_t a, uint32_t (&v)[4]) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a));
}
__device__ __forceinline__ void sts128(uint32_t a, const uint32_t (&v)[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
// Reads of the tables, which stay as they are once the CTA has written them (shared addresses: a load through a
// generic pointer is a slower one).
__device__ __forceinline__ float lds_f(uint32_t a) {
  float v;
  asm("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds_u2(uint32_t a) {
  uint2 v;
  asm("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ float4 lds_f4(uint32_t a) {
  float4 v;
  asm("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
}
__device__ __forceinline__ uint32_t pack2(float2 v) { return pack_bf16(v.x, v.y); }

// Bounded warp-wide wait: one try before the clock is read (most waits find their phase complete).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  if (__all_sync(0xffffffffu, done)) return true;
  return mbar_wait_warp(bar, parity);
}
// Ends of the copying and the multiplying warp, after a wait that ran out too: no copy of the ring's first n tiles
// and no product is in flight when the block leaves.
template <int NS>
__device__ __forceinline__ void copies_landed(uint64_t* full, uint32_t n) {
  for (uint32_t k = n > NS ? n - NS : 0; k < n; ++k) warp_wait(&full[k % NS], (k / NS) & 1);
}
__device__ __forceinline__ void products_done(uint64_t* done, bool leader) {
  if (leader) umma_commit(done);
  __syncwarp();
  warp_wait(done, 0);
}
// A warp's 32 rows x HC columns of a float32 state, a row per lane, from and to global memory in whole lines: the
// 16-byte pieces cross from lane to lane in 32 HC floats of shared memory of the warp's own, permuted so that
// neither side meets a bank twice.  (A lane that read its own row alone cost 12 us a CTA at 128 x 128: every
// request touched 32 lines.)  ld: a multiple of 4; rows and cols (a multiple of 4) that are not there are zeros.
template <int HC>
__device__ __forceinline__ uint32_t state_at(int row, int ch) {
  constexpr int CH = HC / 4;
  static_assert(CH == 4 || CH == 8 || CH == 16, "columns of a warp");
  return uint32_t(row * CH + (ch ^ (CH == 4 ? (row >> 1) & 3 : row & (CH - 1)))) * 16;
}
template <int HC>
__device__ __forceinline__ void state_load(float2 (&s)[HC / 2], uint32_t tile, const float* g, int64_t ld, int rows, int cols) {
  constexpr int CH = HC / 4, BATCH = CH < 8 ? CH : 8;
  const int lane = threadIdx.x & 31, ch = lane % CH;
#pragma unroll
  for (int t0 = 0; t0 < CH; t0 += BATCH) {
    float4 v[BATCH];
#pragma unroll
    for (int t = 0; t < BATCH; ++t) {
      const int row = (t0 + t) * (32 / CH) + lane / CH;
      v[t] = row < rows && ch * 4 < cols ? __ldcg(reinterpret_cast<const float4*>(g + row * ld + ch * 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int t = 0; t < BATCH; ++t) {
      const uint32_t w[4] = {__float_as_uint(v[t].x), __float_as_uint(v[t].y), __float_as_uint(v[t].z), __float_as_uint(v[t].w)};
      sts128(tile + state_at<HC>((t0 + t) * (32 / CH) + lane / CH, ch), w);
    }
  }
  __syncwarp();
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    uint32_t w[4];
    lds128(tile + state_at<HC>(lane, k), w);
    s[2 * k] = make_float2(__uint_as_float(w[0]), __uint_as_float(w[1]));
    s[2 * k + 1] = make_float2(__uint_as_float(w[2]), __uint_as_float(w[3]));
  }
}
template <int HC>
__device__ __forceinline__ void state_store(const float2 (&s)[HC / 2], uint32_t tile, float* g, int64_t ld, int rows, int cols) {
  constexpr int CH = HC / 4;
  const int lane = threadIdx.x & 31, ch = lane % CH;
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    const uint32_t w[4] = {__float_as_uint(s[2 * k].x), __float_as_uint(s[2 * k].y), __float_as_uint(s[2 * k + 1].x),
                           __float_as_uint(s[2 * k + 1].y)};
    sts128(tile + state_at<HC>(lane, k), w);
  }
  __syncwarp();
#pragma unroll
  for (int t = 0; t < CH; ++t) {
    const int row = t * (32 / CH) + lane / CH;
    uint32_t w[4];
    lds128(tile + state_at<HC>(row, ch), w);
    if (row < rows && ch * 4 < cols)
      *reinterpret_cast<uint4*>(g + row * ld + ch * 4) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
// A matrix descriptor (sdesc) whose start moves by whole 16-byte units: the address field is the low 14 bits
// and shared memory ends below 2^18, so a step never carries out of it.
struct Desc {
  uint32_t lo, hi;
  __device__ __forceinline__ Desc(uint32_t saddr, uint32_t lbo) {
    const uint64_t d = sdesc(saddr, lbo, 1024);
    lo = uint32_t(d);
    hi = uint32_t(d >> 32);
  }
  __device__ __forceinline__ uint64_t at(uint32_t bytes) const { return uint64_t(hi) << 32 | (lo + (bytes >> 4)); }
};

// (D, heads, L, B) with a box of 64 columns x `rows` tokens of one head; zeros outside.
static inline bool make_tensor_map(CUtensorMap* m, const Tensor& t, int64_t B, int64_t L, int rows = TC_CHUNK) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[4] = {cuuint64_t(t.d), cuuint64_t(t.heads), cuuint64_t(L), cuuint64_t(B)};
  // the stride of a dimension of one entry is never used, but has to be a valid one
  cuuint64_t st[3] = {cuuint64_t(t.heads > 1 ? t.s.head : t.d) * 2, cuuint64_t(L > 1 ? t.s.token : t.d) * 2,
                      cuuint64_t(B > 1 ? t.s.batch : t.d) * 2};
  cuuint32_t box[4] = {64, 1, cuuint32_t(rows), 1}, es[4] = {1, 1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(t.p), dims, st, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace da
}  // namespace pgf
