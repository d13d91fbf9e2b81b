// Linear attention with a decay for each head on the tensor cores (bf16): one F call of decay_attn.cuh.
//
// A CTA walks one piece of the sequence of one (batch row, head), 128 tokens a chunk.  Per chunk, with x, y, z
// the chunk's rows and S the state before it (forward direction; the walk from the end mirrors the exponents):
//
//   A  = x y^T                                tcgen05.mma, TMEM
//   P  = A * a^(i-j), j <= i                  warps 2..9, bf16, written over A in TMEM
//   D1 = x S                                  S in bf16 from shared memory
//   D2 = P z                                  P read from TMEM
//   o  = scale (D2 + a^(i+1) D1)              warps 2..9, to global memory
//   U  = (a^(n-1-j) y)^T z                    float32-exact operand: three bf16 terms hi + mid + lo
//   S' = a^n S + U                            warps 10..17, float32 in registers
//
// The state is a float32 quantity that outlives the chunk, so the weighted y enters U as three bf16 terms (24
// bits) instead of one rounding, and U is a fresh accumulator per chunk added to the state in registers: the
// tensor cores' own float32 accumulation drops low bits, and 24 short additions (small terms first) keep the
// state to float32 accuracy over any length, where one accumulator over thousands of tokens would not.  Two
// roundings to bf16 are left, P and the copy of S that D1 reads; each is of the size of the output's own.
// With 64-wide y, hi and mid lie side by side as the 128 rows of one product: lanes 0..63 of the state then
// hold hi's and lo's sum and lanes 64..127 mid's, D1 runs over both (K = 128, x used twice), and they are
// added only where the state leaves the kernel.
//
// Roles (576 threads): warp 0 TMA, warp 1 MMA, warps 2..9 scores and output, warps 10..17 the weighted y and
// the state.  Input tiles pass through a ring of slots in the order x, y, z: with four 32 KB slots x of the
// next chunk is there when a chunk begins and y and z arrive while it is worked on.  hi overwrites y in its
// slot once A is done.  Every wait is bounded.
#include "decay_attn_tc.cuh"

namespace pgf {
namespace da {

namespace {

constexpr int C = TC_CHUNK;
constexpr int THREADS = 576;
constexpr uint32_t BLK = 16384;   // 128 rows x 64 bf16 columns, 128B swizzle
constexpr uint32_t TMEM_COLS = 512;

template <int DX, int DZ>
struct Cfg {
  static constexpr uint32_t XB = DX / 64 * BLK, ZB = DZ / 64 * BLK;
  static constexpr uint32_t SLOT = XB > ZB ? XB : ZB;
  static constexpr int NS = SLOT == BLK ? 8 : 4;
  static constexpr uint32_t RING = NS * SLOT;
  static constexpr uint32_t MID = RING, LO = MID + XB, ZERO = LO + XB;  // ZERO only with 64-wide y
  static constexpr uint32_t ST = ZERO + (DX == 64 ? BLK : 0);           // S: 128 rows x DZ bf16
  static constexpr uint32_t TAB = ST + ZB;                              // 256 floats
  static constexpr uint32_t BARS = TAB + 1024;
  static constexpr uint32_t BYTES = BARS + 256 + 1024;
  // TMEM columns
  static constexpr uint32_t T_A = 0, T_D1 = 128, T_D2 = 128 + DZ, T_U = 128 + 2 * DZ;
};

struct Params {
  const float* log_decay;
  const int32_t* lengths;
  const float* start;
  int64_t start_stride;
  void* out;
  float* end;
  float scale, z_scale;
  int64_t L, seg_len;
  int H, segs, dx, dz, start_t, out_f32;
  int gx, gy, gz;              // operator heads per tensor head
};

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
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

template <int DX, int DZ, bool STATE_ONLY, bool REV>
__global__ void __launch_bounds__(THREADS, 1)
walk_tc_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmY,
               const __grid_constant__ CUtensorMap tmZ, const Params p) {
  using G = Cfg<DX, DZ>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* tab = reinterpret_cast<float*>(base + G::TAB);   // tab[127 + e] = a^e for e >= 0, 0 below
  const float* pw = tab + 127;                            // a^0 .. a^128
  uint64_t* full = reinterpret_cast<uint64_t*>(base + G::BARS);
  uint64_t* empty = full + G::NS;
  uint64_t* afull = empty + G::NS;
  uint64_t* pready = afull + 1;
  uint64_t* ofull = afull + 2;
  uint64_t* dfree = afull + 3;
  uint64_t* kready = afull + 4;
  uint64_t* ufull = afull + 5;
  uint64_t* sready = afull + 6;
  uint64_t* aread = afull + 7;    // [4]: both halves of a quarter's rows of A are read
  uint64_t* sumready = afull + 11;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(afull + 12);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int seg = int(blockIdx.x % p.segs);
  const int64_t bh = blockIdx.x / p.segs, b = bh / p.H;
  const int h = int(bh % p.H);
  const int64_t len = row_length(p.lengths, b, p.L);
  const int64_t s0 = min(len, int64_t(seg) * p.seg_len), s1 = min(len, s0 + p.seg_len);
  // (the end state of the walk's last piece enters no other piece)
  const bool idle = STATE_ONLY && seg == (REV ? 0 : p.segs - 1);
  const int chunks = idle ? 0 : int((s1 - s0 + C - 1) / C);
  const float l2 = log2_decay(p.log_decay[h]);

  for (int i = threadIdx.x; i < 256; i += THREADS) tab[i] = i >= 127 ? exp2f(l2 * float(i - 127)) : 0.f;
  if (threadIdx.x == 0) {
    for (int s = 0; s < G::NS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(afull, 1);
    mbar_init(pready, 8);
    mbar_init(ofull, 1);
    mbar_init(dfree, 8);
    mbar_init(kready, 8);
    mbar_init(ufull, 1);
    mbar_init(sready, 8);
    for (int k = 0; k < 4; ++k) mbar_init(&aread[k], 2);
    mbar_init(sumready, 8);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (!STATE_ONLY) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmX)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmY)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmZ)) : "memory");
  }
  if (DX == 64) {
    for (uint32_t i = threadIdx.x * 16; i < BLK; i += THREADS * 16)
      *reinterpret_cast<uint4*>(base + G::ZERO + i) = make_uint4(0, 0, 0, 0);
    fence_async();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tslot)), "r"(TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = *tslot;
  constexpr int PER = STATE_ONLY ? 2 : 3;      // tiles of a chunk
  auto first_token = [&](int c) { return s0 + int64_t(REV ? chunks - 1 - c : c) * C; };

  if (warp == 0) {
    // ---- TMA: x, y, z of each chunk through the ring
    const bool leader = elect_one();
    bool ok = true;
    uint32_t n = 0;
    for (int c = 0; c < chunks && ok; ++c) {
      const int t0 = int(first_token(c));
      for (int k = 3 - PER; k < 3; ++k, ++n) {
        const uint32_t s = n % G::NS, r = n / G::NS;
        if (r > 0 && !mbar_wait_warp(&empty[s], (r - 1) & 1)) { ok = false; break; }
        if (leader) {
          const CUtensorMap* m = k == 0 ? &tmX : k == 1 ? &tmY : &tmZ;
          const int hh = h / (k == 0 ? p.gx : k == 1 ? p.gy : p.gz);
          const int blocks = (k == 2 ? DZ : DX) / 64;
          mbar_expect_tx(&full[s], uint32_t(blocks) * BLK);
          for (int i = 0; i < blocks; ++i)
            tma_load_4d(base + s * G::SLOT + i * BLK, m, &full[s], i * 64, hh, t0, int(b));
        }
        __syncwarp();
      }
    }
  } else if (warp == 1) {
    // ---- MMA
    const bool leader = elect_one();
    const uint32_t id_a = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(C >> 3) << 17) | (uint32_t(C >> 4) << 24);
    const uint32_t id_d = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | (uint32_t(DZ >> 3) << 17) |
                          (uint32_t(C >> 4) << 24);
    const uint32_t id_u = id_d | (1u << 15);
    const uint32_t sbase = smem_u32(base);
    uint32_t n = 0;
    for (int c = 0; c < chunks; ++c, n += PER) {
      const uint32_t nx = n, ny = n + PER - 2, nz = n + PER - 1;
      const uint32_t xs = nx % G::NS, ys = ny % G::NS, zs = nz % G::NS;
      const uint32_t xb = sbase + xs * G::SLOT, yb = sbase + ys * G::SLOT, zb = sbase + zs * G::SLOT;
      if (!STATE_ONLY) {
        if (!mbar_wait_warp(&full[xs], (nx / G::NS) & 1)) break;
        if (!mbar_wait_warp(&full[ys], (ny / G::NS) & 1)) break;
        tc_after();
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < DX / 16; ++kk) {
            const uint32_t off = (kk >> 2) * BLK + (kk & 3) * 32;
            umma_bf16(tmem + G::T_A, sdesc(xb + off, 16, 1024), sdesc(yb + off, 16, 1024), id_a, kk > 0);
          }
          umma_commit(afull);
        }
        __syncwarp();
        if (!mbar_wait_warp(sready, c & 1)) break;
        if (c > 0 && !mbar_wait_warp(dfree, (c - 1) & 1)) break;
        tc_after();
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {  // 128 rows of S: all of x, or x twice
            const int xk = kk % (DX / 16);
            const uint32_t off = (xk >> 2) * BLK + (xk & 3) * 32;
            umma_bf16(tmem + G::T_D1, sdesc(xb + off, 16, 1024), sdesc(sbase + G::ST + kk * 2048, BLK, 1024), id_d, kk > 0);
          }
          umma_commit(&empty[xs]);
        }
        __syncwarp();
      }
      if (!mbar_wait_warp(&full[zs], (nz / G::NS) & 1)) break;
      if (!mbar_wait_warp(kready, c & 1)) break;
      tc_after();
      if (leader) {
        // small terms first, so that the accumulator drops the least
        const uint32_t lo = sbase + G::LO, mid = sbase + G::MID;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const uint64_t bd = sdesc(zb + kk * 2048, BLK, 1024);
          umma_bf16(tmem + G::T_U, sdesc(lo + kk * 2048, BLK, 1024), bd, id_u, kk > 0);
        }
        if (DX == 128) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            umma_bf16(tmem + G::T_U, sdesc(mid + kk * 2048, BLK, 1024), sdesc(zb + kk * 2048, BLK, 1024), id_u, 1);
        }
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          umma_bf16(tmem + G::T_U, sdesc(yb + kk * 2048, DX == 64 ? mid - yb : BLK, 1024), sdesc(zb + kk * 2048, BLK, 1024),
                    id_u, 1);
        umma_commit(ufull);
        umma_commit(&empty[ys]);
        if (STATE_ONLY) umma_commit(&empty[zs]);
      }
      __syncwarp();
      if (!STATE_ONLY) {
        if (!mbar_wait_warp(pready, c & 1)) break;
        tc_after();
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            umma_bf16_ta(tmem + G::T_D2, tmem + G::T_A + 8 * kk, sdesc(zb + kk * 2048, BLK, 1024), id_d, kk > 0);
          umma_commit(ofull);
          umma_commit(&empty[zs]);
        }
        __syncwarp();
      }
    }
  } else if (warp < 10) {
    if (!STATE_ONLY) {
      // ---- scores and output: row i of the chunk is TMEM lane i
      const int q = warp & 3, half = (warp - 2) >> 2, i = q * 32 + lane;
      const uint32_t row = uint32_t(q * 32) << 16;
      const int64_t seg0 = int64_t(seg) * p.seg_len;
      const int64_t pitch = int64_t(p.H) * p.dz;
      const int64_t obase = (b * p.L * p.H + h) * p.dz;
      for (int c = 0; c < chunks; ++c) {
        const int64_t t0 = first_token(c);
        const int n = int(min(int64_t(C), s1 - t0));
        if (!mbar_wait_warp(afull, c & 1)) break;
        tc_after();
        {
          uint32_t r0[32], r1[32];
          tmem_ld32_nowait(tmem + G::T_A + row + half * 64, r0);
          tmem_ld32_nowait(tmem + G::T_A + row + half * 64 + 32, r1);
          tmem_wait_ld();
          tc_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&aread[q]);
          if (!mbar_wait_warp(&aread[q], c & 1)) break;  // both halves are read before P goes over them
          tc_after();
          uint32_t pk[16];
          const int j0 = half * 64;
          const float* t = tab + (REV ? 127 - i + j0 : 127 + i - j0);
#pragma unroll
          for (int g = 0; g < 2; ++g) {
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              float v[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int j = g * 32 + 2 * k + e;
                const float w = REV ? t[j] : t[-j];
                const float a = __uint_as_float(g ? r1[2 * k + e] : r0[2 * k + e]);
                const bool in = REV ? j0 + j >= i && j0 + j < n : j0 + j <= i;
                v[e] = in ? a * w : 0.f;
              }
              pk[k] = pack_bf16(v[0], v[1]);
            }
            tmem_st16(tmem + G::T_A + row + half * 32 + g * 16, pk);
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          tc_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(pready);
        }
        if (!mbar_wait_warp(ofull, c & 1)) break;
        tc_after();
        const float w = i < n ? p.scale * pw[REV ? n - 1 - i : i + 1] : 0.f, w2 = p.scale * p.z_scale;
        const bool on = t0 + i < p.L && t0 + i < seg0 + p.seg_len;
        constexpr int HC = DZ / 2;              // columns of this warp
#pragma unroll
        for (int g = 0; g < HC / 32; ++g) {
          uint32_t d1[32], d2[32];
          const int col = half * HC + g * 32;
          tmem_ld32_nowait(tmem + G::T_D1 + row + col, d1);
          tmem_ld32_nowait(tmem + G::T_D2 + row + col, d2);
          tmem_wait_ld();
          if (g == HC / 32 - 1) {
            tc_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(dfree);
          }
          float o[32];
#pragma unroll
          for (int k = 0; k < 32; ++k)
            o[k] = i < n ? fmaf(w, __uint_as_float(d1[k]), w2 * __uint_as_float(d2[k])) : 0.f;
          if (on) {
            const int64_t at = obase + (t0 + i) * pitch + col;
            if (p.out_f32) {
              float* dst = static_cast<float*>(p.out) + at;
#pragma unroll
              for (int k = 0; k < 8; ++k)
                if (col + 4 * k < p.dz)
                  *reinterpret_cast<float4*>(dst + 4 * k) = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
            } else {
              __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.out) + at;
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (col + 8 * k < p.dz)
                  *reinterpret_cast<uint4*>(dst + 8 * k) =
                      make_uint4(pack_bf16(o[8 * k], o[8 * k + 1]), pack_bf16(o[8 * k + 2], o[8 * k + 3]),
                                 pack_bf16(o[8 * k + 4], o[8 * k + 5]), pack_bf16(o[8 * k + 6], o[8 * k + 7]));
            }
          }
        }
      }
      // whole chunks past the length are zeros
      const int64_t z0 = max(seg0, s0 + int64_t(chunks) * C), z1 = min(p.L, seg0 + p.seg_len);
      const int per = p.dz / 8;
      for (int64_t k = threadIdx.x - 64; k < (z1 - z0) * per; k += 256) {
        const int64_t at = obase + (z0 + k / per) * pitch + (k % per) * 8;
        const uint4 z = make_uint4(0, 0, 0, 0);
        if (p.out_f32) {
          uint4* dst = reinterpret_cast<uint4*>(static_cast<float*>(p.out) + at);
          dst[0] = z;
          dst[1] = z;
        } else {
          *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + at) = z;
        }
      }
    }
  } else {
    // ---- the weighted y and the state: lane i of TMEM is row i of the state (64-wide y: row i % 64)
    const int q = warp & 3, half = (warp - 10) >> 2, i = q * 32 + lane;
    const int tid = int(threadIdx.x) - 320;
    const uint32_t row = uint32_t(q * 32) << 16;
    const uint32_t sbase = smem_u32(base);
    constexpr int HC = DZ / 2;
    const int64_t n_state = int64_t(p.dx) * p.dz;
    float s[HC];
    {
      const float* st = p.start && !STATE_ONLY ? p.start + bh * p.start_stride + int64_t(seg) * n_state : nullptr;
#pragma unroll
      for (int k = 0; k < HC; ++k) {
        const int c = half * HC + k;
        s[k] = st && i < p.dx && i < DX && c < p.dz ? (p.start_t ? st[int64_t(c) * p.dx + i] : st[int64_t(i) * p.dz + c]) : 0.f;
      }
    }
    auto publish = [&]() {  // S as the bf16 operand of D1
#pragma unroll
      for (int k = 0; k < HC / 8; ++k) {
        const uint32_t w[4] = {pack_bf16(s[8 * k], s[8 * k + 1]), pack_bf16(s[8 * k + 2], s[8 * k + 3]),
                               pack_bf16(s[8 * k + 4], s[8 * k + 5]), pack_bf16(s[8 * k + 6], s[8 * k + 7])};
        const int ch = half * (HC / 8) + k;  // 16-byte chunk of the row
        sts128(sbase + G::ST + uint32_t(ch >> 3) * BLK + uint32_t(i) * 128 + (uint32_t((ch & 7) ^ (i & 7)) << 4), w);
      }
      fence_async();
      tc_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sready);
    };
    if (!STATE_ONLY && chunks > 0) publish();
    uint32_t n_tile = 0;
    bool ok = true;
    for (int c = 0; c < chunks; ++c, n_tile += PER) {
      const uint32_t ny = n_tile + PER - 2, nz = n_tile + PER - 1;
      const uint32_t ys = ny % G::NS, zs = nz % G::NS;
      const int64_t t0 = first_token(c);
      const int n = int(min(int64_t(C), s1 - t0));
      if (STATE_ONLY) {
        if (!mbar_wait_warp(&full[ys], (ny / G::NS) & 1)) { ok = false; break; }
      } else if (!mbar_wait_warp(afull, c & 1)) {
        ok = false;
        break;
      }
#pragma unroll
      for (int k = 0; k < DX / 64 * 4; ++k) {
        const uint32_t u = uint32_t(tid + 256 * k), off = u * 16;
        const int j = int(u >> 3) & 127;       // token
        uint32_t v[4], hi[4], mid[4], lo[4];
        lds128(sbase + ys * G::SLOT + off, v);
        const float w = j < n ? pw[REV ? j + 1 : n - 1 - j] : 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float a = __uint_as_float(v[e] << 16) * w, d = __uint_as_float(v[e] & 0xFFFF0000u) * w;
          if (j >= n) a = d = 0.f;              // what lies there may be anything
          hi[e] = pack_bf16(a, d);
          a -= __uint_as_float(hi[e] << 16);
          d -= __uint_as_float(hi[e] & 0xFFFF0000u);
          mid[e] = pack_bf16(a, d);
          a -= __uint_as_float(mid[e] << 16);
          d -= __uint_as_float(mid[e] & 0xFFFF0000u);
          lo[e] = pack_bf16(a, d);
        }
        sts128(sbase + ys * G::SLOT + off, hi);
        sts128(sbase + G::MID + off, mid);
        sts128(sbase + G::LO + off, lo);
      }
      if (n < C) {
        if (!mbar_wait_warp(&full[zs], (nz / G::NS) & 1)) { ok = false; break; }
        const uint32_t zero[4] = {0, 0, 0, 0};
        for (uint32_t u = uint32_t(tid); u < G::ZB / 16; u += 256)
          if ((int(u >> 3) & 127) >= n) sts128(sbase + zs * G::SLOT + u * 16, zero);
      }
      fence_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(kready);
      if (!mbar_wait_warp(ufull, c & 1)) { ok = false; break; }
      tc_after();
      const float an = pw[n];
#pragma unroll
      for (int g = 0; g < HC / 32; ++g) {
        uint32_t u[32];
        tmem_ld32(tmem + G::T_U + row + half * HC + g * 32, u);
#pragma unroll
        for (int k = 0; k < 32; ++k) s[g * 32 + k] = fmaf(an, s[g * 32 + k], p.z_scale * __uint_as_float(u[k]));
      }
      if (STATE_ONLY) tc_before();
      else if (c + 1 < chunks) publish();
    }
    // the state leaves: a piece's own (STATE_ONLY) or the whole walk's
    float* end = nullptr;
    if (STATE_ONLY) end = idle ? nullptr : const_cast<float*>(p.start) + bh * p.start_stride + int64_t(seg) * n_state;
    else if (p.end && seg == (REV ? 0 : p.segs - 1)) end = p.end + bh * n_state;
    if (end && ok) {
      if (DX == 64) {
        // rows 64..127 hold the middle terms' part
        float* sum = reinterpret_cast<float*>(base + G::ST);
        if (i >= 64) {
#pragma unroll
          for (int k = 0; k < HC; ++k) sum[(i - 64) + (half * HC + k) * 64] = s[k];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(sumready);
        if (!mbar_wait_warp(sumready, 0)) ok = false;
        if (i < 64) {
#pragma unroll
          for (int k = 0; k < HC; ++k) s[k] += sum[i + (half * HC + k) * 64];
        }
      }
      if (ok && i < DX && i < p.dx) {
#pragma unroll
        for (int k = 0; k < HC; k += 4) {
          const int c = half * HC + k;
          if (c < p.dz) *reinterpret_cast<float4*>(end + int64_t(i) * p.dz + c) = make_float4(s[k], s[k + 1], s[k + 2], s[k + 3]);
        }
      }
    }
  }
  tc_before();
  __syncthreads();
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS));
}

// (D, heads, L, B) with a box of 64 columns x 128 tokens of one head; zeros outside.
bool make_tensor_map(CUtensorMap* m, const Tensor& t, int64_t B, int64_t L) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[4] = {cuuint64_t(t.d), cuuint64_t(t.heads), cuuint64_t(L), cuuint64_t(B)};
  // the stride of a dimension of one entry is never used, but has to be a valid one
  cuuint64_t st[3] = {cuuint64_t(t.heads > 1 ? t.s.head : t.d) * 2, cuuint64_t(L > 1 ? t.s.token : t.d) * 2,
                      cuuint64_t(B > 1 ? t.s.batch : t.d) * 2};
  cuuint32_t box[4] = {64, 1, C, 1}, es[4] = {1, 1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(t.p), dims, st, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool fits(const Tensor& t, int64_t B, int64_t L) {
  auto ok = [](int64_t n, int64_t s) { return n <= 1 || (s > 0 && s % 8 == 0 && s < (int64_t(1) << 38)); };
  return t.d % 8 == 0 && t.d <= 128 && aligned(t.p, 16) && ok(t.heads, t.s.head) && ok(L, t.s.token) && ok(B, t.s.batch);
}

template <int DX, int DZ, bool STATE_ONLY, bool REV>
int launch(const Job& j, cudaStream_t s) {
  static int limit = 0;
  using G = Cfg<DX, DZ>;
  CUtensorMap mx = {}, my, mz;
  if ((!STATE_ONLY && !make_tensor_map(&mx, j.x, j.B, j.L)) || !make_tensor_map(&my, j.y, j.B, j.L) ||
      !make_tensor_map(&mz, j.z, j.B, j.L)) {
    set_error("decay_attn: tensor map");
    return PGF_ERR_CUDA;
  }
  Params p;
  p.log_decay = j.log_decay;
  p.lengths = j.lengths;
  p.start = j.start;
  p.start_stride = j.start_stride;
  p.out = j.out;
  p.end = j.end;
  p.scale = j.scale;
  p.z_scale = j.z_scale;
  p.L = j.L;
  p.seg_len = j.seg_len;
  p.H = j.H;
  p.segs = j.segs;
  p.dx = j.y.d;
  p.dz = j.z.d;
  p.start_t = j.start_t;
  p.out_f32 = j.out_f32;
  p.gx = STATE_ONLY ? 1 : j.H / j.x.heads;
  p.gy = j.H / j.y.heads;
  p.gz = j.H / j.z.heads;
  PGF_CUDA(ensure_dynamic_smem(walk_tc_kernel<DX, DZ, STATE_ONLY, REV>, G::BYTES, limit));
  walk_tc_kernel<DX, DZ, STATE_ONLY, REV><<<unsigned(j.B * j.H * j.segs), THREADS, G::BYTES, s>>>(mx, my, mz, p);
  PGF_LAUNCH_CHECK();
  return PGF_OK;
}

template <bool STATE_ONLY, bool REV>
int dispatch(const Job& j, cudaStream_t s) {
  if (j.y.d <= 64)
    return j.z.d <= 64 ? launch<64, 64, STATE_ONLY, REV>(j, s) : launch<64, 128, STATE_ONLY, REV>(j, s);
  return j.z.d <= 64 ? launch<128, 64, STATE_ONLY, REV>(j, s) : launch<128, 128, STATE_ONLY, REV>(j, s);
}

}  // namespace

bool tc_fits(const Tensor& t, int64_t B, int64_t L) { return fits(t, B, L); }
int tc_walk(const Job& j, bool state_only, cudaStream_t s) {
  if (state_only) return j.rev ? dispatch<true, true>(j, s) : dispatch<true, false>(j, s);
  return j.rev ? dispatch<false, true>(j, s) : dispatch<false, false>(j, s);
}

}  // namespace da

int decay_tc_fault() { return take_tc_fault(); }

}  // namespace pgf
