// The pieces' own end states of the decay attention on the tensor cores (bf16): for each piece of a cut walk,
// from zero,
//
//   S' = a^n S + (a^(n-1-j) y)^T z       chunk by chunk of n <= 128 tokens, to float32 accuracy
//
// with y's weighted rows as three bf16 terms, a fresh accumulator per chunk and the state in registers, as in the
// walk itself (decay_attn_tc.cu).  65536 tokens x 8 heads of 128: 61 us, 4.3 TB/s (77 with whole chunks and one
// accumulator, weigh - product - state one after the other).  Nothing else is formed, so the reads of y and z and shared memory set the
// pace: per chunk and 128 x 128 state 1,000 wavefronts to weigh y, 1,500 for the products' operands, 500 for the
// tiles.  y is weighed by halves of 64 tokens into two buffers and there are two accumulators, so that the
// products of one half run while the next is weighed and the state of a chunk is stepped a chunk later.
//
// Roles (640 threads): warp 0 TMA, warp 1 MMA, warps 4..19 weigh y and hold a quarter of the state's columns.
#include "decay_attn_tc.cuh"

namespace pgf {
namespace da {

namespace {

constexpr int C = TC_CHUNK;
constexpr int THREADS = 640;
constexpr uint32_t HALF = BLK / 2;     // 64 rows x 64 bf16 columns

template <int DX, int DZ>
struct Cfg {
  static constexpr int NS = DX + DZ == 256 ? 5 : DX + DZ == 192 ? 6 : 8;  // halves of y and z in flight
  static constexpr uint32_t YH = DX / 64 * HALF, ZH = DZ / 64 * HALF;
  static constexpr uint32_t TERMS = NS * (YH + ZH);            // two buffers of mid, lo (64-wide y: mid, lo, zeros)
  static constexpr uint32_t BUF = DX == 64 ? 3 * HALF : 2 * YH;
  static constexpr uint32_t TAB = TERMS + 2 * BUF;
  static constexpr uint32_t BARS = TAB + 528;
  static constexpr uint32_t BYTES = BARS + 256 + 1024;
  static_assert(BYTES <= 232448 && 128 * DZ * 4 <= TERMS, "fits an SM");
};

struct Params {
  const float* log_decay;
  const int32_t* lengths;
  float* pieces;
  int64_t stride, L, seg_len;
  float z_scale;
  int H, segs, dx, dz, last_too, gy, gz;
  Link link;
};

template <int DX, int DZ, bool REV>
__global__ void __launch_bounds__(THREADS, 1)
pieces_tc_kernel(const __grid_constant__ CUtensorMap tmY, const __grid_constant__ CUtensorMap tmZ, const Params p) {
  using G = Cfg<DX, DZ>;
  constexpr int NS = G::NS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(base);
  float* tab = reinterpret_cast<float*>(base + G::TAB);
  uint64_t* full = reinterpret_cast<uint64_t*>(base + G::BARS);
  uint64_t* empty = full + NS;
  uint64_t* weighed = empty + NS;    // [2] a buffer's terms are there
  uint64_t* freed = weighed + 2;     // [2] and have been read
  uint64_t* ufull = freed + 2;       // [2] an accumulator is complete
  uint64_t* sumready = ufull + 2;
  uint64_t* done = sumready + 1;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(done + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const int seg = int(blockIdx.x % p.segs);
  const int64_t bh = blockIdx.x / p.segs, b = bh / p.H;
  const int h = int(bh % p.H);
  const int64_t len = row_length(p.lengths, b, p.L);
  const int64_t s0 = min(len, int64_t(seg) * p.seg_len), s1 = min(len, s0 + p.seg_len);
  // the end state of the walk's last piece enters no other piece
  chain_begin(p.link);
  if (!p.last_too && seg == (REV ? 0 : p.segs - 1)) {
    chain_end();
    return;
  }
  const int chunks = int((s1 - s0 + C - 1) / C);
  auto first_token = [&](int c) { return s0 + int64_t(REV ? chunks - 1 - c : c) * C; };
  auto tokens = [&](int c) { return int(min(int64_t(C), s1 - first_token(c))); };

  const float l2 = log2_decay(p.log_decay[h]);
  if (threadIdx.x <= C) tab[threadIdx.x] = exp2f(l2 * float(threadIdx.x));
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2 * NS; ++s) mbar_init(&full[s], 1);
    for (int k = 0; k < 2; ++k) {
      mbar_init(&weighed[k], 16);
      mbar_init(&freed[k], 1);
      mbar_init(&ufull[k], 1);
    }
    mbar_init(sumready, 16);
    mbar_init(done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (DX == 64) {
    for (uint32_t i = threadIdx.x * 16; i < 2 * HALF; i += THREADS * 16)
      *reinterpret_cast<uint4*>(base + G::TERMS + (i / HALF) * G::BUF + 2 * HALF + i % HALF) = make_uint4(0, 0, 0, 0);
    fence_async();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tslot)), "r"(uint32_t(2 * DZ)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = *tslot;
  const int halves = 2 * chunks;
  auto y_at = [&](int t) { return sbase + uint32_t(t % NS) * (G::YH + G::ZH); };

  if (warp == 0) {
    const bool leader = elect_one();
    int t = 0;
    for (; t < halves; ++t) {
      const int s = t % NS;
      if (t >= NS && !warp_wait(&empty[s], (t / NS - 1) & 1)) break;
      if (leader) {
        const int t0 = int(first_token(t >> 1)) + (t & 1) * 64;
        uint8_t* dst = base + uint32_t(s) * (G::YH + G::ZH);
        mbar_expect_tx(&full[s], G::YH + G::ZH);
        for (int k = 0; k < DX / 64; ++k) tma_load_4d(dst + k * HALF, &tmY, &full[s], k * 64, h / p.gy, t0, int(b));
        for (int k = 0; k < DZ / 64; ++k) tma_load_4d(dst + G::YH + k * HALF, &tmZ, &full[s], k * 64, h / p.gz, t0, int(b));
      }
      __syncwarp();
    }
    copies_landed<NS>(full, uint32_t(t));
  } else if (warp == 1) {
    const bool leader = elect_one();
    const uint32_t id = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) | (uint32_t(DZ >> 3) << 17) |
                        (uint32_t(C >> 4) << 24);
    for (int t = 0; t < halves; ++t) {
      const int c = t >> 1;
      if (!warp_wait(&full[t % NS], (t / NS) & 1) || !warp_wait(&weighed[t & 1], c & 1)) break;
      tc_after();
      if (leader) {
        // small terms first, so that the accumulator drops the least
        const uint32_t yb = y_at(t), mid = sbase + G::TERMS + (t & 1) * G::BUF, lo = mid + G::YH;
        const uint32_t u = tmem + uint32_t(c & 1) * DZ;
        const Desc dz(yb + G::YH, HALF), dlo(lo, HALF), dmid(mid, HALF), dhi(yb, DX == 64 ? mid - yb : HALF);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) umma_bf16(u, dlo.at(kk * 2048), dz.at(kk * 2048), id, (t & 1) || kk > 0);
        if (DX == 128) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) umma_bf16(u, dmid.at(kk * 2048), dz.at(kk * 2048), id, 1);
        }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) umma_bf16(u, dhi.at(kk * 2048), dz.at(kk * 2048), id, 1);
        umma_commit(&freed[t & 1]);
        umma_commit(&empty[t % NS]);
        if (t & 1) umma_commit(&ufull[c & 1]);
      }
      __syncwarp();
    }
    products_done(done, leader);
  } else if (warp >= 4) {
    const int q = warp & 3, cg = (warp - 4) >> 2, i = q * 32 + lane, tid = int(threadIdx.x) - 128;
    constexpr int HC = DZ / 4;
    float2 s[HC / 2];
#pragma unroll
    for (int k = 0; k < HC / 2; ++k) s[k] = f2(0.f);
    bool ok = true;
    auto step = [&](int c) {           // the state over chunk c
      if (!warp_wait(&ufull[c & 1], (c >> 1) & 1)) return false;
      tc_after();
      const float2 an = f2(lds_f(sbase + G::TAB + 4 * tokens(c))), zs = f2(p.z_scale);
#pragma unroll
      for (int g = 0; g < HC / 16; ++g) {
        uint32_t u[16];
        tmem_ld16_nowait(tmem + (uint32_t(q * 32) << 16) + uint32_t(c & 1) * DZ + cg * HC + g * 16, u);
        tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 8; ++k)
          s[g * 8 + k] = fma2(an, s[g * 8 + k], mul2(zs, f2(__uint_as_float(u[2 * k]), __uint_as_float(u[2 * k + 1]))));
      }
      tc_before();
      return true;
    };
    for (int t = 0; t < halves && ok; ++t) {
      const int c = t >> 1, n = tokens(c);
      const uint32_t yb = y_at(t), mid = sbase + G::TERMS + (t & 1) * G::BUF, lo = mid + G::YH;
      if (!warp_wait(&full[t % NS], (t / NS) & 1) || (t >= 2 && !warp_wait(&freed[t & 1], (c - 1) & 1))) {
        ok = false;
        break;
      }
      constexpr int PIECES = DX / 64;
      uint32_t v[PIECES][4];
#pragma unroll
      for (int k = 0; k < PIECES; ++k) lds128(yb + uint32_t(tid + 512 * k) * 16, v[k]);
      const int j = (t & 1) * 64 + ((tid >> 3) & 63);
      const float w = j < n ? lds_f(sbase + G::TAB + 4 * (REV ? j + 1 : n - 1 - j)) : 0.f;
      const float2 w2 = f2(w), minus = f2(-1.f);
#pragma unroll
      for (int k = 0; k < PIECES; ++k) {
        const uint32_t off = uint32_t(tid + 512 * k) * 16;
        uint32_t a[3][4];
        if (j >= n) v[k][0] = v[k][1] = v[k][2] = v[k][3] = 0;  // what lies there may be anything
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          float2 x = mul2(unpack2(v[k][m]), w2);
          a[0][m] = pack2(x);
          x = fma2(unpack2(a[0][m]), minus, x);
          a[1][m] = pack2(x);
          x = fma2(unpack2(a[1][m]), minus, x);
          a[2][m] = pack2(x);
        }
        sts128(yb + off, a[0]);
        sts128(mid + off, a[1]);
        sts128(lo + off, a[2]);
      }
      if (n < (t & 1) * 64 + 64) {
        const uint32_t zero[4] = {0, 0, 0, 0};
        for (uint32_t u = uint32_t(tid); u < G::ZH / 16; u += 512)
          if ((t & 1) * 64 + int((u >> 3) & 63) >= n) sts128(yb + G::YH + u * 16, zero);
      }
      fence_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&weighed[t & 1]);
      if ((t & 1) && c > 0) ok = step(c - 1);
    }
    if (ok && chunks > 0) ok = step(chunks - 1);
    float* end = p.pieces + bh * p.stride + int64_t(seg) * p.dx * p.dz;
    if (DX == 64) {
      // rows 64..127 hold the middle terms' part; the tiles are done with
      float2* sum = reinterpret_cast<float2*>(base);
      if (i >= 64) {
#pragma unroll
        for (int k = 0; k < HC / 2; ++k) sum[(i - 64) + (cg * (HC / 2) + k) * 64] = s[k];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(sumready);
      ok = mbar_wait_warp(sumready, 0) && ok;
      if (i < 64) {
#pragma unroll
        for (int k = 0; k < HC / 2; ++k) s[k] = add2(s[k], sum[i + (cg * (HC / 2) + k) * 64]);
      }
    }
    const int r0 = q * 32, c0 = cg * HC;
    if (ok && r0 < DX)      // through the tiles' places, 64-wide: behind the sum
      state_store<HC>(s, sbase + (DX == 64 ? 64 * DZ * 4 : 0) + uint32_t(q * 4 + cg) * HC * 128,
                      end + int64_t(r0) * p.dz + c0, p.dz, p.dx - r0, p.dz - c0);
  }
  tc_before();
  __syncthreads();
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(uint32_t(2 * DZ)));
  chain_end();
}

template <int DX, int DZ, bool REV>
int launch(const Job& j, const Link& link, cudaStream_t s) {
  static int limit = 0;
  using G = Cfg<DX, DZ>;
  CUtensorMap my, mz;
  if (!make_tensor_map(&my, j.y, j.B, j.L, 64) || !make_tensor_map(&mz, j.z, j.B, j.L, 64)) {
    set_error("decay_attn: tensor map");
    return PGF_ERR_CUDA;
  }
  const Params p = {j.log_decay, j.lengths, const_cast<float*>(j.start), j.start_stride, j.L, j.seg_len, j.z_scale, j.H,
                    j.segs, j.y.d, j.z.d, j.last_too, j.H / j.y.heads, j.H / j.z.heads,
                    link};
  PGF_CUDA(ensure_dynamic_smem(pieces_tc_kernel<DX, DZ, REV>, G::BYTES, limit));
  PGF_CUDA(launch_link(link, pieces_tc_kernel<DX, DZ, REV>, unsigned(j.B * j.H * j.segs), THREADS, G::BYTES, s, my, mz, p));
  PGF_LAUNCH_CHECK();
  return PGF_OK;
}

template <bool REV>
int dispatch(const Job& j, const Link& l, cudaStream_t s) {
  if (j.y.d <= 64) return j.z.d <= 64 ? launch<64, 64, REV>(j, l, s) : launch<64, 128, REV>(j, l, s);
  return j.z.d <= 64 ? launch<128, 64, REV>(j, l, s) : launch<128, 128, REV>(j, l, s);
}

}  // namespace

int tc_pieces(const Job& j, const Link& l, cudaStream_t s) { return j.rev ? dispatch<true>(j, l, s) : dispatch<false>(j, l, s); }

}  // namespace da

int decay_pieces_tc_fault() { return take_tc_fault(); }

}  // namespace pgf
