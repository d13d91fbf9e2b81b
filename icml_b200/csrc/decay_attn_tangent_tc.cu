// The gradient of ln a of the decay attention on the tensor cores (bf16), to float32 accuracy.
//
// With S' = dS / d ln a (S'_t = a (S'_{t-1} + S_{t-1}) along the walk), a chunk of n tokens from (S, S') gives
//
//   sum_{j <= i} (i-j) a^(i-j) (q_i k_j) (g_i v_j)  +  <S, V1>  +  <S', V2>
//   V1 = sum_i (i+1) a^(i+1) q_i g_i^T,   V2 = sum_i a^(i+1) q_i g_i^T
//   S <- a^n S + U,                       U  = sum_j a^(n-1-j) k_j v_j^T
//   S' <- a^n (S' + n S) + U',            U' = sum_j (n-1-j) a^(n-1-j) k_j v_j^T
//
// and the state behind the piece adds <its adjoint, S'>.  Terms of either sign are added over all tokens and
// all but cancel, so nothing here is rounded to 16 bits: the pair sum takes the two score products from their
// float32 accumulators, and the four weighted products take their weighted operand as three bf16 terms.
//
// Everything is bilinear in (q, k) x (v, g) columns, so the widths are cut into 64 x 64 blocks that are walked
// by CTAs of their own and added: one kernel for every width.  Two weights of the same 64 columns fill the 128
// rows of one product: U over U' (lanes 0..63 and 64..127) and V1 over V2, so S stands in lanes 0..63 next to
// V1 and S' in lanes 64..127 next to V2; only n S crosses over, through shared memory.
//
// Roles (640 threads): warp 0 TMA, warp 1 MMA, warps 2..17 work.  Per chunk a worker weighs its share of k and q
// by halves of 64 tokens (k, q, k, q: two buffers, so that the products of one run while the other is weighed),
// adds its block of the pair sum, adds its part of <S, V1> + <S', V2> and steps its 16 columns of the state.
// Shared memory is what it needs most: per chunk 1,500 wavefronts to write the weighted terms, 2,800 for the
// products to read them and 512 for the tiles.  16 x 2048 tokens x 16 heads of 64: 132 us (161 with whole chunks
// weighed before their products).
#include "decay_attn_tc.cuh"

namespace pgf {
namespace da {

namespace {

constexpr int C = TC_CHUNK;
constexpr int THREADS = 640;
constexpr int NS = 7;                                     // ring: k, v, q, g of a chunk, three of the next
constexpr uint32_t HALF = BLK / 2;                        // 64 rows
constexpr uint32_t BUF = NS * BLK;                        // k, q: three terms x two weights of 64 rows
constexpr uint32_t XCH = BUF + 6 * BLK;                   // 64 x 64 float32
constexpr uint32_t TAB = XCH + BLK;                       // 132 + 32 floats
constexpr uint32_t BARS = TAB + 656 + 64;
constexpr uint32_t BYTES = BARS + 256 + 1024;
static_assert(BYTES <= 232448, "fits an SM");
constexpr uint32_t T_A = 0, T_B = 128, T_U = 256, T_V = 320;
enum { B_AB = 0, B_U, B_V, B_K, B_Q, B_X, B_DONE, B_COUNT };      // B_U, B_V, B_K, B_Q: a phase per half

struct Params {
  const float* log_decay;
  const int32_t* lengths;
  const float *start, *behind;
  int64_t start_stride, behind_stride;
  float* part;
  float scale;
  int64_t B, L, seg_len;
  int H, segs, dk, dv, gq, gk, gv, gg;
  Link link;
};

__global__ void __launch_bounds__(THREADS, 1)
tangent_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmG, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(base);
  float* tab = reinterpret_cast<float*>(base + TAB);
  float* sums = tab + 164;
  uint64_t* full = reinterpret_cast<uint64_t*>(base + BARS);
  uint64_t* empty = full + NS;
  uint64_t* bars = empty + NS;
  uint32_t* tslot = reinterpret_cast<uint32_t*>(bars + B_COUNT);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const int nv = (p.dv + 63) / 64, blocks = (p.dk + 63) / 64 * nv;
  int64_t id = blockIdx.x;
  const int blk = int(id % blocks);
  id /= blocks;
  const int seg = int(id % p.segs);
  const int64_t bh = id / p.segs, b = bh / p.H;
  const int h = int(bh % p.H);
  const int r0 = blk / nv * 64, c0 = blk % nv * 64;       // the block's rows (q, k) and columns (v, g)
  const int64_t len = row_length(p.lengths, b, p.L);
  const int64_t s0 = min(len, int64_t(seg) * p.seg_len), s1 = min(len, s0 + p.seg_len);
  const int chunks = int((s1 - s0 + C - 1) / C);

  chain_begin(p.link);
  const float l2 = log2_decay(p.log_decay[h]);
  if (threadIdx.x <= C) tab[threadIdx.x] = exp2f(l2 * float(threadIdx.x));
  if (threadIdx.x < 32) tab[132 + threadIdx.x] = exp2f(l2 * float(31 - threadIdx.x));
  if (threadIdx.x < 16) sums[threadIdx.x] = 0.f;
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2 * NS; ++s) mbar_init(&full[s], 1);
    for (int k = 0; k < B_COUNT; ++k) mbar_init(&bars[k], k == B_K || k == B_Q ? 16 : k == B_X ? 8 : 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tslot)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = *tslot;
  auto wait_full = [&](uint32_t n) { return warp_wait(&full[n % NS], (n / NS) & 1); };
  auto wait = [&](int which, int c) { return warp_wait(&bars[which], c & 1); };
  auto arrive = [&](int which) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars[which]);
  };
  auto tile = [&](uint32_t n) { return sbase + (n % NS) * BLK; };

  if (warp == 0) {
    const bool leader = elect_one();
    uint32_t n = 0;
    bool ok = true;
    for (int c = 0; c < chunks && ok; ++c) {
      for (int k = 0; k < 4; ++k, ++n) {
        const uint32_t s = n % NS, r = n / NS;
        if (r > 0 && !warp_wait(&empty[s], (r - 1) & 1)) { ok = false; break; }
        if (leader) {
          const CUtensorMap* m = k == 0 ? &tmK : k == 1 ? &tmV : k == 2 ? &tmQ : &tmG;
          const int hh = h / (k == 0 ? p.gk : k == 1 ? p.gv : k == 2 ? p.gq : p.gg);
          mbar_expect_tx(&full[s], BLK);
          tma_load_4d(base + s * BLK, m, &full[s], k & 1 ? c0 : r0, hh, int(s0 + int64_t(c) * C), int(b));
        }
        __syncwarp();
      }
    }
    copies_landed<NS>(full, n);
  } else if (warp == 1) {
    const bool leader = elect_one();
    const uint32_t id_a = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(C >> 3) << 17) | (uint32_t(C >> 4) << 24);
    const uint32_t id_u = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) | (uint32_t(64 >> 3) << 17) |
                          (uint32_t(C >> 4) << 24);
    const Desc terms_k(sbase + BUF, HALF), terms_q(sbase + BUF + 6 * HALF, HALF);
    bool ok = true;
    for (int c = 0; c < chunks && ok; ++c) {
      const uint32_t n = uint32_t(c) * 4;
      if (!wait_full(n) || !wait_full(n + 1) || !wait_full(n + 2) || !wait_full(n + 3)) break;
      for (int half = 0; half < 2; ++half) {
        const int t = 2 * c + half;
        // (a worker weighs the next k when it is done with A, B, U and V of the chunk before)
        if (!wait(B_K, t)) { ok = false; break; }
        tc_after();
        if (leader) {
          const Desc v(tile(n + 1) + half * HALF, BLK);
          for (int m = 2; m >= 0; --m)   // small terms first
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma_bf16(tmem + T_U, terms_k.at(m * 2 * HALF + kk * 2048), v.at(kk * 2048), id_u, half || m < 2 || kk > 0);
          umma_commit(&bars[B_U]);
          if (half == 0) {
            const Desc k(tile(n), 16), v1(tile(n + 1), 16), q(tile(n + 2), 16), g(tile(n + 3), 16);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) umma_bf16(tmem + T_A, q.at(kk * 32), k.at(kk * 32), id_a, kk > 0);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) umma_bf16(tmem + T_B, g.at(kk * 32), v1.at(kk * 32), id_a, kk > 0);
            umma_commit(&bars[B_AB]);
          } else {
            umma_commit(&empty[n % NS]);
            umma_commit(&empty[(n + 1) % NS]);
          }
        }
        __syncwarp();
        if (!wait(B_Q, t)) { ok = false; break; }
        tc_after();
        if (leader) {
          const Desc g(tile(n + 3) + half * HALF, BLK);
          for (int m = 2; m >= 0; --m)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma_bf16(tmem + T_V, terms_q.at(m * 2 * HALF + kk * 2048), g.at(kk * 2048), id_u, half || m < 2 || kk > 0);
          umma_commit(&bars[B_V]);
          if (half) {
            umma_commit(&empty[(n + 2) % NS]);
            umma_commit(&empty[(n + 3) % NS]);
          }
        }
        __syncwarp();
      }
    }
    products_done(&bars[B_DONE], leader);
  } else if (warp < 18) {
    const int q = warp & 3, cg = (warp - 2) >> 2, i = q * 32 + lane, tid = int(threadIdx.x) - 64;
    const uint32_t row = uint32_t(q * 32) << 16;
    const bool tangent = i >= 64;                          // these lanes hold S'
    const int64_t n_state = int64_t(p.dk) * p.dv;
    auto pw = [&](int e) { return lds_f(sbase + TAB + 4 * e); };
    // A half of the tile's rows times two weights of their token, each as three terms; rows past the length as zeros.
    auto weigh = [&](uint32_t src, int half, int n, bool keys) {
      uint32_t v[4];
      const uint32_t off = uint32_t(tid) * 16;
      lds128(src + half * HALF + off, v);
      const int j = half * 64 + (tid >> 3);
      if (j >= n) v[0] = v[1] = v[2] = v[3] = 0;
      const int e = j >= n ? 0 : keys ? n - 1 - j : j + 1;
      const float w = pw(e), we = w * float(e);
      const uint32_t dst = sbase + BUF + (keys ? 0 : 6 * HALF) + off;
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        // first 64 rows of the product: a^e of the keys (U), e a^e of the queries (V1)
        const float2 w2 = f2((z == 0) == keys ? w : we), minus = f2(-1.f);
        uint32_t t[3][4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          float2 a = __fmul2_rn(unpack2(v[m]), w2);
          t[0][m] = pack2(a);
          a = __ffma2_rn(unpack2(t[0][m]), minus, a);
          t[1][m] = pack2(a);
          a = __ffma2_rn(unpack2(t[1][m]), minus, a);
          t[2][m] = pack2(a);
        }
#pragma unroll
        for (int m = 0; m < 3; ++m) sts128(dst + uint32_t(m * 2 + z) * HALF, t[m]);
      }
      fence_async();
      arrive(keys ? B_K : B_Q);
    };
    auto clear_rows = [&](uint32_t dst, int n) {
      const uint32_t zero[4] = {0, 0, 0, 0};
      for (uint32_t u = uint32_t(tid); u < 1024; u += 512)
        if (int(u >> 3) >= n) sts128(dst + u * 16, zero);
    };
    float s[16];
    const int sr = r0 + (i & 63);
    {
      const float* st = p.start && !tangent ? p.start + bh * p.start_stride + int64_t(seg) * n_state + int64_t(sr) * p.dv : nullptr;
#pragma unroll
      for (int k = 0; k < 16; k += 4) {
        const int cc = c0 + cg * 16 + k;
        const float4 v = st && sr < p.dk && cc < p.dv ? __ldcg(reinterpret_cast<const float4*>(st + cc)) : make_float4(0.f, 0.f, 0.f, 0.f);
        s[k] = v.x;
        s[k + 1] = v.y;
        s[k + 2] = v.z;
        s[k + 3] = v.w;
      }
    }
    float* xch = reinterpret_cast<float*>(base + XCH) + cg * 16 * 64 + (i & 63);
    float acc = 0.f, acc_end = 0.f;
    bool ok = true;
    for (int c = 0; c < chunks; ++c) {
      const uint32_t nt = uint32_t(c) * 4;
      const int n = int(min(int64_t(C), s1 - (s0 + int64_t(c) * C)));
      // the buffers are free: this warp has seen U and V of the chunk before
      if (!tangent) {
#pragma unroll
        for (int k = 0; k < 16; ++k) xch[k * 64] = s[k];
        arrive(B_X);
      }
      const float an = pw(n), cross = an * float(n);
      if (!wait_full(nt)) { ok = false; break; }
      if (n < C) {
        if (!wait_full(nt + 1) || !wait_full(nt + 3)) { ok = false; break; }
        clear_rows(tile(nt + 1), n);
        clear_rows(tile(nt + 3), n);
      }
      weigh(tile(nt), 0, n, true);
      if (!wait_full(nt + 2)) { ok = false; break; }
      weigh(tile(nt + 2), 0, n, false);
      float u[16];
      if (tangent) {                            // S of this chunk, before its place is written again
        if (!wait(B_X, c)) { ok = false; break; }
#pragma unroll
        for (int k = 0; k < 16; ++k) u[k] = cross * xch[k * 64];
      } else {
#pragma unroll
        for (int k = 0; k < 16; ++k) u[k] = 0.f;
      }
      if (!wait(B_U, 2 * c)) { ok = false; break; }
      weigh(tile(nt), 1, n, true);
      if (!wait(B_V, 2 * c)) { ok = false; break; }
      weigh(tile(nt + 2), 1, n, false);
      // the pair sum: this warp's rows, columns 32 cg .. + 31
      if (cg <= q) {
        if (!wait(B_AB, c)) { ok = false; break; }
        tc_after();
        float t = 0.f;
        const float e0 = float(i - 32 * cg);
        const float rf = cg < q ? pw(i - 32 * cg - 31) : 1.f;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          uint32_t a[16], g[16];
          tmem_ld16_nowait(tmem + T_A + row + cg * 32 + z * 16, a);
          tmem_ld16_nowait(tmem + T_B + row + cg * 32 + z * 16, g);
          tmem_wait_ld();
          if (cg < q) {
#pragma unroll
            for (int k = 0; k < 16; k += 4) {
              const float4 w = lds_f4(sbase + TAB + 528 + 4 * (z * 16 + k));
              const float wf[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int m = 0; m < 4; ++m)
                t = fmaf(__uint_as_float(a[k + m]) * __uint_as_float(g[k + m]), wf[m] * (e0 - float(z * 16 + k + m)), t);
            }
          } else {
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const int j = z * 16 + k;
              const float w = pw(lane - j) * (e0 - float(j));            // masked lanes read what lies in front
              t += j <= lane ? __uint_as_float(a[k]) * __uint_as_float(g[k]) * w : 0.f;
            }
          }
        }
        t *= rf;
        if (i < n) acc += t;
      }
      uint32_t r[16];
      if (!wait(B_U, 2 * c + 1)) { ok = false; break; }
      tc_after();
      tmem_ld16_nowait(tmem + T_U + row + cg * 16, r);
      tmem_wait_ld();
#pragma unroll
      for (int k = 0; k < 16; ++k) u[k] += __uint_as_float(r[k]);
      if (!wait(B_V, 2 * c + 1)) { ok = false; break; }
      tc_after();
      tmem_ld16_nowait(tmem + T_V + row + cg * 16, r);
      tmem_wait_ld();
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        t = fmaf(s[k], __uint_as_float(r[k]), t);
        s[k] = fmaf(an, s[k], u[k]);
      }
      acc += t;
      tc_before();
    }
    if (tangent && p.behind && sr < p.dk) {
      const float* x = p.behind + bh * p.behind_stride + int64_t(seg) * n_state + int64_t(sr) * p.dv;
#pragma unroll
      for (int k = 0; k < 16; k += 4) {
        const int cc = c0 + cg * 16 + k;
        if (cc >= p.dv) continue;
        const float4 v = __ldcg(reinterpret_cast<const float4*>(x + cc));
        acc_end = fmaf(v.x, s[k], fmaf(v.y, s[k + 1], fmaf(v.z, s[k + 2], fmaf(v.w, s[k + 3], acc_end))));
      }
    }
    const float sum = warp_sum(fmaf(acc, p.scale, acc_end));
    if (lane == 0 && ok) sums[warp - 2] = sum;
  }
  tc_before();
  __syncthreads();
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  if (threadIdx.x == 0) {
    float s = 0.f;
    for (int k = 0; k < 16; ++k) s += sums[k];
    p.part[((int64_t(h) * p.B + b) * p.segs + seg) * blocks + blk] = s;
  }
  chain_end();
}

}  // namespace

int tc_tangent(const TangentJob& j, const Link& link, cudaStream_t s) {
  static int limit = 0;
  CUtensorMap mq, mk, mv, mg;
  if (!make_tensor_map(&mq, j.q, j.B, j.L) || !make_tensor_map(&mk, j.k, j.B, j.L) || !make_tensor_map(&mv, j.v, j.B, j.L) ||
      !make_tensor_map(&mg, j.g, j.B, j.L)) {
    set_error("decay_attn: tensor map");
    return PGF_ERR_CUDA;
  }
  Params p;
  p.log_decay = j.log_decay;
  p.lengths = j.lengths;
  p.start = j.start;
  p.behind = j.behind;
  p.start_stride = j.start_stride;
  p.behind_stride = j.behind_stride;
  p.part = j.part;
  p.scale = j.scale;
  p.B = j.B;
  p.L = j.L;
  p.seg_len = j.seg_len;
  p.H = j.H;
  p.segs = j.segs;
  p.dk = j.q.d;
  p.dv = j.v.d;
  p.link = link;
  p.gq = j.H / j.q.heads;
  p.gk = j.H / j.k.heads;
  p.gv = j.H / j.v.heads;
  p.gg = j.H / j.g.heads;
  PGF_CUDA(ensure_dynamic_smem(tangent_tc_kernel, BYTES, limit));
  const int64_t grid = j.B * j.H * j.segs * tc_tangent_blocks(j.q.d, j.v.d);
  PGF_CUDA(launch_link(link, tangent_tc_kernel, unsigned(grid), THREADS, BYTES, s, mq, mk, mv, mg, p));
  PGF_LAUNCH_CHECK();
  return PGF_OK;
}

}  // namespace da

int decay_tangent_tc_fault() { return take_tc_fault(); }

}  // namespace pgf
