// Norms of queries and keys for each head with the position rotation in the same pass, forward and
// backward.
//
//   r = 1 / sqrt(mean(x^2) + eps)      over the D elements of one head
//   u = x r w                          w (D) shared by all heads, queries and keys have their own
//   y = Rot(theta) u                   pair i of the first R elements turned by theta_i
//
// theta_i = 2 pi frac(position * f_i).  The frequencies come as 64-bit fixed-point fractions of a turn
// per position, so the product's whole turns fall off the top of a 64-bit integer multiply and the
// remaining fraction is exact for every position; a float32 product position * f would be off by
// 0.06 rad at position 10^6.
//
// Backward, with gu = Rot(-theta) g and xh = x r (both recomputed from x; nothing is kept):
//   grad w = sum over tokens and heads of gu xh
//   grad x = r (gu w - xh mean(gu w xh))
//
// Bound by HBM: the forward reads and writes each element once, the backward reads x and g and writes
// grad x.  A CTA owns a tile of tokens with all their heads: it forms the tile's cosines and sines once
// in shared memory (the heads share them) and then walks the rows (token, head), a power-of-two group
// of lanes per row.  A lane holds two 16-byte chunks that are each other's rotation partners, so the
// rotation needs no exchange between lanes and the row sums are a few shuffles.  The backward's CTAs
// walk the tiles in a fixed order and leave one partial of grad w each, added in CTA order by a second
// kernel: no atomics, the same bits on every run.
#include "common.cuh"

namespace pgf {
namespace qkr {

constexpr int THREADS = 256;
constexpr int MAX_D = 256;
constexpr int MAX_TILE = 64;
constexpr int BWD_CTAS = 148 * 4;

struct Args {
  const void* x[2];        // queries, keys
  const void* g[2];        // their output gradients (contiguous), backward only
  const float* w[2];       // NULL: ones
  void* y[2];              // outputs, or input gradients (contiguous)
  pgf_strides xs[2];
  int H[2];
  const int64_t* turns;    // R / 2
  const int64_t* positions;  // (B, L) or NULL
  int64_t start;
  int64_t tokens, L;
  int D, R, tile;
  float eps;
  float* part;             // (grid, 2, D), backward only
};

__device__ __forceinline__ float2 turn_of(const Args& a, int64_t pos, int i) {
  float2 cs = make_float2(1.f, 0.f);
  if (2 * i < a.R) {
    const int64_t phase = int64_t(uint64_t(pos) * uint64_t(a.turns[i]));
    sincospif(__ll2float_rn(phase) * 1.0842021724855044e-19f /* 2^-63: half turns */, &cs.y, &cs.x);
  }
  return cs;
}

__device__ __forceinline__ int64_t position_of(const Args& a, int64_t t) {
  return a.positions ? a.positions[t] : a.start + t % a.L;
}

template <class T> struct Vec;
template <> struct Vec<float> {
  static constexpr int W = 4;
  static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y);
    f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int W = 8;
  static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f[2 * k] = __uint_as_float(w[k] << 16);
      f[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * k], f[2 * k + 1]);
      w[k] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// v: the lane's two chunks, [0, W) and [W, 2W).  HALVES: element e of the first is turned with element
// e of the second; otherwise neighbours (2e, 2e + 1) of the lane's 2W consecutive elements.
template <int W, bool HALVES>
__device__ __forceinline__ void rotate(float (&v)[2 * W], const float2* cs, float sign) {
#pragma unroll
  for (int e = 0; e < W; ++e) {
    const float2 c = cs[e];
    const int i = HALVES ? e : 2 * e, j = HALVES ? W + e : 2 * e + 1;
    const float s = sign * c.y;
    const float p = v[i], q = v[j];
    v[i] = p * c.x - q * s;
    v[j] = p * s + q * c.x;
  }
}

// One group of G lanes per row; slot = lane within the group (slots >= D / (2 W) idle along).
template <class T, bool HALVES, bool BWD>
__global__ void __launch_bounds__(THREADS) rotate_kernel(const Args a, int G) {
  constexpr int W = Vec<T>::W;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t soff[2][MAX_TILE];
  const int D = a.D, np = D / 2;
  float2* cs = reinterpret_cast<float2*>(smem);               // (tile, D / 2)
  float* sw = reinterpret_cast<float*>(cs + a.tile * np);     // (2, D) weights, then grad w partials
  const int slot = threadIdx.x & (G - 1);
  const int group = threadIdx.x / G, groups = THREADS / G;
  const bool live = slot < D / (2 * W);
  // places of the lane's two chunks: for HALVES the rotated part and the rest are each cut in half
  int i0, i1;
  if (HALVES) {
    const int rs = a.R / (2 * W);
    if (slot < rs) { i0 = slot * W; i1 = a.R / 2 + slot * W; }
    else { i0 = a.R + (slot - rs) * W; i1 = i0 + (D - a.R) / 2; }
  } else {
    i0 = 2 * slot * W;
    i1 = i0 + W;
  }
  for (int i = threadIdx.x; i < 2 * D; i += THREADS) {
    const float* w = a.w[i >= D];
    sw[i] = w ? w[i >= D ? i - D : i] : 1.f;
  }
  float acc[BWD ? 2 : 1][BWD ? 2 * W : 1];
  if (BWD) {
#pragma unroll
    for (int e = 0; e < 2 * W; ++e) acc[0][e] = acc[BWD ? 1 : 0][e] = 0.f;
  }
  const float inv_d = 1.0f / float(D);
  const int64_t tiles = (a.tokens + a.tile - 1) / a.tile;
  for (int64_t tl = blockIdx.x; tl < tiles; tl += gridDim.x) {
    const int64_t t0 = tl * a.tile;
    const int nt = int(min(int64_t(a.tile), a.tokens - t0));
    __syncthreads();
    for (int i = threadIdx.x; i < nt * np; i += THREADS) cs[i] = turn_of(a, position_of(a, t0 + i / np), i % np);
    if (threadIdx.x < nt) {
      const int64_t b = (t0 + threadIdx.x) / a.L, l = (t0 + threadIdx.x) % a.L;
      for (int z = 0; z < 2; ++z) soff[z][threadIdx.x] = b * a.xs[z].batch + l * a.xs[z].token;
    }
    __syncthreads();
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      const int H = a.H[z];
      const T* x = static_cast<const T*>(a.x[z]);
      T* y = static_cast<T*>(a.y[z]) + t0 * H * D;
      const T* g = BWD ? static_cast<const T*>(a.g[z]) + t0 * H * D : nullptr;
      const int rows = nt * H;
      // every lane of a warp takes the same number of turns, so that the shuffles see all of them
      for (int r0 = 0; r0 < rows; r0 += groups) {
        const int r = r0 + group;
        const bool on = live && r < rows;
        const int t = on ? r / H : 0, h = on ? r - t * H : 0;
        float v[2 * W], d[BWD ? 2 * W : 1];
        if (on) {
          const T* xr = x + soff[z][t] + h * a.xs[z].head;
          const uint4 u0 = __ldg(reinterpret_cast<const uint4*>(xr + i0));
          const uint4 u1 = __ldg(reinterpret_cast<const uint4*>(xr + i1));
          Vec<T>::unpack(u0, v);
          Vec<T>::unpack(u1, v + W);
          if (BWD) {
            const uint4 g0 = __ldg(reinterpret_cast<const uint4*>(g + int64_t(r) * D + i0));
            const uint4 g1 = __ldg(reinterpret_cast<const uint4*>(g + int64_t(r) * D + i1));
            Vec<T>::unpack(g0, d);
            Vec<T>::unpack(g1, d + (BWD ? W : 0));
          }
        } else {
#pragma unroll
          for (int e = 0; e < 2 * W; ++e) {
            v[e] = 0.f;
            if (BWD) d[BWD ? e : 0] = 0.f;
          }
        }
        const float2* csr = cs + t * np + (live ? slot * W : 0);
        const float* w0 = sw + z * D + (live ? i0 : 0);
        const float* w1 = sw + z * D + (live ? i1 : 0);
        float ss = 0.f, sg = 0.f;
        if constexpr (BWD) {
          rotate<W, HALVES>(d, csr, -1.f);
#pragma unroll
          for (int e = 0; e < 2 * W; ++e) {
            const float w = e < W ? w0[e] : w1[e - W];
            ss = fmaf(v[e], v[e], ss);
            sg = fmaf(d[e] * w, v[e], sg);
          }
          for (int o = G >> 1; o > 0; o >>= 1) {
            ss += __shfl_xor_sync(0xffffffffu, ss, o);
            sg += __shfl_xor_sync(0xffffffffu, sg, o);
          }
          const float rinv = 1.0f / sqrtf(fmaf(ss, inv_d, a.eps));
          const float mean = sg * rinv * inv_d;
#pragma unroll
          for (int e = 0; e < 2 * W; ++e) {
            const float w = e < W ? w0[e] : w1[e - W];
            const float xh = v[e] * rinv;
            acc[z][e] = fmaf(d[e], xh, acc[z][e]);
            v[e] = rinv * fmaf(-xh, mean, d[e] * w);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 2 * W; ++e) ss = fmaf(v[e], v[e], ss);
          for (int o = G >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          const float rinv = 1.0f / sqrtf(fmaf(ss, inv_d, a.eps));
#pragma unroll
          for (int e = 0; e < 2 * W; ++e) v[e] = v[e] * rinv * (e < W ? w0[e] : w1[e - W]);
          rotate<W, HALVES>(v, csr, 1.f);
        }
        if (on) {
          *reinterpret_cast<uint4*>(y + int64_t(r) * D + i0) = Vec<T>::pack(v);
          *reinterpret_cast<uint4*>(y + int64_t(r) * D + i1) = Vec<T>::pack(v + W);
        }
      }
    }
  }
  if constexpr (BWD) {
    // lanes of a warp that hold the same slot, then the warps in order
#pragma unroll
    for (int z = 0; z < 2; ++z)
#pragma unroll
      for (int e = 0; e < 2 * W; ++e)
        for (int o = G; o < 32; o <<= 1) acc[z][e] += __shfl_xor_sync(0xffffffffu, acc[z][e], o);
    __syncthreads();
    float* red = reinterpret_cast<float*>(smem);  // (warps, 2, D): the tables are done with
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane < G && live) {
#pragma unroll
      for (int z = 0; z < 2; ++z)
#pragma unroll
        for (int e = 0; e < 2 * W; ++e) red[(warp * 2 + z) * D + (e < W ? i0 + e : i1 + e - W)] = acc[z][e];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * D; c += THREADS) {
      float s = 0.f;
      for (int k = 0; k < THREADS / 32; ++k) s += red[k * 2 * D + c];
      a.part[int64_t(blockIdx.x) * 2 * D + c] = s;
    }
  }
}

// Any layout: a warp per row, element by element.
template <class T, bool BWD>
__global__ void __launch_bounds__(THREADS) rotate_any_kernel(const Args a, bool halves) {
  constexpr int UPL = MAX_D / 32;  // units per lane: a unit is a rotated pair or a single element behind R
  __shared__ float sacc[2][MAX_D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = THREADS / 32;
  const int D = a.D, np = a.R / 2, units = np + (D - a.R);
  const float inv_d = 1.0f / float(D);
  float acc[BWD ? 2 : 1][BWD ? UPL : 1][2];
  if (BWD)
    for (int u = 0; u < UPL; ++u)
      for (int z = 0; z < 2; ++z) acc[BWD ? z : 0][BWD ? u : 0][0] = acc[BWD ? z : 0][BWD ? u : 0][1] = 0.f;
#pragma unroll
  for (int z = 0; z < 2; ++z) {
    const int H = a.H[z];
    const float* w = a.w[z];
    const int64_t rows = a.tokens * H;
    for (int64_t r = int64_t(blockIdx.x) * warps + warp; r < rows; r += int64_t(gridDim.x) * warps) {
      const int64_t t = r / H, b = t / a.L, l = t % a.L, pos = position_of(a, t);
      const int64_t xo = b * a.xs[z].batch + l * a.xs[z].token + (r - t * H) * a.xs[z].head;
      const T* x = static_cast<const T*>(a.x[z]);
      const T* g = static_cast<const T*>(a.g[z]);
      T* y = static_cast<T*>(a.y[z]);
      float v[UPL][2], d[UPL][2];
      float ss = 0.f, sg = 0.f;
#pragma unroll
      for (int u = 0; u < UPL; ++u) {
        const int p = u * 32 + lane;
        const bool pair = p < np, one = !pair && p < units;
        const int i = pair ? (halves ? p : 2 * p) : a.R + p - np, j = pair ? (halves ? np + p : 2 * p + 1) : i;
        v[u][0] = pair || one ? ld(x, xo + i) : 0.f;
        v[u][1] = pair ? ld(x, xo + j) : 0.f;
        ss = fmaf(v[u][0], v[u][0], fmaf(v[u][1], v[u][1], ss));
        if (BWD) {
          float p0 = pair || one ? ld(g, r * D + i) : 0.f, p1 = pair ? ld(g, r * D + j) : 0.f;
          if (pair) {
            const float2 c = turn_of(a, pos, p);
            const float q0 = p0 * c.x + p1 * c.y;
            p1 = p1 * c.x - p0 * c.y;
            p0 = q0;
          }
          d[u][0] = p0;
          d[u][1] = p1;
          const float wi = w && (pair || one) ? w[i] : 1.f, wj = w && pair ? w[j] : 1.f;
          sg = fmaf(p0 * wi, v[u][0], fmaf(p1 * wj, v[u][1], sg));
        }
      }
      ss = warp_sum(ss);
      const float rinv = 1.0f / sqrtf(fmaf(ss, inv_d, a.eps));
      const float mean = BWD ? warp_sum(sg) * rinv * inv_d : 0.f;
#pragma unroll
      for (int u = 0; u < UPL; ++u) {
        const int p = u * 32 + lane;
        const bool pair = p < np, one = !pair && p < units;
        if (!pair && !one) continue;
        const int i = pair ? (halves ? p : 2 * p) : a.R + p - np, j = pair ? (halves ? np + p : 2 * p + 1) : i;
        const float wi = w ? w[i] : 1.f, wj = w && pair ? w[j] : 1.f;
        const float x0 = v[u][0] * rinv, x1 = v[u][1] * rinv;
        if (BWD) {
          acc[BWD ? z : 0][BWD ? u : 0][0] = fmaf(d[u][0], x0, acc[BWD ? z : 0][BWD ? u : 0][0]);
          acc[BWD ? z : 0][BWD ? u : 0][1] = fmaf(d[u][1], x1, acc[BWD ? z : 0][BWD ? u : 0][1]);
          st(y, r * D + i, rinv * fmaf(-x0, mean, d[u][0] * wi));
          if (pair) st(y, r * D + j, rinv * fmaf(-x1, mean, d[u][1] * wj));
        } else if (pair) {
          const float2 c = turn_of(a, pos, p);
          const float p0 = x0 * wi, p1 = x1 * wj;
          st(y, r * D + i, p0 * c.x - p1 * c.y);
          st(y, r * D + j, p0 * c.y + p1 * c.x);
        } else {
          st(y, r * D + i, x0 * wi);
        }
      }
    }
  }
  if (BWD) {
    for (int k = 0; k < warps; ++k) {  // the warps in order
      if (warp == k)
        for (int z = 0; z < 2; ++z)
          for (int u = 0; u < UPL; ++u) {
            const int p = u * 32 + lane;
            const bool pair = p < np, one = !pair && p < units;
            if (!pair && !one) continue;
            const int i = pair ? (halves ? p : 2 * p) : a.R + p - np, j = pair ? (halves ? np + p : 2 * p + 1) : i;
            sacc[z][i] = (k ? sacc[z][i] : 0.f) + acc[BWD ? z : 0][BWD ? u : 0][0];
            if (pair) sacc[z][j] = (k ? sacc[z][j] : 0.f) + acc[BWD ? z : 0][BWD ? u : 0][1];
          }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < 2 * D; c += THREADS)
      a.part[int64_t(blockIdx.x) * 2 * D + c] = sacc[c >= D][c >= D ? c - D : c];
  }
}

// grad w of queries (columns [0, D)) and keys: the CTAs' partials in CTA order, 32 warps' strided sums
// joined in warp order.
__global__ void __launch_bounds__(1024) weight_reduce_kernel(const float* part, int nparts, int D, float* gq, float* gk,
                                                             int accumulate) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < 2 * D) {
#pragma unroll 8
    for (int k = warp; k < nparts; k += 32) s += part[int64_t(k) * 2 * D + c];
  }
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < 2 * D) {
    float v = 0.f;
    for (int k = 0; k < 32; ++k) v += red[k][lane];
    float* out = c < D ? gq : gk;
    if (out) {
      float* o = out + (c < D ? c : c - D);
      *o = accumulate ? *o + v : v;
    }
  }
}

static bool strides_vec(const pgf_strides& s, int W) { return s.batch % W == 0 && s.token % W == 0 && s.head % W == 0; }

template <class T, bool BWD>
static int launch(Args a, bool halves, cudaStream_t s, int* parts) {
  constexpr int W = Vec<T>::W;
  bool vec = a.D % (2 * W) == 0 && (!halves || a.R % (2 * W) == 0);
  for (int z = 0; z < 2; ++z)
    vec = vec && aligned(a.x[z], 16) && aligned(a.y[z], 16) && (!BWD || aligned(a.g[z], 16)) && strides_vec(a.xs[z], W);
  if (!vec) {
    const int64_t rows = a.tokens * (a.H[0] > a.H[1] ? a.H[0] : a.H[1]);
    int64_t ctas = (rows + THREADS / 32 - 1) / (THREADS / 32);
    if (ctas > BWD_CTAS) ctas = BWD_CTAS;
    *parts = int(ctas);
    rotate_any_kernel<T, BWD><<<unsigned(ctas), THREADS, 0, s>>>(a, halves);
    PGF_LAUNCH_CHECK();
    return PGF_OK;
  }
  int G = 1;
  while (G < a.D / (2 * W)) G *= 2;
  // about 16K elements a tile; fewer tokens when they would leave SMs without a tile
  int64_t tile = 16384 / (int64_t(a.H[0] + a.H[1]) * a.D);
  const int64_t share = (a.tokens + BWD_CTAS - 1) / BWD_CTAS;
  if (tile > share) tile = share;
  if (tile > 8192 / a.D) tile = 8192 / a.D;
  if (tile > MAX_TILE) tile = MAX_TILE;
  if (tile < 1) tile = 1;
  a.tile = int(tile);
  int64_t ctas = (a.tokens + tile - 1) / tile;
  if (BWD && ctas > BWD_CTAS) ctas = BWD_CTAS;
  if (ctas > 0x7fffffff) ctas = 0x7fffffff;
  *parts = int(ctas);
  size_t smem = size_t(tile) * (a.D / 2) * 8 + size_t(2) * a.D * 4;
  const size_t red = size_t(THREADS / 32) * 2 * a.D * 4;
  if (BWD && smem < red) smem = red;  // at most 34 KB: within the default limit
  if (halves) rotate_kernel<T, true, BWD><<<unsigned(ctas), THREADS, smem, s>>>(a, G);
  else rotate_kernel<T, false, BWD><<<unsigned(ctas), THREADS, smem, s>>>(a, G);
  PGF_LAUNCH_CHECK();
  return PGF_OK;
}

static int check(const char* what, const Args& a, int64_t Bsz, int64_t L, int64_t Hq, int64_t Hk, int64_t D, int64_t R,
                 int pairs, int dtype, bool bwd) {
  PGF_CHECK_ARG(Bsz >= 0 && L >= 0 && Hq >= 0 && Hk >= 0 && Hq < (1 << 16) && Hk < (1 << 16) &&
                    Bsz * L <= (int64_t(1) << 40),
                "%s: bad shape B=%lld L=%lld Hq=%lld Hk=%lld", what, (long long)Bsz, (long long)L, (long long)Hq,
                (long long)Hk);
  PGF_CHECK_ARG(D >= 1 && D <= MAX_D, "%s: head width %lld (1 to %d)", what, (long long)D, MAX_D);
  PGF_CHECK_ARG(R >= 0 && R <= D && R % 2 == 0, "%s: rotated width %lld of %lld (even)", what, (long long)R, (long long)D);
  PGF_CHECK_ARG(pairs == PGF_PAIRS_HALVES || pairs == PGF_PAIRS_NEIGHBOURS, "%s: pairs %d", what, pairs);
  PGF_CHECK_ARG(dtype == PGF_DTYPE_F32 || dtype == PGF_DTYPE_BF16, "%s: dtype %d", what, dtype);
  if (Bsz * L == 0) return PGF_OK;
  for (int z = 0; z < 2; ++z)
    PGF_CHECK_ARG(a.H[z] == 0 || (a.x[z] && a.y[z] && (!bwd || a.g[z])), "%s: null pointer", what);
  PGF_CHECK_ARG(R == 0 || a.turns, "%s: null rotation table", what);
  return PGF_OK;
}

static Args make(const void* q, const pgf_strides* qs, const void* k, const pgf_strides* ks, const float* wq,
                 const float* wk, const int64_t* turns, const int64_t* positions, int64_t start, void* yq, void* yk,
                 int64_t Bsz, int64_t L, int64_t Hq, int64_t Hk, int64_t D, int64_t R, float eps) {
  Args a = {};
  a.x[0] = q; a.x[1] = k;
  a.w[0] = wq; a.w[1] = wk;
  a.y[0] = yq; a.y[1] = yk;
  const pgf_strides dq = {L * Hq * D, Hq * D, D}, dk = {L * Hk * D, Hk * D, D};
  a.xs[0] = qs ? *qs : dq;
  a.xs[1] = ks ? *ks : dk;
  a.H[0] = int(Hq); a.H[1] = int(Hk);
  a.turns = turns; a.positions = positions; a.start = start;
  a.tokens = Bsz * L; a.L = L;
  a.D = int(D); a.R = int(R); a.eps = eps;
  return a;
}

}  // namespace qkr
}  // namespace pgf

using namespace pgf;

extern "C" int pgf_qk_norm_rotate_fwd(const void* q, const pgf_strides* q_strides, const void* k,
                                      const pgf_strides* k_strides, const float* wq, const float* wk,
                                      const int64_t* turns, const int64_t* positions, int64_t start, void* q_out,
                                      void* k_out, int64_t Bsz, int64_t L, int64_t Hq, int64_t Hk, int64_t D, int64_t R,
                                      int pairs, float eps, int dtype, pgf_stream_t stream) {
  clear_error();
  qkr::Args a = qkr::make(q, q_strides, k, k_strides, wq, wk, turns, positions, start, q_out, k_out, Bsz, L, Hq, Hk, D,
                          R, eps);
  PGF_TRY(qkr::check("qk_norm_rotate_fwd", a, Bsz, L, Hq, Hk, D, R, pairs, dtype, false));
  if (a.tokens * (Hq + Hk) == 0) return PGF_OK;
  int parts;
  if (dtype == PGF_DTYPE_BF16)
    return qkr::launch<__nv_bfloat16, false>(a, pairs == PGF_PAIRS_HALVES, as_stream(stream), &parts);
  return qkr::launch<float, false>(a, pairs == PGF_PAIRS_HALVES, as_stream(stream), &parts);
}

extern "C" size_t pgf_qk_norm_rotate_bwd_workspace(int64_t D) {
  return Workspace::round(size_t(qkr::BWD_CTAS) * 2 * size_t(D > 0 ? D : 1) * sizeof(float));
}

extern "C" int pgf_qk_norm_rotate_bwd(const void* q, const pgf_strides* q_strides, const void* k,
                                      const pgf_strides* k_strides, const void* gq, const void* gk, const float* wq,
                                      const float* wk, const int64_t* turns, const int64_t* positions, int64_t start,
                                      void* grad_q, void* grad_k, float* grad_wq, float* grad_wk, int accumulate,
                                      int64_t Bsz, int64_t L, int64_t Hq, int64_t Hk, int64_t D, int64_t R, int pairs,
                                      float eps, int dtype, void* ws, size_t ws_bytes, pgf_stream_t stream) {
  clear_error();
  qkr::Args a = qkr::make(q, q_strides, k, k_strides, wq, wk, turns, positions, start, grad_q, grad_k, Bsz, L, Hq, Hk,
                          D, R, eps);
  a.g[0] = gq; a.g[1] = gk;
  PGF_TRY(qkr::check("qk_norm_rotate_bwd", a, Bsz, L, Hq, Hk, D, R, pairs, dtype, true));
  cudaStream_t s = as_stream(stream);
  int parts = 0;
  if (a.tokens * (Hq + Hk) != 0) {
    Workspace w(ws, ws_bytes);
    a.part = w.take<float>(size_t(qkr::BWD_CTAS) * 2 * D);
    if (!ws || !a.part) {
      set_error("qk_norm_rotate_bwd: workspace of %zu bytes is too small", ws_bytes);
      return PGF_ERR_WORKSPACE;
    }
    if (dtype == PGF_DTYPE_BF16)
      PGF_TRY((qkr::launch<__nv_bfloat16, true>(a, pairs == PGF_PAIRS_HALVES, s, &parts)));
    else
      PGF_TRY((qkr::launch<float, true>(a, pairs == PGF_PAIRS_HALVES, s, &parts)));
  }
  if (!grad_wq && !grad_wk) return PGF_OK;
  qkr::weight_reduce_kernel<<<unsigned(ceil_div(2 * D, 32)), 1024, 0, s>>>(a.part, parts, int(D), grad_wq, grad_wk,
                                                                           accumulate);
  PGF_LAUNCH_CHECK();
  return PGF_OK;
}
