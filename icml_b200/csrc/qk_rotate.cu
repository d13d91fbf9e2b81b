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
// grad x.  Measured (bf16): forward 16 x 2048 x 32 heads of 64 49 us, 5.5 TB/s; backward 65536 x 16 heads of 128
// 153 us, 5.3 TB/s.  Widths or tensors that 16-byte pieces do not fit take rotate_any_kernel, a warp per row (765
// and 3,050 us at these sizes).
//
// A warp takes a token with all its heads: it forms the token's cosines and sines once (the heads share them) and
// then walks the rows (token, head), a power-of-two group of lanes per row.  A lane holds two 16-byte chunks that
// are each other's rotation partners, so the rotation needs no exchange between lanes and the row sums are a few
// shuffles.  The backward's CTAs walk the tiles in a fixed order and leave one partial of grad w each, added in CTA
// order by a second kernel: no atomics, the same bits on every run.
#include "chain.cuh"
#include "f32x2.cuh"

namespace pgf {
namespace qkr {

constexpr int THREADS = 256;
constexpr int MAX_D = 256;
constexpr int RING = 96 * 1024;        // copies in flight, two CTAs an SM
constexpr int CTAS = 148 * 2;         // two CTAs an SM, every warp walking tiles of its own

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
  int D, R;
  int flat[2];             // token t of row b stands at (b L + t) times the token stride
  int tw[2], ctas[2];      // tokens of a warp's tile, CTAs
  float eps;
  float* part;             // (CTAs, D) of the queries, then of the keys, backward only
};

// (cos, sin) of 2 pi frac(position * turns / 2^64).  The integer phase is cut at the eighths of a turn: its top two
// bits, rounded, are the quadrant, and the rest is an angle within pi / 4, where the Taylor series to x^11 and x^10
// are exact to float32 (remainders 2e-11 and 1e-10).
__device__ __forceinline__ float2 turn_of(int64_t turns, int64_t pos) {
  const uint64_t phase = uint64_t(pos) * uint64_t(turns);
  const uint32_t hi = uint32_t(phase >> 32) + 0x20000000u;
  const uint32_t quadrant = hi >> 30;
  // the rest, within an eighth of a turn, to 2^-34 of a turn
  const int32_t rest = int32_t(uint32_t(phase >> 30));   // the quadrant's bits fall off
  const float x = float(rest) * 3.6572952e-10f;          // 2 pi / 2^34
  const float z = x * x;
  float s = fmaf(z, -1.0f / 39916800.0f, 1.0f / 362880.0f);
  s = fmaf(s, z, -1.0f / 5040.0f);
  s = fmaf(s, z, 1.0f / 120.0f);
  s = fmaf(s, z, -1.0f / 6.0f);
  s = fmaf(s * z, x, x);
  float c = fmaf(z, -1.0f / 3628800.0f, 1.0f / 40320.0f);
  c = fmaf(c, z, -1.0f / 720.0f);
  c = fmaf(c, z, 1.0f / 24.0f);
  c = fmaf(c, z, -0.5f);
  c = fmaf(c, z, 1.0f);
  const float p = quadrant & 1 ? s : c, q = quadrant & 1 ? c : s;
  return make_float2(quadrant == 1 || quadrant == 2 ? -p : p, quadrant >= 2 ? -q : q);
}

__device__ __forceinline__ int64_t position_of(const Args& a, int64_t t) {
  return a.positions ? a.positions[t] : a.start + t % a.L;
}

// 1 / sqrt(x) from the hardware's approximation and a Newton step (within 2 ulp); x > 0, or infinite: 0
__device__ __forceinline__ float inv_sqrt(float x) {
  const float r = rsqrtf(x);
  const float e = fmaf(-x * r, r, 1.0f);
  return x < INFINITY ? fmaf(0.5f * r, e, r) : r;
}

__device__ __forceinline__ float4 lds4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at));
  return v;
}

template <class T> struct Vec;
template <> struct Vec<float> {
  static constexpr int W = 4;
  static __device__ __forceinline__ void unpack(const uint4& u, float2* f) {
    f[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
    f[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
  }
  static __device__ __forceinline__ uint4 pack(const float2* f) {
    return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
  }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int W = 8;
  static __device__ __forceinline__ void unpack(const uint4& u, float2* f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = make_float2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xFFFF0000u));
  }
  static __device__ __forceinline__ uint4 pack(const float2* f) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[k].x, f[k].y);
      w[k] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// v: the lane's two chunks, W / 2 pairs of elements each.  HALVES: an element of the first chunk is turned with
// the same place of the second, and cs / sn hold the angles of the places in pairs; otherwise the pairs
// themselves are turned, pair i by cs / sn's place i.  BACK: by the opposite angle.
template <int W, bool HALVES, bool BACK>
__device__ __forceinline__ void rotate(float2 (&v)[W], const float2 (&cs)[W / 2], const float2 (&sn)[W / 2]) {
  if (HALVES) {
#pragma unroll
    for (int e = 0; e < W / 2; ++e) {
      const float2 p = v[e], q = v[W / 2 + e], c = cs[e], s = sn[e];
      const float2 pc = mul2(p, c), qc = mul2(q, c);
      if (BACK) {
        v[e] = fma2(q, s, pc);
        v[W / 2 + e] = make_float2(fmaf(-p.x, s.x, qc.x), fmaf(-p.y, s.y, qc.y));
      } else {
        v[e] = make_float2(fmaf(-q.x, s.x, pc.x), fmaf(-q.y, s.y, pc.y));
        v[W / 2 + e] = fma2(p, s, qc);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const float c = e & 1 ? cs[e / 2].y : cs[e / 2].x, s0 = e & 1 ? sn[e / 2].y : sn[e / 2].x, s = BACK ? -s0 : s0;
      const float2 p = v[e];
      v[e] = make_float2(fmaf(-p.y, s, p.x * c), fmaf(p.x, s, p.y * c));
    }
  }
}

// CTAs [0, ctas[0]) take the queries, the rest the keys.  A group of G lanes holds a row (slot = lane within the
// group; slots >= D / (2 W) idle along), and a warp walks tiles of `tw` tokens (a power of two): group g of the warp
// takes token g / hs and heads g % hs, g % hs + hs, ... (hs = groups / tw), so that a thread's cosines, sines and
// weights stay in registers over a token's heads and neighbouring groups read neighbouring heads.  An item is U
// rows per lane of a tile.  A lane copies the 16-byte pieces that it will read into a ring of its own in shared
// memory (cp.async), STAGES - 1 items ahead, so what is in flight (8 to 10 KB a warp) does not cost registers and
// nothing but the lane's own copies is ever waited for.
template <class T, bool HALVES, bool BWD>
__global__ void __launch_bounds__(THREADS, 2) rotate_kernel(const Args a, int G) {
  constexpr int W = Vec<T>::W;
  constexpr int U = 2;
  constexpr int WARPS = THREADS / 32;
  constexpr int PER = BWD ? 4 : 2;             // 16-byte pieces of a row
  constexpr int PIECES = PER * U;              // and of an item
  constexpr int STAGES = RING / (PIECES * THREADS * 16);
  extern __shared__ __align__(16) uint8_t smem[];
  if (BWD) chain_begin(Link{0, 0});
  const int z = int(blockIdx.x) >= a.ctas[0];
  const int cta = int(blockIdx.x) - (z ? a.ctas[0] : 0);
  const int D = a.D, np = D / 2, tw = a.tw[z], H = a.H[z];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + threadIdx.x * 16;
  // Cosines and sines of this warp's tokens (tw, W / 4 of cosines and of sines, slots) in fours: the slots of a
  // group read neighbouring words.
  const int slots = D / (2 * W);
  int64_t* st = reinterpret_cast<int64_t*>(smem + RING);             // (R / 2)
  float4* cs = reinterpret_cast<float4*>(st + (np + 1) / 2 * 2) + warp * tw * (W / 2) * slots;
  const int slot = lane & (G - 1), gi = lane / G, hs = 32 / G / tw, t = gi / hs, h0 = gi % hs;
  const bool live = slot < slots;
  const int place = live ? slot : 0;
  // places of the lane's two chunks: for HALVES the rotated part and the rest are each cut in half
  int i0 = 0, i1 = 0;
  if (live) {
    if (HALVES) {
      const int rs = a.R / (2 * W);
      if (slot < rs) { i0 = slot * W; i1 = a.R / 2 + slot * W; }
      else { i0 = a.R + (slot - rs) * W; i1 = i0 + (D - a.R) / 2; }
    } else {
      i0 = 2 * slot * W;
      i1 = i0 + W;
    }
  }
  // the lane's weights: registers in the forward; the backward, whose registers are full, reads them for each row
  // from shared memory (W / 2 fours, slots)
  float2 w[W];
#pragma unroll
  for (int e = 0; e < W; ++e) {
    const int i = e < W / 2 ? i0 + 2 * e : i1 + 2 * e - W;
    w[e] = a.w[z] ? make_float2(a.w[z][i], a.w[z][i + 1]) : f2(1.f);
  }
  float4* sw = reinterpret_cast<float4*>(st + (np + 1) / 2 * 2) + WARPS * tw * (W / 2) * slots;
  if (BWD && warp == 0 && gi == 0 && live) {
#pragma unroll
    for (int e = 0; e < W / 2; ++e) sw[e * slots + slot] = make_float4(w[2 * e].x, w[2 * e].y, w[2 * e + 1].x, w[2 * e + 1].y);
  }
  const uint32_t w_at = static_cast<uint32_t>(__cvta_generic_to_shared(sw + place));
  for (int i = threadIdx.x; i < a.R / 2; i += THREADS) st[i] = a.turns[i];
  __syncthreads();
  float2 acc[BWD ? W : 1];
#pragma unroll
  for (int e = 0; e < (BWD ? W : 1); ++e) acc[e] = f2(0.f);
  const float inv_d = 1.0f / float(D);
  const int64_t tiles = (a.tokens + tw - 1) / tw, step = int64_t(a.ctas[z]) * WARPS;
  const int turns = (H + hs * U - 1) / (hs * U), apart = i1 - i0;
  const int64_t stride = a.xs[z].head * hs;
  const T* const any = static_cast<const T*>(a.x[z]);   // what an empty copy names

  // the item that is copied next: its tile and turn, the lane's first chunk of its next row
  int64_t tile_a = int64_t(warp) * a.ctas[z] + cta;
  int k_a = 0;
  bool mine_a = false;
  const T *px = any, *pg = any;
  auto locate = [&]() {
    const int64_t tok = tile_a * tw + t;
    mine_a = live && tok < a.tokens;
    if (!mine_a) return;
    int64_t at = tok * a.xs[z].token;
    if (!a.flat[z]) at += tok / a.L * (a.xs[z].batch - a.L * a.xs[z].token);
    px = any + at + h0 * a.xs[z].head + i0;
    if (BWD) pg = static_cast<const T*>(a.g[z]) + (tok * H + h0) * D + i0;
  };
  auto copy = [&](int at, const T* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ring + uint32_t(at) * (THREADS * 16)),
                 "l"(on ? src : any), "r"(on ? 16 : 0) : "memory");
  };
  auto issue = [&](int stage) {
    if (tile_a < tiles) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool on = mine_a && h0 + (k_a * U + u) * hs < H;
        copy(stage * PIECES + u * PER, px, on);
        copy(stage * PIECES + u * PER + 1, px + apart, on);
        px += stride;
        if (BWD) {
          copy(stage * PIECES + u * PER + 2, pg, on);
          copy(stage * PIECES + u * PER + 3, pg + apart, on);
          pg += hs * D;
        }
      }
      if (++k_a == turns) {
        k_a = 0;
        tile_a += step;
        if (tile_a < tiles) locate();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto piece = [&](int stage, int k) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(ring + uint32_t(stage * PIECES + k) * (THREADS * 16)));
    return v;
  };
  int64_t tile = tile_a;
  // lane tt < tw: the position of token tt of the next tile, a tile ahead of its use
  auto position_at = [&](int64_t tl) {
    const int64_t tk = tl * tw + lane;
    return lane < tw && tl < tiles && tk < a.tokens ? position_of(a, tk) : 0;
  };
  int64_t pos_next = position_at(tile);
  if (tile < tiles) locate();
  for (int q = 0; q < STAGES - 1; ++q) issue(q);
  int stage = 0;
  for (; tile < tiles; tile += step) {
    const int64_t pos_tile = pos_next;
    pos_next = position_at(tile + step);
    __syncwarp();
    for (int tt = 0; tt < tw; ++tt) {
      const int64_t pos = __shfl_sync(0xffffffffu, pos_tile, tt);
      for (int j = lane; j < np; j += 32) {
        float2 v = make_float2(1.f, 0.f);
        if (2 * j < a.R) v = turn_of(st[j], pos);
        float* d = reinterpret_cast<float*>(cs + (tt * (W / 2) + j % W / 4) * slots + j / W) + j % 4;
        d[0] = v.x;
        d[W * slots] = v.y;             // the sines follow, W / 4 fours of each slot later
      }
    }
    __syncwarp();
    float2 c[W / 2], sn[W / 2];
#pragma unroll
    for (int e = 0; e < W / 4; ++e) {
      const float4 v = cs[(t * (W / 2) + e) * slots + place], q = cs[(t * (W / 2) + W / 4 + e) * slots + place];
      c[2 * e] = make_float2(v.x, v.y);
      c[2 * e + 1] = make_float2(v.z, v.w);
      sn[2 * e] = make_float2(q.x, q.y);
      sn[2 * e + 1] = make_float2(q.z, q.w);
    }
    const int64_t tok = tile * tw + t;
    const int rows = live && tok < a.tokens ? H - h0 : 0;   // of the lane's token from its first head on
    T* y = static_cast<T*>(a.y[z]) + (tok * H + h0) * D + i0;
    for (int k = 0; k < turns; ++k) {
      issue(stage == 0 ? STAGES - 1 : stage - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
#pragma unroll(BWD ? 1 : U)  // the backward's registers hold one row
      for (int u = 0; u < U; ++u) {
        float2 v[W], d[BWD ? W : 1];
        Vec<T>::unpack(piece(stage, u * PER), v);
        Vec<T>::unpack(piece(stage, u * PER + 1), v + W / 2);
        float2 ss2 = f2(0.f), sg2 = ss2;
        if constexpr (BWD) {
          Vec<T>::unpack(piece(stage, u * PER + 2), d);
          Vec<T>::unpack(piece(stage, u * PER + 3), d + W / 2);
          rotate<W, HALVES, true>(d, c, sn);
#pragma unroll
          for (int e = 0; e < W / 2; ++e) {
            const float4 f = lds4(w_at + uint32_t(e * slots) * 16);
            ss2 = fma2(v[2 * e], v[2 * e], fma2(v[2 * e + 1], v[2 * e + 1], ss2));
            sg2 = fma2(mul2(d[2 * e], lo2(f)), v[2 * e], fma2(mul2(d[2 * e + 1], hi2(f)), v[2 * e + 1], sg2));
          }
          float ss = hsum2(ss2), sg = hsum2(sg2);
          for (int o = G >> 1; o > 0; o >>= 1) {
            ss += __shfl_xor_sync(0xffffffffu, ss, o);
            sg += __shfl_xor_sync(0xffffffffu, sg, o);
          }
          const float rinv = inv_sqrt(fmaf(ss, inv_d, a.eps));
          const float2 r2 = f2(rinv), mean = f2(-sg * rinv * inv_d);
#pragma unroll
          for (int e = 0; e < W; ++e) {
            const float4 f = lds4(w_at + uint32_t(e / 2 * slots) * 16);
            v[e] = mul2(v[e], r2);
            acc[e] = fma2(d[e], v[e], acc[e]);
            v[e] = mul2(r2, fma2(v[e], mean, mul2(d[e], e & 1 ? hi2(f) : lo2(f))));
          }
        } else {
#pragma unroll
          for (int e = 0; e < W; ++e) ss2 = fma2(v[e], v[e], ss2);
          float ss = hsum2(ss2);
          for (int o = G >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          const float2 r2 = f2(inv_sqrt(fmaf(ss, inv_d, a.eps)));
#pragma unroll
          for (int e = 0; e < W; ++e) v[e] = mul2(mul2(v[e], r2), w[e]);
          rotate<W, HALVES, false>(v, c, sn);
        }
        if ((k * U + u) * hs < rows) {
          *reinterpret_cast<uint4*>(y) = Vec<T>::pack(v);
          *reinterpret_cast<uint4*>(y + apart) = Vec<T>::pack(v + W / 2);
        }
        y += hs * D;
      }
      stage = stage == STAGES - 1 ? 0 : stage + 1;
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if constexpr (BWD) {
    // lanes of a warp that hold the same slot, then the warps in order
#pragma unroll
    for (int e = 0; e < W; ++e)
      for (int o = G; o < 32; o <<= 1) {
        acc[e].x += __shfl_xor_sync(0xffffffffu, acc[e].x, o);
        acc[e].y += __shfl_xor_sync(0xffffffffu, acc[e].y, o);
      }
    __syncthreads();
    float* red = reinterpret_cast<float*>(smem);  // (warps, D): the ring is done with
    if (gi == 0 && live) {
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const int i = e < W / 2 ? i0 + 2 * e : i1 + 2 * e - W;
        red[warp * D + i] = acc[e].x;
        red[warp * D + i + 1] = acc[e].y;
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < D; i += THREADS) {
      float sum = 0.f;
      for (int q = 0; q < WARPS; ++q) sum += red[q * D + i];
      a.part[int64_t(blockIdx.x) * D + i] = sum;
    }
  }
}

// Any layout: a warp per row, element by element.
template <class T, bool BWD>
__global__ void __launch_bounds__(THREADS) rotate_any_kernel(const Args a, bool halves) {
  constexpr int UPL = MAX_D / 32;  // units per lane: a unit is a rotated pair or a single element behind R
  __shared__ float sacc[MAX_D];
  if (BWD) chain_begin(Link{0, 0});
  const int z = int(blockIdx.x) >= a.ctas[0];
  const int cta = int(blockIdx.x) - (z ? a.ctas[0] : 0);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = THREADS / 32;
  const int D = a.D, np = a.R / 2, units = np + (D - a.R);
  const float inv_d = 1.0f / float(D);
  float acc[BWD ? UPL : 1][2];
  if (BWD)
    for (int u = 0; u < UPL; ++u) acc[BWD ? u : 0][0] = acc[BWD ? u : 0][1] = 0.f;
  {
    const int H = a.H[z];
    const float* w = a.w[z];
    const int64_t rows = a.tokens * H;
    for (int64_t r = int64_t(cta) * warps + warp; r < rows; r += int64_t(a.ctas[z]) * warps) {
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
            const float2 c = turn_of(a.turns[p], pos);
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
      const float rinv = inv_sqrt(fmaf(ss, inv_d, a.eps));
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
          acc[BWD ? u : 0][0] = fmaf(d[u][0], x0, acc[BWD ? u : 0][0]);
          acc[BWD ? u : 0][1] = fmaf(d[u][1], x1, acc[BWD ? u : 0][1]);
          st(y, r * D + i, rinv * fmaf(-x0, mean, d[u][0] * wi));
          if (pair) st(y, r * D + j, rinv * fmaf(-x1, mean, d[u][1] * wj));
        } else if (pair) {
          const float2 c = turn_of(a.turns[p], pos);
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
        for (int u = 0; u < UPL; ++u) {
          const int p = u * 32 + lane;
          const bool pair = p < np, one = !pair && p < units;
          if (!pair && !one) continue;
          const int i = pair ? (halves ? p : 2 * p) : a.R + p - np, j = pair ? (halves ? np + p : 2 * p + 1) : i;
          sacc[i] = (k ? sacc[i] : 0.f) + acc[BWD ? u : 0][0];
          if (pair) sacc[j] = (k ? sacc[j] : 0.f) + acc[BWD ? u : 0][1];
        }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < D; c += THREADS) a.part[int64_t(blockIdx.x) * D + c] = sacc[c];
  }
}

// grad w of the queries (blockIdx.y 0) and keys: the CTAs' partials in CTA order, 32 warps' strided sums joined
// in warp order.
__global__ void __launch_bounds__(1024) weight_reduce_kernel(const float* part, int n_q, int n_k, int D, float* gq,
                                                             float* gk, int accumulate, const Link link) {
  __shared__ float red[32][33];
  chain_begin(link);
  float* out = blockIdx.y ? gk : gq;
  if (!out) return;
  const float* p = part + (blockIdx.y ? int64_t(n_q) * D : 0);
  const int n = blockIdx.y ? n_k : n_q;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < D) {
#pragma unroll 8
    for (int k = warp; k < n; k += 32) s += p[int64_t(k) * D + c];
  }
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < D) {
    float v = 0.f;
    for (int k = 0; k < 32; ++k) v += red[k][lane];
    out[c] = accumulate ? out[c] + v : v;
  }
}

static bool strides_vec(const pgf_strides& s, int W) { return s.batch % W == 0 && s.token % W == 0 && s.head % W == 0; }

template <class T, bool BWD>
static int launch(Args& a, bool halves, cudaStream_t s) {
  constexpr int W = Vec<T>::W;
  bool vec = a.D % (2 * W) == 0 && (!halves || a.R % (2 * W) == 0);
  for (int z = 0; z < 2; ++z)
    vec = vec && aligned(a.x[z], 16) && aligned(a.y[z], 16) && (!BWD || aligned(a.g[z], 16)) && strides_vec(a.xs[z], W);
  int G = 1;
  while (G < a.D / (2 * W)) G *= 2;
  int tw_most = 1;
  for (int z = 0; z < 2; ++z) {
    int64_t ctas;
    if (vec) {
      // (131072 tokens x 2 + 2 heads of 64: 62 us in tiles of 4, 164 in tiles of one)
      // more tokens a tile while the heads of one leave groups idle and there are tiles enough for the warps
      a.tw[z] = 1;
      while (2 * a.tw[z] <= 32 / G && 32 / G / a.tw[z] > a.H[z] && a.tokens / (2 * a.tw[z]) >= 148 * 16) a.tw[z] *= 2;
      if (a.tw[z] > tw_most) tw_most = a.tw[z];
      ctas = a.H[z] ? (a.tokens + a.tw[z] - 1) / a.tw[z] : 0;
    } else {
      ctas = (a.tokens * a.H[z] + THREADS / 32 - 1) / (THREADS / 32);
    }
    // as many as run at once, shared out by the heads; few tiles go to warps of different SMs
    int64_t most = int64_t(CTAS) * a.H[z] / (a.H[0] + a.H[1]);
    if (most < 1) most = 1;
    if (ctas > most) ctas = most;
    a.ctas[z] = int(ctas);
  }
  const unsigned grid = unsigned(a.ctas[0] + a.ctas[1]);
  if (!vec) {
    rotate_any_kernel<T, BWD><<<grid, THREADS, 0, s>>>(a, halves);
    PGF_LAUNCH_CHECK();
    return PGF_OK;
  }
  const size_t smem = size_t(RING) + (size_t(a.D / 2) + 1) / 2 * 16 + size_t(THREADS / 32) * tw_most * (a.D / 2) * 8 +
                      size_t(a.D) * 4;
  static int limit[2] = {0, 0};
  if (halves) {
    PGF_CUDA(ensure_dynamic_smem(rotate_kernel<T, true, BWD>, smem, limit[0]));
    rotate_kernel<T, true, BWD><<<grid, THREADS, smem, s>>>(a, G);
  } else {
    PGF_CUDA(ensure_dynamic_smem(rotate_kernel<T, false, BWD>, smem, limit[1]));
    rotate_kernel<T, false, BWD><<<grid, THREADS, smem, s>>>(a, G);
  }
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
  for (int z = 0; z < 2; ++z) a.flat[z] = Bsz == 1 || a.xs[z].batch == L * a.xs[z].token;
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
  if (dtype == PGF_DTYPE_BF16)
    return qkr::launch<__nv_bfloat16, false>(a, pairs == PGF_PAIRS_HALVES, as_stream(stream));
  return qkr::launch<float, false>(a, pairs == PGF_PAIRS_HALVES, as_stream(stream));
}

extern "C" size_t pgf_qk_norm_rotate_bwd_workspace(int64_t D) {
  return Workspace::round((size_t(qkr::CTAS) + 2) * size_t(D > 0 ? D : 1) * sizeof(float));
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
  if (a.tokens * (Hq + Hk) != 0) {
    Workspace w(ws, ws_bytes);
    a.part = w.take<float>((size_t(qkr::CTAS) + 2) * D);
    if (!ws || !a.part) {
      set_error("qk_norm_rotate_bwd: workspace of %zu bytes is too small", ws_bytes);
      return PGF_ERR_WORKSPACE;
    }
    if (dtype == PGF_DTYPE_BF16)
      PGF_TRY((qkr::launch<__nv_bfloat16, true>(a, pairs == PGF_PAIRS_HALVES, s)));
    else
      PGF_TRY((qkr::launch<float, true>(a, pairs == PGF_PAIRS_HALVES, s)));
  }
  if (!grad_wq && !grad_wk) return PGF_OK;
  const Link link = {1, 1};
  PGF_CUDA(launch_link(link, qkr::weight_reduce_kernel, dim3(unsigned(ceil_div(D, 32)), 2), 1024, 0, s, a.part, a.ctas[0],
                       a.ctas[1], int(D), grad_wq, grad_wk, accumulate, link));
  PGF_LAUNCH_CHECK();
  return PGF_OK;
}
