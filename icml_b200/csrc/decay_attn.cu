// Linear attention with a decay for each head: the float32 engine (any width up to 256, any strides,
// both types), the single-token step, and the entry points.  decay_attn.cuh has the formulas.
#include "decay_attn_tc.cuh"

namespace pgf {
namespace da {

// ---------------------------------------------------------------------------------------------
// The float32 engine.  A CTA walks one piece of the sequence of one (batch row, head) for a slice of
// 64 state columns: the slice of the state stays in shared memory, a chunk's x, y (full width) and z
// (slice) are staged as float32, and three register-tiled products (4 x 4 per thread and pass) form
// the chunk: the decayed scores, the output, the state's update.  Sums are float32 FMAs throughout.
// MODE_STATE only updates (a piece's own end state from zero); MODE_TANGENT carries the state's
// derivative with respect to ln a as well and adds up <g, d out / d ln a>.  Bound by the chain of a chunk's products,
// each behind a barrier, on few CTAs: a backward of 2 x 777 tokens x 6 heads of 48 and 80 takes 94 us (139 with one
// launch a walk, 209 with loads through registers).  Rows above 128 take chunks of 32 tokens, or the staged chunk
// would not fit shared memory.
// ---------------------------------------------------------------------------------------------
constexpr int THREADS = 256;
constexpr int E = 64;               // state columns of one CTA
enum { MODE_OUT = 0, MODE_STATE = 1, MODE_TANGENT = 2 };

// Walks that run side by side in one launch: CTAs [first[k], first[k + 1]) take job k.
struct Jobs {
  Job job[3];
  int first[4];
  Link link;
};

struct TangentArgs {
  Tensor g;               // output gradients, slices like z
  const float* behind;    // (B, H, segs, x.d, z.d): adjoint of the state behind each piece, or NULL (zeros)
  int64_t behind_stride;
  float* part;            // (H, B, segs, slices) partial sums
  float scale;            // of g
};

static inline int chunk_of(int dk) { return dk > 128 ? 32 : 64; }

static size_t smem_bytes(int dx, int mode) {
  const int C = chunk_of(dx), px = dx + 4;
  size_t f = size_t(C) * px + size_t(C) * E + size_t(dx) * E + 3 * (C + 1) + 64;  // y, z, state, powers
  if (mode != MODE_STATE) f += size_t(C) * px + size_t(C) * (C + 4);              // x, scores
  if (mode == MODE_TANGENT) f += size_t(C) * E + size_t(dx) * E;                   // g, derivative
  return f * sizeof(float) + 64;
}

// rows [t0, t0 + n) x columns [c0, c0 + w) of one head as float32 with row pitch `pitch`; zeros elsewhere
// (to C rows and wpad columns, a multiple of 4), so nothing that a padded place holds is read.  float32 goes by
// asynchronous copies (16 bytes where the tensor allows, else 4), so that all of a chunk's tensors are on
// their way together; bfloat16 through registers, eight pieces at a time.  The caller waits (staged()).
template <class T>
__device__ __forceinline__ void stage(float* dst, int pitch, const Tensor& t, int64_t b, int64_t t0, int n, int h, int c0,
                                      int w, int wpad, int C) {
  const T* p = static_cast<const T*>(t.p) + b * t.s.batch + t0 * t.s.token + int64_t(h) * t.s.head + c0;
  const int w4 = wpad / 4;
  if constexpr (sizeof(T) == 4) {
    const uint32_t d0 = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
    if (t.vec) {
      for (int i = threadIdx.x; i < C * w4; i += THREADS) {
        const int r = i / w4, c = (i - r * w4) * 4;
        const int bytes = r < n && c < w ? min(16, (w - c) * 4) : 0;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d0 + uint32_t(r * pitch + c) * 4),
                     "l"(bytes ? p + int64_t(r) * t.s.token + c : static_cast<const T*>(t.p)), "r"(bytes) : "memory");
      }
    } else {
      for (int i = threadIdx.x; i < C * wpad; i += THREADS) {
        const int r = i / wpad, c = i - r * wpad;
        const bool in = r < n && c < w;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(d0 + uint32_t(r * pitch + c) * 4),
                     "l"(in ? p + int64_t(r) * t.s.token + c : static_cast<const T*>(t.p)), "r"(in ? 4 : 0) : "memory");
      }
    }
  } else {
    constexpr int U = 8;
    for (int i0 = threadIdx.x; i0 < C * w4; i0 += U * THREADS) {
      float4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * THREADS, r = i / w4, c = (i - r * w4) * 4;
        const T* q = p + int64_t(r) * t.s.token + c;
        v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < n && r < C) {
          if (c < w) v[u].x = ld(q, 0);
          if (c + 1 < w) v[u].y = ld(q, 1);
          if (c + 2 < w) v[u].z = ld(q, 2);
          if (c + 3 < w) v[u].w = ld(q, 3);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * THREADS, r = i / w4, c = (i - r * w4) * 4;
        if (r < C) *reinterpret_cast<float4*>(dst + r * pitch + c) = v[u];
      }
    }
  }
}
__device__ __forceinline__ void staged() {
  asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
}

template <class T, int C, int MODE>
__global__ void __launch_bounds__(THREADS) walk_kernel(const __grid_constant__ Jobs jobs, const TangentArgs tan) {
  extern __shared__ __align__(16) float sm[];
  const int which = int(blockIdx.x) >= jobs.first[2] ? 2 : int(blockIdx.x) >= jobs.first[1] ? 1 : 0;
  const Job& job = jobs.job[which];
  const int dx = job.x.d, dz = job.z.d, dxp = (dx + 3) & ~3, px = dxp + 4;
  const int slices = (dz + E - 1) / E;
  int64_t id = int(blockIdx.x) - jobs.first[which];
  const int sl = int(id % slices);
  id /= slices;
  const int seg = int(id % job.segs);
  id /= job.segs;
  const int h = int(id % job.H);
  const int64_t b = id / job.H;
  const int c0 = sl * E, cw = min(E, dz - c0);
  const int hx = h / (job.H / job.x.heads), hy = h / (job.H / job.y.heads), hz = h / (job.H / job.z.heads);

  float* sY = sm;                                  // (C, px)
  float* sZ = sY + C * px;                         // (C, E)
  float* sS = sZ + C * E;                          // (dxp, E)
  float* sPow = sS + dxp * E;                      // a^0 .. a^C
  float* sUpd = sPow + (C + 4);                    // weight of row j in the update
  float* sX = sUpd + (C + 4);                      // (C, px)
  float* sP = sX + (MODE != MODE_STATE ? C * px : 0);   // (C, C + 4)
  float* sG = sP + (MODE != MODE_STATE ? C * (C + 4) : 0);
  float* sD = sG + (MODE == MODE_TANGENT ? C * E : 0);  // (dxp, E): d state / d ln a

  chain_begin(jobs.link);
  const float l2 = log2_decay(job.log_decay[h]);
  for (int e = threadIdx.x; e <= C; e += THREADS) sPow[e] = exp2f(l2 * float(e));
  const int64_t len = row_length(job.lengths, b, job.L);
  const int64_t s0 = min(len, int64_t(seg) * job.seg_len), s1 = min(len, s0 + job.seg_len);

  const float* start = MODE != MODE_STATE && job.start ? job.start + (b * job.H + h) * job.start_stride + int64_t(seg) * dx * dz
                                                       : nullptr;
  for (int i = threadIdx.x; i < dxp * E; i += THREADS) {
    const int r = i / E, c = i % E;
    float v = 0.f;
    if (start && r < dx && c < cw)
      v = __ldcg(job.start_t ? start + int64_t(c0 + c) * dx + r : start + int64_t(r) * dz + c0 + c);
    sS[i] = v;
    if (MODE == MODE_TANGENT) sD[i] = 0.f;
  }
  float tsum = 0.f, tend = 0.f;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  // (the end state of the walk's last piece enters no other piece)
  const bool idle = MODE == MODE_STATE && !job.last_too && seg == (job.rev ? 0 : job.segs - 1);
  const int chunks = idle ? 0 : int((s1 - s0 + C - 1) / C);
  for (int ci = 0; ci < chunks; ++ci) {
    const int64_t t0 = s0 + int64_t(job.rev ? chunks - 1 - ci : ci) * C;
    const int n = int(min(int64_t(C), s1 - t0));
    __syncthreads();
    stage<T>(sY, px, job.y, b, t0, n, hy, 0, dx, dxp, C);
    stage<T>(sZ, E, job.z, b, t0, n, hz, c0, cw, E, C);
    if (MODE != MODE_STATE) stage<T>(sX, px, job.x, b, t0, n, hx, 0, dx, dxp, C);
    if (MODE == MODE_TANGENT) stage<T>(sG, E, tan.g, b, t0, n, h / (job.H / tan.g.heads), c0, cw, E, C);
    if (threadIdx.x < C) {
      const int j = threadIdx.x;
      sUpd[j] = j < n ? sPow[job.rev ? j + 1 : n - 1 - j] * job.z_scale : 0.f;
    }
    staged();
    __syncthreads();
    if (MODE != MODE_STATE) {
      // scores of the pairs inside the chunk: rows i = ty + 16 r, columns j = tx + 16 c
      constexpr int RT = C / 16;
      float acc[RT][RT];
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < RT; ++c) acc[r][c] = 0.f;
      for (int k = 0; k < dxp; k += 4) {
        float4 xa[RT], ya[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) xa[r] = *reinterpret_cast<const float4*>(sX + (ty + 16 * r) * px + k);
#pragma unroll
        for (int c = 0; c < RT; ++c) ya[c] = *reinterpret_cast<const float4*>(sY + (tx + 16 * c) * px + k);
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int c = 0; c < RT; ++c) {
            acc[r][c] = fmaf(xa[r].x, ya[c].x, acc[r][c]);
            acc[r][c] = fmaf(xa[r].y, ya[c].y, acc[r][c]);
            acc[r][c] = fmaf(xa[r].z, ya[c].z, acc[r][c]);
            acc[r][c] = fmaf(xa[r].w, ya[c].w, acc[r][c]);
          }
      }
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < RT; ++c) {
          const int i = ty + 16 * r, j = tx + 16 * c, e = job.rev ? j - i : i - j;
          float w = e >= 0 ? sPow[e] * job.z_scale : 0.f;
          if (MODE == MODE_TANGENT) w *= float(e);
          sP[i * (C + 4) + j] = e >= 0 ? acc[r][c] * w : 0.f;
        }
      __syncthreads();
      // output rows i = ty RT + r, columns 4 tx .. 4 tx + 3 of the slice
      float o[RT][4], p[MODE == MODE_TANGENT ? RT : 1][4];
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          o[r][c] = 0.f;
          if (MODE == MODE_TANGENT) p[MODE == MODE_TANGENT ? r : 0][c] = 0.f;
        }
      for (int k = 0; k < dx; ++k) {
        const float4 s = *reinterpret_cast<const float4*>(sS + k * E + 4 * tx);
        float4 d;
        if (MODE == MODE_TANGENT) d = *reinterpret_cast<const float4*>(sD + k * E + 4 * tx);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const float x = sX[(ty * RT + r) * px + k];
          o[r][0] = fmaf(x, s.x, o[r][0]);
          o[r][1] = fmaf(x, s.y, o[r][1]);
          o[r][2] = fmaf(x, s.z, o[r][2]);
          o[r][3] = fmaf(x, s.w, o[r][3]);
          if (MODE == MODE_TANGENT) {
            const int q = MODE == MODE_TANGENT ? r : 0;
            p[q][0] = fmaf(x, d.x, p[q][0]);
            p[q][1] = fmaf(x, d.y, p[q][1]);
            p[q][2] = fmaf(x, d.z, p[q][2]);
            p[q][3] = fmaf(x, d.w, p[q][3]);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const int i = ty * RT + r;
        const int e = job.rev ? n - 1 - i : i + 1;
        const float w = e >= 0 && e <= C ? sPow[e] : 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (MODE == MODE_TANGENT) o[r][c] = w * fmaf(float(e), o[r][c], p[MODE == MODE_TANGENT ? r : 0][c]);
          else o[r][c] *= w;
        }
      }
      for (int j = 0; j < C; j += 4) {
        float4 pv[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) pv[r] = *reinterpret_cast<const float4*>(sP + (ty * RT + r) * (C + 4) + j);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float4 z = *reinterpret_cast<const float4*>(sZ + (j + q) * E + 4 * tx);
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const float w = q == 0 ? pv[r].x : q == 1 ? pv[r].y : q == 2 ? pv[r].z : pv[r].w;
            o[r][0] = fmaf(w, z.x, o[r][0]);
            o[r][1] = fmaf(w, z.y, o[r][1]);
            o[r][2] = fmaf(w, z.z, o[r][2]);
            o[r][3] = fmaf(w, z.w, o[r][3]);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const int i = ty * RT + r;
        if (i >= n) continue;
        if (MODE == MODE_TANGENT) {
          const float4 g = *reinterpret_cast<const float4*>(sG + i * E + 4 * tx);
          tsum = fmaf(o[r][0], g.x, fmaf(o[r][1], g.y, fmaf(o[r][2], g.z, fmaf(o[r][3], g.w, tsum))));
        } else {
          const int64_t at = ((b * job.L + t0 + i) * job.H + h) * dz + c0 + 4 * tx;
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (4 * tx + c < cw) {
              if (job.out_f32) static_cast<float*>(job.out)[at + c] = o[r][c] * job.scale;
              else st(static_cast<T*>(job.out), at + c, o[r][c] * job.scale);
            }
        }
      }
      __syncthreads();
    }
    // the update: state rows 4 (ty + 16 i) .. + 3, columns 4 tx .. 4 tx + 3
    const float an = sPow[n];
    for (int k0 = ty * 4; k0 < dxp; k0 += 64) {
      float s[4][4], d[4][4];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[r][c] = d[r][c] = 0.f;
      for (int j = 0; j < n; ++j) {
        const float w = sUpd[j];
        const float4 y = *reinterpret_cast<const float4*>(sY + j * px + k0);
        const float4 z = *reinterpret_cast<const float4*>(sZ + j * E + 4 * tx);
        const float yv[4] = {y.x * w, y.y * w, y.z * w, y.w * w}, zv[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            s[r][c] = fmaf(yv[r], zv[c], s[r][c]);
            if (MODE == MODE_TANGENT) d[r][c] = fmaf(yv[r] * float(n - 1 - j), zv[c], d[r][c]);
          }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int i = (k0 + r) * E + 4 * tx + c;
          const float old = sS[i];
          sS[i] = fmaf(an, old, s[r][c]);
          if (MODE == MODE_TANGENT) sD[i] = fmaf(an, fmaf(float(n), old, sD[i]), d[r][c]);
        }
    }
  }
  __syncthreads();
  if (MODE == MODE_OUT) {
    // rows past the length are zeros
    const int64_t e0 = max(len, int64_t(seg) * job.seg_len), e1 = min(job.L, (int64_t(seg) + 1) * job.seg_len);
    for (int64_t i = threadIdx.x; i < (e1 - e0) * cw; i += THREADS) {
      const int64_t at = ((b * job.L + e0 + i / cw) * job.H + h) * dz + c0 + i % cw;
      if (job.out_f32) static_cast<float*>(job.out)[at] = 0.f;
      else st(static_cast<T*>(job.out), at, 0.f);
    }
  }
  if (MODE != MODE_TANGENT) {
    // MODE_STATE: the piece's own end state; MODE_OUT: the whole walk's
    float* end = MODE == MODE_STATE
                     ? const_cast<float*>(job.start) + (b * job.H + h) * job.start_stride + int64_t(seg) * dx * dz
                     : (job.end && seg == (job.rev ? 0 : job.segs - 1) ? job.end + (b * job.H + h) * dx * dz : nullptr);
    if (end && !idle)
      for (int i = threadIdx.x; i < dx * cw; i += THREADS) end[int64_t(i / cw) * dz + c0 + i % cw] = sS[(i / cw) * E + i % cw];
  } else {
    if (tan.behind) {
      const float* x = tan.behind + (b * job.H + h) * tan.behind_stride + int64_t(seg) * dx * dz;
      for (int i = threadIdx.x; i < dx * cw; i += THREADS)
        tend = fmaf(__ldcg(x + int64_t(i / cw) * dz + c0 + i % cw), sD[(i / cw) * E + i % cw], tend);
    }
    __shared__ float red[THREADS / 32];
    tsum = warp_sum(fmaf(tsum, tan.scale, tend));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = tsum;
    __syncthreads();
    if (threadIdx.x == 0) {
      float s = 0.f;
      for (int w = 0; w < THREADS / 32; ++w) s += red[w];
      tan.part[((int64_t(h) * job.B + b) * job.segs + seg) * slices + sl] = s;
    }
  }
  chain_end();
}

// The pieces' own end states (B, H, segs, n) become the states that enter each piece: one thread per
// state element walks the pieces in the direction of time (or back), eight loads ahead of their use.
// last: the state behind the walk (the last piece's own end state has to be there), or NULL.
struct EnterSet {
  float* pieces[2];
  const float* first[2];
  float* last[2];
  int rev[2];
  const float* log_decay;
  const int32_t* lengths;
  int64_t L, seg_len, n;
  int H, segs, blocks;
  Link link;
};
__global__ void __launch_bounds__(128) enter_kernel(const __grid_constant__ EnterSet a) {
  constexpr int U = 8;
  chain_begin(a.link);
  const int w = blockIdx.y, rev = a.rev[w], segs = a.segs;
  const int64_t bh = blockIdx.x / a.blocks, b = bh / a.H, n = a.n;
  const float l2 = log2_decay(a.log_decay[bh % a.H]);
  const int64_t len = row_length(a.lengths, b, a.L);
  const int64_t i = int64_t(blockIdx.x % a.blocks) * 128 + threadIdx.x;
  if (i >= n) return;
  float cur = a.first[w] ? a.first[w][bh * n + i] : 0.f;
  float* __restrict__ p = a.pieces[w] + bh * segs * n + i;
  const int own_segs = a.last[w] ? segs : segs - 1;
  for (int k0 = 0; k0 < segs; k0 += U) {
    float own[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u;
      own[u] = k < own_segs ? p[int64_t(rev ? segs - 1 - k : k) * n] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u, s = rev ? segs - 1 - k : k;
      if (k >= segs) break;
      const int64_t s0 = min(len, s * a.seg_len), s1 = min(len, s0 + a.seg_len);
      p[int64_t(s) * n] = cur;
      if (s1 > s0) cur = fmaf(exp2f(l2 * float(s1 - s0)), cur, own[u]);   // (no tokens: a^0, of a NaN too)
    }
  }
  if (a.last[w]) a.last[w][bh * n + i] = cur;
}

// out (tokens, heads, d) = sum over the H / heads operator heads that share each head of part (tokens, H, d),
// for up to three tensors (blockIdx.y)
struct ShareSet {
  const float* part[3];
  void* out[3];
  int64_t n[3];
  int heads[3], group[3], d[3];
  Link link;
};
template <class T>
__global__ void __launch_bounds__(256) share_sum_kernel(const __grid_constant__ ShareSet a) {
  chain_begin(a.link);
  const int w = blockIdx.y, heads = a.heads[w], group = a.group[w], d = a.d[w];
  T* out = static_cast<T*>(a.out[w]);
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < a.n[w]; i += int64_t(gridDim.x) * 256) {
    const int64_t th = i / d;
    const int64_t t = th / heads, hh = th % heads;
    const float* p = a.part[w] + (t * heads * group + hh * group) * d + i % d;
    float s = 0.f;
    for (int r = 0; r < group; ++r) s += __ldcg(p + int64_t(r) * d);
    st(out, i, s);
  }
}

// grad ln a of head h: its partials in order
__global__ void __launch_bounds__(256) decay_sum_kernel(const float* part, float* out, int64_t n, int accumulate,
                                                        const Link link) {
  chain_begin(link);
  __shared__ float red[8];
  const float* p = part + int64_t(blockIdx.x) * n;
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += 256) s += p[i];
  s = warp_sum(s);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    float v = 0.f;
    for (int w = 0; w < 8; ++w) v += red[w];
    out[blockIdx.x] = accumulate ? out[blockIdx.x] + v : v;
  }
}

template <class T, int C, int MODE>
static int walk_as(const Jobs& jobs, int rows, const TangentArgs& tan, cudaStream_t s) {
  static int limit = 0;
  const size_t smem = smem_bytes((rows + 3) & ~3, MODE);
  PGF_CUDA(ensure_dynamic_smem(walk_kernel<T, C, MODE>, smem, limit));
  PGF_CUDA(launch_link(jobs.link, walk_kernel<T, C, MODE>, unsigned(jobs.first[3]), THREADS, smem, s, jobs, tan));
  PGF_LAUNCH_CHECK();
  return PGF_OK;
}

template <int MODE>
static int walk(const Job* job, int count, const TangentArgs& tan, const Link& link, int dtype, cudaStream_t s) {
  Jobs jobs = {};
  int64_t ctas = 0;
  int rows = 0;
  for (int k = 0; k < 3; ++k) {
    jobs.first[k] = int(ctas);
    if (k >= count) continue;
    jobs.job[k] = job[k];
    ctas += job[k].B * job[k].H * job[k].segs * ceil_div(job[k].z.d, E);
    if (job[k].x.d > rows) rows = job[k].x.d;
  }
  PGF_CHECK_ARG(ctas < 0x7fffffff, "decay_attn: too many pieces");
  jobs.first[3] = int(ctas);
  jobs.link = link;
  if (dtype == PGF_DTYPE_BF16)
    return rows > 128 ? walk_as<__nv_bfloat16, 32, MODE>(jobs, rows, tan, s)
                      : walk_as<__nv_bfloat16, 64, MODE>(jobs, rows, tan, s);
  return rows > 128 ? walk_as<float, 32, MODE>(jobs, rows, tan, s) : walk_as<float, 64, MODE>(jobs, rows, tan, s);
}

// ---------------------------------------------------------------------------------------------
// One token: S' = a S + k v^T, o = scale q S'.  It reads and writes the state (8 Dk Dv bytes per head), but what it
// waits for is the chain of a short CTA (vectors, barrier, state, barrier; 4 resident, 3.5 waves at the first size
// below): DRAM and L2 are at 24 and 22%, issue slots at 44%.  A CTA owns a slice of the columns of one (row, head); a
// thread keeps four columns and walks the rows, its loads ahead of its arithmetic; the row sums of o meet in shared
// memory in a fixed order.
// 128 rows x 16 heads of 64 x 64: 16.5 us for 67 MB (22 with single columns instead of four); 1 row x 8 heads
// of 128 x 128: 3.2 us, the length of its chain of loads.
// ---------------------------------------------------------------------------------------------
struct StepArgs {
  Tensor q, k, v;            // one token each: the token stride is unused
  const float* log_decay;
  const float* state;        // (n_src, H, Dk, Dv)
  const int64_t* rows;       // (B) row of `state` that each row goes on from, or NULL
  int64_t n_src;
  void* out;                 // (B, H, Dv)
  float* state_out;          // (B, H, Dk, Dv)
  int H, slice;              // columns of one CTA
  float scale;
};

template <class T, int W>
__global__ void __launch_bounds__(256) step_kernel(const StepArgs a) {
  __shared__ float sq[MAX_D], sk[MAX_D];
  __shared__ float so[256 * W];
  const int Dk = a.q.d, Dv = a.v.d;
  const int slices = (Dv + a.slice - 1) / a.slice;
  const int64_t bh = blockIdx.x / slices, b = bh / a.H;
  const int h = int(bh % a.H), c0 = int(blockIdx.x % slices) * a.slice;
  const int nx = a.slice / W, ny = 256 / nx;          // threads across the slice, row groups
  const int tx = threadIdx.x % nx, ty = threadIdx.x / nx, c = c0 + tx * W;
  const bool on = c < Dv;
  const T* q = static_cast<const T*>(a.q.p) + b * a.q.s.batch + int64_t(h / (a.H / a.q.heads)) * a.q.s.head;
  const T* k = static_cast<const T*>(a.k.p) + b * a.k.s.batch + int64_t(h / (a.H / a.k.heads)) * a.k.s.head;
  const T* v = static_cast<const T*>(a.v.p) + b * a.v.s.batch + int64_t(h / (a.H / a.v.heads)) * a.v.s.head;
  if (threadIdx.x < Dk) {
    sq[threadIdx.x] = ld(q, threadIdx.x);
    sk[threadIdx.x] = ld(k, threadIdx.x);
  }
  const int64_t from = a.rows ? a.rows[b] : b;
  const bool known = from >= 0 && from < a.n_src;  // a row out of range goes on from zeros
  const float* s = a.state + ((known ? from : 0) * a.H + h) * Dk * Dv + c;
  float* s2 = a.state_out + bh * Dk * Dv + c;
  const float an = exp2f(log2_decay(a.log_decay[h]));
  float vv[W], o[W];
#pragma unroll
  for (int e = 0; e < W; ++e) {
    vv[e] = on ? ld(v, c + e) : 0.f;
    o[e] = 0.f;
  }
  __syncthreads();
  if (on) {
    constexpr int U = 4;
    for (int r0 = ty; r0 < Dk; r0 += U * ny) {
      float t[U][W];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * ny;
        if (r < Dk && known) {
          if constexpr (W == 4) {
            const float4 f = *reinterpret_cast<const float4*>(s + int64_t(r) * Dv);
            t[u][0] = f.x; t[u][1] = f.y; t[u][2] = f.z; t[u][3] = f.w;
          } else {
            t[u][0] = s[int64_t(r) * Dv];
          }
        } else {
#pragma unroll
          for (int e = 0; e < W; ++e) t[u][e] = 0.f;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * ny;
        if (r < Dk) {
          const float kr = sk[r], qr = sq[r];
#pragma unroll
          for (int e = 0; e < W; ++e) {
            t[u][e] = fmaf(an, t[u][e], kr * vv[e]);
            o[e] = fmaf(qr, t[u][e], o[e]);
          }
          if constexpr (W == 4) *reinterpret_cast<float4*>(s2 + int64_t(r) * Dv) = make_float4(t[u][0], t[u][1], t[u][2], t[u][3]);
          else s2[int64_t(r) * Dv] = t[u][0];
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < W; ++e) so[ty * a.slice + tx * W + e] = o[e];
  __syncthreads();
  for (int i = threadIdx.x; i < a.slice && c0 + i < Dv; i += 256) {
    float sum = 0.f;
    for (int y = 0; y < ny; ++y) sum += so[y * a.slice + i];
    st(static_cast<T*>(a.out), bh * Dv + c0 + i, sum * a.scale);
  }
}

// ---------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------
// How the sequence is cut.  Pieces run side by side, but all except one have their y and z read a second time
// (for the states that enter the others), so the cut is the one with the least time over the waves of CTAs, in
// units of a chunk's time in a walk: a piece's chunks plus 2.5 for its start and end, the same for the states' pass
// at 0.6 of the walk's pace (0.8 in a backward, whose two passes end before its walks begin), and 3 for the two more
// launches.  walks and passes count what one call runs side by side
// (a backward's launches overlap).  Measured with and without a cut: 65536 tokens x 8 heads of 128, forward,
// 188 and 1929 us; 7 rows of 1999 x 8 heads of 64, 37 and 34 us; backward of 9 x 3000 x 8 heads of 128,
// 440 and 355 us; of 1 x 2000 x 8 heads of 128, 65 and 73 us.
// The float32 engine's walk of a chunk is longer beside its other parts and several CTAs share an SM: with its own
// constants below, 2 x 777 tokens x 6 heads take 94 us backward in 13 pieces, 100 in 7, 138 in 4 and 425 in one.
struct Cut {
  int segs;
  int64_t seg_len;
};
static Cut cut(int64_t ctas, int64_t L, int chunk, bool tc, int resident, int walks, int passes) {
  const int64_t chunks = (L + chunk - 1) / chunk, slots = 148 * resident;
  Cut best = {1, (chunks ? chunks : 1) * chunk};
  if (ctas == 0) return best;
  auto waves = [&](int64_t n) { return double((ctas * n + slots - 1) / slots); };
  double least = 0;
  // (more than two waves of pieces never pay)
  for (int64_t s = 1; s <= chunks && (s == 1 || ctas * s <= 2 * slots); ++s) {
    const int64_t per = (chunks + s - 1) / s, n = (chunks + per - 1) / per;
    if (n != s) continue;
    double t;
    if (tc) t = waves(walks * n) * (per + 2.5) + (n > 1 ? waves(passes * n) * (per + 2.5) * (passes > 1 ? 0.8 : 0.6) + 3.0 : 0.0);
    else t = waves(n) * (per * (n > 1 ? 1.5 : 1.0) + 2.5) + (n > 1 ? 3.0 : 0.0);
    if (s == 1 || t < least) {
      least = t;
      best = {int(n), per * chunk};
    }
  }
  return best;
}

struct Shape {
  int64_t B, L, H, Hq, Hk, Hv, Dk, Dv;
};

static int check(const char* what, const Shape& s, int dtype) {
  PGF_CHECK_ARG(s.B >= 0 && s.L >= 0 && s.B <= (1 << 22) && s.H >= 1 && s.H <= (1 << 22) && s.B * s.H <= (1 << 22) &&
                    s.L < (int64_t(1) << 31),
                "%s: bad shape B=%lld L=%lld H=%lld", what, (long long)s.B, (long long)s.L, (long long)s.H);
  PGF_CHECK_ARG(s.Hq >= 1 && s.Hk >= 1 && s.Hv >= 1 && s.H % s.Hq == 0 && s.H % s.Hk == 0 && s.H % s.Hv == 0,
                "%s: %lld query, %lld key and %lld value heads for %lld states (each must divide)", what, (long long)s.Hq,
                (long long)s.Hk, (long long)s.Hv, (long long)s.H);
  PGF_CHECK_ARG(s.Dk >= 1 && s.Dk <= MAX_D && s.Dv >= 1 && s.Dv <= MAX_D, "%s: head widths %lld and %lld (1 to %d)", what,
                (long long)s.Dk, (long long)s.Dv, MAX_D);
  PGF_CHECK_ARG(dtype == PGF_DTYPE_F32 || dtype == PGF_DTYPE_BF16, "%s: dtype %d", what, dtype);
  return PGF_OK;
}

static Tensor tensor(const void* p, const pgf_strides* s, int64_t L, int64_t heads, int64_t d) {
  Tensor t;
  t.p = p;
  t.heads = int(heads);
  t.d = int(d);
  if (s) t.s = *s;
  else t.s = {L * heads * d, heads * d, d};
  t.vec = aligned(p, 16) && t.s.batch % 4 == 0 && t.s.token % 4 == 0 && t.s.head % 4 == 0;
  return t;
}

// The calls of one entry point take one engine and one cut.
struct Plan {
  bool tc;
  Cut c;
};
static Plan plan(const Shape& p, bool tc, bool backward) {
  const int walks = backward ? 4 : 1, passes = backward ? 2 : 1;   // (grad ln a is a walk of its own)
  if (tc) return {true, cut(p.B * p.H, p.L, TC_CHUNK, true, 1, walks, passes)};
  // a backward's calls have either width as columns and either as rows
  const int64_t cols = backward && p.Dk < p.Dv ? p.Dk : p.Dv, rows = backward && p.Dv > p.Dk ? p.Dv : p.Dk;
  const int resident = int(233472 / (smem_bytes((int(rows) + 3) & ~3, MODE_OUT) + 1024));
  return {false, cut(p.B * p.H * ceil_div(cols, E), p.L, chunk_of(int(rows)), false, resident, walks, passes)};
}

// The state that enters each piece of a walk: (B, H, segs, rows, columns).
struct Entering {
  const float* p;       // NULL: zeros (an uncut walk without a first state)
  int64_t stride;
};

static int f_calls(const Job* job, int count, const Plan& pl, Chain& chain, int dtype, cudaStream_t s) {
  if (!pl.tc) return walk<MODE_OUT>(job, count, TangentArgs{}, chain.next(), dtype, s);
  for (int k = 0; k < count; ++k) PGF_TRY(tc_walk(job[k], chain.next(), s));
  return PGF_OK;
}

// What enters the pieces of one or two walks of the same shape that begin with `first`; `pieces` is scratch for
// them.  last: where the state behind a cut walk goes, or NULL (an uncut one gives it by itself).
static int entering(Job* job, int count, const Plan& pl, const float* const* first, float* const* pieces,
                    float* const* last, Entering* e, Chain& chain, int dtype, cudaStream_t s) {
  const int64_t n = int64_t(job[0].y.d) * job[0].z.d;
  const int segs = job[0].segs;
  for (int k = 0; k < count; ++k) e[k] = {first[k], n};
  if (segs == 1) return PGF_OK;
  EnterSet set;
  for (int k = 0; k < count; ++k) {
    job[k].start = pieces[k];
    job[k].start_stride = segs * n;
    job[k].start_t = 0;
    job[k].last_too = last[k] != nullptr;
    set.pieces[k] = pieces[k];
    set.first[k] = first[k];
    set.last[k] = last[k];
    set.rev[k] = job[k].rev;
    e[k] = {pieces[k], segs * n};
  }
  if (pl.tc) {
    for (int k = 0; k < count; ++k) PGF_TRY(tc_pieces(job[k], chain.next(), s));
  } else {
    PGF_TRY(walk<MODE_STATE>(job, count, TangentArgs{}, chain.next(), dtype, s));
  }
  set.log_decay = job[0].log_decay;
  set.lengths = job[0].lengths;
  set.L = job[0].L;
  set.seg_len = job[0].seg_len;
  set.n = n;
  set.H = job[0].H;
  set.segs = segs;
  set.blocks = ceil_div(n, 128);
  chain.wait = 1;
  set.link = chain.next();
  PGF_CUDA(launch_link(set.link, enter_kernel, dim3(unsigned(job[0].B * job[0].H * set.blocks), unsigned(count)), 128, 0, s,
                       set));
  PGF_LAUNCH_CHECK();
  chain.wait = 1;
  return PGF_OK;
}

static size_t workspace(const Shape& p, bool backward) {
  const size_t state = size_t(p.B) * p.H * p.Dk * p.Dv * sizeof(float);
  const Plan f = plan(p, false, backward), t = plan(p, true, backward);
  size_t pieces = 0;
  for (const Plan& q : {f, t})
    if (q.c.segs > 1 && q.c.segs * state > pieces) pieces = q.c.segs * state;
  size_t n = 0;
  if (pieces) n += (backward ? 2 : 1) * (Workspace::round(pieces) + 256);
  if (backward) {
    const int segs = f.c.segs > t.c.segs ? f.c.segs : t.c.segs;
    n += Workspace::round(size_t(p.H) * p.B * segs * ceil_div(p.Dk, 64) * ceil_div(p.Dv, 64) * sizeof(float)) + 256;
    const size_t tok = size_t(p.B) * p.L * p.H * sizeof(float);
    if (p.Hq < p.H) n += Workspace::round(tok * p.Dk) + 256;
    if (p.Hk < p.H) n += Workspace::round(tok * p.Dk) + 256;
    if (p.Hv < p.H) n += Workspace::round(tok * p.Dv) + 256;
  }
  return n;
}

}  // namespace da
}  // namespace pgf

using namespace pgf;

extern "C" size_t pgf_decay_attn_workspace(int64_t Bsz, int64_t L, int64_t H, int64_t Hq, int64_t Hk, int64_t Hv,
                                           int64_t Dk, int64_t Dv, int dtype, int backward) {
  const da::Shape p = {Bsz, L, H, Hq, Hk, Hv, Dk, Dv};
  if (da::check("decay_attn_workspace", p, dtype) != PGF_OK) return 0;
  return da::workspace(p, backward != 0);
}

extern "C" int pgf_decay_attn_fwd(const void* q, const pgf_strides* q_strides, const void* k,
                                  const pgf_strides* k_strides, const void* v, const pgf_strides* v_strides,
                                  const float* log_decay, const float* state, const int32_t* lengths, void* out,
                                  float* state_out, int64_t Bsz, int64_t L, int64_t H, int64_t Hq, int64_t Hk, int64_t Hv,
                                  int64_t Dk, int64_t Dv, float scale, int dtype, void* ws, size_t ws_bytes,
                                  pgf_stream_t stream) {
  clear_error();
  const da::Shape p = {Bsz, L, H, Hq, Hk, Hv, Dk, Dv};
  PGF_TRY(da::check("decay_attn_fwd", p, dtype));
  if (Bsz == 0) return PGF_OK;
  PGF_CHECK_ARG(log_decay && (L == 0 || (q && k && v && out)), "decay_attn_fwd: null pointer");
  cudaStream_t s = as_stream(stream);
  da::Job job = {};
  job.x = da::tensor(q, q_strides, L, Hq, Dk);
  job.y = da::tensor(k, k_strides, L, Hk, Dk);
  job.z = da::tensor(v, v_strides, L, Hv, Dv);
  job.log_decay = log_decay;
  job.lengths = lengths;
  job.out = out;
  job.out_f32 = dtype == PGF_DTYPE_F32;
  job.end = state_out;
  job.scale = scale;
  job.z_scale = 1.f;
  job.B = Bsz; job.L = L; job.H = int(H);
  const bool tc = dtype == PGF_DTYPE_BF16 && L > 0 && da::tc_fits(job.x, Bsz, L) && da::tc_fits(job.y, Bsz, L) &&
                  da::tc_fits(job.z, Bsz, L) && aligned(out, 16) && aligned(state, 16) && aligned(state_out, 16);
  const da::Plan pl = da::plan(p, tc, false);
  job.segs = pl.c.segs;
  job.seg_len = pl.c.seg_len;
  float* pieces = nullptr;
  if (job.segs > 1) {
    Workspace w(ws, ws_bytes);
    pieces = w.take<float>(size_t(Bsz) * H * job.segs * Dk * Dv);
    if (!ws || !pieces) {
      set_error("decay_attn_fwd: workspace of %zu bytes is too small", ws_bytes);
      return PGF_ERR_WORKSPACE;
    }
  }
  da::Entering S;
  Chain chain;
  da::Job js = job;
  PGF_TRY(da::entering(&js, 1, pl, &state, &pieces, &state_out, &S, chain, dtype, s));
  if (job.segs > 1) job.end = nullptr;
  job.start = S.p;
  job.start_stride = S.stride;
  return da::f_calls(&job, 1, pl, chain, dtype, s);
}

extern "C" int pgf_decay_attn_bwd(const void* q, const pgf_strides* q_strides, const void* k,
                                  const pgf_strides* k_strides, const void* v, const pgf_strides* v_strides,
                                  const float* log_decay, const float* state, const int32_t* lengths, const void* g,
                                  const pgf_strides* g_strides, const float* g_state, void* grad_q, void* grad_k,
                                  void* grad_v, float* grad_log_decay, float* grad_state, int accumulate, int64_t Bsz,
                                  int64_t L, int64_t H, int64_t Hq, int64_t Hk, int64_t Hv, int64_t Dk, int64_t Dv,
                                  float scale, int dtype, void* ws, size_t ws_bytes, pgf_stream_t stream) {
  clear_error();
  const da::Shape p = {Bsz, L, H, Hq, Hk, Hv, Dk, Dv};
  PGF_TRY(da::check("decay_attn_bwd", p, dtype));
  cudaStream_t s = as_stream(stream);
  if (Bsz == 0) {
    if (grad_log_decay && !accumulate) PGF_CUDA(cudaMemsetAsync(grad_log_decay, 0, size_t(H) * sizeof(float), s));
    return PGF_OK;
  }
  PGF_CHECK_ARG(log_decay && (L == 0 || (q && k && v && g && grad_q && grad_k && grad_v)), "decay_attn_bwd: null pointer");
  const da::Tensor tq = da::tensor(q, q_strides, L, Hq, Dk), tk = da::tensor(k, k_strides, L, Hk, Dk),
                   tv = da::tensor(v, v_strides, L, Hv, Dv), tg = da::tensor(g, g_strides, L, H, Dv);
  const bool tc = dtype == PGF_DTYPE_BF16 && L > 0 && da::tc_fits(tq, Bsz, L) && da::tc_fits(tk, Bsz, L) &&
                  da::tc_fits(tv, Bsz, L) && da::tc_fits(tg, Bsz, L) && aligned(grad_q, 16) && aligned(grad_k, 16) &&
                  aligned(grad_v, 16) && aligned(state, 16) && aligned(g_state, 16) && aligned(grad_state, 16);
  const da::Plan pl = da::plan(p, tc, true);
  da::Job job = {};
  job.log_decay = log_decay;
  job.lengths = lengths;
  job.B = Bsz; job.L = L; job.H = int(H);
  job.scale = 1.f;
  job.segs = pl.c.segs;
  job.seg_len = pl.c.seg_len;
  Workspace w(ws, ws_bytes);
  const size_t states = size_t(Bsz) * H * job.segs * Dk * Dv;
  float* sp = job.segs > 1 ? w.take<float>(states) : nullptr;
  float* xp = job.segs > 1 ? w.take<float>(states) : nullptr;
  float* part = grad_log_decay ? w.take<float>(size_t(H) * Bsz * job.segs * ceil_div(Dk, 64) * ceil_div(Dv, 64)) : nullptr;
  const int64_t tokens = Bsz * L;
  float* pq = Hq < H ? w.take<float>(size_t(tokens) * H * Dk) : nullptr;
  float* pk = Hk < H ? w.take<float>(size_t(tokens) * H * Dk) : nullptr;
  float* pv = Hv < H ? w.take<float>(size_t(tokens) * H * Dv) : nullptr;
  if ((grad_log_decay && !part) || (job.segs > 1 && (!sp || !xp)) || (Hq < H && !pq) || (Hk < H && !pk) || (Hv < H && !pv)) {
    set_error("decay_attn_bwd: workspace of %zu bytes is too small", ws_bytes);
    return PGF_ERR_WORKSPACE;
  }
  // what enters the pieces from both ends; X carries the scale of g
  da::Entering ends[2];
  Chain chain;
  {
    da::Job js[2] = {job, job};
    js[0].x = js[0].y = tk; js[0].z = tv;
    js[0].z_scale = 1.f;
    js[1].x = js[1].y = tq; js[1].z = tg;
    js[1].z_scale = scale;
    js[1].rev = 1;
    const float* first[2] = {state, g_state};
    float *pieces[2] = {sp, xp}, *last[2] = {nullptr, grad_state};
    PGF_TRY(da::entering(js, 2, pl, first, pieces, last, ends, chain, dtype, s));
  }
  const da::Entering S = ends[0], X = ends[1];
  const int f32 = dtype == PGF_DTYPE_F32;
  // grad q = scale F(g, v, k; S^T)
  da::Job calls[3] = {job, job, job};
  da::Job &jq = calls[0], &jv = calls[1], &jk = calls[2];
  jq.x = tg; jq.y = tv; jq.z = tk;
  jq.start = S.p; jq.start_stride = S.stride; jq.start_t = 1;
  jq.scale = scale; jq.z_scale = 1.f;
  jq.out = pq ? static_cast<void*>(pq) : grad_q;
  jq.out_f32 = f32 || pq;
  // grad v = F(k, q, scale g; X) from the end
  jv.x = tk; jv.y = tq; jv.z = tg;
  jv.start = X.p; jv.start_stride = X.stride; jv.rev = 1;
  jv.z_scale = scale;
  jv.out = pv ? static_cast<void*>(pv) : grad_v;
  jv.out_f32 = f32 || pv;
  jv.end = job.segs > 1 ? nullptr : grad_state;
  // grad k = F(v, g, scale q; X^T) from the end
  jk.x = tv; jk.y = tg; jk.z = tq;
  jk.start = X.p; jk.start_stride = X.stride; jk.start_t = 1; jk.rev = 1;
  jk.z_scale = scale;
  jk.out = pk ? static_cast<void*>(pk) : grad_k;
  jk.out_f32 = f32 || pk;
  PGF_TRY(da::f_calls(calls, 3, pl, chain, dtype, s));
  if (grad_log_decay) {
    int parts;
    if (tc) {
      da::TangentJob t = {};
      t.q = tq; t.k = tk; t.v = tv; t.g = tg;
      t.log_decay = log_decay;
      t.lengths = lengths;
      t.start = S.p; t.start_stride = S.stride;
      t.behind = X.p; t.behind_stride = X.stride;
      t.part = part;
      t.scale = scale;
      t.B = Bsz; t.L = L; t.seg_len = job.seg_len;
      t.H = int(H); t.segs = job.segs;
      PGF_TRY(da::tc_tangent(t, chain.next(), s));
      parts = da::tc_tangent_blocks(Dk, Dv);
    } else {
      da::Job jt = job;
      jt.x = tq; jt.y = tk; jt.z = tv;
      jt.start = S.p; jt.start_stride = S.stride;
      jt.z_scale = 1.f;
      da::TangentArgs t = {};
      t.g = tg;
      t.behind = X.p;
      t.behind_stride = X.stride;
      t.part = part;
      t.scale = scale;
      PGF_TRY(da::walk<da::MODE_TANGENT>(&jt, 1, t, chain.next(), dtype, s));
      parts = ceil_div(Dv, da::E);
    }
    chain.wait = 1;
    const Link sum = chain.next();
    PGF_CUDA(launch_link(sum, da::decay_sum_kernel, unsigned(H), 256, 0, s, part, grad_log_decay,
                             int64_t(Bsz * job.segs * parts), accumulate, sum));
    PGF_LAUNCH_CHECK();
  }
  if (L == 0) return PGF_OK;
  const struct { float* part; void* out; int64_t heads, d; } sums[3] = {{pq, grad_q, Hq, Dk}, {pk, grad_k, Hk, Dk}, {pv, grad_v, Hv, Dv}};
  da::ShareSet set;
  int count = 0;
  int64_t most = 0;
  for (const auto& t : sums) {
    if (!t.part) continue;
    set.part[count] = t.part;
    set.out[count] = t.out;
    set.n[count] = tokens * t.heads * t.d;
    set.heads[count] = int(t.heads);
    set.group[count] = int(H / t.heads);
    set.d[count] = int(t.d);
    if (set.n[count] > most) most = set.n[count];
    ++count;
  }
  if (count) {
    int64_t ctas = (most + 255) / 256;
    if (ctas > 148 * 16) ctas = 148 * 16;
    chain.wait = 1;
    set.link = chain.next();
    PGF_CUDA(launch_link(set.link, f32 ? da::share_sum_kernel<float> : da::share_sum_kernel<__nv_bfloat16>,
                             dim3(unsigned(ctas), unsigned(count)), 256, 0, s, set));
    PGF_LAUNCH_CHECK();
  }
  return PGF_OK;
}

extern "C" int pgf_decay_attn_step(const void* q, const pgf_strides* q_strides, const void* k,
                                   const pgf_strides* k_strides, const void* v, const pgf_strides* v_strides,
                                   const float* log_decay, const float* state, const int64_t* rows, int64_t n_src,
                                   void* out, float* state_out, int64_t Bsz, int64_t H, int64_t Hq, int64_t Hk, int64_t Hv,
                                   int64_t Dk, int64_t Dv, float scale, int dtype, pgf_stream_t stream) {
  clear_error();
  const da::Shape p = {Bsz, 1, H, Hq, Hk, Hv, Dk, Dv};
  PGF_TRY(da::check("decay_attn_step", p, dtype));
  PGF_CHECK_ARG(n_src >= 0 && (rows || n_src == Bsz), "decay_attn_step: %lld states for %lld rows", (long long)n_src,
                (long long)Bsz);
  if (Bsz == 0) return PGF_OK;
  PGF_CHECK_ARG(q && k && v && log_decay && (state || n_src == 0) && out && state_out, "decay_attn_step: null pointer");
  const float *a0 = state, *a1 = state + n_src * H * Dk * Dv, *b0 = state_out, *b1 = state_out + Bsz * H * Dk * Dv;
  PGF_CHECK_ARG((!rows && a0 == b0) || a1 <= b0 || b1 <= a0,
                "decay_attn_step: the new states would overwrite states that other rows read");
  da::StepArgs a;
  a.q = da::tensor(q, q_strides, 1, Hq, Dk);
  a.k = da::tensor(k, k_strides, 1, Hk, Dk);
  a.v = da::tensor(v, v_strides, 1, Hv, Dv);
  a.log_decay = log_decay;
  a.state = state; a.rows = rows; a.n_src = n_src;
  a.out = out; a.state_out = state_out;
  a.H = int(H); a.scale = scale;
  const bool vec = Dv % 4 == 0 && aligned(state, 16) && aligned(state_out, 16);
  // whole rows of the state per CTA; narrower slices while that leaves SMs without work (8 heads of 128 x 128:
  // 3.2 us in slices of 16 and 4.6 whole; 2048 heads of 64 x 64: 46 us in slices of 16 and 16.5 whole)
  int slice = vec ? 4 : 1;
  while (slice < Dv) slice *= 2;
  const int least = vec ? 16 : 8;
  while (slice > least && Bsz * H * ceil_div(Dv, slice) < 148) slice /= 2;
  a.slice = slice;
  const unsigned grid = unsigned(Bsz * H * ceil_div(Dv, slice));
  cudaStream_t s = as_stream(stream);
  if (dtype == PGF_DTYPE_BF16) {
    if (vec) da::step_kernel<__nv_bfloat16, 4><<<grid, 256, 0, s>>>(a);
    else da::step_kernel<__nv_bfloat16, 1><<<grid, 256, 0, s>>>(a);
  } else {
    if (vec) da::step_kernel<float, 4><<<grid, 256, 0, s>>>(a);
    else da::step_kernel<float, 1><<<grid, 256, 0, s>>>(a);
  }
  PGF_LAUNCH_CHECK();
  return PGF_OK;
}
