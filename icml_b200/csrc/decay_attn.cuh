// Linear attention with a decay for each head: what its engines share.
//
//   S_t = a S_{t-1} + k_t v_t^T         (Dk x Dv, float32),  a = exp(log_decay) of the head
//   o_t = scale q_t S_t
//
// Over a chunk of n tokens from the state S (tokens 0 .. n-1):
//   o_i = sum_{j <= i} a^(i-j) (q_i k_j) v_j + a^(i+1) q_i S
//   S'  = a^n S + sum_j a^(n-1-j) k_j v_j^T
// and, walked from the end with X the adjoint of the state behind the chunk (the same sums mirrored):
//   r_j = sum_{i >= j} a^(i-j) (x_j y_i) z_i + a^(n-1-j) x_j X
//   X'  = a^n X + sum_i a^(i+1) y_i z_i^T
//
// One operator F(x, y, z; state, direction) therefore gives the forward pass and every gradient:
//   out    = F(q, k, v; S)            forward
//   grad q = F(g, v, k; S^T)          forward
//   grad v = F(k, q, g; X)            from the end, X = sum a^(..) q g^T + the final state's gradient
//   grad k = F(v, g, q; X^T)          from the end
// with g the output's gradient.  X' before the first token is the initial state's gradient.
//
// A chunk's pairs are formed by products whose masked weights are zeros, so a value that is infinite or NaN reaches
// its column from the first token of its chunk on (at most 128 tokens, counted from the sequence's start), not from
// its own token.  Rows past the length are replaced by zeros first: whatever lies there reaches nothing.
#pragma once
#include "chain.cuh"

namespace pgf {
namespace da {

constexpr int MAX_D = 256;

struct Tensor {
  const void* p;
  pgf_strides s;
  int heads;      // divides H: head h of the operator reads head h / (H / heads)
  int d;
  int vec;        // base and strides are whole 16-byte units of float32
};

// One F call.
struct Job {
  Tensor x, y, z;            // widths x.d == y.d == rows of the state, z.d its columns
  const float* log_decay;    // (H)
  const int32_t* lengths;    // (B) or NULL: tokens past a row's length are not there
  const float* start;        // (B, H, segs, x.d, z.d), or its transpose; NULL: zeros
  int64_t start_stride;      // floats between (b, h) entries of start
  int start_t;               // start holds (z.d, x.d)
  void* out;                 // (B, L, H, z.d) contiguous
  int out_f32;               // out is float32 (else the inputs' type)
  float* end;                // (B, H, x.d, z.d) the state after the walk, or NULL
  float scale;               // of out
  float z_scale;             // of z, in the output and in the state
  int64_t B, L;
  int H;
  int rev;                   // walk from the end
  int segs;                  // pieces of the sequence walked in parallel
  int64_t seg_len;           // tokens of a piece, a multiple of the engine's chunk
  int last_too;              // pieces' own end states: the walk's last piece as well
};

// a^e for the exponents of one head.  log2(a) is clamped so that e = 0 gives 1 for a decay of zero; a NaN stays one.
__device__ __forceinline__ float log2_decay(float log_decay) {
  const float l2 = log_decay * 1.4426950408889634f;
  return l2 < -1.0e4f ? -1.0e4f : l2;
}

__device__ __forceinline__ int64_t row_length(const int32_t* lengths, int64_t b, int64_t L) {
  if (!lengths) return L;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : n > L ? L : n;
}

}  // namespace da
}  // namespace pgf
