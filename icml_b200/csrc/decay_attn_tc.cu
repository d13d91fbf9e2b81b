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
// Roles (640 threads): warp 0 TMA loads, warp 1 MMA, warps 2..9 scores and output ("X"), warps 10..17 the
// weighted y and the state ("Y"), warp 18 the output's TMA stores.  The chunk's steps overlap with its
// neighbours': X forms P of chunk c beside the output of c - 1, so that it seldom waits for a product;
// Y publishes S and weighs y before it waits for U (64-wide heads have two buffers of A, U and y's smaller terms, so
// that y of the next chunk is weighed while this one's U is formed).  Input tiles pass through a ring of slots in the
// order y, x, z; hi overwrites y in its slot once A is done, and the output is staged in z's slot.  Every wait is
// bounded.
//
// What bounds it: the chain of a chunk's steps (weigh, product, state) in shared memory, which the products' operands
// and the warps share (4,350 wavefronts of a 128-wide chunk's 7,500 cycles).  65536 tokens x 8 heads of 128
// take 129 us (16 x 2048 x 16 heads of 64: 72 us), 4.2 TB/s of its four tensors; a 128-wide chunk takes 3.2 us where
// 32 SMs walk and 4.2 where all do, and the warps that weigh y are the ones that the others wait for.  Measured
// and slower: the output stored straight from registers (157 against 129 us), half of y weighed by X (148 against
// 137), y weighed by parts of 32 tokens out of place (139 against 128), the next A in front of D1 (144 against 129).
// 640 threads leave 96 registers each: the walks with 128-wide z spill 48 to 144 bytes a thread, those with 64-wide z
// none.
// The float32 engine (decay_attn.cu) takes 3350 us for the first of these sizes: bf16 inputs of widths that are
// multiples of 8 up to 128, in 16-byte aligned tensors, go here whatever their number.
//
// P takes two multiplications for 32 x 32 blocks off the diagonal (a^(i-j) as a row factor times a column factor,
// both with exponents >= 0: no overflow for any decay), a table look-up for the four on it, nothing for the rest.
#include "decay_attn_tc.cuh"

namespace pgf {
namespace da {

namespace {

constexpr int C = TC_CHUNK;
constexpr int THREADS = 640;
constexpr uint32_t TMEM_COLS = 512;

// NT: bf16 terms of the weighted y.  3 keep the state to float32 accuracy; 2 (2^-17) are enough where the state
// only feeds D1, which reads it in bf16, and leave room for a fifth slot.
template <int DX, int DZ, int NT>
struct Cfg {
  static constexpr uint32_t XB = DX / 64 * BLK, ZB = DZ / 64 * BLK;
  static constexpr uint32_t SLOT = XB > ZB ? XB : ZB;
  static constexpr int NS = SLOT == BLK ? 8 : NT == 2 ? 5 : 4;
  static constexpr int NA = NS == 8 ? 2 : 1;                            // buffers of A, of U and of y's smaller terms
  static constexpr uint32_t RING = NS * SLOT;
  static constexpr uint32_t MID = RING, LO = MID + NA * XB, ZERO = LO + NA * XB;  // ZERO only with 64-wide y
  static constexpr uint32_t ST = NT == 2 ? LO : DX == 64 ? ZERO + BLK : ZERO;  // S: 128 rows x DZ bf16
  // at the walk's end: the middle terms' part of a 64-wide y's state lies in MID .. SUM_END, and the state leaves
  // through LEAVES on
  static constexpr uint32_t SUM_END = MID + (DX == 64 ? 64 * DZ * 4 : 0), LEAVES = DX == 64 ? LO : MID;
  static constexpr uint32_t WTAB = ST + ZB;                             // 130 x 8 bytes
  static constexpr uint32_t TAB = WTAB + 1040;                          // 132 + 32 floats
  static constexpr uint32_t BARS = TAB + 656;
  static constexpr uint32_t BYTES = BARS + 256 + 1024;
  // TMEM columns
  static constexpr uint32_t T_A = 0, T_D1 = NA * 128, T_D2 = T_D1 + DZ, T_U = T_D2 + DZ;
  static_assert(T_U + NA * DZ <= TMEM_COLS && BYTES <= 232448, "fits an SM");
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
  Link link;
};

// Barriers behind full[NS] and empty[NS].  A and P take turns where there are two A buffers: X may be a chunk
// ahead of the product that reads P.
enum { B_A = 0, B_A1, B_P, B_P1, B_K, B_K1, B_U, B_U1, B_O, B_DFREE, B_S, B_OSTAGED, B_STORED, B_SUM, B_DONE, B_COUNT };

template <int DX, int DZ, int NT, bool REV>
struct Walk {
  using G = Cfg<DX, DZ, NT>;
  static constexpr int PER = 3;                       // tiles of a chunk
  static constexpr int HC = DZ / 2;                   // columns of one X or Y warp
  static constexpr int CONV = 256;                    // threads that weigh y

  const Params& p;
  uint8_t* base;
  uint32_t sbase;
  uint64_t* full;
  uint64_t* empty;
  uint64_t* bars;
  uint32_t tmem;
  int warp, lane, seg, h, chunks;
  int64_t b, bh, len, s0, s1;

  // a^e; a^e as two bf16 terms, each twice; column factors of a block off the diagonal: a^(31-k), from the end a^k
  __device__ __forceinline__ uint32_t pw_at(int e) const { return sbase + G::TAB + 4 * e; }
  __device__ __forceinline__ float pw(int e) const { return lds_f(pw_at(e)); }
  __device__ __forceinline__ uint2 wt(int e) const { return lds_u2(sbase + G::WTAB + 8 * e); }
  __device__ __forceinline__ float4 cf4(int k) const { return lds_f4(sbase + G::TAB + 528 + 4 * k); }

  __device__ __forceinline__ int64_t first_token(int c) const { return s0 + int64_t(REV ? chunks - 1 - c : c) * C; }
  __device__ __forceinline__ int tokens(int c) const { return int(min(int64_t(C), s1 - first_token(c))); }
  __device__ __forceinline__ uint32_t slot(uint32_t n) const { return n % G::NS; }
  __device__ __forceinline__ bool wait(int which, int c) const { return warp_wait(&bars[which], c & 1); }
  __device__ __forceinline__ bool wait_turn(int which, int c) const {
    return warp_wait(&bars[which + c % G::NA], (c / G::NA) & 1);
  }
  __device__ __forceinline__ bool wait_full(uint32_t n) const { return warp_wait(&full[n % G::NS], (n / G::NS) & 1); }
  __device__ __forceinline__ void arrive(int which) const {
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars[which]);
  }

  // Places of a chunk's tiles in the ring's order y, x, z.
  __device__ __forceinline__ uint32_t tile_y(int c) const { return uint32_t(c) * PER; }
  __device__ __forceinline__ uint32_t tile_x(int c) const { return uint32_t(c) * PER + 1; }
  __device__ __forceinline__ uint32_t tile_z(int c) const { return uint32_t(c) * PER + PER - 1; }

  // ---- warp 0
  __device__ void load(const CUtensorMap* mx, const CUtensorMap* my, const CUtensorMap* mz) const {
    const bool leader = elect_one();
    uint32_t n = 0;
    bool ok = true;
    for (int c = 0; c < chunks && ok; ++c) {
      const int t0 = int(first_token(c));
      for (int i = 0; i < PER; ++i, ++n) {
        const int k = i == 0 ? 1 : i == PER - 1 ? 2 : 0;
        const uint32_t s = slot(n), r = n / G::NS;
        if (r > 0 && !warp_wait(&empty[s], (r - 1) & 1)) { ok = false; break; }
        if (leader) {
          const CUtensorMap* m = k == 0 ? mx : k == 1 ? my : mz;
          const int hh = h / (k == 0 ? p.gx : k == 1 ? p.gy : p.gz);
          const int blocks = (k == 2 ? DZ : DX) / 64;
          mbar_expect_tx(&full[s], uint32_t(blocks) * BLK);
          for (int blk = 0; blk < blocks; ++blk)
            tma_load_4d(base + s * G::SLOT + blk * BLK, m, &full[s], blk * 64, hh, t0, int(b));
        }
        __syncwarp();
      }
    }
    copies_landed<G::NS>(full, n);
  }

  // ---- warp 1.  A tile's slot is released by the last product that reads it (z's by the output's store).  With
  // two A buffers A of the next chunk goes first; with one it comes last.
  __device__ void mma(const bool leader) const {
    const uint32_t id_a = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(C >> 3) << 17) | (uint32_t(C >> 4) << 24);
    const uint32_t id_d = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | (uint32_t(DZ >> 3) << 17) |
                          (uint32_t(C >> 4) << 24);
    const uint32_t id_u = id_d | (1u << 15);
    const Desc d_s(sbase + G::ST, BLK);
    auto at = [&](uint32_t n) { return sbase + slot(n) * G::SLOT; };
    auto product_a = [&](int c) {
      if (!wait_full(tile_y(c)) || !wait_full(tile_x(c))) return false;
      tc_after();
      if (leader) {
        const Desc dx(at(tile_x(c)), 16), dy(at(tile_y(c)), 16);
#pragma unroll
        for (int kk = 0; kk < DX / 16; ++kk) {
          const uint32_t off = (kk >> 2) * BLK + (kk & 3) * 32;
          umma_bf16(tmem + G::T_A + uint32_t(c % G::NA) * 128, dx.at(off), dy.at(off), id_a, kk > 0);
        }
        umma_commit(&bars[B_A + c % G::NA]);
      }
      __syncwarp();
      return true;
    };
    if (chunks > 0 && !product_a(0)) return;
    for (int c = 0; c < chunks; ++c) {
      const bool more = c + 1 < chunks;
      if (G::NA == 2 && more && !product_a(c + 1)) return;
      if (!wait_full(tile_z(c)) || !wait_turn(B_K, c)) return;
      tc_after();
      const Desc dz(at(tile_z(c)), BLK);
      if (leader) {
        // small terms first, so that the accumulator drops the least
        const uint32_t yb = at(tile_y(c));
        const uint32_t mid = sbase + G::MID + uint32_t(c % G::NA) * G::XB, lo = sbase + G::LO + uint32_t(c % G::NA) * G::XB;
        const Desc dy(yb, DX == 64 ? mid - yb : BLK), d_mid(mid, BLK), d_lo(lo, DX == 64 ? sbase + G::ZERO - lo : BLK);
        if (NT == 3) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) umma_bf16(tmem + G::T_U + uint32_t(c % G::NA) * DZ, d_lo.at(kk * 2048), dz.at(kk * 2048), id_u, kk > 0);
        }
        if (DX == 128) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            umma_bf16(tmem + G::T_U + uint32_t(c % G::NA) * DZ, d_mid.at(kk * 2048), dz.at(kk * 2048), id_u, NT == 3 || kk > 0);
        }
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          umma_bf16(tmem + G::T_U + uint32_t(c % G::NA) * DZ, dy.at(kk * 2048), dz.at(kk * 2048), id_u, NT == 3 || DX == 128 || kk > 0);
        umma_commit(&bars[B_U + c % G::NA]);
        umma_commit(&empty[slot(tile_y(c))]);
      }
      __syncwarp();
      if (!wait_turn(B_P, c)) return;
      if (c > 0 && !wait(B_DFREE, c - 1)) return;
      tc_after();
      if (leader) {
        const uint32_t pa = tmem + G::T_A + uint32_t(c % G::NA) * 128;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)  // P of columns 0..63 and 64..127 lies where each half of A was
          umma_bf16_ta(tmem + G::T_D2, pa + (kk >> 2) * 64 + (kk & 3) * 8, dz.at(kk * 2048), id_d, kk > 0);
      }
      __syncwarp();
      if (!wait(B_S, c)) return;
      tc_after();
      if (leader) {
        const Desc dx(at(tile_x(c)), 16);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {  // 128 rows of S: all of x, or x twice
          const int xk = kk % (DX / 16);
          umma_bf16(tmem + G::T_D1, dx.at((xk >> 2) * BLK + (xk & 3) * 32), d_s.at(kk * 2048), id_d, kk > 0);
        }
        umma_commit(&empty[slot(tile_x(c))]);
        umma_commit(&bars[B_O]);
      }
      __syncwarp();
      if (G::NA == 1 && more && !product_a(c + 1)) return;
    }
  }

  // ---- X: row i of the chunk is TMEM lane i
  __device__ __forceinline__ bool scores(int c) const {
    const int q = warp & 3, half = (warp - 2) >> 2, i = q * 32 + lane;
    const uint32_t ta = tmem + G::T_A + uint32_t(c % G::NA) * 128 + (uint32_t(q * 32) << 16) + half * 64;
    const int n = tokens(c);
    if (!wait_turn(B_A, c)) return false;
    tc_after();
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int cb = half * 2 + g;      // block of 32 columns
      uint32_t pk[16];
      if (REV ? cb < q : cb > q) {
#pragma unroll
        for (int k = 0; k < 16; ++k) pk[k] = 0;
      } else {
        uint32_t r[32];
        tmem_ld32(ta + g * 32, r);
        const int lim = REV ? n - 32 * cb : 32;   // columns past the length
        if (cb != q && lim >= 32) {
          const float rf = pw(REV ? 32 * cb - i : i - 32 * cb - 31);
          const float2 rf2 = make_float2(rf, rf);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float4 w = cf4(4 * k);
            const float2 lo = __fmul2_rn(make_float2(w.x, w.y), rf2), hi = __fmul2_rn(make_float2(w.z, w.w), rf2);
            pk[2 * k] = pack2(__fmul2_rn(make_float2(__uint_as_float(r[4 * k]), __uint_as_float(r[4 * k + 1])), lo));
            pk[2 * k + 1] = pack2(__fmul2_rn(make_float2(__uint_as_float(r[4 * k + 2]), __uint_as_float(r[4 * k + 3])), hi));
          }
        } else {
          const uint32_t t = pw_at(REV ? 32 * cb - i : i - 32 * cb);  // masked lanes read what lies in front
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float v[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int j = 2 * k + e;
              const bool in = REV ? 32 * cb + j >= i && j < lim : 32 * cb + j <= i;
              v[e] = in ? __uint_as_float(r[j]) * lds_f(t + (REV ? 4 * j : -4 * j)) : 0.f;
            }
            pk[k] = pack_bf16(v[0], v[1]);
          }
        }
      }
      tmem_st16(ta + g * 16, pk);
    }
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    tc_before();
    arrive(B_P + c % G::NA);
    return true;
  }

  __device__ __forceinline__ bool output(int c) const {
    const int q = warp & 3, half = (warp - 2) >> 2, i = q * 32 + lane;
    const uint32_t row = uint32_t(q * 32) << 16;
    const int64_t t0 = first_token(c);
    const int n = tokens(c);
    if (!wait(B_O, c)) return false;
    tc_after();
    const float w = i < n ? p.scale * pw(REV ? n - 1 - i : i + 1) : 0.f, w2 = p.scale * p.z_scale;
    const uint32_t stage = sbase + slot(tile_z(c)) * G::SLOT;
#pragma unroll
    for (int g = 0; g < HC / 32; ++g) {
      uint32_t d1[32], d2[32];
      const int col = half * HC + g * 32;
      tmem_ld32_nowait(tmem + G::T_D1 + row + col, d1);
      tmem_ld32_nowait(tmem + G::T_D2 + row + col, d2);
      tmem_wait_ld();
      if (g == HC / 32 - 1) {
        tc_before();
        arrive(B_DFREE);
      }
      float2 o[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        o[k] = __ffma2_rn(make_float2(w, w), make_float2(__uint_as_float(d1[2 * k]), __uint_as_float(d1[2 * k + 1])),
                          __fmul2_rn(make_float2(w2, w2), make_float2(__uint_as_float(d2[2 * k]), __uint_as_float(d2[2 * k + 1]))));
        if (i >= n) o[k] = make_float2(0.f, 0.f);
      }
      if (p.out_f32) {
        if (t0 + i < p.L) {
          float* dst = static_cast<float*>(p.out) + ((b * p.L + t0 + i) * p.H + h) * p.dz + col;
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (col + 4 * k < p.dz)
              *reinterpret_cast<float4*>(dst + 4 * k) = make_float4(o[2 * k].x, o[2 * k].y, o[2 * k + 1].x, o[2 * k + 1].y);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t v[4] = {pack2(o[4 * k]), pack2(o[4 * k + 1]), pack2(o[4 * k + 2]), pack2(o[4 * k + 3])};
          // 128-wide: a 128-byte row of the half's block; 64-wide: a 64-byte row of the warp's own 2 KB
          const uint32_t a = DZ == 128 ? half * BLK + uint32_t(i) * 128 + (uint32_t((g * 4 + k) ^ (i & 7)) << 4)
                                       : uint32_t(q * 2 + half) * 2048 + uint32_t(lane) * 64 + (uint32_t(k ^ ((lane >> 1) & 3)) << 4);
          sts128(stage + a, v);
        }
      }
    }
    fence_async();
    // The store warp has seen the chunk before: with eight slots X could otherwise stage two more chunks while that
    // warp waits for a slow store, and a barrier two phases ahead looks as if it had not moved.
    if (c > 0 && !wait(B_STORED, c - 1)) return false;
    arrive(B_OSTAGED);
    return true;
  }

  // ---- X: whole chunks past the length are zeros
  __device__ void zeros() const {
    const int64_t seg0 = int64_t(seg) * p.seg_len;
    const int64_t z0 = max(seg0, s0 + int64_t(chunks) * C), z1 = min(p.L, seg0 + p.seg_len);
    const int per = p.dz / 8;
    for (int64_t k = int(threadIdx.x) - 64; k < (z1 - z0) * per; k += 256) {
      const int64_t at = ((b * p.L + z0 + k / per) * p.H + h) * p.dz + (k % per) * 8;
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

  // ---- warp 18: stores the staged output and hands z's slot back
  __device__ void store(const CUtensorMap* mo) const {
    for (int c = 0; c < chunks; ++c) {
      const uint32_t nz = tile_z(c);
      if (!wait(B_OSTAGED, c)) return;
      arrive(B_STORED);
      if (lane == 0) {
        if (!p.out_f32) {
          const int t0 = int(first_token(c));
          const uint32_t src = sbase + slot(nz) * G::SLOT;
          for (int k = 0; k < 8; ++k) {
            const int q = k >> 1, half = k & 1;
            if (t0 + q * 32 < p.L && half * HC < p.dz)
              tma_store_4d(mo, src + (DZ == 128 ? half * BLK + q * 4096 : k * 2048), half * HC, h, t0 + q * 32, int(b));
          }
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        }
        mbar_arrive(&empty[slot(nz)]);
      }
      __syncwarp();
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }

  // ---- the weighted y of chunk c as bf16 terms (this thread's 16-byte pieces); z's rows past the length
  __device__ __forceinline__ bool weigh(int c, int tid) const {
    const uint32_t ny = tile_y(c), nz = tile_z(c);
    const int n = tokens(c);
    const uint32_t yb = sbase + slot(ny) * G::SLOT, buf = sbase + uint32_t(c % G::NA) * G::XB;
    if (!wait_turn(B_A, c)) return false;
    constexpr int PIECES = DX / 64 * 1024 / CONV, BATCH = PIECES < 4 ? PIECES : 4;
#pragma unroll
    for (int k0 = 0; k0 < PIECES; k0 += BATCH) {
      uint32_t v[BATCH][4];
#pragma unroll
      for (int k = 0; k < BATCH; ++k) lds128(yb + uint32_t(tid + CONV * (k0 + k)) * 16, v[k]);
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        const uint32_t u = uint32_t(tid + CONV * (k0 + k)), off = u * 16;
        const int j = int(u >> 3) & 127;       // token
        uint32_t hi[4], mid[4], lo[4];
        const int e = REV ? j + 1 : n - 1 - j;
        if (j >= n) v[k][0] = v[k][1] = v[k][2] = v[k][3] = 0;  // what lies there may be anything
        if (NT == 2) {
          // in packed bf16: hi = rn(y w1), its error y w1 - hi exactly, mid = rn(that + y w2)
          const uint2 w = wt(j < n ? e : 0);
          const __nv_bfloat162 w1 = *reinterpret_cast<const __nv_bfloat162*>(&w.x);
          const __nv_bfloat162 w2 = *reinterpret_cast<const __nv_bfloat162*>(&w.y);
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const __nv_bfloat162 y = *reinterpret_cast<const __nv_bfloat162*>(&v[k][m]);
            const __nv_bfloat162 h = __hmul2_rn(y, w1);
            const __nv_bfloat162 r = __hfma2(y, w2, __hfma2(y, w1, __hneg2(h)));
            hi[m] = *reinterpret_cast<const uint32_t*>(&h);
            mid[m] = *reinterpret_cast<const uint32_t*>(&r);
          }
        } else {
          const float w = pw(j < n ? e : 0);
          const float2 w2 = make_float2(w, w), minus = make_float2(-1.f, -1.f);
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            float2 a = __fmul2_rn(unpack2(v[k][m]), w2);
            hi[m] = pack2(a);
            a = __ffma2_rn(unpack2(hi[m]), minus, a);
            mid[m] = pack2(a);
            a = __ffma2_rn(unpack2(mid[m]), minus, a);
            lo[m] = pack2(a);
          }
        }
        sts128(yb + off, hi);
        sts128(buf + G::MID + off, mid);
        if (NT == 3) sts128(buf + G::LO + off, lo);
      }
    }
    if (n < C) {
      if (!wait_full(nz)) return false;
      const uint32_t zero[4] = {0, 0, 0, 0};
      for (uint32_t u = uint32_t(tid); u < G::ZB / 16; u += CONV)
        if ((int(u >> 3) & 127) >= n) sts128(sbase + slot(nz) * G::SLOT + u * 16, zero);
    }
    fence_async();
    arrive(B_K + c % G::NA);
    return true;
  }

  // ---- Y: lane i of TMEM is row i of the state (64-wide y: row i % 64)
  __device__ void state() const {
    const int q = warp & 3, half = (warp - 10) >> 2, i = q * 32 + lane;
    const int tid = int(threadIdx.x) - 320;
    const uint32_t row = uint32_t(q * 32) << 16;
    const int64_t n_state = int64_t(p.dx) * p.dz;
    float2 s[HC / 2];
    chain_begin(p.link);    // only the state may come from the launches in front
    const float* st = p.start ? p.start + bh * p.start_stride + int64_t(seg) * n_state : nullptr;
    if (st && !p.start_t && q * 32 < DX) {
      // through where the terms of y and S will be
      static_assert(G::MID + DX * DZ * 4 <= (DX == 64 && NT == 3 ? G::ZERO : G::ST + G::ZB), "the states fit");
      const int r0 = q * 32, c0 = half * HC;
      state_load<HC>(s, sbase + G::MID + uint32_t(q * 2 + half) * HC * 128, st + int64_t(r0) * p.dz + c0, p.dz,
                     p.dx - r0, p.dz - c0);
    } else {
#pragma unroll
      for (int k = 0; k < HC; ++k) {
        const int c = half * HC + k;
        const float v = st && i < p.dx && i < DX && c < p.dz ? __ldcg(st + int64_t(c) * p.dx + i) : 0.f;
        if (k & 1) s[k / 2].y = v;
        else s[k / 2].x = v;
      }
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");   // all Y: the states have left where y's terms go
    if (G::NA == 2 && chunks > 0 && !weigh(0, tid)) return;
    for (int c = 0; c < chunks; ++c) {
      if (G::NA == 1 && !weigh(c, tid)) return;
      {
        // S as the bf16 operand of D1, once D1 of the chunk before has read its own
        if (c > 0 && !wait(B_O, c - 1)) return;
#pragma unroll
        for (int k = 0; k < HC / 8; ++k) {
          const uint32_t w[4] = {pack2(s[4 * k]), pack2(s[4 * k + 1]), pack2(s[4 * k + 2]), pack2(s[4 * k + 3])};
          const int ch = half * (HC / 8) + k;  // 16-byte piece of the row
          sts128(sbase + G::ST + uint32_t(ch >> 3) * BLK + uint32_t(i) * 128 + (uint32_t((ch & 7) ^ (i & 7)) << 4), w);
        }
        fence_async();
        arrive(B_S);
      }
      // with two buffers y of the next chunk is weighed while this one's U is formed
      if (G::NA == 2 && c + 1 < chunks && !weigh(c + 1, tid)) return;
      if (!wait_turn(B_U, c)) return;
      tc_after();
      const float an = pw(tokens(c));
      const float2 an2 = make_float2(an, an), zs = make_float2(p.z_scale, p.z_scale);
#pragma unroll
      for (int g = 0; g < HC / 16; ++g) {
        uint32_t u[16];
        tmem_ld16_nowait(tmem + G::T_U + uint32_t(c % G::NA) * DZ + row + half * HC + g * 16, u);
        tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 8; ++k)
          s[g * 8 + k] = __ffma2_rn(an2, s[g * 8 + k],
                                    __fmul2_rn(zs, make_float2(__uint_as_float(u[2 * k]), __uint_as_float(u[2 * k + 1]))));
      }
      tc_before();
    }
    // the state behind the whole walk leaves
    float* end = p.end && seg == (REV ? 0 : p.segs - 1) ? p.end + bh * n_state : nullptr;
    if (!end) return;
    if (DX == 64) {
      // rows 64..127 hold the middle terms' part; the ring is done with
      float2* sum = reinterpret_cast<float2*>(base + G::MID);
      static_assert(NT == 2 || G::SUM_END <= G::ST, "the sum fits");
      if (i >= 64) {
#pragma unroll
        for (int k = 0; k < HC / 2; ++k) sum[(i - 64) + (half * (HC / 2) + k) * 64] = s[k];
      }
      arrive(B_SUM);
      if (!mbar_wait_warp(&bars[B_SUM], 0)) return;
      if (i < 64) {
#pragma unroll
        for (int k = 0; k < HC / 2; ++k) s[k] = __fadd2_rn(s[k], sum[i + (half * (HC / 2) + k) * 64]);
      }
      // 128-wide z: the sum takes both terms' places, the second of which the state leaves through; no warp writes
      // there before all have read
      if constexpr (G::SUM_END > G::LEAVES) {
        arrive(B_SUM);
        if (!mbar_wait_warp(&bars[B_SUM], 1)) return;
      }
    }
    const int r0 = q * 32, c0 = half * HC;
    if (r0 < DX) {
      // (all products that read y's terms are done; D1 of the last chunk may still read S)
      static_assert(NT == 2 || G::LEAVES + DX * DZ * 4 <= G::ST, "the states fit");
      state_store<HC>(s, sbase + G::LEAVES + uint32_t(q * 2 + half) * HC * 128, end + int64_t(r0) * p.dz + c0, p.dz,
                      p.dx - r0, p.dz - c0);
    }
  }
};

template <int DX, int DZ, int NT, bool REV>
__global__ void __launch_bounds__(THREADS, 1)
walk_tc_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmY,
               const __grid_constant__ CUtensorMap tmZ, const __grid_constant__ CUtensorMap tmO, const Params p) {
  using W = Walk<DX, DZ, NT, REV>;
  using G = typename W::G;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint2* wt = reinterpret_cast<uint2*>(base + G::WTAB);
  float* tab = reinterpret_cast<float*>(base + G::TAB);
  uint64_t* full = reinterpret_cast<uint64_t*>(base + G::BARS);
  uint64_t* bars = full + 2 * G::NS;
  static_assert((2 * G::NS + B_COUNT) * 8 + 4 <= 256, "barriers fit");
  uint32_t* tslot = reinterpret_cast<uint32_t*>(bars + B_COUNT);
  W w{p, base, smem_u32(base), full, full + G::NS, bars, 0u, int(threadIdx.x >> 5),
      int(threadIdx.x & 31)};
  w.seg = int(blockIdx.x % p.segs);
  w.bh = blockIdx.x / p.segs;
  w.b = w.bh / p.H;
  w.h = int(w.bh % p.H);
  w.len = row_length(p.lengths, w.b, p.L);
  w.s0 = min(w.len, int64_t(w.seg) * p.seg_len);
  w.s1 = min(w.len, w.s0 + p.seg_len);
  w.chunks = int((w.s1 - w.s0 + C - 1) / C);

  const float l2 = log2_decay(p.log_decay[w.h]);
  if (threadIdx.x <= C) {
    const float a = exp2f(l2 * float(threadIdx.x));
    const float a1 = __bfloat162float(__float2bfloat16_rn(a));
    tab[threadIdx.x] = a;
    wt[threadIdx.x] = make_uint2(pack_bf16(a1, a1), pack_bf16(a - a1, a - a1));
  }
  if (threadIdx.x < 32) tab[132 + threadIdx.x] = exp2f(l2 * float(REV ? threadIdx.x : 31 - threadIdx.x));
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2 * G::NS; ++s) mbar_init(&full[s], 1);
    for (int k = 0; k < B_COUNT; ++k) mbar_init(&bars[k], k <= B_A1 || k == B_U || k == B_U1 || k == B_O || k == B_STORED || k == B_DONE ? 1 : 8);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmX)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmY)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmZ)) : "memory");
  }
  if (DX == 64 && NT == 3) {
    for (uint32_t i = threadIdx.x * 16; i < BLK; i += THREADS * 16)
      *reinterpret_cast<uint4*>(base + G::ZERO + i) = make_uint4(0, 0, 0, 0);
    fence_async();
  }
  if (w.warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tslot)), "r"(TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_before();
  __syncthreads();
  tc_after();
  w.tmem = *tslot;

  if (w.warp == 0) {
    w.load(&tmX, &tmY, &tmZ);
  } else if (w.warp == 1) {
    const bool leader = elect_one();
    w.mma(leader);
    products_done(&bars[B_DONE], leader);
  } else if (w.warp < 10) {
    {
      bool ok = true;
      // with one A buffer the output goes first: the product that reads P waits for its accumulators
      for (int c = 0; c < w.chunks && ok; ++c) {
        if (G::NA == 1 && c > 0) ok = w.output(c - 1);
        ok = ok && w.scores(c);
        if (G::NA == 2 && c > 0) ok = ok && w.output(c - 1);
      }
      if (ok && w.chunks > 0) w.output(w.chunks - 1);
      w.zeros();
    }
  } else if (w.warp < 18) {
    w.state();
  } else if (w.warp == 18) {
    w.store(&tmO);
  }
  tc_before();
  __syncthreads();
  if (w.warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(w.tmem), "r"(TMEM_COLS));
  chain_end();
}

bool fits(const Tensor& t, int64_t B, int64_t L) {
  auto ok = [](int64_t n, int64_t s) { return n <= 1 || (s > 0 && s % 8 == 0 && s < (int64_t(1) << 38)); };
  return t.d % 8 == 0 && t.d <= 128 && aligned(t.p, 16) && ok(t.heads, t.s.head) && ok(L, t.s.token) && ok(B, t.s.batch);
}

// The output as (D, H, L, B), a box of 32 tokens and one X warp's columns, in the swizzle that it is staged in.
bool make_store_map(CUtensorMap* m, const Job& j, int cols) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t d = cuuint64_t(j.z.d);
  cuuint64_t dims[4] = {d, cuuint64_t(j.H), cuuint64_t(j.L), cuuint64_t(j.B)};
  cuuint64_t st[3] = {d * 2, d * 2 * j.H, d * 2 * j.H * cuuint64_t(j.L)};
  cuuint32_t box[4] = {cuuint32_t(cols), 1, 32, 1}, es[4] = {1, 1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, j.out, dims, st, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DX, int DZ, int NT, bool REV>
int launch(const Job& j, const Link& link, cudaStream_t s) {
  static int limit = 0;
  using G = Cfg<DX, DZ, NT>;
  CUtensorMap mx, my, mz, mo = {};
  if (!make_tensor_map(&mx, j.x, j.B, j.L) || !make_tensor_map(&my, j.y, j.B, j.L) ||
      !make_tensor_map(&mz, j.z, j.B, j.L) || (!j.out_f32 && !make_store_map(&mo, j, DZ / 2))) {
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
  p.link = link;
  p.gx = j.H / j.x.heads;
  p.gy = j.H / j.y.heads;
  p.gz = j.H / j.z.heads;
  PGF_CUDA(ensure_dynamic_smem(walk_tc_kernel<DX, DZ, NT, REV>, G::BYTES, limit));
  PGF_CUDA(launch_link(link, walk_tc_kernel<DX, DZ, NT, REV>, unsigned(j.B * j.H * j.segs), THREADS, G::BYTES, s, mx, my, mz,
                       mo, p));
  PGF_LAUNCH_CHECK();
  return PGF_OK;
}

template <int NT, bool REV>
int dispatch(const Job& j, const Link& l, cudaStream_t s) {
  if (j.y.d <= 64) return j.z.d <= 64 ? launch<64, 64, NT, REV>(j, l, s) : launch<64, 128, NT, REV>(j, l, s);
  return j.z.d <= 64 ? launch<128, 64, NT, REV>(j, l, s) : launch<128, 128, NT, REV>(j, l, s);
}

}  // namespace

bool tc_fits(const Tensor& t, int64_t B, int64_t L) { return fits(t, B, L); }
int tc_walk(const Job& j, const Link& l, cudaStream_t s) {
  if (j.end) return j.rev ? dispatch<3, true>(j, l, s) : dispatch<3, false>(j, l, s);
  return j.rev ? dispatch<2, true>(j, l, s) : dispatch<2, false>(j, l, s);
}

}  // namespace da

int decay_tc_fault() { return take_tc_fault(); }

}  // namespace pgf
