// Shared parts of the gated delta rule kernels (plastic_*.cu): the argument block, fragments of the
// tensor-core products and the staging of token tiles.
//
// The rule, per batch row and value head, with a state S of (dk, dv):
//   u_t = beta_t (v_t - e^{g_t} S_{t-1}^T k_t),  S_t = e^{g_t} S_{t-1} + k_t u_t^T,  o_t = scale S_t^T q_t
// and over a chunk of C = 64 tokens with G = cumsum(g), Gamma_ij = e^{G_i - G_j} (i >= j):
//   T = (I + A)^{-1},  A_ij = beta_i Gamma_ij k_i.k_j (j < i),   P_ij = scale Gamma_ij q_i.k_j (j <= i)
//   U = T diag(beta) (V - diag(e^G) K S0),   O = scale diag(e^G) Q S0 + P U,
//   S' = e^{G_C} S0 + (diag(e^{G_C - G}) K)^T U
//
// Products run on tf32 tensor instructions (16x8x8, 32-bit sums).  bf16 and fp16 values are exact in tf32; a 32-bit
// operand is split into hi + lo tf32 parts (22 bits), so a product with one 16-bit operand takes two instructions
// and one of two 32-bit operands three (lo x lo, 2^-22 of the product, is dropped).  Everything the state, its
// cotangent and the gate gradients depend on is computed this way; only the last product before a bf16 output uses
// the hi parts alone (2^-12 before a rounding of 2^-9).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace bsx {
namespace plastic {

constexpr int kC = 64;           // tokens of a chunk
constexpr size_t kMaxSmem = 227 * 1024;   // dynamic shared memory of a block
constexpr int kVec = 5 * kC;     // e^G, e^{G_C-G}, beta, G (high part), G (low part)

struct Args {
  const void *q, *k, *v;
  const float *g, *beta, *initial;
  const int32_t* lengths;
  int64_t qs[3], ks[3], vs[3], gs[3], bs[3];  // batch, token, head strides in elements
  int64_t T;
  int B, Hk, Hv, dk, dv, NC;
  float scale;
  // per (row, head, chunk): T, P, A / beta (64 x 64 each; entries above the diagonal blocks are not written), vectors
  float *Tm, *Pm, *Bm, *vec;
  // per (row, head, chunk), transposed: state before the chunk (dv, DK), U (dv, 64); backward only
  float *Sn, *U;
  void* o;
  float* state;
  // backward
  const void* dout;
  const float* dstate;
  float *dS, *dY;
  void *dq, *dk_, *dv_;
  float *dg, *dbeta, *dinitial;
  float *dq32, *dk32;     // per value head, when heads share keys
  bool vec_qk, vec_v, vec_do;
};

template <typename E> __device__ __forceinline__ float to_f(E x);
template <> __device__ __forceinline__ float to_f<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }
template <typename E> __device__ __forceinline__ E from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16(x); }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half(x); }

template <typename E> struct IsExact { static constexpr bool value = sizeof(E) == 2; };
// Types whose own rounding (2^-9) hides that of one tf32 operand (2^-12): the last product before an output of such a
// type takes the hi parts alone.
template <typename E> struct IsShort { static constexpr bool value = false; };
template <> struct IsShort<__nv_bfloat16> { static constexpr bool value = true; };

// Two neighbouring elements of shared memory as floats (p: even element offset, 2-element aligned).
__device__ __forceinline__ float2 pair(const float* p) { return *reinterpret_cast<const float2*>(p); }
__device__ __forceinline__ float2 pair(const __nv_bfloat16* p) {
  const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 pair(const __half* p) {
  return __half22float2(*reinterpret_cast<const __half2*>(p));
}

__device__ __forceinline__ void mma(float* c, const float* a, float b0, float b1) {
  asm(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(__float_as_uint(a[0])), "r"(__float_as_uint(a[1])), "r"(__float_as_uint(a[2])), "r"(__float_as_uint(a[3])),
        "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}

// Nearest tf32 value.
__device__ __forceinline__ float tf32(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return __uint_as_float(r);
}
// x = hi + lo with hi the nearest tf32 value (integer form: a NaN may lose itself in hi, but then lo is NaN).
__device__ __forceinline__ void split(float x, float& hi, float& lo) {
  hi = __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xffffe000u);
  lo = x - hi;
}
__device__ __forceinline__ void split4(const float* x, float* hi, float* lo) {
#pragma unroll
  for (int i = 0; i < 4; ++i) split(x[i], hi[i], lo[i]);
}
// The rows x columns of an accumulator tile (row g, columns 2t, 2t+1; row g + 8) are those of a 16x8 left operand
// whose inner index is taken in the order (0, 2, 4, 6, 1, 3, 5, 7): an accumulator is the next product's operand
// without leaving its registers, and the right operand's values are neighbours in memory.
__device__ __forceinline__ void as_left(const float* c, float* a) {
  a[0] = c[0];
  a[1] = c[2];
  a[2] = c[1];
  a[3] = c[3];
}

// c[n] += a b[n] for N tiles, a 32-bit (hi, lo), b exact or 32-bit: the small terms of all tiles first, so that
// instructions that follow each other do not wait for each other's sums.
template <bool BEXACT, int N>
__device__ __forceinline__ void mma_split(float (*c)[4], const float* ahi, const float* alo, const float2* b) {
  if (BEXACT) {
#pragma unroll
    for (int n = 0; n < N; ++n) mma(c[n], alo, b[n].x, b[n].y);
#pragma unroll
    for (int n = 0; n < N; ++n) mma(c[n], ahi, b[n].x, b[n].y);
  } else {
    float2 h[N], l[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      split(b[n].x, h[n].x, l[n].x);
      split(b[n].y, h[n].y, l[n].y);
    }
#pragma unroll
    for (int n = 0; n < N; ++n) mma(c[n], alo, h[n].x, h[n].y);
#pragma unroll
    for (int n = 0; n < N; ++n) mma(c[n], ahi, l[n].x, l[n].y);
#pragma unroll
    for (int n = 0; n < N; ++n) mma(c[n], ahi, h[n].x, h[n].y);
  }
}

__device__ __forceinline__ void cp16(void* dst, const void* src, bool ok) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
  const int n = ok ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Stages `rows` (of 64) token rows x `cols` (of COLS) of a (token, column) tile; the rest is zero.  vec: rows start on
// 16-byte boundaries and cols is a multiple of a 16-byte stretch.
template <typename E>
__device__ __forceinline__ void stage(E* sm, int pitch, const E* src, int64_t stride, int rows, int cols, int colspad,
                                      bool vec, int tid, int nthr) {
  if (vec) {
    constexpr int V = 16 / sizeof(E);
    const int per = colspad / V;
    for (int i = tid; i < kC * per; i += nthr) {
      const int r = i / per, c = (i - r * per) * V;
      const bool ok = r < rows && c < cols;
      cp16(sm + r * pitch + c, ok ? src + r * stride + c : src, ok);
    }
  } else {
    for (int i = tid; i < kC * colspad; i += nthr) {
      const int r = i / colspad, c = i - r * colspad;
      sm[r * pitch + c] = (r < rows && c < cols) ? src[r * stride + c] : from_f<E>(0.f);
    }
  }
}
// Stages the lower block triangle (16x16 blocks) of a 64x64 matrix.
__device__ __forceinline__ void stage_lower(float* sm, int pitch, const float* src, int tid, int nthr) {
  for (int i = tid; i < kC * 16; i += nthr) {
    const int r = i >> 4, c = (i & 15) * 4;
    if (c < ((r >> 4) + 1) * 16) cp16(sm + r * pitch + c, src + r * kC + c, true);
  }
}

__device__ __forceinline__ int row_length(const Args& a, int b) {
  if (!a.lengths) return (int)a.T;
  const int64_t n = a.lengths[b];
  return (int)(n < 0 ? 0 : (n > a.T ? a.T : n));
}

// Launchers (one translation unit per kernel family).
int launch_prepare(const Args& a, int dtype, bool backward, cudaStream_t st);
int launch_scan(const Args& a, int dtype, bool save, cudaStream_t st);
int launch_backward_scan(const Args& a, int dtype, cudaStream_t st);
int launch_backward_chunks(const Args& a, int dtype, cudaStream_t st);

}  // namespace plastic
}  // namespace bsx
