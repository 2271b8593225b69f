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
// and one of two 32-bit operands three (lo x lo, 2^-22 of the product, is dropped).  The products with bf16 keys and
// queries that carry the state run on bf16 instructions instead (16x8x16, the same time for twice the depth): the 32-bit
// operand is then three bf16 parts (24 bits), three instructions where tf32 takes four, and the bf16 operand goes in as
// it lies in memory.  Everything the state, its cotangent and the gate gradients depend on is computed this way; only
// products that go straight into a bf16 output take fewer parts (2^-12 or 2^-17 before a rounding of 2^-9).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "bulk_copy.cuh"
#include "common.cuh"

namespace bsx {
namespace plastic {

constexpr int kC = 64;           // tokens of a chunk
constexpr size_t kMaxSmem = 227 * 1024 - 64;   // dynamic shared memory of a block, beside its few static bytes
constexpr int kVec = 5 * kC;     // e^G, e^{G_C-G}, beta, G (high part), G (low part)
constexpr int kTri = 36 * 64;    // lower triangle of a 64x64 matrix: 8x8 tiles by rows, each row-major
constexpr int kRecord = 2 * kTri + kVec;   // T, P and the vectors of a chunk, one contiguous record

struct Args {
  const void *q, *k, *v;
  const float *g, *beta, *initial;
  const int32_t* lengths;
  int64_t qs[3], ks[3], vs[3], gs[3], bs[3];  // batch, token, head strides in elements
  int64_t T;
  int B, Hk, Hv, dk, dv, NC;
  float scale;
  // per (row, key head, chunk): K and Q tiles, 64 rows of DK + 8 elements each, as they lie in shared memory
  void* kq;
  // per (row, value head, chunk): T, P and vectors (kRecord floats); A / beta (kTri), backward only
  float *rec, *Bm;
  // per (row, head, chunk), transposed: state before the chunk (dv rows of DK + 4), U (dv rows of 68); backward only.  The
  // rows lie as in shared memory, so that a block of them is one copy; dS (after the chunk) and dY likewise
  float *Sn, *U;
  void* o;
  float* state;
  // backward
  uint32_t* taken;      // chunks that blocks took beyond their first; cleared by the preparing kernel
  const void* dout;
  const float* dstate;
  float *dS, *dY;
  void *dq, *dk_, *dv_;
  float *dg, *dbeta, *dinitial;
  float *dq32, *dk32;     // per value head, when heads share keys
  bool four_do, four_v;   // dO, V: four neighbouring elements can be loaded together
  bool vec_qk;            // rows of q and k start on 16-byte boundaries and are whole 16-byte stretches
};

constexpr int kPU = kC + 4;

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
// (used where the tiles are first read, by the kernel that packs them)
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
// Place of 8x8 tile (row tile n, column tile k <= n) in a packed lower triangle.
__device__ __forceinline__ constexpr int tri(int n, int k) { return (n * (n + 1) / 2 + k) * 64; }

// Waits for the bytes of a stage; false when the bounded wait ran out (the caller then spoils its results with NaN).
__device__ __forceinline__ bool stage_wait(uint64_t* bar, uint32_t parity) {
  for (uint32_t i = 0; i < (1u << 20); ++i)
    if (mbar_try_wait(bar, parity)) return true;
  return false;
}

// Operand tiles (16 value columns x 8) handed from one warp of a group to the others, already split: 1 KB a tile, the
// four registers of the left operand together (anything else costs moves).
__device__ __forceinline__ void put_split(float4* base, int tile, int lane, const float* c) {
  float h[4], l[4];
  split4(c, h, l);
  base[tile * 64 + lane] = make_float4(h[0], h[2], h[1], h[3]);
  base[tile * 64 + 32 + lane] = make_float4(l[0], l[2], l[1], l[3]);
}
__device__ __forceinline__ void get_split(const float4* base, int tile, int lane, float* hi, float* lo) {
  const float4 x = base[tile * 64 + lane], y = base[tile * 64 + 32 + lane];
  hi[0] = x.x; hi[1] = x.y; hi[2] = x.z; hi[3] = x.w;
  lo[0] = y.x; lo[1] = y.y; lo[2] = y.z; lo[3] = y.w;
}

// The same in three bf16 parts, two tiles (16 inner entries) together: 1.5 KB, each part the four registers of a left
// operand of the bf16 instruction (first tile in .x .y, second in .z .w).
struct Parts { uint32_t w[3]; };     // a pair of neighbouring entries
__device__ __forceinline__ Parts parts_of(float x0, float x1) {
  Parts p;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(p.w[i]) : "f"(x1), "f"(x0));
    if (i < 2) {
      x0 -= __uint_as_float(p.w[i] << 16);
      x1 -= __uint_as_float(p.w[i] & 0xffff0000u);
    }
  }
  return p;
}
__device__ __forceinline__ void put_parts(float4* base, int tile, int lane, const float* c) {
  const Parts a = parts_of(c[0], c[1]), b = parts_of(c[2], c[3]);
  uint2* o = reinterpret_cast<uint2*>(base + (tile >> 1) * 96 + lane) + (tile & 1);
#pragma unroll
  for (int i = 0; i < 3; ++i) o[i * 64] = make_uint2(a.w[i], b.w[i]);
}
__device__ __forceinline__ uint4 get_part(const float4* base, int pair, int part, int lane) {
  return reinterpret_cast<const uint4*>(base)[pair * 96 + part * 32 + lane];
}
__device__ __forceinline__ void mma16(float* c, const uint4& a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// s^T times the transposed (token, key row) tile X for token tiles own[0], own[1], s in parts: large and small sums; only
// the first two parts with TWO.
template <int DK, int PK, bool TWO>
__device__ __forceinline__ void state_times(float (*h)[4], float (*l)[4], const uint4* a, const __nv_bfloat16* X, int kp,
                                            const int* own, int g, int t) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const uint32_t* x = reinterpret_cast<const uint32_t*>(X + (own[e] * 8 + g) * PK + kp * 16) + t;
    const uint32_t b0 = x[0], b1 = x[4];
    if (!TWO) mma16(l[e], a[2], b0, b1);
    mma16(l[e], a[1], b0, b1);
    mma16(h[e], a[0], b0, b1);
  }
}
// u (16 tokens of it, in parts) times tiles n = 0 .. N - 1 of a (token, key row) tile at `at`.
template <int N, int PK>
__device__ __forceinline__ void update_state(float (*h)[4], float (*l)[4], const uint4* a, const __nv_bfloat16* at, int lane) {
  const int row = (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
  for (int n = 0; n < N; n += 2) {
    uint32_t r[4];
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_u32(at + row * PK + n * 8 + (lane >> 4) * 8)) : "memory");
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      mma16(l[n + m], a[2], r[2 * m], r[2 * m + 1]);
      mma16(l[n + m], a[1], r[2 * m], r[2 * m + 1]);
      mma16(h[n + m], a[0], r[2 * m], r[2 * m + 1]);
    }
  }
}

// Right-operand tiles from a (row, column) tile in shared memory: N 8x8 tiles whose rows are the outer index (pairs of
// neighbouring columns) ...
__device__ __forceinline__ float2 unpack(uint32_t w, const __nv_bfloat16*) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack(uint32_t w, const __half*) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// ... and N tiles side by side whose rows are the inner index (pairs of neighbouring rows).
template <int N, typename E>
__device__ __forceinline__ void tiles_by_row(float2* b, const E* at, int pitch, int lane) {
  if constexpr (sizeof(E) == 2) {
    uint32_t r[4];
    const uint32_t addr = smem_u32(at + (lane & 7) * pitch + ((lane >> 3) % N) * 8);
    if constexpr (N == 4)
      asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                   : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
    else if constexpr (N == 2)
      asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
    else
      asm volatile("ldmatrix.sync.aligned.m8n8.x1.trans.shared.b16 {%0}, [%1];" : "=r"(r[0]) : "r"(addr) : "memory");
#pragma unroll
    for (int n = 0; n < N; ++n) b[n] = unpack(r[n], at);
  } else {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < N; ++n) b[n] = make_float2(at[2 * t * pitch + n * 8 + g], at[(2 * t + 1) * pitch + n * 8 + g]);
  }
}

// c (sum of the small terms) and ch (sum of the large ones) += a b, a given as hi + lo.  The two sums are kept apart
// because the tensor unit cuts its sums: each is cut relative to its own size.
template <bool BEXACT>
__device__ __forceinline__ void mma_apart(float* ch, float* cl, const float* hi, const float* lo, float2 b) {
  if (BEXACT) {
    mma(cl, lo, b.x, b.y);
    mma(ch, hi, b.x, b.y);
  } else {
    float h0, l0, h1, l1;
    split(b.x, h0, l0);
    split(b.y, h1, l1);
    mma(cl, lo, h0, h1);
    mma(ch, hi, h0, h1);
    mma(cl, hi, l0, l1);
  }
}
// Values of a (token, column) array of global memory for this warp's two token tiles, in accumulator order; those past the
// sequence's end or the last column are zero.  row0: the chunk's first token, column g of the group's first.
template <typename E>
__device__ __forceinline__ void fetch_own(E (*x)[4], const E* row0, int64_t stride, const int* own, int t, int left, bool in0,
                                          bool in1) {
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int tok = own[e] * 8 + 2 * t + j;
      const E* p = row0 + tok * stride;
      x[e][j] = tok < left && in0 ? p[0] : from_f<E>(0.f);
      x[e][2 + j] = tok < left && in1 ? p[8] : from_f<E>(0.f);
    }
}
__device__ __forceinline__ void clear(float* c) { c[0] = c[1] = c[2] = c[3] = 0.f; }

__device__ __forceinline__ int row_length(const Args& a, int b) {
  if (!a.lengths) return (int)a.T;
  const int64_t n = a.lengths[b];
  return (int)(n < 0 ? 0 : (n > a.T ? a.T : n));
}

// Barrier of the four warps of a group.
__device__ __forceinline__ void group_sync(int grp) { asm volatile("bar.sync %0, 128;" ::"r"(grp + 1) : "memory"); }

int scan_groups(const Args& a, int sms);   // groups of 16 value columns to a block (plastic_scan.cu)

// Launchers (one translation unit per kernel family).
int launch_prepare(const Args& a, int dtype, bool backward, cudaStream_t st);
int launch_scan(const Args& a, int dtype, bool save, cudaStream_t st);
int launch_backward_scan(const Args& a, int dtype, cudaStream_t st);
int launch_backward_chunks(const Args& a, int dtype, cudaStream_t st);

}  // namespace plastic
}  // namespace bsx
