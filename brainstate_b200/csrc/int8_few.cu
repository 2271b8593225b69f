// Dense 8-bit product for few rows (up to 32): bound by reading the weights once.
//
// The weights' output channels are the rows of the tensor instructions (16 x 8 x 32, 32-bit sums), the activations
// their columns.  A block has 16 channels; its warps share the inner dimension in stretches of 64, loaded straight into
// the instructions' registers with 16-byte loads (the order of the inner index is free as long as both operands agree),
// and their sums meet in shared memory.  Integer sums: the order does not matter.
#include "int8.cuh"

namespace bsx {
namespace int8 {

constexpr int kFewWarps = 16;

__device__ __forceinline__ void mma_s8(int* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename E, int NT>
__global__ void __launch_bounds__(kFewWarps * 32) few_kernel(Product p) {
  __shared__ int part[kFewWarps][NT * 4][32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  // rows beyond the last are read from the last: their sums are dropped
  const int64_t r0 = min(n0 + g, p.N - 1), r1 = min(n0 + g + 8, p.N - 1);
  const int8_t* w0 = p.w + r0 * p.Kp;
  const int8_t* w1 = p.w + r1 * p.Kp;
  const int8_t* xr[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) xr[n] = p.x + min((int64_t)(n * 8 + g), p.M - 1) * p.Kp;
  int acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0;
  constexpr int U = 4;    // stretches in flight
  constexpr int kStep = kFewWarps * 64;
  const uint4 none = make_uint4(0u, 0u, 0u, 0u);
  const int Kp = (int)p.Kp;
  uint4 a[U], b[U];
  auto weights = [&](int k0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * kStep + t * 16;
      a[u] = k < Kp ? __ldg(reinterpret_cast<const uint4*>(w0 + k)) : none;
      b[u] = k < Kp ? __ldg(reinterpret_cast<const uint4*>(w1 + k)) : none;
    }
  };
  weights(warp * 64);
  wait_for_rows();
  for (int k0 = warp * 64; k0 < Kp; k0 += U * kStep) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * kStep + t * 16;
      uint4 x[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) x[n] = k < Kp ? *reinterpret_cast<const uint4*>(xr[n] + k) : none;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma_s8(acc[n], a[u].x, b[u].x, a[u].y, b[u].y, x[n].x, x[n].y);
        mma_s8(acc[n], a[u].z, b[u].z, a[u].w, b[u].w, x[n].z, x[n].w);
      }
    }
    if (k0 + U * kStep < Kp) weights(k0 + U * kStep);
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[warp][n * 4 + i][lane] = acc[n][i];
  __syncthreads();
  // entry (n, i, lane): channel g + 8 (i >> 1), row n * 8 + 2 t + (i & 1)
  for (int e = tid; e < NT * 128; e += kFewWarps * 32) {
    const int ch = e & 15, m = e >> 4;
    const int ni = (m >> 3) * 4 + (m & 1) + 2 * (ch >> 3), l = (ch & 7) * 4 + ((m & 7) >> 1);
    int s = 0;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) s += part[w][ni][l];
    const int64_t n = n0 + ch;
    if (m < p.M && n < p.N) static_cast<E*>(p.out)[m * p.N + n] = scaled<E>(s, p.sx[m], __ldg(p.sw + n));
  }
}

// Up to 8 rows cost what one costs.  Up to 32 the rows' own traffic shows: measured (with quantisation, 24 rows),
// 1000 x 2000 5.6 us here and 9.4 us on tiles, 2048 x 8192 14.7 and 11.3, 8192 x 4096 21.8 and 14.1.
bool few_applies(int64_t M, int64_t N, int64_t Kp) { return M <= 8 || (M <= 32 && N * Kp <= 1 << 23); }

template <typename E>
static int launch_typed(const Product& p, cudaStream_t st) {
  const unsigned grid = (unsigned)((p.N + 15) / 16);
  const int nt = (int)((p.M + 7) / 8);
  auto kernel = nt <= 1 ? few_kernel<E, 1> : nt == 2 ? few_kernel<E, 2> : nt == 3 ? few_kernel<E, 3> : few_kernel<E, 4>;
  const cudaError_t e = launch_behind(p.after_rows, kernel, grid, kFewWarps * 32, 0, st, p);
  return e == cudaSuccess ? BSX_OK : cuda_fail(e, "int8 few_kernel");
}

int launch_few(const Product& p, int dtype, cudaStream_t st) {
  if (dtype == BSX_T_F32) return launch_typed<float>(p, st);
  if (dtype == BSX_T_BF16) return launch_typed<__nv_bfloat16>(p, st);
  return launch_typed<__half>(p, st);
}

}  // namespace int8
}  // namespace bsx
