// Dense 8-bit product for few rows (up to 32): bound by reading the weights once.
//
// The weights' output channels are the rows of the tensor instructions (16 x 8 x 32, 32-bit sums), the activations
// their columns.  A block has 16 channels; its warps share the inner dimension in stretches of 64, loaded straight into
// the instructions' registers with 16-byte loads (the order of the inner index is free as long as both operands agree),
// and their sums meet in shared memory.  Integer sums: the order does not matter.
//
// Up to four rows are quantised by the product's own blocks, each for itself, while their first weights are on the way: the
// rows come from L2, and neither a second kernel nor a workspace is needed.
#include "int8.cuh"

namespace bsx {
namespace int8 {

constexpr int kFewWarps = 16;

__device__ __forceinline__ void mma_s8(int* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int kFewThreads = kFewWarps * 32;

// The maxima of the rows, then their 8-bit values in shared memory (rows of Kp bytes) and their scales; kFewWarps / R
// warps to a row, R >= M a power of two.  X: float, bf16, fp16, or a spike format.
// ask_weights() is called once the first loads of the rows are on their way: behind the weights they would wait for those.
template <typename X, int EVENT, int R, typename F>
__device__ __forceinline__ void take_rows(const void* x, int64_t stride, int M, int K, int Kp, bool vec, int8_t* q, float* scale,
                                          float* part, F ask_weights) {
  constexpr int WPR = kFewWarps / R, T = WPR * 32;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = warp / WPR, at = tid - row * T;
  const bool on = row < M;
  int8_t* qr = q + row * Kp;
  if constexpr (EVENT >= 0) {
    ask_weights();
    for (int c = at * 4; on && c < Kp; c += T * 4) {
      uint32_t r = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < K && spike_at<EVENT>(x, row * stride + c + j)) r |= 1u << (8 * j);
      *reinterpret_cast<uint32_t*>(qr + c) = r;
    }
    if (tid < R) scale[tid] = 1.f;
  } else {
    constexpr int V = 16 / sizeof(X);
    const X* xr = static_cast<const X*>(x) + row * stride;
    const int4* x4 = reinterpret_cast<const int4*>(xr);
    float top = 0.f;
    const int n = on ? K / V : 0;
    int4 held[2];      // the first two stretches stay in registers between the passes
    if (vec) {
#pragma unroll
      for (int i = 0; i < 2; ++i) held[i] = at + i * T < n ? __ldg(x4 + at + i * T) : make_int4(0, 0, 0, 0);
      ask_weights();
      Top<X> look;
      look.look(held[0]);
      look.look(held[1]);
#pragma unroll 4
      for (int c = at + 2 * T; c < n; c += T) look.look(__ldg(x4 + c));
      top = look.get();
    } else {
      ask_weights();
      for (int c = at; on && c < K; c += T) top = max_nan(top, fabsf(to_f<X>(xr[c])));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) part[warp] = top;
    __syncthreads();
    top = part[row * WPR];
#pragma unroll
    for (int w = 1; w < WPR; ++w) top = max_nan(top, part[row * WPR + w]);
    const float s = scale_of(top);
    if (at == 0) scale[row] = s;
    const bool zero = !(s > 0.f);
    const float inv = s < 1e-30f ? __int_as_float(0x7fffffff) : 1.f / s;
    if (vec) {
      auto put = [&](int c, const int4& w) {
        const Stretch<X> h = *reinterpret_cast<const Stretch<X>*>(&w);
#pragma unroll
        for (int e = 0; e < V; e += 4)
          *reinterpret_cast<uint32_t*>(qr + c * V + e) =
              zero ? 0u : four(make_float4(to_f<X>(h.v[e]), to_f<X>(h.v[e + 1]), to_f<X>(h.v[e + 2]), to_f<X>(h.v[e + 3])), s, inv);
      };
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (at + i * T < n) put(at + i * T, held[i]);
      for (int c = at + 2 * T; c < n; c += T) put(c, __ldg(x4 + c));
      for (int c = K + at * 4; on && c < Kp; c += T * 4) *reinterpret_cast<uint32_t*>(qr + c) = 0u;
    } else {
      for (int c = at * 4; on && c < Kp; c += T * 4) {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = c + j < K ? to_f<X>(xr[c + j]) : 0.f;
        *reinterpret_cast<uint32_t*>(qr + c) = zero ? 0u : four(make_float4(v[0], v[1], v[2], v[3]), s, inv);
      }
    }
  }
  __syncthreads();
}

struct Given {          // rows that are not quantised yet
  const void* x;
  int64_t stride;
  int K;
  bool vec;
};

// NT tiles of eight rows, quantised before (R = 0) or taken from `given` (R >= M rows, NT = 1).
template <typename E, int NT, typename X, int EVENT, int R>
__global__ void __launch_bounds__(kFewThreads, NT == 1 ? 2 : 1) few_kernel(Product p, Given given) {
  __shared__ int part[kFewWarps][NT * 4][32];
  __shared__ float row_scale[R > 0 ? R : 1];
  extern __shared__ __align__(16) int8_t rows[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int8_t* xr[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) xr[n] = (R > 0 ? rows : p.x) + min((int64_t)(n * 8 + g), p.M - 1) * p.Kp;
  constexpr int U = 4;    // stretches in flight
  constexpr int kStep = kFewWarps * 64;
  const uint4 none = make_uint4(0u, 0u, 0u, 0u);
  const int Kp = (int)p.Kp;
  const int tiles = (int)((p.N + 15) / 16);
  uint4 a[U], b[U];
  auto weights = [&](int tile, int k0) {
    // channels beyond the last are read from the last: their sums are dropped
    const int8_t* w0 = p.w + min((int64_t)tile * 16 + g, p.N - 1) * p.Kp;
    const int8_t* w1 = p.w + min((int64_t)tile * 16 + g + 8, p.N - 1) * p.Kp;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * kStep + t * 16;
      a[u] = k < Kp ? __ldg(reinterpret_cast<const uint4*>(w0 + k)) : none;
      b[u] = k < Kp ? __ldg(reinterpret_cast<const uint4*>(w1 + k)) : none;
    }
  };
  if constexpr (R > 0) {
    take_rows<X, EVENT, R>(given.x, given.stride, (int)p.M, given.K, Kp, given.vec, rows, row_scale,
                           reinterpret_cast<float*>(&part[0][0][0]), [&] { weights(blockIdx.x, warp * 64); });
  } else {
    weights(blockIdx.x, warp * 64);
    wait_for_rows();
  }
  for (int tile = blockIdx.x; tile < tiles; tile += R > 0 ? gridDim.x : tiles) {
    int acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][i] = 0;
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
      if (k0 + U * kStep < Kp) weights(tile, k0 + U * kStep);
    }
    if (R > 0 && tile + (int)gridDim.x < tiles) weights(tile + gridDim.x, warp * 64);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[warp][n * 4 + i][lane] = acc[n][i];
    __syncthreads();
    // entry (n, i, lane): channel g + 8 (i >> 1), row n * 8 + 2 t + (i & 1)
    for (int e = tid; e < NT * 128; e += kFewThreads) {
      const int ch = e & 15, m = e >> 4;
      const int ni = (m >> 3) * 4 + (m & 1) + 2 * (ch >> 3), l = (ch & 7) * 4 + ((m & 7) >> 1);
      const int64_t n = (int64_t)tile * 16 + ch;
      if (m >= p.M || n >= p.N) continue;
      int s = 0;
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) s += part[w][ni][l];
      static_cast<E*>(p.out)[m * p.N + n] = scaled<E>(s, R > 0 ? row_scale[m] : p.sx[m], __ldg(p.sw + n));
    }
    __syncthreads();
  }
}

// Up to 8 rows cost what one costs.  Up to 32 the rows' own traffic shows: measured (with quantisation, 24 rows),
// 1000 x 2000 5.6 us here and 9.4 us on tiles, 2048 x 8192 14.7 and 11.3, 8192 x 4096 21.8 and 14.1.
bool few_applies(int64_t M, int64_t N, int64_t Kp) { return M <= 8 || (M <= 32 && N * Kp <= 1 << 23); }

template <typename E>
static int launch_typed(const Product& p, cudaStream_t st) {
  const int nt = (int)((p.M + 7) / 8);
  const unsigned grid = (unsigned)((p.N + 15) / 16);
  auto kernel = nt <= 1   ? few_kernel<E, 1, float, -1, 0>
                : nt == 2 ? few_kernel<E, 2, float, -1, 0>
                : nt == 3 ? few_kernel<E, 3, float, -1, 0>
                          : few_kernel<E, 4, float, -1, 0>;
  const cudaError_t e = launch_behind(p.after_rows, kernel, grid, kFewThreads, 0, st, p, Given{});
  return e == cudaSuccess ? BSX_OK : cuda_fail(e, "int8 few_kernel");
}

int launch_few(const Product& p, int dtype, cudaStream_t st) {
  if (dtype == BSX_T_F32) return launch_typed<float>(p, st);
  if (dtype == BSX_T_BF16) return launch_typed<__nv_bfloat16>(p, st);
  return launch_typed<__half>(p, st);
}

// Every block reads and quantises all rows: M / 8 of the weights' traffic (for 16-bit rows), from L2, and M * K / 512 values a
// thread.  One row of 8192 x 4096: 9.1 us replayed in a graph against 7.8 us with a kernel of its own for the rows, but
// 11.1 us against 15.3 us of host time where calls are launched one by one; 1000 x 2000 3.5 us against 3.8 us.
bool few_takes_rows(int64_t M, int64_t K) { return M <= 4 && M * padded(K) <= 40704; }

template <typename E, typename X, int EVENT>
static int launch_rows(const Product& p, const Given& given, cudaStream_t st) {
  // as many blocks as run at once: each quantises the rows once and takes one group of channels after the other
  const int64_t tiles = (p.N + 15) / 16, most = 2ll * sm_count();
  const unsigned grid = (unsigned)(tiles < most ? tiles : most);
  auto kernel = p.M <= 1 ? few_kernel<E, 1, X, EVENT, 1> : p.M == 2 ? few_kernel<E, 1, X, EVENT, 2> : few_kernel<E, 1, X, EVENT, 4>;
  kernel<<<grid, kFewThreads, (size_t)(p.M * p.Kp), st>>>(p, given);
  BSX_LAUNCH_CHECK("int8 few_kernel");
  return BSX_OK;
}

template <typename E>
static int launch_rows_typed(const Product& p, const Given& given, int format, cudaStream_t st) {
  switch (format) {
    case BSX_T_F32: return launch_rows<E, float, -1>(p, given, st);
    case BSX_T_BF16: return launch_rows<E, __nv_bfloat16, -1>(p, given, st);
    case BSX_T_F16: return launch_rows<E, __half, -1>(p, given, st);
    case BSX_T_EVENT8: return launch_rows<E, float, BSX_SPK_BOOL8>(p, given, st);
    default: return launch_rows<E, float, BSX_SPK_F32>(p, given, st);
  }
}

int launch_few_rows(const Product& p, const void* x, int format, int64_t stride, int64_t K, int dtype, cudaStream_t st) {
  const int V = format == BSX_T_F32 ? 4 : 8;
  const Given given = {x, stride, (int)K, aligned16(x) && (p.M == 1 || stride % V == 0) && K % V == 0};
  if (dtype == BSX_T_F32) return launch_rows_typed<float>(p, given, format, st);
  if (dtype == BSX_T_BF16) return launch_rows_typed<__nv_bfloat16>(p, given, format, st);
  return launch_rows_typed<__half>(p, given, format, st);
}

}  // namespace int8
}  // namespace bsx
