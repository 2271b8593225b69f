// Dense 8-bit product: rows of activations and columns of weights to 8 bits, and the C entry points.
//
// A row's scale is max|x| / 127 (32 bits); its values are the nearest integers of x / scale.  Spike rows become 0 and 1
// with scale 1.  A row with an entry that is not finite gets the scale NaN and zeros, so that its outputs are NaN.
#include "int8.cuh"

namespace bsx {
namespace int8 {

constexpr int kHeld = 4;   // 16-byte stretches a thread keeps between the two passes over its row

// One block per row: the maximum, then the values.  Bound by reading the row once and writing a byte per entry; the first
// kHeld 16-byte stretches of a thread stay in registers in between, the rest comes from L2 the second time.  4096 rows of 4096
// in bf16: 15.6 us, 3.2 TB/s.
template <typename E, bool VEC, int THREADS>
__global__ void __launch_bounds__(THREADS)
quantize_rows_kernel(const E* __restrict__ x, int64_t stride, int64_t K, int64_t Kp, int8_t* __restrict__ q,
                     float* __restrict__ scale) {
  constexpr int V = 16 / sizeof(E);
  __shared__ float part[THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31;
  const int64_t row = blockIdx.x;
  const E* xr = x + row * stride;
  int8_t* qr = q + row * Kp;
  let_dependents_start();
  int4 held[kHeld];
  float top = 0.f;
  const int n = (int)(K / V);
  const int4* x4 = reinterpret_cast<const int4*>(xr);
  if (VEC) {
    Top<E> look;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) held[i] = tid + i * THREADS < n ? __ldg(x4 + tid + i * THREADS) : make_int4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) look.look(held[i]);
    for (int c = tid + kHeld * THREADS; c < n; c += THREADS) look.look(__ldg(x4 + c));
    top = look.get();
  } else {
    for (int c = tid; c < K; c += THREADS) top = max_nan(top, fabsf(to_f<E>(xr[c])));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) part[tid >> 5] = top;
  __syncthreads();
  top = part[lane % (THREADS / 32)];
#pragma unroll
  for (int o = THREADS / 64; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float s = scale_of(top);
  if (tid == 0) scale[row] = s;
  const bool zero = !(s > 0.f);
  const float inv = s < 1e-30f ? __int_as_float(0x7fffffff) : 1.f / s;   // tiny scales: every quotient in 64 bits
  if (VEC) {
    auto put = [&](int c, const int4& x) {
      const Stretch<E> h = *reinterpret_cast<const Stretch<E>*>(&x);
      uint32_t w[V / 4];
#pragma unroll
      for (int e = 0; e < V; e += 4)
        w[e / 4] = zero ? 0u : four(make_float4(to_f<E>(h.v[e]), to_f<E>(h.v[e + 1]), to_f<E>(h.v[e + 2]), to_f<E>(h.v[e + 3])),
                                    s, inv);
      if (V == 8) reinterpret_cast<uint2*>(qr)[c] = make_uint2(w[0], w[V / 4 - 1]);
      else reinterpret_cast<uint32_t*>(qr)[c] = w[0];
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (tid + i * THREADS < n) put(tid + i * THREADS, held[i]);
    for (int c = tid + kHeld * THREADS; c < n; c += THREADS) put(c, __ldg(x4 + c));
    for (int c = n + tid; c < (int)(Kp / V); c += THREADS) {
      if (V == 8) reinterpret_cast<uint2*>(qr)[c] = make_uint2(0u, 0u);
      else reinterpret_cast<uint32_t*>(qr)[c] = 0u;
    }
  } else {
    for (int c = tid * 4; c < Kp; c += THREADS * 4) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = c + j < K ? to_f<E>(xr[c + j]) : 0.f;
      *reinterpret_cast<uint32_t*>(qr + c) = zero ? 0u : four(make_float4(v[0], v[1], v[2], v[3]), s, inv);
    }
  }
}

// Spike rows: 1 where an entry is not zero; 16 entries a thread.
template <int FORMAT, bool VEC>
__global__ void __launch_bounds__(256)
event_rows_kernel(const void* __restrict__ x, int64_t stride, int64_t M, int64_t K, int64_t Kp, int8_t* __restrict__ q,
                  float* __restrict__ scale) {
  let_dependents_start();
  const int64_t words = Kp / 16, total = M * words;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / words, c = (i - row * words) * 16;
    uint4 r;
    if (VEC && FORMAT == BSX_SPK_BOOL8) {
      r = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(x) + row * stride + c));
      r.x = __vsetgtu4(r.x, 0u);
      r.y = __vsetgtu4(r.y, 0u);
      r.z = __vsetgtu4(r.z, 0u);
      r.w = __vsetgtu4(r.w, 0u);
    } else {
      uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (c + j < K && spike_at<FORMAT>(x, row * stride + c + j)) w[j / 4] |= 1u << (8 * (j % 4));
      r = make_uint4(w[0], w[1], w[2], w[3]);
    }
    *reinterpret_cast<uint4*>(q + row * Kp + c) = r;
    if (c == 0) scale[row] = 1.f;
  }
}

// Weights (K, N), 32 columns a block: the maxima over a range of rows, met in `top` as the bits of non-negative floats
// (infinity for what is not finite) ...
template <typename E>
__global__ void __launch_bounds__(256) column_top_kernel(const E* __restrict__ w, int64_t K, int64_t N, uint32_t* __restrict__ top) {
  __shared__ float part[8][32];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t n = (int64_t)blockIdx.x * 32 + tx;
  float t = 0.f;
  if (n < N)
#pragma unroll 4
    for (int64_t k = (int64_t)blockIdx.y * 8 + ty; k < K; k += (int64_t)gridDim.y * 8) t = max_nan(t, fabsf(to_f<E>(w[k * N + n])));
  part[ty][tx] = t <= 3.402823466e38f ? t : __int_as_float(0x7f800000);
  __syncthreads();
  if (ty == 0 && n < N) {
#pragma unroll
    for (int i = 0; i < 8; ++i) t = fmaxf(t, part[i][tx]);
    atomicMax(top + n, __float_as_uint(t));
  }
}

// ... then tiles of 128 rows, turned through shared memory ...
template <typename E>
__global__ void __launch_bounds__(256)
quantize_columns_kernel(const E* __restrict__ w, int64_t K, int64_t N, int64_t Kp, int8_t* __restrict__ q,
                        const uint32_t* __restrict__ top) {
  __shared__ __align__(16) int8_t tile[32][132];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t n0 = (int64_t)blockIdx.x * 32, n = n0 + tx, k0 = (int64_t)blockIdx.y * 128;
  const float t = n < N ? __uint_as_float(top[n]) : 0.f;
  const float s = scale_of(t);
  const bool zero = !(s > 0.f);
  const float inv = s < 1e-30f ? __int_as_float(0x7fffffff) : 1.f / s;
#pragma unroll 4
  for (int i = 0; i < 16; ++i) {
    const int64_t k = k0 + ty + 8 * i;
    tile[tx][ty + 8 * i] = (n < N && k < K && !zero) ? (int8_t)quantized(to_f<E>(w[k * N + n]), s, inv) : (int8_t)0;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = ty + 8 * i, c = tx * 4;
    if (n0 + r < N && k0 + c < Kp)
      *reinterpret_cast<uint32_t*>(q + (n0 + r) * Kp + k0 + c) = *reinterpret_cast<const uint32_t*>(&tile[r][c]);
  }
}

// ... and the maxima become scales.
__global__ void __launch_bounds__(256) column_scale_kernel(float* scale, int64_t N) {
  const int64_t n = blockIdx.x * 256ll + threadIdx.x;
  if (n < N) scale[n] = scale_of(scale[n]);
}

template <typename E>
static int launch_columns(const void* w, int64_t K, int64_t N, int8_t* q, float* scale, cudaStream_t st) {
  const E* p = static_cast<const E*>(w);
  const int64_t Kp = padded(K), cols = (N + 31) / 32, want = 8ll * sm_count() / cols + 1, most = (K + 63) / 64;
  BSX_CUDA(cudaMemsetAsync(scale, 0, N * sizeof(float), st));
  column_top_kernel<E><<<dim3((unsigned)cols, (unsigned)(want < most ? want : most)), 256, 0, st>>>(
      p, K, N, reinterpret_cast<uint32_t*>(scale));
  BSX_LAUNCH_CHECK("column_top_kernel");
  quantize_columns_kernel<E><<<dim3((unsigned)cols, (unsigned)((Kp + 127) / 128)), 256, 0, st>>>(
      p, K, N, Kp, q, reinterpret_cast<const uint32_t*>(scale));
  BSX_LAUNCH_CHECK("quantize_columns_kernel");
  column_scale_kernel<<<(unsigned)((N + 255) / 256), 256, 0, st>>>(scale, N);
  BSX_LAUNCH_CHECK("column_scale_kernel");
  return BSX_OK;
}

template <typename E, bool VEC>
static void launch_rows_vec(const E* x, int64_t stride, int64_t M, int64_t K, int8_t* q, float* scale, cudaStream_t st) {
  const int64_t Kp = padded(K);
  // few rows: the time is that of one row, so that as many threads as its stretches fill share it
  if (M < 148 && K * (int64_t)sizeof(E) > 128 * 16)
    quantize_rows_kernel<E, VEC, 1024><<<(unsigned)M, 1024, 0, st>>>(x, stride, K, Kp, q, scale);
  else
    quantize_rows_kernel<E, VEC, 128><<<(unsigned)M, 128, 0, st>>>(x, stride, K, Kp, q, scale);
}

template <typename E>
static int launch_rows(const void* x, int64_t stride, int64_t M, int64_t K, int8_t* q, float* scale, cudaStream_t st) {
  constexpr int V = 16 / sizeof(E);
  const E* p = static_cast<const E*>(x);
  if (aligned16(x) && (M == 1 || stride % V == 0) && K % V == 0) launch_rows_vec<E, true>(p, stride, M, K, q, scale, st);
  else launch_rows_vec<E, false>(p, stride, M, K, q, scale, st);
  BSX_LAUNCH_CHECK("quantize_rows_kernel");
  return BSX_OK;
}

static int rows(const void* x, int format, int64_t stride, int64_t M, int64_t K, int8_t* q, float* scale, cudaStream_t st) {
  switch (format) {
    case BSX_T_F32: return launch_rows<float>(x, stride, M, K, q, scale, st);
    case BSX_T_BF16: return launch_rows<__nv_bfloat16>(x, stride, M, K, q, scale, st);
    case BSX_T_F16: return launch_rows<__half>(x, stride, M, K, q, scale, st);
    default: break;
  }
  const int64_t Kp = padded(K), want = (M * (Kp / 16) + 255) / 256, most = 8ll * sm_count();
  const unsigned grid = (unsigned)(want < most ? want : most);
  if (format == BSX_T_EVENT32)
    event_rows_kernel<BSX_SPK_F32, false><<<grid, 256, 0, st>>>(x, stride, M, K, Kp, q, scale);
  else if (aligned16(x) && (M == 1 || stride % 16 == 0) && K % 16 == 0)
    event_rows_kernel<BSX_SPK_BOOL8, true><<<grid, 256, 0, st>>>(x, stride, M, K, Kp, q, scale);
  else
    event_rows_kernel<BSX_SPK_BOOL8, false><<<grid, 256, 0, st>>>(x, stride, M, K, Kp, q, scale);
  BSX_LAUNCH_CHECK("event_rows_kernel");
  return BSX_OK;
}

static int check_sizes(int64_t M, int64_t K, int64_t N) {
  if (M < 0 || K < 0 || N < 0) return fail(BSX_ERR_INVALID_ARG, "negative size");
  if (M > INT32_MAX || N > INT32_MAX) return fail(BSX_ERR_UNSUPPORTED, "sizes must fit int32");
  // |sum| <= 127^2 K has to fit 32 bits
  if (K > 131072) return fail(BSX_ERR_UNSUPPORTED, "more than 131072 inputs: sums would leave 32 bits");
  return BSX_OK;
}
static int check_format(int format) {
  if (format < BSX_T_F32 || format > BSX_T_EVENT32) return fail(BSX_ERR_INVALID_ARG, "unknown element type");
  return BSX_OK;
}

static size_t aligned(size_t n) { return (n + 255) / 256 * 256; }

// Bytes of the parts of the workspace: rows in 8 bits, their scales, partial sums.
static size_t partial_bytes(int64_t M, int64_t K, int64_t N, int sms) {
  if (few_applies(M, N, padded(K))) return 0;
  const int splits = plan_tiles(M, N, padded(K), sms).splits;
  return splits > 1 ? (size_t)splits * M * N * sizeof(int32_t) : 0;
}

static int product(bool after_rows, const int8_t* q, const float* sx, const int8_t* w, const float* sw, int64_t M, int64_t K, int64_t N,
                   void* out, int out_type, void* partial, cudaStream_t st) {
  Product p;
  p.x = q; p.sx = sx; p.w = w; p.sw = sw; p.out = out;
  p.partial = static_cast<int32_t*>(partial);
  p.M = M; p.N = N; p.Kp = padded(K);
  p.after_rows = after_rows;
  if (few_applies(M, N, p.Kp)) return launch_few(p, out_type, st);
  return launch_tiles(p, plan_tiles(M, N, p.Kp, sm_count()), out_type, st);
}

}  // namespace int8
}  // namespace bsx

using namespace bsx;
using namespace bsx::int8;

extern "C" int64_t bsx_int8_row_bytes(int64_t K) { return K < 0 ? 0 : padded(K); }

extern "C" int bsx_int8_quantize_rows(const void* x, int format, int64_t row_stride, int64_t M, int64_t K, int8_t* q,
                                      float* scale, bsx_stream_t stream) {
  BSX_TRACE("bsx_int8_quantize_rows");
  int rc;
  if ((rc = check_sizes(M, K, 0)) != BSX_OK || (rc = check_format(format)) != BSX_OK) return rc;
  if (M == 0) return BSX_OK;
  if ((K > 0 && (!x || !q)) || !scale) return fail(BSX_ERR_INVALID_ARG, "NULL buffer");
  if (K > 0 && !aligned16(q)) return fail(BSX_ERR_INVALID_ARG, "q must start on a 16-byte boundary");
  if (sm_count() <= 0) return fail(BSX_ERR_CUDA, "no CUDA device");
  if (K == 0) return fail(BSX_ERR_UNSUPPORTED, "rows without entries have no scale");
  return rows(x, format, row_stride, M, K, q, scale, as_stream(stream));
}

extern "C" int bsx_int8_quantize_weights(const void* w, int dtype, int64_t K, int64_t N, int8_t* q, float* scale,
                                         bsx_stream_t stream) {
  BSX_TRACE("bsx_int8_quantize_weights");
  int rc;
  if ((rc = check_sizes(0, K, N)) != BSX_OK) return rc;
  if (dtype < BSX_T_F32 || dtype > BSX_T_F16) return fail(BSX_ERR_INVALID_ARG, "unknown element type");
  if (N == 0) return BSX_OK;
  if (K == 0) return fail(BSX_ERR_UNSUPPORTED, "columns without entries have no scale");
  if (!w || !q || !scale) return fail(BSX_ERR_INVALID_ARG, "NULL buffer");
  if (!aligned16(q)) return fail(BSX_ERR_INVALID_ARG, "q must start on a 16-byte boundary");
  if (sm_count() <= 0) return fail(BSX_ERR_CUDA, "no CUDA device");
  cudaStream_t st = as_stream(stream);
  if (dtype == BSX_T_F32) return launch_columns<float>(w, K, N, q, scale, st);
  if (dtype == BSX_T_BF16) return launch_columns<__nv_bfloat16>(w, K, N, q, scale, st);
  return launch_columns<__half>(w, K, N, q, scale, st);
}

extern "C" size_t bsx_int8_matmul_workspace_bytes(int64_t M, int64_t K, int64_t N) {
  return check_sizes(M, K, N) == BSX_OK ? partial_bytes(M, K, N, sm_count()) : 0;
}

extern "C" int bsx_int8_matmul(const int8_t* q, const float* scale, const int8_t* wq, const float* wscale, int64_t M,
                               int64_t K, int64_t N, void* out, int out_dtype, void* ws, size_t ws_bytes,
                               bsx_stream_t stream) {
  BSX_TRACE("bsx_int8_matmul");
  int rc;
  if ((rc = check_sizes(M, K, N)) != BSX_OK) return rc;
  if (out_dtype < BSX_T_F32 || out_dtype > BSX_T_F16) return fail(BSX_ERR_INVALID_ARG, "unknown output type");
  if (M == 0 || N == 0) return BSX_OK;
  if (K == 0) return fail(BSX_ERR_UNSUPPORTED, "product over no inputs");
  if (!q || !scale || !wq || !wscale || !out) return fail(BSX_ERR_INVALID_ARG, "NULL buffer");
  if (!aligned16(q) || !aligned16(wq)) return fail(BSX_ERR_INVALID_ARG, "8-bit operands must start on a 16-byte boundary");
  const int sms = sm_count();
  if (sms <= 0) return fail(BSX_ERR_CUDA, "no CUDA device");
  const size_t need = partial_bytes(M, K, N, sms);
  if (need > 0 && (!ws || !aligned16(ws) || ws_bytes < need))
    return fail(BSX_ERR_WORKSPACE, "workspace missing, misaligned or too small");
  return product(false, q, scale, wq, wscale, M, K, N, out, out_dtype, ws, as_stream(stream));
}

extern "C" size_t bsx_int8_dense_workspace_bytes(int64_t M, int64_t K, int64_t N) {
  if (check_sizes(M, K, N) != BSX_OK || few_takes_rows(M, K)) return 0;
  return aligned((size_t)M * padded(K)) + aligned((size_t)M * sizeof(float)) + partial_bytes(M, K, N, sm_count());
}

extern "C" int bsx_int8_dense(const void* x, int format, int64_t row_stride, const int8_t* wq, const float* wscale,
                              int64_t M, int64_t K, int64_t N, void* out, int out_dtype, void* ws, size_t ws_bytes,
                              bsx_stream_t stream) {
  BSX_TRACE("bsx_int8_dense");
  int rc;
  if ((rc = check_sizes(M, K, N)) != BSX_OK || (rc = check_format(format)) != BSX_OK) return rc;
  if (out_dtype < BSX_T_F32 || out_dtype > BSX_T_F16) return fail(BSX_ERR_INVALID_ARG, "unknown output type");
  if (M == 0 || N == 0) return BSX_OK;
  if (K == 0) return fail(BSX_ERR_UNSUPPORTED, "product over no inputs");
  if (!x || !wq || !wscale || !out) return fail(BSX_ERR_INVALID_ARG, "NULL buffer");
  if (!aligned16(wq)) return fail(BSX_ERR_INVALID_ARG, "8-bit operands must start on a 16-byte boundary");
  const int sms = sm_count();
  if (sms <= 0) return fail(BSX_ERR_CUDA, "no CUDA device");
  if (few_takes_rows(M, K)) {     // one kernel, no workspace
    Product p = {};
    p.w = wq; p.sw = wscale; p.out = out;
    p.M = M; p.N = N; p.Kp = padded(K);
    return launch_few_rows(p, x, format, row_stride, K, out_dtype, as_stream(stream));
  }
  const size_t qb = aligned((size_t)M * padded(K)), sb = aligned((size_t)M * sizeof(float));
  if (!ws || !aligned16(ws) || ws_bytes < qb + sb + partial_bytes(M, K, N, sms))
    return fail(BSX_ERR_WORKSPACE, "workspace missing, misaligned or too small");
  char* base = static_cast<char*>(ws);
  int8_t* q = reinterpret_cast<int8_t*>(base);
  float* sx = reinterpret_cast<float*>(base + qb);
  cudaStream_t st = as_stream(stream);
  if ((rc = rows(x, format, row_stride, M, K, q, sx, st)) != BSX_OK) return rc;
  return product(true, q, sx, wq, wscale, M, K, N, out, out_dtype, base + qb + sb, st);
}
