// Shared parts of the dense 8-bit product (int8_*.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace bsx {
namespace int8 {

template <typename E> __device__ __forceinline__ float to_f(E x);
template <> __device__ __forceinline__ float to_f<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }
template <typename E> __device__ __forceinline__ E from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16(x); }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half(x); }

// The scaled output: the sum is exact, each of the three roundings is 2^-24 of the value.  Factors on both sides of 1
// are joined first: no intermediate result leaves the range of numbers that the operands and the output lie in.
template <typename E>
__device__ __forceinline__ E scaled(int sum, float sx, float sw) {
  const float s = (float)sum;
  const bool mixed = (sx < 1.f) != (sw < 1.f);
  return from_f<E>(__fmul_rn(__fmul_rn(mixed ? sw : s, sx), mixed ? s : sw));
}

// The scale of a row or column from its max|x| (max_nan): max / 127 in one rounding; NaN where an entry is not finite.
__device__ __forceinline__ float scale_of(float top) {
  return top <= 3.402823466e38f ? __fdiv_rn(top, 127.f) : __int_as_float(0x7fffffff);
}

// x / s to the nearest integer, ties to even, decided on the exact quotient: the 32-bit product x * (1/s), |x/s| <= 127, is
// within 127 * 2 * 2^-24 = 1.6e-5 of it (half of that without the product's own rounding), so only values that come as
// near to a border need the 64-bit quotient.
__device__ __forceinline__ int quantized(float x, float s, float inv) {
  const float y = x * inv;
  float n = rintf(y);
  if (!(fabsf(y - n) < 0.49998f)) n = (float)rint((double)x / (double)s);
  return (int)fminf(fmaxf(n, -127.f), 127.f);
}

template <typename E> struct Stretch { E v[16 / sizeof(E)]; };

// The larger of two, NaN if either is: a maximum of |x| that is finite says that all are.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// Four values in one word.  The nearest integer comes from the sum with 1.5 * 2^23, whose low byte is it; where a value
// comes near a border the exact rule decides, out of line.
static __device__ __noinline__ uint32_t four_exact(float4 x, float s, float inv) {
  return (uint32_t)(uint8_t)(int8_t)quantized(x.x, s, inv) | (uint32_t)(uint8_t)(int8_t)quantized(x.y, s, inv) << 8 |
         (uint32_t)(uint8_t)(int8_t)quantized(x.z, s, inv) << 16 | (uint32_t)(uint8_t)(int8_t)quantized(x.w, s, inv) << 24;
}
__device__ __forceinline__ uint32_t four(float4 x, float s, float inv) {
  constexpr float M = 12582912.f;
  const float t0 = fmaf(x.x, inv, M), t1 = fmaf(x.y, inv, M), t2 = fmaf(x.z, inv, M), t3 = fmaf(x.w, inv, M);
  const float d = fmaxf(fmaxf(fabsf(fmaf(x.x, inv, M - t0)), fabsf(fmaf(x.y, inv, M - t1))),
                        fmaxf(fabsf(fmaf(x.z, inv, M - t2)), fabsf(fmaf(x.w, inv, M - t3))));
  if (!(d < 0.49999f)) return four_exact(x, s, inv);
  return __byte_perm(__byte_perm(__float_as_uint(t0), __float_as_uint(t1), 0x0040),
                     __byte_perm(__float_as_uint(t2), __float_as_uint(t3), 0x0040), 0x5410);
}

// The running max|x| of 16-byte stretches: two 16-bit entries an instruction.
template <typename X> struct Top {
  float t = 0.f;
  __device__ __forceinline__ void look(const int4& w) {
    const Stretch<X> h = *reinterpret_cast<const Stretch<X>*>(&w);
#pragma unroll
    for (int e = 0; e < 4; ++e) t = max_nan(t, fabsf(h.v[e]));
  }
  __device__ __forceinline__ float get() const { return t; }
};
template <typename X2, typename X> struct Top2 {
  X2 t;
  __device__ __forceinline__ Top2() { *reinterpret_cast<uint32_t*>(&t) = 0u; }
  __device__ __forceinline__ void look(const int4& w) {
    const X2* h = reinterpret_cast<const X2*>(&w);
#pragma unroll
    for (int e = 0; e < 4; ++e) t = __hmax2_nan(t, __habs2(h[e]));
  }
  __device__ __forceinline__ float get() const { return max_nan(to_f<X>(t.x), to_f<X>(t.y)); }
};
template <> struct Top<__nv_bfloat16> : Top2<__nv_bfloat162, __nv_bfloat16> {};
template <> struct Top<__half> : Top2<__half2, __half> {};

// Rows of a product's left operand are padded to whole 16-byte stretches.
inline int64_t padded(int64_t k) { return (k + 15) / 16 * 16; }

struct Product {
  const int8_t* x;      // (M, Kp)
  const float* sx;      // (M)
  const int8_t* w;      // (N, Kp)
  const float* sw;      // (N)
  void* out;            // (M, N)
  int32_t* partial;     // (splits, M, N), or NULL
  int64_t M, N, Kp;
  bool after_rows;      // launched right behind the kernel that writes x and sx: may start before that has ended
};

// A product's kernel is launched while the kernel that quantises its rows still runs, sets itself up (and asks for
// weights, which that kernel does not touch), and waits here for the rows.
__device__ __forceinline__ void let_dependents_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_rows() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... P, typename... A>
inline cudaError_t launch_behind(bool early, void (*kernel)(P...), unsigned grid, unsigned threads, size_t smem,
                                 cudaStream_t st, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

struct Plan { int rows, splits; };

bool few_applies(int64_t M, int64_t N, int64_t Kp);
int launch_few(const Product& p, int dtype, cudaStream_t st);
// Rows that are not quantised yet, by the same kernel (p.x and p.sx unused).
bool few_takes_rows(int64_t M, int64_t K);
int launch_few_rows(const Product& p, const void* x, int format, int64_t stride, int64_t K, int dtype, cudaStream_t st);
Plan plan_tiles(int64_t M, int64_t N, int64_t Kp, int sms);
int launch_tiles(const Product& p, Plan plan, int dtype, cudaStream_t st);

}  // namespace int8
}  // namespace bsx
