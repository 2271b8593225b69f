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

// max|x| of a row or column as the ABI defines its scale: max / 127 in one rounding; NaN where an entry is not finite.
__device__ __forceinline__ float scale_of(float top, bool finite) {
  return finite ? __fdiv_rn(top, 127.f) : __int_as_float(0x7fffffff);
}

// x / s to the nearest integer, ties to even, decided on the exact quotient: the 32-bit product x * (1/s) is within
// 5e-5 of it, so only values that come within 1e-4 of a border need the 64-bit quotient.
__device__ __forceinline__ int quantized(float x, float s, float inv) {
  const float y = x * inv;
  float n = rintf(y);
  if (!(fabsf(y - n) < 0.4999f)) n = (float)rint((double)x / (double)s);
  return (int)fminf(fmaxf(n, -127.f), 127.f);
}

template <typename E> struct Stretch { E v[16 / sizeof(E)]; };

__device__ __forceinline__ bool note(float x, float& top) {   // true for what is not finite
  const float a = fabsf(x);
  top = fmaxf(top, a);
  return !(a <= 3.402823466e38f);
}

// Four values in one word.  The nearest integer comes from the sum with 1.5 * 2^23, whose low byte is it; where a value
// comes near a border the exact rule decides, out of line.
static __device__ __noinline__ uint32_t four_exact(float4 x, float s, float inv) {
  return (uint32_t)(uint8_t)(int8_t)quantized(x.x, s, inv) | (uint32_t)(uint8_t)(int8_t)quantized(x.y, s, inv) << 8 |
         (uint32_t)(uint8_t)(int8_t)quantized(x.z, s, inv) << 16 | (uint32_t)(uint8_t)(int8_t)quantized(x.w, s, inv) << 24;
}
__device__ __forceinline__ uint32_t four(float4 x, float s, float inv) {
  constexpr float M = 12582912.f;
  const float y0 = x.x * inv, y1 = x.y * inv, y2 = x.z * inv, y3 = x.w * inv;
  const float t0 = __fadd_rn(y0, M), t1 = __fadd_rn(y1, M), t2 = __fadd_rn(y2, M), t3 = __fadd_rn(y3, M);
  const float d = fmaxf(fmaxf(fabsf(y0 - __fsub_rn(t0, M)), fabsf(y1 - __fsub_rn(t1, M))),
                        fmaxf(fabsf(y2 - __fsub_rn(t2, M)), fabsf(y3 - __fsub_rn(t3, M))));
  if (!(d < 0.4999f)) return four_exact(x, s, inv);
  return __byte_perm(__byte_perm(__float_as_uint(t0), __float_as_uint(t1), 0x0040),
                     __byte_perm(__float_as_uint(t2), __float_as_uint(t3), 0x0040), 0x5410);
}

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
