// Gated delta rule, token by token: the form for single tokens and short sequences.
//
// One block owns all dk key rows of 32 * VEC value columns of one head.  Its eight warps hold dk / 8 rows each in
// registers; the state is read once and written once whatever the number of tokens (8 dk dv bytes a head, which is what
// bounds a single token).  Per token the sums S^T k and S^T q are taken together, so there is one exchange between the
// warps: o = scale (e^g S^T q + u (k.q)).
//
// 256 rows x 16 heads of 128 x 128: 105 us, 5.1 TB/s, 78 % of the measured copy rate; one row of 8 heads of 64 x 64 2.9 us.
#include "plastic.cuh"

namespace bsx {
namespace plastic {

template <int VEC> struct __align__(4 * VEC) Cols { float v[VEC]; };

template <typename E, int ROWS, int VEC>
__global__ void __launch_bounds__(256) step_kernel(Args a) {
  constexpr int W = 32 * VEC;
  __shared__ float sk[128], sq[128];
  __shared__ float part[2][8][2][W];
  __shared__ float skq[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per_head = (a.dv + W - 1) / W;
  const int bh = blockIdx.x / per_head, c0 = (blockIdx.x - bh * per_head) * W + lane * VEC;
  const int b = bh / a.Hv, h = bh - b * a.Hv, hk = h / (a.Hv / a.Hk);
  const int len = row_length(a, b);
  const bool on = c0 < a.dv;     // VEC divides dv
  const int64_t base = (int64_t)bh * a.dk * a.dv + c0;

  Cols<VEC> s[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int kr = warp * ROWS + r;
    const bool ok = on && kr < a.dk && a.initial != nullptr;
    if (ok) {
      s[r] = *reinterpret_cast<const Cols<VEC>*>(a.initial + base + (int64_t)kr * a.dv);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[r].v[e] = 0.f;
    }
  }
  const E* kp = static_cast<const E*>(a.k) + b * a.ks[0] + hk * a.ks[2];
  const E* qp = static_cast<const E*>(a.q) + b * a.qs[0] + hk * a.qs[2];
  const E* vp = static_cast<const E*>(a.v) + b * a.vs[0] + h * a.vs[2];
  const float* gp = a.g + b * a.gs[0] + h * a.gs[2];
  const float* bp = a.beta + b * a.bs[0] + h * a.bs[2];
  E* op = static_cast<E*>(a.o) + ((int64_t)b * a.T * a.Hv + h) * a.dv;

  for (int tok = 0; tok < len; ++tok) {
    const int buf = tok & 1;
    if (tok > 0) __syncthreads();      // everybody has read the previous token's k and q
    if (tid < 128) sk[tid] = tid < a.dk ? to_f<E>(kp[tok * a.ks[1] + tid]) : 0.f;
    else sq[tid - 128] = tid - 128 < a.dk ? to_f<E>(qp[tok * a.qs[1] + tid - 128]) : 0.f;
    const float eg = expf(gp[tok * a.gs[1]]), be = bp[tok * a.bs[1]];
    float v[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = on ? to_f<E>(vp[tok * a.vs[1] + c0 + e]) : 0.f;
    __syncthreads();
    if (warp == 0) {
      float x = 0.f;
      for (int i = lane; i < 128; i += 32) x = fmaf(sk[i], sq[i], x);
      x = warp_sum(x);
      if (lane == 0) skq[buf] = x;
    }
    float pk[VEC], pq[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) pk[e] = pq[e] = 0.f;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float kv = sk[warp * ROWS + r], qv = sq[warp * ROWS + r];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        pk[e] = fmaf(s[r].v[e], kv, pk[e]);
        pq[e] = fmaf(s[r].v[e], qv, pq[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      part[buf][warp][0][lane * VEC + e] = pk[e];
      part[buf][warp][1][lane * VEC + e] = pq[e];
    }
    __syncthreads();
    float u[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float x = 0.f;
#pragma unroll
      for (int p = 0; p < 8; ++p) x += part[buf][p][0][lane * VEC + e];
      u[e] = be * (v[e] - eg * x);
    }
    if (warp == 0 && on) {
      const float kq = skq[buf];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float x = 0.f;
#pragma unroll
        for (int p = 0; p < 8; ++p) x += part[buf][p][1][lane * VEC + e];
        op[(int64_t)tok * a.Hv * a.dv + c0 + e] = from_f<E>(a.scale * fmaf(u[e], kq, eg * x));
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float kv = sk[warp * ROWS + r];
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[r].v[e] = fmaf(kv, u[e], eg * s[r].v[e]);
    }
  }
  if (!a.state) return;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int kr = warp * ROWS + r;
    if (!on || kr >= a.dk) continue;
    *reinterpret_cast<Cols<VEC>*>(a.state + base + (int64_t)kr * a.dv) = s[r];
  }
}

template <typename E, int ROWS>
static int launch_rows(const Args& a, cudaStream_t st) {
  // Two columns a lane (64 a block) keep more blocks in flight while one waits; where there are many waves of blocks the
  // wider rows of four columns count for more.  16-bit inputs, 16 heads of 128 x 128: 64 rows 27.8 us with two, 29.6 with
  // four; 256 rows 109 us and 105 us.
  const bool vec = a.dv % 4 == 0 && a.dv > 32 && aligned16(a.initial) && aligned16(a.state);
  const int64_t heads = (int64_t)a.B * a.Hv;
  const bool wide = vec && heads * ((a.dv + 127) / 128) >= 16ll * sm_count();
  const int W = wide ? 128 : vec ? 64 : 32;
  const unsigned grid = (unsigned)(heads * ((a.dv + W - 1) / W));
  if (wide) step_kernel<E, ROWS, 4><<<grid, 256, 0, st>>>(a);
  else if (vec) step_kernel<E, ROWS, 2><<<grid, 256, 0, st>>>(a);
  else step_kernel<E, ROWS, 1><<<grid, 256, 0, st>>>(a);
  BSX_LAUNCH_CHECK("plastic step_kernel");
  return BSX_OK;
}

template <typename E>
static int launch_typed(const Args& a, cudaStream_t st) {
  return a.dk <= 64 ? launch_rows<E, 8>(a, st) : launch_rows<E, 16>(a, st);
}

int launch_step(const Args& a, int dtype, cudaStream_t st) {
  if (dtype == BSX_T_F32) return launch_typed<float>(a, st);
  if (dtype == BSX_T_BF16) return launch_typed<__nv_bfloat16>(a, st);
  return launch_typed<__half>(a, st);
}

}  // namespace plastic
}  // namespace bsx
