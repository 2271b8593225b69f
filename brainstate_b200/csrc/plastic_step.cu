// Gated delta rule, token by token: the form for single tokens and short sequences.
//
// One block owns all dk key rows of 32 * VEC value columns of one head.  Its eight warps hold dk / 8 rows each in
// registers; the state is read once and written once whatever the number of tokens (8 dk dv bytes a head, which is what
// bounds a single token).  Per token the sums S^T k and S^T q are taken together, so there is one exchange between the
// warps: o = scale (e^g S^T q + u (k.q)).
//
// 128 rows x 16 heads of 128 x 128: 57 us, 4.7 TB/s; one row of 8 heads of 64 x 64 2.9 us.  Many large states take
// step_stream_kernel below.
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

// One token for many rows: bound by moving the states through, so the moving is done by bulk copies that run ahead.  One
// block an SM takes every gridDim-th (row, head): its state (up to 64 KB, contiguous) comes into one of three places of
// shared memory while earlier ones are worked on, passes through the registers once and goes back with a bulk copy.  The
// arithmetic is that of step_kernel, in the same order.  256 rows x 16 heads of 128 x 128: 95 us, 5.66 TB/s, 86 % of the
// measured copy rate.
constexpr int kStages = 3;

template <typename E>
__global__ void __launch_bounds__(256, 1) step_stream_kernel(Args a) {
  constexpr int ROWS = 16, stages = kStages;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float sk[2][128], sq[2][128], skq[2];
  __shared__ __align__(16) float part[8][2][128];
  __shared__ __align__(8) uint64_t full[kStages];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, c0 = lane * 4;
  const uint32_t items = (uint32_t)a.B * a.Hv, tile = (uint32_t)a.dk * a.dv;
  const bool on = c0 < a.dv;
  if (tid < stages) mbar_init(&full[tid], 1);
  __syncthreads();
  auto place = [&](uint32_t nth) { return reinterpret_cast<float*>(smem) + (nth % stages) * tile; };
  auto load = [&](uint32_t nth, uint32_t item) {    // one thread
    mbar_expect_tx(&full[nth % stages], tile * 4);
    bulk_g2s(place(nth), a.initial + (int64_t)item * tile, tile * 4, &full[nth % stages]);
  };
  // this item's inputs: an entry of k or q, the gates, four of v
  float x = 0.f, eg = 0.f, be = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
  auto fetch = [&](uint32_t item) {
    const uint32_t b = item / a.Hv, h = item - b * a.Hv, hk = h / (a.Hv / a.Hk);
    const int c = tid & 127;
    const E* p = tid < 128 ? static_cast<const E*>(a.k) + b * a.ks[0] + hk * a.ks[2] : static_cast<const E*>(a.q) + b * a.qs[0] + hk * a.qs[2];
    x = c < a.dk ? to_f<E>(p[c]) : 0.f;
    const E* vp = static_cast<const E*>(a.v) + b * a.vs[0] + h * a.vs[2] + c0;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = on ? to_f<E>(vp[e]) : 0.f;
    eg = a.g[b * a.gs[0] + h * a.gs[2]];
    be = a.beta[b * a.bs[0] + h * a.bs[2]];
  };
  if (tid == 0)
    for (int i = 0; i < stages - 1 && blockIdx.x + i * gridDim.x < items; ++i) load(i, blockIdx.x + i * gridDim.x);
  if (blockIdx.x < items) fetch(blockIdx.x);
  uint32_t nth = 0;
  for (uint32_t item = blockIdx.x; item < items; item += gridDim.x, ++nth) {
    const int buf = nth & 1;
    (tid < 128 ? sk[buf] : sq[buf])[tid & 127] = x;
    const float decay = expf(eg), rate = be, vv[4] = {v[0], v[1], v[2], v[3]};
    __syncthreads();
    if (item + gridDim.x < items) fetch(item + gridDim.x);
    if (warp == 0) {
      float y = 0.f;
      for (int i = lane; i < 128; i += 32) y = fmaf(sk[buf][i], sq[buf][i], y);
      y = warp_sum(y);
      if (lane == 0) skq[buf] = y;
    }
    const bool there = stage_wait(&full[nth % stages], (nth / stages) & 1);
    float* S = place(nth);
    float4 s[ROWS];
    float pk[4] = {0.f, 0.f, 0.f, 0.f}, pq[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int kr = warp * ROWS + r;
      s[r] = on && kr < a.dk ? *reinterpret_cast<const float4*>(S + kr * a.dv + c0) : make_float4(0.f, 0.f, 0.f, 0.f);
      if (!there) s[r].x = s[r].y = s[r].z = s[r].w = __int_as_float(0x7fffffff);
      const float kv = sk[buf][kr], qv = sq[buf][kr];
      pk[0] = fmaf(s[r].x, kv, pk[0]); pk[1] = fmaf(s[r].y, kv, pk[1]);
      pk[2] = fmaf(s[r].z, kv, pk[2]); pk[3] = fmaf(s[r].w, kv, pk[3]);
      pq[0] = fmaf(s[r].x, qv, pq[0]); pq[1] = fmaf(s[r].y, qv, pq[1]);
      pq[2] = fmaf(s[r].z, qv, pq[2]); pq[3] = fmaf(s[r].w, qv, pq[3]);
    }
    *reinterpret_cast<float4*>(&part[warp][0][c0]) = make_float4(pk[0], pk[1], pk[2], pk[3]);
    *reinterpret_cast<float4*>(&part[warp][1][c0]) = make_float4(pq[0], pq[1], pq[2], pq[3]);
    __syncthreads();
    float u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float y = 0.f;
#pragma unroll
      for (int p = 0; p < 8; ++p) y += part[p][0][c0 + e];
      u[e] = rate * (vv[e] - decay * y);
    }
    if (warp == 0 && on) {
      const float kq = skq[buf];
      E* op = static_cast<E*>(a.o) + (int64_t)item * a.dv + c0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float y = 0.f;
#pragma unroll
        for (int p = 0; p < 8; ++p) y += part[p][1][c0 + e];
        op[e] = from_f<E>(a.scale * fmaf(u[e], kq, decay * y));
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int kr = warp * ROWS + r;
      if (!on || kr >= a.dk) continue;
      const float kv = sk[buf][kr];
      *reinterpret_cast<float4*>(S + kr * a.dv + c0) =
          make_float4(fmaf(kv, u[0], decay * s[r].x), fmaf(kv, u[1], decay * s[r].y), fmaf(kv, u[2], decay * s[r].z),
                      fmaf(kv, u[3], decay * s[r].w));
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    if (tid == 0) {
      bulk_s2g(a.state + (int64_t)item * tile, S, tile * 4);
      // the place of the item before is free once its copy has been read; the item `stages - 1` ahead goes there
      const uint64_t ahead = item + (uint64_t)(stages - 1) * gridDim.x;
      if (ahead < items) {
        bulk_read_wait_but_one();
        load(nth + stages - 1, (uint32_t)ahead);
      }
    }
  }
  if (tid == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

template <typename E, int ROWS>
static int launch_rows(const Args& a, cudaStream_t st) {
  // Many large states of one token each are streamed: 16 heads of 128 x 128, 256 rows 96 us against 105 us, 128 rows 51 us
  // against 57 us, 64 rows 28 us either way; smaller states do not pay for the barriers (128 x 96 39 us either way).
  const int64_t tile = (int64_t)a.dk * a.dv * 4;
  if constexpr (ROWS == 16)
    if (a.T == 1 && !a.lengths && a.initial && a.state && a.dv % 4 == 0 && a.dv <= 128 && tile >= 57344 && aligned16(a.initial) &&
        aligned16(a.state) && (int64_t)a.B * a.Hv >= 8ll * sm_count()) {
      static std::atomic<uint64_t> seen;
      const int rc = allow_smem(step_stream_kernel<E>, kStages * 65536, seen);
      if (rc != BSX_OK) return rc;
      step_stream_kernel<E><<<sm_count(), 256, (size_t)(kStages * tile), st>>>(a);
      BSX_LAUNCH_CHECK("plastic step_stream_kernel");
      return BSX_OK;
    }
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
