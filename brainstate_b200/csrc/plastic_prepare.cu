// Gated delta rule: what a chunk needs that does not depend on the state — T, P and the decay vectors — for all
// chunks at once, one block of four warps per (row, head, chunk).
//
// The K and Q tiles are also written back in the layout they have in shared memory, once per key head.
// K K^T and Q K^T are 64x64xdk products (only the tiles on and below the diagonal); T = (I + A)^{-1} is built by
// substitution: the four 16x16 diagonal blocks by columns (one lane each), then by block distance
// T_ij = -sum_l (T_ii A_il) T_lj, warp i having block row i, on split operands.  (A power series would need fewer steps but
// loses all digits when the keys of a chunk are alike.)  The sums of g are taken in 64 bits and kept as two floats, so
// that a strong decay (g is cut at -128, where e^g is 0 in 32 bits) leaves the differences behind it exact.
//
// A chain of short phases whose waits blocks hide for each other, six to an SM (T and A lie where K and Q were; with four
// it took 52 us): 2048 chunks of dk = 128 in bf16 take 46 us, of which reading the tiles and writing them, T and P would
// take 31 us.
#include "plastic.cuh"

namespace bsx {
namespace plastic {

template <typename E, int DK>
struct PrepLayout {
  static constexpr int PK = DK + 8;  // pair loads of 8 rows hit distinct banks
  static constexpr size_t tile = (size_t)kC * PK * sizeof(E);
  static constexpr int PA = kC + 4;  // as right operand rows 2t, 2t + 1 hit distinct banks
  // T and A take the place of the K and Q tiles
  static constexpr size_t matrix = sizeof(float) * kC * PA, shared = tile > matrix ? 2 * tile : 2 * matrix;
  static constexpr size_t bytes = shared + sizeof(float) * 3 * kC;
};

// 16 x 8 x 16 with 16-bit operands: their products are exact in the float32 sums.
template <typename E>
__device__ __forceinline__ void mma_exact(float* c, const uint4& a, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<E, __nv_bfloat16>::value)
    mma16(c, a, b0, b1);
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// A left operand: four 8 x 8 tiles, a row's address from each lane.
__device__ __forceinline__ uint4 four_tiles(const void* row) {
  uint4 r;
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(smem_u32(row)) : "memory");
  return r;
}

// Clears this head's outputs (gradients) of a chunk's tokens from `live` on, which no later kernel writes.  Gradients of
// shared keys are written whole where they are summed.
template <typename E, bool BACK>
__device__ __forceinline__ void clear_tail(const Args& a, int b, int h, int64_t t0, int live) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, end = (int)min((int64_t)kC, a.T - t0);
  auto rows = [&](void* p, int width) {      // (batch, tokens, Hv, width)
    constexpr int V = 16 / sizeof(E);
    const bool wide = width % V == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
    for (int r = live + warp; r < end; r += 4) {
      E* x = static_cast<E*>(p) + (((int64_t)b * a.T + t0 + r) * a.Hv + h) * width;
      if (wide)
        for (int c = lane; c < width / V; c += 32) reinterpret_cast<int4*>(x)[c] = make_int4(0, 0, 0, 0);
      else
        for (int c = lane; c < width; c += 32) x[c] = from_f<E>(0.f);
    }
  };
  if (!BACK) {
    rows(a.o, a.dv);
    return;
  }
  rows(a.dv_, a.dv);
  if (a.Hk == a.Hv) {
    rows(a.dq, a.dk);
    rows(a.dk_, a.dk);
  }
  for (int r = live + threadIdx.x; r < end; r += 128) {
    const int64_t at = ((int64_t)b * a.T + t0 + r) * a.Hv + h;
    a.dg[at] = 0.f;
    a.dbeta[at] = 0.f;
  }
}

template <typename E, int DK, bool BACK>
__global__ void __launch_bounds__(128) prepare_kernel(Args a) {
  using L = PrepLayout<E, DK>;
  extern __shared__ __align__(16) unsigned char smem[];
  E* sk = reinterpret_cast<E*>(smem);
  E* sq = reinterpret_cast<E*>(smem + L::tile);
  float* sT = reinterpret_cast<float*>(smem);      // once K and Q are not needed any more
  float* sA = reinterpret_cast<float*>(smem + L::matrix);
  float* sHi = reinterpret_cast<float*>(smem + L::shared);
  float* sLo = sHi + kC;
  float* sBeta = sLo + kC;

  if (BACK && blockIdx.x == 0 && threadIdx.x == 0) *a.taken = 0u;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int chunk = blockIdx.x % a.NC;
  const int bh = blockIdx.x / a.NC, b = bh / a.Hv, h = bh - b * a.Hv, hk = h / (a.Hv / a.Hk);
  const int len = row_length(a, b);
  const int64_t t0 = (int64_t)chunk * kC;
  const int rows = t0 < len ? (int)min((int64_t)kC, len - t0) : 0;
  if (a.lengths && rows < kC) clear_tail<E, BACK>(a, b, h, t0, rows);
  if (rows == 0) return;
  const int64_t ci = (int64_t)bh * a.NC + chunk;

  // g and beta first: their sums are a chain that starts with these loads
  float gv[2] = {0.f, 0.f}, bv[2] = {0.f, 0.f};
  if (warp == 0) {
    const float* gp = a.g + b * a.gs[0] + t0 * a.gs[1] + h * a.gs[2];
    const float* bp = a.beta + b * a.bs[0] + t0 * a.bs[1] + h * a.bs[2];
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (2 * lane + e < rows) {
        gv[e] = gp[(2 * lane + e) * a.gs[1]];
        bv[e] = bp[(2 * lane + e) * a.bs[1]];
      }
  }
  const E* kp = static_cast<const E*>(a.k) + b * a.ks[0] + t0 * a.ks[1] + hk * a.ks[2];
  const E* qp = static_cast<const E*>(a.q) + b * a.qs[0] + t0 * a.qs[1] + hk * a.qs[2];
  stage(sk, L::PK, kp, a.ks[1], rows, a.dk, DK, a.vec_qk, tid, 128);
  stage(sq, L::PK, qp, a.qs[1], rows, a.dk, DK, a.vec_qk, tid, 128);
  cp_commit();
  if (warp == 0) {  // sums of g: two tokens a lane, then across the lanes
    const double x0 = gv[0] < -128.f ? -128.f : gv[0], x1 = gv[1] < -128.f ? -128.f : gv[1];
    const float b0 = bv[0], b1 = bv[1];
    double s = x0 + x1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    const double G1 = s, G0 = s - x1, GC = __shfl_sync(0xffffffffu, s, 31);
    // s - x1 is not the sum in order, but within 2^-52 of it
    float* vec = a.rec + ci * kRecord + 2 * kTri;
    const float h0 = (float)G0, h1 = (float)G1;
    const float l0 = (float)(G0 - h0), l1 = (float)(G1 - h1);
    sHi[2 * lane] = h0; sHi[2 * lane + 1] = h1;
    sLo[2 * lane] = l0; sLo[2 * lane + 1] = l1;
    sBeta[2 * lane] = b0; sBeta[2 * lane + 1] = b1;
    *reinterpret_cast<float2*>(vec + 2 * lane) = make_float2(expf((float)G0), expf((float)G1));
    *reinterpret_cast<float2*>(vec + kC + 2 * lane) = make_float2(expf((float)(GC - G0)), expf((float)(GC - G1)));
    *reinterpret_cast<float2*>(vec + 2 * kC + 2 * lane) = make_float2(b0, b1);
    *reinterpret_cast<float2*>(vec + 3 * kC + 2 * lane) = make_float2(h0, h1);
    *reinterpret_cast<float2*>(vec + 4 * kC + 2 * lane) = make_float2(l0, l1);
  }
  cp_wait<0>();
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncthreads();
  const bool packs = tid == 0 && h % (a.Hv / a.Hk) == 0;
  if (packs) {   // both tiles as they lie here, in one copy: later kernels take them with one copy too
    unsigned char* kq = static_cast<unsigned char*>(a.kq) + (((int64_t)b * a.Hk + hk) * a.NC + chunk) * (2 * L::tile);
    bulk_s2g(kq, smem, (uint32_t)(2 * L::tile));
  }

  // K K^T and Q K^T: the 20 tiles (16 x 8) on and below the diagonal by rows, five to a warp
  float kk[5][4], qk[5][4];
  int r0[5], nt[5];       // first row (of this lane) and column tile
#pragma unroll
  for (int u = 0; u < 5; ++u) {
    const int i = 5 * warp + u, r = i < 2 ? 0 : i < 6 ? 1 : i < 12 ? 2 : 3;
    nt[u] = i - r * (r + 1);
    r0[u] = r * 16 + g;
    clear(kk[u]);
    clear(qk[u]);
  }
  if constexpr (IsExact<E>::value) {
#pragma unroll 2
    for (int kp = 0; kp < DK / 16; ++kp)
#pragma unroll
      for (int u = 0; u < 5; ++u) {
        const int left = (r0[u] - g + (lane & 15)) * L::PK + kp * 16 + (lane >> 4) * 8;
        const int right = (nt[u] * 8 + (lane & 7)) * L::PK + kp * 16 + ((lane >> 3) & 1) * 8;
        uint32_t b0, b1;
        asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];" : "=r"(b0), "=r"(b1) : "r"(smem_u32(sk + right)) : "memory");
        mma_exact<E>(kk[u], four_tiles(sk + left), b0, b1);
        mma_exact<E>(qk[u], four_tiles(sq + left), b0, b1);
      }
  } else {
#pragma unroll 2
    for (int ks = 0; ks < DK / 8; ++ks) {
      const int c = ks * 8 + 2 * t;
#pragma unroll
      for (int u = 0; u < 5; ++u) {
        const float2 k0 = pair(sk + r0[u] * L::PK + c), k1 = pair(sk + (r0[u] + 8) * L::PK + c);
        const float2 q0 = pair(sq + r0[u] * L::PK + c), q1 = pair(sq + (r0[u] + 8) * L::PK + c);
        const float ak[4] = {k0.x, k1.x, k0.y, k1.y}, aq[4] = {q0.x, q1.x, q0.y, q1.y};
        const float2 bb = pair(sk + (nt[u] * 8 + g) * L::PK + c);
        float h[4], l[4];
        split4(ak, h, l);
        mma_split<false, 1>(kk + u, h, l, &bb);
        split4(aq, h, l);
        mma_split<false, 1>(qk + u, h, l, &bb);
      }
    }
  }
  if (packs) bulk_read_wait();
  __syncthreads();      // the tiles are free
  float* Tm = a.rec + ci * kRecord;
  float* Pm = Tm + kTri;
  float* Bm = BACK ? a.Bm + ci * kTri : nullptr;
#pragma unroll
  for (int u = 0; u < 5; ++u)
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int i = r0[u] + 8 * hf, n = nt[u], j = n * 8 + 2 * t;
      float p[2], m[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float gam = j + e <= i ? expf((sHi[i] - sHi[j + e]) + (sLo[i] - sLo[j + e])) : 0.f;
        p[e] = j + e <= i ? a.scale * gam * qk[u][2 * hf + e] : 0.f;
        m[e] = j + e < i ? gam * kk[u][2 * hf + e] : 0.f;
        sA[i * L::PA + j + e] = sBeta[i] * m[e];
      }
      if (n <= i >> 3) {
        const int at = tri(i >> 3, n) + lane * 2;
        *reinterpret_cast<float2*>(Pm + at) = make_float2(p[0], p[1]);
        if (BACK) *reinterpret_cast<float2*>(Bm + at) = make_float2(m[0], m[1]);
      }
    }
  __syncthreads();

  // diagonal blocks of T: lane j solves column j of block `warp`
  if (lane < 16) {
    float x[16];
    const float* Ad = sA + (16 * warp) * L::PA + 16 * warp;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float r[16];
#pragma unroll
      for (int l = 0; l < i; l += 4) *reinterpret_cast<float4*>(r + l) = *reinterpret_cast<const float4*>(Ad + i * L::PA + l);
      float v = i == lane ? 1.f : 0.f, u = 0.f;     // two chains
#pragma unroll
      for (int l = 0; l < i; ++l) {
        if (l & 1) u = fmaf(-r[l], x[l], u);
        else v = fmaf(-r[l], x[l], v);
      }
      x[i] = v + u;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) sT[(16 * warp + i) * L::PA + 16 * warp + lane] = x[i];
  }
  __syncwarp();
  // -T_ii A_il for l < i = warp, kept as left operands
  float z[3][2][4];
#pragma unroll
  for (int l = 0; l < 3; ++l) {
    if (l >= warp) break;
    clear(z[l][0]);
    clear(z[l][1]);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const float* p = sT + (16 * warp + g) * L::PA + 16 * warp + ks * 8 + 2 * t;
      const float2 p0 = pair(p), p1 = pair(p + 8 * L::PA);
      const float x[4] = {-p0.x, -p1.x, -p0.y, -p1.y};
      float hi[4], lo[4];
      split4(x, hi, lo);
      const float* r = sA + (16 * warp + ks * 8 + 2 * t) * L::PA + 16 * l + g;
      const float2 y[2] = {make_float2(r[0], r[L::PA]), make_float2(r[8], r[L::PA + 8])};
      mma_split<false, 2>(z[l], hi, lo, y);
    }
  }
  for (int d = 1; d < 4; ++d) {
    __syncthreads();
    const int j = warp - d;
    if (j < 0) continue;
    float c[2][4];
    clear(c[0]);
    clear(c[1]);
#pragma unroll
    for (int l = 0; l < 3; ++l) {
      if (l < j || l >= warp) continue;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        float x[4], hi[4], lo[4];
        as_left(z[l][ks], x);
        split4(x, hi, lo);
        const float* r = sT + (16 * l + ks * 8 + 2 * t) * L::PA + 16 * j + g;
        const float2 y[2] = {make_float2(r[0], r[L::PA]), make_float2(r[8], r[L::PA + 8])};
        mma_split<false, 2>(c, hi, lo, y);
      }
    }
    float* o = sT + (16 * warp + g) * L::PA + 16 * j + 2 * t;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      *reinterpret_cast<float2*>(o + n * 8) = make_float2(c[n][0], c[n][1]);
      *reinterpret_cast<float2*>(o + n * 8 + 8 * L::PA) = make_float2(c[n][2], c[n][3]);
    }
  }
  __syncthreads();
  for (int n = warp; n < 8; n += 4)
    for (int k = 0; k <= n; ++k) {
      const float* x = sT + (n * 8 + g) * L::PA + k * 8 + 2 * t;
      *reinterpret_cast<float2*>(Tm + tri(n, k) + lane * 2) = make_float2(x[0], x[1]);
    }
}

template <typename E, int DK>
static int launch_typed(const Args& a, bool backward, cudaStream_t st) {
  const size_t bytes = PrepLayout<E, DK>::bytes;
  const unsigned grid = (unsigned)((int64_t)a.B * a.Hv * a.NC);
  static std::atomic<uint64_t> seen[2];
  int rc;
  if (backward) {
    if ((rc = allow_smem(prepare_kernel<E, DK, true>, bytes, seen[1])) != BSX_OK) return rc;
    prepare_kernel<E, DK, true><<<grid, 128, bytes, st>>>(a);
  } else {
    if ((rc = allow_smem(prepare_kernel<E, DK, false>, bytes, seen[0])) != BSX_OK) return rc;
    prepare_kernel<E, DK, false><<<grid, 128, bytes, st>>>(a);
  }
  BSX_LAUNCH_CHECK("plastic prepare_kernel");
  return BSX_OK;
}

template <typename E>
static int launch_width(const Args& a, bool backward, cudaStream_t st) {
  return a.dk <= 64 ? launch_typed<E, 64>(a, backward, st) : launch_typed<E, 128>(a, backward, st);
}

int launch_prepare(const Args& a, int dtype, bool backward, cudaStream_t st) {
  if (dtype == BSX_T_F32) return launch_width<float>(a, backward, st);
  if (dtype == BSX_T_BF16) return launch_width<__nv_bfloat16>(a, backward, st);
  return launch_width<__half>(a, backward, st);
}

}  // namespace plastic
}  // namespace bsx
