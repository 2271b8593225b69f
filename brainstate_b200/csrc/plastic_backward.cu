// Gated delta rule, reverse mode.
//
// backward_scan_kernel: the pass over the chunks from the last to the first that carries the cotangent of the state,
// in the same form as the forward pass (groups of 16 value columns, transposed, accumulators used as left
// operands).  With dS the cotangent of the state after the chunk:
//   dU = P^T dO + diag(e^{G_C-G}) K dS,  dY = T^T dU,  dV = beta dY,  dR = -beta e^G dY,
//   dS <- e^{G_C} dS + Q^T (scale e^G dO) + K^T dR.
// It leaves dS (before the update) and dY for every chunk.  4 x 2048 tokens of 16 heads of 128 x 128 in bf16: 259 us, bound
// like the forward pass (shared memory 53 %, tensor unit 41 %).
//
// backward_chunk_kernel: everything else, independent of the order of the chunks; each block of 16 warps takes one (row, head,
// chunk) after the other and copies the next one's data while it finishes one.  Over blocks of 32 value columns it
// sums D1 = dY S0^T, Dq = dO S0^T, D3 = U dS^T (64 x dk) and dP = dO U^T, dA = -dY U^T (64 x 64), then
//   dQ = scale e^G Dq + E K,                         E = scale Gamma dP (j <= i)
//   dK = -beta e^G D1 + e^{G_C-G} D3 + E^T Q + (F + F^T) K,   F = beta Gamma dA (j < i)
//   dbeta_i = dY_i.V_i - e^{G_i} K_i.D1_i + sum_j dA_ij (A/beta)_ij
//   dG_i = -beta e^G K_i.D1_i + scale e^G Q_i.Dq_i - e^{G_C-G} K_i.D3_i + (row - column sums of dP P + dA A)_i,
//   dG_C += sum_i e^{G_C-G_i} K_i.D3_i + e^{G_C} <S0, dS>,   dg = sums of dG from the chunk's end.
// The same sizes: 464 us (tensor unit 40 %, issue slots 47 %).  Its 128 registers a thread hold the sums of all five
// products, which is what bounds the tiles; eight warps with twice the registers took 820 us.
#include <type_traits>

#include "plastic.cuh"

namespace bsx {
namespace plastic {

// ------------------------------------------------------------------------------------------------ pass over chunks

template <typename E, int DK>
struct BackScanLayout {
  static constexpr int PK = DK + 8;
  static constexpr size_t tile = (size_t)kC * PK * sizeof(E);
  static constexpr uint32_t rec = (2 * kTri + 3 * kC) * sizeof(float);
  static constexpr size_t set = 2 * tile + rec;        // K, Q, record (T, P, vectors)
  // a group's exchange: dS (then dR and scale e^G dO), dU, dO
  static constexpr size_t group = 16384 + 8192 + 4096;
  static constexpr size_t bytes(int groups, int stages) { return stages * set + groups * group; }
};

// The pair (row 2t, row 2t + 1) of column g of a packed 8x8 tile.
__device__ __forceinline__ float2 column_pair(const float* tile, int lane) {
  const float* p = tile + (lane & 3) * 16 + (lane >> 2);
  return make_float2(p[0], p[8]);
}

// r += dO^T P of token tiles W and 7 - W.
template <int W, bool X>
__device__ __forceinline__ void gather_own(const float4* gO, const float* Pm, int lane, float (*r)[4]) {
  float h[2][4], x[2][4];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    clear(h[e]);
    clear(x[e]);
  }
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) {
    if (ks < W && ks < 7 - W) continue;
    const float4 v = gO[ks * 32 + lane];
    const float c[4] = {v.x, v.y, v.z, v.w};
    float hi[4], lo[4];
    if (!X) split4(c, hi, lo);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int n = e ? 7 - W : W;
      if (ks < n) continue;
      const float2 pp = column_pair(Pm + tri(ks, n), lane);
      if (X) {
        float h0, l0, h1, l1;
        split(pp.x, h0, l0);
        split(pp.y, h1, l1);
        mma(x[e], c, l0, l1);
        mma(h[e], c, h0, h1);
      } else {
        mma_apart<false>(h[e], x[e], hi, lo, pp);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int i = 0; i < 4; ++i) r[e][i] += h[e][i] + x[e][i];
}

// dY^T = dU^T T of the same token tiles.
template <int W>
__device__ __forceinline__ void solve_back_own(const float4* gU, const float* Tm, int lane, float (*y)[4]) {
  float h[2][4], x[2][4], z[2][4];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    clear(h[e]);
    clear(x[e]);
    clear(z[e]);
  }
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) {
    if (ks < W && ks < 7 - W) continue;
    float hi[4], lo[4];
    get_split(gU, ks, lane, hi, lo);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int n = e ? 7 - W : W;
      if (ks < n) continue;
      const float2 tt = column_pair(Tm + tri(ks, n), lane);
      float h0, l0, h1, l1;
      split(tt.x, h0, l0);
      split(tt.y, h1, l1);
      mma(x[e], lo, h0, h1);
      mma(z[e], hi, l0, l1);
      mma(h[e], hi, h0, h1);
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int i = 0; i < 4; ++i) y[e][i] = h[e][i] + (x[e][i] + z[e][i]);
}

template <typename E, int DK, int THREADS>
__global__ void __launch_bounds__(THREADS, 1) backward_scan_kernel(Args a, int groups, int stages) {
  using L = BackScanLayout<E, DK>;
  constexpr bool X = IsExact<E>::value;
  constexpr bool B16 = std::is_same<E, __nv_bfloat16>::value;
  constexpr int DKW = DK / 4, NT = DKW / 8;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ __align__(8) uint64_t bars[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int grp = warp >> 2, w = warp & 3;
  const int per_head = (a.dv + 16 * groups - 1) / (16 * groups);
  const int bh = blockIdx.x / per_head, vb = (blockIdx.x - bh * per_head) * groups * 16;
  const int b = bh / a.Hv, h = bh - b * a.Hv, hk = h / (a.Hv / a.Hk);
  const int len = row_length(a, b), nc = (len + kC - 1) / kC;
  float4* gS = reinterpret_cast<float4*>(smem + stages * L::set + grp * L::group);   // dS; then dR, scale e^G dO
  float4* gX = gS + 512;
  float4* gU = gS + 1024;
  float4* gO = gU + 512;
  const int d0 = vb + grp * 16 + g;
  const bool in0 = d0 < a.dv, in1 = d0 + 8 < a.dv;
  const int kb = w * DKW;
  const int own[2] = {w, 7 - w};

  float s[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int kr = kb + n * 8 + 2 * t + (i & 1), d = d0 + (i >> 1) * 8;
      s[n][i] = (a.dstate && kr < a.dk && d < a.dv) ? a.dstate[((int64_t)bh * a.dk + kr) * a.dv + d] : 0.f;
    }

  if (tid < 2) mbar_init(&bars[tid], 1);
  __syncthreads();
  const unsigned char* kq = static_cast<const unsigned char*>(a.kq) + ((int64_t)b * a.Hk + hk) * a.NC * (2 * L::tile);
  auto load = [&](int c, int buf) {    // one thread
    unsigned char* base = smem + buf * L::set;
    mbar_expect_tx(&bars[buf], (uint32_t)L::set);
    bulk_g2s(base, kq + (int64_t)c * (2 * L::tile), (uint32_t)(2 * L::tile), &bars[buf]);
    bulk_g2s(base + 2 * L::tile, a.rec + ((int64_t)bh * a.NC + c) * kRecord, L::rec, &bars[buf]);
  };
  const int64_t os = (int64_t)a.Hv * a.dv;      // token stride of the outputs and their cotangents
  const E* dop = static_cast<const E*>(a.dout) + (int64_t)b * a.T * os + (int64_t)h * a.dv + d0;
  E on[2][4];
  if (nc > 0) {
    if (tid == 0) load(nc - 1, 0);
    fetch_own(on, dop + (int64_t)(nc - 1) * kC * os, os, own, t, len - (nc - 1) * kC, in0, in1);
  }
  for (int i = 0; i < nc; ++i) {
    const int c = nc - 1 - i;
    const int buf = stages == 2 ? (i & 1) : 0;
    if (stages == 2 && c > 0 && tid == 0) load(c - 1, buf ^ 1);
    const bool there = stage_wait(&bars[buf], stages == 2 ? ((i >> 1) & 1) : (i & 1));
    if (!there) s[0][0] = s[0][1] = s[0][2] = s[0][3] = __int_as_float(0x7fffffff);
    const unsigned char* base = smem + buf * L::set;
    const E* K = reinterpret_cast<const E*>(base);
    const E* Q = reinterpret_cast<const E*>(base + L::tile);
    const float* Tm = reinterpret_cast<const float*>(base + 2 * L::tile);
    const float* Pm = Tm + kTri;
    const float* eG = Pm + kTri;
    const float* eD = eG + kC;
    const float* beta = eG + 2 * kC;
    const int64_t ci = (int64_t)bh * a.NC + c;
    const int64_t t0 = (int64_t)c * kC;

    {
      float* out = a.dS + ci * a.dv * (DK + 4);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
          if (d0 + 8 * hf < a.dv)
            *reinterpret_cast<float2*>(out + (d0 + 8 * hf) * (DK + 4) + kb + n * 8 + 2 * t) =
                make_float2(s[n][2 * hf], s[n][2 * hf + 1]);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if constexpr (B16) put_parts(gS, w * NT + n, lane, s[n]);
      else put_split(gS, w * NT + n, lane, s[n]);
    }
    float x[2][4];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[e][j] = to_f<E>(on[e][j]);
      gO[own[e] * 32 + lane] = make_float4(x[e][0], x[e][2], x[e][1], x[e][3]);
    }
    if (c > 0) fetch_own(on, dop + (t0 - kC) * os, os, own, t, kC, in0, in1);
    group_sync(grp);

    // dU^T = e^{G_C-G} dS^T K^T + dO^T P of this warp's tokens
    float rh[2][4], rl[2][4];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      clear(rh[e]);
      clear(rl[e]);
    }
    if constexpr (B16) {
#pragma unroll
      for (int kp = 0; kp < DK / 16; ++kp) {
        const uint4 p[3] = {get_part(gS, kp, 0, lane), get_part(gS, kp, 1, lane), get_part(gS, kp, 2, lane)};
        state_times<DK, L::PK, false>(rh, rl, p, K, kp, own, g, t);
      }
    } else {
#pragma unroll 4
      for (int ks = 0; ks < DK / 8; ++ks) {
        float hi[4], lo[4];
        get_split(gS, ks, lane, hi, lo);
#pragma unroll
        for (int e = 0; e < 2; ++e)
          mma_apart<X>(rh[e], rl[e], hi, lo, pair(K + (own[e] * 8 + g) * L::PK + ks * 8 + 2 * t));
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float2 ed = pair(eD + own[e] * 8 + 2 * t);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float f = (j & 1) ? ed.y : ed.x;
        rh[e][j] *= f;
        rl[e][j] *= f;
      }
    }
    float u[2][4], y[2][4];
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int j = 0; j < 4; ++j) u[e][j] = rh[e][j] + rl[e][j];
    switch (w) {
      case 0: gather_own<0, X>(gO, Pm, lane, u); break;
      case 1: gather_own<1, X>(gO, Pm, lane, u); break;
      case 2: gather_own<2, X>(gO, Pm, lane, u); break;
      default: gather_own<3, X>(gO, Pm, lane, u);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) put_split(gU, own[e], lane, u[e]);
    group_sync(grp);

    switch (w) {
      case 0: solve_back_own<0>(gU, Tm, lane, y); break;
      case 1: solve_back_own<1>(gU, Tm, lane, y); break;
      case 2: solve_back_own<2>(gU, Tm, lane, y); break;
      default: solve_back_own<3>(gU, Tm, lane, y);
    }
    float* Y = a.dY + ci * a.dv * kPU;
    E* dv = static_cast<E*>(a.dv_) + ((int64_t)b * a.T + t0) * os + (int64_t)h * a.dv + d0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int tok = own[e] * 8 + 2 * t;
      const float2 be = pair(beta + tok), eg = pair(eG + tok);
      if (in0) *reinterpret_cast<float2*>(Y + d0 * kPU + tok) = make_float2(y[e][0], y[e][1]);
      if (in1) *reinterpret_cast<float2*>(Y + (d0 + 8) * kPU + tok) = make_float2(y[e][2], y[e][3]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        E* o = dv + (tok + j) * os;
        const float bj = j ? be.y : be.x;
        if (tok + j < len - c * kC) {
          if (in0) o[0] = from_f<E>(bj * y[e][j]);
          if (in1) o[8] = from_f<E>(bj * y[e][2 + j]);
        }
      }
      // dR^T and scale e^G dO^T: left operands of the state's cotangent
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float f = (j & 1) ? eg.y : eg.x;
        y[e][j] *= -f * ((j & 1) ? be.y : be.x);
        x[e][j] *= a.scale * f;
      }
      if constexpr (B16) {
        put_parts(gS, own[e], lane, y[e]);
        put_parts(gX, own[e], lane, x[e]);
      } else {
        put_split(gS, own[e], lane, y[e]);
        put_split(gX, own[e], lane, x[e]);
      }
    }
    group_sync(grp);

    float ah[NT][4], al[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      clear(ah[n]);
      clear(al[n]);
    }
    if constexpr (B16) {
#pragma unroll
      for (int tp = 0; tp < 4; ++tp) {
        const uint4 p[3] = {get_part(gS, tp, 0, lane), get_part(gS, tp, 1, lane), get_part(gS, tp, 2, lane)};
        update_state<NT, L::PK>(ah, al, p, K + tp * 16 * L::PK + kb, lane);
        const uint4 q[3] = {get_part(gX, tp, 0, lane), get_part(gX, tp, 1, lane), get_part(gX, tp, 2, lane)};
        update_state<NT, L::PK>(ah, al, q, Q + tp * 16 * L::PK + kb, lane);
      }
    } else {
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        float hi[4], lo[4];
        float2 kk[NT];
        get_split(gS, ks, lane, hi, lo);
        tiles_by_row<NT>(kk, K + ks * 8 * L::PK + kb, L::PK, lane);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_apart<X>(ah[n], al[n], hi, lo, kk[n]);
        get_split(gX, ks, lane, hi, lo);
        tiles_by_row<NT>(kk, Q + ks * 8 * L::PK + kb, L::PK, lane);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_apart<X>(ah[n], al[n], hi, lo, kk[n]);
      }
    }
    const float eC = eG[kC - 1];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[n][j] = fmaf(eC, s[n][j], ah[n][j] + al[n][j]);
    __syncthreads();      // the tiles and the group's exchange are free
    if (stages == 1 && c > 0 && tid == 0) load(c - 1, 0);
  }
  if (a.dinitial) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int kr = kb + n * 8 + 2 * t + (i & 1), d = d0 + (i >> 1) * 8;
        if (kr < a.dk && d < a.dv) a.dinitial[((int64_t)bh * a.dk + kr) * a.dv + d] = s[n][i];
      }
  }
}

template <typename E, int DK, int THREADS>
static int launch_scan_threads(const Args& a, int groups, cudaStream_t st) {
  using L = BackScanLayout<E, DK>;
  static std::atomic<uint64_t> seen;
  int rc = allow_smem(backward_scan_kernel<E, DK, THREADS>, kMaxSmem, seen);
  if (rc != BSX_OK) return rc;
  const int stages = L::bytes(groups, 2) <= kMaxSmem ? 2 : 1;
  const int per_head = (a.dv + 16 * groups - 1) / (16 * groups);
  const unsigned grid = (unsigned)((int64_t)a.B * a.Hv * per_head);
  backward_scan_kernel<E, DK, THREADS><<<grid, groups * 128, L::bytes(groups, stages), st>>>(a, groups, stages);
  BSX_LAUNCH_CHECK("plastic backward_scan_kernel");
  return BSX_OK;
}

template <typename E, int DK>
static int launch_scan_typed(const Args& a, cudaStream_t st) {
  const int sms = sm_count();
  if (sms <= 0) return fail(BSX_ERR_CUDA, "no CUDA device");
  const int groups = scan_groups(a, sms);
  return groups == 4 ? launch_scan_threads<E, DK, 512>(a, groups, st) : launch_scan_threads<E, DK, 256>(a, groups, st);
}

// ------------------------------------------------------------------------------------------------ all chunks at once

constexpr int kVB = 32;   // value columns of a block
constexpr int kChunkThreads = 512;

template <typename E, int DK>
struct BackChunkLayout {
  static constexpr int PK = DK + 8, PS = DK + 4, PO = kVB + 8, PE = kC + 8;
  static constexpr size_t tile = (size_t)kC * PK * sizeof(E);
  // floats of one set of block buffers: S0, dS, U, dY
  static constexpr int ds = kVB * PS, u = 2 * kVB * PS, dy = u + kVB * kPU, used = dy + kVB * kPU,
                       set = used > 2 * kC * PE ? used : 2 * kC * PE;   // E and F have to fit as well
  // floats after the K and Q tiles
  static constexpr int dof = 2 * set, pm = dof + kC * PO, vecs = pm + kTri, bm = vecs + kVec, parts = bm + kTri,
                       end = parts + 36 * kC;
  // E and F, then the finished gradients, take the set that the next chunk's first block does not
  static constexpr int f = kC * PE;
  static constexpr size_t bytes = 2 * tile + (size_t)end * sizeof(float);
};

// Four neighbouring elements as they come from memory: taken apart only where they are used, so that a load a block ahead
// is not waited for where it is issued.
template <typename E> struct Four;
template <> struct Four<float> {
  float4 w;
  __device__ __forceinline__ void load(const float* p) { w = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ void gather(const float* p, int left) {
    w.x = left > 0 ? p[0] : 0.f;
    w.y = left > 1 ? p[1] : 0.f;
    w.z = left > 2 ? p[2] : 0.f;
    w.w = left > 3 ? p[3] : 0.f;
  }
  __device__ __forceinline__ float4 get() const { return w; }
};
template <typename H> struct FourHalves {
  uint2 w;
  __device__ __forceinline__ void load(const H* p) { w = *reinterpret_cast<const uint2*>(p); }
  __device__ __forceinline__ void gather(const H* p, int left) {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < left ? q[i] : 0u;
    w = make_uint2(v[0] | v[1] << 16, v[2] | v[3] << 16);
  }
  __device__ __forceinline__ float4 get() const {
    const float2 a = unpack(w.x, (const H*)nullptr), b = unpack(w.y, (const H*)nullptr);
    return make_float4(a.x, a.y, b.x, b.y);
  }
};
template <> struct Four<__nv_bfloat16> : FourHalves<__nv_bfloat16> {};
template <> struct Four<__half> : FourHalves<__half> {};

// Rows of a finished (token, column) tile from shared memory, pitch `pitch`, to global memory.
template <typename O>
__device__ __forceinline__ void store_rows(O* dst, int64_t stride, const O* sm, int pitch, int rows, int cols, bool vec, int tid,
                                           int nthr) {
  constexpr int V = 16 / sizeof(O);
  if (vec) {
    const int per = cols / V;
    for (int i = tid; i < rows * per; i += nthr) {
      const int r = i / per, c = (i - r * per) * V;
      *reinterpret_cast<int4*>(dst + r * stride + c) = *reinterpret_cast<const int4*>(sm + r * pitch + c);
    }
  } else {
    for (int i = tid; i < rows * cols; i += nthr) {
      const int r = i / cols, c = i - r * cols;
      dst[r * stride + c] = sm[r * pitch + c];
    }
  }
}

// t[m][n] += a b over the four 8-column steps of a block: a (32 rows of this warp, two tiles) from a transposed (column,
// row) array or, with ROWS, from a (row, column) one; b from two (column, outer) arrays, N tiles of the first and one of
// the second.  All in 32 bits except a where AEXACT.
template <bool AEXACT, bool ROWS, int N, bool SECOND>
__device__ __forceinline__ void block_products(float (*t1)[N][4], float (*t2)[4], const float* a, int pa, const float* b1, int p1,
                                               const float* b2, int p2, int g, int t) {
#pragma unroll 1   // unrolled, the accumulators (112 of 128 registers) do not stay in registers: 463 -> 521 us
  for (int ks = 0; ks < kVB / 8; ++ks) {
    const int v = ks * 8 + 2 * t;
    constexpr int M = N + (SECOND ? 1 : 0);
    float2 h[M], l[M];
#pragma unroll
    for (int n = 0; n < M; ++n) {
      const float* p = n < N ? b1 + v * p1 + n * 8 + g : b2 + v * p2 + g;
      split(p[0], h[n].x, l[n].x);
      split(p[n < N ? p1 : p2], h[n].y, l[n].y);
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      float x[4], hi[4], lo[4];
      if (ROWS) {
        const float2 p0 = pair(a + (m * 16 + g) * pa + v), q0 = pair(a + (m * 16 + g + 8) * pa + v);
        x[0] = p0.x; x[1] = q0.x; x[2] = p0.y; x[3] = q0.y;
      } else {
        const float* p = a + v * pa + m * 16 + g;
        x[0] = p[0]; x[1] = p[8]; x[2] = p[pa]; x[3] = p[pa + 8];
      }
      if (AEXACT) {
#pragma unroll
        for (int i = 0; i < 4; ++i) hi[i] = x[i];
      } else {
        split4(x, hi, lo);
      }
      auto at = [&](int n) { return n < N ? t1[m][n < N ? n : 0] : t2[m]; };
      if (!AEXACT)
#pragma unroll
        for (int n = 0; n < M; ++n) mma(at(n), lo, h[n].x, h[n].y);
#pragma unroll
      for (int n = 0; n < M; ++n) mma(at(n), hi, l[n].x, l[n].y);
#pragma unroll
      for (int n = 0; n < M; ++n) mma(at(n), hi, h[n].x, h[n].y);
    }
  }
}

template <typename E, int DK>
__global__ void __launch_bounds__(kChunkThreads, 1) backward_chunk_kernel(Args a) {
  using L = BackChunkLayout<E, DK>;
  constexpr bool X = IsExact<E>::value;
  constexpr bool SHORT = IsShort<E>::value;
  constexpr int N = DK / 64;    // 8-wide column tiles of a warp in the (64, DK) products
  constexpr int kT = kChunkThreads;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ __align__(8) uint64_t bars[3];
  __shared__ uint32_t next_item;
  E* K = reinterpret_cast<E*>(smem);
  E* Q = reinterpret_cast<E*>(smem + L::tile);
  float* F = reinterpret_cast<float*>(smem + 2 * L::tile);
  float* sDO = F + L::dof;
  const float* Pm = F + L::pm;
  const float* Bm = F + L::bm;
  float* eG = F + L::vecs;
  float* eD = eG + kC;
  float* beta = eG + 2 * kC;
  float* gHi = eG + 3 * kC;
  float* gLo = eG + 4 * kC;
  // sums by column eighth, then added: [0,8) rows of dP P + dA A (later dA A/beta), [8,10) its columns, [10,18) K.D1,
  // [18,26) Q.Dq, [26,34) K.D3, 34 dY.V, 35 <S0,dS>
  float* parts = F + L::parts;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int wr = warp & 1, wc = warp >> 1;     // rows 32 wr .. + 31; column eighth wc
  const int64_t os = (int64_t)a.Hv * a.dv;
  const int tok = tid >> 3, vc = (tid & 7) * 4;      // this thread's values of dO and V
  const uint32_t items = (uint32_t)a.B * a.Hv * a.NC, NC = a.NC, Hv = a.Hv;

  // Where rows differ in length, items are taken as blocks become free; the first is the block's own number.
  auto ask = [&](uint32_t i) { return a.lengths ? gridDim.x + atomicAdd(a.taken, 1u) : i + gridDim.x; };
  auto valid = [&](uint32_t i) {    // the first from i on that has tokens
    if (a.lengths)
      while (i < items && (int)(i % NC) * kC >= row_length(a, (int)(i / NC / Hv))) i = ask(i);
    return i;
  };
  auto load = [&](uint32_t ci, int v0, int buf) {    // one thread
    const uint32_t nv = (uint32_t)min(kVB, a.dv - v0);
    float* f = F + buf * L::set;
    uint64_t* bar = &bars[buf];
    const int64_t row = (int64_t)ci * a.dv + v0;
    mbar_expect_tx(bar, nv * (2 * L::PS + 2 * kPU) * 4);
    bulk_g2s(f, a.Sn + row * L::PS, nv * L::PS * 4, bar);
    bulk_g2s(f + L::ds, a.dS + row * L::PS, nv * L::PS * 4, bar);
    bulk_g2s(f + L::u, a.U + row * kPU, nv * kPU * 4, bar);
    bulk_g2s(f + L::dy, a.dY + row * kPU, nv * kPU * 4, bar);
  };
  auto load_chunk = [&](uint32_t ci) {    // one thread: K, Q, P, the vectors, A / beta
    const uint32_t bh = ci / NC, b = bh / Hv, hk = (bh - b * Hv) / (Hv / a.Hk);
    mbar_expect_tx(&bars[2], (uint32_t)(2 * L::tile) + (2 * kTri + kVec) * 4);
    bulk_g2s(smem, static_cast<const unsigned char*>(a.kq) + (((int64_t)b * a.Hk + hk) * NC + ci % NC) * (2 * L::tile),
             (uint32_t)(2 * L::tile), &bars[2]);
    bulk_g2s(F + L::pm, a.rec + (int64_t)ci * kRecord + kTri, (kTri + kVec) * 4, &bars[2]);
    bulk_g2s(F + L::bm, a.Bm + (int64_t)ci * kTri, kTri * 4, &bars[2]);
  };
  // columns past dv of the last block count as zero
  auto blank = [&](int v0, int buf) {
    const int nv = a.dv - v0;
    if (nv >= kVB) return;
    float* f = F + buf * L::set;
    for (int i = tid; i < (kVB - nv) * L::PS; i += kT) f[nv * L::PS + i] = f[L::ds + nv * L::PS + i] = 0.f;
    for (int i = tid; i < (kVB - nv) * kPU; i += kT) f[L::u + nv * kPU + i] = f[L::dy + nv * kPU + i] = 0.f;
  };
  Four<E> xo, xv;
  const E *po = nullptr, *pv = nullptr;     // this thread's dO and V of an item, at column vc; NULL past the sequence's end
  auto locate = [&](uint32_t ci) {
    const uint32_t bh = ci / NC, b = bh / Hv, h = bh - b * Hv;
    const int64_t tk = (int64_t)(ci - bh * NC) * kC + tok;
    po = tk < row_length(a, b) ? static_cast<const E*>(a.dout) + ((int64_t)b * a.T + tk) * os + (int64_t)h * a.dv + vc : nullptr;
    pv = static_cast<const E*>(a.v) + b * a.vs[0] + tk * a.vs[1] + h * a.vs[2] + vc;
  };
  auto fetch = [&](int v0) {
    const int left = po ? a.dv - v0 - vc : 0;
    if (left > 0 && a.four_do) xo.load(po + v0);       // dv is a multiple of four
    else xo.gather(po + v0, left);
    if (left > 0 && a.four_v) xv.load(pv + v0);
    else xv.gather(pv + v0, left);
  };

  if (tid < 3) mbar_init(&bars[tid], 1);
  __syncthreads();
  if (tid == 0) next_item = valid(blockIdx.x);
  __syncthreads();
  uint32_t item = next_item;
  if (item < items) {
    if (tid == 0) {
      load(item, 0, 0);
      load_chunk(item);
    }
    blank(0, 0);
    locate(item);
    fetch(0);
  }
  uint32_t blk = 0;       // blocks taken so far: sets alternate across chunks
  for (uint32_t nth = 0; item < items; ++nth) {
  uint32_t asked = 0;    // looked at after the blocks: the answer takes its time
  if (tid == 0) asked = ask(item);

  float d1[2][N][4], dqa[2][N][4], d3[2][N][4], dp[2][4], da[2][4];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      clear(d1[m][n]);
      clear(dqa[m][n]);
      clear(d3[m][n]);
    }
    clear(dp[m]);
    clear(da[m]);
  }
  float ss = 0.f;     // <S0, dS>
  float yv = 0.f;     // dY.V of this thread's token, its columns
  bool there = true;
  for (int v0 = 0; v0 < a.dv; v0 += kVB, ++blk) {
    const int buf = blk & 1;
    const float* f = F + buf * L::set;
    *reinterpret_cast<float4*>(sDO + tok * L::PO + vc) = xo.get();
    const float4 v4 = xv.get();
    const float v[4] = {v4.x, v4.y, v4.z, v4.w};
    if (v0 + kVB < a.dv) {
      if (tid == 0) load(item, v0 + kVB, buf ^ 1);
      blank(v0 + kVB, buf ^ 1);
      fetch(v0 + kVB);
    }
    there &= stage_wait(&bars[buf], (blk >> 1) & 1);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) yv = fmaf(f[L::dy + (vc + i) * kPU + tok], v[i], yv);
    for (int i = tid; i < kVB * DK / 4; i += kT) {
      const int at = (i / (DK / 4)) * L::PS + (i % (DK / 4)) * 4;
      const float4 x = *reinterpret_cast<const float4*>(f + at), y = *reinterpret_cast<const float4*>(f + L::ds + at);
      ss += (x.x * y.x + x.y * y.y) + (x.z * y.z + x.w * y.w);
    }
    // each block's sums are started afresh and added in one rounding (the tensor unit cuts its sums)
    float t1[2][N][4], t2[2][4];
    auto zero = [&] {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
#pragma unroll
        for (int n = 0; n < N; ++n) clear(t1[m][n]);
        clear(t2[m]);
      }
    };
    auto add = [&](float (*x1)[N][4], float (*x2)[4]) {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) x1[m][n][i] += t1[m][n][i];
        if (x2)
#pragma unroll
          for (int i = 0; i < 4; ++i) x2[m][i] += t2[m][i];
      }
    };
    const float* s0 = f + wc * (DK / 8);
    const float* u8 = f + L::u + wc * 8;
    zero();
    block_products<false, false, N, true>(t1, t2, f + L::dy + wr * 32, kPU, s0, L::PS, u8, kPU, g, t);
    add(d1, da);
    zero();
    block_products<X, true, N, true>(t1, t2, sDO + wr * 32 * L::PO, L::PO, s0, L::PS, u8, kPU, g, t);
    add(dqa, dp);
    zero();
    block_products<false, false, N, false>(t1, t2, f + L::u + wr * 32, kPU, s0 + L::ds, L::PS, u8, kPU, g, t);
    add(d3, nullptr);
    __syncthreads();
  }
  if (tid == 0) next_item = valid(asked);
  __syncthreads();
  const uint32_t next = next_item;
  const uint32_t bh = item / NC, b = bh / Hv, h = bh - b * Hv, hk = h / (Hv / a.Hk);
  const int64_t t0 = (int64_t)(item - bh * NC) * kC;
  const int rows = (int)min((int64_t)kC, row_length(a, b) - t0);
  // the next chunk's first block goes to one set, E, F and the gradients to the other
  float* sE = F + ((blk & 1) ^ 1) * L::set;
  float* sF = sE + L::f;
  if (next < items) {
    if (tid == 0) load(next, 0, blk & 1);
    blank(0, blk & 1);
    locate(next);
    fetch(0);
  }
  there &= stage_wait(&bars[2], nth & 1);
  if (!there) yv = ss = d1[0][0][0] = dqa[0][0][0] = __int_as_float(0x7fffffff);

  // dot products over the key rows
#pragma unroll
  for (int r = 0; r < 4; ++r) {   // row wr * 32 + (r >> 1) * 16 + (r & 1) * 8 + g
    const int i = wr * 32 + (r >> 1) * 16 + (r & 1) * 8 + g;
    float x1 = 0.f, xq = 0.f, x3 = 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int col = wc * (DK / 8) + n * 8 + 2 * t;
      const float2 kk = pair(K + i * L::PK + col), qq = pair(Q + i * L::PK + col);
      const int e = 2 * (r & 1);
      x1 += kk.x * d1[r >> 1][n][e] + kk.y * d1[r >> 1][n][e + 1];
      xq += qq.x * dqa[r >> 1][n][e] + qq.y * dqa[r >> 1][n][e + 1];
      x3 += kk.x * d3[r >> 1][n][e] + kk.y * d3[r >> 1][n][e + 1];
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      x1 += __shfl_xor_sync(0xffffffffu, x1, o);
      xq += __shfl_xor_sync(0xffffffffu, xq, o);
      x3 += __shfl_xor_sync(0xffffffffu, x3, o);
    }
    if (t == 0) {
      parts[(10 + wc) * kC + i] = x1;
      parts[(18 + wc) * kC + i] = xq;
      parts[(26 + wc) * kC + i] = x3;
    }
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) yv += __shfl_xor_sync(0xffffffffu, yv, o);
  if ((tid & 7) == 0) parts[34 * kC + tok] = yv;
  ss = warp_sum(ss);
  if (lane == 0) parts[35 * kC + warp] = ss;

  // E, F and the sums of dP P + dA A, dA (A/beta)
  float cs[2] = {0.f, 0.f};
  float bsum[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = wr * 32 + (r >> 1) * 16 + (r & 1) * 8 + g;
    const int j0 = wc * 8 + 2 * t;
    float rs = 0.f, bsr = 0.f;
    float2 pm = make_float2(0.f, 0.f), bm = pm, ev = pm, fv = pm;
    if (wc <= (i >> 3)) {
      const int at = tri(i >> 3, wc) + (i & 7) * 8 + 2 * t;
      pm = *reinterpret_cast<const float2*>(Pm + at);
      bm = *reinterpret_cast<const float2*>(Bm + at);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int j = j0 + e;
      if (j <= i) {
        const float gam = expf((gHi[i] - gHi[j]) + (gLo[i] - gLo[j]));
        const float dpv = dp[r >> 1][2 * (r & 1) + e];
        float m = dpv * (e ? pm.y : pm.x);
        (e ? ev.y : ev.x) = a.scale * gam * dpv;
        if (j < i) {
          const float dav = -da[r >> 1][2 * (r & 1) + e];
          const float nb = dav * (e ? bm.y : bm.x);
          bsr += nb;
          m = fmaf(beta[i], nb, m);
          (e ? fv.y : fv.x) = beta[i] * gam * dav;
        }
        rs += m;
        cs[e] += m;
      }
    }
    *reinterpret_cast<float2*>(sE + i * L::PE + j0) = ev;
    *reinterpret_cast<float2*>(sF + i * L::PE + j0) = fv;
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      rs += __shfl_xor_sync(0xffffffffu, rs, o);
      bsr += __shfl_xor_sync(0xffffffffu, bsr, o);
    }
    if (t == 0) parts[wc * kC + i] = rs;
    bsum[r] = bsr;
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    float x = cs[e];
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if (g == 0) parts[(8 + wr) * kC + wc * 8 + 2 * t + e] = x;
  }
  __syncthreads();

  // gates: thread i < 64 has token i
  float dG = 0.f, dbe = 0.f, tailC = 0.f;
  if (tid < kC) {
    const int i = tid;
    float c1 = 0.f, cq = 0.f, c3 = 0.f, rs = 0.f;
    for (int p = 0; p < 8; ++p) {
      rs += parts[p * kC + i];
      c1 += parts[(10 + p) * kC + i];
      cq += parts[(18 + p) * kC + i];
      c3 += parts[(26 + p) * kC + i];
    }
    const float cc = parts[8 * kC + i] + parts[9 * kC + i];
    const float L3 = eD[i] * c3;
    dbe = parts[34 * kC + i] - eG[i] * c1;
    dG = (rs - cc) - beta[i] * eG[i] * c1 + a.scale * eG[i] * cq - L3;
    tailC = L3;
  }
  __syncthreads();
  if (t == 0) {
#pragma unroll
    for (int r = 0; r < 4; ++r) parts[wc * kC + wr * 32 + (r >> 1) * 16 + (r & 1) * 8 + g] = bsum[r];
  }
  if (tid < kC) {
    parts[8 * kC + tid] = dG;
    parts[9 * kC + tid] = tailC;
  }
  __syncthreads();
  if (tid < kC) {
    for (int p = 0; p < 8; ++p) dbe += parts[p * kC + tid];
    if (tid < rows) a.dbeta[((int64_t)b * a.T + t0 + tid) * a.Hv + h] = dbe;
  }
  if (warp == 2) {   // dg: sums of dG from the end; the chunk's last G takes the tail terms
    const float* sdG = parts + 8 * kC;
    const float* sTail = parts + 9 * kC;
    const float x0 = sdG[2 * lane], x1 = sdG[2 * lane + 1];
    float tail = warp_sum(sTail[2 * lane] + sTail[2 * lane + 1]);
    float in = 0.f;
    for (int p = 0; p < kT / 32; ++p) in += parts[35 * kC + p];
    tail += eG[kC - 1] * in;
    float s = x0 + x1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float y = __shfl_down_sync(0xffffffffu, s, o);
      if (lane + o < 32) s += y;
    }
    const float e0 = s + tail, e1 = (s - x0) + tail;
    if (2 * lane < rows) a.dg[((int64_t)b * a.T + t0 + 2 * lane) * a.Hv + h] = e0;
    if (2 * lane + 1 < rows) a.dg[((int64_t)b * a.T + t0 + 2 * lane + 1) * a.Hv + h] = e1;
  }

  // dQ and dK on top of the parts that came through the state
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = wr * 32 + m * 16 + g + 8 * (i >> 1);
        dqa[m][n][i] *= a.scale * eG[r];
        d1[m][n][i] = fmaf(-beta[r] * eG[r], d1[m][n][i], eD[r] * d3[m][n][i]);
      }
  // sums of their own, added in one rounding
  float (*ek)[N][4] = d3;      // E^T Q + (F + F^T) K
  float eq[2][N][4];           // E K
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < N; ++n) {
      clear(ek[m][n]);
      clear(eq[m][n]);
    }
#pragma unroll 2
  for (int ks = 0; ks < 8; ++ks) {
    const int c0 = ks * 8 + 2 * t;
    float2 kk[N], qq[N];
    tiles_by_row<N>(kk, K + ks * 8 * L::PK + wc * (DK / 8), L::PK, lane);
    tiles_by_row<N>(qq, Q + ks * 8 * L::PK + wc * (DK / 8), L::PK, lane);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int i0 = wr * 32 + m * 16, i = i0 + g;
      float hi[4], lo[4];
      auto prepare = [&](const float* x) {
        if (SHORT) {
#pragma unroll
          for (int e = 0; e < 4; ++e) hi[e] = tf32(x[e]);
        } else {
          split4(x, hi, lo);
        }
      };
      auto product = [&](float (*c)[4], const float2* y) {
        if (SHORT) {
#pragma unroll
          for (int n = 0; n < N; ++n) mma(c[n], hi, y[n].x, y[n].y);
        } else {
          mma_split<X, N>(c, hi, lo, y);
        }
      };
      if (ks * 8 <= i0 + 15) {           // E is lower triangular
        const float2 p0 = pair(sE + i * L::PE + c0), p1 = pair(sE + (i + 8) * L::PE + c0);
        const float x[4] = {p0.x, p1.x, p0.y, p1.y};
        prepare(x);
        product(eq[m], kk);
      }
      if (ks * 8 + 7 >= i0) {
        const float* et = sE + c0 * L::PE + i;
        const float x[4] = {et[0], et[8], et[L::PE], et[L::PE + 8]};
        prepare(x);
        product(ek[m], qq);
      }
      {
        const float2 f0 = pair(sF + i * L::PE + c0), f1 = pair(sF + (i + 8) * L::PE + c0);
        const float* ft = sF + c0 * L::PE + i;
        const float x[4] = {f0.x + ft[0], f1.x + ft[8], f0.y + ft[L::PE], f1.y + ft[L::PE + 8]};
        prepare(x);
        product(ek[m], kk);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        dqa[m][n][i] += eq[m][n][i];
        d1[m][n][i] += ek[m][n][i];
      }
  __syncthreads();      // K, Q, E and F are free
  if (tid == 0 && next < items) load_chunk(next);
  auto finish = [&](auto* dq, auto* dk, int heads, int ho) {
    using O = typename std::remove_pointer<decltype(dq)>::type;
    O* sm = reinterpret_cast<O*>(sE);
    const int64_t at = (((int64_t)b * a.T + t0) * heads + ho) * a.dk, stride = (int64_t)heads * a.dk;
    const bool vec = a.dk % (16 / (int)sizeof(O)) == 0 && (reinterpret_cast<uintptr_t>(dq) & 15) == 0 &&
                     (reinterpret_cast<uintptr_t>(dk) & 15) == 0;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      if (which) __syncthreads();
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const float* c = which ? d1[m][n] : dqa[m][n];
            O* o = sm + (wr * 32 + m * 16 + g + 8 * hf) * L::PK + wc * (DK / 8) + n * 8 + 2 * t;
            o[0] = from_f<O>(c[2 * hf]);
            o[1] = from_f<O>(c[2 * hf + 1]);
          }
      __syncthreads();
      store_rows<O>((which ? dk : dq) + at, stride, sm, L::PK, rows, a.dk, vec, tid, kT);
    }
  };
  if (a.Hk != a.Hv) finish(a.dq32, a.dk32, a.Hv, h);
  else finish(static_cast<E*>(a.dq), static_cast<E*>(a.dk_), a.Hk, hk);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // bulk copies will follow these writes
  __syncthreads();      // the set is free
  item = next;
  }
}

// Gradients of keys and queries that several value heads share: 32-bit sums in head order.
template <typename E>
__global__ void __launch_bounds__(256) head_sum_kernel(Args a) {
  const int group = a.Hv / a.Hk;
  const int64_t n = (int64_t)a.B * a.T * a.Hk * a.dk;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / a.dk, tb = row / a.Hk, tok = tb % a.T;
    const int c = (int)(i - row * a.dk), b = (int)(tb / a.T);
    float xq = 0.f, xk = 0.f;
    if (tok < row_length(a, b)) {
      const int64_t at = row * group * a.dk + c;
      for (int p = 0; p < group; ++p) {
        xq += a.dq32[at + (int64_t)p * a.dk];
        xk += a.dk32[at + (int64_t)p * a.dk];
      }
    }
    static_cast<E*>(a.dq)[i] = from_f<E>(xq);
    static_cast<E*>(a.dk_)[i] = from_f<E>(xk);
  }
}

template <typename E, int DK>
static int launch_chunks_typed(const Args& a, cudaStream_t st) {
  const size_t bytes = BackChunkLayout<E, DK>::bytes;
  static std::atomic<uint64_t> seen;
  int rc = allow_smem(backward_chunk_kernel<E, DK>, bytes, seen);
  if (rc != BSX_OK) return rc;
  const int64_t items = (int64_t)a.B * a.Hv * a.NC;
  const int sms = sm_count();
  backward_chunk_kernel<E, DK><<<(unsigned)(items < sms ? items : sms), kChunkThreads, bytes, st>>>(a);
  BSX_LAUNCH_CHECK("plastic backward_chunk_kernel");
  if (a.Hk != a.Hv) {
    const int64_t n = (int64_t)a.B * a.T * a.Hk * a.dk;
    const int64_t want = (n + 255) / 256, most = 16ll * sm_count();
    head_sum_kernel<E><<<(unsigned)(want < most ? want : most), 256, 0, st>>>(a);
    BSX_LAUNCH_CHECK("plastic head_sum_kernel");
  }
  return BSX_OK;
}

int launch_backward_scan(const Args& a, int dtype, cudaStream_t st) {
  const bool narrow = a.dk <= 64;
  if (dtype == BSX_T_F32) return narrow ? launch_scan_typed<float, 64>(a, st) : launch_scan_typed<float, 128>(a, st);
  if (dtype == BSX_T_BF16)
    return narrow ? launch_scan_typed<__nv_bfloat16, 64>(a, st) : launch_scan_typed<__nv_bfloat16, 128>(a, st);
  return narrow ? launch_scan_typed<__half, 64>(a, st) : launch_scan_typed<__half, 128>(a, st);
}

int launch_backward_chunks(const Args& a, int dtype, cudaStream_t st) {
  const bool narrow = a.dk <= 64;
  if (dtype == BSX_T_F32) return narrow ? launch_chunks_typed<float, 64>(a, st) : launch_chunks_typed<float, 128>(a, st);
  if (dtype == BSX_T_BF16)
    return narrow ? launch_chunks_typed<__nv_bfloat16, 64>(a, st) : launch_chunks_typed<__nv_bfloat16, 128>(a, st);
  return narrow ? launch_chunks_typed<__half, 64>(a, st) : launch_chunks_typed<__half, 128>(a, st);
}

}  // namespace plastic
}  // namespace bsx
