// Gated delta rule: the pass over the chunks that carries the state, and the outputs.
//
// The state is held transposed in registers: WS warps own 16 value columns of one head, each of them DK / WS key
// rows, as accumulator tiles (16 x 8).  Every product of a chunk has the value columns as its rows, so the
// accumulator of one is the left operand of the next without a pass through shared memory:
//   R^T = S^T K^T -> Y^T = beta (V^T - e^G R^T) -> U^T = Y^T T^T -> S^T = e^{G_C} S^T + (e^{G_C-G} U)^T K,
//   O^T = scale e^G S^T Q^T + U^T P^T.
// Warps share nothing but the staged tiles of K, Q, T, P and V (copied one chunk ahead where two sets fit); with
// WS > 1 the partial sums of R and S^T Q^T over the key rows meet in shared memory, added in warp order.
// What a chunk adds to the state is summed apart and added in one rounding, because the tensor unit's sums are cut,
// not rounded, and would drift over many chunks.
#include "plastic.cuh"

namespace bsx {
namespace plastic {

template <typename E, int DK, bool OUT>
struct ScanLayout {
  static constexpr int PK = DK + 8, PT = kC + 8;
  static constexpr size_t tile = (size_t)kC * PK * sizeof(E);
  static constexpr size_t tri = (size_t)kC * PT * sizeof(float);
  static constexpr int stages = (sizeof(E) == 4 && DK == 128 && OUT) ? 1 : 2;
  static constexpr size_t q_off = tile, t_off = tile * (OUT ? 2 : 1), p_off = t_off + tri,
                          vec_off = t_off + tri * (OUT ? 2 : 1), v_off = vec_off + 3 * kC * sizeof(float);
  static size_t v_bytes(int groups) { return (size_t)kC * (groups * 16 + 8) * sizeof(E); }
  static size_t red_bytes(int groups, int ws) { return ws > 1 ? (size_t)groups * ws * (OUT ? 64 : 32) * 32 * 4 : 0; }
  static size_t bytes(int groups, int ws) { return stages * (v_off + v_bytes(groups)) + red_bytes(groups, ws); }
};

template <int WS>
__device__ __forceinline__ void group_sync(int grp) {
  asm volatile("bar.sync %0, %1;" ::"r"(grp + 1), "n"(WS * 32) : "memory");
}

template <typename E, int DK, int WS, bool OUT, bool SAVE>
__global__ void __launch_bounds__(256) scan_kernel(Args a, int groups) {
  using L = ScanLayout<E, DK, OUT>;
  constexpr bool X = IsExact<E>::value;
  constexpr bool SHORT = IsShort<E>::value;   // the last products before the outputs take the hi parts alone
  constexpr int DKW = DK / WS, NT = DKW / 8, NB = NT < 4 ? NT : 4;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, nthr = blockDim.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int grp = warp / WS, w = warp - grp * WS;
  const int per_head = (a.dv + 16 * groups - 1) / (16 * groups);
  const int bh = blockIdx.x / per_head, vb = (blockIdx.x - bh * per_head) * groups * 16;
  const int b = bh / a.Hv, h = bh - b * a.Hv, hk = h / (a.Hv / a.Hk);
  const int len = row_length(a, b), nc = (len + kC - 1) / kC;
  const int PV = groups * 16 + 8;
  const size_t set = L::v_off + (size_t)kC * PV * sizeof(E);
  float* red = reinterpret_cast<float*>(smem + L::stages * set);
  const int d0 = vb + grp * 16 + g;  // value columns d0 and d0 + 8
  const int kb = w * DKW;            // first key row of this warp

  const E* kp = static_cast<const E*>(a.k) + b * a.ks[0] + hk * a.ks[2];
  const E* qp = static_cast<const E*>(a.q) + b * a.qs[0] + hk * a.qs[2];
  const E* vp = static_cast<const E*>(a.v) + b * a.vs[0] + h * a.vs[2] + vb;

  float s[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int kr = kb + n * 8 + 2 * t + (i & 1), d = d0 + (i >> 1) * 8;
      s[n][i] = (a.initial && kr < a.dk && d < a.dv) ? a.initial[((int64_t)bh * a.dk + kr) * a.dv + d] : 0.f;
    }

  auto load = [&](int c, int buf) {
    unsigned char* base = smem + buf * set;
    const int64_t t0 = (int64_t)c * kC;
    const int rows = min(kC, len - c * kC);
    const int64_t ci = (int64_t)bh * a.NC + c;
    stage(reinterpret_cast<E*>(base), L::PK, kp + t0 * a.ks[1], a.ks[1], rows, a.dk, DK, a.vec_qk, tid, nthr);
    if (OUT) {
      stage(reinterpret_cast<E*>(base + L::q_off), L::PK, qp + t0 * a.qs[1], a.qs[1], rows, a.dk, DK, a.vec_qk, tid, nthr);
      stage_lower(reinterpret_cast<float*>(base + L::p_off), L::PT, a.Pm + ci * kC * kC, tid, nthr);
    }
    stage_lower(reinterpret_cast<float*>(base + L::t_off), L::PT, a.Tm + ci * kC * kC, tid, nthr);
    for (int i = tid; i < 3 * kC / 4; i += nthr)
      cp16(base + L::vec_off + i * 16, a.vec + ci * kVec + i * 4, true);
    stage(reinterpret_cast<E*>(base + L::v_off), PV, vp + t0 * a.vs[1], a.vs[1], rows, min(a.dv - vb, groups * 16),
          groups * 16, a.vec_v, tid, nthr);
    cp_commit();
  };

  if (L::stages == 2 && nc > 0) load(0, 0);
  for (int c = 0; c < nc; ++c) {
    const int buf = L::stages == 2 ? (c & 1) : 0;
    if (L::stages == 2) {
      if (c + 1 < nc) {
        load(c + 1, buf ^ 1);
        cp_wait<1>();
      } else {
        cp_wait<0>();
      }
    } else {
      load(c, 0);
      cp_wait<0>();
    }
    __syncthreads();
    const unsigned char* base = smem + buf * set;
    const E* K = reinterpret_cast<const E*>(base);
    const E* Q = reinterpret_cast<const E*>(base + L::q_off);
    const float* Tm = reinterpret_cast<const float*>(base + L::t_off);
    const float* Pm = reinterpret_cast<const float*>(base + L::p_off);
    const float* eG = reinterpret_cast<const float*>(base + L::vec_off);
    const float* eD = eG + kC;
    const float* beta = eG + 2 * kC;
    const E* V = reinterpret_cast<const E*>(base + L::v_off) + grp * 16;
    const int64_t ci = (int64_t)bh * a.NC + c;
    const int64_t t0 = (int64_t)c * kC;

    if (SAVE) {  // the state before this chunk, transposed
      float* Sn = a.Sn + ci * a.dv * DK;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
          if (d0 + 8 * hf < a.dv)
            *reinterpret_cast<float2*>(Sn + (int64_t)(d0 + 8 * hf) * DK + kb + n * 8 + 2 * t) =
                make_float2(s[n][2 * hf], s[n][2 * hf + 1]);
    }

    // R^T and S^T Q^T over this warp's key rows
    float r[8][4], z[8][4];
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) r[n][i] = z[n][i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < NT; ++ks) {
      float x[4], hi[4], lo[4], rn[4];
      as_left(s[ks], x);
      split4(x, hi, lo);
      if (OUT && SHORT)
#pragma unroll
        for (int i = 0; i < 4; ++i) rn[i] = tf32(x[i]);
      const int col = kb + ks * 8 + 2 * t;
      float2 kk[8];
#pragma unroll
      for (int n = 0; n < 8; ++n) kk[n] = pair(K + (n * 8 + g) * L::PK + col);
      mma_split<X, 8>(r, hi, lo, kk);
      if (OUT) {
#pragma unroll
        for (int n = 0; n < 8; ++n) kk[n] = pair(Q + (n * 8 + g) * L::PK + col);
        if (SHORT) {
#pragma unroll
          for (int n = 0; n < 8; ++n) mma(z[n], rn, kk[n].x, kk[n].y);
        } else {
          mma_split<X, 8>(z, hi, lo, kk);
        }
      }
    }
    if (WS > 1) {
      constexpr int NR = OUT ? 64 : 32;
      float* mine = red + (size_t)grp * WS * NR * 32 + lane;   // free since the barrier at the chunk's end
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          mine[(w * NR + n * 4 + i) * 32] = r[n][i];
          if (OUT) mine[(w * NR + 32 + n * 4 + i) * 32] = z[n][i];
        }
      group_sync<WS>(grp);
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = mine[(n * 4 + i) * 32], y = (OUT && n % WS == w) ? mine[(32 + n * 4 + i) * 32] : 0.f;
#pragma unroll
          for (int p = 1; p < WS; ++p) {
            x += mine[(p * NR + n * 4 + i) * 32];
            if (OUT && n % WS == w) y += mine[(p * NR + 32 + n * 4 + i) * 32];
          }
          r[n][i] = x;
          z[n][i] = y;
        }
    }

    // Y^T = beta (V^T - e^G R^T)
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const int tok = n * 8 + 2 * t;
      const float2 eg = pair(eG + tok), be = pair(beta + tok);
      r[n][0] = be.x * (to_f<E>(V[tok * PV + g]) - eg.x * r[n][0]);
      r[n][1] = be.y * (to_f<E>(V[(tok + 1) * PV + g]) - eg.y * r[n][1]);
      r[n][2] = be.x * (to_f<E>(V[tok * PV + g + 8]) - eg.x * r[n][2]);
      r[n][3] = be.y * (to_f<E>(V[(tok + 1) * PV + g + 8]) - eg.y * r[n][3]);
    }
    // U^T = Y^T T^T
    float u[8][4];
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) u[n][i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      float x[4], hi[4], lo[4];
      as_left(r[ks], x);
      split4(x, hi, lo);
      // column ks of tiles; those above the diagonal are zero
      float2 tt[8];
#pragma unroll
      for (int n = ks; n < 8; ++n) tt[n] = pair(Tm + (n * 8 + g) * L::PT + ks * 8 + 2 * t);
      float2 th[8], tl[8];
#pragma unroll
      for (int n = ks; n < 8; ++n) {
        split(tt[n].x, th[n].x, tl[n].x);
        split(tt[n].y, th[n].y, tl[n].y);
      }
#pragma unroll
      for (int n = ks; n < 8; ++n) mma(u[n], lo, th[n].x, th[n].y);
#pragma unroll
      for (int n = ks; n < 8; ++n) mma(u[n], hi, tl[n].x, tl[n].y);
#pragma unroll
      for (int n = ks; n < 8; ++n) mma(u[n], hi, th[n].x, th[n].y);
    }
    if (SAVE && w == 0) {
      float* U = a.U + ci * a.dv * kC;
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
          if (d0 + 8 * hf < a.dv)
            *reinterpret_cast<float2*>(U + (int64_t)(d0 + 8 * hf) * kC + n * 8 + 2 * t) =
                make_float2(u[n][2 * hf], u[n][2 * hf + 1]);
    }
    if (OUT) {  // O^T: this warp's tokens
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const float2 eg = pair(eG + n * 8 + 2 * t);
        z[n][0] *= a.scale * eg.x;
        z[n][1] *= a.scale * eg.y;
        z[n][2] *= a.scale * eg.x;
        z[n][3] *= a.scale * eg.y;
      }
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        float x[4], hi[4], lo[4];
        as_left(u[ks], x);
        if (SHORT) {
#pragma unroll
          for (int i = 0; i < 4; ++i) hi[i] = tf32(x[i]);
        } else {
          split4(x, hi, lo);
        }
#pragma unroll
        for (int n = ks; n < 8; ++n) {
          if (WS > 1 && n % WS != w) continue;
          const float2 pp = pair(Pm + (n * 8 + g) * L::PT + ks * 8 + 2 * t);
          if (SHORT) mma(z[n], hi, tf32(pp.x), tf32(pp.y));
          else mma_split<false, 1>(z + n, hi, lo, &pp);
        }
      }
      E* op = static_cast<E*>(a.o) + (((int64_t)b * a.T + t0) * a.Hv + h) * a.dv;
      const int64_t ts = (int64_t)a.Hv * a.dv;
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        if (WS > 1 && n % WS != w) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int tok = n * 8 + 2 * t + (i & 1), d = d0 + 8 * (i >> 1);
          if (t0 + tok < len && d < a.dv) op[tok * ts + d] = from_f<E>(z[n][i]);
        }
      }
    }
    // S^T = e^{G_C} S^T + (e^{G_C-G} U)^T K
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const float2 ed = pair(eD + n * 8 + 2 * t);
      u[n][0] *= ed.x;
      u[n][1] *= ed.y;
      u[n][2] *= ed.x;
      u[n][3] *= ed.y;
    }
    const float eC = eG[kC - 1];
#pragma unroll
    for (int n0 = 0; n0 < NT; n0 += NB) {
      float acc[NB][4];
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        float x[4], hi[4], lo[4];
        as_left(u[ks], x);
        split4(x, hi, lo);
        float2 kk[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          const E* kc = K + (ks * 8 + 2 * t) * L::PK + kb + (n0 + n) * 8 + g;
          kk[n] = make_float2(to_f<E>(kc[0]), to_f<E>(kc[L::PK]));
        }
        mma_split<X, NB>(acc, hi, lo, kk);
      }
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n0 + n][i] = fmaf(eC, s[n0 + n][i], acc[n][i]);
    }
    __syncthreads();
  }
  if (a.state && !SAVE) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int kr = kb + n * 8 + 2 * t + (i & 1), d = d0 + (i >> 1) * 8;
        if (kr < a.dk && d < a.dv) a.state[((int64_t)bh * a.dk + kr) * a.dv + d] = s[n][i];
      }
  }
}

template <typename E, int DK, int WS, bool OUT, bool SAVE>
static int launch_one(const Args& a, int groups, cudaStream_t st) {
  const size_t bytes = ScanLayout<E, DK, OUT>::bytes(groups, WS);
  static std::atomic<uint64_t> seen;
  int rc = allow_smem(scan_kernel<E, DK, WS, OUT, SAVE>, kMaxSmem, seen);
  if (rc != BSX_OK) return rc;
  const int per_head = (a.dv + 16 * groups - 1) / (16 * groups);
  const unsigned grid = (unsigned)((int64_t)a.B * a.Hv * per_head);
  scan_kernel<E, DK, WS, OUT, SAVE><<<grid, groups * WS * 32, bytes, st>>>(a, groups);
  BSX_LAUNCH_CHECK("plastic scan_kernel");
  return BSX_OK;
}

template <typename E, int DK>
static int launch_typed(const Args& a, bool save, cudaStream_t st) {
  const int64_t total = (int64_t)a.B * a.Hv * ((a.dv + 15) / 16);
  const int most = (a.dv + 15) / 16;
  int sms = sm_count();
  if (sms <= 0) return fail(BSX_ERR_CUDA, "no CUDA device");
  // Few 16-column groups: four warps share the key rows of each, one group a block, so that a chunk takes a quarter of
  // the steps; many groups: one warp each, up to four to a block.
  const int ws = total <= 2 * (int64_t)sms ? 4 : (total <= 4 * (int64_t)sms ? 2 : 1);
  int groups = ws == 4 ? 1 : 4;
  while (groups > most) groups >>= 1;
  while (groups > 1 && ScanLayout<E, DK, true>::bytes(groups, ws) > kMaxSmem) groups >>= 1;
#define BSX_SCAN(WS)                                                            \
  return save ? launch_one<E, DK, WS, false, true>(a, groups, st) : launch_one<E, DK, WS, true, false>(a, groups, st)
  if (ws == 4) BSX_SCAN(4);
  if (ws == 2) BSX_SCAN(2);
  BSX_SCAN(1);
#undef BSX_SCAN
}

template <typename E>
static int launch_width(const Args& a, bool save, cudaStream_t st) {
  return a.dk <= 64 ? launch_typed<E, 64>(a, save, st) : launch_typed<E, 128>(a, save, st);
}

int launch_scan(const Args& a, int dtype, bool save, cudaStream_t st) {
  if (dtype == BSX_T_F32) return launch_width<float>(a, save, st);
  if (dtype == BSX_T_BF16) return launch_width<__nv_bfloat16>(a, save, st);
  return launch_width<__half>(a, save, st);
}

}  // namespace plastic
}  // namespace bsx
