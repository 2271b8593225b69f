// Gated delta rule: the pass over the chunks that carries the state, and the outputs.
//
// Four warps own 16 value columns of one head (a group); a block has one to four groups that share the staged tiles
// of K, Q, T and P (two bulk copies by one thread, a chunk ahead where two sets fit; a copy for every row of the
// tiles took 4300 of a chunk's 11000 clocks).  V goes from global memory to registers, a chunk ahead.  The state is held
// transposed in registers, each warp a quarter of the key rows, as accumulator tiles (16 x 8).  All products of a chunk have the value columns as their
// rows, so that one product's accumulator is the next one's left operand:
//   R^T = S^T K^T -> Y^T = beta (V^T - e^G R^T) -> U^T = Y^T T^T -> S^T = e^{G_C} S^T + (e^{G_C-G} U)^T K,
//   O^T = scale e^G S^T Q^T + U^T P^T.
// R, Y, U and O are divided among the warps by tokens (8-token tiles w and 7 - w, whose triangular products are together
// equally long for every w), the state by key rows; S, Y and U change hands through shared memory, already split into
// the parts that the instructions take.
// What a chunk adds to the state is summed apart and added in one rounding, because the tensor unit's sums are cut,
// not rounded, and would drift over many chunks.
//
// Bound by the chain of its phases: a chunk is four exchanges between the warps.  bf16, heads of 128 x 128: 8192 tokens of
// one row and 16 heads 289 us (one group a block, 2.3 us a chunk); 4 x 2048 tokens of 16 heads 204 us (four groups a block:
// shared memory 56 %, tensor unit 46 % busy), 181 us where it leaves the states for the reverse pass instead of the
// outputs.  Eight warps to a group measured no better (330 us for the first).
#include "plastic.cuh"

namespace bsx {
namespace plastic {

template <typename E, int DK>
struct ScanLayout {
  static constexpr int PK = DK + 8;
  static constexpr size_t tile = (size_t)kC * PK * sizeof(E);
  static constexpr uint32_t rec = (2 * kTri + 3 * kC) * sizeof(float);
  static constexpr size_t set = 2 * tile + rec;        // K, Q, record (T, P, vectors)
  // a group's exchange: S (then U, split and plain), Y
  static constexpr size_t s_bytes = (size_t)DK * 128 > 12288 ? (size_t)DK * 128 : 12288;
  static constexpr size_t group = s_bytes + 8192;
  static constexpr size_t bytes(int groups, int stages) { return stages * set + groups * group; }
};

// U^T = Y^T T^T of token tiles W and 7 - W: nine tile products whatever W is, all known to the compiler.
template <int W>
__device__ __forceinline__ void solve_own(const float4* gY, const float* Tm, int lane, float (*u)[4]) {
  float h[2][4], x[2][4], y[2][4];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    clear(h[e]);
    clear(x[e]);
    clear(y[e]);
  }
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) {
    if (ks > W && ks > 7 - W) continue;
    float hi[4], lo[4];
    get_split(gY, ks, lane, hi, lo);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int n = e ? 7 - W : W;
      if (ks > n) continue;
      const float2 tt = pair(Tm + tri(n, ks) + lane * 2);
      float h0, l0, h1, l1;
      split(tt.x, h0, l0);
      split(tt.y, h1, l1);
      mma(x[e], lo, h0, h1);
      mma(y[e], hi, l0, l1);
      mma(h[e], hi, h0, h1);
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int i = 0; i < 4; ++i) u[e][i] = h[e][i] + (x[e][i] + y[e][i]);
}

// o += U^T P^T of the same token tiles.
template <int W, bool SHORT>
__device__ __forceinline__ void answer_own(const float4* gU, const float* Pm, int lane, float (*o)[4]) {
  float h[2][4], x[2][4];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    clear(h[e]);
    clear(x[e]);
  }
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) {
    if (ks > W && ks > 7 - W) continue;
    const float4 v = gU[ks * 32 + lane];
    const float c[4] = {v.x, v.y, v.z, v.w};
    float hi[4], lo[4];
    if (SHORT) {
#pragma unroll
      for (int i = 0; i < 4; ++i) hi[i] = tf32(c[i]);
    } else {
      split4(c, hi, lo);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int n = e ? 7 - W : W;
      if (ks > n) continue;
      const float2 pp = pair(Pm + tri(n, ks) + lane * 2);
      if (SHORT) mma(h[e], hi, tf32(pp.x), tf32(pp.y));
      else mma_apart<false>(h[e], x[e], hi, lo, pp);
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[e][i] += SHORT ? h[e][i] : h[e][i] + x[e][i];
}

template <typename E, int DK, bool OUT, bool SAVE, int THREADS>
__global__ void __launch_bounds__(THREADS, 1) scan_kernel(Args a, int groups, int stages) {
  using L = ScanLayout<E, DK>;
  constexpr bool X = IsExact<E>::value;
  constexpr bool SHORT = IsShort<E>::value;   // the last products before the outputs take the hi parts alone
  constexpr int DKW = DK / 4, NT = DKW / 8;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ __align__(8) uint64_t bars[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int grp = warp >> 2, w = warp & 3;
  const int per_head = (a.dv + 16 * groups - 1) / (16 * groups);
  const int bh = blockIdx.x / per_head, vb = (blockIdx.x - bh * per_head) * groups * 16;
  const int b = bh / a.Hv, h = bh - b * a.Hv, hk = h / (a.Hv / a.Hk);
  const int len = row_length(a, b), nc = (len + kC - 1) / kC;
  float4* gS = reinterpret_cast<float4*>(smem + stages * L::set + grp * L::group);   // S; then U split (8 KB), U plain
  float4* gU = gS + 512;
  float4* gY = reinterpret_cast<float4*>(reinterpret_cast<unsigned char*>(gS) + L::s_bytes);
  const int d0 = vb + grp * 16 + g;  // value columns d0 and d0 + 8
  const bool in0 = d0 < a.dv, in1 = d0 + 8 < a.dv;
  const int kb = w * DKW;            // first key row of this warp
  const int own[2] = {w, 7 - w};     // token tiles of this warp

  float s[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int kr = kb + n * 8 + 2 * t + (i & 1), d = d0 + (i >> 1) * 8;
      s[n][i] = (a.initial && kr < a.dk && d < a.dv) ? a.initial[((int64_t)bh * a.dk + kr) * a.dv + d] : 0.f;
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
  const E* vp = static_cast<const E*>(a.v) + b * a.vs[0] + h * a.vs[2] + d0;
  E vn[2][4];
  if (nc > 0) {
    if (tid == 0) load(0, 0);
    fetch_own(vn, vp, a.vs[1], own, t, len, in0, in1);
  }
  for (int c = 0; c < nc; ++c) {
    const int buf = stages == 2 ? (c & 1) : 0;
    if (stages == 2 && c + 1 < nc && tid == 0) load(c + 1, buf ^ 1);
    const bool there = stage_wait(&bars[buf], stages == 2 ? ((c >> 1) & 1) : (c & 1));
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

    if (SAVE) {  // the state before this chunk, transposed
      float* Sn = a.Sn + ci * a.dv * (DK + 4);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
          if (d0 + 8 * hf < a.dv)
            *reinterpret_cast<float2*>(Sn + (d0 + 8 * hf) * (DK + 4) + kb + n * 8 + 2 * t) =
                make_float2(s[n][2 * hf], s[n][2 * hf + 1]);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if constexpr (SHORT) put_parts(gS, w * NT + n, lane, s[n]);
      else put_split(gS, w * NT + n, lane, s[n]);
    }
    group_sync(grp);

    // R^T and S^T Q^T of this warp's tokens
    float rh[2][4], rl[2][4], zh[2][4], zl[2][4];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      clear(rh[e]);
      clear(rl[e]);
      clear(zh[e]);
      clear(zl[e]);
    }
    if constexpr (SHORT) {
#pragma unroll
      for (int kp = 0; kp < DK / 16; ++kp) {
        const uint4 x[3] = {get_part(gS, kp, 0, lane), get_part(gS, kp, 1, lane), get_part(gS, kp, 2, lane)};
        state_times<DK, L::PK, false>(rh, rl, x, K, kp, own, g, t);
        if (OUT) state_times<DK, L::PK, true>(zh, zl, x, Q, kp, own, g, t);
      }
    } else {
#pragma unroll
      for (int ks = 0; ks < DK / 8; ++ks) {
        float hi[4], lo[4];
        get_split(gS, ks, lane, hi, lo);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int at = (own[e] * 8 + g) * L::PK + ks * 8 + 2 * t;
          mma_apart<X>(rh[e], rl[e], hi, lo, pair(K + at));
          if (OUT) mma_apart<X>(zh[e], zl[e], hi, lo, pair(Q + at));
        }
      }
    }
    // Y^T = beta (V^T - e^G R^T)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int tok = own[e] * 8 + 2 * t;
      const float2 eg = pair(eG + tok), be = pair(beta + tok);
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        y[i] = ((i & 1) ? be.y : be.x) * (to_f<E>(vn[e][i]) - ((i & 1) ? eg.y : eg.x) * (rh[e][i] + rl[e][i]));
      put_split(gY, own[e], lane, y);
    }
    if (c + 1 < nc) fetch_own(vn, vp + (t0 + kC) * a.vs[1], a.vs[1], own, t, len - (c + 1) * kC, in0, in1);
    group_sync(grp);

    float u[2][4];
    switch (w) {
      case 0: solve_own<0>(gY, Tm, lane, u); break;
      case 1: solve_own<1>(gY, Tm, lane, u); break;
      case 2: solve_own<2>(gY, Tm, lane, u); break;
      default: solve_own<3>(gY, Tm, lane, u);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int tok = own[e] * 8 + 2 * t;
      if (SAVE) {
        float* U = a.U + ci * a.dv * kPU;
        if (in0) *reinterpret_cast<float2*>(U + d0 * kPU + tok) = make_float2(u[e][0], u[e][1]);
        if (in1) *reinterpret_cast<float2*>(U + (d0 + 8) * kPU + tok) = make_float2(u[e][2], u[e][3]);
      }
      if (OUT) gU[own[e] * 32 + lane] = make_float4(u[e][0], u[e][2], u[e][1], u[e][3]);
      const float2 ed = pair(eD + tok);
      u[e][0] *= ed.x;
      u[e][1] *= ed.y;
      u[e][2] *= ed.x;
      u[e][3] *= ed.y;
      if constexpr (SHORT) put_parts(gS, own[e], lane, u[e]);
      else put_split(gS, own[e], lane, u[e]);
    }
    group_sync(grp);

    // S^T = e^{G_C} S^T + (e^{G_C-G} U)^T K
    float ah[NT][4], al[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      clear(ah[n]);
      clear(al[n]);
    }
    if constexpr (SHORT) {
#pragma unroll
      for (int tp = 0; tp < 4; ++tp) {
        const uint4 x[3] = {get_part(gS, tp, 0, lane), get_part(gS, tp, 1, lane), get_part(gS, tp, 2, lane)};
        update_state<NT, L::PK>(ah, al, x, K + tp * 16 * L::PK + kb, lane);
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
      }
    }
    const float eC = eG[kC - 1];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] = fmaf(eC, s[n][i], ah[n][i] + al[n][i]);

    if (OUT) {  // O^T of this warp's tokens
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 eg = pair(eG + own[e] * 8 + 2 * t);
#pragma unroll
        for (int i = 0; i < 4; ++i) zh[e][i] = a.scale * ((i & 1) ? eg.y : eg.x) * (zh[e][i] + zl[e][i]);
      }
      switch (w) {
        case 0: answer_own<0, SHORT>(gU, Pm, lane, zh); break;
        case 1: answer_own<1, SHORT>(gU, Pm, lane, zh); break;
        case 2: answer_own<2, SHORT>(gU, Pm, lane, zh); break;
        default: answer_own<3, SHORT>(gU, Pm, lane, zh);
      }
      const int64_t ts = (int64_t)a.Hv * a.dv;
      E* op = static_cast<E*>(a.o) + ((int64_t)b * a.T + t0) * ts + (int64_t)h * a.dv + d0;
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int tok = own[e] * 8 + 2 * t + j;
          E* o = op + tok * ts;
          if (tok < len - c * kC) {
            if (in0) o[0] = from_f<E>(zh[e][j]);
            if (in1) o[8] = from_f<E>(zh[e][2 + j]);
          }
        }
    }
    __syncthreads();      // the tiles and the group's exchange are free
    if (stages == 1 && c + 1 < nc && tid == 0) load(c + 1, 0);
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

// Groups of 16 value columns to a block: as few as give every SM a block, since a chunk of one group takes least time;
// more where there are more groups than that (they share the staged tiles and hide each other's waits).
int scan_groups(const Args& a, int sms) {
  const int most = (a.dv + 15) / 16;
  const int64_t total = (int64_t)a.B * a.Hv * most;
  return total <= sms || most < 2 ? 1 : (total <= 2 * (int64_t)sms || most < 4 ? 2 : 4);
}

template <typename E, int DK, bool OUT, bool SAVE, int THREADS>
static int launch_threads(const Args& a, int groups, cudaStream_t st) {
  using L = ScanLayout<E, DK>;
  static std::atomic<uint64_t> seen;
  int rc = allow_smem(scan_kernel<E, DK, OUT, SAVE, THREADS>, kMaxSmem, seen);
  if (rc != BSX_OK) return rc;
  const int stages = L::bytes(groups, 2) <= kMaxSmem ? 2 : 1;
  const int per_head = (a.dv + 16 * groups - 1) / (16 * groups);
  const unsigned grid = (unsigned)((int64_t)a.B * a.Hv * per_head);
  scan_kernel<E, DK, OUT, SAVE, THREADS><<<grid, groups * 128, L::bytes(groups, stages), st>>>(a, groups, stages);
  BSX_LAUNCH_CHECK("plastic scan_kernel");
  return BSX_OK;
}

template <typename E, int DK, bool OUT, bool SAVE>
static int launch_one(const Args& a, cudaStream_t st) {
  const int sms = sm_count();
  if (sms <= 0) return fail(BSX_ERR_CUDA, "no CUDA device");
  const int groups = scan_groups(a, sms);
  return groups == 4 ? launch_threads<E, DK, OUT, SAVE, 512>(a, groups, st)
                     : launch_threads<E, DK, OUT, SAVE, 256>(a, groups, st);
}

template <typename E>
static int launch_typed(const Args& a, bool save, cudaStream_t st) {
  if (a.dk <= 64) return save ? launch_one<E, 64, false, true>(a, st) : launch_one<E, 64, true, false>(a, st);
  return save ? launch_one<E, 128, false, true>(a, st) : launch_one<E, 128, true, false>(a, st);
}

int launch_scan(const Args& a, int dtype, bool save, cudaStream_t st) {
  if (dtype == BSX_T_F32) return launch_typed<float>(a, save, st);
  if (dtype == BSX_T_BF16) return launch_typed<__nv_bfloat16>(a, save, st);
  return launch_typed<__half>(a, save, st);
}

}  // namespace plastic
}  // namespace bsx
