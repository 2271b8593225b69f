// Gated delta rule: C entry points, argument checks and the layout of the workspace.
#include "plastic.cuh"

namespace bsx {
namespace plastic {

int launch_step(const Args& a, int dtype, cudaStream_t st);

static int64_t chunks_of(int64_t tokens) { return (tokens + kC - 1) / kC; }
static int width_of(int dk) { return dk <= 64 ? 64 : 128; }

static size_t workspace(const bsx_delta_t* d, bool backward) {
  const int64_t n = d->batch * d->v_heads * chunks_of(d->tokens);
  const size_t size = d->dtype == BSX_T_F32 ? 4 : 2;
  size_t f = (size_t)n * kRecord + (size_t)(n / (d->v_heads / d->k_heads)) * (2 * kC * (width_of(d->dk) + 8) * size / 4);
  if (backward) {
    f += 4 + (size_t)n * (kTri + 2 * (size_t)d->dv * (width_of(d->dk) + 4 + kPU));
    if (d->k_heads != d->v_heads) f += 2 * (size_t)d->batch * d->tokens * d->v_heads * d->dk;
  }
  return f * sizeof(float);
}

// Clears the outputs behind each row's length, `per` bytes a token (sequences that go token by token; the chunks of others
// are cleared where they are prepared).
__global__ void __launch_bounds__(256) clear_tails_kernel(Args a, int64_t per) {
  for (int b = blockIdx.y; b < a.B; b += gridDim.y) {
    const int len = row_length(a, b);
    // whole elements of two bytes at least: to a 16-byte boundary, 16 bytes at a time, the rest
    uint16_t* x = reinterpret_cast<uint16_t*>(static_cast<unsigned char*>(a.o) + ((int64_t)b * a.T + len) * per);
    const int64_t n = (a.T - len) * per / 2;
    int64_t head = ((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / 2;
    head = head < n ? head : n;
    const int64_t body = (n - head) / 8;
    const int64_t first = blockIdx.x * 256ll + threadIdx.x, step = gridDim.x * 256ll;
    int4* y = reinterpret_cast<int4*>(x + head);
    for (int64_t i = first; i < body; i += step) y[i] = make_int4(0, 0, 0, 0);
    if (first < head) x[first] = 0;
    const int64_t tail = head + body * 8 + first;
    if (first < 8 && tail < n) x[tail] = 0;
  }
}

static int check_sizes(const bsx_delta_t* d) {
  if (!d) return fail(BSX_ERR_INVALID_ARG, "description is NULL");
  if (d->batch < 0 || d->tokens < 0) return fail(BSX_ERR_INVALID_ARG, "negative size");
  if (d->dtype < BSX_T_F32 || d->dtype > BSX_T_F16) return fail(BSX_ERR_INVALID_ARG, "unknown element type");
  if (d->k_heads < 1 || d->v_heads < 1 || d->v_heads % d->k_heads != 0)
    return fail(BSX_ERR_INVALID_ARG, "v_heads must be a positive multiple of k_heads");
  if (d->dk < 1 || d->dv < 1) return fail(BSX_ERR_INVALID_ARG, "dk and dv must be positive");
  if (d->dk > 128) return fail(BSX_ERR_UNSUPPORTED, "dk above 128");
  if (d->dv > 4096) return fail(BSX_ERR_UNSUPPORTED, "dv above 4096");
  if (d->tokens > INT32_MAX - kC || d->batch > INT32_MAX) return fail(BSX_ERR_UNSUPPORTED, "batch and tokens must fit int32");
  const int64_t blocks_per_head = chunks_of(d->tokens) > (d->dv + 15) / 16 ? chunks_of(d->tokens) : (d->dv + 15) / 16;
  if (d->batch > 0 && d->v_heads > INT32_MAX / blocks_per_head / d->batch)
    return fail(BSX_ERR_UNSUPPORTED, "batch * v_heads * chunks must fit int32");
  return BSX_OK;
}

static int clear_tails(const Args& a, int dtype, cudaStream_t st) {
  if (!a.lengths) return BSX_OK;
  const dim3 grid(8, (unsigned)(a.B < 65535 ? a.B : 65535));
  clear_tails_kernel<<<grid, 256, 0, st>>>(a, (int64_t)a.Hv * a.dv * (dtype == BSX_T_F32 ? 4 : 2));
  BSX_LAUNCH_CHECK("plastic clear_tails_kernel");
  return BSX_OK;
}

static int fill(const bsx_delta_t* d, Args& a) {
  int rc = check_sizes(d);
  if (rc != BSX_OK) return rc;
  if (d->batch > 0 && d->tokens > 0 && (!d->q || !d->k || !d->v || !d->g || !d->beta))
    return fail(BSX_ERR_INVALID_ARG, "NULL input");
  a = Args{};
  a.q = d->q; a.k = d->k; a.v = d->v; a.g = d->g; a.beta = d->beta;
  a.initial = d->initial; a.lengths = d->lengths;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = d->q_stride[i]; a.ks[i] = d->k_stride[i]; a.vs[i] = d->v_stride[i];
    a.gs[i] = d->g_stride[i]; a.bs[i] = d->beta_stride[i];
  }
  // the stride of a dimension of one entry says nothing and must not spoil the alignment rule
  auto single = [](int64_t* s, int64_t batch, int64_t tokens, int64_t heads) {
    if (batch == 1) s[0] = 0;
    if (tokens == 1) s[1] = 0;
    if (heads == 1) s[2] = 0;
  };
  single(a.qs, d->batch, d->tokens, d->k_heads);
  single(a.ks, d->batch, d->tokens, d->k_heads);
  single(a.vs, d->batch, d->tokens, d->v_heads);
  a.T = d->tokens; a.B = (int)d->batch; a.Hk = d->k_heads; a.Hv = d->v_heads; a.dk = d->dk; a.dv = d->dv;
  a.NC = (int)chunks_of(d->tokens);
  a.scale = d->scale;
  const int per = d->dtype == BSX_T_F32 ? 4 : 8;     // elements of a 16-byte stretch
  auto vec = [per](const void* p, const int64_t* s, int cols) {
    return aligned16(p) && s[0] % per == 0 && s[1] % per == 0 && s[2] % per == 0 && cols % per == 0;
  };
  a.vec_qk = vec(a.q, a.qs, a.dk) && vec(a.k, a.ks, a.dk);
  return BSX_OK;
}

static void place(Args& a, const bsx_delta_t* d, float* ws, bool backward) {
  const int64_t n = (int64_t)a.B * a.Hv * a.NC;
  a.kq = ws; ws += (int64_t)a.B * a.Hk * a.NC * (2 * kC * (width_of(a.dk) + 8) * (d->dtype == BSX_T_F32 ? 4 : 2) / 4);
  a.rec = ws; ws += n * kRecord;
  if (!backward) return;
  a.taken = reinterpret_cast<uint32_t*>(ws); ws += 4;
  const int64_t wide = width_of(a.dk) + 4;
  a.Bm = ws; ws += n * kTri;
  a.Sn = ws; ws += n * a.dv * wide;
  a.dS = ws; ws += n * a.dv * wide;
  a.U = ws; ws += n * a.dv * kPU;
  a.dY = ws; ws += n * a.dv * kPU;
  if (a.Hk != a.Hv) {
    a.dq32 = ws; ws += (int64_t)a.B * a.T * a.Hv * a.dk;
    a.dk32 = ws;
  }
}

}  // namespace plastic
}  // namespace bsx

using namespace bsx;
using namespace bsx::plastic;

extern "C" size_t bsx_delta_workspace_bytes(const bsx_delta_t* d) {
  return check_sizes(d) == BSX_OK ? workspace(d, false) : 0;
}
extern "C" size_t bsx_delta_backward_workspace_bytes(const bsx_delta_t* d) {
  return check_sizes(d) == BSX_OK ? workspace(d, true) : 0;
}

extern "C" int bsx_delta_forward(const bsx_delta_t* d, void* out, float* state, void* ws, size_t ws_bytes,
                                 bsx_stream_t stream) {
  BSX_TRACE("bsx_delta_forward");
  Args a;
  int rc = fill(d, a);
  if (rc != BSX_OK) return rc;
  if (a.B == 0) return BSX_OK;
  if (a.NC > 0 && !out) return fail(BSX_ERR_INVALID_ARG, "out is NULL");
  if (a.NC == 0 && !state) return BSX_OK;
  if (a.NC > 0 && (!ws || !aligned16(ws) || ws_bytes < workspace(d, false)))
    return fail(BSX_ERR_WORKSPACE, "workspace missing, misaligned or too small");
  if (sm_count() <= 0) return fail(BSX_ERR_CUDA, "no CUDA device");
  a.o = out;
  a.state = state;
  place(a, d, static_cast<float*>(ws), false);
  cudaStream_t st = as_stream(stream);
  if (a.NC > 0 && (rc = launch_prepare(a, d->dtype, false, st)) != BSX_OK) return rc;
  return launch_scan(a, d->dtype, false, st);
}

extern "C" int bsx_delta_recurrent(const bsx_delta_t* d, void* out, float* state, bsx_stream_t stream) {
  BSX_TRACE("bsx_delta_recurrent");
  Args a;
  int rc = fill(d, a);
  if (rc != BSX_OK) return rc;
  if (a.B == 0) return BSX_OK;
  if (a.T > 0 && !out) return fail(BSX_ERR_INVALID_ARG, "out is NULL");
  if (a.T == 0 && !state) return BSX_OK;
  if (sm_count() <= 0) return fail(BSX_ERR_CUDA, "no CUDA device");
  a.o = out;
  a.state = state;
  cudaStream_t st = as_stream(stream);
  if (a.T > 0 && (rc = clear_tails(a, d->dtype, st)) != BSX_OK) return rc;
  return launch_step(a, d->dtype, st);
}

extern "C" int bsx_delta_backward(const bsx_delta_t* d, const void* dout, const float* dstate, void* dq, void* dk,
                                  void* dv, float* dg, float* dbeta, float* dinitial, void* ws, size_t ws_bytes,
                                  bsx_stream_t stream) {
  BSX_TRACE("bsx_delta_backward");
  Args a;
  int rc = fill(d, a);
  if (rc != BSX_OK) return rc;
  if (a.B == 0) return BSX_OK;
  if (a.NC > 0 && (!dout || !dq || !dk || !dv || !dg || !dbeta)) return fail(BSX_ERR_INVALID_ARG, "NULL buffer");
  if (a.NC == 0 && !dinitial) return BSX_OK;
  if (a.NC > 0 && (!ws || !aligned16(ws) || ws_bytes < workspace(d, true)))
    return fail(BSX_ERR_WORKSPACE, "workspace missing, misaligned or too small");
  if (sm_count() <= 0) return fail(BSX_ERR_CUDA, "no CUDA device");
  const uintptr_t four = 4 * (d->dtype == BSX_T_F32 ? 4 : 2) - 1;
  a.four_do = a.dv % 4 == 0 && (reinterpret_cast<uintptr_t>(dout) & four) == 0;
  a.four_v = a.dv % 4 == 0 && (reinterpret_cast<uintptr_t>(a.v) & four) == 0 && a.vs[0] % 4 == 0 && a.vs[1] % 4 == 0 &&
             a.vs[2] % 4 == 0;
  a.dout = dout; a.dstate = dstate;
  a.dq = dq; a.dk_ = dk; a.dv_ = dv; a.dg = dg; a.dbeta = dbeta; a.dinitial = dinitial;
  place(a, d, static_cast<float*>(ws), true);
  cudaStream_t st = as_stream(stream);
  if (a.NC > 0) {
    if ((rc = launch_prepare(a, d->dtype, true, st)) != BSX_OK) return rc;
    if ((rc = launch_scan(a, d->dtype, true, st)) != BSX_OK) return rc;
  }
  if ((rc = launch_backward_scan(a, d->dtype, st)) != BSX_OK) return rc;
  return a.NC > 0 ? launch_backward_chunks(a, d->dtype, st) : BSX_OK;
}
