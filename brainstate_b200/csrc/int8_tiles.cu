// Dense 8-bit product on the fifth-generation tensor cores, for more than a few rows.
//
// Output channels are the rows of the tensor instructions and activations their columns, so that the 32 lanes of an
// output warp hold neighbouring channels of one activation row and store them together.  A pair of blocks on
// neighbouring SMs computes a tile of 256 channels x BT rows: each holds its 128 channels and half of the activation
// rows, one instruction (256 x BT x 32, 32-bit integer sums in tensor memory) reads both blocks' shared memory, and each
// operand byte is copied once per pair — the traffic from L2, not the instructions, limits this product
// on single blocks.  In each block one warp copies 128-byte wide tiles into a ring of stages (tensor-map
// copies, 128-byte swizzle) that reports to the first block's barriers, the first block's second warp issues the
// instructions, and four warps scale and store the finished tile while the next one is summed in the other half of
// tensor memory.  Pairs take tiles in a fixed stride; for few tiles and a long inner dimension several pairs share a
// tile's inner dimension, write their integer sums to the workspace, and a second kernel adds them.
//
// 4096 x 4096 by 4096 x 8192: 122 us, 2.25e15 operations a second (69 % of twice the measured bf16 rate), the tensor unit 56 %
// busy: 32 KB a block and step come from L2 at 43 bytes a clock and SM, 12 TB/s over the card, in 775 clocks where the
// instructions take 512.  Blocks of their own (128 x 256) read half as much again and took 125 us.
//
// Every wait is bounded.  A block whose wait runs out waits (again with a bound) for its copies in flight, takes no more
// part and leaves NaN in its tiles.
#include <cuda.h>

#include "bulk_copy.cuh"
#include "int8.cuh"

namespace bsx {
namespace int8 {

constexpr int kBM = 128, kBK = 128;    // channels of a block, bytes of a step
constexpr int kThreads = 192;          // copies, instructions, four warps of output
constexpr uint32_t kWaitLimit = 1u << 20;   // polls of 20 ns and more: far above any wait of a block that makes progress
constexpr int kNoSum = -2147483647 - 1;   // stands for a sum that was not computed (real ones stay below 127^2 * 131072)

template <int BT> struct Tiles {
  static constexpr int rows = BT / 2;                      // activation rows of a block
  static constexpr int stage = kBM * kBK + rows * kBK;
  static constexpr int stages = BT == 256 ? 6 : (BT == 128 ? 8 : (BT == 64 ? 9 : 10));
  static constexpr int columns = 2 * BT;                   // of tensor memory: a power of two from 32 to 512
  static constexpr size_t bytes = (size_t)stages * stage + 1024;
};

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* dead) {
  for (uint32_t i = 0; i < kWaitLimit; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 1023) == 1023 && *dead) return false;
  }
  *dead = 1;
  return false;
}
// Address of a shared variable in the pair's first block.
__device__ __forceinline__ uint32_t in_first(const void* p) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
  return r;
}
__device__ __forceinline__ void arrive_first(uint64_t* bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_first(bar)) : "memory");
}
__device__ __forceinline__ void pair_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Copies a tile into this block; its bytes count on the first block's barrier.
__device__ __forceinline__ void copy_tile(void* dst, const CUtensorMap* map, int x, int y, uint32_t first_bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], "
      "[%4];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(first_bar)
      : "memory");
}
// Operand tile in shared memory: rows of 128 bytes, 128-byte swizzle, groups of eight rows 1024 bytes apart.
__device__ __forceinline__ uint64_t operand(uint32_t addr) {
  return (uint64_t)((addr & 0x3ffff) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Signals the barrier at the same place in both blocks once the instructions issued so far have finished.
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void load32(uint32_t addr, int* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}

struct Work {
  int64_t tiles_c, tiles_t, total;   // channel tiles, row tiles; total includes the splits
  int splits, steps;                 // steps of 128 over the inner dimension
  __device__ __forceinline__ void tile(int64_t i, int& c, int& r, int& k0, int& k1, int& split) const {
    split = (int)(i % splits);
    i /= splits;
    r = (int)(i % tiles_t);          // tiles that share weights follow each other
    c = (int)(i / tiles_t);
    k0 = (int)((int64_t)steps * split / splits);
    k1 = (int)((int64_t)steps * (split + 1) / splits);
  }
};

template <typename E, int BT, bool SPLIT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
tiles_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, Product p, Work work) {
  using L = Tiles<BT>;
  extern __shared__ unsigned char raw[];
  // full (copies of both blocks) and taken (their output warps) live in the first block, empty and done in each
  __shared__ __align__(8) uint64_t full[L::stages], empty[L::stages], done[2], taken[2];
  __shared__ uint32_t tmem_base;
  __shared__ int dead_flag;
  volatile int* dead = &dead_flag;
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int side = blockIdx.x & 1;
  const int64_t pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    dead_flag = 0;
    for (int i = 0; i < L::stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&done[i], 1);
      mbar_init(&taken[i], 8);
    }
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)),
                 "n"(L::columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  pair_sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_base;
  wait_for_rows();

  if (warp == 0) {
    if (lane == 0) {
      uint32_t n = 0;   // stages filled so far
      bool ok = true;
      for (int64_t i = pair; ok && i < work.total; i += pairs) {
        int c, r, k0, k1, split;
        work.tile(i, c, r, k0, k1, split);
        for (int k = k0; k < k1; ++k) {
          const int s = n % L::stages;
          if (n >= L::stages && !wait(&empty[s], ((n / L::stages) - 1) & 1, dead)) { ok = false; break; }
          unsigned char* at = ring + s * L::stage;
          const uint32_t bar = in_first(&full[s]);
          if (side == 0) mbar_expect_tx(&full[s], 2 * L::stage);
          copy_tile(at, &map_w, k * kBK, c * 2 * kBM + side * kBM, bar);
          copy_tile(at + kBM * kBK, &map_x, k * kBK, r * BT + side * L::rows, bar);
          ++n;
        }
      }
      if (!ok) {   // copies in flight land before the pair may end: both blocks' count on the first's barriers
        const uint32_t open = n < L::stages ? n : L::stages;
        for (uint32_t j = n - open; side == 0 && j < n; ++j)
          for (uint32_t w = 0; w < kWaitLimit && !mbar_try_wait(&full[j % L::stages], (j / L::stages) & 1); ++w) {}
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && side == 0) {
      // 32-bit integer sums, signed 8-bit operands, both with the inner dimension contiguous
      const uint32_t idesc =
          (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BT >> 3) << 17) | ((uint32_t)(2 * kBM >> 4) << 24);
      uint32_t used = 0, t = 0;
      bool ok = true;
      for (int64_t i = pair; ok && i < work.total; i += pairs, ++t) {
        int c, r, k0, k1, split;
        work.tile(i, c, r, k0, k1, split);
        const int half = t & 1;
        if (t >= 2 && !wait(&taken[half], ((t >> 1) - 1) & 1, dead)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (int k = k0; k < k1; ++k, ++used) {
          const int s = used % L::stages;
          if (!wait(&full[s], (used / L::stages) & 1, dead)) { ok = false; break; }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t at = smem_u32(ring + s * L::stage);
#pragma unroll
          for (int j = 0; j < kBK / 32; ++j)
            mma_i8(tmem + half * BT, operand(at + j * 32), operand(at + kBM * kBK + j * 32), idesc, k > k0 || j > 0);
          commit(&empty[s]);     // the stage is free in both blocks when these have read it
        }
        if (ok) commit(&done[half]);
      }
    }
  } else {
    const int quarter = warp & 3;      // the 32 tensor-memory lanes a warp can read
    uint32_t t = 0;
    bool alive = true;
    for (int64_t i = pair; i < work.total; i += pairs, ++t) {
      int c, r0, k0, k1, split;
      work.tile(i, c, r0, k0, k1, split);
      const int half = t & 1;
      if (alive) {
        alive = wait(&done[half], (t >> 1) & 1, dead);
        alive = __all_sync(0xffffffffu, alive);
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int64_t ch = (int64_t)c * 2 * kBM + side * kBM + quarter * 32 + lane, row0 = (int64_t)r0 * BT;
      const bool mine = ch < p.N;
      const float sw = alive ? (!SPLIT && mine ? __ldg(p.sw + ch) : 0.f) : __int_as_float(0x7fffffff);
#pragma unroll 1
      for (int b = 0; b < BT; b += 32) {
        if (row0 + b >= p.M) break;
        int r[32];
        __syncwarp();
        if (alive) {
          load32(tmem + ((uint32_t)(quarter * 32) << 16) + half * BT + b, r);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) r[j] = kNoSum;
        }
        // the rows' scales: one load a lane, handed round (as loads of their own they would wait for the stores)
        float sxs[32];
        if (!SPLIT) {
          const float sx = row0 + b + lane < p.M ? p.sx[row0 + b + lane] : 0.f;
#pragma unroll
          for (int j = 0; j < 32; ++j) sxs[j] = __shfl_sync(0xffffffffu, sx, j);
        }
        if (mine) {
          const int m = (int)min((int64_t)32, p.M - row0 - b);
          if (SPLIT) {
            int32_t* o = p.partial + ((int64_t)split * p.M + row0 + b) * p.N + ch;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j < m) o[j * p.N] = r[j];
          } else {
            E* o = static_cast<E*>(p.out) + (row0 + b) * p.N + ch;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j < m) o[j * p.N] = scaled<E>(r[j], sxs[j], sw);
          }
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) arrive_first(&taken[half]);
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  pair_sync();       // neither block leaves while the other's copies, instructions or signals may reach it
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(L::columns) : "memory");
  }
}

// Adds the partial sums of a split inner dimension and scales: four channels a thread, a block 1024 of a row.
template <typename E, bool VEC>
__global__ void __launch_bounds__(256) add_splits_kernel(Product p, int splits) {
  const int64_t n = (int64_t)blockIdx.x * 1024 + threadIdx.x * 4;
  if (n >= p.N) return;
  float sw[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) sw[j] = n + j < p.N ? __ldg(p.sw + n + j) : 0.f;
  for (int64_t m = blockIdx.y; m < p.M; m += gridDim.y) {
    const int32_t* x = p.partial + m * p.N + n;
    int s[4] = {0, 0, 0, 0};
    bool whole = true;
    for (int k = 0; k < splits; ++k, x += p.M * p.N) {
      int v[4];
      if (VEC) {
        const int4 q = __ldg(reinterpret_cast<const int4*>(x));
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = n + j < p.N ? __ldg(x + j) : 0;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        whole &= v[j] != kNoSum;
        s[j] += v[j];
      }
    }
    const float sx = whole ? __ldg(p.sx + m) : __int_as_float(0x7fffffff);
    E* o = static_cast<E*>(p.out) + m * p.N + n;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < p.N) o[j] = scaled<E>(s[j], sx, sw[j]);
  }
}

static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How a product is divided: rows of a tile and splits of the inner dimension, the cheapest by an estimate in clocks.
// Measured on a B200: a step of 128 takes 776 clocks with 256 rows and 653 with 128 (about 284 and 0.015 a byte that a
// block copies, whose rate from L2 is the limit; the instructions alone would take 512 and 256); a tile's output about
// 1000 and 20 a row; adding splits costs a launch and its latency (7000) and its bytes (3000 a clock over the card).
Plan plan_tiles(int64_t M, int64_t N, int64_t Kp, int sms) {
  const int64_t pairs = sms > 1 ? sms / 2 : 74, steps = ceil_div(Kp, kBK);
  Plan best = {32, 1};
  double least = 0;
  for (int bt = 32; bt <= 256; bt *= 2) {
    const double step = 284 + 0.015 * (kBM + bt / 2) * kBK, out = 1000 + 20.0 * bt;
    for (int s = 1; s <= 8 && s <= steps; s *= 2) {
      const int64_t waves = ceil_div(ceil_div(N, 2 * kBM) * ceil_div(M, bt) * s, pairs);
      double cost = waves * ceil_div(steps, s) * step + out;
      if (s > 1) cost += 7000 + (double)M * N * s * 8 / 3000;
      if (least == 0 || cost < least) {
        least = cost;
        best = {bt, s};
      }
    }
  }
  return best;
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encoder() {
  static EncodeTiled fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult got;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &got) != cudaSuccess ||
        got != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiled>(f);
  }();
  return fn;
}

static int encode(CUtensorMap* map, const int8_t* base, int64_t rows, int64_t Kp, int box_rows) {
  EncodeTiled fn = encoder();
  if (!fn) return fail(BSX_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[2] = {(cuuint64_t)Kp, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)Kp};
  const cuuint32_t box[2] = {kBK, (cuuint32_t)box_rows}, step[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(base), dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(BSX_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", (int)r);
  return BSX_OK;
}

template <typename E, int BT, bool SPLIT>
static int launch_height(const Product& p, int splits, int sms, cudaStream_t st) {
  CUtensorMap mw, mx;
  int rc;
  if ((rc = encode(&mw, p.w, p.N, p.Kp, kBM)) != BSX_OK || (rc = encode(&mx, p.x, p.M, p.Kp, Tiles<BT>::rows)) != BSX_OK)
    return rc;
  Work w;
  w.tiles_c = ceil_div(p.N, 2 * kBM);
  w.tiles_t = ceil_div(p.M, BT);
  w.splits = splits;
  w.steps = (int)ceil_div(p.Kp, kBK);
  w.total = w.tiles_c * w.tiles_t * splits;
  static std::atomic<uint64_t> seen;
  if ((rc = allow_smem(tiles_kernel<E, BT, SPLIT>, Tiles<BT>::bytes, seen)) != BSX_OK) return rc;
  const int64_t pairs = w.total < sms / 2 ? w.total : sms / 2;
  const cudaError_t e = launch_behind(p.after_rows, tiles_kernel<E, BT, SPLIT>, (unsigned)(2 * pairs), kThreads,
                                      Tiles<BT>::bytes, st, mw, mx, p, w);
  if (e != cudaSuccess) return cuda_fail(e, "int8 tiles_kernel");
  if (SPLIT) {
    const dim3 grid((unsigned)ceil_div(p.N, 1024), (unsigned)(p.M < 65535 ? p.M : 65535));
    if (p.N % 4 == 0 && aligned16(p.partial)) add_splits_kernel<E, true><<<grid, 256, 0, st>>>(p, splits);
    else add_splits_kernel<E, false><<<grid, 256, 0, st>>>(p, splits);
    BSX_LAUNCH_CHECK("int8 add_splits_kernel");
  }
  return BSX_OK;
}

template <typename E>
static int launch_typed(const Product& p, Plan plan, cudaStream_t st) {
  const int sms = sm_count();
  if (sms <= 0) return fail(BSX_ERR_CUDA, "no CUDA device");
#define BSX_TILES(BT) \
  return plan.splits > 1 ? launch_height<E, BT, true>(p, plan.splits, sms, st) : launch_height<E, BT, false>(p, 1, sms, st)
  if (plan.rows == 256) BSX_TILES(256);
  if (plan.rows == 128) BSX_TILES(128);
  if (plan.rows == 64) BSX_TILES(64);
  BSX_TILES(32);
#undef BSX_TILES
}

int launch_tiles(const Product& p, Plan plan, int dtype, cudaStream_t st) {
  if (dtype == BSX_T_F32) return launch_typed<float>(p, plan, st);
  if (dtype == BSX_T_BF16) return launch_typed<__nv_bfloat16>(p, plan, st);
  return launch_typed<__half>(p, plan, st);
}

}  // namespace int8
}  // namespace bsx
