// Dense 8-bit product on the fifth-generation tensor cores: out = (x w^T) sx sw for more than a few rows.
//
// A block computes tiles of 128 rows x BN output channels.  One warp copies 128 x 128 and BN x 128 byte tiles of both
// operands into a ring of shared-memory stages (tensor-map copies with the 128-byte swizzle), one warp issues the tensor
// instructions (128 x BN x 32, 32-bit integer sums in tensor memory), and four warps scale and write the finished tile
// while the next one is summed in the other half of tensor memory.  Blocks take tiles in a fixed stride; for few tiles
// and a long inner dimension several blocks share a tile's inner dimension, write their integer sums to the workspace,
// and a second kernel adds them.
//
// Every wait is bounded.  A block whose wait runs out stops taking part, waits (again with a bound) for its copies in
// flight and leaves NaN in the rest of its tiles.
#include <cuda.h>

#include "bulk_copy.cuh"
#include "int8.cuh"

namespace bsx {
namespace int8 {

constexpr int kBM = 128, kBK = 128;
constexpr int kThreads = 192;          // copies, instructions, four warps of output
constexpr uint32_t kWaitLimit = 1u << 20;   // polls of 20 ns and more: far above any wait of a block that makes progress

constexpr int kNoSum = -2147483647 - 1;   // stands for a sum that was not computed (real ones stay below 127^2 * 131072)

template <int BN> struct Tiles {
  static constexpr int stage = kBM * kBK + BN * kBK;
  static constexpr int stages = BN == 256 ? 4 : (BN == 128 ? 6 : 8);
  static constexpr int columns = 2 * BN;                   // of tensor memory: a power of two from 32 to 512
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
__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void copy_tile(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
// Operand tile in shared memory: rows of 128 bytes, 128-byte swizzle, groups of eight rows 1024 bytes apart.
__device__ __forceinline__ uint64_t operand(uint32_t addr) {
  return (uint64_t)((addr & 0x3ffff) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
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
  int64_t tiles_m, tiles_n, total;   // total includes the splits
  int splits, steps;                 // steps of 128 over the inner dimension
  __device__ __forceinline__ void tile(int64_t i, int& m, int& n, int& k0, int& k1, int& split) const {
    split = (int)(i % splits);
    i /= splits;
    m = (int)(i % tiles_m);          // tiles that share weights follow each other
    n = (int)(i / tiles_m);
    k0 = (int)((int64_t)steps * split / splits);
    k1 = (int)((int64_t)steps * (split + 1) / splits);
  }
};

template <typename E, int BN, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
tiles_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, Product p, Work work,
             bool wide_out) {
  using L = Tiles<BN>;
  extern __shared__ unsigned char raw[];
  __shared__ __align__(8) uint64_t full[L::stages], empty[L::stages], done[2], taken[2];
  __shared__ uint32_t tmem_base;
  __shared__ int dead_flag;
  volatile int* dead = &dead_flag;
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    dead_flag = 0;
    for (int i = 0; i < L::stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&done[i], 1);
      mbar_init(&taken[i], 4);
    }
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)),
                 "n"(L::columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_base;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t n_issued = 0;   // stages filled so far
      bool ok = true;
      for (int64_t i = blockIdx.x; ok && i < work.total; i += gridDim.x) {
        int m, n, k0, k1, split;
        work.tile(i, m, n, k0, k1, split);
        for (int k = k0; k < k1; ++k) {
          const int s = n_issued % L::stages;
          if (n_issued >= L::stages && !wait(&empty[s], ((n_issued / L::stages) - 1) & 1, dead)) { ok = false; break; }
          unsigned char* at = ring + s * L::stage;
          mbar_expect_tx(&full[s], L::stage);
          copy_tile(at, &map_x, k * kBK, m * kBM, &full[s]);
          copy_tile(at + kBM * kBK, &map_w, k * kBK, n * BN, &full[s]);
          ++n_issued;
        }
      }
      if (!ok) {   // copies in flight land before the block may end
        const uint32_t open = n_issued < L::stages ? n_issued : L::stages;
        for (uint32_t j = n_issued - open; j < n_issued; ++j)
          for (uint32_t w = 0; w < kWaitLimit && !mbar_try_wait(&full[j % L::stages], (j / L::stages) & 1); ++w) {}
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // 32-bit integer sums, signed 8-bit operands, both with the inner dimension contiguous
      const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(kBM >> 4) << 24);
      uint32_t used = 0, t = 0;
      bool ok = true;
      for (int64_t i = blockIdx.x; ok && i < work.total; i += gridDim.x, ++t) {
        int m, n, k0, k1, split;
        work.tile(i, m, n, k0, k1, split);
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
            mma_i8(tmem + half * BN, operand(at + j * 32), operand(at + kBM * kBK + j * 32), idesc, k > k0 || j > 0);
          commit(&empty[s]);     // the stage is free when these have read it
        }
        if (ok) commit(&done[half]);
      }
    }
  } else {
    const int quarter = warp & 3;      // the 32 tensor-memory lanes a warp can read
    uint32_t t = 0;
    bool alive = true;
    for (int64_t i = blockIdx.x; i < work.total; i += gridDim.x, ++t) {
      int m, n, k0, k1, split;
      work.tile(i, m, n, k0, k1, split);
      const int half = t & 1;
      if (alive) {
        alive = wait(&done[half], (t >> 1) & 1, dead);
        alive = __all_sync(0xffffffffu, alive);
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int64_t row = (int64_t)m * kBM + quarter * 32 + lane;
      float sx = (!SPLIT && row < p.M) ? __ldg(p.sx + row) : 0.f;
      if (!alive) sx = __int_as_float(0x7fffffff);
#pragma unroll 1
      for (int c = 0; c < BN; c += 32) {
        const int64_t col = (int64_t)n * BN + c;
        if (col >= p.N) break;
        int r[32];
        __syncwarp();
        if (alive) {
          load32(tmem + ((uint32_t)(quarter * 32) << 16) + half * BN + c, r);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) r[j] = kNoSum;
        }
        if (row < p.M) {
          if (SPLIT) {
            int32_t* o = p.partial + ((int64_t)split * p.M + row) * p.N + col;
            if (wide_out) {
#pragma unroll
              for (int j = 0; j < 32; j += 4)
                if (col + j < p.N) *reinterpret_cast<int4*>(o + j) = make_int4(r[j], r[j + 1], r[j + 2], r[j + 3]);
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (col + j < p.N) o[j] = r[j];
            }
          } else {
            E* o = static_cast<E*>(p.out) + row * p.N + col;
            constexpr int V = 16 / sizeof(E);
            if (wide_out) {
#pragma unroll
              for (int j = 0; j < 32; j += V) {
                if (col + j < p.N) {
                  union { E e[V]; int4 q; } w;
#pragma unroll
                  for (int x = 0; x < V; ++x) w.e[x] = scaled<E>(r[j + x], sx, __ldg(p.sw + col + j + x));
                  *reinterpret_cast<int4*>(o + j) = w.q;
                }
              }
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (col + j < p.N) o[j] = scaled<E>(r[j], sx, __ldg(p.sw + col + j));
            }
          }
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) arrive(&taken[half]);
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(L::columns) : "memory");
  }
}

// Adds the partial sums of a split inner dimension and scales.
template <typename E>
__global__ void __launch_bounds__(256) add_splits_kernel(Product p, int splits) {
  const int64_t total = p.M * p.N;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    int s = 0;
    bool whole = true;
    for (int k = 0; k < splits; ++k) {
      const int x = __ldg(p.partial + k * total + i);
      whole &= x != kNoSum;
      s += x;
    }
    const int64_t m = i / p.N, n = i - m * p.N;
    static_cast<E*>(p.out)[i] = scaled<E>(s, whole ? __ldg(p.sx + m) : __int_as_float(0x7fffffff), __ldg(p.sw + n));
  }
}

static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Width of the tiles: the widest that still gives every SM a tile; narrow ones read the rows more often.
static int width(int64_t M, int64_t N, int sms) {
  const int64_t tm = ceil_div(M, kBM);
  if (tm * ceil_div(N, 256) >= sms) return 256;
  if (tm * ceil_div(N, 128) >= sms) return 128;
  return 64;
}

int tiles_splits(int64_t M, int64_t N, int64_t Kp, int sms) {
  if (sms <= 0) sms = 148;
  const int64_t tiles = ceil_div(M, kBM) * ceil_div(N, width(M, N, sms)), steps = ceil_div(Kp, kBK);
  // A split has at least 16 steps (2048 of the inner dimension), so that its sums are worth their round trip.
  int s = 1;
  while (s < 8 && tiles * s * 2 <= sms && steps / (s * 2) >= 16) s *= 2;
  return s;
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

template <typename E, int BN, bool SPLIT>
static int launch_width(const Product& p, int splits, int sms, cudaStream_t st) {
  CUtensorMap mx, mw;
  int rc;
  if ((rc = encode(&mx, p.x, p.M, p.Kp, kBM)) != BSX_OK || (rc = encode(&mw, p.w, p.N, p.Kp, BN)) != BSX_OK) return rc;
  Work w;
  w.tiles_m = ceil_div(p.M, kBM);
  w.tiles_n = ceil_div(p.N, BN);
  w.splits = splits;
  w.steps = (int)ceil_div(p.Kp, kBK);
  w.total = w.tiles_m * w.tiles_n * splits;
  const size_t bytes = Tiles<BN>::bytes;
  BSX_CUDA(cudaFuncSetAttribute(tiles_kernel<E, BN, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  const unsigned grid = (unsigned)(w.total < sms ? w.total : sms);
  constexpr int V = SPLIT ? 4 : 16 / (int)sizeof(E);
  const bool wide = p.N % V == 0 && aligned16(SPLIT ? static_cast<const void*>(p.partial) : p.out);
  tiles_kernel<E, BN, SPLIT><<<grid, kThreads, bytes, st>>>(mx, mw, p, w, wide);
  BSX_LAUNCH_CHECK("int8 tiles_kernel");
  if (SPLIT) {
    const int64_t want = ceil_div(p.M * p.N, 256), most = 8ll * sms;
    add_splits_kernel<E><<<(unsigned)(want < most ? want : most), 256, 0, st>>>(p, splits);
    BSX_LAUNCH_CHECK("int8 add_splits_kernel");
  }
  return BSX_OK;
}

template <typename E>
static int launch_typed(const Product& p, int splits, cudaStream_t st) {
  const int sms = sm_count();
  if (sms <= 0) return fail(BSX_ERR_CUDA, "no CUDA device");
  const int bn = width(p.M, p.N, sms);
  if (splits > 1) {   // only where there are few tiles: the narrow ones
    return bn == 64 ? launch_width<E, 64, true>(p, splits, sms, st) : launch_width<E, 128, true>(p, splits, sms, st);
  }
  if (bn == 256) return launch_width<E, 256, false>(p, 1, sms, st);
  if (bn == 128) return launch_width<E, 128, false>(p, 1, sms, st);
  return launch_width<E, 64, false>(p, 1, sms, st);
}

int launch_tiles(const Product& p, int splits, int dtype, cudaStream_t st) {
  if (dtype == BSX_T_F32) return launch_typed<float>(p, splits, st);
  if (dtype == BSX_T_BF16) return launch_typed<__nv_bfloat16>(p, splits, st);
  return launch_typed<__half>(p, splits, st);
}

}  // namespace int8
}  // namespace bsx
