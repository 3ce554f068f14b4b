// Dense GEMM with epilogue for few rows of x:  y[M, N] = T( act(x W^T + bias) + residual ),  M up to a few hundred.
//
// With few rows the product is bound by the one read of W, and the dense kernel (gemm_tcgen05.cu) has too few
// tiles for it: 128 rows of x by up to 256 of W leave most SMs idle at N = 4096.  Here W is the 128-row operand
// of tcgen05.mma and the rows of x are its columns (16..256, as many as there are), so a tile is 128 outputs wide
// whatever M is, and K is split over a cluster of 1..8 CTAs, which puts every SM to work: the partial sums [rows of
// x][128] meet in shared memory and each CTA finishes an equal share of them, reading its peers' over DSMEM in rank
// order -- no workspace, no atomics, the same bits every time.
//
// CTA: warp 0 TMA producer (stages of 128 of k: two 64-wide boxes of W and of x, 128-byte swizzle), warp 1 TMEM owner
// and tcgen05.mma issuer, warps 2-9 move the accumulator (TMEM lane = output, column = row of x) to shared memory or,
// unsplit, straight through the epilogue; lanes are consecutive outputs, so stores and residual loads are coalesced,
// and the residual is on its way before the sums are there.  Up to two CTAs share an SM.  Every wait is bounded (npb_set_wait_limit_ns); on give-up the kernel records it, lets
// its copies land, frees its TMEM and returns.
#include <type_traits>

#include "activation.cuh"
#include "common.cuh"
#include "tcgen05.cuh"

namespace npb {

// gemm_tcgen05.cu
int make_tensor_map_2d(CUtensorMap* map, CUtensorMapDataType type, int elem_bytes, const void* base, int64_t rows,
                       int64_t cols, int box_rows, int box_cols, CUtensorMapSwizzle swizzle);

__device__ int g_skinny_status = 0;  // 0 ok; 1..3: the role whose wait gave up

namespace {

using namespace sm100;

constexpr int BN = 128;             // outputs per tile
constexpr int BK = 128;             // of k per stage, as two halves of 64 (one swizzle row each)
constexpr int kThreads = 320;
constexpr int kWHalf = BN * 64 * 2; // 16 KiB
constexpr int kMaxStages = 8;
constexpr int kHead = 1024;         // barriers

struct SkinnyParams {
  const float* bias;
  const void* residual;
  void* y;
  int M, N, act;
  int rows;       // of x per tile: multiple of 16, at most 256
  int stages, k_blocks, split;
  uint64_t wait_ns;
};

template <typename T>
__device__ __forceinline__ float residual_at(const SkinnyParams& p, int m, int n) {
  return to_f32(static_cast<const T*>(p.residual)[(int64_t)m * p.N + n]);
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2)
gemm_skinny_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                   const SkinnyParams p) {
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem);  // [stages]
  uint64_t* empty = full + kMaxStages;
  uint64_t* done = empty + kMaxStages;                 // the accumulator is complete
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint8_t* ring = smem + kHead;
  const int x_half = p.rows * 128, stage_bytes = 2 * kWHalf + 2 * x_half;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = p.split > 1 ? (int)cluster_ctarank() : 0;
  const int n0 = blockIdx.x / p.split * BN, m0 = blockIdx.y * p.rows;
  const int kb0 = (int)((int64_t)p.k_blocks * rank / p.split), kb1 = (int)((int64_t)p.k_blocks * (rank + 1) / p.split);
  const uint32_t tmem_cols = p.rows <= 32 ? 32 : p.rows <= 64 ? 64 : p.rows <= 128 ? 128 : 256;

  if (tid == 0) {
    *abort_flag = 0;
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    fence_barrier_init();
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_x);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 1;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_bounded(&empty[s], ph, abort_flag, p.wait_ns)) {
          atomicExch(&g_skinny_status, 1);
          break;
        }
        uint8_t* st = ring + (size_t)s * stage_bytes;
        mbar_arrive_expect_tx(&full[s], (uint32_t)stage_bytes);
        tma_load_2d(st, &map_w, &full[s], kb * BK, n0);
        tma_load_2d(st + kWHalf, &map_w, &full[s], kb * BK + 64, n0);
        tma_load_2d(st + 2 * kWHalf, &map_x, &full[s], kb * BK, m0);
        tma_load_2d(st + 2 * kWHalf + x_half, &map_x, &full[s], kb * BK + 64, m0);
        if (++s == p.stages) { s = 0; ph ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = umma_idesc_f16(std::is_same<T, __nv_bfloat16>::value ? 1 : 0, BN, p.rows);
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_bounded(&full[s], ph, abort_flag, p.wait_ns)) {
          atomicExch(&g_skinny_status, 2);
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t st = smem_u32(ring + (size_t)s * stage_bytes);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint64_t a = umma_desc_sw128(st + h * kWHalf), b = umma_desc_sw128(st + 2 * kWHalf + h * x_half);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16(tmem, a + 2 * k, b + 2 * k, idesc, (kb > kb0 || h > 0 || k > 0) ? 1u : 0u);
        }
        umma_commit(&empty[s]);
        if (++s == p.stages) { s = 0; ph ^= 1; }
      }
      if (ok) umma_commit(done);
    }
  } else {
    // 16 rows of x at a time: two warps share the 32 outputs of a TMEM quadrant
    const int quad = warp & 3, n = quad * 32 + lane, c0 = warp < 6 ? 0 : 16;  // TMEM lane = output of the tile
    const int rows = min(p.rows, p.M - m0);
    const bool in = n0 + n < p.N, adds = p.split == 1 && p.residual != nullptr && in;
    const float bias = p.split == 1 && p.bias && in ? __ldg(p.bias + n0 + n) : 0.f;
    float r[16];
    auto load_residual = [&](int c) {
#pragma unroll
      for (int i = 0; i < 16; ++i) r[i] = adds && c + i < rows ? residual_at<T>(p, m0 + c + i, n0 + n) : 0.f;
    };
    load_residual(c0);
    const bool got = mbar_wait_bounded(done, 0, abort_flag, p.wait_ns, 64u);
    if (__all_sync(0xffffffffu, got)) {
      tc_fence_after();
      float* part = reinterpret_cast<float*>(ring);   // every stage has been read
      for (int c = c0; c < rows; c += 32) {
        uint32_t v[16];
        tmem_ld_32x32_x16(tmem + ((uint32_t)(quad * 32) << 16) + c, v);
        tmem_ld_wait();
        if (p.split > 1) {
#pragma unroll
          for (int i = 0; i < 16; ++i) part[(c + i) * BN + n] = __uint_as_float(v[i]);
        } else {
          T* y = static_cast<T*>(p.y) + (int64_t)(m0 + c) * p.N + n0 + n;
          float o[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = activate(__uint_as_float(v[i]) + bias, p.act) + r[i];
          load_residual(c + 32);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (in && c + i < rows) y[(int64_t)i * p.N] = from_f32<T>(o[i]);
        }
      }
    } else {
      atomicExch(&g_skinny_status, 3);
    }
    tc_fence_before();
  }
  __syncwarp();
  if (p.split > 1) {
    // each CTA of the cluster finishes an equal share of the tile, four outputs of a row of x at a time, adding the
    // partial sums in rank order
    const int rows = min(p.rows, p.M - m0), total = rows * (BN / 4);
    const int last = (int)((int64_t)total * (rank + 1) / p.split);
    int i = (int)((int64_t)total * rank / p.split) + tid;
    struct alignas(8) Four { T e[4]; };
    const bool wide = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 7) == 0 &&
                      (reinterpret_cast<uintptr_t>(p.residual) & 7) == 0;
    float r[4], bias[4];
    auto load_rest = [&](int u) {
      const int n = n0 + u % (BN / 4) * 4, m = m0 + u / (BN / 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        bias[k] = p.bias && u < last && n + k < p.N ? __ldg(p.bias + n + k) : 0.f;
        r[k] = 0.f;
      }
      if (p.residual && u < last) {
        if (wide && n < p.N) {
          const Four f = *reinterpret_cast<const Four*>(static_cast<const T*>(p.residual) + (int64_t)m * p.N + n);
#pragma unroll
          for (int k = 0; k < 4; ++k) r[k] = to_f32(f.e[k]);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (n + k < p.N) r[k] = residual_at<T>(p, m, n + k);
        }
      }
    };
    load_rest(i);
    cluster_sync_all();
    const uint32_t part = smem_u32(ring);
    for (; i < last; i += kThreads) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int c = 0; c < p.split; ++c) {
        float4 q;
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(q.x), "=f"(q.y), "=f"(q.z), "=f"(q.w)
                     : "r"(map_to_cta(part + i * 16, c))
                     : "memory");
        v.x += q.x; v.y += q.y; v.z += q.z; v.w += q.w;
      }
      const int n = n0 + i % (BN / 4) * 4, m = m0 + i / (BN / 4);
      T* y = static_cast<T*>(p.y) + (int64_t)m * p.N + n;
      Four f;
      const float sum[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) f.e[k] = from_f32<T>(activate(sum[k] + bias[k], p.act) + r[k]);
      if (wide && n < p.N) {
        *reinterpret_cast<Four*>(y) = f;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (n + k < p.N) y[k] = f.e[k];
      }
      load_rest(i + kThreads);
    }
    __syncwarp();
    cluster_sync_all();  // nobody leaves while its sums are read
  }
  if (*abort_flag) {
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
}

}  // namespace

// Tiles of at most 256 rows of x; W is read once per tile of rows.
int gemm_skinny(const void* x, const void* w, const float* bias, int act, const void* residual, void* y, int64_t M,
                int64_t N, int64_t K, int dtype, cudaStream_t st) {
  SkinnyParams p{};
  p.bias = bias;
  p.residual = residual;
  p.y = y;
  p.M = (int)M; p.N = (int)N; p.act = act;
  const int row_tiles = (int)((M + 255) / 256);
  p.rows = (int)(((M + row_tiles - 1) / row_tiles + 15) / 16 * 16);
  p.k_blocks = (int)((K + BK - 1) / BK);
  p.wait_ns = wait_limit_ns();
  const int stage_bytes = 2 * kWHalf + 2 * p.rows * 128;
  // two CTAs on an SM where three stages of each fit
  const int half = max_dynamic_smem() / 2 - 1024 - 2048, whole = max_dynamic_smem() - 2048;
  const int per_sm = (half - kHead) / stage_bytes >= 3 ? 2 : 1;
  p.stages = ((per_sm == 2 ? half : whole) - kHead) / stage_bytes;
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  const int64_t tiles = (N + BN - 1) / BN, slots = (int64_t)sm_count() * per_sm;
  p.split = 1;
  while (p.split < 8 && tiles * row_tiles * p.split * 2 <= slots && p.k_blocks >= p.split * 4) p.split *= 2;
  const int parts = p.rows * BN * 4;
  int ring = p.stages * stage_bytes;
  if (ring < parts) ring = parts;
  const int smem = 1024 + kHead + ring;
  const bool bf16 = dtype == NPB_BF16;
  const void* kern = bf16 ? reinterpret_cast<const void*>(gemm_skinny_kernel<__nv_bfloat16>)
                          : reinterpret_cast<const void*>(gemm_skinny_kernel<__half>);
  int resident = 0;
  if (int rc = blocks_per_sm(kern, kThreads, smem, &resident)) return rc;
  if (resident < 1) return NPB_ERR_TOO_LARGE;
  CUtensorMap map_w, map_x;
  const CUtensorMapDataType type = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  if (int rc = make_tensor_map_2d(&map_w, type, 2, w, N, K, BN, 64, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  if (int rc = make_tensor_map_2d(&map_x, type, 2, x, M, K, p.rows, 64, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(tiles * p.split), (unsigned)row_tiles);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = p.split;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (bf16) NPB_CUDA_TRY(cudaLaunchKernelEx(&cfg, gemm_skinny_kernel<__nv_bfloat16>, map_w, map_x, p));
  else NPB_CUDA_TRY(cudaLaunchKernelEx(&cfg, gemm_skinny_kernel<__half>, map_w, map_x, p));
  NPB_LAUNCH_CHECK();
  return NPB_OK;
}

// Reads and clears the give-up record (npb_gemm_device_status collects it).
int gemm_skinny_device_status(int* host_out) {
  NPB_CUDA_TRY(cudaMemcpyFromSymbol(host_out, g_skinny_status, sizeof(int)));
  if (*host_out != 0) {
    const int zero = 0;
    NPB_CUDA_TRY(cudaMemcpyToSymbol(g_skinny_status, &zero, sizeof(int)));
  }
  return NPB_OK;
}

}  // namespace npb
