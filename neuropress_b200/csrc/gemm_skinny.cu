// Dense GEMM with epilogue for products of few tiles:  y[M, N] = T( act(x W^T + bias) + residual ).  That is few rows, up to
// a few hundred, or any number of rows with so few outputs that the tiles fill at most half of the SMs
// (gemm_skinny_takes).
//
// With few rows the product is bound by the one read of W, and the dense kernel (gemm_tcgen05.cu) has too few
// tiles for it: 128 rows of x by up to 256 of W leave most SMs idle at N = 4096.  Here W is the 128-row operand
// of tcgen05.mma and the rows of x are its columns (16..256, as many as there are), so a tile is 128 outputs wide
// whatever M is, and K is split over a cluster of 1..8 CTAs, which puts every SM to work.  Each CTA finishes a share of
// the tile's outputs: the others push their partial sums of them into its shared memory, it adds them in rank order --
// no workspace, no atomics, the same bits every time.  (Reading the peers' sums instead is a DSMEM round trip per addend:
// 201 x 4096 x 14336 took 39 us with it, 33 with the push.)
//
// CTA: warp 0 TMA producer (stages of 64 or 128 of k: 64-wide boxes of W and of x, 128-byte swizzle), warp 1 TMEM owner
// and tcgen05.mma issuer, both by an elected lane of a converged warp; then all eight warps move the accumulator (TMEM
// lane = output, column = row of x) to its shares or, unsplit, straight through the epilogue; the residual is fetched
// before the sums are there.  Up to two CTAs share an SM.  Every wait is bounded (npb_set_wait_limit_ns); on give-up
// the kernel records it, lets its copies land, frees its TMEM and returns.
//
// In a CUDA graph (launched one by one in brackets): 1 x 4096 x 4096 10.3 us (10.9; floor at the copy bandwidth 5.1), 16 x
// 14336 x 4096 25.7 us (26.6; 18.0), 201 x 4096 x 14336 34.0 us (37.5; 19.3; 9 TB/s into the SMs).
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
constexpr int kThreads = 256;  // eight warps: two CTAs fit an SM's register banks (ten warps of 96 registers do not)
constexpr int kWBox = BN * 64 * 2;  // 16 KiB: 64 of k (one swizzle row) of the tile's rows of W
constexpr int kMaxStages = 8;
constexpr int kHead = 1024;         // barriers

struct SkinnyParams {
  const float* bias;
  const void* residual;
  void* y;
  int M, N, act;
  int rows;       // of x per tile: multiple of 16, at most 256
  int boxes;      // of 64 of k per stage: 1 or 2
  int stages, k_stages, split;
  int part_rows;  // rows of x of the largest tile: their partial sums lie in the ring, or
  int part_at;    // behind it, so many bytes from its start (0: in it)
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
  const int x_box = p.rows * 128, stage_bytes = p.boxes * (kWBox + x_box);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = p.split > 1 ? (int)cluster_ctarank() : 0;  // share of K
  const int n0 = blockIdx.x / p.split * BN, m0 = blockIdx.y * p.rows;
  const int kb0 = (int)((int64_t)p.k_stages * rank / p.split), kb1 = (int)((int64_t)p.k_stages * (rank + 1) / p.split);
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
  if (p.split > 1 && p.part_at != 0) {
    __syncwarp();
    cluster_arrive();
  }

  if (warp == 0) {
    int s = 0;
    uint32_t ph = 1;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&empty[s], ph, abort_flag, p.wait_ns))) {
        atomicExch(&g_skinny_status, 1);
        break;
      }
      if (elect_one()) {
        uint8_t* st = ring + (size_t)s * stage_bytes;
        mbar_arrive_expect_tx(&full[s], (uint32_t)stage_bytes);
        for (int h = 0; h < p.boxes; ++h) {
          const int k = (kb * p.boxes + h) * 64;
          tma_load_2d(st + h * kWBox, &map_w, &full[s], k, n0);
          tma_load_2d(st + p.boxes * kWBox + h * x_box, &map_x, &full[s], k, m0);
        }
      }
      __syncwarp();
      if (++s == p.stages) { s = 0; ph ^= 1; }
    }
  } else if (warp == 1) {
    const uint32_t idesc = umma_idesc_f16(std::is_same<T, __nv_bfloat16>::value ? 1 : 0, BN, p.rows);
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&full[s], ph, abort_flag, p.wait_ns))) {
        atomicExch(&g_skinny_status, 2);
        ok = false;
        break;
      }
      tc_fence_after();
      if (elect_one()) {
        const uint32_t st = smem_u32(ring + (size_t)s * stage_bytes);
        for (int h = 0; h < p.boxes; ++h) {
          const uint64_t a = umma_desc_sw128(st + h * kWBox), b = umma_desc_sw128(st + p.boxes * kWBox + h * x_box);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16(tmem, a + 2 * k, b + 2 * k, idesc, (kb > kb0 || h > 0 || k > 0) ? 1u : 0u);
        }
        umma_commit(&empty[s]);
      }
      __syncwarp();
      if (++s == p.stages) { s = 0; ph ^= 1; }
    }
    if (ok && elect_one()) umma_commit(done);
  }
  __syncwarp();
  // Epilogue, 16 rows of x at a time: two warps share the 32 outputs of a TMEM quadrant.
  const int quad = warp & 3, lane_n = quad * 32 + lane, c0 = warp < 4 ? 0 : 16;  // TMEM lane = output of the tile
  const int rows = min(p.rows, p.M - m0);
  const uint32_t acc = tmem + ((uint32_t)(quad * 32) << 16);
  if (p.split == 1) {
    const bool in = n0 + lane_n < p.N, adds = p.residual != nullptr && in;
    const float bias = p.bias && in ? __ldg(p.bias + n0 + lane_n) : 0.f;
    float r[16];
    auto load_residual = [&](int c) {
#pragma unroll
      for (int i = 0; i < 16; ++i) r[i] = adds && c + i < rows ? residual_at<T>(p, m0 + c + i, n0 + lane_n) : 0.f;
    };
    load_residual(c0);
    if (__all_sync(0xffffffffu, mbar_wait_bounded(done, 0, abort_flag, p.wait_ns, 64u))) {
      tc_fence_after();
      for (int c = c0; c < rows; c += 32) {
        uint32_t v[16];
        tmem_ld_32x32_x16(acc + c, v);
        tmem_ld_wait();
        T* y = static_cast<T*>(p.y) + (int64_t)(m0 + c) * p.N + n0 + lane_n;
        float o[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = __uint_as_float(v[i]) + bias;
        activate_all(o, p.act);
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] += r[i];
        load_residual(c + 32);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (in && c + i < rows) y[(int64_t)i * p.N] = from_f32<T>(o[i]);
      }
    } else {
      atomicExch(&g_skinny_status, 3);
    }
    tc_fence_before();
  } else {
    // A CTA of the cluster finishes its share of the tile's outputs.  The others push their partial sums of them into
    // its shared memory, [rank][row of x][share]; it adds them in rank order, four outputs of a row at a time.
    struct alignas(8) Four { T e[4]; };
    constexpr int kAhead = 16;  // units of a thread, at most (256 rows, a split in two)
    const bool wide = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 7) == 0 &&
                      (reinterpret_cast<uintptr_t>(p.residual) & 7) == 0;
    const int share = BN / p.split, units = share / 4, row_step = kThreads / units;
    const int n = n0 + rank * share + tid % units * 4;  // this thread's outputs
    float bias[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) bias[k] = p.bias && n + k < p.N ? __ldg(p.bias + n + k) : 0.f;
    Four rest[kAhead];  // the residual: fetched before the sums are there, kept in shared memory while they are joined
    auto fetch = [&](int j) {
      rest[j] = Four{};
      const int row = tid / units + j * row_step;
      if (p.residual == nullptr || row >= rows) return;
      const T* from = static_cast<const T*>(p.residual) + (int64_t)(m0 + row) * p.N + n;
      if (wide) {
        if (n < p.N) rest[j] = *reinterpret_cast<const Four*>(from);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (n + k < p.N) rest[j].e[k] = from[k];
      }
    };
    const bool more = rows > row_step;  // few rows skip the code for many
    fetch(0);
    if (more) {
#pragma unroll
      for (int j = 1; j < kAhead; ++j) fetch(j);
    }
    const bool got = __all_sync(0xffffffffu, mbar_wait_bounded(done, 0, abort_flag, p.wait_ns, 64u));
    if (!got) atomicExch(&g_skinny_status, 3);
    tc_fence_after();
    const uint32_t part = smem_u32(ring) + p.part_at;
    Four* kept = reinterpret_cast<Four*>(ring + p.part_at + p.part_rows * BN * 4);  // [row][units]
    const uint32_t to = map_to_cta(part + (rank * p.part_rows * share + lane_n % share) * 4, lane_n / share);
    __syncwarp();
    if (p.part_at != 0) cluster_wait();  // the others have started
    else cluster_sync_all();             // the others are through with their rings
    if (tid / units < rows) kept[tid] = rest[0];
    if (more) {
#pragma unroll
      for (int j = 1; j < kAhead; ++j)
        if (tid / units + j * row_step < rows) kept[j * kThreads + tid] = rest[j];
    }
    if (got) {
      for (int c = c0; c < rows; c += 32) {
        uint32_t v[16];
        tmem_ld_32x32_x16(acc + c, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (c + i < rows)
            asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(to + (c + i) * share * 4), "r"(v[i]) : "memory");
      }
    }
    __syncwarp();
    cluster_sync_all();
    const float4* from = reinterpret_cast<const float4*>(ring + p.part_at) + tid;
#pragma unroll 1  // a short body: it runs a few times, and fetching it costs more than running it
    for (int row = tid / units; row < rows; row += 2 * row_step, from += 2 * kThreads) {
      const bool two = row + row_step < rows;
      const int next = two ? kThreads : 0;
      float sum[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) sum[k] = 0.f;
#pragma unroll 2
      for (int c = 0; c < p.split; ++c) {
        const float4 q = from[c * p.part_rows * units], r = from[c * p.part_rows * units + next];
        sum[0] += q.x; sum[1] += q.y; sum[2] += q.z; sum[3] += q.w;
        sum[4] += r.x; sum[5] += r.y; sum[6] += r.z; sum[7] += r.w;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) sum[k] += bias[k & 3];
      activate_all(sum, p.act);
      const Four* rest = kept + row * units + tid % units;
      T* y = static_cast<T*>(p.y) + (int64_t)(m0 + row) * p.N + n;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const Four r = rest[j * next];
        Four f;
#pragma unroll
        for (int k = 0; k < 4; ++k) f.e[k] = from_f32<T>(sum[j * 4 + k] + to_f32(r.e[k]));
        if (j == 1 && !two) break;
        if (wide) {
          if (n < p.N) *reinterpret_cast<Four*>(y) = f;
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (n + k < p.N) y[k] = f.e[k];
        }
        y += (int64_t)row_step * p.N;
      }
    }
    tc_fence_before();
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

template <typename T>
int launch_skinny(const cudaLaunchConfig_t& cfg, const CUtensorMap& map_w, const CUtensorMap& map_x,
                  const SkinnyParams& p) {
  auto kern = gemm_skinny_kernel<T>;
  int resident = 0;
  if (int rc = blocks_per_sm(reinterpret_cast<const void*>(kern), kThreads, cfg.dynamicSmemBytes, &resident)) return rc;
  if (resident < 1) return NPB_ERR_TOO_LARGE;
  NPB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, map_w, map_x, p));
  NPB_LAUNCH_CHECK();
  return NPB_OK;
}

}  // namespace

// CTAs of this kernel that run at once, one to an SM, in clusters of a size (a GPC's SMs do not divide evenly: 132 in
// clusters of four, 120 in clusters of eight on a B200).
int resident_ctas(int cluster, int* ctas) {
  static int cached[64][4] = {};
  int dev = 0, slot = cluster == 1 ? 0 : cluster == 2 ? 1 : cluster == 4 ? 2 : 3;
  NPB_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return NPB_ERR_CUDA;
  if (cached[dev][slot] == 0) {
    auto kern = gemm_skinny_kernel<__half>;
    int per_sm = 0;
    const int smem = max_dynamic_smem() / 2 + 2048;
    if (int rc = blocks_per_sm(reinterpret_cast<const void*>(kern), kThreads, smem, &per_sm)) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(sm_count() / cluster * cluster));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    NPB_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
    cached[dev][slot] = n > 0 ? n * cluster : cluster;
  }
  *ctas = cached[dev][slot];
  return NPB_OK;
}

// Whether this form is the faster one (this / the dense kernel, us): while tiles can be split over the SMs (201 rows, 4096
// x 14336: 34 / 58; 512 rows, 2048 x 8192: 25 / 36); in one wave of two tiles to an SM (64 rows, 14336 x 4096: 28 / 31;
// 160 rows: 34 / 39; 201 rows, with pairs of CTAs in this form as in the dense kernel: 39 / 39); in two waves, whose
// epilogues the dense kernel overlaps, with fewer rows (64 rows, 28672 x 8192: 89 / 90; 96 rows: 93 / 89); and with a few
// rows always (16 rows, 49152 x 4096: 78 / 82; 64 rows: 89 / 79).
bool gemm_skinny_takes(int64_t M, int64_t N) {
  const int64_t row_tiles = (M + 255) / 256, all = row_tiles * ((N + BN - 1) / BN);
  const int64_t rows = row_tiles ? (M + row_tiles - 1) / row_tiles : 0;
  if (all * 2 <= sm_count()) return true;
  if (all <= sm_count()) return rows <= 160;
  return row_tiles == 1 && rows <= (all <= 2 * sm_count() ? 64 : 32);
}

// Tiles of at most 256 rows of x; W is read once per tile of rows.
int gemm_skinny(const void* x, const void* w, const float* bias, int act, const void* residual, void* y, int64_t M,
                int64_t N, int64_t K, int dtype, cudaStream_t st) {
  SkinnyParams p{};
  p.bias = bias;
  p.residual = residual;
  p.y = y;
  p.M = (int)M; p.N = (int)N; p.act = act;
  const int row_tiles = (int)((M + 255) / 256);
  const int rows = (int)((M + row_tiles - 1) / row_tiles);
  const int64_t tiles = (N + BN - 1) / BN;
  const int half = max_dynamic_smem() / 2 - 1024 - 2048, whole = max_dynamic_smem() - 2048;
  p.rows = (rows + 15) / 16 * 16;
  p.wait_ns = wait_limit_ns();
  const int box_bytes = kWBox + p.rows * 128;  // of W and x, 64 of k
  // Too many tiles for a split in two, one CTA to an SM: two CTAs to an SM (128 rows, 14336 x 4096: 32 us, one to an SM
  // 39 us; the dense kernel takes the rows that leave no room for two).  Otherwise one CTA with the whole ring is better
  // (128 rows, 4096 x 4096: 14.8 us, two to an SM 16.3 us).
  const int per_sm = tiles * row_tiles * 2 > sm_count() ? 2 : 1, room = (per_sm == 2 ? half : whole) - kHead;
  p.boxes = room / box_bytes >= 6 ? 2 : 1;
  const int stage_bytes = p.boxes * box_bytes;
  p.stages = room / stage_bytes < kMaxStages ? room / stage_bytes : kMaxStages;
  p.k_stages = (int)((K + p.boxes * 64 - 1) / (p.boxes * 64));
  p.split = 1;
  while (p.split < 8 && p.k_stages >= p.split * 4) {
    int room_for = 0;  // CTAs that run at once, one to an SM, in clusters of twice the size
    if (int rc = resident_ctas(p.split * 2, &room_for)) return rc;
    // where two share an SM a tenth more than run at once is better than half as many
    const int64_t most = per_sm == 2 ? room_for * 2 * 11 / 10 : room_for;
    if (tiles * row_tiles * p.split * 2 > most) break;
    p.split *= 2;
  }
  const int ring = p.stages * stage_bytes, most_rows = (int)(M < p.rows ? M : p.rows);
  const int rest = most_rows * (BN / p.split) * 2;  // the residual's share
  // partial sums behind the ring need no wait for it; in it they have room whatever the sizes are (16 rows to spare at
  // least, with 227 KB to a CTA)
  const int join = p.split > 1 ? most_rows * BN * 4 + rest : 0;
  const bool behind = join > 0 && ring + join <= room;
  if (!behind && join > ring) return NPB_ERR_TOO_LARGE;
  p.part_at = behind ? ring : 0;
  p.part_rows = most_rows;
  const bool bf16 = dtype == NPB_BF16;
  CUtensorMap map_w, map_x;
  const CUtensorMapDataType type = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  if (int rc = make_tensor_map_2d(&map_w, type, 2, w, N, K, BN, 64, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  if (int rc = make_tensor_map_2d(&map_x, type, 2, x, M, K, p.rows, 64, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(tiles * p.split), (unsigned)row_tiles);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = 1024 + kHead + ring + (behind ? join : 0);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = p.split;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return bf16 ? launch_skinny<__nv_bfloat16>(cfg, map_w, map_x, p) : launch_skinny<__half>(cfg, map_w, map_x, p);
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
