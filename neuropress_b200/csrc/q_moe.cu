// A mixture-of-experts layer for a few tokens over 4-bit group-affine experts, in two kernels:
//
//   p = softmax(l_t);  S_t = the top_k largest l_t (equal logits: lowest expert);
//   w_te = p_e, or p_e / sum_{S_t} p
//   h_te[i] = w_te * silu(G_e x_t)[i] * (U_e x_t)[i]              kernel 1: routing, gate / up, silu
//   y_t     = T( sum_{e in S_t} D_e h_te )                         kernel 2: routing, down, sum
//   W[n, k] = (q[n, k] - z) * s  in fp32, z and s per group of k (z = 8 without a zero point)
//
// Each active expert's codes are read once; HBM-bound (0.56 bytes per weight at group 32).  Every CTA of the first
// kernel routes by itself (a warp per token); the second reads the outcome with h.  (Programmatic serialisation
// between the two was measured and dropped: the first kernel's CTAs fill the SMs, so the second cannot start under
// them; one token, 8 of 64 experts, 2048 x 1024: 22.5 us with it, 21.7 us without.)
//
// Product: mma.sync.m16n8k16 in fp16 with the weights as the A operand (16 rows) built in registers.  A code
// q becomes 1024 + q or, four bits higher in the mantissa, 1024 + 16 q with one bit operation per two
// codes; the activations that meet the latter are stored divided by 16.  With x' the stored activations
//   sum_k (q - z) x = D - 1024 sum_k x' - z sum_k x,   D the mma's sum
// is applied per 32-wide block, with the weight's scale, in fp32.  Activations are stored as fp16 after division by a
// power of two that brings the largest to 2^14 (so that next to all of fp16's range lies below it), one per token for x
// and one per 32-block and token for h.  Relative to the power of two at or below that largest, x is stored as it is down
// to 2^-27 (bf16) or 2^-24 (fp16) and h with 11 significant bits down to 2^-24; what is smaller is off by at most 2^-35.
//
// The eight columns of an mma are NT = 8 / G tokens times G neighbouring 32-blocks (G = 4, 2, 1): lane (g, t)
// of a warp loads G words, the t-th part of G blocks, of rows g and g + 8, so the k slots of an mma hold
// G different blocks, and the B operand keeps them apart by being block-diagonal.  Lane (g, t) of the result
// then holds two tokens of exactly the block whose scale it loaded.  A step of four blocks takes the same
// sixteen mmas for two 16-row tiles whatever G is (8 cycles of a scheduler's tensor pipe each, measured);
// G = 4 has the widest loads and the fewest results to scale, G = 1 the most tokens per weight read.
//
// Weights stream through a ring of rounds in shared memory, filled by producer warps: codes as TMA boxes of 64 bytes of
// k with the 64-byte swizzle (no bank conflicts when read, nothing in the L1 path), scales and zero points as TMA
// boxes or, where their rows are not aligned, by cp.async.  In a round each of the sixteen consumer warps takes one
// step of two 16-row tiles.  Kernel 1 keeps the tokens of a unit (up to NT tokens of one expert), or all of them
// where there are no more than NT, in shared memory in the order of the mma operands and writes h in that order;
// kernel 2 brings h along with the weights.  An expert with more tokens than a unit is read again (from L2).  Every
// sum has a fixed order: results do not depend on scheduling.  Waits on the barriers are bounded like those of the
// GEMMs.
//
// What bounds it: the consumers' own latency.  Without the loads the two kernels take 101 + 49 us of 103 + 52 (4 tokens, 2 of
// 8 experts, 4096 x 14336), without the products 79 + 36, so the products are the longer part; but they use 54-60 % of the
// issue slots (about 300 instructions a step: 16 mma.sync, 80 that turn codes into operands), and their largest stall is
// the fixed-latency wait: four warps a scheduler with one chain each do not cover it.  Most forms of kernel 1 spill a few
// registers at 96 (up to 150 bytes a thread).  In a CUDA graph: that case 152 us (floor at the copy bandwidth 83), 32
// tokens, 8 of 64 experts, 4096 x 1376 188 us (92), 1 token, 8 of 64, 2048 x 1024 21 us, of which 9 are launches, routing and
// fills.  More than 32 tokens take a pair of launches for every 32, which read and convert their experts again: 512 tokens of
// 4096 x 1376 3.0 ms, 2048 12 ms (expert by expert through the framework's 4-bit linears 4.5 and 5.1 ms).
// Measured and left: register double buffers (a third of the bandwidth: waiting for one step's loads waits for the
// next step's too); a ring of each warp's own (80-110 more instructions a step: 185 us for the first case, 206 for the
// second); 32 consumer warps of 64 registers (spills: 242 and 366 us); 16 warps that fetch in turn (190 and 234 us).
#include <type_traits>

#include "common.cuh"
#include "order_key.cuh"
#include "tcgen05.cuh"

namespace npb {

// gemm_tcgen05.cu
int make_tensor_map_2d(CUtensorMap* map, CUtensorMapDataType type, int elem_bytes, const void* base, int64_t rows,
                       int64_t cols, int box_rows, int box_cols, CUtensorMapSwizzle swizzle);

__device__ int g_moe_status = 0;  // 0 ok; 1, 2: the kernel one of whose waits gave up

namespace {

constexpr int kMaxTokens = 32;   // bits of an expert's token mask
constexpr int kMaxExperts = 512;
constexpr int kMaxTopK = 16;
constexpr int kMaxUnits = kMaxTokens * kMaxTopK;
constexpr int kMaxWidth = 16384;  // of H and I: two tokens of H in shared memory next to the rings

struct Units;

struct MoeWeight {
  const uint8_t* codes;
  const __half* scale;
  const __half* zp;  // null: symmetric, z = 8
  int group_shift;   // log2 of the 32-blocks per group, or -1: divide
  int group_blocks;
};

struct MoeParams {
  const void* x;
  const void* logits;
  int logits_dtype, dtype;
  int T, E, H, I, top_k, renormalize;
  MoeWeight gate, up, down;
  uint8_t* h;      // [pair of tokens of a unit][I / 32, padded to whole steps] records
  Units* units;
  void* y;
  uint64_t wait_ns;
  int stages;      // of the ring
  int window;      // bytes of a row's groups in a round
  int slices;      // kernel 2: of k in a round; 16 / slices warps side by side over the rows
  int split;       // kernel 2: CTAs of a cluster
};

// One 32-block of h of two tokens: 32 stored fp16 values of each (64 bytes), then {m0, m1, m0, m1, f0, f1, s2 of both}.
constexpr int kRecord = 160;

// ---- routing ---------------------------------------------------------------------------------
// The work lists: a unit is up to NT tokens of one expert.
struct Units {
  int n;
  int unused[3];
  uint32_t mask[kMaxUnits];      // the unit's tokens
  uint16_t expert[kMaxUnits];
  uint16_t slot[kMaxUnits];      // row of h of its first pair
};

struct Routing {
  float weight[kMaxTokens][kMaxTopK];
  uint16_t id[kMaxTokens][kMaxTopK];     // 0xffff: none
  Units units;
};

__device__ __forceinline__ float load_logit(const MoeParams& p, int64_t i) {
  if (p.logits_dtype == NPB_F32) return __ldg(static_cast<const float*>(p.logits) + i);
  if (p.logits_dtype == NPB_BF16) return to_f32(static_cast<const __nv_bfloat16*>(p.logits)[i]);
  return to_f32(static_cast<const __half*>(p.logits)[i]);
}

// The choices of every token, a warp per token; a lane holds experts lane, lane + 32, ...
template <int PER_LANE>
__device__ void choose(const MoeParams& p, Routing& r, uint32_t* tokens) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  for (int t = warp; t < p.T; t += warps) {
    uint32_t key[PER_LANE];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) {
      key[i] = i * 32 + lane < p.E ? order_key(load_logit(p, (int64_t)t * p.E + i * 32 + lane)) : 0u;
      top = max(top, key[i]);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    const float m = top <= 1u ? -INFINITY : key_value(top);  // a row of NaN alone has no maximum
    float all = 0.f;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i)
      if (key[i] != 0) {
        all += expf(key_value(key[i]) - m);
        nan |= key[i] == 1u;
      }
    all = warp_sum(all);
    // a row with NaN or +inf has NaN weights (all is NaN); a row of -inf alone is routed nowhere
    const bool nowhere = m == -INFINITY && !__any_sync(0xffffffffu, nan);
    uint32_t mine = 0, mine_e = 0;  // lane j: the j-th largest
    for (int j = 0; j < p.top_k; ++j) {
      uint32_t best = 0;
      int at = 0;
#pragma unroll
      for (int i = 0; i < PER_LANE; ++i)
        if (key[i] > best) { best = key[i]; at = i; }
      top = __reduce_max_sync(0xffffffffu, best);
      const uint32_t e = __reduce_min_sync(0xffffffffu, best == top ? (uint32_t)(at * 32 + lane) : 0xffffffffu);
#pragma unroll
      for (int i = 0; i < PER_LANE; ++i)
        if (i * 32 + lane == (int)e) key[i] = 0;
      if (lane == j) {
        mine = top;
        mine_e = e;
      }
    }
    const float l = key_value(mine), w = lane < p.top_k ? expf(l - m) : 0.f;
    const float norm = p.renormalize ? (all != all ? all : warp_sum(w)) : all;
    if (lane < p.top_k) {
      const bool none = nowhere || (l == -INFINITY && all == all);  // probability 0: not read
      r.id[t][lane] = none ? 0xffffu : (uint16_t)mine_e;
      r.weight[t][lane] = w / norm;
      if (!none) atomicOr(&tokens[mine_e], 1u << t);
    }
  }
}

// All threads of the CTA; ends with a barrier.  A unit is up to NT tokens of one expert.  `tokens` [kMaxExperts] is
// scratch that TMA may write afterwards.
template <int NT>
__device__ void route(const MoeParams& p, Routing& r, uint32_t* tokens) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) tokens[e] = 0;
  __syncthreads();
  if (p.E <= 64) choose<2>(p, r, tokens);
  else if (p.E <= 128) choose<4>(p, r, tokens);
  else choose<kMaxExperts / 32>(p, r, tokens);
  __syncthreads();
  if (warp == 0) {
    int units = 0, slots = 0;
    for (int base = 0; base < p.E; base += 32) {
      const int e = base + lane;
      const int n = e < p.E ? __popc(tokens[e]) : 0;
      const int u = (n + NT - 1) / NT, pairs = (n + 1) / 2;
      int iu = u, in = pairs;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, iu, o), b = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) { iu += a; in += b; }
      }
      uint32_t m = n > 0 ? tokens[e] : 0u;
      for (int i = 0; i < u; ++i) {
        const int at = units + iu - u + i;
        uint32_t rest = m;
        for (int j = 0; j < NT && rest; ++j) rest &= rest - 1;
        r.units.expert[at] = (uint16_t)e;
        r.units.mask[at] = m & ~rest;
        r.units.slot[at] = (uint16_t)(slots + in - pairs + i * (NT / 2));
        m = rest;
      }
      units += __shfl_sync(0xffffffffu, iu, 31);
      slots += __shfl_sync(0xffffffffu, in, 31);
    }
    if (lane == 0) r.units.n = units;
  }
  sm100::fence_proxy_async_smem();
  __syncthreads();
}

// ---- weights ---------------------------------------------------------------------------------
__device__ __forceinline__ int group_of(const MoeWeight& w, int blk) {
  return w.group_shift >= 0 ? blk >> w.group_shift : blk / w.group_blocks;
}

// 16 bytes, of which the first `bytes` are read and the rest is zero.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// The barrier counts one arrival once this thread's copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(sm100::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(sm100::smem_u32(bar))
               : "memory");
}

// For the producers.  A consumer whose wait gave up raises the flag, then goes on to free stages that copies may still land
// in: those are not filled again.
__device__ __forceinline__ bool stage_is_free(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint64_t wait_ns) {
  return sm100::mbar_wait_bounded(bar, parity, abort_flag, wait_ns) && *abort_flag == 0;
}

// How groups come: kOnePerBlock (a group is a block) and kPowerOfTwo (a group is 2^n blocks) have rows of whole 16-byte
// pieces, which TMA takes; kAny is the rest.
enum { kAny = 0, kOnePerBlock = 1, kPowerOfTwo = 2 };

constexpr int kConsumers = 16;                    // warps
// Producer warps: one issues TMA, all copy the windows that TMA cannot take (four against one: 111 -> 83 us for 32
// tokens of 64 experts 4096 x 1376; without windows to copy the three would only cost, 118 -> 126 us for 4096 -> 14336).
constexpr int producers(int mode) { return mode == kAny ? 4 : 1; }
constexpr int threads_of(int mode) { return (kConsumers + producers(mode)) * 32; }
constexpr int kMaxStages = 4;

// A round's groups of a row lie in a window of p.window bytes that starts with group window_start of the row: a multiple
// of eight (counted in the matrix for kAny, where rows start anywhere).
template <int MODE>
__device__ __forceinline__ int window_start(const MoeWeight& w, int first_blk) {
  return MODE == kAny ? group_of(w, first_blk) : group_of(w, first_blk) & ~7;
}
// The swizzle that TMA gives a window of 64 or 32 bytes, for rows that are r modulo 8.
template <int MODE>
__device__ __forceinline__ int window_swizzle(int bytes, int r) {
  return MODE == kAny ? 0 : bytes == 64 ? r >> 1 & 3 : bytes == 32 ? r >> 2 & 1 : 0;
}
// Copies the windows of `rows` rows (kAny; by the producer warps, a lane per row): row i starts at group at + i * n_group
// of `total`.
__device__ __forceinline__ void copy_windows(uint32_t dst, const __half* groups, int rows, int bytes, int64_t at,
                                             int n_group, int64_t total, int lane) {
  for (int row = lane; row < rows; row += producers(kAny) * 32) {
    const int64_t first = (at + row * n_group) & ~7ll;
    const int left = (int)min((int64_t)bytes, (total - first) * 2);  // what the matrix still holds
    const __half* src = groups + (left > 0 ? first : 0);
#pragma unroll 1
    for (int b = 0; b < bytes; b += 16) {
      const int n = min(16, max(0, left - b));
      cp_async16(dst + row * bytes + b, n ? src + b / 2 : src, n);
    }
  }
}

// Tile row of lane group g: G = 2 reads half pieces, which needs every other pair of rows in a phase.
template <int G>
__device__ __forceinline__ int row_of(int g) { return G == 2 ? (g & 1) | (g & 2) << 1 | (g & 4) >> 1 : g; }

__device__ __forceinline__ float half_bits(uint32_t v) { return __half2float(__ushort_as_half((unsigned short)v)); }

// The value of this lane's block of set j among the four of a step.
template <int G>
__device__ __forceinline__ float group_value(const uint2& v, int j, int t) {
  const uint32_t w = G == 4 ? (t & 2 ? v.y : v.x) : (G == 2 ? j : j / 2) ? v.y : v.x;
  const __half2 pair = *reinterpret_cast<const __half2*>(&w);
  if (G == 1) return j & 1 ? __high2float(pair) : __low2float(pair);
  return half_bits(w >> (G == 4 ? (t & 1) * 16 : t / 2 * 16));
}

// Pair j of a word's codes, j and j + 4, as two fp16 values: 1024 + q (j even) or 1024 + 16 q (j odd).
__device__ __forceinline__ uint32_t code_pair(uint32_t word, int odd) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(word), "r"(odd ? 0x00f000f0u : 0x000f000fu), "r"(0x64006400u));
  return r;
}

// The A operands of one word of rows (l, h): two mmas of 16 k slots each.
__device__ __forceinline__ void a_operands(uint32_t l, uint32_t h, uint32_t (&a)[2][4]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    a[k][0] = code_pair(l, 0);
    a[k][1] = code_pair(h, 0);
    a[k][2] = code_pair(l, 1);
    a[k][3] = code_pair(h, 1);
    l >>= 8;
    h >>= 8;
  }
}

// ---- stored activations --------------------------------------------------------------------
// The power of two that values up to a magnitude are divided by, as its exponent field (15..241): the magnitude comes to
// [2^14, 2^15), which fp16 holds even where its rounding goes up.  At least 2^-112, so that the product with a normal fp16
// scale stays normal.  (Infinite values stay so, and their products become NaN.)
__device__ __forceinline__ uint32_t storage_exponent(float top) { return max(__float_as_uint(top) >> 23, 29u) - 14u; }
__device__ __forceinline__ float power_of(uint32_t exponent) { return __uint_as_float(exponent << 23); }
__device__ __forceinline__ float reciprocal_of(uint32_t exponent) { return __uint_as_float((254u - exponent) << 23); }

// A block's m and s2 from the sums of its stored values at k = 0, 2 mod 4 (`even`) and 1, 3 mod 4 (`odd`, divided
// by 16).
__device__ __forceinline__ void put_sides(float* m, float* s2, float even, float odd, bool asym) {
  const float sum = even + 16.f * odd, magic = -1024.f * (even + odd);
  m[0] = m[2] = asym ? magic : magic - 8.f * sum;
  if (s2) *s2 = sum;
}

// mma.sync.m16n8k16 fp16; a plain (not volatile) asm, so that the compiler may interleave the tiles
__device__ __forceinline__ void mma_add(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                         const float4& c) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c.x), "f"(c.y), "f"(c.z), "f"(c.w));
}

// What a block of two tokens brings besides its values: {m0, m1, m0, m1}, minus what the magic (and, for a
// symmetric weight, z = 8) adds, as the first mma's C operand; their powers of two and their sums.
struct Sides {
  const uint8_t *m, *f, *s2;
};

// Where one step of two 16-row tiles lies: codes of a row 64 bytes apart, TILE bytes from tile to tile; windows of a
// row `pitch` bytes apart, `window_tile` bytes from tile to tile, zero points `zeros` behind the scales.
struct StepAt {
  const uint8_t* codes;
  const uint8_t* window;
  int pitch, window_tile, zeros;
};

// Adds step s to acc[tile] (rows row_of(g) and + 8 of two tokens, as the mma has them).  `start` is the group that the
// windows start with, `first` the place of that group in this lane's row (kAny); `operand` this lane's part of the
// first set in B order, BLOCK bytes from block to block (a lane off the diagonal: zeros); `sides` belong to its two
// tokens and its block of the first set, MS and FS bytes from block to block.
template <int G, bool ASYM, int MODE, bool SCALED, int TILE, int BLOCK, int MS, int FS>
__device__ __forceinline__ void add_step(float (&acc)[2][4], const StepAt& at, int start, int first,
                                         const uint8_t* operand, const Sides& sides, int g, int t, int s, int n_blk,
                                         const MoeWeight& w) {
  const int r0 = row_of<G>(g), swizzle = window_swizzle<MODE>(at.pitch, r0);
  const uint8_t* row = at.window + r0 * at.pitch;
  // place of group x of a row in its window
  auto place = [&](int x) {
    const int byte = (x - start + first) * 2;
    return ((byte >> 4 ^ swizzle) << 4) + (byte & 15);
  };
  uint2 sc[2][2], zp[ASYM ? 2 : 1][2];
  if constexpr (MODE == kOnePerBlock) {
    const uint8_t* from = row + place(s * 4);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sc[i][h] = *reinterpret_cast<const uint2*>(from + i * at.window_tile + h * 8 * at.pitch);
        if (ASYM)
          zp[ASYM ? i : 0][h] = *reinterpret_cast<const uint2*>(from + i * at.window_tile + h * 8 * at.pitch + at.zeros);
      }
  }
  // kPowerOfTwo: a step has one group or (64-wide) two; in the halves of a word the groups of the first and the second
  // two blocks, or this lane's twice
  uint32_t sw[MODE == kPowerOfTwo ? 2 : 1][2], zw[MODE == kPowerOfTwo && ASYM ? 2 : 1][2];
  if constexpr (MODE == kPowerOfTwo) {
    const int group = group_of(w, s * 4);
    const uint8_t* from = row + place(group & ~1);
    const uint32_t lower = 0x1010, upper = 0x3232;
    const uint32_t halves = w.group_shift > 1 ? (group & 1 ? upper : lower) : G < 4 ? 0x3210 : t & 2 ? upper : lower;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* value = from + i * at.window_tile + h * 8 * at.pitch;
        sw[i][h] = __byte_perm(*reinterpret_cast<const uint32_t*>(value), 0u, halves);
        if (ASYM)
          zw[ASYM ? i : 0][h] = __byte_perm(*reinterpret_cast<const uint32_t*>(value + at.zeros), 0u, halves);
      }
  }
#pragma unroll
  for (int j = 0; j < 4 / G; ++j) {
    // this lane's G words of the set: 16-byte piece (block) of the row, word t mod 4 / G times G
    const int piece = ((j * G + t / (4 / G)) ^ (r0 >> 1 & 3)) * 16 + t % (4 / G) * (4 * G);
    uint32_t c[4][G];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t* from = at.codes + r0 * 64 + piece + i / 2 * TILE + i % 2 * 512;
      if constexpr (G == 4) *reinterpret_cast<uint4*>(c[i]) = *reinterpret_cast<const uint4*>(from);
      else if constexpr (G == 2) *reinterpret_cast<uint2*>(c[i]) = *reinterpret_cast<const uint2*>(from);
      else c[i][0] = *reinterpret_cast<const uint32_t*>(from);
    }
    const float4 m = *reinterpret_cast<const float4*>(sides.m + j * G * MS);
    float d[2][4];
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(operand + j * G * BLOCK + i * 16);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint32_t a[2][4];
        a_operands(c[2 * q][i], c[2 * q + 1][i], a);
        if (i == 0) mma_from(d[q], a[0], v.x, v.y, m);
        else mma_add(d[q], a[0], v.x, v.y);
        mma_add(d[q], a[1], v.z, v.w);
      }
    }
    float2 f = make_float2(1.f, 1.f), s2 = make_float2(0.f, 0.f);
    if (SCALED) f = *reinterpret_cast<const float2*>(sides.f + j * G * FS);
    if (ASYM) s2 = *reinterpret_cast<const float2*>(sides.s2 + j * G * FS);
    // this lane's block of the set; past the row's last (whose products are zero) the last one's scale will do
    int own = s * 4 + j * G + t / (4 / G);
    if (MODE == kAny) own = min(own, n_blk - 1);
    const uint8_t* from = MODE == kAny ? row + place(group_of(w, own)) : row;
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float scale, z = 0.f;
        if constexpr (MODE == kOnePerBlock) {
          scale = group_value<G>(sc[q][h], j, t);
          if (ASYM) z = group_value<G>(zp[ASYM ? q : 0][h], j, t);
        } else if constexpr (MODE == kPowerOfTwo) {
          constexpr int kHalf = 4 / G / 2;  // sets of the first two blocks
          const bool second = kHalf > 0 && j >= kHalf;
          scale = half_bits(second ? sw[q][h] >> 16 : sw[q][h]);
          if (ASYM) z = half_bits(second ? zw[ASYM ? q : 0][h] >> 16 : zw[ASYM ? q : 0][h]);
        } else {
          const uint8_t* value = from + q * at.window_tile + h * 8 * at.pitch;
          scale = half_bits(*reinterpret_cast<const uint16_t*>(value));
          if (ASYM) z = half_bits(*reinterpret_cast<const uint16_t*>(value + at.zeros));
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float fk = k ? f.y : f.x, sk = k ? s2.y : s2.x;
          float v = d[q][2 * h + k];
          if (ASYM) v = fmaf(-z, sk, v);
          acc[q][2 * h + k] = fmaf(SCALED ? scale * fk : scale, v, acc[q][2 * h + k]);
        }
      }
  }
}

__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// Sum over the lanes of a quad that hold the same tokens of different blocks; lanes t < 4 / G then hold
// tokens 2 t and 2 t + 1.
template <int G>
__device__ __forceinline__ float block_sum(float v) {
  if (G == 4) v += __shfl_xor_sync(0xffffffffu, v, 1);
  if (G >= 2) v += __shfl_xor_sync(0xffffffffu, v, 2);
  return v;
}

__device__ __forceinline__ void consumer_barrier() { asm volatile("bar.sync 1, 512;" ::: "memory"); }

// ---- kernel 1: gate / up products, silu, routing weight ------------------------------------------
constexpr int kUpRows = 32;      // rows of gate and of up per item: one 32-block of h
constexpr int kUpSlices = 8;     // steps of k in a round: a warp takes one, of 16 rows of gate and of up
constexpr int kUpCodes = kUpSlices * 2 * kUpRows * 64;  // [slice][gate, up][32][64]

// Shared memory of kernel 1 behind the routing: the ring (codes, then windows [scales of gate, of up, zero points of
// either][32][window]), tokens [NT][4 * steps] blocks of 64 bytes (neighbouring rows in the other half of the banks),
// their m [NT / 2][blocks + 1] (pairs in different banks) and s2 [NT / 2][blocks], the partial products of two items
// [slice][gate, up][NT][32] (while one is finished the next is computed), 256 bytes of zeros, barriers.
struct UpLayout {
  int windows, window_stage, x, row, m, s2, red, red_item, zeros, bars, bytes;
  __host__ __device__ UpLayout(int n_blk, int nt, bool asym, int window, int stages) {
    const int blocks = (n_blk + 3) / 4 * 4;
    windows = stages * kUpCodes;
    window_stage = (asym ? 4 : 2) * kUpRows * window;
    x = windows + stages * window_stage;
    row = blocks * 64 + 64;
    m = x + row * nt;
    s2 = m + nt / 2 * (blocks + 1) * 16;
    red = s2 + (asym ? nt / 2 * blocks * 8 : 0);
    red_item = kUpSlices * 2 * nt * kUpRows * 4;
    zeros = red + 2 * red_item;
    bars = zeros + 256;
    bytes = bars + 2 * kMaxStages * 8 + 1024;  // + alignment of the start
  }
};

// Stores eight elements of a token (thread j of a row: elements 8 j ...), times `by`, in the order of the mma
// operands, and their block's sides; the lanes of a quad share a block.
template <typename T>
__device__ __forceinline__ void store_operand(const uint4& raw, float by, uint4* to, float* m, float* s2, bool write,
                                              bool asym) {
  const T* v = reinterpret_cast<const T*>(&raw);
  __half2 o[4];
  float even = 0.f, odd = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float f = k & 1 ? by * 0.0625f : by;
    o[k] = __floats2half2_rn(to_f32(v[k]) * f, to_f32(v[k + 4]) * f);
    (k & 1 ? odd : even) += __low2float(o[k]) + __high2float(o[k]);
  }
  even = quad_sum(even);
  odd = quad_sum(odd);
  if (write) {
    *to = *reinterpret_cast<const uint4*>(o);
    if ((threadIdx.x & 3) == 0) put_sides(m, s2, even, odd, asym);
  }
}
template <typename T>
__device__ __forceinline__ float largest(const uint4& raw) {
  const T* v = reinterpret_cast<const T*>(&raw);
  float top = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(to_f32(v[k])));
  return top;
}

struct UpMaps {
  CUtensorMap codes[2], scale[2], zero[2];  // gate, up
};

template <int G, bool ASYM, int MODE>
__global__ void __launch_bounds__(threads_of(MODE), 1)
moe_up_kernel(const __grid_constant__ UpMaps maps, const MoeParams p) {
  constexpr int NT = 8 / G, kStagers = kConsumers * 32, kThreads = threads_of(MODE);
  extern __shared__ uint8_t dyn_raw[];
  uint8_t* dyn = dyn_raw + ((1024u - (sm100::smem_u32(dyn_raw) & 1023u)) & 1023u);
  __shared__ Routing r;
  __shared__ uint32_t x_top[NT];     // bits of the largest magnitude of each token
  __shared__ float x_f[NT];
  __shared__ int abort_flag;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int n_blk = p.H / 32, n_steps = (n_blk + 3) / 4, blocks = n_steps * 4;
  const int rounds = (n_steps + kUpSlices - 1) / kUpSlices, n_group = n_blk / p.gate.group_blocks;
  const UpLayout at(n_blk, NT, ASYM, p.window, p.stages);
  uint64_t* full = reinterpret_cast<uint64_t*>(dyn + at.bars);
  uint64_t* empty = full + kMaxStages;
  if (tid < 64) reinterpret_cast<uint32_t*>(dyn + at.zeros)[tid] = 0;
  if (tid == 0) {
    abort_flag = 0;
    for (int i = 0; i < p.stages; ++i) {
      sm100::mbar_init(&full[i], MODE == kAny ? producers(MODE) * 32 + 1 : 1);
      sm100::mbar_init(&empty[i], kConsumers);
    }
    sm100::fence_barrier_init();
  }

  // The tokens whose columns the mma computes: those of the unit at hand, or all of them where they fit.
  const bool resident = p.T <= NT, bf16 = p.dtype == NPB_BF16, held = blocks * 4 <= kStagers;
  uint32_t staged = resident ? (p.T < 32 ? (1u << p.T) - 1u : ~0u) : 0u;
  uint4 raw[NT] = {};
  auto load = [&](int j) {  // eight elements of each
    uint32_t m = staged;
#pragma unroll
    for (int i = 0; i < NT; ++i, m &= m - 1) {
      raw[i] = make_uint4(0, 0, 0, 0);
      if (m != 0 && j < n_blk * 4)
        raw[i] = __ldg(reinterpret_cast<const uint4*>(p.x) + (int64_t)(__ffs(m) - 1) * (n_blk * 4) + j);
    }
  };
  // Brings the staged tokens to shared memory: the largest magnitude of each, then the stored values; rows of up to
  // 4096 stay in registers between the two.  (Columns past the last token hold what was there: nothing reads their
  // sums.)  By the consumers; `loaded` if raw holds them already.
  auto stage_tokens = [&](bool loaded) {
    const int n = __popc(staged);
    if (tid < NT) x_top[tid] = 0;
    consumer_barrier();  // everybody is through with the tokens before
    float top[NT] = {};
#pragma unroll 1
    for (int j = tid; j < blocks * 4; j += kStagers) {
      if (!(loaded && held)) load(j);
#pragma unroll
      for (int i = 0; i < NT; ++i)
        top[i] = fmaxf(top[i], bf16 ? largest<__nv_bfloat16>(raw[i]) : largest<__half>(raw[i]));
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top[i]));
      if (lane == 0 && i < n) atomicMax(&x_top[i], bits);
    }
    consumer_barrier();
    if (tid < n) x_f[tid] = power_of(storage_exponent(__uint_as_float(x_top[tid])));
#pragma unroll 1
    for (int j0 = 0; j0 < blocks * 4; j0 += kStagers) {  // whole warps
      const int j = j0 + tid;
      if (!held) load(j);
#pragma unroll
      for (int i = 0; i < NT; ++i)
        if (i < n) {
          // a division (exact), not reciprocal_of: with that the compiler spills (32 tokens, 8 of 64 experts: 192 us, 188 us)
          const float by = 1.f / power_of(storage_exponent(__uint_as_float(x_top[i])));
          uint4* to = reinterpret_cast<uint4*>(dyn + at.x + i * at.row + j * 16);
          float* to_m = reinterpret_cast<float*>(dyn + at.m) + (i / 2 * (blocks + 1) + (j >> 2)) * 4 + (i & 1);
          float* to_s2 = ASYM ? reinterpret_cast<float*>(dyn + at.s2) + (i / 2 * blocks + (j >> 2)) * 2 + (i & 1) : nullptr;
          const bool write = j < blocks * 4;
          if (bf16) store_operand<__nv_bfloat16>(raw[i], by, to, to_m, to_s2, write, ASYM);
          else store_operand<__half>(raw[i], by, to, to_m, to_s2, write, ASYM);
        }
    }
    consumer_barrier();
  };
  if (resident && held && warp < kConsumers) load(tid);  // on their way while the tokens are routed
  route<NT>(p, r, reinterpret_cast<uint32_t*>(dyn));

  if (blockIdx.x == 0) {  // for kernel 2
    if (tid == 0) p.units->n = r.units.n;
    for (int i = tid; i < r.units.n; i += kThreads) {
      p.units->mask[i] = r.units.mask[i];
      p.units->expert[i] = r.units.expert[i];
      p.units->slot[i] = r.units.slot[i];
    }
  }
  const int tiles = p.I / kUpRows;
  const int64_t items = (int64_t)tiles * r.units.n;
  const int first = (int)(items * blockIdx.x / gridDim.x), last = (int)(items * (blockIdx.x + 1) / gridDim.x);
  int stage = 0;
  uint32_t parity = 0;
  auto advance = [&] {
    if (++stage == p.stages) {
      stage = 0;
      parity ^= 1;
    }
  };
  bool ok = true;

  if (warp >= kConsumers) {
    // ---- producers ----
    const int thread = tid - kConsumers * 32;
    const uint32_t base = sm100::smem_u32(dyn);
    const int64_t total_groups = (int64_t)p.E * p.I * n_group;
    for (int item = first; item < last && ok; ++item) {
      const int u = item / tiles, row = r.units.expert[u] * p.I + (item - u * tiles) * kUpRows;
      for (int round = 0; round < rounds; ++round, advance()) {
        ok = stage_is_free(&empty[stage], parity ^ 1, &abort_flag, p.wait_ns);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        const int s0 = round * kUpSlices, n = min(kUpSlices, n_steps - s0);
        const int start = window_start<MODE>(p.gate, s0 * 4);
        uint8_t* codes = dyn + stage * kUpCodes;
        const int windows = at.windows + stage * at.window_stage, part = kUpRows * p.window;
        if (warp == kConsumers && sm100::elect_one()) {
          sm100::mbar_arrive_expect_tx(&full[stage], n * 2 * kUpRows * 64 + (MODE == kAny ? 0 : at.window_stage));
          for (int i = 0; i < n; ++i)
#pragma unroll
            for (int w = 0; w < 2; ++w)
              sm100::tma_load_2d(codes + (i * 2 + w) * kUpRows * 64, &maps.codes[w], &full[stage], (s0 + i) * 64, row);
          if (MODE != kAny) {
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              sm100::tma_load_2d(dyn + windows + w * part, &maps.scale[w], &full[stage], start, row);
              if (ASYM) sm100::tma_load_2d(dyn + windows + (2 + w) * part, &maps.zero[w], &full[stage], start, row);
            }
          }
        }
        if (MODE == kAny) {
          const int64_t group = (int64_t)row * n_group + start;
#pragma unroll 1
          for (int w = 0; w < (ASYM ? 4 : 2); ++w) {
            const MoeWeight& from = w & 1 ? p.up : p.gate;
            copy_windows(base + windows + w * part, w < 2 ? from.scale : from.zp, kUpRows, p.window, group, n_group,
                         total_groups, thread);
          }
          cp_async_arrive(&full[stage]);
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    // ---- consumers ----
    const int mt = warp & 1, ks = warp >> 1;
    const int lane_blk = t / (4 / G);      // this lane's block of a set
    const bool diag = g / NT == lane_blk;  // it holds the nonzero part of column g
    const uint8_t* operand = dyn + (diag ? at.x + (g % NT) * at.row + lane_blk * 64 + t % (4 / G) * G * 16 : at.zeros);
    const int operand_step = diag ? 256 : 0, pair = t % (4 / G);
    const Sides sides{dyn + at.m + (pair * (blocks + 1) + lane_blk) * 16, nullptr,
                      dyn + at.s2 + (pair * blocks + lane_blk) * 8};
    if (resident) stage_tokens(true);
    for (int item = first; item < last; ++item) {
      const int u = item / tiles, i0 = (item - u * tiles) * kUpRows, e = r.units.expert[u];
      const uint32_t mask = r.units.mask[u];
      if (!resident && mask != staged) {
        staged = mask;
        stage_tokens(false);
      }
      float acc[2][4] = {};
      for (int round = 0; round < rounds; ++round, advance()) {
        const int s = round * kUpSlices + ks;
        ok = sm100::mbar_wait_bounded(&full[stage], parity, &abort_flag, p.wait_ns) && ok;
        if (s < n_steps) {
          const int start = window_start<MODE>(p.gate, round * kUpSlices * 4);
          const int place = MODE == kAny ? (row_of<G>(g) * n_group + start) & 7 : 0;
          const uint8_t* windows = dyn + at.windows + stage * at.window_stage;
          const StepAt here{dyn + stage * kUpCodes + ks * 2 * kUpRows * 64 + mt * 1024, windows + mt * 16 * p.window,
                            p.window, kUpRows * p.window, 2 * kUpRows * p.window};
          add_step<G, ASYM, MODE, false, kUpRows * 64, 64, 16, 8>(
              acc, here, start, place, operand + s * operand_step,
              Sides{sides.m + s * 64, nullptr, sides.s2 + s * 32}, g, t, s, n_blk, p.gate);
        }
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&empty[stage]);
      }
      float* red = reinterpret_cast<float*>(dyn + at.red + (item & 1) * at.red_item);
      // the blocks of a set, then the slices of K
      float* part = red + ks * 2 * NT * kUpRows;
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float q = block_sum<G>(acc[w][2 * h + c]);
            if (t < 4 / G) part[(w * NT + 2 * t + c) * kUpRows + mt * 16 + row_of<G>(g) + h * 8] = q;
          }
      consumer_barrier();
      // a warp per column, a lane per row; the warps take turns, as the others go on
      const int column = (warp - item * NT) & (kConsumers - 1);
      uint32_t m = staged;
      for (int i = 0; i < column; ++i) m &= m - 1;
      const int token = __ffs(m) - 1;
      if (column < NT && token >= 0 && (mask >> token & 1)) {
        float gate = 0.f, up = 0.f;
#pragma unroll
        for (int k = 0; k < kUpSlices; ++k) {
          const float* from = red + (k * 2 * NT + column) * kUpRows + lane;
          gate += from[0];
          up += from[NT * kUpRows];
        }
        gate *= x_f[column];
        up *= x_f[column];
        const bool chosen = lane < p.top_k && r.id[token][lane] == e;
        const int j = __ffs(__ballot_sync(0xffffffffu, chosen)) - 1;
        const float h = r.weight[token][j] * (gate / (1.f + expf(-gate)) * up);
        const uint32_t f = storage_exponent(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(h)))));
        const bool is_odd = lane & 1;  // pair (lane & 3) of its word
        const __half v = __float2half_rn(h * reciprocal_of(is_odd ? f + 4u : f));
        const float even = warp_sum(is_odd ? 0.f : __half2float(v)), odd = warp_sum(is_odd ? __half2float(v) : 0.f);
        const int rank = __popc(mask & ((1u << token) - 1u)), side = rank & 1;
        const int padded = (tiles + 3) / 4 * 4;
        uint8_t* rec = p.h + ((int64_t)(r.units.slot[u] + rank / 2) * padded + i0 / 32) * kRecord;
        reinterpret_cast<__half*>(rec)[side * 32 + (lane & 24) + (lane & 3) * 2 + ((lane >> 2) & 1)] = v;
        if (lane == 0) {
          float* to = reinterpret_cast<float*>(rec + 128) + side;
          put_sides(to, to + 6, even, odd, p.down.zp != nullptr);
          to[4] = power_of(f);
        }
        if (i0 / 32 == tiles - 1)  // zeros behind the last block, up to a whole step
          for (int i = tiles; i < padded; ++i) {
            rec += kRecord;
            reinterpret_cast<__half*>(rec)[side * 32 + lane] = __ushort_as_half(0);
            if (lane < 4) reinterpret_cast<float*>(rec + 128)[side + lane * 2] = 0.f;
          }
      }
    }
  }
  if (!ok) {
    atomicExch(&g_moe_status, 1);
    const uint64_t t0 = sm100::global_timer_ns();  // let copies that were issued land
    while (sm100::global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
}

// ---- kernel 2: down product and the sum over experts ----------------------------------------------
// A CTA has 512 / slices rows of the output, 32 to each of 16 / slices warps side by side, and takes a share of the
// (unit, round) pairs of its cluster.
// Shared memory of kernel 2 behind the lists: the ring (codes [slice][rows][64], then windows [scales, zero points]
// [rows][window], then h records [NT / 2][4 * slices], pairs in different banks), the sums [T][rows], the
// partial products of two units [slice][NT][rows], zeros that cover the reach of a step's operands, barriers.
struct DownLayout {
  int rows, windows, window_stage, h, h_pair, h_stage, sums, red, red_unit, zeros, bars, bytes;
  __host__ __device__ DownLayout(int T, int nt, bool asym, int window, int slices, int stages) {
    rows = 512 / slices;
    windows = stages * 512 * 64;
    window_stage = (asym ? 2 : 1) * rows * window;
    h = windows + stages * window_stage;
    h_pair = 4 * slices * kRecord + 32;
    h_stage = nt / 2 * h_pair;
    sums = h + stages * h_stage;
    red = sums + T * rows * 4;
    red_unit = 512 * nt * 4;
    zeros = red + 2 * red_unit;
    bars = zeros + 4 * kRecord;
    bytes = bars + 2 * kMaxStages * 8 + 1024;
  }
};

struct DownMaps {
  CUtensorMap codes, scale, zero;
};

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

template <int G, bool ASYM, int MODE>
__global__ void __launch_bounds__(threads_of(MODE), 1)
moe_down_kernel(const __grid_constant__ DownMaps maps, const MoeParams p) {
  constexpr int NT = 8 / G, kThreads = threads_of(MODE);
  extern __shared__ uint8_t dyn_raw[];
  uint8_t* dyn = dyn_raw + ((1024u - (sm100::smem_u32(dyn_raw) & 1023u)) & 1023u);
  __shared__ Units lists;
  __shared__ int abort_flag;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int n_blk = p.I / 32, n_steps = (n_blk + 3) / 4, n_group = n_blk / p.down.group_blocks;
  const int rounds = (n_steps + p.slices - 1) / p.slices;
  const int rank = p.split > 1 ? (int)sm100::cluster_ctarank() : 0;
  const DownLayout at(p.T, NT, ASYM, p.window, p.slices, p.stages);
  const int rows = at.rows, j0 = blockIdx.x / p.split * rows, rows_left = min(rows, p.H - j0);
  float* sums = reinterpret_cast<float*>(dyn + at.sums);
  uint64_t* full = reinterpret_cast<uint64_t*>(dyn + at.bars);
  uint64_t* empty = full + kMaxStages;
  for (int i = tid; i < p.T * rows; i += kThreads) sums[i] = 0.f;
  for (int i = tid; i < kRecord; i += kThreads) reinterpret_cast<uint32_t*>(dyn + at.zeros)[i] = 0;
  if (tid == 0) {
    abort_flag = 0;
    for (int i = 0; i < p.stages; ++i) {
      sm100::mbar_init(&full[i], MODE == kAny ? producers(MODE) * 32 + 1 : 1);
      sm100::mbar_init(&empty[i], kConsumers);
    }
    sm100::fence_barrier_init();
  }
  const int n_units = __ldcg(&p.units->n);
  for (int i = tid; i < n_units; i += kThreads) {
    lists.mask[i] = __ldcg(&p.units->mask[i]);
    lists.expert[i] = __ldcg(&p.units->expert[i]);
    lists.slot[i] = __ldcg(&p.units->slot[i]);
  }
  __syncthreads();

  const int64_t total = (int64_t)n_units * rounds;
  const int first = (int)(total * rank / p.split), last = (int)(total * (rank + 1) / p.split);
  const int first_u = first / rounds;
  int u = first_u, round = first - first_u * rounds;  // of the pair at hand
  int stage = 0;
  uint32_t parity = 0;
  auto advance = [&] {
    if (++round == rounds) {
      round = 0;
      ++u;
    }
    if (++stage == p.stages) {
      stage = 0;
      parity ^= 1;
    }
  };
  bool ok = true;

  if (warp >= kConsumers) {
    // ---- producers ----
    const int thread = tid - kConsumers * 32;
    const uint32_t base = sm100::smem_u32(dyn);
    const int64_t total_groups = (int64_t)p.E * p.H * n_group;
    for (int q = first; q < last; ++q, advance()) {
      ok = stage_is_free(&empty[stage], parity ^ 1, &abort_flag, p.wait_ns);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      const int row = lists.expert[u] * p.H + j0, s0 = round * p.slices, n = min(p.slices, n_steps - s0);
      const int start = window_start<MODE>(p.down, s0 * 4), pairs = (__popc(lists.mask[u]) + 1) / 2;
      const int windows = at.windows + stage * at.window_stage, part = rows * p.window;
      const uint32_t h_bytes = n * 4 * kRecord;
      if (warp == kConsumers && sm100::elect_one()) {
        sm100::mbar_arrive_expect_tx(&full[stage], n * rows * 64 + pairs * h_bytes + (MODE == kAny ? 0 : at.window_stage));
        for (int i = 0; i < n; ++i)
          sm100::tma_load_2d(dyn + stage * 512 * 64 + i * rows * 64, &maps.codes, &full[stage], (s0 + i) * 64, row);
        if (MODE != kAny) {
          sm100::tma_load_2d(dyn + windows, &maps.scale, &full[stage], start, row);
          if (ASYM) sm100::tma_load_2d(dyn + windows + part, &maps.zero, &full[stage], start, row);
        }
        for (int i = 0; i < pairs; ++i)
          bulk_load(base + at.h + stage * at.h_stage + i * at.h_pair,
                    p.h + ((int64_t)(lists.slot[u] + i) * (n_steps * 4) + s0 * 4) * kRecord, h_bytes, &full[stage]);
      }
      if (MODE == kAny) {
        const int64_t group = (int64_t)row * n_group + start;
        copy_windows(base + windows, p.down.scale, rows, p.window, group, n_group, total_groups, thread);
        if (ASYM) copy_windows(base + windows + part, p.down.zp, rows, p.window, group, n_group, total_groups, thread);
        cp_async_arrive(&full[stage]);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    // ---- consumers ----
    const int ks = warp % p.slices, r0 = warp / p.slices * 32;  // slice of a round, rows of the CTA's
    const int lane_blk = t / (4 / G);
    const bool diag = g / NT == lane_blk;
    const uint8_t* operand = dyn + (diag ? at.h + g % NT / 2 * at.h_pair + (ks * 4 + lane_blk) * kRecord + (g & 1) * 64 +
                                               t % (4 / G) * G * 16
                                         : at.zeros);
    const int operand_stage = diag ? at.h_stage : 0;
    const uint8_t* sides = dyn + at.h + t % (4 / G) * at.h_pair + (ks * 4 + lane_blk) * kRecord + 128;
    float acc[2][4] = {};
    for (int q = first; q < last; ++q, advance()) {
      const int s = round * p.slices + ks;
      ok = sm100::mbar_wait_bounded(&full[stage], parity, &abort_flag, p.wait_ns) && ok;
      if (s < n_steps) {
        const int start = window_start<MODE>(p.down, round * p.slices * 4);
        const int place = MODE == kAny ? (row_of<G>(g) * n_group + start) & 7 : 0;
        const StepAt here{dyn + stage * 512 * 64 + (ks * rows + r0) * 64,
                          dyn + at.windows + stage * at.window_stage + r0 * p.window, p.window, 16 * p.window,
                          rows * p.window};
        const uint8_t* side = sides + stage * at.h_stage;
        add_step<G, ASYM, MODE, true, 1024, kRecord, kRecord, kRecord>(
            acc, here, start, place, operand + stage * operand_stage, Sides{side, side + 16, side + 24}, g, t, s, n_blk,
            p.down);
      }
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&empty[stage]);
      if (round == rounds - 1 || q == last - 1) {
        // the unit (or this CTA's share of it) is done: its slices of k, and its tokens into the sums
        float* red = reinterpret_cast<float*>(dyn + at.red + (u & 1) * at.red_unit);
        float* part = red + ks * NT * rows + r0;
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const float v = block_sum<G>(acc[w][2 * h + c]);
              if (t < 4 / G) part[(2 * t + c) * rows + w * 16 + h * 8 + row_of<G>(g)] = v;
              acc[w][2 * h + c] = 0.f;
            }
        consumer_barrier();
        const uint32_t mask = lists.mask[u];
        const int n = __popc(mask);
        const int row = tid & (rows - 1), step = kConsumers * 32 / rows;  // rows: a power of two
        uint32_t m = mask;
        for (int c = tid / rows, at_c = 0; c < n; c += step) {
          for (; at_c < c; ++at_c) m &= m - 1;
          float v = 0.f;
#pragma unroll 4
          for (int k = 0; k < p.slices; ++k) v += red[(k * NT + c) * rows + row];
          sums[(__ffs(m) - 1) * rows + row] += v;
        }
      }
    }
  }
  if (!ok) {
    atomicExch(&g_moe_status, 2);
    const uint64_t t0 = sm100::global_timer_ns();
    while (sm100::global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  __syncthreads();
  // the CTAs of the cluster: each finishes an equal share of the rows
  if (p.split > 1) {
    __syncwarp();
    sm100::cluster_sync_all();
  }
  const int each = rows / p.split;
  for (int i = tid; i < p.T * each; i += kThreads) {
    const int token = i / each, row = rank * each + i % each;
    float v = 0.f;
    if (p.split > 1) {
      for (int c = 0; c < p.split; ++c)
        v += ld_cluster_f32(sm100::map_to_cta(sm100::smem_u32(sums) + (token * rows + row) * 4, c));
    } else {
      v = sums[token * rows + row];
    }
    if (row >= rows_left) continue;
    const int64_t to = (int64_t)token * p.H + j0 + row;
    if (p.dtype == NPB_BF16) static_cast<__nv_bfloat16*>(p.y)[to] = from_f32<__nv_bfloat16>(v);
    else static_cast<__half*>(p.y)[to] = from_f32<__half>(v);
  }
  if (p.split > 1) {
    __syncwarp();
    sm100::cluster_sync_all();  // nobody leaves while its sums are read
  }
}

// ---- host ----------------------------------------------------------------------------------------
int mode_of(const MoeWeight& w, int n_blk) {
  if (w.group_shift < 0 || (n_blk / w.group_blocks) % 8 != 0) return kAny;
  return w.group_blocks == 1 ? kOnePerBlock : kPowerOfTwo;
}

// Bytes of a row's groups in a round of `slices` steps.
int window_bytes(const MoeWeight& w, int n_blk, int slices) {
  const int blocks = 4 * slices, gb = w.group_blocks;
  switch (mode_of(w, n_blk)) {
    case kOnePerBlock: return blocks * 2;
    case kPowerOfTwo: return blocks * 2 / gb > 16 ? blocks * 2 / gb : 16;
    default:  // the groups that `blocks` blocks touch, behind up to seven others
      return (((blocks - 1 + gb - 1) / gb + 1 + 7) * 2 + 15) / 16 * 16;
  }
}

// Codes [rows, bytes of a row] in boxes of 64 bytes x box_rows, and groups [rows, n_group] in boxes of a window.
int make_code_map(CUtensorMap* map, const uint8_t* codes, int64_t rows, int64_t row_bytes, int box_rows) {
  return make_tensor_map_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, codes, rows, row_bytes, box_rows, 64,
                            CU_TENSOR_MAP_SWIZZLE_64B);
}
int make_group_map(CUtensorMap* map, const __half* groups, int64_t rows, int64_t n_group, int box_rows, int window) {
  return make_tensor_map_2d(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, groups, rows, n_group, box_rows, window / 2,
                            window == 64   ? CU_TENSOR_MAP_SWIZZLE_64B
                            : window == 32 ? CU_TENSOR_MAP_SWIZZLE_32B
                                           : CU_TENSOR_MAP_SWIZZLE_NONE);
}

// Ring stages that fit next to the rest (2..4; 0: not even two do).
template <typename Bytes>
int pick_stages(Bytes bytes, int static_bytes) {
  int stages = kMaxStages;
  while (stages >= 2 && bytes(stages) + static_bytes > max_dynamic_smem()) --stages;
  return stages >= 2 ? stages : 0;
}

// Fills in the ring of a kernel; false: it does not fit.
bool plan_up(MoeParams& p, int g) {
  p.window = window_bytes(p.gate, p.H / 32, kUpSlices);
  p.stages = pick_stages(
      [&](int n) { return UpLayout(p.H / 32, 8 / g, p.gate.zp != nullptr, p.window, n).bytes; }, (int)sizeof(Routing) + 128);
  return p.stages != 0;
}
bool plan_down(MoeParams& p, int g) {
  // 128 rows to a CTA and a cluster of up to four, as long as that makes a CTA for most SMs; fewer rows otherwise
  p.slices = p.H >= 4096 ? 4 : p.H >= 2048 ? 8 : 16;
  const int rows = 512 / p.slices, tiles = (p.H + rows - 1) / rows;
  p.split = 1;
  while (p.split < 4 && tiles * p.split * 2 <= sm_count()) p.split *= 2;
  p.window = window_bytes(p.down, p.I / 32, p.slices);
  p.stages = pick_stages(
      [&](int n) { return DownLayout(p.T, 8 / g, p.down.zp != nullptr, p.window, p.slices, n).bytes; },
      (int)sizeof(Units) + 512);
  return p.stages != 0;
}

template <int G, bool ASYM, int MODE>
int launch_up(MoeParams p, cudaStream_t st) {
  auto kern = moe_up_kernel<G, ASYM, MODE>;
  if (!plan_up(p, G)) return NPB_ERR_TOO_LARGE;
  const int n_blk = p.H / 32, smem = UpLayout(n_blk, 8 / G, ASYM, p.window, p.stages).bytes;
  int per_sm = 0;
  if (int rc = blocks_per_sm(reinterpret_cast<const void*>(kern), threads_of(MODE), smem, &per_sm)) return rc;
  if (per_sm < 1) return NPB_ERR_TOO_LARGE;
  UpMaps maps{};
  const int64_t rows = (int64_t)p.E * p.I, n_group = n_blk / p.gate.group_blocks;
  const MoeWeight* w[2] = {&p.gate, &p.up};
  for (int i = 0; i < 2; ++i) {
    if (int rc = make_code_map(&maps.codes[i], w[i]->codes, rows, p.H / 2, kUpRows)) return rc;
    if (MODE == kAny) continue;
    if (int rc = make_group_map(&maps.scale[i], w[i]->scale, rows, n_group, kUpRows, p.window)) return rc;
    if (!ASYM) continue;
    if (int rc = make_group_map(&maps.zero[i], w[i]->zp, rows, n_group, kUpRows, p.window)) return rc;
  }
  const int64_t active = p.T * p.top_k < p.E ? p.T * p.top_k : p.E;
  const int64_t most = active * (p.I / kUpRows), slots = (int64_t)sm_count() * per_sm;
  kern<<<(unsigned)(most < slots ? most : slots), threads_of(MODE), smem, st>>>(maps, p);
  NPB_LAUNCH_CHECK();
  return NPB_OK;
}

template <int G, bool ASYM, int MODE>
int launch_down(MoeParams p, cudaStream_t st) {
  auto kern = moe_down_kernel<G, ASYM, MODE>;
  if (!plan_down(p, G)) return NPB_ERR_TOO_LARGE;
  const DownLayout at(p.T, 8 / G, ASYM, p.window, p.slices, p.stages);
  int per_sm = 0;
  if (int rc = blocks_per_sm(reinterpret_cast<const void*>(kern), threads_of(MODE), at.bytes, &per_sm)) return rc;
  if (per_sm < 1) return NPB_ERR_TOO_LARGE;
  DownMaps maps{};
  const int64_t rows = (int64_t)p.E * p.H, n_group = p.I / 32 / p.down.group_blocks;
  if (int rc = make_code_map(&maps.codes, p.down.codes, rows, p.I / 2, at.rows)) return rc;
  if (MODE != kAny) {
    if (int rc = make_group_map(&maps.scale, p.down.scale, rows, n_group, at.rows, p.window)) return rc;
    if (ASYM)
      if (int rc = make_group_map(&maps.zero, p.down.zp, rows, n_group, at.rows, p.window)) return rc;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((p.H + at.rows - 1) / at.rows * p.split));
  cfg.blockDim = dim3(threads_of(MODE));
  cfg.dynamicSmemBytes = at.bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = p.split;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  NPB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, maps, p));
  NPB_LAUNCH_CHECK();
  return NPB_OK;
}

template <int G, bool ASYM>
int launch_up_mode(const MoeParams& p, cudaStream_t st) {
  switch (mode_of(p.gate, p.H / 32)) {
    case kOnePerBlock: return launch_up<G, ASYM, kOnePerBlock>(p, st);
    case kPowerOfTwo: return launch_up<G, ASYM, kPowerOfTwo>(p, st);
    default: return launch_up<G, ASYM, kAny>(p, st);
  }
}
template <int G, bool ASYM>
int launch_down_mode(const MoeParams& p, cudaStream_t st) {
  switch (mode_of(p.down, p.I / 32)) {
    case kOnePerBlock: return launch_down<G, ASYM, kOnePerBlock>(p, st);
    case kPowerOfTwo: return launch_down<G, ASYM, kPowerOfTwo>(p, st);
    default: return launch_down<G, ASYM, kAny>(p, st);
  }
}
template <int G>
int launch(const MoeParams& p, cudaStream_t st) {
  if (int rc = p.gate.zp ? launch_up_mode<G, true>(p, st) : launch_up_mode<G, false>(p, st)) return rc;
  return p.down.zp ? launch_down_mode<G, true>(p, st) : launch_down_mode<G, false>(p, st);
}

int launch_tokens(const MoeParams& p, cudaStream_t st) {
  // an expert has at most T tokens; both kernels need two stages next to a unit's tokens
  auto fits = [&](int g) {
    MoeParams q = p;
    return plan_up(q, g) && plan_down(q, g);
  };
  if (p.T > 4 && fits(1)) return launch<1>(p, st);
  if (p.T > 2 && fits(2)) return launch<2>(p, st);
  return fits(4) ? launch<4>(p, st) : NPB_ERR_TOO_LARGE;
}

int make_weight(const npb_q_weight* w, int64_t N, int64_t K, MoeWeight* out) {
  if (int rc = validate_q(w, N, K)) return rc;
  if (w->nbits != 4 || w->group_size % 32 != 0) return NPB_ERR_UNSUPPORTED;
  if (!aligned_to(w->codes, 16) || !aligned_to(w->scale, 16) || !aligned_to(w->zero_point, 16)) return NPB_ERR_ALIGNMENT;
  out->codes = w->codes;
  out->scale = static_cast<const __half*>(w->scale);
  out->zp = static_cast<const __half*>(w->zero_point);
  out->group_blocks = w->group_size / 32;
  out->group_shift = -1;
  for (int s = 0; s < 16; ++s)
    if (out->group_blocks == 1 << s) out->group_shift = s;
  return NPB_OK;
}

}  // namespace

// Reads and clears the give-up record (npb_gemm_device_status collects it).
int q_moe_device_status(int* host_out) {
  NPB_CUDA_TRY(cudaMemcpyFromSymbol(host_out, g_moe_status, sizeof(int)));
  if (*host_out != 0) {
    const int zero = 0;
    NPB_CUDA_TRY(cudaMemcpyToSymbol(g_moe_status, &zero, sizeof(int)));
  }
  return NPB_OK;
}

int64_t q_moe_workspace_bytes(int64_t T, int top_k, int64_t I) {
  if (T < 0 || top_k <= 0 || I <= 0 || T > kMaxTokens || top_k > kMaxTopK || I % 32 != 0) return 0;
  // a pair of tokens of an expert is at least one of the T * top_k
  return (int64_t)sizeof(Units) + T * top_k * ((I / 32 + 3) / 4 * 4) * kRecord;
}

int q_moe(const void* x, int dtype, const void* logits, int logits_dtype, int64_t T, int64_t E, int64_t H, int64_t I,
          const npb_q_weight* gate, const npb_q_weight* up, const npb_q_weight* down, int top_k, int renormalize,
          void* workspace, int64_t workspace_bytes, void* y, cudaStream_t st) {
  if (T < 0 || E <= 0 || H <= 0 || I <= 0 || top_k <= 0 || top_k > E) return NPB_ERR_INVALID_ARG;
  if (gate == nullptr || up == nullptr || down == nullptr) return NPB_ERR_INVALID_ARG;
  if (dtype != NPB_BF16 && dtype != NPB_F16) return NPB_ERR_UNSUPPORTED;
  if (logits_dtype != NPB_BF16 && logits_dtype != NPB_F16 && logits_dtype != NPB_F32) return NPB_ERR_UNSUPPORTED;
  if (T > kMaxTokens || E > kMaxExperts || top_k > kMaxTopK || H > kMaxWidth || I > kMaxWidth) return NPB_ERR_UNSUPPORTED;
  if (H % 32 != 0 || I % 32 != 0) return NPB_ERR_SHAPE;
  MoeParams p{};
  if (int rc = make_weight(gate, E * I, H, &p.gate)) return rc;
  if (int rc = make_weight(up, E * I, H, &p.up)) return rc;
  if (int rc = make_weight(down, E * H, I, &p.down)) return rc;
  if ((p.gate.zp == nullptr) != (p.up.zp == nullptr) || gate->group_size != up->group_size) return NPB_ERR_UNSUPPORTED;
  if (T == 0) return NPB_OK;
  if (x == nullptr || logits == nullptr || y == nullptr || workspace == nullptr) return NPB_ERR_INVALID_ARG;
  if (workspace_bytes < q_moe_workspace_bytes(T, top_k, I)) return NPB_ERR_TOO_LARGE;
  const size_t logit_size = logits_dtype == NPB_F32 ? 4 : 2;
  if (!aligned_to(x, 16) || !aligned_to(workspace, 16) || !aligned_to(y, 2) || !aligned_to(logits, logit_size))
    return NPB_ERR_ALIGNMENT;
  p.x = x;
  p.logits = logits;
  p.logits_dtype = logits_dtype;
  p.dtype = dtype;
  p.T = (int)T; p.E = (int)E; p.H = (int)H; p.I = (int)I;
  p.top_k = top_k;
  p.renormalize = renormalize != 0;
  p.units = static_cast<Units*>(workspace);
  p.h = static_cast<uint8_t*>(workspace) + sizeof(Units);
  p.y = y;
  p.wait_ns = wait_limit_ns();
  return launch_tokens(p, st);
}

}  // namespace npb
