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
// is applied per 32-wide block, with the weight's scale, in fp32.  Activations are stored as fp16 after division by a power of two, one per token for x and one per
// 32-block and token for h, so their size does not matter: x loses nothing down to 2^-13 (bf16) or 2^-10
// (fp16) of the token's largest and at most 2^-21 of the largest below that; h keeps 11 significant bits
// between the kernels, 1/8 of a bf16 half step.
//
// The eight columns of an mma are NT = 8 / G tokens times G neighbouring 32-blocks (G = 4, 2, 1): lane (g, t)
// of a warp loads G words, the t-th part of G blocks, of rows g and g + 8, so the k slots of an mma hold
// G different blocks, and the B operand keeps them apart by being block-diagonal.  Lane (g, t) of the result
// then holds two tokens of exactly the block whose scale it loaded.  A step of four blocks takes the same
// sixteen mmas for two 16-row tiles whatever G is (8 cycles of a scheduler's tensor pipe each, measured);
// G = 4 has the widest loads and the fewest results to scale, G = 1 the most tokens per weight read.
//
// Every warp streams its own weights through a ring of steps in shared memory: codes as TMA boxes of 64 bytes x 16
// rows with the 64-byte swizzle (no bank conflicts when read, no load instructions, nothing in the L1 path),
// scales and zero points by cp.async as 16- or 32-byte windows that serve several steps.  What is in flight
// does not depend on registers: register double buffers of the same kernels reached a third of the bandwidth
// (waiting for one step's loads waits for the next step's too), and cp.async for the codes left the L1 path
// 72 % busy.  Kernel 1 keeps the tokens of its unit (up to NT tokens of one expert) in shared memory in the
// order of the mma operands and writes h in that order; kernel 2 brings h along with the weights.  An expert
// with more tokens than a unit is read again (from L2).  Every sum has a fixed order: results do not depend
// on scheduling.  Waits on the TMA barriers are bounded like those of the GEMMs.
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
  int window;        // steps that a window of groups serves
};

struct MoeParams {
  const void* x;
  const void* logits;
  int logits_dtype, dtype;
  int T, E, H, I, top_k, renormalize;
  MoeWeight gate, up, down;
  uint8_t* h;      // [pair of tokens of a unit][I / 32] records
  Units* units;
  void* y;
  uint64_t wait_ns;
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
  uint32_t mask[kMaxExperts];            // tokens of each expert
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
__device__ void choose(const MoeParams& p, Routing& r) {
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
      if (!none) atomicOr(&r.mask[mine_e], 1u << t);
    }
  }
}

// All threads of the CTA; ends with a barrier.  A unit is up to NT tokens of one expert.
template <int NT>
__device__ void route(const MoeParams& p, Routing& r) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) r.mask[e] = 0;
  __syncthreads();
  if (p.E <= 64) choose<2>(p, r);
  else if (p.E <= 128) choose<4>(p, r);
  else choose<kMaxExperts / 32>(p, r);
  __syncthreads();
  if (warp == 0) {
    int units = 0, slots = 0;
    for (int base = 0; base < p.E; base += 32) {
      const int e = base + lane;
      const int n = e < p.E ? __popc(r.mask[e]) : 0;
      const int u = (n + NT - 1) / NT, pairs = (n + 1) / 2;
      int iu = u, in = pairs;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, iu, o), b = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) { iu += a; in += b; }
      }
      uint32_t m = n > 0 ? r.mask[e] : 0u;
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
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits until at most `pending` (1..3) of the committed groups are under way.
__device__ __forceinline__ void cp_async_wait(int pending) {
  if (pending == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else if (pending == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else asm volatile("cp.async.wait_group 3;" ::: "memory");
}

// A warp's ring over R 16-row tiles.  A stage holds one step (four 32-blocks of k): per row 64 bytes of codes as TMA's
// 64-byte swizzle leaves them (16-byte piece c of row r at c ^ (r / 2 mod 4)).  A window holds per row the 16 or 32
// bytes, from a 16-byte boundary on, with the groups of several steps; there are as many windows as stages: the
// steps in the ring need no more.  MODE: kOnePerBlock (a group is a block; a step's four values are eight aligned
// bytes) and kPowerOfTwo (a group is 2^n blocks) take rows of whole 16-byte windows, one for every eight groups;
// kAny the rest, 32 bytes at a run's first step and every `window`-th after it.
enum { kAny = 0, kOnePerBlock = 1, kPowerOfTwo = 2 };

template <int G, int R, bool ASYM, int MODE>
struct Ring {
  static constexpr int kRows = 16 * R, kWindowRow = MODE == kAny ? 32 : 16;
  static constexpr int kCodes = kRows * 64;
  static constexpr int kWindow = kRows * kWindowRow * (ASYM ? 2 : 1);
  static constexpr int kZeros = kRows * kWindowRow;  // of the zero points in a window

  // Tile row of lane group g: G = 2 reads half pieces, which needs every other pair of rows in a phase.
  __device__ static int row_of(int g) { return G == 2 ? (g & 1) | (g & 2) << 1 | (g & 4) >> 1 : g; }

  // The step after s (which brings a window) that brings the next one in its run.
  __device__ static int next_window(const MoeWeight& w, int s) {
    if (MODE == kOnePerBlock) return (s | 1) + 1;
    if (MODE == kPowerOfTwo) return (s | ((2 << w.group_shift) - 1)) + 1;
    return s + w.window;
  }
  // Place of step s's first group in the window that step w_s brought, for rows that are row_of(g) modulo 8.
  __device__ static int index_of(const MoeWeight& w, int s, int w_s, int g, int n_group) {
    if (MODE == kOnePerBlock) return (s & 1) * 4;
    if (MODE == kPowerOfTwo) return (s * 4 >> w.group_shift) & 7;
    const int g0 = group_of(w, w_s * 4);
    return ((row_of(g) * n_group + g0) & 7) + group_of(w, s * 4) - g0;
  }

  // Windows of rows row0 + lane / PIECES ..: `at` is the first group of ring row 0's step, counted in the matrix of
  // `total` groups; rows are n_group apart.
  template <int ROWS>
  __device__ static void fetch_window(uint32_t window, int row0, const MoeWeight& w, int64_t at, int n_group,
                                      int64_t total, int lane) {
    constexpr int PIECES = kWindowRow / 16;
#pragma unroll
    for (int i = 0; i < (ROWS * PIECES + 31) / 32; ++i) {
      const int row = i * (32 / PIECES) + lane / PIECES, piece = lane % PIECES;
      if (row >= ROWS) break;
      const int64_t first = ((at + row * n_group) & ~7ll) + piece * 8;
      const int bytes = first + 8 <= total ? 16 : first < total ? (int)(total - first) * 2 : 0;
      const uint32_t dst = window + (row0 + row) * kWindowRow + piece * 16;
      const int64_t from = bytes ? first : 0;
      cp_async16(dst, w.scale + from, bytes);
      if (ASYM) cp_async16(dst + kZeros, w.zp + from, bytes);
    }
  }
};

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
// The power of two at or below a magnitude (1 for zero, subnormal, inf, NaN).
__device__ __forceinline__ float power_below(float top) {
  const uint32_t exponent = __float_as_uint(top) >> 23;
  return exponent == 0 || exponent == 255 ? 1.f : __uint_as_float(exponent << 23);
}

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

// Adds one step to acc[tile] (rows row_of(g) and + 8 of two tokens, as the mma has them).  `codes` and `window` are the ring's; `index` the place
// of the step's first group in this lane's row of the window; `operand` this lane's part of the first set in B
// order, BLOCK bytes from block to block (a lane off the diagonal: zeros); `sides` belong to its two tokens and its
// block of the first set, MS and FS bytes from block to block.
template <int G, int R, bool ASYM, int MODE, bool SCALED, int BLOCK, int MS, int FS>
__device__ __forceinline__ void add_step(float (&acc)[R][4], const uint8_t* codes, const uint8_t* window, int index,
                                         const uint8_t* operand, const Sides& sides, int g, int t, int s, int n_blk,
                                         const MoeWeight& w) {
  using Rg = Ring<G, R, ASYM, MODE>;
  const int r0 = Rg::row_of(g);
  const uint8_t* at = window + r0 * Rg::kWindowRow + index * 2;
  uint2 sc[R][2], zp[ASYM ? R : 1][2];
  if constexpr (MODE == kOnePerBlock) {
#pragma unroll
    for (int i = 0; i < 2 * R; ++i) {
      sc[i / 2][i % 2] = *reinterpret_cast<const uint2*>(at + i * 8 * Rg::kWindowRow);
      if (ASYM) zp[ASYM ? i / 2 : 0][i % 2] = *reinterpret_cast<const uint2*>(at + i * 8 * Rg::kWindowRow + Rg::kZeros);
    }
  }
#pragma unroll
  for (int j = 0; j < 4 / G; ++j) {
    // its G words: 16-byte piece (block) of the row, word t mod 4 / G times G
    const int piece = ((j * G + t / (4 / G)) ^ (r0 >> 1 & 3)) * 16 + t % (4 / G) * (4 * G);
    uint32_t c[2 * R][G];
#pragma unroll
    for (int i = 0; i < 2 * R; ++i) {
      const uint8_t* from = codes + (i * 8 + r0) * 64 + piece;
      if constexpr (G == 4) *reinterpret_cast<uint4*>(c[i]) = *reinterpret_cast<const uint4*>(from);
      else if constexpr (G == 2) *reinterpret_cast<uint2*>(c[i]) = *reinterpret_cast<const uint2*>(from);
      else c[i][0] = *reinterpret_cast<const uint32_t*>(from);
    }
    const float4 m = *reinterpret_cast<const float4*>(sides.m + j * G * MS);
    float d[R][4];
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(operand + j * G * BLOCK + i * 16);
#pragma unroll
      for (int q = 0; q < R; ++q) {
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
    const int group = MODE == kOnePerBlock ? 0 : (group_of(w, own) - group_of(w, s * 4)) * 2;
#pragma unroll
    for (int q = 0; q < R; ++q)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float scale, z = 0.f;
        if constexpr (MODE == kOnePerBlock) {
          scale = group_value<G>(sc[q][h], j, t);
          if (ASYM) z = group_value<G>(zp[ASYM ? q : 0][h], j, t);
        } else {
          const uint8_t* from = at + (q * 16 + h * 8) * Rg::kWindowRow + group;
          scale = half_bits(*reinterpret_cast<const uint16_t*>(from));
          if (ASYM) z = half_bits(*reinterpret_cast<const uint16_t*>(from + Rg::kZeros));
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

// ---- kernel 1: gate / up products, silu, routing weight ------------------------------------------
constexpr int kUpThreads = 512;  // two 16-row tile pairs (gate, up) x eight slices of K
constexpr int kUpWarps = kUpThreads / 32;
constexpr int kUpRows = 32;      // rows of gate and of up per item: one 32-block of h
constexpr int kUpSlices = 8;
constexpr int kMaxStages = 4;    // of a ring

// Shared memory of kernel 1 behind the routing: the warps' rings (codes, windows), tokens [NT][4 * steps] blocks of
// 64 bytes (neighbouring rows in the other half of the banks), their m [NT / 2][blocks + 1] (pairs in different
// banks) and s2 [NT / 2][blocks], the partial
// products, 256 bytes of zeros, barriers.
struct UpLayout {
  int windows, x, row, m, s2, red, zeros, bars, bytes;
  __host__ __device__ UpLayout(int n_blk, int nt, bool asym, int code_bytes, int window_bytes, int stages) {
    const int blocks = (n_blk + 3) / 4 * 4;
    windows = kUpWarps * stages * code_bytes;
    x = windows + kUpWarps * stages * window_bytes;
    row = blocks * 64 + 64;
    m = x + row * nt;
    s2 = m + nt / 2 * (blocks + 1) * 16;
    red = s2 + (asym ? nt / 2 * blocks * 8 : 0);
    zeros = red + kUpSlices * 2 * kUpRows * nt * 4;
    bars = zeros + 256;
    bytes = bars + kUpWarps * kMaxStages * 8 + 1024;  // + alignment of the start
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
  CUtensorMap gate, up;
};

template <int G, bool ASYM, int MODE>
__global__ void __launch_bounds__(kUpThreads, 1)
moe_up_kernel(const __grid_constant__ UpMaps maps, const MoeParams p, const int stages) {
  constexpr int NT = 8 / G;
  using Rg = Ring<G, 2, ASYM, MODE>;
  extern __shared__ uint8_t dyn_raw[];
  uint8_t* dyn = dyn_raw + ((1024u - (sm100::smem_u32(dyn_raw) & 1023u)) & 1023u);
  __shared__ Routing r;
  __shared__ uint32_t x_top[NT];     // bits of the largest magnitude of each token
  __shared__ float x_f[NT];
  __shared__ int abort_flag;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int n_blk = p.H / 32, n_steps = (n_blk + 3) / 4, blocks = n_steps * 4;
  const int n_group = n_blk / p.gate.group_blocks;
  const UpLayout at(n_blk, NT, ASYM, Rg::kCodes, Rg::kWindow, stages);
  float* red = reinterpret_cast<float*>(dyn + at.red);  // [slice][gate, up][NT][32]
  uint64_t* bars = reinterpret_cast<uint64_t*>(dyn + at.bars) + warp * kMaxStages;
  const uint32_t base = sm100::smem_u32(dyn);
  if (tid < 64) reinterpret_cast<uint32_t*>(dyn + at.zeros)[tid] = 0;
  if (tid == 0) {
    abort_flag = 0;
    sm100::tma_prefetch_desc(&maps.gate);
    sm100::tma_prefetch_desc(&maps.up);
  }
  if (lane == 0) {
    for (int i = 0; i < stages; ++i) sm100::mbar_init(&bars[i], 1);
    sm100::fence_barrier_init();
  }
  route<NT>(p, r);

  if (blockIdx.x == 0) {  // for kernel 2
    if (tid == 0) p.units->n = r.units.n;
    for (int i = tid; i < r.units.n; i += kUpThreads) {
      p.units->mask[i] = r.units.mask[i];
      p.units->expert[i] = r.units.expert[i];
      p.units->slot[i] = r.units.slot[i];
    }
  }
  const int tiles = p.I / kUpRows;
  const int64_t items = (int64_t)tiles * r.units.n;
  const int first = (int)(items * blockIdx.x / gridDim.x), last = (int)(items * (blockIdx.x + 1) / gridDim.x);
  const int mt = warp & 1, ks = warp >> 1;
  const int s_first = n_steps * ks / kUpSlices, s_last = n_steps * (ks + 1) / kUpSlices;
  const int lane_blk = t / (4 / G);      // this lane's block of a set
  const bool diag = g / NT == lane_blk;  // it holds the nonzero part of column g
  const uint8_t* operand = dyn + (diag ? at.x + (g % NT) * at.row + lane_blk * 64 + t % (4 / G) * G * 16 : at.zeros);
  const int operand_step = diag ? 256 : 0;
  const int pair = t % (4 / G);
  const Sides sides{dyn + at.m + (pair * (blocks + 1) + lane_blk) * 16, nullptr,
                    dyn + at.s2 + (pair * blocks + lane_blk) * 8};

  // the warp's ring runs through its steps of all items
  const int code_ring = warp * stages * Rg::kCodes, window_ring = at.windows + warp * stages * Rg::kWindow;
  const int64_t total_groups = (int64_t)p.E * p.I * n_group;
  int f_item = s_first < s_last ? first : last, f_s = s_first, f_stage = 0, f_window = 0, f_row = 0, f_next = s_first;
  auto f_start = [&] {
    if (f_item < last) {
      const int u = f_item / tiles;
      f_row = r.units.expert[u] * p.I + (f_item - u * tiles) * kUpRows + mt * 16;
    }
  };
  f_start();
  auto fetch = [&] {
    if (f_item < last) {
      if (lane == 0) {
        uint8_t* to = dyn + code_ring + f_stage * Rg::kCodes;
        sm100::mbar_arrive_expect_tx(&bars[f_stage], Rg::kCodes);
        sm100::tma_load_2d(to, &maps.gate, &bars[f_stage], f_s * 64, f_row);
        sm100::tma_load_2d(to + 1024, &maps.up, &bars[f_stage], f_s * 64, f_row);
      }
      if (f_s == f_next) {
        f_next = Rg::next_window(p.gate, f_s);
        const uint32_t to = base + window_ring + f_window * Rg::kWindow;
        if (++f_window == stages) f_window = 0;
        const int64_t group = (int64_t)f_row * n_group + group_of(p.gate, f_s * 4);
        Rg::template fetch_window<16>(to, 0, p.gate, group, n_group, total_groups, lane);
        Rg::template fetch_window<16>(to, 16, p.up, group, n_group, total_groups, lane);
      }
      if (++f_s == s_last) {
        f_s = f_next = s_first;
        ++f_item;
        f_start();
      }
      if (++f_stage == stages) f_stage = 0;
    }
    cp_async_commit();
  };
  for (int i = 0; i < stages; ++i) fetch();

  int unit = -1, n = 0, stage = 0, window = -1;  // of the step at hand
  uint32_t parity = 0;
  bool ok = true;
  for (int item = first; item < last; ++item) {
    const int u = item / tiles, i0 = (item - u * tiles) * kUpRows;
    const int e = r.units.expert[u];
    if (u != unit) {
      if (tid < NT) x_top[tid] = 0;
      __syncthreads();  // everybody is through with the unit before
      unit = u;
      const uint32_t mask = r.units.mask[u];
      n = __popc(mask);
      // the unit's tokens, eight elements of each to a thread (columns of an mma past the last token hold what was
      // there: nothing reads their sums): the largest magnitude of each, then the stored values.  Rows of up to 4096
      // stay in registers between the two.
      uint4 raw[NT] = {};
      auto load = [&](int j) {
        uint32_t m = mask;
#pragma unroll
        for (int i = 0; i < NT; ++i, m &= m - 1) {
          raw[i] = make_uint4(0, 0, 0, 0);
          if (i < n && j < n_blk * 4)
            raw[i] = __ldg(reinterpret_cast<const uint4*>(p.x) + (int64_t)(__ffs(m) - 1) * (n_blk * 4) + j);
        }
      };
      const bool bf16 = p.dtype == NPB_BF16, held = blocks * 4 <= kUpThreads;
      float top[NT] = {};
#pragma unroll 1
      for (int j = tid; j < blocks * 4; j += kUpThreads) {
        load(j);
#pragma unroll
        for (int i = 0; i < NT; ++i)
          top[i] = fmaxf(top[i], bf16 ? largest<__nv_bfloat16>(raw[i]) : largest<__half>(raw[i]));
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top[i]));
        if (lane == 0 && i < n) atomicMax(&x_top[i], bits);
      }
      __syncthreads();
      if (tid < n) x_f[tid] = power_below(__uint_as_float(x_top[tid]));
#pragma unroll 1
      for (int j0 = 0; j0 < blocks * 4; j0 += kUpThreads) {  // whole warps
        const int j = j0 + tid;
        if (!held) load(j);
#pragma unroll
        for (int i = 0; i < NT; ++i)
          if (i < n) {
            const float by = 1.f / power_below(__uint_as_float(x_top[i]));
            uint4* to = reinterpret_cast<uint4*>(dyn + at.x + i * at.row + j * 16);
            float* to_m = reinterpret_cast<float*>(dyn + at.m) + (i / 2 * (blocks + 1) + (j >> 2)) * 4 + (i & 1);
            float* to_s2 = ASYM ? reinterpret_cast<float*>(dyn + at.s2) + (i / 2 * blocks + (j >> 2)) * 2 + (i & 1) : nullptr;
            const bool write = j < blocks * 4;
            if (bf16) store_operand<__nv_bfloat16>(raw[i], by, to, to_m, to_s2, write, ASYM);
            else store_operand<__half>(raw[i], by, to, to_m, to_s2, write, ASYM);
          }
      }
      __syncthreads();
    }
    float acc[2][4] = {};
    int w_s = 0, w_next = s_first;
    for (int s = s_first; s < s_last; ++s) {
      ok = sm100::mbar_wait_bounded(&bars[stage], parity, &abort_flag, p.wait_ns) && ok;
      cp_async_wait(stages - 1);
      __syncwarp();
      if (s == w_next) {
        if (++window == stages) window = 0;
        w_s = s;
        w_next = Rg::next_window(p.gate, s);
      }
      const int index = Rg::index_of(p.gate, s, w_s, g, n_group);
      const Sides here{sides.m + s * 64, nullptr, sides.s2 + s * 32};
      add_step<G, 2, ASYM, MODE, false, 64, 16, 8>(acc, dyn + code_ring + stage * Rg::kCodes,
                                               dyn + window_ring + window * Rg::kWindow, index, operand + s * operand_step, here, g, t, s, n_blk, p.gate);
      __syncwarp();
      fetch();
      if (++stage == stages) { stage = 0; parity ^= 1; }
    }
    __syncthreads();  // the item before is read
    // the blocks of a set, then the slices of K
    float* part = red + ks * 2 * NT * kUpRows;
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float q = block_sum<G>(acc[w][2 * h + c]);
          if (t < 4 / G) part[(w * NT + 2 * t + c) * kUpRows + mt * 16 + Rg::row_of(g) + h * 8] = q;
        }
      }
    __syncthreads();
    if (warp < n) {  // a warp per token, a lane per row
      float gate = 0.f, up = 0.f;
#pragma unroll
      for (int k = 0; k < kUpSlices; ++k) {
        const float* from = red + (k * 2 * NT + warp) * kUpRows + lane;
        gate += from[0];
        up += from[NT * kUpRows];
      }
      gate *= x_f[warp];
      up *= x_f[warp];
      uint32_t m = r.units.mask[u];
      for (int i = 0; i < warp; ++i) m &= m - 1;
      const int token = __ffs(m) - 1;
      float weight = 0.f;
      for (int j = 0; j < p.top_k; ++j)
        if (r.id[token][j] == e) weight = r.weight[token][j];
      const float h = weight * (gate / (1.f + expf(-gate)) * up);
      float top = fabsf(h);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float f = power_below(top);
      const bool is_odd = lane & 1;  // pair (lane & 3) of its word
      const __half v = __float2half_rn(h * ((is_odd ? 0.0625f : 1.f) / f));
      const float even = warp_sum(is_odd ? 0.f : __half2float(v)), odd = warp_sum(is_odd ? __half2float(v) : 0.f);
      uint8_t* rec = p.h + ((int64_t)(r.units.slot[u] + warp / 2) * (p.I / 32) + i0 / 32) * kRecord;
      reinterpret_cast<__half*>(rec)[(warp & 1) * 32 + (lane & 24) + (lane & 3) * 2 + ((lane >> 2) & 1)] = v;
      if (lane == 0) {
        float* to = reinterpret_cast<float*>(rec + 128) + (warp & 1);
        put_sides(to, to + 6, even, odd, p.down.zp != nullptr);
        to[4] = f;
      }
    }
  }
  if (!ok) atomicExch(&g_moe_status, 1);
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (!ok) {  // let copies that were issued land before the shared memory is released
    const uint64_t t0 = sm100::global_timer_ns();
    while (sm100::global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
}

// ---- kernel 2: down product and the sum over experts ----------------------------------------------
constexpr int kDownThreads = 256;
constexpr int kDownWarps = kDownThreads / 32;
constexpr int kDownTiles = 4;                 // 16-row tiles per warp: h is brought once for all of them
constexpr int kDownRows = 16 * kDownTiles;    // output rows per cluster
constexpr int kDownSplit = 4;                 // CTAs of a cluster: each takes a share of the (unit, step) sequence

// Shared memory of kernel 2 behind the routing: per warp a ring of codes, a ring of windows and h records
// [NT / 2][4], the partial sums [T][64]; then zeros that cover the reach of a step's operands, barriers.
struct DownLayout {
  int rest, stage, windows, warp_rest, zeros, bars, bytes;
  __host__ __device__ DownLayout(int T, int nt, int code_bytes, int window_bytes, int stages) {
    rest = kDownWarps * stages * code_bytes;
    stage = window_bytes + nt / 2 * 4 * kRecord;
    warp_rest = stages * stage + T * kDownRows * 4;
    zeros = rest + kDownWarps * warp_rest;
    bars = zeros + 4 * kRecord;
    bytes = bars + kDownWarps * kMaxStages * 8 + 1024;
  }
};

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

template <int G, bool ASYM, int MODE>
__global__ void __cluster_dims__(kDownSplit, 1, 1) __launch_bounds__(kDownThreads, G == 1 ? 1 : 2)
moe_down_kernel(const __grid_constant__ CUtensorMap map, const MoeParams p, const int stages) {
  constexpr int NT = 8 / G;
  using Rg = Ring<G, kDownTiles, ASYM, MODE>;
  extern __shared__ uint8_t dyn_raw[];
  uint8_t* dyn = dyn_raw + ((1024u - (sm100::smem_u32(dyn_raw) & 1023u)) & 1023u);
  __shared__ Units u;
  __shared__ int abort_flag;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int n_blk = p.I / 32, n_steps = (n_blk + 3) / 4, n_group = n_blk / p.down.group_blocks;
  const int rank = (int)sm100::cluster_ctarank();
  const int j0 = blockIdx.x / kDownSplit * kDownRows;
  const int rows_left = min(kDownRows, p.H - j0);  // 32 in the last cluster of an odd H / 32
  const DownLayout at(p.T, NT, Rg::kCodes, Rg::kWindow, stages);
  const uint32_t base = sm100::smem_u32(dyn);
  uint64_t* bars = reinterpret_cast<uint64_t*>(dyn + at.bars) + warp * kMaxStages;
  const int code_ring = warp * stages * Rg::kCodes, rest_ring = at.rest + warp * at.warp_rest;
  auto sums_of = [&](int w) {
    return reinterpret_cast<float*>(dyn + at.rest + w * at.warp_rest + stages * at.stage);  // [T][64]
  };
  float* sums = sums_of(warp);
  for (int i = lane; i < p.T * kDownRows; i += 32) sums[i] = 0.f;
  for (int i = tid; i < kRecord; i += kDownThreads) reinterpret_cast<uint32_t*>(dyn + at.zeros)[i] = 0;
  if (tid == 0) {
    abort_flag = 0;
    sm100::tma_prefetch_desc(&map);
  }
  if (lane == 0) {
    for (int i = 0; i < stages; ++i) sm100::mbar_init(&bars[i], 1);
    sm100::fence_barrier_init();
  }
  const int n_units = __ldcg(&p.units->n);
  for (int i = tid; i < n_units; i += kDownThreads) {
    u.mask[i] = __ldcg(&p.units->mask[i]);
    u.expert[i] = __ldcg(&p.units->expert[i]);
    u.slot[i] = __ldcg(&p.units->slot[i]);
  }
  __syncthreads();

  // (unit, step) pairs in a row, an equal share of consecutive ones per warp of the cluster
  const int64_t total = (int64_t)n_units * n_steps;
  const int share = rank * kDownWarps + warp, shares = kDownSplit * kDownWarps;
  const int first = (int)(total * share / shares), last = (int)(total * (share + 1) / shares);
  const int lane_blk = t / (4 / G);
  const bool diag = g / NT == lane_blk;
  const uint8_t* operand = dyn + (diag ? rest_ring + Rg::kWindow + (g % NT / 2 * 4 + lane_blk) * kRecord + (g & 1) * 64 +
                                             t % (4 / G) * G * 16
                                       : at.zeros);
  const int operand_stage = diag ? at.stage : 0;
  const uint8_t* sides = dyn + rest_ring + Rg::kWindow + (t % (4 / G) * 4 + lane_blk) * kRecord + 128;

  const int64_t total_groups = (int64_t)p.E * p.H * n_group;
  const int first_u = first / n_steps, first_s = first - first_u * n_steps;
  // a run of windows is what the warp does of one unit
  int f_at = first, f_u = first_u, f_s = first_s, f_stage = 0, f_window = 0, f_next = first_s;
  auto fetch_weights = [&] {
    const int row0 = u.expert[f_u] * p.H + j0;
    if (lane == 0) {
      sm100::mbar_arrive_expect_tx(&bars[f_stage], Rg::kCodes);
      sm100::tma_load_2d(dyn + code_ring + f_stage * Rg::kCodes, &map, &bars[f_stage], f_s * 64, row0);
    }
    if (f_s == f_next) {
      f_next = Rg::next_window(p.down, f_s);
      Rg::template fetch_window<kDownRows>(base + rest_ring + f_window * at.stage, 0, p.down,
                                           (int64_t)row0 * n_group + group_of(p.down, f_s * 4), n_group, total_groups,
                                           lane);
      if (++f_window == stages) f_window = 0;
    }
  };
  constexpr int kPieces = kRecord / 16, kParts = (NT / 2 * 4 * kPieces + 31) / 32;
  int part_src[kParts];  // of this lane's 16-byte pieces of a step's records, from the unit's first of the step on
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    const int c = i * 32 + lane, pair = c / (4 * kPieces);
    part_src[i] = pair * n_blk * kRecord + (c - pair * 4 * kPieces) * 16;
  }
  auto fetch_records = [&] {  // blocks 4 f_s .. + 4 of the unit's tokens; zeros past n_blk
    const uint8_t* rec = p.h + ((int64_t)u.slot[f_u] * n_blk + f_s * 4) * kRecord;
    const int pieces = (__popc(u.mask[f_u]) + 1) / 2 * 4 * kPieces;
    const uint32_t to = base + rest_ring + f_stage * at.stage + Rg::kWindow + lane * 16;
    const int whole = (n_blk - f_s * 4) * kPieces;  // pieces of a pair that exist
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int c = i * 32 + lane;
      const bool valid = MODE != kAny || c % (4 * kPieces) < whole;
      if (c < pieces) cp_async16(to + i * 512, valid ? rec + part_src[i] : p.h, valid ? 16 : 0);
    }
  };
  auto advance = [&] {
    cp_async_commit();
    if (f_at < last) {
      ++f_at;
      if (++f_s == n_steps) {
        f_s = f_next = 0;
        ++f_u;
      }
      if (++f_stage == stages) f_stage = 0;
    }
  };

  float acc[kDownTiles][4] = {};
  int unit = -1;
  auto flush = [&] {
    uint32_t m = unit >= 0 ? u.mask[unit] : 0u;
    for (int i = 0; i < 2 * t; ++i) m &= m - 1;  // of this lane's two tokens
    const int token[2] = {__ffs(m) - 1, __ffs(m & (m - 1)) - 1};
#pragma unroll
    for (int w = 0; w < kDownTiles; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float q = block_sum<G>(acc[w][2 * h + c]);
          if (t < 4 / G && token[c] >= 0) sums[token[c] * kDownRows + w * 16 + h * 8 + Rg::row_of(g)] += q;
          acc[w][2 * h + c] = 0.f;
        }
      }
    __syncwarp();
  };

  int c_u = first_u, c_s = first_s, stage = 0, window = -1, w_s = 0, w_next = first_s;
  uint32_t parity = 0;
  bool ok = true;
  for (int q = first - stages; q < last; ++q) {
    if (q >= first) {
      if (c_u != unit) {
        flush();
        unit = c_u;
      }
      ok = sm100::mbar_wait_bounded(&bars[stage], parity, &abort_flag, p.wait_ns) && ok;
      cp_async_wait(stages - 1);
      __syncwarp();
      if (c_s == w_next) {
        if (++window == stages) window = 0;
        w_s = c_s;
        w_next = Rg::next_window(p.down, c_s);
      }
      const int index = Rg::index_of(p.down, c_s, w_s, g, n_group);
      const uint8_t* side = sides + stage * at.stage;
      add_step<G, kDownTiles, ASYM, MODE, true, kRecord, kRecord, kRecord>(acc, dyn + code_ring + stage * Rg::kCodes,
                                                                  dyn + rest_ring + window * at.stage, index, operand + stage * operand_stage,
                                                                  Sides{side, side + 16, side + 24}, g, t, c_s, n_blk,
                                                                  p.down);
      __syncwarp();
      if (++c_s == n_steps) {
        c_s = w_next = 0;
        ++c_u;
      }
      if (++stage == stages) {
        stage = 0;
        parity ^= 1;
      }
    }
    if (f_at < last) {
      fetch_weights();
      fetch_records();
    }
    advance();
  }
  flush();
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (!ok) {
    atomicExch(&g_moe_status, 2);
    const uint64_t t0 = sm100::global_timer_ns();
    while (sm100::global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
  }
  __syncthreads();
  // the warps of the CTA (into warp 0's sums), then the CTAs of the cluster: each finishes a quarter of the rows
  float* cta_sums = sums_of(0);
  for (int i = tid; i < p.T * kDownRows; i += kDownThreads) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kDownWarps; ++w) v += sums_of(w)[i];
    cta_sums[i] = v;
  }
  __syncwarp();
  sm100::cluster_sync_all();
  constexpr int kRowsEach = kDownRows / kDownSplit;
  for (int i = tid; i < p.T * kRowsEach; i += kDownThreads) {
    const int token = i / kRowsEach, row = rank * kRowsEach + i % kRowsEach;
    float v = 0.f;
#pragma unroll
    for (int c = 0; c < kDownSplit; ++c)
      v += ld_cluster_f32(sm100::map_to_cta(sm100::smem_u32(cta_sums) + (token * kDownRows + row) * 4, c));
    if (row >= rows_left) continue;
    const int64_t to = (int64_t)token * p.H + j0 + row;
    if (p.dtype == NPB_BF16) static_cast<__nv_bfloat16*>(p.y)[to] = from_f32<__nv_bfloat16>(v);
    else static_cast<__half*>(p.y)[to] = from_f32<__half>(v);
  }
  __syncwarp();
  sm100::cluster_sync_all();  // nobody leaves while its sums are read
}

// ---- host ----------------------------------------------------------------------------------------
int mode_of(const MoeWeight& w, int n_blk) {
  if (w.group_shift < 0 || (n_blk / w.group_blocks) % 8 != 0) return kAny;
  return w.group_blocks == 1 ? kOnePerBlock : kPowerOfTwo;
}

// Codes [rows, bytes of a row] in boxes of 64 bytes x box_rows.
int make_code_map(CUtensorMap* map, const uint8_t* codes, int64_t rows, int64_t row_bytes, int box_rows) {
  return make_tensor_map_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, codes, rows, row_bytes, box_rows, 64,
                            CU_TENSOR_MAP_SWIZZLE_64B);
}

// Ring stages that fit next to the rest (2..4; 0: not even two do).
template <typename Bytes>
int pick_stages(Bytes bytes, int static_bytes, int ctas_per_sm) {
  const int cap = ctas_per_sm == 1 ? max_dynamic_smem() : (max_dynamic_smem() - 1024) / ctas_per_sm - 1024;
  int stages = kMaxStages;
  while (stages >= 2 && bytes(stages) + static_bytes > cap) --stages;
  return stages >= 2 ? stages : 0;
}

int window_bytes(int rows, bool asym, int mode) { return rows * (mode == kAny ? 32 : 16) * (asym ? 2 : 1); }

int up_bytes(const MoeParams& p, int g, int stages) {
  return UpLayout(p.H / 32, 8 / g, p.gate.zp != nullptr, 32 * 64,
                  window_bytes(32, p.gate.zp != nullptr, mode_of(p.gate, p.H / 32)), stages).bytes;
}
int up_stages(const MoeParams& p, int g) {
  return pick_stages([&](int n) { return up_bytes(p, g, n); }, (int)sizeof(Routing) + 256, 1);
}
int down_bytes(const MoeParams& p, int g, int stages) {
  return DownLayout(p.T, 8 / g, kDownRows * 64,
                    window_bytes(kDownRows, p.down.zp != nullptr, mode_of(p.down, p.I / 32)), stages).bytes;
}
int down_stages(const MoeParams& p, int g) {
  auto bytes = [&](int n) { return down_bytes(p, g, n); };
  const int two = g == 1 ? 0 : pick_stages(bytes, (int)sizeof(Units) + 256, 2);  // two CTAs on an SM where they fit
  return two ? two : pick_stages(bytes, (int)sizeof(Units) + 256, 1);
}

template <int G, bool ASYM, int MODE>
int launch_up(const MoeParams& p, cudaStream_t st) {
  auto kern = moe_up_kernel<G, ASYM, MODE>;
  const int stages = up_stages(p, G), smem = up_bytes(p, G, stages);
  int per_sm = 0;
  if (int rc = blocks_per_sm(reinterpret_cast<const void*>(kern), kUpThreads, smem, &per_sm)) return rc;
  if (per_sm < 1) return NPB_ERR_TOO_LARGE;
  UpMaps maps;
  if (int rc = make_code_map(&maps.gate, p.gate.codes, (int64_t)p.E * p.I, p.H / 2, 16)) return rc;
  if (int rc = make_code_map(&maps.up, p.up.codes, (int64_t)p.E * p.I, p.H / 2, 16)) return rc;
  const int64_t active = p.T * p.top_k < p.E ? p.T * p.top_k : p.E;
  const int64_t most = active * (p.I / kUpRows), slots = (int64_t)sm_count() * per_sm;
  kern<<<(unsigned)(most < slots ? most : slots), kUpThreads, smem, st>>>(maps, p, stages);
  NPB_LAUNCH_CHECK();
  return NPB_OK;
}

template <int G, bool ASYM, int MODE>
int launch_down(const MoeParams& p, cudaStream_t st) {
  auto kern = moe_down_kernel<G, ASYM, MODE>;
  const int stages = down_stages(p, G), smem = down_bytes(p, G, stages);
  int per_sm = 0;
  if (int rc = blocks_per_sm(reinterpret_cast<const void*>(kern), kDownThreads, smem, &per_sm)) return rc;
  if (per_sm < 1) return NPB_ERR_TOO_LARGE;
  CUtensorMap map;
  if (int rc = make_code_map(&map, p.down.codes, (int64_t)p.E * p.H, p.I / 2, kDownRows)) return rc;
  kern<<<(unsigned)((p.H + kDownRows - 1) / kDownRows * kDownSplit), kDownThreads, smem, st>>>(map, p, stages);
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
  auto fits = [&](int g) { return up_stages(p, g) && down_stages(p, g); };
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
  // the last group of the last step lies at most eight groups behind the first, which lies at most seven behind
  // the window's start: sixteen values hold them
  out->window = out->group_blocks >= 4 ? 8 : 2 * out->group_blocks;
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
  return (int64_t)sizeof(Units) + T * top_k * (I / 32) * kRecord;  // a pair of tokens of an expert is at least one of the T * top_k
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
