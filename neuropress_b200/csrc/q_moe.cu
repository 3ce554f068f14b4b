// A mixture-of-experts layer for a few tokens over 4-bit group-affine experts, in two kernels:
//
//   p = softmax(l_t);  S_t = the top_k largest l_t (equal logits: lowest expert);
//   w_te = p_e, or p_e / sum_{S_t} p
//   h_te[i] = w_te * silu(G_e x_t)[i] * (U_e x_t)[i]              kernel 1: routing, gate / up, silu
//   y_t     = T( sum_{e in S_t} D_e h_te )                         kernel 2: routing, down, sum
//   W[n, k] = (q[n, k] - z) * s  in fp32, z and s per group of k (z = 8 without a zero point)
//
// Each active expert's codes are read once; HBM-bound (0.56 bytes per weight at group 32).  Both kernels
// route by themselves (a warp per token, every CTA alike: a microsecond, no hand-over between kernels),
// and the second is launched with programmatic serialisation, so it routes and fetches its first
// weights under the end of the first.
//
// Product: mma.sync.m16n8k16 in fp16 with the weights as the A operand (16 rows) built in registers.  A code
// q becomes 1024 + q or, four bits higher in the mantissa, 1024 + 16 q with one bit operation per two
// codes; the activations that meet the latter are stored divided by 16.  With x' the stored activations
//   sum_k (q - z) x = D - 1024 sum_k x' - z sum_k x,   D the mma's sum
// is applied per 32-wide block, with the weight's scale, in fp32.  Activations are stored as fp16 with a power
// of two per 32-block and token, so their size does not matter: a bf16 or fp16 x loses nothing down to
// 2^-13 of its block's largest (below that at most 2^-21 of the largest), and h keeps 11 significant bits
// between the kernels, 1/8 of a bf16 half step.
//
// The eight columns of an mma are NT = 8 / G tokens times G neighbouring 32-blocks (G = 4, 2, 1): lane (g, t)
// of a warp loads G words, the t-th part of G blocks, of rows g and g + 8, so the k slots of an mma hold
// G different blocks, and the B operand keeps them apart by being block-diagonal.  Lane (g, t) of the result
// then holds two tokens of exactly the block whose scale it loaded.  A step of four blocks takes the same
// sixteen mmas for two 16-row tiles whatever G is (8 cycles of a scheduler's tensor pipe each, measured);
// G = 4 has the widest loads and the fewest results to scale, G = 1 the most tokens per weight read.
//
// Kernel 1 keeps the tokens of its unit (up to NT tokens of one expert) in shared memory in the order of
// the mma operands and writes h in that order; kernel 2 brings h along with the weights by cp.async.  An
// expert with more tokens than a unit is read again (from L2).  Every sum has a fixed order: results do
// not depend on scheduling.
#include <type_traits>

#include "common.cuh"
#include "mma_sync.cuh"
#include "order_key.cuh"
#include "tcgen05.cuh"

namespace npb {
namespace {

constexpr int kMaxTokens = 32;   // bits of an expert's token mask
constexpr int kMaxExperts = 512;
constexpr int kMaxTopK = 16;
constexpr int kMaxUnits = kMaxTokens * kMaxTopK;
constexpr int kMaxWidth = 32768;  // of H and I: two tokens of H in shared memory

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
  uint8_t* h;      // [pair of tokens of a unit][I / 32] records
  void* y;
};

// One 32-block of h of two tokens: 32 stored fp16 values of each (64 bytes), then their Factors.
constexpr int kRecord = 160;

// ---- routing ---------------------------------------------------------------------------------
struct Routing {
  uint32_t mask[kMaxExperts];            // tokens of each expert
  float weight[kMaxTokens][kMaxTopK];
  uint16_t id[kMaxTokens][kMaxTopK];     // 0xffff: none
  uint16_t unit_expert[kMaxUnits];
  uint32_t unit_mask[kMaxUnits];         // its tokens
  uint16_t unit_slot[kMaxUnits];         // row of h of its first pair
  int n_units;
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
    float chosen = 0.f;
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
      const float l = key_value(top);
      const float w = expf(l - m);
      chosen += w;
      if (lane == 0) {
        const bool none = nowhere || (l == -INFINITY && all == all);  // probability 0: not read
        r.id[t][j] = none ? 0xffffu : (uint16_t)e;
        r.weight[t][j] = w;
        if (!none) atomicOr(&r.mask[e], 1u << t);
      }
    }
    __syncwarp();
    const float norm = p.renormalize ? (all != all ? all : chosen) : all;
    for (int j = lane; j < p.top_k; j += 32) r.weight[t][j] /= norm;
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
        r.unit_expert[at] = (uint16_t)e;
        r.unit_mask[at] = m & ~rest;
        r.unit_slot[at] = (uint16_t)(slots + in - pairs + i * (NT / 2));
        m = rest;
      }
      units += __shfl_sync(0xffffffffu, iu, 31);
      slots += __shfl_sync(0xffffffffu, in, 31);
    }
    if (lane == 0) r.n_units = units;
  }
  __syncthreads();
}

// ---- weights ---------------------------------------------------------------------------------
__device__ __forceinline__ int group_of(const MoeWeight& w, int blk) {
  return w.group_shift >= 0 ? blk >> w.group_shift : blk / w.group_blocks;
}

// This lane's part of one step (four 32-blocks) of four rows (g and g + 8 of two tiles).
template <int G, bool ASYM>
struct Step {
  uint32_t c[4][4];              // [row][set * G + word]
  uint2 s[4], z[ASYM ? 4 : 1];   // scales, zero points as fp16: of the four blocks (G = 4: of the lane's own)
};

__device__ __forceinline__ uint32_t ldg_u16(const __half* p) {
  return __ldg(reinterpret_cast<const unsigned short*>(p));
}

// Four consecutive blocks' values of one row, the first in group `group`.
template <int G, bool WIDE>
__device__ __forceinline__ uint2 fetch_groups(const __half* v, const MoeWeight& w, int64_t at_row, int first, int own,
                                              int n_blk) {
  if constexpr (G == 4) return make_uint2(ldg_u16(v + at_row + group_of(w, own)), 0u);
  if constexpr (WIDE) {
    if (w.group_blocks == 1) return __ldg(reinterpret_cast<const uint2*>(v + at_row + first));
    if (w.group_blocks == 2) {
      const uint32_t q = __ldg(reinterpret_cast<const uint32_t*>(v + at_row + first / 2));
      return make_uint2(__byte_perm(q, q, 0x1010), __byte_perm(q, q, 0x3232));
    }
    const uint32_t q = ldg_u16(v + at_row + group_of(w, first)) * 0x10001u;
    return make_uint2(q, q);
  } else {
    uint32_t q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = first + j < n_blk ? ldg_u16(v + at_row + group_of(w, first + j)) : 0u;
    return make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
  }
}

// Row i of step s: codes from block `at_blk` of the matrix on (the row's first), groups from `at_row` on.  WIDE:
// every step is whole and the groups of a step are read at once; otherwise blocks past n_blk become zeros.
template <int G, bool ASYM, bool WIDE>
__device__ __forceinline__ void fetch_row(Step<G, ASYM>& b, int i, const MoeWeight& w, int64_t at_blk, int64_t at_row,
                                          int s, int n_blk, int t) {
  const int own = s * 4 + t / (4 / G);
  const uint8_t* codes = w.codes + (at_blk + own) * 16 + (t % (4 / G)) * (4 * G);
#pragma unroll
  for (int j = 0; j < 4 / G; ++j) {
    uint32_t* c = &b.c[i][j * G];
    if (WIDE || own + j * G < n_blk) {
      if constexpr (G == 4)
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3]) : "l"(codes));
      else if constexpr (G == 2)
        asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(c[0]), "=r"(c[1])
                     : "l"(codes + j * 32));
      else  // two requests share a 32-byte sector
        asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(c[0]) : "l"(codes + j * 16));
    } else {
#pragma unroll
      for (int k = 0; k < G; ++k) c[k] = 0;
    }
  }
  if (WIDE || G != 4 || own < n_blk) {
    b.s[i] = fetch_groups<G, WIDE>(w.scale, w, at_row, s * 4, own, n_blk);
    if (ASYM) b.z[ASYM ? i : 0] = fetch_groups<G, WIDE>(w.zp, w, at_row, s * 4, own, n_blk);
  } else {
    b.s[i] = make_uint2(0u, 0u);
    if (ASYM) b.z[ASYM ? i : 0] = make_uint2(0u, 0u);
  }
}

// The value of this lane's block of set j.
template <int G>
__device__ __forceinline__ float group_value(const uint2& v, int j, int t) {
  if (G == 4) return __half2float(__ushort_as_half((unsigned short)v.x));
  if (G == 2) return __half2float(__ushort_as_half((unsigned short)((j ? v.y : v.x) >> (t / 2 * 16))));
  const uint32_t w = j < 2 ? v.x : v.y;
  return __half2float(__ushort_as_half((unsigned short)(j & 1 ? w >> 16 : w)));
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
// Of one 32-block of two tokens: the powers of two they were divided by, what to subtract from D for the magic
// (and, for a symmetric weight, for z = 8), the sums that a zero point multiplies.
struct alignas(16) Factors {
  float f[2], c[2], s2[2], unused[2];
};

// The power of two at or below a magnitude (1 for zero, subnormal, inf, NaN).
__device__ __forceinline__ float power_below(float top) {
  const uint32_t exponent = __float_as_uint(top) >> 23;
  return exponent == 0 || exponent == 255 ? 1.f : __uint_as_float(exponent << 23);
}

// Token c of a pair, from the sums of its block's stored values at k = 0, 2 mod 4 (`even`) and 1, 3 mod 4 (`odd`,
// divided by 16).
__device__ __forceinline__ void put_factors(Factors* to, int c, float f, float even, float odd, bool asym) {
  const float s2 = even + 16.f * odd, m = 1024.f * (even + odd);
  to->f[c] = f;
  to->c[c] = asym ? m : m + 8.f * s2;
  to->s2[c] = s2;
}

// Two floats in a register pair, for the packed fp32 instructions.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 pack(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack(const F2& x, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v));
}
__device__ __forceinline__ F2 sub2(const F2& a, const F2& b) {  // a - b
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(b.v), "l"(0xbf800000bf800000ull), "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 mul2(const F2& a, const F2& b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(const F2& a, const F2& b, const F2& c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 lds_f2(uint32_t addr) {
  F2 r;
  asm volatile("ld.shared.u64 %0, [%1];" : "=l"(r.v) : "r"(addr));
  return r;
}
__device__ __forceinline__ void lds_2f2(uint32_t addr, F2& a, F2& b) {
  asm volatile("ld.shared.v2.u64 {%0, %1}, [%2];" : "=l"(a.v), "=l"(b.v) : "r"(addr));
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

// Adds one step of two 16-row tiles to acc[tile][row g, g + 8] (two tokens each).  `operand` is the shared address
// of this lane's part of the first set in B order, BLOCK bytes from block to block (a lane off the diagonal:
// zeros); `factors` that of the Factors of its two tokens and its block of the first set, FAC bytes from block
// to block.
template <int G, bool ASYM, int BLOCK, int FAC>
__device__ __forceinline__ void add_step(F2 (&acc)[2][2], const Step<G, ASYM>& b, uint32_t operand, uint32_t factors,
                                         int t) {
#pragma unroll
  for (int j = 0; j < 4 / G; ++j) {
    float d[2][4];
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const uint4 v = lds128(operand + j * G * BLOCK + i * 16);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        uint32_t a[2][4];
        a_operands(b.c[2 * w][j * G + i], b.c[2 * w + 1][j * G + i], a);
        if (i == 0) mma16816_first<__half>(d[w], a[0], v.x, v.y);
        else mma16816<__half>(d[w], a[0], v.x, v.y);
        mma16816<__half>(d[w], a[1], v.z, v.w);
      }
    }
    F2 f, c, s2{};
    lds_2f2(factors + j * G * FAC, f, c);
    if (ASYM) s2 = lds_f2(factors + j * G * FAC + 16);
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float sc = group_value<G>(b.s[2 * w + h], j, t);
        F2 v = sub2(pack(d[w][2 * h], d[w][2 * h + 1]), c);
        if (ASYM) {
          const float z = -group_value<G>(b.z[ASYM ? 2 * w + h : 0], j, t);
          v = fma2(pack(z, z), s2, v);
        }
        acc[w][h] = fma2(mul2(pack(sc, sc), f), v, acc[w][h]);
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
constexpr int kUpThreads = 256;  // two 16-row tiles x four slices of K
constexpr int kUpRows = 32;      // rows of gate and of up per item: one 32-block of h
constexpr int kUpSlices = 4;

// Shared memory of kernel 1 behind the routing: tokens [NT][4 * steps] blocks of 64 bytes (neighbouring rows
// in the other half of the banks), their Factors, the partial products, 256 bytes of zeros.
struct UpLayout {
  int row, factors, red, zeros, bytes;
  __host__ __device__ UpLayout(int n_blk, int nt) {
    const int blocks = (n_blk + 3) / 4 * 4;
    row = blocks * 64 + 64;
    factors = row * nt;
    red = factors + nt / 2 * blocks * (int)sizeof(Factors);
    zeros = red + kUpSlices * 2 * 2 * nt * 16 * 4;
    bytes = zeros + 256;
  }
};

// Stores eight elements of a token (thread j of a row: elements 8 j ...) in the order of the mma operands, and
// their block's Factors; the lanes of a quad share a block.
template <typename T>
__device__ __forceinline__ void store_operand(const uint4& raw, uint4* to, Factors* fac, int c, bool write, bool asym) {
  const T* v = reinterpret_cast<const T*>(&raw);
  float top = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(to_f32(v[k])));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const float f = power_below(top), even_by = 1.f / f, odd_by = 0.0625f / f;
  __half2 o[4];
  float even = 0.f, odd = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float by = k & 1 ? odd_by : even_by;
    o[k] = __floats2half2_rn(to_f32(v[k]) * by, to_f32(v[k + 4]) * by);
    (k & 1 ? odd : even) += __low2float(o[k]) + __high2float(o[k]);
  }
  even = quad_sum(even);
  odd = quad_sum(odd);
  if (write) {
    *to = *reinterpret_cast<const uint4*>(o);
    if ((threadIdx.x & 3) == 0) put_factors(fac, c, f, even, odd, asym);
  }
}

template <int G, bool ASYM, bool WIDE>
__global__ void __launch_bounds__(kUpThreads, 2)
moe_up_kernel(const MoeParams p) {
  constexpr int NT = 8 / G;
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ Routing r;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int n_blk = p.H / 32, n_steps = (n_blk + 3) / 4, blocks = n_steps * 4;
  const int n_group = n_blk / p.gate.group_blocks;
  const UpLayout at(n_blk, NT);
  Factors* fac = reinterpret_cast<Factors*>(dyn + at.factors);  // [NT / 2][blocks]
  float* red = reinterpret_cast<float*>(dyn + at.red);          // [slice][tile][matrix][NT][16]
  const uint32_t base = sm100::smem_u32(dyn);
  if (tid < 64) reinterpret_cast<uint32_t*>(dyn + at.zeros)[tid] = 0;
  route<NT>(p, r);

  const int tiles = p.I / kUpRows;
  const int64_t items = (int64_t)tiles * r.n_units;
  const int first = (int)(items * blockIdx.x / gridDim.x), last = (int)(items * (blockIdx.x + 1) / gridDim.x);
  const int mt = warp & 1, ks = warp >> 1;
  const int s_first = n_steps * ks / kUpSlices, s_last = n_steps * (ks + 1) / kUpSlices;
  const int lane_blk = t / (4 / G);      // this lane's block of a set
  const bool diag = g / NT == lane_blk;  // it holds the nonzero part of column g
  const uint32_t operand = diag ? base + (g % NT) * at.row + lane_blk * 64 + t % (4 / G) * G * 16 : base + at.zeros;
  const int operand_step = diag ? 256 : 0;
  const uint32_t factors = base + at.factors + (t % (4 / G) * blocks + lane_blk) * (int)sizeof(Factors);

  int unit = -1, n = 0, e = 0;
  for (int item = first; item < last; ++item) {
    const int u = item / tiles, i0 = (item - u * tiles) * kUpRows;
    e = r.unit_expert[u];
    const int64_t row = (int64_t)e * p.I + i0 + mt * 16 + g;
    const int64_t row_blk = row * n_blk, row_group = row * n_group;
    using S = Step<G, ASYM>;
    auto fetch = [&](S& b, int s) {
      if (s < s_last) {
        fetch_row<G, ASYM, WIDE>(b, 0, p.gate, row_blk, row_group, s, n_blk, t);
        fetch_row<G, ASYM, WIDE>(b, 1, p.gate, row_blk + 8 * n_blk, row_group + 8 * n_group, s, n_blk, t);
        fetch_row<G, ASYM, WIDE>(b, 2, p.up, row_blk, row_group, s, n_blk, t);
        fetch_row<G, ASYM, WIDE>(b, 3, p.up, row_blk + 8 * n_blk, row_group + 8 * n_group, s, n_blk, t);
      }
    };
    S b0, b1;
    fetch(b0, s_first);
    fetch(b1, s_first + 1);
    if (u != unit) {
      unit = u;
      uint32_t m = r.unit_mask[u];
      n = __popc(m);
      // the unit's tokens: a thread takes eight elements (columns of an mma past the last token hold what was
      // there: nothing reads their sums)
#pragma unroll 1
      for (int i = 0; i < n; ++i, m &= m - 1) {
        const uint4* src = reinterpret_cast<const uint4*>(p.x) + (int64_t)(__ffs(m) - 1) * (n_blk * 4);
        for (int j0 = 0; j0 < blocks * 4; j0 += kUpThreads) {  // whole warps
          const int j = j0 + tid;
          uint4 raw = make_uint4(0, 0, 0, 0);
          if (j < n_blk * 4) raw = __ldg(src + j);
          uint4* to = reinterpret_cast<uint4*>(dyn + i * at.row + j * 16);
          Factors* f = fac + i / 2 * blocks + (j >> 2);
          if (p.dtype == NPB_BF16) store_operand<__nv_bfloat16>(raw, to, f, i & 1, j < blocks * 4, ASYM);
          else store_operand<__half>(raw, to, f, i & 1, j < blocks * 4, ASYM);
        }
      }
      __syncthreads();
    }
    F2 acc[2][2] = {};
    auto compute = [&](const S& b, int s) {
      add_step<G, ASYM, 64, sizeof(Factors)>(acc, b, operand + s * operand_step, factors + s * 4 * (int)sizeof(Factors), t);
    };
    for (int s = s_first; s < s_last; s += 2) {
      compute(b0, s);
      fetch(b0, s + 2);
      if (s + 1 < s_last) compute(b1, s + 1);
      fetch(b1, s + 3);
    }
    // the blocks of a set, then the slices of K
    float* part = red + (ks * 2 + mt) * 2 * NT * 16;
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[2];
        unpack(acc[w][h], v[0], v[1]);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float q = block_sum<G>(v[c]);
          if (t < 4 / G) part[(w * NT + 2 * t + c) * 16 + g + h * 8] = q;
        }
      }
    __syncthreads();
    if (warp < n) {  // a warp per token, a lane per row
      float gate = 0.f, up = 0.f;
#pragma unroll
      for (int k = 0; k < kUpSlices; ++k) {
        const float* from = red + ((k * 2 + (lane >> 4)) * 2 * NT + warp) * 16 + (lane & 15);
        gate += from[0];
        up += from[NT * 16];
      }
      uint32_t m = r.unit_mask[u];
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
      uint8_t* rec = p.h + ((int64_t)(r.unit_slot[u] + warp / 2) * (p.I / 32) + i0 / 32) * kRecord;
      reinterpret_cast<__half*>(rec)[(warp & 1) * 32 + (lane & 24) + (lane & 3) * 2 + ((lane >> 2) & 1)] = v;
      if (lane == 0)
        put_factors(reinterpret_cast<Factors*>(rec + 128), warp & 1, f, even, odd, p.down.zp != nullptr);
    }
    __syncthreads();
  }
}

// ---- kernel 2: down product and the sum over experts ----------------------------------------------
constexpr int kDownThreads = 256;
constexpr int kDownWarps = kDownThreads / 32;
constexpr int kDownRows = 32;    // output rows per cluster: two 16-row tiles per warp
constexpr int kDownSplit = 4;    // CTAs of a cluster: each takes a share of the (unit, step) sequence
constexpr int kDownStages = 2;

// Shared memory of kernel 2 behind the routing: per warp the partial sums [T][32] and a ring of h records
// [stage][NT / 2][4], then zeros that cover the reach of a step's operands.
struct DownLayout {
  int sums, ring, warp, zeros, bytes;
  __host__ __device__ DownLayout(int T, int nt) {
    sums = T * kDownRows * 4;
    ring = kDownStages * (nt / 2) * 4 * kRecord;
    warp = sums + ring;
    zeros = warp * kDownWarps;
    bytes = zeros + 4 * kRecord;
  }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

template <int G, bool ASYM, bool WIDE>
__global__ void __cluster_dims__(kDownSplit, 1, 1) __launch_bounds__(kDownThreads, 2)
moe_down_kernel(const MoeParams p) {
  constexpr int NT = 8 / G;
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ Routing r;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int n_blk = p.I / 32, n_steps = (n_blk + 3) / 4, n_group = n_blk / p.down.group_blocks;
  const int rank = (int)sm100::cluster_ctarank();
  const int j0 = blockIdx.x / kDownSplit * kDownRows;
  const DownLayout at(p.T, NT);
  const uint32_t base = sm100::smem_u32(dyn);
  float* sums = reinterpret_cast<float*>(dyn + warp * at.warp);  // [T][32]
  for (int i = lane; i < p.T * kDownRows; i += 32) sums[i] = 0.f;
  for (int i = tid; i < kRecord; i += kDownThreads) reinterpret_cast<uint32_t*>(dyn + at.zeros)[i] = 0;
  route<NT>(p, r);

  // (unit, step) pairs in a row, an equal share of consecutive ones per warp of the cluster
  const int64_t total = (int64_t)r.n_units * n_steps;
  const int share = rank * kDownWarps + warp, shares = kDownSplit * kDownWarps;
  const int first = (int)(total * share / shares), last = (int)(total * (share + 1) / shares);
  const int lane_blk = t / (4 / G);
  const bool diag = g / NT == lane_blk;
  const uint32_t ring = base + warp * at.warp + at.sums;
  constexpr int kStage = NT / 2 * 4 * kRecord;
  const uint32_t operand = diag ? ring + (g % NT / 2 * 4 + lane_blk) * kRecord + (g & 1) * 64 + t % (4 / G) * G * 16
                                : base + at.zeros;
  const int operand_stage = diag ? kStage : 0;
  const uint32_t factors = ring + (t % (4 / G) * 4 + lane_blk) * kRecord + 128;

  // position of the next fetch, its unit's rows and records
  int fu = first / n_steps, fs = first - fu * n_steps, fetched = first, fn = 0;
  int64_t row_blk = 0, row_group = 0;
  const uint8_t* rec = nullptr;
  auto fetch_unit = [&] {
    if (fetched >= last) return;
    const int64_t row = (int64_t)r.unit_expert[fu] * p.H + j0 + g;
    row_blk = row * n_blk;
    row_group = row * n_group;
    rec = p.h + (int64_t)r.unit_slot[fu] * n_blk * kRecord;
    fn = __popc(r.unit_mask[fu]);
  };
  using S = Step<G, ASYM>;
  auto fetch_weights = [&](S& b) {
    if (fetched < last) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        fetch_row<G, ASYM, WIDE>(b, i, p.down, row_blk + 8 * i * n_blk, row_group + 8 * i * n_group, fs, n_blk, t);
    }
  };
  auto fetch_records = [&](int stage) {  // blocks fs * 4 .. + 4 of the unit's tokens; zeros past n_blk
    constexpr int kPieces = kRecord / 16;
    if (fetched < last)
#pragma unroll
      for (int c0 = 0; c0 < NT / 2 * 4 * kPieces; c0 += 32) {
        const int c = c0 + lane;
        const int k = c / kPieces, piece = c - k * kPieces, pair = k >> 2, blk = fs * 4 + (k & 3);
        const bool valid = blk < n_blk;
        if (c < NT / 2 * 4 * kPieces && 2 * pair < fn)
          cp_async16(ring + stage * kStage + c * 16, valid ? rec + ((int64_t)pair * n_blk + blk) * kRecord + piece * 16
                                                           : p.h, valid);
      }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto advance = [&] {
    ++fetched;
    if (++fs == n_steps) {
      fs = 0;
      ++fu;
      fetch_unit();
    }
  };

  F2 acc[2][2] = {};
  int unit = -1;
  auto flush = [&] {
    uint32_t m = unit >= 0 ? r.unit_mask[unit] : 0u;
    for (int i = 0; i < 2 * t; ++i) m &= m - 1;  // of this lane's two tokens
    const int token[2] = {__ffs(m) - 1, __ffs(m & (m - 1)) - 1};
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[2];
        unpack(acc[w][h], v[0], v[1]);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float q = block_sum<G>(v[c]);
          if (t < 4 / G && token[c] >= 0) sums[token[c] * kDownRows + w * 16 + h * 8 + g] += q;
        }
        acc[w][h] = F2{0ull};
      }
    __syncwarp();
  };
  int cu = fu, cs = fs;  // position of the computation
  auto compute = [&](const S& b, int stage) {
    if (cu != unit) {
      flush();
      unit = cu;
    }
    add_step<G, ASYM, kRecord, kRecord>(acc, b, operand + stage * operand_stage, factors + stage * kStage, t);
    if (++cs == n_steps) { cs = 0; ++cu; }
    __syncwarp();  // the stage may be filled again
  };

  S b0, b1;
  fetch_unit();
  // the first weights are under way before kernel 1 ends; h exists only after it
  fetch_weights(b0);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  fetch_records(0);
  advance();
  fetch_weights(b1);
  fetch_records(1);
  advance();
  for (int q = first; q < last; q += 2) {
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    compute(b0, 0);
    fetch_weights(b0);
    fetch_records(0);
    advance();
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    if (q + 1 < last) compute(b1, 1);
    fetch_weights(b1);
    fetch_records(1);
    advance();
  }
  flush();
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  // the warps of the CTA (into warp 0's sums), then the CTAs of the cluster: each finishes eight rows
  for (int i = tid; i < p.T * kDownRows; i += kDownThreads) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kDownWarps; ++w) v += reinterpret_cast<const float*>(dyn + w * at.warp)[i];
    reinterpret_cast<float*>(dyn)[i] = v;
  }
  __syncwarp();
  sm100::cluster_sync_all();
  constexpr int kRowsEach = kDownRows / kDownSplit;
  for (int i = tid; i < p.T * kRowsEach; i += kDownThreads) {
    const int token = i / kRowsEach, row = rank * kRowsEach + i % kRowsEach;
    float v = 0.f;
#pragma unroll
    for (int c = 0; c < kDownSplit; ++c)
      v += ld_cluster_f32(sm100::map_to_cta(base + (token * kDownRows + row) * 4, c));
    const int64_t to = (int64_t)token * p.H + j0 + row;
    if (p.dtype == NPB_BF16) static_cast<__nv_bfloat16*>(p.y)[to] = from_f32<__nv_bfloat16>(v);
    else static_cast<__half*>(p.y)[to] = from_f32<__half>(v);
  }
  __syncwarp();
  sm100::cluster_sync_all();  // nobody leaves while its sums are read
}

// ---- host ----------------------------------------------------------------------------------------
// Every step of a row of n_blk blocks is whole, and the groups of a step are aligned words.
bool is_wide(const MoeWeight& w, int n_blk) {
  const int gb = w.group_blocks;
  return n_blk % 4 == 0 && (gb == 1 || gb == 2 || gb % 4 == 0) && aligned_to(w.scale, 8) && aligned_to(w.zp, 8);
}

template <int G, bool ASYM, bool WIDE>
int launch_up(const MoeParams& p, cudaStream_t st) {
  auto kern = moe_up_kernel<G, ASYM, WIDE>;
  const size_t smem = UpLayout(p.H / 32, 8 / G).bytes;
  int per_sm = 0;
  if (int rc = blocks_per_sm(reinterpret_cast<const void*>(kern), kUpThreads, smem, &per_sm)) return rc;
  if (per_sm < 1) return NPB_ERR_TOO_LARGE;
  const int64_t active = p.T * p.top_k < p.E ? p.T * p.top_k : p.E;
  const int64_t most = active * (p.I / kUpRows), slots = (int64_t)sm_count() * per_sm;
  kern<<<(unsigned)(most < slots ? most : slots), kUpThreads, smem, st>>>(p);
  NPB_LAUNCH_CHECK();
  return NPB_OK;
}

template <int G, bool ASYM, bool WIDE>
int launch_down(const MoeParams& p, cudaStream_t st) {
  auto kern = moe_down_kernel<G, ASYM, WIDE>;
  const size_t smem = DownLayout(p.T, 8 / G).bytes;
  int per_sm = 0;
  if (int rc = blocks_per_sm(reinterpret_cast<const void*>(kern), kDownThreads, smem, &per_sm)) return rc;
  if (per_sm < 1) return NPB_ERR_TOO_LARGE;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.H / kDownRows * kDownSplit));
  cfg.blockDim = dim3(kDownThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  NPB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p));
  NPB_LAUNCH_CHECK();
  return NPB_OK;
}

template <int G>
int launch(const MoeParams& p, cudaStream_t st) {
  const bool wide_up = is_wide(p.gate, p.H / 32) && is_wide(p.up, p.H / 32), wide_down = is_wide(p.down, p.I / 32);
  int rc;
  if (p.gate.zp) rc = wide_up ? launch_up<G, true, true>(p, st) : launch_up<G, true, false>(p, st);
  else rc = wide_up ? launch_up<G, false, true>(p, st) : launch_up<G, false, false>(p, st);
  if (rc) return rc;
  if (p.down.zp) return wide_down ? launch_down<G, true, true>(p, st) : launch_down<G, true, false>(p, st);
  return wide_down ? launch_down<G, false, true>(p, st) : launch_down<G, false, false>(p, st);
}

int launch_tokens(const MoeParams& p, cudaStream_t st) {
  // an expert has at most T tokens; a unit's tokens have to fit the shared memory of kernel 1
  int g = p.T <= 2 ? 4 : p.T <= 4 ? 2 : 1;
  while (g < 4 && UpLayout(p.H / 32, 8 / g).bytes + (int)sizeof(Routing) > max_dynamic_smem() / 2) g *= 2;
  if (g == 4) return launch<4>(p, st);
  if (g == 2) return launch<2>(p, st);
  return launch<1>(p, st);
}

int make_weight(const npb_q_weight* w, int64_t N, int64_t K, MoeWeight* out) {
  if (int rc = validate_q(w, N, K)) return rc;
  if (w->nbits != 4 || w->group_size % 32 != 0) return NPB_ERR_UNSUPPORTED;
  if (!aligned_to(w->codes, 16)) return NPB_ERR_ALIGNMENT;
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

int64_t q_moe_workspace_bytes(int64_t T, int top_k, int64_t I) {
  if (T < 0 || top_k <= 0 || I <= 0 || T > kMaxTokens || top_k > kMaxTopK || I % 32 != 0) return 0;
  return T * top_k * (I / 32) * kRecord;  // a pair of tokens of an expert is at least one of the T * top_k
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
  p.h = static_cast<uint8_t*>(workspace);
  p.y = y;
  return launch_tokens(p, st);
}

}  // namespace npb
