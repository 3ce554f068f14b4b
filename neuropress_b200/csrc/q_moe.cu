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
// Every warp streams its own weights: a ring of steps in shared memory filled by cp.async, so that what is in flight
// does not depend on registers (register double buffers of the same kernels reached a third of the
// bandwidth: waiting for one step's loads waits for the next step's too).  Kernel 1 keeps the tokens of its
// unit (up to NT tokens of one expert) in shared memory in the order of the mma operands and writes h in
// that order; kernel 2 brings h along with the weights.  An expert with more tokens than a unit is read again
// (from L2).  Every sum has a fixed order: results do not depend on scheduling.
#include <type_traits>

#include "common.cuh"
#include "order_key.cuh"
#include "tcgen05.cuh"

namespace npb {
namespace {

constexpr int kMaxTokens = 32;   // bits of an expert's token mask
constexpr int kMaxExperts = 512;
constexpr int kMaxTopK = 16;
constexpr int kMaxUnits = kMaxTokens * kMaxTopK;
constexpr int kMaxWidth = 16384;  // of H and I: two tokens of H in shared memory next to the rings

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

// One 32-block of h of two tokens: 32 stored fp16 values of each (64 bytes), then {f0, f1, c0, c1, s2 of both}.
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

template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool valid = true) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES),
                 "r"(valid ? BYTES : 0)
                 : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits until at most `pending` (1..3) of the committed groups are under way.
__device__ __forceinline__ void cp_async_wait(int pending) {
  if (pending == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else if (pending == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else asm volatile("cp.async.wait_group 3;" ::: "memory");
}

// One step (four 32-blocks of k) of R 16-row tiles in a warp's ring: per row 64 bytes of codes, the 16-byte pieces
// permuted so that the reads below are free of bank conflicts, then per row 16 bytes with the scales of the
// step's groups and, if ASYM, with the zero points.  FAST: one group per block and rows of whole steps, the
// four values sit in the first eight bytes; otherwise the three words that hold them, which start at an odd
// fp16 where the row's first group is odd.
template <int G, int R, bool ASYM, bool FAST>
struct Ring {
  static constexpr int kRows = 16 * R;
  static constexpr int kScales = kRows * 64, kZeros = kScales + kRows * 16;
  static constexpr int kBytes = kZeros + (ASYM ? kRows * 16 : 0);

  __device__ static int swizzle(int row) { return G == 2 ? (row >> 1 & 1) * 2 : row >> 1 & 3; }

  // Codes of rows 8 i + lane / 4, i < N, to ring rows from `row0` on; `src` points at block 0 of row lane / 4.
  template <int N>
  __device__ static void fetch_codes(uint32_t stage, int row0, const uint8_t* src, int s, int n_blk, int lane) {
    const int c = lane & 3, row = row0 + (lane >> 2);
    const uint32_t dst = stage + row * 64 + (c ^ swizzle(row)) * 16;  // rows 8 apart have the same swizzle
    const bool valid = FAST || s * 4 + c < n_blk;
    src += (s * 4 + c) * 16;
#pragma unroll
    for (int i = 0; i < N; ++i) cp_async<16>(dst + i * 512, valid ? src + (int64_t)i * 8 * n_blk * 16 : src - c * 16, valid);
  }
  // Groups of one row; `at_row` is its first, `total` the number of groups of the matrix.
  __device__ static void fetch_groups(uint32_t stage, int row, const MoeWeight& w, int64_t at_row, int64_t total, int s) {
    const uint32_t dst = stage + kScales + row * 16;
    if constexpr (FAST) {
      cp_async<8>(dst, w.scale + at_row + s * 4);
      if (ASYM) cp_async<8>(dst + kRows * 16, w.zp + at_row + s * 4);
    } else {
      const int64_t word = (at_row + group_of(w, s * 4)) >> 1;
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const bool in = 2 * (word + i) < total;  // total is even: 32 rows to a multiple
        const int64_t at = in ? 2 * (word + i) : 0;
        cp_async<4>(dst + i * 4, w.scale + at, in);
        if (ASYM) cp_async<4>(dst + kRows * 16 + i * 4, w.zp + at, in);
      }
    }
  }
};

// The values of the four blocks of a step of one row.
struct GroupReader {
  uint32_t pick_lo, pick_hi, keep_lo, keep_hi;
  int shift;
  // p: 1 if the row's first group of the step is odd; the selectors are the same for every lane
  __device__ GroupReader(const MoeWeight& w, int s, int n_blk, int p) {
    shift = p * 16;
    if (w.group_blocks == 1) {
      pick_lo = pick_hi = 0;
    } else {
      const int first = group_of(w, s * 4);
      auto byte2 = [&](int j) { return group_of(w, s * 4 + j) != first ? 0x32u : 0x10u; };
      pick_lo = byte2(0) | byte2(1) << 8;
      pick_hi = byte2(2) | byte2(3) << 8;
    }
    const int left = n_blk - s * 4;  // blocks past the row's last have scale 0
    keep_lo = left >= 2 ? 0xffffffffu : 0x0000ffffu;
    keep_hi = left >= 4 ? 0xffffffffu : left >= 3 ? 0x0000ffffu : 0u;
  }
  __device__ uint2 operator()(const uint4& v) const {
    const uint32_t a = __funnelshift_r(v.x, v.y, shift), b = __funnelshift_r(v.y, v.z, shift);
    uint2 r = make_uint2(a, b);
    if (pick_lo) r = make_uint2(__byte_perm(a, a, pick_lo), __byte_perm(a, a, pick_hi));
    return make_uint2(r.x & keep_lo, r.y & keep_hi);
  }
};

// The value of this lane's block of set j.
template <int G>
__device__ __forceinline__ float group_value(const uint2& v, int j, int t) {
  if (G == 4) return __half2float(__ushort_as_half((unsigned short)((t & 2 ? v.y : v.x) >> ((t & 1) * 16))));
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
// Of one 32-block of two tokens: the powers of two f they were divided by and what to subtract from D for the
// magic and, for a symmetric weight, for z = 8: floats {f0, f1, c0, c1}; apart from them, {s2 of both}, the sums
// that a zero point multiplies.
// The power of two at or below a magnitude (1 for zero, subnormal, inf, NaN).
__device__ __forceinline__ float power_below(float top) {
  const uint32_t exponent = __float_as_uint(top) >> 23;
  return exponent == 0 || exponent == 255 ? 1.f : __uint_as_float(exponent << 23);
}

// From the sums of a block's stored values at k = 0, 2 mod 4 (`even`) and 1, 3 mod 4 (`odd`, divided by 16), to
// this token's place in fc = {f0, f1, c0, c1} and s2.
__device__ __forceinline__ void put_factors(float* fc, float* s2, float f, float even, float odd, bool asym) {
  const float sum = even + 16.f * odd, m = 1024.f * (even + odd);
  fc[0] = f;
  fc[2] = asym ? m : m + 8.f * sum;
  if (s2) *s2 = sum;
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
// mma.sync.m16n8k16 fp16; a plain (not volatile) asm, so that the compiler may interleave the tiles
__device__ __forceinline__ void mma_step(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool first) {
  if (first)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Adds one step to acc[tile][row g, g + 8] (two tokens each).  `stage` is the warp's ring stage; `operand` this
// lane's part of the first set in B order, BLOCK bytes from block to block (a lane off the diagonal: zeros);
// `factors` the Factors {f, c} of its two tokens and its block of the first set, FAC bytes from block to block,
// and `sums` their s2, SUM bytes from block to block.
template <int G, int R, bool ASYM, bool FAST, int BLOCK, int FAC, int SUM>
__device__ __forceinline__ void add_step(F2 (&acc)[R][2], const uint8_t* stage, const uint8_t* operand,
                                         const uint8_t* factors, const uint8_t* sums, int g, int t, int s, int n_blk,
                                         const MoeWeight& w) {
  using Rg = Ring<G, R, ASYM, FAST>;
  const int sw = Rg::swizzle(g);
  uint2 sc[R][2], zp[ASYM ? R : 1][2];
  {
    const int p = FAST ? 0 : (g * (n_blk / w.group_blocks) + group_of(w, s * 4)) & 1;
    const GroupReader reader(w, s, n_blk, p);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* at = stage + Rg::kScales + (i * 16 + h * 8 + g) * 16;
        if (FAST) {
          sc[i][h] = *reinterpret_cast<const uint2*>(at);
          if (ASYM) zp[ASYM ? i : 0][h] = *reinterpret_cast<const uint2*>(at + Rg::kRows * 16);
        } else {
          sc[i][h] = reader(*reinterpret_cast<const uint4*>(at));
          if (ASYM) zp[ASYM ? i : 0][h] = reader(*reinterpret_cast<const uint4*>(at + Rg::kRows * 16));
        }
      }
  }
#pragma unroll
  for (int j = 0; j < 4 / G; ++j) {
    // this lane's G words of the set: piece (block) j G + t / (4 / G) of the row, word t mod 4 / G times G
    const int piece = ((j * G + t / (4 / G)) ^ sw) * 16 + t % (4 / G) * (4 * G);
    uint32_t c[2 * R][G];
#pragma unroll
    for (int i = 0; i < 2 * R; ++i) {
      const uint8_t* at = stage + (i * 8 + g) * 64 + piece;
      if constexpr (G == 4) *reinterpret_cast<uint4*>(c[i]) = *reinterpret_cast<const uint4*>(at);
      else if constexpr (G == 2) *reinterpret_cast<uint2*>(c[i]) = *reinterpret_cast<const uint2*>(at);
      else c[i][0] = *reinterpret_cast<const uint32_t*>(at);
    }
    float d[R][4];
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(operand + j * G * BLOCK + i * 16);
#pragma unroll
      for (int q = 0; q < R; ++q) {
        uint32_t a[2][4];
        a_operands(c[2 * q][i], c[2 * q + 1][i], a);
        mma_step(d[q], a[0], v.x, v.y, i == 0);
        mma_step(d[q], a[1], v.z, v.w, false);
      }
    }
    const ulonglong2 fc = *reinterpret_cast<const ulonglong2*>(factors + j * G * FAC);
    const F2 f{fc.x}, m{fc.y};
    F2 s2{};
    if (ASYM) s2.v = *reinterpret_cast<const unsigned long long*>(sums + j * G * SUM);
#pragma unroll
    for (int q = 0; q < R; ++q)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float scale = group_value<G>(sc[q][h], j, t);
        F2 v = sub2(pack(d[q][2 * h], d[q][2 * h + 1]), m);
        if (ASYM) {
          const float z = -group_value<G>(zp[ASYM ? q : 0][h], j, t);
          v = fma2(pack(z, z), s2, v);
        }
        acc[q][h] = fma2(mul2(pack(scale, scale), f), v, acc[q][h]);
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

// Shared memory of kernel 1 behind the routing: tokens [NT][4 * steps] blocks of 64 bytes (neighbouring rows
// in the other half of the banks), their Factors, the partial products of two items, 256 bytes of zeros, the
// warps' rings.
struct UpLayout {
  int row, factors, sums, red, zeros, rings, bytes;
  __host__ __device__ UpLayout(int n_blk, int nt, bool asym, int stage_bytes, int stages) {
    const int blocks = (n_blk + 3) / 4 * 4;
    row = blocks * 64 + 64;
    factors = row * nt;
    sums = factors + nt / 2 * blocks * 16;
    red = sums + (asym ? nt / 2 * blocks * 8 : 0);
    zeros = red + 2 * kUpSlices * 2 * kUpRows * nt * 4;
    rings = zeros + 256;
    bytes = rings + kUpWarps * stages * stage_bytes;
  }
};

// Stores eight elements of a token (thread j of a row: elements 8 j ...) in the order of the mma operands, and
// their block's Factors; the lanes of a quad share a block.
template <typename T>
__device__ __forceinline__ void store_operand(const uint4& raw, uint4* to, float* fc, float* s2, bool write, bool asym) {
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
    if ((threadIdx.x & 3) == 0) put_factors(fc, s2, f, even, odd, asym);
  }
}

template <int G, bool ASYM, bool FAST>
__global__ void __launch_bounds__(kUpThreads, 1)
moe_up_kernel(const MoeParams p, const int stages) {
  constexpr int NT = 8 / G;
  using Rg = Ring<G, 2, ASYM, FAST>;
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ Routing r;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int n_blk = p.H / 32, n_steps = (n_blk + 3) / 4, blocks = n_steps * 4;
  const int n_group = n_blk / p.gate.group_blocks;
  const UpLayout at(n_blk, NT, ASYM, Rg::kBytes, stages);
  float* red = reinterpret_cast<float*>(dyn + at.red);  // [item parity][slice][gate, up][NT][32]
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
  const uint8_t* operand = dyn + (diag ? (g % NT) * at.row + lane_blk * 64 + t % (4 / G) * G * 16 : at.zeros);
  const int operand_step = diag ? 256 : 0;
  const int pair_blk = t % (4 / G) * blocks + lane_blk;
  const uint8_t *factors = dyn + at.factors + pair_blk * 16, *sums = dyn + at.sums + pair_blk * 8;

  // the warp's ring runs through its steps of all items
  const int ring = at.rings + warp * stages * Rg::kBytes;
  const int64_t total_groups = (int64_t)p.E * p.I * n_group;
  int f_item = first, f_s = s_first, f_stage = 0;
  auto fetch = [&] {
    if (f_item < last && s_first < s_last) {
      const int u = f_item / tiles;
      const int64_t row0 = (int64_t)r.unit_expert[u] * p.I + (f_item - u * tiles) * kUpRows + mt * 16;
      const uint32_t stage = base + ring + f_stage * Rg::kBytes;
      const int64_t code_row = (row0 + g) * n_blk * 16;
      Rg::template fetch_codes<2>(stage, 0, p.gate.codes + code_row, f_s, n_blk, lane);
      Rg::template fetch_codes<2>(stage, 16, p.up.codes + code_row, f_s, n_blk, lane);
      Rg::fetch_groups(stage, lane, lane < 16 ? p.gate : p.up, (row0 + (lane & 15)) * n_group, total_groups, f_s);
      if (++f_s == s_last) { f_s = s_first; ++f_item; }
      if (++f_stage == stages) f_stage = 0;
    }
    cp_async_commit();
  };
  for (int i = 0; i < stages; ++i) fetch();

  int unit = -1, n = 0, stage = 0;
  for (int item = first; item < last; ++item) {
    const int u = item / tiles, i0 = (item - u * tiles) * kUpRows;
    const int e = r.unit_expert[u];
    if (u != unit) {
      if (unit >= 0) __syncthreads();  // everybody is through with the unit before
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
          const int pb = i / 2 * blocks + (j >> 2);
          float* fc = reinterpret_cast<float*>(dyn + at.factors) + pb * 4 + (i & 1);
          float* s2 = ASYM ? reinterpret_cast<float*>(dyn + at.sums) + pb * 2 + (i & 1) : nullptr;
          if (p.dtype == NPB_BF16) store_operand<__nv_bfloat16>(raw, to, fc, s2, j < blocks * 4, ASYM);
          else store_operand<__half>(raw, to, fc, s2, j < blocks * 4, ASYM);
        }
      }
      __syncthreads();
    }
    F2 acc[2][2] = {};
    for (int s = s_first; s < s_last; ++s) {
      cp_async_wait(stages - 1);
      __syncwarp();
      add_step<G, 2, ASYM, FAST, 64, 16, 8>(acc, dyn + ring + stage * Rg::kBytes, operand + s * operand_step,
                                            factors + s * 64, sums + s * 32, g, t, s, n_blk, p.gate);
      __syncwarp();
      fetch();
      if (++stage == stages) stage = 0;
    }
    // the blocks of a set, then the slices of K
    float* part = red + ((item & 1) * kUpSlices + ks) * 2 * NT * kUpRows;
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[2];
        unpack(acc[w][h], v[0], v[1]);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float q = block_sum<G>(v[c]);
          if (t < 4 / G) part[(w * NT + 2 * t + c) * kUpRows + mt * 16 + g + h * 8] = q;
        }
      }
    __syncthreads();
    if (warp < n) {  // a warp per token, a lane per row
      float gate = 0.f, up = 0.f;
#pragma unroll
      for (int k = 0; k < kUpSlices; ++k) {
        const float* from = red + (((item & 1) * kUpSlices + k) * 2 * NT + warp) * kUpRows + lane;
        gate += from[0];
        up += from[NT * kUpRows];
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
      if (lane == 0) {
        float* to = reinterpret_cast<float*>(rec + 128) + (warp & 1);
        put_factors(to, to + 4, f, even, odd, p.down.zp != nullptr);
      }
    }
    // the next item writes the other half of `red`, the one after it only behind the next barrier
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// ---- kernel 2: down product and the sum over experts ----------------------------------------------
constexpr int kDownThreads = 256;
constexpr int kDownWarps = kDownThreads / 32;
constexpr int kDownTiles = 4;                 // 16-row tiles per warp: h is brought once for all of them
constexpr int kDownRows = 16 * kDownTiles;    // output rows per cluster
constexpr int kDownSplit = 4;                 // CTAs of a cluster: each takes a share of the (unit, step) sequence

// Shared memory of kernel 2 behind the routing: per warp the partial sums [T][64] and a ring of steps, each followed
// by h records [NT / 2][4]; then zeros that cover the reach of a step's operands.
struct DownLayout {
  int sums, stage, warp, zeros, bytes;
  __host__ __device__ DownLayout(int T, int nt, int stage_bytes, int stages) {
    sums = T * kDownRows * 4;
    stage = stage_bytes + nt / 2 * 4 * kRecord;
    warp = sums + stages * stage;
    zeros = warp * kDownWarps;
    bytes = zeros + 4 * kRecord;
  }
};

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

template <int G, bool ASYM, bool FAST>
__global__ void __cluster_dims__(kDownSplit, 1, 1) __launch_bounds__(kDownThreads, G == 1 ? 1 : 2)
moe_down_kernel(const MoeParams p, const int stages) {
  constexpr int NT = 8 / G;
  using Rg = Ring<G, kDownTiles, ASYM, FAST>;
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ Routing r;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int n_blk = p.I / 32, n_steps = (n_blk + 3) / 4, n_group = n_blk / p.down.group_blocks;
  const int rank = (int)sm100::cluster_ctarank();
  const int j0 = blockIdx.x / kDownSplit * kDownRows;
  const int rows_left = min(kDownRows, p.H - j0);  // 32 in the last cluster of an odd H / 32
  const DownLayout at(p.T, NT, Rg::kBytes, stages);
  const uint32_t base = sm100::smem_u32(dyn);
  float* sums = reinterpret_cast<float*>(dyn + warp * at.warp);  // [T][64]
  for (int i = lane; i < p.T * kDownRows; i += 32) sums[i] = 0.f;
  for (int i = tid; i < kRecord; i += kDownThreads) reinterpret_cast<uint32_t*>(dyn + at.zeros)[i] = 0;
  route<NT>(p, r);

  // (unit, step) pairs in a row, an equal share of consecutive ones per warp of the cluster
  const int64_t total = (int64_t)r.n_units * n_steps;
  const int share = rank * kDownWarps + warp, shares = kDownSplit * kDownWarps;
  const int first = (int)(total * share / shares), last = (int)(total * (share + 1) / shares);
  const int lane_blk = t / (4 / G);
  const bool diag = g / NT == lane_blk;
  const int ring = warp * at.warp + at.sums;
  const uint8_t* operand = dyn + (diag ? ring + Rg::kBytes + (g % NT / 2 * 4 + lane_blk) * kRecord + (g & 1) * 64 +
                                             t % (4 / G) * G * 16
                                       : at.zeros);
  const int operand_stage = diag ? at.stage : 0;
  const uint8_t* factors = dyn + ring + Rg::kBytes + (t % (4 / G) * 4 + lane_blk) * kRecord + 128;

  const int64_t total_groups = (int64_t)p.E * p.H * n_group;
  int f_at = first, f_u = first / n_steps, f_s = first - f_u * n_steps, f_stage = 0;
  auto fetch_weights = [&] {
    const int64_t row0 = (int64_t)r.unit_expert[f_u] * p.H + j0;
    const uint32_t to = base + ring + f_stage * at.stage;
    Rg::template fetch_codes<4>(to, 0, p.down.codes + (row0 + g) * n_blk * 16, f_s, n_blk, lane);
    if (rows_left == kDownRows)
      Rg::template fetch_codes<4>(to, 32, p.down.codes + (row0 + 32 + g) * n_blk * 16, f_s, n_blk, lane);
#pragma unroll
    for (int i = 0; i < kDownRows; i += 32)
      if (i < rows_left) Rg::fetch_groups(to, i + lane, p.down, (row0 + i + lane) * n_group, total_groups, f_s);
  };
  auto fetch_records = [&] {  // blocks 4 f_s .. + 4 of the unit's tokens; zeros past n_blk
    constexpr int kPieces = kRecord / 16;
    const uint8_t* rec = p.h + ((int64_t)r.unit_slot[f_u] * n_blk + f_s * 4) * kRecord;
    const int pieces = (__popc(r.unit_mask[f_u]) + 1) / 2 * 4 * kPieces;
    const uint32_t to = base + ring + f_stage * at.stage + Rg::kBytes;
#pragma unroll
    for (int c0 = 0; c0 < NT / 2 * 4 * kPieces; c0 += 32) {
      const int c = c0 + lane, pair = c / (4 * kPieces), rest = c - pair * 4 * kPieces;
      const bool valid = f_s * 4 + rest / kPieces < n_blk;
      if (c < pieces) cp_async<16>(to + c * 16, valid ? rec + (int64_t)pair * n_blk * kRecord + rest * 16 : p.h, valid);
    }
  };
  auto advance = [&] {
    cp_async_commit();
    if (f_at < last) {
      ++f_at;
      if (++f_s == n_steps) { f_s = 0; ++f_u; }
      if (++f_stage == stages) f_stage = 0;
    }
  };

  F2 acc[kDownTiles][2] = {};
  int unit = -1;
  auto flush = [&] {
    uint32_t m = unit >= 0 ? r.unit_mask[unit] : 0u;
    for (int i = 0; i < 2 * t; ++i) m &= m - 1;  // of this lane's two tokens
    const int token[2] = {__ffs(m) - 1, __ffs(m & (m - 1)) - 1};
#pragma unroll
    for (int w = 0; w < kDownTiles; ++w)
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

  // the first weights are under way before kernel 1 ends; h exists only after it
  const int f0 = f_at, u0 = f_u, s0 = f_s;
  for (int i = 0; i < stages; ++i) {
    if (f_at < last) fetch_weights();
    advance();
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  f_at = f0;
  f_u = u0;
  f_s = s0;
  f_stage = 0;
  for (int i = 0; i < stages; ++i) {
    if (f_at < last) fetch_records();
    advance();
  }
  int c_u = first / n_steps, c_s = first - c_u * n_steps, stage = 0;
  for (int q = first; q < last; ++q) {
    if (c_u != unit) {
      flush();
      unit = c_u;
    }
    cp_async_wait(stages - 1);
    __syncwarp();
    const uint8_t* f = factors + stage * at.stage;
    add_step<G, kDownTiles, ASYM, FAST, kRecord, kRecord, kRecord>(acc, dyn + ring + stage * at.stage,
                                                                   operand + stage * operand_stage, f, f + 16, g, t, c_s,
                                                                   n_blk, p.down);
    __syncwarp();
    if (f_at < last) {
      fetch_weights();
      fetch_records();
    }
    advance();
    if (++c_s == n_steps) { c_s = 0; ++c_u; }
    if (++stage == stages) stage = 0;
  }
  flush();
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  // the warps of the CTA (into warp 0's sums), then the CTAs of the cluster: each finishes a quarter of the rows
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
    if (row >= rows_left) continue;
    const int64_t to = (int64_t)token * p.H + j0 + row;
    if (p.dtype == NPB_BF16) static_cast<__nv_bfloat16*>(p.y)[to] = from_f32<__nv_bfloat16>(v);
    else static_cast<__half*>(p.y)[to] = from_f32<__half>(v);
  }
  __syncwarp();
  sm100::cluster_sync_all();  // nobody leaves while its sums are read
}

// ---- host ----------------------------------------------------------------------------------------
// One group per block, rows of whole steps, eight-byte words of groups.
bool is_fast(const MoeWeight& w, int n_blk) {
  return n_blk % 4 == 0 && w.group_blocks == 1 && aligned_to(w.scale, 8) && aligned_to(w.zp, 8);
}

constexpr int kMaxStages = 4;

// Ring stages that fit next to the rest (2..4; 0: not even two do).
template <typename Bytes>
int pick_stages(Bytes bytes, int ctas_per_sm) {
  const int cap = ctas_per_sm == 1 ? max_dynamic_smem() : (max_dynamic_smem() - 1024) / ctas_per_sm - 1024;
  int stages = kMaxStages;
  while (stages >= 2 && bytes(stages) + (int)sizeof(Routing) + 64 > cap) --stages;
  return stages >= 2 ? stages : 0;
}

template <int G, bool ASYM, bool FAST>
int up_stages(const MoeParams& p) {
  return pick_stages([&](int n) { return UpLayout(p.H / 32, 8 / G, ASYM, Ring<G, 2, ASYM, FAST>::kBytes, n).bytes; }, 1);
}

template <int G, bool ASYM, bool FAST>
int launch_up(const MoeParams& p, cudaStream_t st) {
  auto kern = moe_up_kernel<G, ASYM, FAST>;
  const int stages = up_stages<G, ASYM, FAST>(p);
  if (stages == 0) return NPB_ERR_TOO_LARGE;
  const size_t smem = UpLayout(p.H / 32, 8 / G, ASYM, Ring<G, 2, ASYM, FAST>::kBytes, stages).bytes;
  int per_sm = 0;
  if (int rc = blocks_per_sm(reinterpret_cast<const void*>(kern), kUpThreads, smem, &per_sm)) return rc;
  if (per_sm < 1) return NPB_ERR_TOO_LARGE;
  const int64_t active = p.T * p.top_k < p.E ? p.T * p.top_k : p.E;
  const int64_t most = active * (p.I / kUpRows), slots = (int64_t)sm_count() * per_sm;
  kern<<<(unsigned)(most < slots ? most : slots), kUpThreads, smem, st>>>(p, stages);
  NPB_LAUNCH_CHECK();
  return NPB_OK;
}

template <int G, bool ASYM, bool FAST>
int launch_down(const MoeParams& p, cudaStream_t st) {
  auto kern = moe_down_kernel<G, ASYM, FAST>;
  auto bytes = [&](int n) { return DownLayout(p.T, 8 / G, Ring<G, kDownTiles, ASYM, FAST>::kBytes, n).bytes; };
  int stages = pick_stages(bytes, 2);
  if (stages == 0) stages = pick_stages(bytes, 1);
  if (stages == 0) return NPB_ERR_TOO_LARGE;
  int per_sm = 0;
  if (int rc = blocks_per_sm(reinterpret_cast<const void*>(kern), kDownThreads, bytes(stages), &per_sm)) return rc;
  if (per_sm < 1) return NPB_ERR_TOO_LARGE;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((p.H + kDownRows - 1) / kDownRows * kDownSplit));
  cfg.blockDim = dim3(kDownThreads);
  cfg.dynamicSmemBytes = bytes(stages);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  NPB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p, stages));
  NPB_LAUNCH_CHECK();
  return NPB_OK;
}

template <int G>
int launch(const MoeParams& p, cudaStream_t st) {
  const bool fast_up = is_fast(p.gate, p.H / 32) && is_fast(p.up, p.H / 32), fast_down = is_fast(p.down, p.I / 32);
  int rc;
  if (p.gate.zp) rc = fast_up ? launch_up<G, true, true>(p, st) : launch_up<G, true, false>(p, st);
  else rc = fast_up ? launch_up<G, false, true>(p, st) : launch_up<G, false, false>(p, st);
  if (rc) return rc;
  if (p.down.zp) return fast_down ? launch_down<G, true, true>(p, st) : launch_down<G, true, false>(p, st);
  return fast_down ? launch_down<G, false, true>(p, st) : launch_down<G, false, false>(p, st);
}

int launch_tokens(const MoeParams& p, cudaStream_t st) {
  // an expert has at most T tokens; a unit's tokens have to fit the shared memory of kernel 1 (ASYM's larger ring)
  if (p.T > 4 && up_stages<1, true, false>(p)) return launch<1>(p, st);
  if (p.T > 2 && up_stages<2, true, false>(p)) return launch<2>(p, st);
  return launch<4>(p, st);
}

int make_weight(const npb_q_weight* w, int64_t N, int64_t K, MoeWeight* out) {
  if (int rc = validate_q(w, N, K)) return rc;
  if (w->nbits != 4 || w->group_size % 32 != 0) return NPB_ERR_UNSUPPORTED;
  if (!aligned_to(w->codes, 16) || !aligned_to(w->scale, 4) || !aligned_to(w->zero_point, 4)) return NPB_ERR_ALIGNMENT;
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
