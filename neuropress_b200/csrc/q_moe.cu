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
// Product: mma.sync.m16n8k16 with the weights as the A operand (16 rows) built in registers: a code q is
// the float (magic + q) with one bit operation per two codes (magic 128 in bf16, 1024 in fp16), and
//   sum_k (q - z) x = sum_k (magic + q) x - (magic + z) sum_k x
// is applied per 32-wide block with its scale, in fp32.  Lane (g, t) of a warp loads 16 bytes = one
// whole 32-block of rows g and g + 8 (64 contiguous bytes per row and quad), i.e. the four lanes of a
// quad bring four different blocks to the k slots of an mma.  The B operand keeps them apart: it is
// block-diagonal, column 2 t + c holds block t of token c, so lane (g, t) of the result holds exactly
// the block whose scale it loaded.  An mma thus serves 256 weights for two columns: two tokens in
// kernel 1, and the high and the low bf16 half of one token's h in kernel 2 -- h keeps 16
// significant bits, which leaves the output's own rounding as the only one that shows.
//
// An expert's tokens are taken in units of up to NT; an expert with more tokens is read again (from L2).
// Every sum has a fixed order: results do not depend on scheduling.
#include <type_traits>

#include "common.cuh"
#include "mma_sync.cuh"
#include "order_key.cuh"

namespace npb {
namespace {

constexpr int kMaxTokens = 32;   // bits of an expert's token mask
constexpr int kMaxExperts = 512;
constexpr int kMaxTopK = 16;
constexpr int kMaxUnits = kMaxTokens * kMaxTopK;

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
  int logits_dtype;
  int T, E, H, I, top_k, renormalize;
  MoeWeight gate, up, down;
  uint16_t* h;     // [T * top_k][I / 32][2][32] bf16 bits: high and low half, in mma order
  float* h_sum;    // [T * top_k][I / 32]
  void* y;
};

// ---- routing ---------------------------------------------------------------------------------
struct Routing {
  uint32_t mask[kMaxExperts];            // tokens of each expert
  float weight[kMaxTokens][kMaxTopK];
  uint16_t id[kMaxTokens][kMaxTopK];     // 0xffff: none
  uint16_t unit_expert[kMaxUnits];
  uint8_t unit_first[kMaxUnits];         // rank of the unit's first token among the expert's
  uint16_t unit_slot[kMaxUnits];         // row of h of the unit's first token
  int n_units;
};

__device__ __forceinline__ float load_logit(const MoeParams& p, int64_t i) {
  if (p.logits_dtype == NPB_F32) return __ldg(static_cast<const float*>(p.logits) + i);
  if (p.logits_dtype == NPB_BF16) return to_f32(static_cast<const __nv_bfloat16*>(p.logits)[i]);
  return to_f32(static_cast<const __half*>(p.logits)[i]);
}

// All threads of the CTA; ends with a barrier.  A unit is up to NT tokens of one expert.
template <int NT>
__device__ void route(const MoeParams& p, Routing& r) {
  constexpr int PER_LANE = kMaxExperts / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) r.mask[e] = 0;
  __syncthreads();
  for (int t = warp; t < p.T; t += warps) {
    uint32_t key[PER_LANE];
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) {
      key[i] = 0;
      if (i * 32 < p.E && i * 32 + lane < p.E) {
        const float l = load_logit(p, (int64_t)t * p.E + i * 32 + lane);
        key[i] = order_key(l);
        m = fmaxf(m, l);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
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
        if (i * 32 < p.E && key[i] > best) { best = key[i]; at = i; }
      const uint32_t top = __reduce_max_sync(0xffffffffu, best);
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
  __syncthreads();
  if (warp == 0) {
    int units = 0, slots = 0;
    for (int base = 0; base < p.E; base += 32) {
      const int e = base + lane;
      const int n = e < p.E ? __popc(r.mask[e]) : 0;
      const int u = (n + NT - 1) / NT;
      int iu = u, in = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, iu, o), b = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) { iu += a; in += b; }
      }
      for (int i = 0; i < u; ++i) {
        const int at = units + iu - u + i;
        r.unit_expert[at] = (uint16_t)e;
        r.unit_first[at] = (uint8_t)(i * NT);
        r.unit_slot[at] = (uint16_t)(slots + in - n + i * NT);
      }
      units += __shfl_sync(0xffffffffu, iu, 31);
      slots += __shfl_sync(0xffffffffu, in, 31);
    }
    if (lane == 0) r.n_units = units;
  }
  __syncthreads();
}

// Tokens of a unit: count, and the tokens themselves (those past the count repeat the last).
template <int NT>
__device__ __forceinline__ int unit_tokens(const Routing& r, int u, int (&tok)[NT]) {
  uint32_t m = r.mask[r.unit_expert[u]];
  for (int i = r.unit_first[u]; i > 0; --i) m &= m - 1;
  const int n = min(NT, __popc(m));
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    tok[i] = __ffs(m) - 1;
    if (m & (m - 1)) m &= m - 1;
  }
  return n;
}

// ---- weights ---------------------------------------------------------------------------------
__device__ __forceinline__ uint4 ld_stream(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// Codes, scales and zero points of R rows for one 32-block.
template <int R, bool ASYM>
struct Blocks {
  uint4 c[R];
  __half s[R];
  __half z[ASYM ? R : 1];
};

__device__ __forceinline__ int group_of(const MoeWeight& w, int blk) {
  return w.group_shift >= 0 ? blk >> w.group_shift : blk / w.group_blocks;
}

template <int R, bool ASYM>
__device__ __forceinline__ void fetch_row(Blocks<R, ASYM>& b, int i, const MoeWeight& w, int64_t row, int n_blk, int blk,
                                          bool valid) {
  if (valid) {
    b.c[i] = ld_stream(w.codes + (row * n_blk + blk) * 16);
    const int64_t g = row * (n_blk / w.group_blocks) + group_of(w, blk);
    b.s[i] = __ldg(w.scale + g);
    if (ASYM) b.z[ASYM ? i : 0] = __ldg(w.zp + g);
  } else {
    b.c[i] = make_uint4(0, 0, 0, 0);
    b.s[i] = __ushort_as_half(0);
    if (ASYM) b.z[ASYM ? i : 0] = __ushort_as_half(0);
  }
}

// Codes j and j + 4 of a word as two floats (magic + q) of type T.
template <typename T>
__device__ __forceinline__ uint32_t code_pair(uint32_t word, int j) {
  constexpr uint32_t magic = std::is_same<T, __half>::value ? 0x64006400u : 0x43004300u;
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(word >> (4 * j)), "r"(0x000f000fu), "r"(magic));
  return r;
}
template <typename T>
constexpr float magic_of() { return std::is_same<T, __half>::value ? 1024.f : 128.f; }

__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// The A operands of word i of rows (lo, hi): two mmas of 16 k slots each.
template <typename T>
__device__ __forceinline__ void a_operands(const uint4& lo, const uint4& hi, int i, uint32_t (&a0)[4],
                                           uint32_t (&a1)[4]) {
  const uint32_t l = word_of(lo, i), h = word_of(hi, i);
  a0[0] = code_pair<T>(l, 0); a0[1] = code_pair<T>(h, 0); a0[2] = code_pair<T>(l, 1); a0[3] = code_pair<T>(h, 1);
  a1[0] = code_pair<T>(l, 2); a1[1] = code_pair<T>(h, 2); a1[2] = code_pair<T>(l, 3); a1[3] = code_pair<T>(h, 3);
}

// ---- kernel 1: gate / up products, silu, routing weight ------------------------------------------
constexpr int kUpThreads = 256;  // two 16-row tiles x four slices of K
constexpr int kUpRows = 32;      // rows of gate and of up per item: one 32-block of h
constexpr int kUpSlices = 4;

template <typename T, int NT, bool ASYM>
__global__ void __launch_bounds__(kUpThreads, 2)
moe_up_kernel(const MoeParams p) {
  constexpr int NP = NT / 2;  // pairs of tokens
  extern __shared__ float dyn[];
  __shared__ Routing r;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const T* x = static_cast<const T*>(p.x);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int n_blk = p.H / 32, n_steps = (n_blk + 3) / 4;
  float* x_sum = dyn;                                  // [T][n_blk]
  float* red = dyn + (p.T * n_blk + 3) / 4 * 4;        // [slice][tile][matrix][NT][16]

  for (int i = tid; i < p.T * n_blk; i += kUpThreads) {
    const uint4* q = reinterpret_cast<const uint4*>(x + (int64_t)i * 32);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint4 v = __ldg(q + j);
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int k = 0; k < 8; ++k) s += to_f32(e[k]);
    }
    x_sum[i] = s;
  }
  route<NT>(p, r);

  const int tiles = p.I / kUpRows, items = tiles * r.n_units;
  const int mt = warp & 1, ks = warp >> 1;
  const int s_first = n_steps * ks / kUpSlices, s_last = n_steps * (ks + 1) / kUpSlices;
  const bool diag = (lane >> 3) == t;  // this lane holds the nonzero part of column lane / 4
  const int column = (lane >> 2) & 1;  // token of the pair in that column

  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int u = item % r.n_units, i0 = item / r.n_units * kUpRows;
    const int e = r.unit_expert[u];
    int tok[NT];
    const int n = unit_tokens<NT>(r, u, tok);
    const int64_t row = (int64_t)e * p.I + i0 + mt * 16 + g;
    const T* xp[NP];
    bool has[NP];
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      has[q] = diag && 2 * q + column < n;
      xp[q] = x + (int64_t)(column ? tok[2 * q + 1] : tok[2 * q]) * p.H;
    }
    float acc[2][NP][4] = {};
    using B = Blocks<4, ASYM>;
    auto fetch = [&](B& b, int s) {
      const int blk = s * 4 + t;
      const bool valid = s < s_last && blk < n_blk;
      fetch_row(b, 0, p.gate, row, n_blk, blk, valid);
      fetch_row(b, 1, p.gate, row + 8, n_blk, blk, valid);
      fetch_row(b, 2, p.up, row, n_blk, blk, valid);
      fetch_row(b, 3, p.up, row + 8, n_blk, blk, valid);
    };
    auto compute = [&](const B& b, int s) {
      const int blk = s * 4 + t;
      const bool valid = blk < n_blk;
      float d[2][NP][4] = {};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t a[2][2][4];
        a_operands<T>(b.c[0], b.c[1], i, a[0][0], a[0][1]);
        a_operands<T>(b.c[2], b.c[3], i, a[1][0], a[1][1]);
#pragma unroll
        for (int q = 0; q < NP; ++q) {
          if (2 * q < n) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (has[q] && valid) v = __ldg(reinterpret_cast<const uint4*>(xp[q] + blk * 32 + i * 8));
            // k slots in the order of the code pairs: (0, 4) (1, 5) and (2, 6) (3, 7)
            const uint32_t b0 = __byte_perm(v.x, v.z, 0x5410), b1 = __byte_perm(v.x, v.z, 0x7632);
            const uint32_t b2 = __byte_perm(v.y, v.w, 0x5410), b3 = __byte_perm(v.y, v.w, 0x7632);
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              mma16816<T>(d[w][q], a[w][0], b0, b1);
              mma16816<T>(d[w][q], a[w][1], b2, b3);
            }
          }
        }
      }
#pragma unroll
      for (int q = 0; q < NP; ++q) {
        if (2 * q < n) {
          const float s0 = valid ? x_sum[tok[2 * q] * n_blk + blk] : 0.f;
          const float s1 = valid ? x_sum[tok[2 * q + 1] * n_blk + blk] : 0.f;
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float sc = __half2float(b.s[2 * w + h]);
              const float mz = magic_of<T>() + (ASYM ? __half2float(b.z[ASYM ? 2 * w + h : 0]) : 8.f);
              acc[w][q][2 * h] = fmaf(sc, fmaf(-mz, s0, d[w][q][2 * h]), acc[w][q][2 * h]);
              acc[w][q][2 * h + 1] = fmaf(sc, fmaf(-mz, s1, d[w][q][2 * h + 1]), acc[w][q][2 * h + 1]);
            }
        }
      }
    };
    B b0, b1;
    fetch(b0, s_first);
    for (int s = s_first; s < s_last; s += 2) {
      fetch(b1, s + 1);
      compute(b0, s);
      fetch(b0, s + 2);
      if (s + 1 < s_last) compute(b1, s + 1);
    }
    // the four blocks of a quad, then the slices of K
    float* mine = red + (ks * 2 + mt) * 2 * NT * 16;
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v = acc[w][q][c];
          v += __shfl_xor_sync(0xffffffffu, v, 1);
          v += __shfl_xor_sync(0xffffffffu, v, 2);
          if (t == 0) mine[(w * NT + 2 * q + (c & 1)) * 16 + g + (c >> 1) * 8] = v;
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
      int token = tok[0];
#pragma unroll
      for (int i = 1; i < NT; ++i) token = warp == i ? tok[i] : token;
      float weight = 0.f;
      for (int j = 0; j < p.top_k; ++j)
        if (r.id[token][j] == e) weight = r.weight[token][j];
      const float h = weight * (gate / (1.f + expf(-gate)) * up);
      const __nv_bfloat16 hi = __float2bfloat16_rn(h);
      float rest = h - __bfloat162float(hi);
      if (isinf(__bfloat162float(hi))) rest = 0.f;
      const __nv_bfloat16 lo = __float2bfloat16_rn(rest);
      const float sum = warp_sum(__bfloat162float(hi) + __bfloat162float(lo));
      const int64_t at = (int64_t)(r.unit_slot[u] + warp) * (p.I / 32) + i0 / 32;
      uint16_t* dst = p.h + at * 64 + (lane & 24) + (lane & 3) * 2 + ((lane >> 2) & 1);
      dst[0] = __bfloat16_as_ushort(hi);
      dst[32] = __bfloat16_as_ushort(lo);
      if (lane == 0) p.h_sum[at] = sum;
    }
    __syncthreads();
  }
}

// ---- kernel 2: down product and the sum over experts ----------------------------------------------
constexpr int kDownThreads = 512;
constexpr int kDownWarps = kDownThreads / 32;

template <typename T, int NT, bool ASYM>
__global__ void __launch_bounds__(kDownThreads, 1)
moe_down_kernel(const MoeParams p) {
  extern __shared__ float dyn[];  // [warp][T][16]
  __shared__ Routing r;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int n_blk = p.I / 32, n_steps = (n_blk + 3) / 4;
  const int j0 = blockIdx.x * 16;
  float* mine = dyn + warp * p.T * 16;
  for (int i = tid; i < kDownWarps * p.T * 16; i += kDownThreads) dyn[i] = 0.f;
  route<NT>(p, r);

  // (unit, step) pairs in a row, an equal share of consecutive ones per warp
  const int total = r.n_units * n_steps;
  const int first = (int)((int64_t)total * warp / kDownWarps), last = (int)((int64_t)total * (warp + 1) / kDownWarps);
  const bool diag = (lane >> 3) == t;
  const int half = (lane >> 2) & 1;  // 0: the high, 1: the low half of h
  using B = Blocks<2, ASYM>;
  auto fetch = [&](B& b, int q) {
    const int u = q < last ? q / n_steps : 0, blk = (q - u * n_steps) * 4 + t;
    const bool valid = q < last && blk < n_blk;
    const int64_t row = valid ? (int64_t)r.unit_expert[u] * p.H + j0 + g : 0;
    fetch_row(b, 0, p.down, row, n_blk, blk, valid);
    fetch_row(b, 1, p.down, row + 8, n_blk, blk, valid);
  };
  float acc[NT][2] = {};
  int unit = -1, n = 0, tok[NT];
  int64_t slot = 0;
  auto flush = [&] {
#pragma unroll
    for (int i = 0; i < NT; ++i)
      if (i < n) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v = acc[i][h];
          v += __shfl_xor_sync(0xffffffffu, v, 1);
          v += __shfl_xor_sync(0xffffffffu, v, 2);
          if (t == 0) mine[tok[i] * 16 + g + 8 * h] += v;
          acc[i][h] = 0.f;
        }
      }
    __syncwarp();
  };
  auto compute = [&](const B& b, int q) {
    const int u = q / n_steps, blk = (q - u * n_steps) * 4 + t;
    if (u != unit) {
      if (unit >= 0) flush();
      unit = u;
      n = unit_tokens<NT>(r, u, tok);
      slot = r.unit_slot[u];
    }
    const bool valid = blk < n_blk;
    float d[NT][4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t a0[4], a1[4];
      a_operands<__nv_bfloat16>(b.c[0], b.c[1], i, a0, a1);
#pragma unroll
      for (int c = 0; c < NT; ++c)
        if (c < n) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (diag && valid)
            v = *reinterpret_cast<const uint4*>(p.h + (((slot + c) * n_blk + blk) * 2 + half) * 32 + i * 8);
          mma16816<__nv_bfloat16>(d[c], a0, v.x, v.y);
          mma16816<__nv_bfloat16>(d[c], a1, v.z, v.w);
        }
    }
#pragma unroll
    for (int c = 0; c < NT; ++c)
      if (c < n) {
        const float s = valid ? p.h_sum[(slot + c) * n_blk + blk] : 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float mz = magic_of<__nv_bfloat16>() + (ASYM ? __half2float(b.z[ASYM ? h : 0]) : 8.f);
          acc[c][h] = fmaf(__half2float(b.s[h]), fmaf(-mz, s, d[c][2 * h] + d[c][2 * h + 1]), acc[c][h]);
        }
      }
  };
  constexpr int DEPTH = 4;
  B b[DEPTH];
#pragma unroll
  for (int i = 0; i < DEPTH; ++i) fetch(b[i], first + i);
  asm volatile("griddepcontrol.wait;" ::: "memory");  // h is written
  for (int q = first; q < last; q += DEPTH) {
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) {
      if (q + i < last) compute(b[i], q + i);
      fetch(b[i], q + i + DEPTH);
    }
  }
  if (unit >= 0) flush();
  __syncthreads();
  T* y = static_cast<T*>(p.y);
  for (int i = tid; i < p.T * 16; i += kDownThreads) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kDownWarps; ++w) v += dyn[w * p.T * 16 + i];
    y[(int64_t)(i >> 4) * p.H + j0 + (i & 15)] = from_f32<T>(v);
  }
}

// ---- host ----------------------------------------------------------------------------------------
template <typename T, int NT, bool ASYM>
int launch_up(const MoeParams& p, cudaStream_t st) {
  auto kern = moe_up_kernel<T, NT, ASYM>;
  const size_t smem = ((size_t)(p.T * (p.H / 32) + 3) / 4 * 4 + kUpSlices * 2 * 2 * NT * 16) * sizeof(float);
  int per_sm = 0;
  if (int rc = blocks_per_sm(reinterpret_cast<const void*>(kern), kUpThreads, smem, &per_sm)) return rc;
  if (per_sm < 1) return NPB_ERR_TOO_LARGE;
  const int64_t active = p.T * p.top_k < p.E ? p.T * p.top_k : p.E;
  const int64_t most = active * (p.I / kUpRows), slots = (int64_t)sm_count() * per_sm;
  kern<<<(unsigned)(most < slots ? most : slots), kUpThreads, smem, st>>>(p);
  NPB_LAUNCH_CHECK();
  return NPB_OK;
}

template <typename T, int NT, bool ASYM>
int launch_down(const MoeParams& p, cudaStream_t st) {
  auto kern = moe_down_kernel<T, NT, ASYM>;
  const size_t smem = (size_t)kDownWarps * p.T * 16 * sizeof(float);
  int per_sm = 0;
  if (int rc = blocks_per_sm(reinterpret_cast<const void*>(kern), kDownThreads, smem, &per_sm)) return rc;
  if (per_sm < 1) return NPB_ERR_TOO_LARGE;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.H / 16));
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

template <typename T, int NT>
int launch(const MoeParams& p, cudaStream_t st) {
  if (int rc = p.gate.zp ? launch_up<T, NT, true>(p, st) : launch_up<T, NT, false>(p, st)) return rc;
  return p.down.zp ? launch_down<T, NT, true>(p, st) : launch_down<T, NT, false>(p, st);
}

template <typename T>
int launch_tokens(const MoeParams& p, cudaStream_t st) {
  // an expert has at most T tokens; eight per unit is what the registers of kernel 1 hold
  if (p.T <= 2) return launch<T, 2>(p, st);
  if (p.T <= 4) return launch<T, 4>(p, st);
  return launch<T, 8>(p, st);
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
  return T * top_k * (I * 4 + I / 32 * 4);
}

int q_moe(const void* x, int dtype, const void* logits, int logits_dtype, int64_t T, int64_t E, int64_t H, int64_t I,
          const npb_q_weight* gate, const npb_q_weight* up, const npb_q_weight* down, int top_k, int renormalize,
          void* workspace, int64_t workspace_bytes, void* y, cudaStream_t st) {
  if (T < 0 || E <= 0 || H <= 0 || I <= 0 || top_k <= 0 || top_k > E) return NPB_ERR_INVALID_ARG;
  if (gate == nullptr || up == nullptr || down == nullptr) return NPB_ERR_INVALID_ARG;
  if (dtype != NPB_BF16 && dtype != NPB_F16) return NPB_ERR_UNSUPPORTED;
  if (logits_dtype != NPB_BF16 && logits_dtype != NPB_F16 && logits_dtype != NPB_F32) return NPB_ERR_UNSUPPORTED;
  if (T > kMaxTokens || E > kMaxExperts || top_k > kMaxTopK || H >= 1 << 20 || I >= 1 << 20) return NPB_ERR_UNSUPPORTED;
  if (H % 32 != 0 || I % 32 != 0) return NPB_ERR_SHAPE;
  MoeParams p{};
  if (int rc = make_weight(gate, E * I, H, &p.gate)) return rc;
  if (int rc = make_weight(up, E * I, H, &p.up)) return rc;
  if (int rc = make_weight(down, E * H, I, &p.down)) return rc;
  if ((p.gate.zp == nullptr) != (p.up.zp == nullptr)) return NPB_ERR_UNSUPPORTED;
  if (T == 0) return NPB_OK;
  if (x == nullptr || logits == nullptr || y == nullptr || workspace == nullptr) return NPB_ERR_INVALID_ARG;
  if (workspace_bytes < q_moe_workspace_bytes(T, top_k, I)) return NPB_ERR_TOO_LARGE;
  const size_t logit_size = logits_dtype == NPB_F32 ? 4 : 2;
  if (!aligned_to(x, 16) || !aligned_to(workspace, 16) || !aligned_to(y, 2) || !aligned_to(logits, logit_size))
    return NPB_ERR_ALIGNMENT;
  p.x = x;
  p.logits = logits;
  p.logits_dtype = logits_dtype;
  p.T = (int)T; p.E = (int)E; p.H = (int)H; p.I = (int)I;
  p.top_k = top_k;
  p.renormalize = renormalize != 0;
  p.h = static_cast<uint16_t*>(workspace);
  p.h_sum = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + T * top_k * I * 4);
  p.y = y;
  return dtype == NPB_BF16 ? launch_tokens<__nv_bfloat16>(p, st) : launch_tokens<__half>(p, st);
}

}  // namespace npb
