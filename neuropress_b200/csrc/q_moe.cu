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
// block-diagonal, column 2 t + c holds block t of token c of a pair, so lane (g, t) of the result holds
// exactly the block whose scale it loaded.  An mma serves 256 weights for two tokens.
//
// Kernel 1 keeps the tokens of its unit (up to NT tokens of one expert) in shared memory, in the order of
// the code pairs; h leaves it as fp16 in that order with a power of two per 32-block, so it keeps 11
// significant bits whatever its size (1/8 of a bf16 half step; nothing overflows).  Kernel 2 brings h
// along with the weights by cp.async.  An expert with more tokens than a unit is read again (from L2).
// Every sum has a fixed order: results do not depend on scheduling.
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
  int logits_dtype;
  int T, E, H, I, top_k, renormalize;
  MoeWeight gate, up, down;
  uint8_t* h;      // [T * top_k][I / 32] records, see kRecord
  void* y;
};

// One 32-block of one token's h: 32 fp16 values h / f in mma order, the power of two f, the sum of the 32
// values, padding to a multiple of 16 bytes.
constexpr int kRecord = 80;

// ---- routing ---------------------------------------------------------------------------------
struct Routing {
  uint32_t mask[kMaxExperts];            // tokens of each expert
  float weight[kMaxTokens][kMaxTopK];
  uint16_t id[kMaxTokens][kMaxTopK];     // 0xffff: none
  uint16_t unit_expert[kMaxUnits];
  uint32_t unit_mask[kMaxUnits];         // its tokens
  uint16_t unit_slot[kMaxUnits];         // row of h of its first token
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
      uint32_t m = n > 0 ? r.mask[e] : 0u;
      for (int i = 0; i < u; ++i) {
        const int at = units + iu - u + i;
        uint32_t rest = m;
        for (int j = 0; j < NT && rest; ++j) rest &= rest - 1;
        r.unit_expert[at] = (uint16_t)e;
        r.unit_mask[at] = m & ~rest;
        r.unit_slot[at] = (uint16_t)(slots + in - n + i * NT);
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
__device__ __forceinline__ uint4 ld_stream(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// Codes, scales and zero points of four rows (two tiles, rows g and g + 8 of each) for one 32-block.
template <bool ASYM>
struct Blocks {
  uint4 c[4];
  __half s[4];
  __half z[ASYM ? 4 : 1];
};

__device__ __forceinline__ int group_of(const MoeWeight& w, int blk) {
  return w.group_shift >= 0 ? blk >> w.group_shift : blk / w.group_blocks;
}

// Block `blk` (counted from the start of the matrix), group `group` likewise.
template <bool ASYM>
__device__ __forceinline__ void fetch_row(Blocks<ASYM>& b, int i, const MoeWeight& w, int64_t blk, int64_t group,
                                          bool valid) {
  b.c[i] = make_uint4(0, 0, 0, 0);
  b.s[i] = __ushort_as_half(0);
  if (ASYM) b.z[ASYM ? i : 0] = __ushort_as_half(0);
  if (valid) {
    b.c[i] = ld_stream(w.codes + blk * 16);
    b.s[i] = __ldg(w.scale + group);
    if (ASYM) b.z[ASYM ? i : 0] = __ldg(w.zp + group);
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
__device__ __forceinline__ void a_operands(const uint4& lo, const uint4& hi, int i, uint32_t (&a)[2][4]) {
  const uint32_t l = word_of(lo, i), h = word_of(hi, i);
  a[0][0] = code_pair<T>(l, 0); a[0][1] = code_pair<T>(h, 0); a[0][2] = code_pair<T>(l, 1); a[0][3] = code_pair<T>(h, 1);
  a[1][0] = code_pair<T>(l, 2); a[1][1] = code_pair<T>(h, 2); a[1][2] = code_pair<T>(l, 3); a[1][3] = code_pair<T>(h, 3);
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

// Eight consecutive elements in the order of the code pairs: (0, 4) (1, 5) (2, 6) (3, 7).
__device__ __forceinline__ uint4 in_pair_order(const uint4& v) {
  return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                    __byte_perm(v.y, v.w, 0x7632));
}

// Adds one step (128 of k, one 32-block per lane of a quad) of two 16-row tiles to acc[tile][pair]: rows g
// (tokens 0, 1 of the pair) and g + 8.  operand(q): shared address of this lane's 64 bytes of pair q (zeros
// for a lane off the diagonal); factors(q): {sum of token 0, of token 1, factor of 0, of 1} of its block.
template <typename T, int NP, bool ASYM, bool SCALED, typename Operand, typename Factors>
__device__ __forceinline__ void add_step(float (&acc)[2][NP][4], const Blocks<ASYM>& b, int n, Operand operand,
                                         Factors factors) {
  float d[2][NP][4];
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
      for (int c = 0; c < 4; ++c) d[w][q][c] = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t a[2][2][4];
    a_operands<T>(b.c[0], b.c[1], i, a[0]);
    a_operands<T>(b.c[2], b.c[3], i, a[1]);
#pragma unroll
    for (int q = 0; q < NP; ++q)
      if (2 * q < n) {
        const uint4 v = lds128(operand(q) + i * 16);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          mma16816<T>(d[w][q], a[w][0], v.x, v.y);
          mma16816<T>(d[w][q], a[w][1], v.z, v.w);
        }
      }
  }
#pragma unroll
  for (int q = 0; q < NP; ++q)
    if (2 * q < n) {
      const float4 f = factors(q);
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float sc = __half2float(b.s[2 * w + h]);
          const float mz = magic_of<T>() + (ASYM ? __half2float(b.z[ASYM ? 2 * w + h : 0]) : 8.f);
          float* to = &acc[w][q][2 * h];
          const float* from = &d[w][q][2 * h];
          to[0] = fmaf(SCALED ? sc * f.z : sc, fmaf(-mz, f.x, from[0]), to[0]);
          to[1] = fmaf(SCALED ? sc * f.w : sc, fmaf(-mz, f.y, from[1]), to[1]);
        }
    }
}

__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// ---- kernel 1: gate / up products, silu, routing weight ------------------------------------------
constexpr int kUpThreads = 256;  // two 16-row tiles x four slices of K
constexpr int kUpRows = 32;      // rows of gate and of up per item: one 32-block of h
constexpr int kUpSlices = 4;

// Shared memory of kernel 1 behind the routing: tokens [NT][4 * steps] blocks of 64 bytes (rows 16 bytes
// apart in the banks), their block sums, the partial products, 64 bytes of zeros.
struct UpLayout {
  int row, sums, red, zeros, bytes;
  __host__ __device__ UpLayout(int n_blk, int nt) {
    const int blocks = (n_blk + 3) / 4 * 4;
    row = blocks * 64 + 16;
    sums = row * nt;
    red = sums + nt * blocks * 4;
    zeros = red + kUpSlices * 2 * 2 * nt * 16 * 4;
    bytes = zeros + 64;
  }
};

template <typename T, int NT, bool ASYM>
__global__ void __launch_bounds__(kUpThreads, 2)
moe_up_kernel(const MoeParams p) {
  constexpr int NP = NT / 2;  // pairs of tokens
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ Routing r;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const T* x = static_cast<const T*>(p.x);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int n_blk = p.H / 32, n_steps = (n_blk + 3) / 4, blocks = n_steps * 4;
  const int n_group = n_blk / p.gate.group_blocks;
  const UpLayout at(n_blk, NT);
  float* x_sum = reinterpret_cast<float*>(dyn + at.sums);  // [NT][blocks]
  float* red = reinterpret_cast<float*>(dyn + at.red);     // [slice][tile][matrix][NT][16]
  const uint32_t base = sm100::smem_u32(dyn);
  if (tid < 16) reinterpret_cast<uint32_t*>(dyn + at.zeros)[tid] = 0;
  route<NT>(p, r);

  const int tiles = p.I / kUpRows;
  const int64_t items = (int64_t)tiles * r.n_units;
  const int first = (int)(items * blockIdx.x / gridDim.x), last = (int)(items * (blockIdx.x + 1) / gridDim.x);
  const int mt = warp & 1, ks = warp >> 1;
  const int s_first = n_steps * ks / kUpSlices, s_last = n_steps * (ks + 1) / kUpSlices;
  const bool diag = (lane >> 3) == t;  // this lane holds the nonzero part of column lane / 4
  const uint32_t mine = base + ((lane >> 2) & 1) * at.row + t * 64;  // of pair 0 in step 0

  int unit = -1, n = 0, e = 0;
  for (int item = first; item < last; ++item) {
    const int u = item / tiles, i0 = (item - u * tiles) * kUpRows;
    e = r.unit_expert[u];
    const int64_t row = (int64_t)e * p.I + i0 + mt * 16 + g;
    const int64_t row_blk = row * n_blk, row_group = row * n_group;
    auto fetch = [&](Blocks<ASYM>& b, int s) {
      const int blk = s * 4 + t, group = group_of(p.gate, blk);
      const bool valid = s < s_last && blk < n_blk;
      const int64_t at_blk = row_blk + blk, at_group = row_group + group;
      fetch_row(b, 0, p.gate, at_blk, at_group, valid);
      fetch_row(b, 1, p.gate, at_blk + 8 * n_blk, at_group + 8 * n_group, valid);
      fetch_row(b, 2, p.up, at_blk, at_group, valid);
      fetch_row(b, 3, p.up, at_blk + 8 * n_blk, at_group + 8 * n_group, valid);
    };
    Blocks<ASYM> b0, b1;
    fetch(b0, s_first);
    fetch(b1, s_first + 1);
    if (u != unit) {
      unit = u;
      uint32_t m = r.unit_mask[u];
      n = __popc(m);
      // the unit's tokens (and zeros behind the last of an odd count) in the order of the code pairs
#pragma unroll 1
      for (int i = 0; i < ((n + 1) & ~1); ++i) {
        const int token = __ffs(m) - 1;
        const uint4* src = reinterpret_cast<const uint4*>(x + (int64_t)(i < n ? token : 0) * p.H);
        m &= m - 1;
        for (int j0 = 0; j0 < blocks * 4; j0 += kUpThreads) {  // whole warps: the quads sum below
          const int j = j0 + tid;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (i < n && j < n_blk * 4) v = __ldg(src + j);
          if (j < blocks * 4) *reinterpret_cast<uint4*>(dyn + i * at.row + j * 16) = in_pair_order(v);
          const T* f = reinterpret_cast<const T*>(&v);
          float s = 0.f;
#pragma unroll
          for (int k = 0; k < 8; ++k) s += to_f32(f[k]);
          s = quad_sum(s);
          if ((j & 3) == 0 && j < blocks * 4) x_sum[i * blocks + (j >> 2)] = s;
        }
      }
      __syncthreads();
    }
    float acc[2][NP][4] = {};
    auto compute = [&](const Blocks<ASYM>& b, int s) {
      add_step<T, NP, ASYM, false>(
          acc, b, n, [&](int q) { return diag ? mine + q * 2 * at.row + s * 256 : base + at.zeros; },
          [&](int q) {
            const float* f = x_sum + 2 * q * blocks + s * 4 + t;
            return make_float4(f[0], f[blocks], 1.f, 1.f);
          });
    };
    for (int s = s_first; s < s_last; s += 2) {
      compute(b0, s);
      fetch(b0, s + 2);
      if (s + 1 < s_last) compute(b1, s + 1);
      fetch(b1, s + 3);
    }
    // the four blocks of a quad, then the slices of K
    float* part = red + (ks * 2 + mt) * 2 * NT * 16;
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int q = 0; q < NP; ++q)
        if (2 * q < n)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float v = quad_sum(acc[w][q][c]);
            if (t == 0) part[(w * NT + 2 * q + (c & 1)) * 16 + g + (c >> 1) * 8] = v;
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
      // the power of two at or below the block's largest magnitude (1 for a block of zeros or with inf / NaN)
      float top = fabsf(h);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const uint32_t exponent = __float_as_uint(top) >> 23;
      const float f = exponent == 0 || exponent == 255 ? 1.f : __uint_as_float(exponent << 23);
      const __half v = __float2half_rn(h / f);
      const float sum = warp_sum(__half2float(v));
      uint8_t* rec = p.h + ((int64_t)(r.unit_slot[u] + warp) * (p.I / 32) + i0 / 32) * kRecord;
      reinterpret_cast<__half*>(rec)[(lane & 24) + (lane & 3) * 2 + ((lane >> 2) & 1)] = v;
      if (lane == 0) *reinterpret_cast<float2*>(rec + 64) = make_float2(f, sum);
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
// [stage][NT][4], then 64 bytes of zeros.
struct DownLayout {
  int sums, ring, warp, zeros, bytes;
  __host__ __device__ DownLayout(int T, int nt) {
    sums = T * kDownRows * 4;
    ring = kDownStages * nt * 4 * kRecord;
    warp = sums + ring;
    zeros = warp * kDownWarps;
    bytes = zeros + 64;
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

template <typename T, int NT, bool ASYM>
__global__ void __cluster_dims__(kDownSplit, 1, 1) __launch_bounds__(kDownThreads, 2)
moe_down_kernel(const MoeParams p) {
  constexpr int NP = NT / 2;
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
  if (tid < 16) reinterpret_cast<uint32_t*>(dyn + at.zeros)[tid] = 0;
  route<NT>(p, r);

  // (unit, step) pairs in a row, an equal share of consecutive ones per warp of the cluster
  const int64_t total = (int64_t)r.n_units * n_steps;
  const int share = rank * kDownWarps + warp, shares = kDownSplit * kDownWarps;
  const int first = (int)(total * share / shares), last = (int)(total * (share + 1) / shares);
  const bool diag = (lane >> 3) == t;
  const uint32_t ring = base + warp * at.warp + at.sums;
  constexpr int kStage = NT * 4 * kRecord;
  const uint32_t mine = ring + (((lane >> 2) & 1) * 4 + t) * kRecord;  // of pair 0 in stage 0

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
  auto fetch_weights = [&](Blocks<ASYM>& b) {
    const int blk = fs * 4 + t;
    const bool valid = fetched < last && blk < n_blk;
    const int group = group_of(p.down, blk);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      fetch_row(b, i, p.down, row_blk + blk + 8 * i * n_blk, row_group + group + 8 * i * n_group, valid);
  };
  auto fetch_records = [&](int stage) {  // blocks fs * 4 .. + 4 of the unit's tokens; zeros past the last
    constexpr int kPieces = kRecord / 16;
    if (fetched < last)
#pragma unroll
      for (int c0 = 0; c0 < NT * 4 * kPieces; c0 += 32) {
        const int c = c0 + lane;
        const int k = c / kPieces, piece = c - k * kPieces, token = k >> 2, blk = fs * 4 + (k & 3);
        const bool valid = token < fn && blk < n_blk;
        if (c < NT * 4 * kPieces && token < ((fn + 1) & ~1))
          cp_async16(ring + stage * kStage + c * 16, valid ? rec + ((int64_t)token * n_blk + blk) * kRecord + piece * 16
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

  float acc[2][NP][4] = {};
  int unit = -1, n = 0;
  auto flush = [&] {
    uint32_t m = unit >= 0 ? r.unit_mask[unit] : 0u;
#pragma unroll
    for (int q = 0; q < NP; ++q)
      if (2 * q < n) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int token = __ffs(m) - 1;
          m &= m - 1;
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float v = quad_sum(acc[w][q][2 * h + c]);
              if (t == 0 && token >= 0) sums[token * kDownRows + w * 16 + h * 8 + g] += v;
              acc[w][q][2 * h + c] = 0.f;
            }
        }
      }
    __syncwarp();
  };
  int cu = fu, cs = fs;  // position of the computation
  auto compute = [&](const Blocks<ASYM>& b, int stage) {
    if (cu != unit) {
      flush();
      unit = cu;
      n = __popc(r.unit_mask[cu]);
    }
    const uint32_t from = mine + stage * kStage;
    add_step<__half, NP, ASYM, true>(
        acc, b, n, [&](int q) { return diag ? from + q * 8 * kRecord : base + at.zeros; },
        [&](int q) {
          const uint32_t f = ring + stage * kStage + (q * 8 + t) * kRecord + 64;
          float4 v;  // {sum 0, sum 1, factor 0, factor 1}
          asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.z), "=f"(v.x) : "r"(f));
          asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.w), "=f"(v.y) : "r"(f + 4 * kRecord));
          return v;
        });
    if (++cs == n_steps) { cs = 0; ++cu; }
    __syncwarp();  // the stage may be filled again
  };

  Blocks<ASYM> b0, b1;
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
  T* y = static_cast<T*>(p.y);
  constexpr int kRowsEach = kDownRows / kDownSplit;
  for (int i = tid; i < p.T * kRowsEach; i += kDownThreads) {
    const int token = i / kRowsEach, row = rank * kRowsEach + i % kRowsEach;
    float v = 0.f;
#pragma unroll
    for (int c = 0; c < kDownSplit; ++c)
      v += ld_cluster_f32(sm100::map_to_cta(base + (token * kDownRows + row) * 4, c));
    y[(int64_t)token * p.H + j0 + row] = from_f32<T>(v);
  }
  __syncwarp();
  sm100::cluster_sync_all();  // nobody leaves while its sums are read
}

// ---- host ----------------------------------------------------------------------------------------
template <typename T, int NT, bool ASYM>
int launch_up(const MoeParams& p, cudaStream_t st) {
  auto kern = moe_up_kernel<T, NT, ASYM>;
  const size_t smem = UpLayout(p.H / 32, NT).bytes;
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
  const size_t smem = DownLayout(p.T, NT).bytes;
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

template <typename T, int NT>
int launch(const MoeParams& p, cudaStream_t st) {
  if (int rc = p.gate.zp ? launch_up<T, NT, true>(p, st) : launch_up<T, NT, false>(p, st)) return rc;
  return p.down.zp ? launch_down<T, NT, true>(p, st) : launch_down<T, NT, false>(p, st);
}

template <typename T>
int launch_tokens(const MoeParams& p, cudaStream_t st) {
  // an expert has at most T tokens; eight per unit is what the registers hold, and a unit's tokens have to
  // fit the shared memory of kernel 1
  int nt = p.T <= 2 ? 2 : p.T <= 4 ? 4 : 8;
  while (nt > 2 && UpLayout(p.H / 32, nt).bytes + (int)sizeof(Routing) > max_dynamic_smem() / 2) nt /= 2;
  if (nt == 2) return launch<T, 2>(p, st);
  if (nt == 4) return launch<T, 4>(p, st);
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
  return T * top_k * (I / 32) * kRecord;
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
  p.T = (int)T; p.E = (int)E; p.H = (int)H; p.I = (int)I;
  p.top_k = top_k;
  p.renormalize = renormalize != 0;
  p.h = static_cast<uint8_t*>(workspace);
  p.y = y;
  return dtype == NPB_BF16 ? launch_tokens<__nv_bfloat16>(p, st) : launch_tokens<__half>(p, st);
}

}  // namespace npb
