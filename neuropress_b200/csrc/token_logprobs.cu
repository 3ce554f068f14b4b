// Log probabilities of given tokens, entropy and the top alternatives, from logits in one pass.
//
//   m = max_v l_v,  s = sum_v e^(l_v - m),  u = sum_v e^(l_v - m) (l_v - m)
//   log p_v = (l_v - m) - ln s,   entropy = ln s - u / s          (nats; log p of the given token)
//   the n largest l_v, equal values by ascending v, as log p_v and v
//
// A row is split over a cluster of 1..8 CTAs; each thread keeps (m, s, u) of its own elements with a
// running maximum (a tile of three or eight 16-byte loads raises m at most once), so every logit is read from
// HBM once.  All sums are fp32; l - m is formed before the multiplication by log2(e), so rows with a
// large common offset lose nothing.  Bound by HBM for many rows, by latency for a few.
//
// The n largest without a second pass: if every full warp's q-th largest THREAD maximum is at least b, with q = n /
// warps rounded up, n elements are at least b, and only a few dozen elements are.  The threads whose maximum
// reaches the least of those q-th largest are re-read (L2), their elements at or above it go to a shared-memory
// list, and an element's rank in the answer is the number of larger (value, index) keys in the list -- no order of
// arrival enters the result.  Rows where that list overflows (masked or constant rows: the bound ties with most of
// the row) find the exact n-th value by bisection over the ordered bits of the values and take the ties in index
// order.  The CTAs of a cluster meet with sorted lists, where a rank is a binary search in each.
//
// Per element of a 16-bit row: one unpacking, half an instruction each for the maximum (on packed pairs), l - m, its
// scaling, and the two sums (packed fp32), one ex2.  The exponentials alone would take 0.7 of the time that HBM
// needs for them.
#include <type_traits>

#include "common.cuh"
#include "order_key.cuh"
#include "tcgen05.cuh"

namespace npb {
namespace {

using sm100::cluster_ctarank;
using sm100::cluster_sync_all;
using sm100::map_to_cta;
using sm100::smem_u32;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kUnroll = 3;      // 16-byte loads per thread and tile with many rows
constexpr int kWide = 8;        // and with few
constexpr int kMaxTop = 32;
constexpr int kListCap = 1024;  // candidate keys in shared memory
constexpr int kMaxSplit = 8;    // CTAs per row (portable cluster size)
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// (value, index): larger value first, equal values by ascending index.
__device__ __forceinline__ uint64_t full_key(uint32_t k, int index) {
  return ((uint64_t)k << 32) | (uint32_t)~index;
}

// Sums of a part of the row, relative to its maximum m (-inf: no element above -inf yet; then s and
// u are 0, or NaN when a NaN was met).
struct Part {
  float m, s, u;
};

__device__ __forceinline__ Part merge(const Part& a, const Part& b) {
  Part r;
  r.m = fmaxf(a.m, b.m);
  // shift of each side; the clamp keeps 0 * shift from being NaN for an empty side
  const float da = a.m == r.m ? 0.f : fmaxf(a.m - r.m, -1e20f), db = b.m == r.m ? 0.f : fmaxf(b.m - r.m, -1e20f);
  const float ca = ex2(da * kLog2e), cb = ex2(db * kLog2e);
  r.s = ca * a.s + cb * b.s;
  r.u = ca * (a.u + da * a.s) + cb * (b.u + db * b.s);
  return r;
}

template <typename T>
struct Tile {
  static constexpr int EPV = 16 / (int)sizeof(T);
  static constexpr uint32_t kMasked =  // -inf, or two
      sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  struct alignas(16) Vec { T e[EPV]; };
};

template <typename T>
__device__ __forceinline__ typename Tile<T>::Vec load_vec(const T* p) {
  const uint4 r = __ldg(reinterpret_cast<const uint4*>(p));
  return *reinterpret_cast<const typename Tile<T>::Vec*>(&r);
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
__device__ __forceinline__ F2 add2(const F2& a, const F2& b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
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

// Element pairs of a vector as floats, and the largest element (NaN only if every element is).
template <typename T>
__device__ __forceinline__ F2 pair_of(const typename Tile<T>::Vec& q, int i) {
  return pack(to_f32(q.e[2 * i]), to_f32(q.e[2 * i + 1]));
}
__device__ __forceinline__ float largest(const Tile<float>::Vec& q) {
  return fmaxf(fmaxf(q.e[0], q.e[1]), fmaxf(q.e[2], q.e[3]));
}
__device__ __forceinline__ float largest(const Tile<__half>::Vec& q) {
  const __half2* h = reinterpret_cast<const __half2*>(q.e);
  const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float largest(const Tile<__nv_bfloat16>::Vec& q) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(q.e);
  const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(__low2float(m), __high2float(m));
}

// Adds N vectors to a part.  CLAMP: d of a masked (-inf) element is raised to -1e20, its e is 0.  Otherwise the product
// e * d of one is 0 * -inf = NaN; such a tile (u is NaN, s is not) is summed again with d clamped, so that the others pay
// nothing.
template <typename T, int N, bool CLAMP>
__device__ __forceinline__ void add_vectors(Part& p, const typename Tile<T>::Vec (&q)[N]) {
  constexpr int PAIRS = Tile<T>::EPV / 2;
  float tm = largest(q[0]);
#pragma unroll
  for (int i = 1; i < N; ++i) tm = fmaxf(tm, largest(q[i]));
  if (tm > p.m) {
    const float d = fmaxf(p.m - tm, -1e20f), c = ex2(d * kLog2e);
    p.u = c * (p.u + d * p.s);
    p.s *= c;
    p.m = tm;
  }
  const float ref = p.m == -INFINITY ? 0.f : p.m;
  const F2 less = pack(-ref, -ref), scale = pack(kLog2e, kLog2e);
  F2 s2 = pack(0.f, 0.f), u2 = s2;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int k = 0; k < PAIRS; ++k) {
      F2 d = add2(pair_of<T>(q[i], k), less);
      float a, b;
      unpack(mul2(d, scale), a, b);
      const F2 e = pack(ex2(a), ex2(b));
      s2 = add2(s2, e);
      if (CLAMP) {
        unpack(d, a, b);
        d = pack(fmaxf(a, -1e20f), fmaxf(b, -1e20f));
      }
      u2 = fma2(e, d, u2);
    }
  float s, s_hi, u, u_hi;
  unpack(s2, s, s_hi);
  unpack(u2, u, u_hi);
  s += s_hi;
  u += u_hi;
  if (!CLAMP && u != u) {
    u = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int k = 0; k < 2 * PAIRS; ++k) {
        const float d = to_f32(q[i].e[k]) - ref;
        u = fmaf(ex2(d * kLog2e), fmaxf(d, -1e20f), u);
      }
  }
  p.s += s;
  p.u += u;
}

// A part of one element.
__device__ __forceinline__ Part part_of(float f) {
  const float d = f - (f == -INFINITY ? 0.f : f);  // 0, or NaN for NaN and +inf
  return {f == f ? f : -INFINITY, f == -INFINITY ? 0.f : ex2(d), f == -INFINITY ? 0.f : d};
}

struct Shared {
  Part warp_part[kWarps];
  Part parts[kMaxSplit];             // rank 0: one per CTA of the cluster
  uint32_t bound;                    // key the n-th largest element is known to reach
  int n_hot, n_list;
  int hot[kThreads];                 // threads whose maximum reaches the bound
  unsigned long long list[kListCap];
  unsigned long long best[kMaxSplit * kMaxTop];  // rank 0: the CTAs' n largest keys, 0 where there is none
  int warp_count[kWarps];
};

__device__ __forceinline__ int block_sum(int v, Shared& sh) {
  v = __reduce_add_sync(0xffffffffu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.warp_count[threadIdx.x >> 5] = v;
  __syncthreads();
  int t = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) t += sh.warp_count[w];
  return t;
}

// Exact selection of the `need` largest keys of row[first, last) by bisection; the slow path.
template <typename T>
__device__ void select_by_bisection(const T* __restrict__ row, int first, int last, int need, Shared& sh) {
  const int tid = threadIdx.x;
  auto count_from = [&](uint32_t k) {
    int c = 0;
    for (int i = first + tid; i < last; i += kThreads) c += order_key(to_f32(row[i])) >= k;
    return block_sum(c, sh);
  };
  // the n-th largest key: the bound itself where it ties (masked and constant rows), else bit by bit
  uint32_t nth = 0;
  const uint32_t bound = sh.bound;
  if (bound > 1u && count_from(bound + 1) < need && count_from(bound) >= need) {
    nth = bound;
  } else {
    for (int b = 31; b >= 0; --b)
      if (count_from(nth | (1u << b)) >= need) nth |= 1u << b;
  }
  __syncthreads();
  if (tid == 0) sh.n_list = 0;
  __syncthreads();
  for (int i = first + tid; i < last; i += kThreads) {  // fewer than `need` keys lie above the n-th
    const uint32_t k = order_key(to_f32(row[i]));
    if (k > nth) sh.list[atomicAdd(&sh.n_list, 1)] = full_key(k, i);
  }
  __syncthreads();
  int have = sh.n_list;
  // ties in index order: eight consecutive elements per thread and step
  for (int base = first; base < last && have < need; base += kThreads * 8) {
    int c = 0;
    for (int j = 0; j < 8; ++j) {
      const int i = base + tid * 8 + j;
      c += i < last && order_key(to_f32(row[i])) == nth;
    }
    int incl = c;  // inclusive scan over the block
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if ((tid & 31) >= o) incl += v;
    }
    __syncthreads();
    if ((tid & 31) == 31) sh.warp_count[tid >> 5] = incl;
    __syncthreads();
    int before = incl - c, total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < (tid >> 5)) before += sh.warp_count[w];
      total += sh.warp_count[w];
    }
    int pos = have + before;
    for (int j = 0; j < 8 && pos < need; ++j) {
      const int i = base + tid * 8 + j;
      if (i < last && order_key(to_f32(row[i])) == nth) sh.list[pos++] = full_key(nth, i);
    }
    have = min(need, have + total);
  }
  __syncthreads();
  if (tid == 0) sh.n_list = have;
  __syncthreads();
}

// Six CTAs on an SM with many rows: what hides the loads is occupancy (4096 x 128000 bf16 in a CUDA graph: 187 us, 5.6
// TB/s, launched one by one 214-219 us; four CTAs with four loads per tile 194 us, three with the next tile prefetched into
// registers 249 us).
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads, WIDE ? 3 : 6)
token_logprobs_kernel(const T* __restrict__ logits, int64_t ld, int V, const int64_t* __restrict__ targets, int top_n,
                      int split, float* __restrict__ logprob, float* __restrict__ entropy,
                      float* __restrict__ top_logprobs, int64_t* __restrict__ top_ids) {
  constexpr int EPV = Tile<T>::EPV;
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = split > 1 ? (int)cluster_ctarank() : 0;
  const int64_t r = blockIdx.x / split;
  const T* row = logits + r * ld;

  // [0, head) and [tail, V) are read by element (rank 0), the vectors between them are split evenly
  const int head = min(V, (int)(((16u - (uint32_t)(reinterpret_cast<uintptr_t>(row) & 15u)) & 15u) / sizeof(T)));
  const int n_vec = (V - head) / EPV, tail = head + n_vec * EPV;
  const int per_cta = (n_vec + split - 1) / split;
  const int v0 = min(n_vec, rank * per_cta), v1 = min(n_vec, v0 + per_cta);
  int odd = -1;  // this thread's element outside the vectors
  if (rank == 0) {
    if (tid < head) odd = tid;
    else if (tid - head < V - tail) odd = tail + tid - head;
  }

  Part p{-INFINITY, 0.f, 0.f};
  const T* vectors = row + head;
  int v = v0 + tid;
  if (WIDE) {
    for (; v < v1; v += kWide * kThreads) {
      typename Tile<T>::Vec q[kWide];
#pragma unroll
      for (int i = 0; i < kWide; ++i) {
        if (v + i * kThreads < v1) {
          q[i] = load_vec(vectors + (int64_t)(v + i * kThreads) * EPV);
        } else {  // masked elements
          const uint32_t f = Tile<T>::kMasked;
          const uint4 none = make_uint4(f, f, f, f);
          q[i] = *reinterpret_cast<const typename Tile<T>::Vec*>(&none);
        }
      }
      add_vectors<T, kWide, true>(p, q);
    }
  } else {
    for (; v + (kUnroll - 1) * kThreads < v1; v += kUnroll * kThreads) {
      typename Tile<T>::Vec q[kUnroll];
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) q[i] = load_vec(vectors + (int64_t)(v + i * kThreads) * EPV);
      add_vectors<T, kUnroll, false>(p, q);
    }
    for (; v < v1; v += kThreads) {
      const typename Tile<T>::Vec q[1] = {load_vec(vectors + (int64_t)v * EPV)};
      add_vectors<T, 1, false>(p, q);
    }
  }
  if (odd >= 0) p = merge(p, part_of(to_f32(row[odd])));

  const bool mine = v0 + tid < v1 || odd >= 0;
  if (top_n > 0) {
    // ---- the n largest keys of this CTA's slice ----
    const int first = rank == 0 ? 0 : head + v0 * EPV;
    const int count = (v1 - v0) * EPV + (rank == 0 ? head + (V - tail) : 0);
    const int need = min(top_n, count);
    const uint32_t my_max = mine ? order_key(p.m) : 0u;
    const int full = min(v1 - v0, kThreads) / 32;  // warps of which every thread has elements
    if (tid == 0) {
      sh.bound = full ? 0xffffffffu : 0u;          // none: everything is a candidate
      sh.n_hot = 0;
      sh.n_list = 0;
    }
    __syncthreads();
    if (warp < full) {
      uint32_t left = my_max, nth = 0;
      for (int q = (need + full - 1) / full; q > 0; --q) {
        nth = __reduce_max_sync(0xffffffffu, left);
        const uint32_t who = __ballot_sync(0xffffffffu, left == nth);
        if (lane == __ffs(who) - 1) left = 0;
      }
      if (lane == 0) atomicMin(&sh.bound, nth);
    }
    __syncthreads();
    const uint32_t bound = sh.bound;
    if (my_max != 0 && my_max >= bound) sh.hot[atomicAdd(&sh.n_hot, 1)] = tid;
    __syncthreads();
    const int n_hot = sh.n_hot, per = (v1 - v0 + kThreads - 1) / kThreads + 1;  // + the odd element
    auto offer = [&](float f, int index) {
      const uint32_t k = order_key(f);
      if (k >= bound) {
        const int pos = atomicAdd(&sh.n_list, 1);
        if (pos < kListCap) sh.list[pos] = full_key(k, index);
      }
    };
    // loads in flight: four for fp32 (300 x 128000: 42 us, one 48 us), whose rows have twice the vectors; 16-bit rows lose
    // (300 x 128000: 33 / 31 us), and with many rows the other CTAs hide the load
    constexpr int kBatch = WIDE && sizeof(T) == 4 ? 4 : 1;
    for (int w0 = tid; w0 < n_hot * per; w0 += kBatch * kThreads) {
      typename Tile<T>::Vec q[kBatch];
      int at[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int w = w0 + b * kThreads;
        at[b] = -1;
        if (w >= n_hot * per) continue;
        const int h = sh.hot[w / per], i = w % per;
        if (i == per - 1) {
          if (rank == 0) {
            const int o = h < head ? h : tail + h - head;
            if (o < V && (h < head || h - head < V - tail)) offer(to_f32(row[o]), o);
          }
        } else if (v0 + h + i * kThreads < v1) {
          at[b] = head + (v0 + h + i * kThreads) * EPV;
          q[b] = load_vec(row + at[b]);
        }
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
        if (at[b] >= 0) {
#pragma unroll
          for (int e = 0; e < EPV; ++e) offer(to_f32(q[b].e[e]), at[b] + e);
        }
    }
    __syncthreads();
    if (sh.n_list > kListCap || sh.n_list < need) {
      if (rank == 0 && split > 1) {
        // rank 0 owns [0, head), its vectors and [tail, V): two ranges.  Select from the vectors and
        // the head together, then add the at most seven tail elements as further candidates.
        const int mid = head + v1 * EPV;
        select_by_bisection(row, 0, mid, min(need, mid), sh);
        if (tail + tid < V && tid < 16) {
          const uint32_t k = order_key(to_f32(row[tail + tid]));
          sh.list[atomicAdd(&sh.n_list, 1)] = full_key(k, tail + tid);
        }
        __syncthreads();
      } else {
        select_by_bisection(row, first, first + count, need, sh);
      }
    }
    // rank of each candidate; the n best of every CTA meet in rank 0
    unsigned long long* dst = sh.best + rank * kMaxTop;
    const int n_list = sh.n_list;
    if (split > 1) {  // rank 0 runs: its shared memory may be written
      __syncwarp();
      cluster_sync_all();
    }
    const uint32_t dst0 = split > 1 ? map_to_cta(smem_u32(dst), 0) : 0u;
    auto put = [&](int pos, unsigned long long key) {
      if (split > 1) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(dst0 + pos * 8), "l"(key) : "memory");
      else dst[pos] = key;
    };
    for (int i = tid; i < n_list; i += kThreads) {
      const unsigned long long key = sh.list[i];
      int pos = 0;
      for (int j = 0; j < n_list; ++j) pos += sh.list[j] > key;
      if (pos < need) put(pos, key);
    }
    if (tid >= need && tid < top_n) put(tid, 0ull);
  } else if (split > 1) {
    cluster_sync_all();
  }

  // ---- the sums: threads -> warps -> CTA -> cluster ----
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Part q;
    q.m = __shfl_xor_sync(0xffffffffu, p.m, o);
    q.s = __shfl_xor_sync(0xffffffffu, p.s, o);
    q.u = __shfl_xor_sync(0xffffffffu, p.u, o);
    // both lanes of a pair merge in the same order, so every lane ends with the same bits
    p = (lane & o) ? merge(q, p) : merge(p, q);
  }
  if (lane == 0) sh.warp_part[warp] = p;
  __syncthreads();
  if (tid == 0) {
    Part a = sh.warp_part[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) a = merge(a, sh.warp_part[w]);
    if (split > 1) {
      const uint32_t at = map_to_cta(smem_u32(&sh.parts[rank]), 0);
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(a.m) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at + 4), "f"(a.s) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at + 8), "f"(a.u) : "memory");
    } else {
      sh.parts[0] = a;
    }
  }
  if (split > 1) {
    __syncwarp();
    cluster_sync_all();
    if (rank != 0) return;
  } else {
    __syncthreads();
  }
  Part a = sh.parts[0];
  for (int c = 1; c < split; ++c) a = merge(a, sh.parts[c]);
  const float ln_s = logf(a.s);
  const bool nothing = a.m == -INFINITY && a.s == 0.f;  // every logit of the row is -inf
  auto log_p = [&](float l) { return nothing ? -INFINITY : (l - a.m) - ln_s; };
  if (tid == 0) {
    const int64_t t = targets[r];
    logprob[r] = t >= 0 && t < V ? log_p(to_f32(row[t])) : 0.f;
    entropy[r] = nothing ? 0.f : ln_s - a.u / a.s;
  }
  if (top_n > 0) {
    for (int i = tid; i < split * top_n; i += kThreads) {
      const unsigned long long key = sh.best[(i / top_n) * kMaxTop + i % top_n];
      if (key == 0) continue;
      int pos = 0;
#pragma unroll
      for (int c = 0; c < kMaxSplit; ++c)
        if (c < split) {  // keys of a CTA that are larger: its list is in descending order
          int n = 0;
#pragma unroll
          for (int step = kMaxTop; step > 0; step >>= 1)
            if (n + step <= top_n && sh.best[c * kMaxTop + n + step - 1] > key) n += step;
          pos += n;
        }
      if (pos < top_n) {
        top_ids[r * top_n + pos] = (int64_t)(uint32_t)~(uint32_t)key;
        top_logprobs[r * top_n + pos] = log_p(key_value((uint32_t)(key >> 32)));
      }
    }
  }
}

// The wide form holds three CTAs on an SM; a grid of one wave of it has one load latency per eight loads of a thread and
// none for a ragged end (20 x 128000 bf16: 10.0 us, narrow 10.8 us; 220 x 128000: 23 / 29 us; 150 x 50001 fp32: 15.7 / 16.3
// us).  More rows have enough CTAs to hide the loads.
constexpr int kWidePerSm = 3;

// CTAs per row: as many as one wave of the wide form has, each with a slice worth its start.
int pick_split(int64_t R, int64_t V) {
  int split = 1;
  while (split < kMaxSplit && R * split * 2 <= (int64_t)sm_count() * kWidePerSm && V / (split * 2) >= 2048) split *= 2;
  return split;
}

template <typename T>
int launch(const void* logits, int64_t ld, int64_t R, int64_t V, const int64_t* targets, int top_n, float* logprob,
           float* entropy, float* top_logprobs, int64_t* top_ids, cudaStream_t st) {
  if (!aligned_to(logits, sizeof(T))) return NPB_ERR_ALIGNMENT;
  const int split = pick_split(R, V);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(R * split));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = split;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const bool wide = R * split <= (int64_t)sm_count() * kWidePerSm;
  NPB_CUDA_TRY(cudaLaunchKernelEx(&cfg, wide ? token_logprobs_kernel<T, true> : token_logprobs_kernel<T, false>,
                                  static_cast<const T*>(logits), ld, (int)V, targets, top_n, split, logprob, entropy,
                                  top_logprobs, top_ids));
  NPB_LAUNCH_CHECK();
  return NPB_OK;
}

}  // namespace

int token_logprobs(const void* logits, int64_t ld, int64_t R, int64_t V, int dtype, const int64_t* targets, int top_n,
                   float* logprob, float* entropy, float* top_logprobs, int64_t* top_ids, cudaStream_t st) {
  if (R < 0 || V <= 0 || top_n < 0 || (R > 1 && ld < V)) return NPB_ERR_INVALID_ARG;
  if (top_n > kMaxTop || top_n > V) return NPB_ERR_UNSUPPORTED;
  if (R >= (int64_t)1 << 27 || V >= (int64_t)1 << 30) return NPB_ERR_UNSUPPORTED;
  if (R == 0) return NPB_OK;
  if (logits == nullptr || targets == nullptr || logprob == nullptr || entropy == nullptr ||
      (top_n > 0 && (top_logprobs == nullptr || top_ids == nullptr)))
    return NPB_ERR_INVALID_ARG;
  switch (dtype) {
    case NPB_BF16: return launch<__nv_bfloat16>(logits, ld, R, V, targets, top_n, logprob, entropy, top_logprobs, top_ids, st);
    case NPB_F16: return launch<__half>(logits, ld, R, V, targets, top_n, logprob, entropy, top_logprobs, top_ids, st);
    case NPB_F32: return launch<float>(logits, ld, R, V, targets, top_n, logprob, entropy, top_logprobs, top_ids, st);
    default: return NPB_ERR_UNSUPPORTED;
  }
}

}  // namespace npb
