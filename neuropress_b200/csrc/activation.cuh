// Activations of the GEMM epilogues, fp32 in and out.
#pragma once

#include <cuda_runtime.h>

#include "neuropress_b200.h"

namespace npb {

// NaN passes through every one of them.  silu and the tanh form of gelu are v * sigmoid(.) with the fast
// exponential and division (a few fp32 ulps; the result is rounded to 16 bits): a negative argument far
// out makes the exponential +inf and the quotient -0.  gelu uses erfc, which does not cancel for
// negative arguments as 1 + erf does.
__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {
    case NPB_ACT_RELU: return v < 0.f ? 0.f : v;
    case NPB_ACT_SILU: return __fdividef(v, 1.f + __expf(-v));
    case NPB_ACT_GELU: return 0.5f * v * erfcf(-0.70710678118654752f * v);
    case NPB_ACT_GELU_TANH: {
      const float u = 0.79788456080286536f * fmaf(0.044715f * v * v, v, v);
      return __fdividef(v, 1.f + __expf(-2.f * u));
    }
    default: return v;
  }
}

// One branch for all of them: the values' chains overlap.
template <int N>
__device__ __forceinline__ void activate_all(float (&v)[N], int act) {
  auto each = [&](int which) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = activate(v[i], which);
  };
  switch (act) {
    case NPB_ACT_RELU: return each(NPB_ACT_RELU);
    case NPB_ACT_SILU: return each(NPB_ACT_SILU);
    case NPB_ACT_GELU: return each(NPB_ACT_GELU);
    case NPB_ACT_GELU_TANH: return each(NPB_ACT_GELU_TANH);
    default: return;
  }
}

}  // namespace npb
