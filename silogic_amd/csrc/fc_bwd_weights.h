// What the FC soft backward's weight kernels share: the one on fp32 inputs
// (fc_soft_bwd.hip) and the one on 8-bit inputs (fc_bwd8.hip).
#pragma once
#include "fc_soft_common.h"

namespace slg {

// dL/da, dL/db and dL/dparam of one node at operands (a, b), given dL/dy = g.
template <int NODE>
__device__ inline void node_grad(float a, float b, float g, const float4& p, float inv_tau,
                                 float& ga, float& gb, float (&gp)[4]) {
  if constexpr (NODE == SLG_NODE_MULTILINEAR2) {
    // y = (1-a)(1-b) s0 + a(1-b) s1 + (1-a) b s2 + a b s3 (nodes.py:174-178)
    const float ua = 1.0f - a, ub = 1.0f - b;
    gp[0] = g * (ua * ub);
    gp[1] = g * (a * ub);
    gp[2] = g * (ua * b);
    gp[3] = g * (a * b);
    ga = g * (ub * (p.y - p.x) + b * (p.w - p.z));
    gb = g * (ua * (p.z - p.x) + a * (p.w - p.y));
  } else {
    float gz = g;
    if constexpr (NODE == SLG_NODE_WALSH) {
      // y = sigmoid(z * inv_tau), z = c0 + c1 a + c2 b + c3 ab (warp.py:14-31)
      const float y = sigmoid_hw(bilinear(a, b, p) * inv_tau);
      gz = g * (y * (1.0f - y)) * inv_tau;
    }
    gp[0] = gz;
    gp[1] = gz * a;
    gp[2] = gz * b;
    gp[3] = gz * (a * b);
    ga = gz * (p.y + p.w * b);
    gb = gz * (p.z + p.w * a);
  }
}

// gw [OUT,2,K], gnp [OUT,4] (either may be null) from the partials
// part [NR][2K+4][OUT] of the sample ranges (NR = 0: zeros).
void fc_bwd_reduce(const float* part, int NR, int64_t OUT, int K, float* gw, float* gnp, hipStream_t st);

}  // namespace slg
