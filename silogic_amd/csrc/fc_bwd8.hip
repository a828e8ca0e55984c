// FC soft backward from an input kept in 8 bits (rows8.h): the gradients of
// slg_fc_soft_bwd at xq[b][i] = lo[b] + step[b] * q[b][i].
//
//   A[b,o]    = sum_k w_a xq[b, ca]   = lo W_a + step * sum_k w_a q[b, ca],   W_a = sum_k w_a
//   gw_a[o,k] = sum_b ga xq[b, ca]    = sum_b ga lo + sum_b (ga step) q[b, ca]
//
// so the gathers read codes and the offsets and steps stay scalars of a
// sample. Operands, operand gradients and every sum are fp32.
//
// A 32-bit word of the codes holds an input's four samples: one LDS read
// gathers what takes a 16-byte one in fp32, the tile is a quarter of the
// LDS and a copy of a row of the codes (no transpose), and the 2K gathered
// words stay in registers from the operands to the weight gradients, where
// the fp32 kernel gathers twice.
//
// Bound by the vector units: each (sample, output) takes 2K conversions and
// 2K products twice, and the node's derivatives. 10000 -> 10000, K = 8, B =
// 4096: 113 us for the weights' part alone (1.3 G fused products and as many
// conversions), 146 with the operand gradients written too (348 MB of 575 in
// all, 3.9 TB/s, and 64% of the vector issue), where the fp32 kernel's weights'
// part takes 318. Halves multiplied straight from registers (fp16 of the codes
// by a byte permutation, mixed-precision products) took the same time with
// fewer instructions; kept from the operands to the weights they spilled (482
// us). The next tile's gy and rows loaded before this one's stores, so that no
// load waits for a store, took 131 us and 169.
#include <algorithm>

#include "fc_bwd_input.h"
#include "fc_bwd_weights.h"
#include "fc_soft_common.h"
#include "rows8.h"

namespace slg {

// Candidate slots of a thread: those past K have input 0 and weight 0, which the
// codes, always finite, leave without a trace; a loop that skips them (16
// slots, 512 threads of twice the registers) only past 8. Weights' part, us,
// against that loop for any K: 10000 -> 10000, B = 4096, K = 8 110 for 218; 16380
// -> 16380, B = 1024, K = 4 45 for 91; 8000 -> 8000, B = 1024, K = 1 22 for 39, 2 25
// for 44, 3 24 for 43, 5 36 for 52, 7 37 for 56. With 512 threads K = 8 and 4 took
// 145 and 71, the loop with 1024 118 for 52 at K = 5.
constexpr int bwd8_slots(int K) { return K <= 1 ? 1 : K <= 2 ? 2 : K <= 4 ? 4 : K <= 8 ? 8 : 16; }
constexpr int bwd8_threads(int KM) { return KM <= 8 ? 1024 : 512; }

// The four codes of a word as floats (v_cvt_f32_ubyte0..3).
__device__ inline float code_of(uint32_t w, int v) { return (float)((w >> (8 * v)) & 255u); }

// One output per thread over a range of 4-sample tiles: part and gbr as
// fc_soft_bwd_w_kernel writes them. AHEAD: two tiles in LDS, the next one's
// codes on their way in registers (up to bwd8_quads quads a thread) while this
// one computes, one barrier a tile; else one tile and two barriers.
constexpr int bwd8_quads(int KM) { return KM == 8 ? 3 : KM == 4 ? 5 : 8; }
template <int NODE, int KM, bool AHEAD>
__global__ void __launch_bounds__(bwd8_threads(KM))
fc_bwd8_w_kernel(const uint32_t* __restrict__ codes, const float* __restrict__ rows, int B, int IN, int ld,
                 int OUT, int K, ParamView pv, float inv_tau, const float* __restrict__ gy, int n_orange,
                 int n_range, int tiles_per_range, float* __restrict__ part, float* __restrict__ gbr) {
  constexpr int S = kRows8Tile, NQ = bwd8_quads(KM);
  constexpr bool SKIP = KM > 8;  // more slots to skip than the branches cost
  extern __shared__ __align__(16) unsigned char smem[];
  // the output ranges of one sample range on one XCD: they stage the same codes
  const uint32_t lid = xcd_logical_id(blockIdx.x, gridDim.x);
  const int r_o = (int)(lid % (uint32_t)n_orange);
  const int r_b = (int)(lid / (uint32_t)n_orange);
  if (r_b >= n_range) return;  // the grid is padded to a multiple of 8
  const int o = r_o * blockDim.x + threadIdx.x;
  const bool valid = o < OUT;
  FcParams<KM> P;
  if (K == KM) load_params<KM, KM, false>(P, min(o, OUT - 1), K, pv);
  else load_params<0, KM, false>(P, min(o, OUT - 1), K, pv);  // free slots: input 0, weight 0
  const uint32_t lim = (uint32_t)IN - 1u;
  uint32_t pk[KM];  // index pairs (inputs below 65536), clamped into the tile
  float Wa = 0.0f, Wb = 0.0f;
#pragma unroll
  for (int k = 0; k < KM; ++k) {
    pk[k] = min((uint32_t)P.ia[k], lim) | (min((uint32_t)P.ib[k], lim) << 16);
    Wa += P.fa[k];
    Wb += P.fb[k];
  }
  float swa[KM], swb[KM], sp[4] = {0.f, 0.f, 0.f, 0.f}, sla = 0.0f, slb = 0.0f;
#pragma unroll
  for (int k = 0; k < KM; ++k) swa[k] = swb[k] = 0.0f;
  const int n_tiles = (B + S - 1) / S;
  const int t0 = r_b * tiles_per_range, t_end = min(n_tiles, t0 + tiles_per_range);
  const int vo = valid ? o * 4 : 0x7ffffffc, n4 = ld >> 2, T = blockDim.x;
  uint4 pf[AHEAD ? NQ : 1];
  auto issue = [&](int t) {
    const auto r = uniform_rsrc(codes + (int64_t)t * ld, ld * 4);
#pragma unroll
    for (int u = 0; u < NQ; ++u)  // zeros past the row
      pf[u] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, (threadIdx.x + u * T) * 16, 0, 0));
  };
  auto place = [&](int t) {
    uint4* dst = reinterpret_cast<uint4*>(smem) + (t & 1) * n4;
#pragma unroll
    for (int u = 0; u < NQ; ++u) {
      const int q = threadIdx.x + u * T;
      if (q < n4) dst[q] = pf[u];
    }
  };
  auto load_g = [&](int t, float (&g)[S]) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int b = t * S + s;
      const auto gr = uniform_rsrc(gy + (int64_t)min(b, B - 1) * OUT, b < B ? OUT * 4 : 0);
      g[s] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(gr, vo, 0, 0));
    }
  };
  if constexpr (AHEAD) {
    if (t0 < t_end) {
      issue(t0);
      place(t0);
      __syncthreads();
    }
  }
  for (int t = t0; t < t_end; ++t) {
    const int b0 = t * S;
    float g[S], lo[S], step[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int64_t b = min(b0 + s, B - 1);
      lo[s] = b0 + s < B ? rows[2 * b] : 0.0f;
      step[s] = b0 + s < B ? rows[2 * b + 1] : 0.0f;
    }
    const uint32_t* xs = reinterpret_cast<const uint32_t*>(smem) + (AHEAD ? (t & 1) * ld : 0);
    if constexpr (!AHEAD) {
      __syncthreads();  // the previous tile's reads are done
      const uint4* src = reinterpret_cast<const uint4*>(codes + (int64_t)t * ld);
      for (int q = threadIdx.x; q < n4; q += T) reinterpret_cast<uint4*>(smem)[q] = src[q];
      __syncthreads();
    }
    load_g(t, g);  // back by the time the operands are there
    if constexpr (AHEAD) {
      if (t + 1 < t_end) issue(t + 1);
    }
    uint32_t qa[KM], qb[KM];
#pragma unroll
    for (int k = 0; k < KM; ++k) {
      if (!SKIP || k < K) {
        qa[k] = xs[pk[k] & 0xffffu];
        qb[k] = xs[pk[k] >> 16];
      }
    }
    float A[S] = {0.f, 0.f, 0.f, 0.f}, Bv[S] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < KM; ++k) {
      if (!SKIP || k < K) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
          A[s] = fmaf(P.fa[k], code_of(qa[k], s), A[s]);
          Bv[s] = fmaf(P.fb[k], code_of(qb[k], s), Bv[s]);
        }
      }
    }
    // converted again for the weight gradients: 64 floats kept would spill
#pragma unroll
    for (int k = 0; k < KM; ++k) asm volatile("" : "+v"(qa[k]), "+v"(qb[k]));
    float ga[S], gb[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      float gp[4];
      node_grad<NODE>(fmaf(step[s], A[s], lo[s] * Wa), fmaf(step[s], Bv[s], lo[s] * Wb), g[s], P.p,
                      inv_tau, ga[s], gb[s], gp);
#pragma unroll
      for (int q = 0; q < 4; ++q) sp[q] += gp[q];
    }
    if (gbr != nullptr) {  // sample rows of 2*OUT; outputs past OUT are not stored
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const auto gr = uniform_rsrc(gbr + (int64_t)(b0 + s) * (2 * OUT), OUT * 8);
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(ga[s]), gr, vo, 0, 0);
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(gb[s]), gr, valid ? vo + OUT * 4 : vo, 0, 0);
      }
    }
#pragma unroll
    for (int s = 0; s < S; ++s) {
      sla = fmaf(ga[s], lo[s], sla);
      slb = fmaf(gb[s], lo[s], slb);
      ga[s] *= step[s];
      gb[s] *= step[s];
    }
#pragma unroll
    for (int k = 0; k < KM; ++k) {
      if (!SKIP || k < K) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
          swa[k] = fmaf(ga[s], code_of(qa[k], s), swa[k]);
          swb[k] = fmaf(gb[s], code_of(qb[k], s), swb[k]);
        }
      }
    }
    if constexpr (AHEAD) {  // the other tile's reads ended at the last barrier
      if (t + 1 < t_end) place(t + 1);
      __syncthreads();
    }
  }
  if (part != nullptr && valid) {
    float* base = part + (int64_t)r_b * (2 * K + 4) * OUT + o;
#pragma unroll
    for (int k = 0; k < KM; ++k) {
      if (k < K) {
        base[(int64_t)k * OUT] = swa[k] + sla;
        base[(int64_t)(K + k) * OUT] = swb[k] + slb;
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) base[(int64_t)(2 * K + q) * OUT] = sp[q];
  }
}

// From the sample ranges' partials to the gradients of a layer's own
// parameters in one launch: the sums over ranges, the connection softmax's
// chain rule and the node's. A workgroup takes 16 outputs; a wave a component
// at a time, its lanes 16 outputs by 4 parts of the ranges (each part
// ascending, the parts added in order of a butterfly), so that a narrow layer
// with many ranges is not walked by one lane. 9.6 us at 16000 outputs with 8
// candidates; as two launches through memory (the sums, then
// slg_layer_params_bwd) 14 us.
constexpr int kPbThreads = 1024, kPbOut = 16;
template <int NODE>
__global__ void __launch_bounds__(kPbThreads)
fc_bwd8_params_kernel(const float* __restrict__ part, int NR, int OUT, int K, const float* __restrict__ w,
                      const float* __restrict__ kept, float* __restrict__ gconn, float* __restrict__ graw) {
  __shared__ float g[36][kPbOut + 1];  // 2 K + 4 components
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int o0 = blockIdx.x * kPbOut, n = 2 * K + 4;
  const int o = min(o0 + (lane & 15), OUT - 1);
  for (int c = wave; c < n; c += kPbThreads / 64) {
    float sum = 0.0f;
    for (int r0 = lane >> 4; r0 < NR; r0 += 32) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = part[((int64_t)min(r0 + 4 * u, NR - 1) * n + c) * OUT + o];
#pragma unroll
      for (int u = 0; u < 8; ++u) sum += r0 + 4 * u < NR ? v[u] : 0.0f;
    }
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (lane < kPbOut) g[c][lane] = sum;
  }
  __syncthreads();
  if (tid < 2 * kPbOut) {  // a softmax row: an output's operand
    const int side = tid / kPbOut, l = tid % kPbOut;
    if (gconn && o0 + l < OUT) {
      const int64_t at = ((int64_t)(o0 + l) * 2 + side) * K;
      float dot = 0.0f;
      for (int k = 0; k < K; ++k) dot = fmaf(w[at + k], g[side * K + k][l], dot);
      for (int k = 0; k < K; ++k) gconn[at + k] = w[at + k] * (g[side * K + k][l] - dot);
    }
  } else if (tid >= 64 && tid < 64 + kPbOut) {
    const int l = tid - 64;
    if (graw && o0 + l < OUT) {
      const int64_t out = o0 + l;
      const float q0 = g[2 * K][l], q1 = g[2 * K + 1][l], q2 = g[2 * K + 2][l], q3 = g[2 * K + 3][l];
      if constexpr (NODE == SLG_NODE_GATE16) {
        // gate i's values by the bits of i: f(a, b) = bit 3 - (2 a + b), in {1, a, b, ab}
        const float* p = kept + 4 * (int64_t)OUT + 16 * out;
        float d[16], dot = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int f0 = (i >> 3) & 1, f1 = (i >> 2) & 1, f2 = (i >> 1) & 1, f3 = i & 1;
          d[i] = f0 * q0 + (f2 - f0) * q1 + (f1 - f0) * q2 + (f3 - f2 - f1 + f0) * q3;
          dot = fmaf(p[i], d[i], dot);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) graw[16 * out + i] = p[i] * (d[i] - dot);
      } else if constexpr (NODE == SLG_NODE_WALSH) {
        graw[4 * out] = q0;
        graw[4 * out + 1] = 2.0f * q1 - q0;
        graw[4 * out + 2] = 2.0f * q2 - q0;
        graw[4 * out + 3] = q0 + 4.0f * q3 - 2.0f * (q1 + q2);
      } else {
        const float q[4] = {q0, q1, q2, q3};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = kept[4 * out + i];
          graw[4 * out + i] = q[i] * (v * (1.0f - v));
        }
      }
    }
  }
}

// Workspace (in 4-byte words): partials | operand gradients | input-gradient part.
struct Bwd8Plan {
  int threads, n_orange, NR, tiles_per_range;
  int64_t part, gbr, in_ws;
  int64_t total() const { return part + gbr + in_ws; }
};

static int64_t bwd8_lds_cap() { return std::min<int64_t>(device_lds_bytes(), 160 * 1024); }

static bool bwd8_takes(int64_t B, int64_t IN, int64_t OUT, int K) {
  return B >= 0 && B < (1LL << 31) - 8 && IN > 0 && OUT > 0 && OUT < (1LL << 28) && K >= 1 && K <= 16 &&
         2 * OUT * K < (1LL << 31) && rows8_ld(IN) * 4 <= bwd8_lds_cap() && B * IN < (1LL << 40);
}

static Bwd8Plan bwd8_plan(int64_t B, int64_t IN, int64_t OUT, int K) {
  Bwd8Plan p{};
  p.threads = bwd8_threads(bwd8_slots(K));
  p.n_orange = (int)cdiv(OUT, p.threads);
  const int64_t n_tiles = cdiv(std::max<int64_t>(B, 1), kRows8Tile);
  // one round of workgroups: as many sample ranges as resident slots allow
  const int64_t per_cu = std::max<int64_t>(1, std::min<int64_t>(1024 / p.threads, 160 * 1024 / (rows8_ld(IN) * 4)));
  const int64_t slots = per_cu * device_cus();
  p.NR = (int)std::max<int64_t>(1, std::min<int64_t>(n_tiles, slots / p.n_orange));
  p.tiles_per_range = (int)cdiv(n_tiles, p.NR);
  p.NR = (int)cdiv(n_tiles, p.tiles_per_range);
  auto round4 = [](int64_t n) { return (n + 3) & ~int64_t(3); };
  p.part = round4((int64_t)p.NR * (2 * K + 4) * OUT);
  p.gbr = round4(2 * OUT * n_tiles * kRows8Tile);  // the last tile's rows whole
  p.in_ws = fc_input_grad_floats(B, IN, OUT, 2, K);
  return p;
}

struct Bwd8Args {
  const uint32_t* codes;
  const float* rows;
  int64_t B, IN, OUT;
  int K;
  const int* cand;
  const float *w, *np;
  float inv_tau;
  const float* gy;
  float *part, *gbr;
};

template <int NODE, int KM>
static int launch_bwd8(const Bwd8Args& a, const Bwd8Plan& p, hipStream_t st) {
  const int64_t ld = rows8_ld(a.IN);
  const bool ahead = p.tiles_per_range > 1 && ld <= bwd8_quads(KM) * 4 * bwd8_threads(KM) &&
                     ld * 8 <= bwd8_lds_cap();
  auto kern = ahead ? fc_bwd8_w_kernel<NODE, KM, true> : fc_bwd8_w_kernel<NODE, KM, false>;
  const size_t lds = (size_t)ld * 4 * (ahead ? 2 : 1);
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)lds);
    SLG_REQUIRE(e == hipSuccess, (int)e, "fc_soft_bwd8: LDS %zu: %s", lds, hipGetErrorString(e));
  }
  // a thread reads its output's parameters once, from where they are: records
  // (as the fp32 kernels take) would be a launch and 5 us to save less
  const ParamView pv{a.cand, a.cand + a.K, a.w, a.w + a.K, a.np, 2 * a.K, 2 * a.K, 4, nullptr};
  hipLaunchKernelGGL(kern, dim3((unsigned)(cdiv((int64_t)p.n_orange * p.NR, 8) * 8)), dim3(bwd8_threads(KM)),
                     lds, st, a.codes, a.rows, (int)a.B, (int)a.IN, (int)ld, (int)a.OUT, a.K, pv,
                     a.inv_tau, a.gy, p.n_orange, p.NR, p.tiles_per_range, a.part, a.gbr);
  SLG_LAUNCH_CHECK("fc_soft_bwd8");
  return 0;
}

template <int NODE>
static int launch_bwd8_k(const Bwd8Args& a, const Bwd8Plan& p, hipStream_t st) {
  switch (bwd8_slots(a.K)) {
    case 1: return launch_bwd8<NODE, 1>(a, p, st);  // fixed wiring
    case 2: return launch_bwd8<NODE, 2>(a, p, st);
    case 4: return launch_bwd8<NODE, 4>(a, p, st);
    case 8: return launch_bwd8<NODE, 8>(a, p, st);
    default: return launch_bwd8<NODE, 16>(a, p, st);
  }
}

// Checks, the weight kernel and the input gradient: partials of the weights'
// and node parameters' gradients (want_w) at the workspace's start, p.NR of
// them (none for an empty batch).
static int bwd8_run(Bwd8Args a, int node_kind, bool want_w, float* gx, float* workspace, int64_t workspace_floats,
                    hipStream_t st, Bwd8Plan& p) {
  SLG_REQUIRE(a.cand && a.w && a.np && workspace && ((a.codes && a.rows && a.gy) || a.B == 0), SLG_E_ARG,
              "fc_soft_bwd8: null pointer");
  SLG_REQUIRE(node_kind == SLG_NODE_GATE16 || node_kind == SLG_NODE_WALSH ||
                  node_kind == SLG_NODE_MULTILINEAR2,
              SLG_E_ARG, "fc_soft_bwd8: node_kind %d", node_kind);
  SLG_REQUIRE(bwd8_takes(a.B, a.IN, a.OUT, a.K), SLG_E_SHAPE, "fc_soft_bwd8: B %lld, IN %lld, OUT %lld, K %d",
              (long long)a.B, (long long)a.IN, (long long)a.OUT, a.K);
  SLG_REQUIRE((((uintptr_t)a.codes | (uintptr_t)a.cand | (uintptr_t)a.w | (uintptr_t)a.np |
                (uintptr_t)workspace) & 15) == 0,
              SLG_E_ARG, "fc_soft_bwd8: codes, cand, w, node_param or workspace not at a multiple of 16 bytes");
  p = bwd8_plan(a.B, a.IN, a.OUT, a.K);
  SLG_REQUIRE(workspace_floats >= p.total(), SLG_E_ARG, "fc_soft_bwd8: workspace of %lld floats, %lld needed",
              (long long)workspace_floats, (long long)p.total());
  if (a.B == 0) {  // no samples: zero gradients
    p.NR = 0;
    return 0;
  }
  if (!want_w && !gx) return 0;
  float* gbr = workspace + p.part;
  a.part = want_w ? workspace : nullptr;
  a.gbr = gx ? gbr : nullptr;
  const int rc = node_kind == SLG_NODE_GATE16  ? launch_bwd8_k<SLG_NODE_GATE16>(a, p, st)
                 : node_kind == SLG_NODE_WALSH ? launch_bwd8_k<SLG_NODE_WALSH>(a, p, st)
                                               : launch_bwd8_k<SLG_NODE_MULTILINEAR2>(a, p, st);
  return rc || !gx ? rc : fc_input_grad(gbr, a.B, a.IN, a.OUT, 2, a.K, a.cand, a.w, gbr + p.gbr, gx, st);
}

}  // namespace slg

using namespace slg;

extern "C" {

int64_t slg_fc_soft_bwd8_workspace(int64_t B, int64_t IN, int64_t OUT, int32_t K) {
  return bwd8_takes(B, IN, OUT, K) ? bwd8_plan(B, IN, OUT, K).total() : -1;
}

int slg_fc_soft_bwd8(const uint8_t* codes, const float* rows, int64_t B, int64_t IN, int64_t OUT, int32_t K,
                     const int32_t* cand, const float* w, int32_t node_kind, const float* node_param,
                     float inv_tau, const float* gy, float* gx, float* gw, float* gnp, float* workspace,
                     int64_t workspace_floats, slg_stream_t stream) {
  const Bwd8Args a{reinterpret_cast<const uint32_t*>(codes), rows, B, IN, OUT, K, cand, w, node_param, inv_tau,
                   gy, nullptr, nullptr};
  Bwd8Plan p{};
  const int rc = bwd8_run(a, node_kind, gw || gnp, gx, workspace, workspace_floats, as_stream(stream), p);
  if (rc || !(gw || gnp)) return rc;
  fc_bwd_reduce(workspace, p.NR, OUT, K, gw, gnp, as_stream(stream));
  SLG_LAUNCH_CHECK("fc_soft_bwd8 sums");
  return 0;
}

int64_t slg_fc_layer8_fwd_workspace(int64_t B, int64_t IN, int64_t OUT, int32_t K) {
  return fc_soft8_rec_floats(B, IN, OUT, K);
}

int slg_fc_layer8_fwd(const float* x, int64_t B, int64_t IN, int64_t OUT, int32_t K, const int32_t* cand,
                      const float* conn, const float* raw, int32_t node_kind, float inv_tau, float* y,
                      uint8_t* codes, float* rows, float* w, float* kept, float* workspace, int64_t workspace_floats,
                      slg_stream_t stream) {
  SLG_REQUIRE(cand && raw && w && kept, SLG_E_ARG, "fc_layer8_fwd: null pointer");
  SLG_REQUIRE(node_kind == SLG_NODE_GATE16 || node_kind == SLG_NODE_WALSH ||
                  node_kind == SLG_NODE_MULTILINEAR2,
              SLG_E_ARG, "fc_layer8_fwd: node_kind %d", node_kind);
  SLG_REQUIRE(K >= 1 && K <= 16 && OUT > 0 && OUT < (1LL << 28) && 2 * OUT * K < (1LL << 31), SLG_E_SHAPE,
              "fc_layer8_fwd: OUT %lld, K %d", (long long)OUT, K);
  const int32_t one = 1;
  const int rc = slg_layer_params(conn, 2 * OUT, K, 1, &raw, &one, OUT, node_kind, 2, 1.0f, w, kept,
                                  node_kind == SLG_NODE_GATE16 ? kept + 4 * OUT : nullptr, stream);
  if (rc) return rc;
  const int64_t rec = fc_soft8_rec_floats(B, IN, OUT, K);
  SLG_REQUIRE(workspace_floats >= rec && (rec == 0 || (workspace && (uintptr_t)workspace % 16 == 0)), SLG_E_ARG,
              "fc_layer8_fwd: workspace of %lld floats, %lld at a multiple of 16 bytes needed",
              (long long)workspace_floats, (long long)rec);
  return fc_soft_fwd8(x, B, IN, OUT, K, cand, w, node_kind, kept, inv_tau, y, codes, rows, rec ? workspace : nullptr,
                      as_stream(stream));
}

int64_t slg_fc_layer8_bwd_workspace(int64_t B, int64_t IN, int64_t OUT, int32_t K) {
  return slg_fc_soft_bwd8_workspace(B, IN, OUT, K);
}

int slg_fc_layer8_bwd(const uint8_t* codes, const float* rows, int64_t B, int64_t IN, int64_t OUT, int32_t K,
                      const int32_t* cand, const float* w, const float* kept, int32_t node_kind, float inv_tau,
                      const float* gy, float* gx, float* gconn, float* graw, float* workspace,
                      int64_t workspace_floats, slg_stream_t stream) {
  const Bwd8Args a{reinterpret_cast<const uint32_t*>(codes), rows, B, IN, OUT, K, cand, w, kept, inv_tau, gy,
                   nullptr, nullptr};
  Bwd8Plan p{};
  hipStream_t st = as_stream(stream);
  const int rc = bwd8_run(a, node_kind, gconn || graw, gx, workspace, workspace_floats, st, p);
  if (rc || !(gconn || graw)) return rc;
  auto kern = node_kind == SLG_NODE_GATE16  ? fc_bwd8_params_kernel<SLG_NODE_GATE16>
              : node_kind == SLG_NODE_WALSH ? fc_bwd8_params_kernel<SLG_NODE_WALSH>
                                            : fc_bwd8_params_kernel<SLG_NODE_MULTILINEAR2>;
  hipLaunchKernelGGL(kern, dim3((unsigned)cdiv(OUT, kPbOut)), dim3(kPbThreads), 0, st, workspace, p.NR, (int)OUT,
                     K, w, kept, gconn, graw);
  SLG_LAUNCH_CHECK("fc_layer8_bwd parameters");
  return 0;
}

}  // extern "C"
