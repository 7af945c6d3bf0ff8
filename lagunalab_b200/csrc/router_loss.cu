// The router's balance loss with its counts, and the gradient of the router's logits.
//
// Scores s_te = softmax or sigmoid of the logits [T, E], as lg_router_topk takes them; shares
// q_te = s_te / sum_e s_te (softmax: s itself). Over the N tokens that the mask keeps:
//   counts_e = picks of e,  f_e = counts_e / sum counts,  P_e = sum_t q_te / N,  loss = E sum_e f_e P_e.
// Its gradient goes through P alone (counts have none):  dq_e = c E f_e / N,
//   softmax: dl = s (dq - sum q dq),   sigmoid: dl = s (1 - s) (dq - sum q dq) / sum_e s.
// Routing weights w_j = s_j / sum over the token's picks of s (norm) or s_j, for dw given:
//   ds_j = (dw_j - sum_i dw_i w_i) / sum s (norm) or dw_j;  a sigmoid's or softmax's backward from there.
//
// A warp a token, E / 32 scores a lane in registers. Both kernels read the logits once and are bound by
// HBM on long batches, by launch latency on short ones.
#include <math.h>

#include <algorithm>

#include "common.cuh"

namespace lg {

constexpr int RB_WARPS = 32;       // warps a CTA of the balance
constexpr int RG_WARPS = 16;       // and of the gradient
constexpr int RB_MAXE = 256;
constexpr int RB_CTA_TOKENS = 64;  // a CTA for so many tokens, up to RB_CTAS: the join reads all of them at once
constexpr int RB_CTAS = 144;
constexpr float RB_LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float rb_exp(float x) {  // within 2^-22 + |x| 2^-23
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * RB_LOG2E));
  return y;
}

// The token's scores in place of its logits (0 past E), and their sum over the experts. For a sigmoid `tail` is
// s (1 - s), without the difference that cancels.
template <int N, bool TAIL>
__device__ __forceinline__ float rb_scores(float (&v)[N], float (&tail)[N], int E, int score_fn) {
  const int lane = threadIdx.x & 31;
  float sum = 0.f;
  if (score_fn == LG_SCORE_SOFTMAX) {
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < N; ++j) mx = fmaxf(mx, v[j]);
    mx = warp_max(mx);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      v[j] = lane + 32 * j < E ? rb_exp(v[j] - mx) : 0.f;
      sum += v[j];
    }
    const float r = 1.f / warp_sum(sum);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] *= r;
    return 1.f;
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float t = rb_exp(-fabsf(v[j]));  // NaN stays
    const float r = __fdividef(1.f, 1.f + t);
    if (TAIL) tail[j] = t * r * r;
    v[j] = lane + 32 * j < E ? (v[j] >= 0.f ? r : t * r) : 0.f;
    sum += v[j];
  }
  return warp_sum(sum);
}

template <int N>
__device__ __forceinline__ void rb_load(float (&v)[N], const float* row, int E) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = lane + 32 * j < E ? __ldg(row + lane + 32 * j) : -INFINITY;
}

struct RbOut {
  float* loss;
  int* counts;
  float* probs;
  int* tokens;
};

// The sums of one expert over all tokens -> outputs; called by whole CTAs of at least E threads.
__device__ __forceinline__ void rb_finish(float prob, int count, int n, int E, const RbOut& o) {
  __shared__ float sh_f[32];
  __shared__ long long sh_c[32];
  const int e = threadIdx.x, lane = e & 31, warp = e >> 5;
  const float p = n > 0 ? prob / (float)n : 0.f;
  if (e < E) {
    o.counts[e] = count;
    o.probs[e] = p;
  }
  if (e >= E) count = 0;
  float fp = e < E ? (float)count * p : 0.f;
  long long c = count;
  fp = warp_sum(fp);
#pragma unroll
  for (int s = 16; s; s >>= 1) c += __shfl_xor_sync(0xffffffffu, c, s);
  if (lane == 0) {
    sh_f[warp] = fp;
    sh_c[warp] = c;
  }
  __syncthreads();
  if (e == 0) {
    float f = 0.f;
    long long all = 0;
    for (int i = 0; i < (int)(blockDim.x + 31) / 32; ++i) {
      f += sh_f[i];
      all += sh_c[i];
    }
    *o.loss = all > 0 ? (float)E * f / (float)all : 0.f;
    *o.tokens = n;
  }
}

// Each CTA's sums over its tokens; a grid of one CTA writes the outputs itself. A warp has four tokens' logits in
// flight, whatever the mask says of them (a load that waits for the mask costs a second trip to memory).
template <int N>
__global__ void __launch_bounds__(RB_WARPS * 32) router_balance_kernel(
    const float* __restrict__ logits, const int* __restrict__ inds, const uint8_t* __restrict__ mask, int T,
    int E, int k, int score_fn, float* __restrict__ part_p, int* __restrict__ part_c, RbOut o) {
  constexpr int U = N > 4 ? 2 : 4;
  __shared__ float sum_p[RB_WARPS][32 * N];
  __shared__ int hist[RB_MAXE + 1];  // the last: tokens kept
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i <= RB_MAXE; i += blockDim.x) hist[i] = 0;
  __syncthreads();
  float acc[N] = {};
  int kept = 0;
  const int step = gridDim.x * RB_WARPS;
  for (int t0 = blockIdx.x * RB_WARPS + warp; t0 < T; t0 += U * step) {
    float v[U][N], unused[N];
    int pick[U];
    bool keep[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u * step;
      keep[u] = t < T;
      pick[u] = -1;
      if (keep[u]) {
        rb_load<N>(v[u], logits + (size_t)t * E, E);
        if (lane < k) pick[u] = inds[(size_t)t * k + lane];
        if (mask) keep[u] = mask[t];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!keep[u]) continue;
      if (pick[u] >= 0 && pick[u] < E) atomicAdd(&hist[pick[u]], 1);
      ++kept;
      const float r = 1.f / rb_scores<N, false>(v[u], unused, E, score_fn);
#pragma unroll
      for (int j = 0; j < N; ++j) acc[j] = fmaf(v[u][j], r, acc[j]);
    }
  }
  pdl_trigger();
#pragma unroll
  for (int j = 0; j < N; ++j) sum_p[warp][lane + 32 * j] = acc[j];
  if (lane == 0) atomicAdd(&hist[RB_MAXE], kept);
  __syncthreads();
  const int e = threadIdx.x;
  float p = 0.f;
  if (e < 32 * N) {
#pragma unroll
    for (int w = 0; w < RB_WARPS; ++w) p += sum_p[w][e];
  }
  if (gridDim.x == 1) {
    rb_finish(p, e < E ? hist[e] : 0, hist[RB_MAXE], E, o);
  } else {
    if (e < E) {
      part_p[(size_t)blockIdx.x * E + e] = p;
      part_c[(size_t)blockIdx.x * E + e] = hist[e];
    }
    if (e == E) part_c[(size_t)RB_CTAS * E + blockIdx.x] = hist[RB_MAXE];
  }
}

// Joins the CTAs' sums, in their order: 1,024 threads, 256 a quarter of the CTAs, each with all of its loads in
// flight.
__global__ void __launch_bounds__(1024) router_balance_join_kernel(const float* __restrict__ part_p,
                                                                   const int* __restrict__ part_c, int C,
                                                                   int E, RbOut o) {
  constexpr int PER = RB_CTAS / 4, HALF = PER / 2;
  __shared__ float sp[4][RB_MAXE];
  __shared__ int sc[4][RB_MAXE];
  __shared__ int sn[32];
  pdl_wait();
  const int e = threadIdx.x & 255, s = threadIdx.x >> 8;
  float p = 0.f;
  int c = 0;
#pragma unroll 1
  for (int h = 0; h < 2; ++h) {
    const int a = s * PER + h * HALF;
    float pv[HALF];
    int cv[HALF];
#pragma unroll
    for (int i = 0; i < HALF; ++i) {
      const bool in = e < E && a + i < C;
      pv[i] = in ? part_p[(size_t)(a + i) * E + e] : 0.f;
      cv[i] = in ? part_c[(size_t)(a + i) * E + e] : 0;
    }
#pragma unroll
    for (int i = 0; i < HALF; ++i) {
      p += pv[i];
      c += cv[i];
    }
  }
  sp[s][e] = p;
  sc[s][e] = c;
  int n = threadIdx.x < C ? part_c[(size_t)RB_CTAS * E + threadIdx.x] : 0;
#pragma unroll
  for (int i = 16; i; i >>= 1) n += __shfl_xor_sync(0xffffffffu, n, i);
  if ((threadIdx.x & 31) == 0) sn[threadIdx.x >> 5] = n;
  __syncthreads();
  const bool first = s == 0;
  p = first ? sp[0][e] + sp[1][e] + sp[2][e] + sp[3][e] : 0.f;
  c = first ? sc[0][e] + sc[1][e] + sc[2][e] + sc[3][e] : 0;
  n = 0;
#pragma unroll
  for (int i = 0; i < (RB_CTAS + 31) / 32; ++i) n += sn[i];
  rb_finish(p, c, n, E, o);
}

struct RgArgs {
  const float* logits;
  const int* inds;
  const float* dw;  // [T, k] or NULL
  const uint8_t* mask;
  const int* counts;  // NULL: no balance loss
  const int* tokens;
  float weight;
  int T, E, k, norm, score_fn;
  float* dl;
};

template <int N>
__global__ void __launch_bounds__(RG_WARPS * 32) router_grad_kernel(const RgArgs a) {
  __shared__ float sh_s[RG_WARPS][32 * N];  // a token's scores, for its picks
  __shared__ float sh_d[RG_WARPS][32 * N];  // its picks' gradients; zeros between tokens
  __shared__ int sh_t[RG_WARPS][32 * N];    // which pick has an expert
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float *ss = sh_s[warp], *sd = sh_d[warp];
  int* st = sh_t[warp];
  float dq[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    sd[lane + 32 * j] = 0.f;
    dq[j] = 0.f;
  }
  if (a.counts) {
    int c[N];
    long long all = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      c[j] = lane + 32 * j < a.E ? a.counts[lane + 32 * j] : 0;
      all += c[j];
    }
#pragma unroll
    for (int s = 16; s; s >>= 1) all += __shfl_xor_sync(0xffffffffu, all, s);
    const int n = *a.tokens;
    const float f = all > 0 && n > 0 ? a.weight * (float)a.E / ((float)all * (float)n) : 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) dq[j] = f * (float)c[j];
  }
  __syncwarp();
  for (int t = blockIdx.x * RG_WARPS + warp; t < a.T; t += gridDim.x * RG_WARPS) {
    float* out = a.dl + (size_t)t * a.E;
    if (a.mask && !a.mask[t]) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (lane + 32 * j < a.E) out[lane + 32 * j] = 0.f;
      continue;
    }
    float s[N], tail[N];
    rb_load<N>(s, a.logits + (size_t)t * a.E, a.E);
    int id = -1;
    float d = 0.f;
    if (a.dw && lane < a.k) {
      id = a.inds[(size_t)t * a.k + lane];
      if (id >= a.E) id = -1;
      d = a.dw[(size_t)t * a.k + lane];
    }
    const float total = rb_scores<N, true>(s, tail, a.E, a.score_fn);
    float pick = 0.f;  // softmax: sum_e s_e ds_e
    if (a.dw) {
#pragma unroll
      for (int j = 0; j < N; ++j) ss[lane + 32 * j] = s[j];
      __syncwarp();
      if (id >= 0) st[id] = lane;
      const float p = id >= 0 ? ss[id] : 0.f;
      const float dot = warp_sum(id >= 0 ? d * p : 0.f);
      if (a.norm) {
        const float r = 1.f / warp_sum(p);
        d = (d - dot * r) * r;
      } else {
        pick = dot;
      }
      __syncwarp();
      const bool twice = id >= 0 && st[id] != lane;
      if (__any_sync(0xffffffffu, twice)) {  // an expert picked twice: its gradients in their order
        for (int j = 0; j < a.k; ++j) {
          if (lane == j && id >= 0) sd[id] += d;
          __syncwarp();
        }
      } else if (id >= 0) {
        sd[id] = d;
      }
      __syncwarp();
    }
    float mean = 0.f;
    if (a.counts) {
#pragma unroll
      for (int j = 0; j < N; ++j) mean = fmaf(s[j], dq[j], mean);
      mean = warp_sum(mean) / total;
    }
    const float r = 1.f / total;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int e = lane + 32 * j;
      float ds = a.dw ? sd[e] : 0.f;
      float g;
      if (a.score_fn == LG_SCORE_SOFTMAX) {
        if (a.counts) ds += dq[j] - mean;
        g = s[j] * (ds - pick);
      } else {
        if (a.counts) ds += (dq[j] - mean) * r;
        g = ds * tail[j];
      }
      if (e < a.E) out[e] = g;
    }
    __syncwarp();
    if (id >= 0) sd[id] = 0.f;
    __syncwarp();
  }
}

static int rb_ctas(int T) {
  return std::max(1, std::min(RB_CTAS, (T + RB_CTA_TOKENS - 1) / RB_CTA_TOKENS));
}

static int rb_check(const char* who, const void* logits, const void* inds, int T, int E, int k, int score_fn) {
  LG_CHECK_ARG(E >= 1 && E <= RB_MAXE, "%s: E=%d not in [1, %d]", who, E, RB_MAXE);
  LG_CHECK_ARG(k >= 1 && k <= 32, "%s: k=%d not in [1, 32]", who, k);
  LG_CHECK_ARG(T >= 0, "%s: T=%d", who, T);
  LG_CHECK_ARG(score_fn == LG_SCORE_SIGMOID || score_fn == LG_SCORE_SOFTMAX, "%s: score_fn %d", who, score_fn);
  LG_CHECK_ARG(T == 0 || (logits && inds), "%s: NULL pointer", who);
  return LG_OK;
}

// N: 32 * N experts a warp's registers hold
#define RB_BY_E(E, CALL)             \
  do {                               \
    if ((E) <= 32) { CALL(1); }      \
    else if ((E) <= 64) { CALL(2); } \
    else if ((E) <= 128) { CALL(4); } \
    else { CALL(8); }                \
  } while (0)

}  // namespace lg

using namespace lg;

extern "C" size_t lg_router_balance_workspace_bytes(int T, int E) {
  const size_t C = rb_ctas(T) > 1 ? RB_CTAS : 0, e = E > 0 ? E : 1;
  return align_up(C * e * 4, 256) + align_up(C * (e + 1) * 4, 256);  // 0: one CTA needs none
}

extern "C" int lg_router_balance(const float* logits, const int32_t* inds, const uint8_t* mask, int T, int E,
                                 int k, int score_fn, float* loss, int32_t* counts, float* probs,
                                 int32_t* tokens, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = rb_check("router_balance", logits, inds, T, E, k, score_fn);
  if (rc != LG_OK) return rc;
  LG_CHECK_ARG(loss && counts && probs && tokens, "router_balance: NULL output");
  const size_t need = lg_router_balance_workspace_bytes(T, E);
  if (need && (!workspace || !aligned(workspace, 256) || workspace_bytes < need))
    return fail(LG_ERR_WORKSPACE, "router_balance: workspace of %zu bytes, need %zu", workspace_bytes, need);
  const int C = rb_ctas(T);
  Carver w(workspace);
  float* pp = w.take<float>((size_t)RB_CTAS * E);
  int* pc = w.take<int>((size_t)RB_CTAS * (E + 1));
  const RbOut o = {loss, counts, probs, tokens};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define RB_CALL(N)                                                                               \
  router_balance_kernel<N><<<C, RB_WARPS * 32, 0, st>>>(logits, inds, mask, T, E, k, score_fn, pp, pc, o)
  RB_BY_E(E, RB_CALL);
#undef RB_CALL
  LG_LAUNCH_CHECK("router_balance");
  if (C > 1) {
    LG_CUDA_TRY(launch_early(router_balance_join_kernel, 1, 1024, 0, st, (const float*)pp, (const int*)pc, C, E, o));
    LG_LAUNCH_CHECK("router_balance_join");
  }
  return LG_OK;
}

extern "C" int lg_router_grad(const float* logits, const int32_t* inds, const float* dw, const uint8_t* mask,
                              int T, int E, int k, int norm_topk_prob, int score_fn, const int32_t* counts,
                              const int32_t* tokens, float weight, float* dlogits, void* stream) {
  int rc = rb_check("router_grad", logits, inds, T, E, k, score_fn);
  if (rc != LG_OK) return rc;
  LG_CHECK_ARG((counts == nullptr) == (tokens == nullptr), "router_grad: counts and tokens go together");
  if (T == 0) return LG_OK;
  LG_CHECK_ARG(dw || counts, "router_grad: neither dw nor a balance loss");
  LG_CHECK_ARG(dlogits, "router_grad: NULL output");
  const RgArgs a = {logits, inds, dw, mask, counts, tokens, weight, T, E, k, norm_topk_prob, score_fn, dlogits};
  const int grid = std::max(1, std::min(2 * device_sm_count(), (T + RG_WARPS - 1) / RG_WARPS));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define RB_CALL(N) router_grad_kernel<N><<<grid, RG_WARPS * 32, 0, st>>>(a)
  RB_BY_E(E, RB_CALL);
#undef RB_CALL
  LG_LAUNCH_CHECK("router_grad");
  return LG_OK;
}
