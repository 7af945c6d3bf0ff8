// The router's balance loss with its counts, and the gradient of the router's logits.
//
// Scores s_te = softmax or sigmoid of the logits [T, E], as lg_router_topk takes them; shares
// q_te = s_te / sum_e s_te (softmax: s itself). Over the N tokens that the mask keeps:
//   counts_e = picks of e,  f_e = counts_e / sum counts,  P_e = sum_t q_te / N,  loss = E sum_e f_e P_e.
// Its gradient goes through P alone (counts have none):  dq_e = c E f_e / N,
//   softmax: dl = s (dq - sum q dq),   sigmoid: dl = s (1 - s) (dq - sum q dq) / sum_e s.
// Routing weights w_j = s_j / sum over the token's picks of s (norm) or s_j, for dw given:
//   ds_j = (dw_j - sum_i dw_i w_i) / sum s (norm) or dw_j;  a sigmoid's or softmax's backward from there.
// Such differences from a mean are taken of values less that of the largest share: where one share is nearly 1 (or the
// only one: k = 1 with norm), its value and the mean are nearly the same number, and their roundings would be the
// result.
// Shares are quotients: where a token's scores (or its picks') are all below 2^-80, down to 0 in fp32, they are taken
// again relative to exp of the largest logit (rb_faint). Gradients are sums of shares times differences, so that
// no score is divided by alone.
//
// A token is worked on by G = 8, 16 or 32 lanes (E up to 64, 128, 256), eight scores a lane, so that a reduction's
// shuffles serve 32 / G tokens at once: with a warp a token the gradient of 32,768 tokens of 64 experts took 254
// instructions a token and 14 us. Both kernels read the logits once; the bound is HBM on long batches, launch
// latency on short ones. 32,768 tokens: balance of 128 experts 11 to 17 us (17 MB: 8 for the sums, 5 for their join,
// the rest between them), gradient of 64 experts 7 to 11 us (19 MB); 64 tokens 5 to 7 us, 4,096 tokens' gradient 4 us.
#include <math.h>

#include <algorithm>

#include "common.cuh"

namespace lg {

constexpr int RB_WARPS = 32;  // warps a CTA of the balance
constexpr int RG_WARPS = 8;   // and of the gradient
constexpr int RB_N = 8;       // scores a lane
constexpr int RB_MAXE = 256;
constexpr int RB_CTAS = 144;  // of the balance, at most
constexpr float RB_LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float rb_exp(float x) {  // within 2^-22 + |x| 2^-23
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * RB_LOG2E));
  return y;
}
__device__ __forceinline__ float rb_rcp(float x) { return __fdividef(1.f, x); }  // within 2^-22

template <int G>
__device__ __forceinline__ float rb_sum(float v) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int G>
__device__ __forceinline__ float rb_max(float v) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// The expert of a lane's score j: fours of neighbours (VEC: E % 4 == 0, 16-byte rows), or every G-th.
template <int G, bool VEC>
__device__ __forceinline__ int rb_expert(int j) {
  const int l = threadIdx.x % G;
  return VEC ? 4 * (l + G * (j / 4)) + j % 4 : l + G * j;
}

template <int G, bool VEC>
__device__ __forceinline__ void rb_load(float (&v)[RB_N], const float* row, int E, bool in) {
  const float none = -INFINITY;
#pragma unroll
  for (int j = 0; j < RB_N; j += VEC ? 4 : 1) {
    const int e = rb_expert<G, VEC>(j);
    if (VEC) {
      float4 q = make_float4(none, none, none, none);
      if (in && e < E) q = __ldg(reinterpret_cast<const float4*>(row + e));
      v[j] = q.x;
      v[j + 1] = q.y;
      v[j + 2] = q.z;
      v[j + 3] = q.w;
    } else {
      v[j] = in && e < E ? __ldg(row + e) : none;
    }
  }
}

__device__ __forceinline__ float rb_sigmoid(float x, float* rest) {  // rest: 1 - s, without the difference
  const float t = rb_exp(-fabsf(x));                                 // NaN stays
  const float r = rb_rcp(1.f + t);
  *rest = x >= 0.f ? t * r : r;
  return x >= 0.f ? r : t * r;
}

// Sums of scores below this are taken again. Above it, what fp32 leaves out of a sum (scores below 2^-126) is nothing.
constexpr float RB_FAINT = 0x1p-80f;

// exp(v - the largest v) in place of logits far below 0, where a sigmoid is exp(v); their sum.
template <int G>
__device__ __forceinline__ float rb_faint(float (&v)[RB_N]) {
  float m = v[0], sum = 0.f;
#pragma unroll
  for (int j = 1; j < RB_N; ++j) m = fmaxf(m, v[j]);
  m = rb_max<G>(m);
#pragma unroll
  for (int j = 0; j < RB_N; ++j) {
    v[j] = rb_exp(v[j] - m);
    sum += v[j];
  }
  return rb_sum<G>(sum);
}

// The token's scores in place of its logits (-inf past E gives 0). A sigmoid: their sum, and 1 - s of each; softmax: 1,
// with what one more logit's score takes (the maximum, and the reciprocal of the sum).
template <int G>
__device__ __forceinline__ float rb_scores(float (&v)[RB_N], float (&rest)[RB_N], int score_fn, float* mx,
                                           float* rs) {
  float sum = 0.f;
  if (score_fn == LG_SCORE_SOFTMAX) {
    float m = v[0];
#pragma unroll
    for (int j = 1; j < RB_N; ++j) m = fmaxf(m, v[j]);
    m = rb_max<G>(m);
#pragma unroll
    for (int j = 0; j < RB_N; ++j) {
      v[j] = rb_exp(v[j] - m);
      sum += v[j];
    }
    const float r = rb_rcp(rb_sum<G>(sum));
#pragma unroll
    for (int j = 0; j < RB_N; ++j) v[j] *= r;
    *mx = m;
    *rs = r;
    return 1.f;
  }
#pragma unroll
  for (int j = 0; j < RB_N; ++j) {
    v[j] = rb_sigmoid(v[j], &rest[j]);
    sum += v[j];
  }
  return rb_sum<G>(sum);
}

// rb_scores' sigmoids and their sum once more for a token whose sum is faint. Called by whole warps.
template <int G, bool VEC>
__device__ __forceinline__ void rb_again(float (&v)[RB_N], float& total, const float* row, int E, bool keep) {
  const bool faint = keep && total < RB_FAINT;
  if (!__any_sync(0xffffffffu, faint)) return;
  float z[RB_N];
  rb_load<G, VEC>(z, row, E, faint);
  const float sum = rb_faint<G>(z);
  if (!faint) return;
  total = sum;
#pragma unroll
  for (int j = 0; j < RB_N; ++j) v[j] = z[j];
}

// `v` of the first lane of this token's G that holds `mine` (of its lane 0 if none does).
template <int G>
__device__ __forceinline__ float rb_first(bool mine, float v) {
  const unsigned lanes = __ballot_sync(0xffffffffu, mine) >> (threadIdx.x % 32 / G * G);
  const int at = G == 32 ? __ffs(lanes) : __ffs(lanes & ((1u << G % 32) - 1));
  return __shfl_sync(0xffffffffu, v, max(at - 1, 0), G);
}

struct RbOut {
  float* loss;
  int* counts;
  float* probs;
  int* tokens;
};

// The sums of expert threadIdx.x over all tokens -> outputs; called by whole CTAs of at least E threads.
__device__ __forceinline__ void rb_finish(float prob, int count, int n, int E, const RbOut& o) {
  __shared__ float sh_f[32];
  __shared__ long long sh_c[32];
  const int e = threadIdx.x, lane = e & 31, warp = e >> 5;
  const float p = n > 0 ? prob / (float)n : 0.f;
  if (e < E) {
    o.counts[e] = count;
    o.probs[e] = p;
  }
  float fp = e < E ? (float)count * p : 0.f;
  long long c = e < E ? count : 0;
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
    for (int i = 0; i < (E + 31) / 32; ++i) {
      f += sh_f[i];
      all += sh_c[i];
    }
    *o.loss = all > 0 ? (float)E * f / (float)all : 0.f;
    *o.tokens = n;
  }
}

// A CTA's sums over its tokens; a grid of one CTA writes the outputs itself. Each lane has the logits of two tokens
// in flight, whatever the mask says of them (a load that waits for the mask costs a second trip to memory).
template <int G, bool VEC>
__global__ void __launch_bounds__(RB_WARPS * 32) router_balance_kernel(
    const float* __restrict__ logits, const int* __restrict__ inds, const uint8_t* __restrict__ mask, int T,
    int E, int k, int score_fn, float* __restrict__ part_p, int* __restrict__ part_c, RbOut o) {
  constexpr int U = 2, PER = 32 / G;  // tokens a warp works on at a time
  __shared__ float sum_p[RB_WARPS][G * RB_N];
  __shared__ int hist[RB_MAXE + 1];  // the last: tokens kept
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % G;
  for (int i = threadIdx.x; i <= RB_MAXE; i += blockDim.x) hist[i] = 0;
  __syncthreads();
  float acc[RB_N] = {};
  int kept = 0;
  const int step = gridDim.x * RB_WARPS * PER;
  for (int t0 = (blockIdx.x * RB_WARPS + warp) * PER; t0 < T; t0 += U * step) {
    float v[U][RB_N], unused[RB_N], mx, rs;
    int pick[U];
    bool keep[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u * step + lane / G;
      keep[u] = t < T;
      rb_load<G, VEC>(v[u], logits + (size_t)t * E, E, keep[u]);
      pick[u] = keep[u] && l < k ? inds[(size_t)t * k + l] : -1;
      if (keep[u] && mask) keep[u] = mask[t];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (keep[u] && pick[u] >= 0 && pick[u] < E) atomicAdd(&hist[pick[u]], 1);
      float total = rb_scores<G>(v[u], unused, score_fn, &mx, &rs);
      rb_again<G, VEC>(v[u], total, logits + (size_t)(t0 + u * step + lane / G) * E, E, keep[u]);
      const float r = rb_rcp(total);
      if (keep[u]) {
        ++kept;
#pragma unroll
        for (int j = 0; j < RB_N; ++j) acc[j] = fmaf(v[u][j], r, acc[j]);
      }
    }
  }
  if (l == 0 && kept) atomicAdd(&hist[RB_MAXE], kept);
#pragma unroll
  for (int s = 16; s >= G; s >>= 1) {
#pragma unroll
    for (int j = 0; j < RB_N; ++j) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], s);
  }
  if (lane < G) {
#pragma unroll
    for (int j = 0; j < RB_N; ++j) sum_p[warp][rb_expert<G, VEC>(j)] = acc[j];
  }
  __syncthreads();
  const int e = threadIdx.x;
  float p = 0.f;
  if (e < E) {
#pragma unroll
    for (int w = 0; w < RB_WARPS; ++w) p += sum_p[w][e];
  }
  if (gridDim.x == 1) {
    rb_finish(p, e < E ? hist[e] : 0, hist[RB_MAXE], E, o);
    return;
  }
  if (e < E) {
    part_p[(size_t)blockIdx.x * E + e] = p;
    part_c[(size_t)blockIdx.x * E + e] = hist[e];
  }
  if (e == E) part_c[(size_t)RB_CTAS * E + blockIdx.x] = hist[RB_MAXE];
}

// Joins the CTAs' sums in their order: W threads a slice of the CTAs (W: E rounded up to 32), 18 rows in flight
// each. (Joining eight CTAs over the shared memory of a cluster before takes longer, 17 us with 4 here against 8 with
// 5: no more than 14 to 16 clusters of eight CTAs of 1,024 threads are on the GPU at once.)
__global__ void __launch_bounds__(1024) router_balance_join_kernel(const float* __restrict__ part_p,
                                                                   const int* __restrict__ part_c, int C,
                                                                   int E, RbOut o) {
  constexpr int ROWS = 18;
  __shared__ float sp[1024];
  __shared__ int sc[1024];
  __shared__ int sn[32];
  const int W = (E + 31) / 32 * 32, S = 1024 / W;
  const int e = threadIdx.x % W, s = threadIdx.x / W;
  const int a = C * s / S, b = s < S ? C * (s + 1) / S : 0;
  float p = 0.f;
  int c = 0;
  int n = threadIdx.x < C ? part_c[(size_t)RB_CTAS * E + threadIdx.x] : 0;
  for (int i = a; i < b; i += ROWS) {
    float pv[ROWS];
    int cv[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const bool in = e < E && i + r < b;
      pv[r] = in ? part_p[(size_t)(i + r) * E + e] : 0.f;
      cv[r] = in ? part_c[(size_t)(i + r) * E + e] : 0;
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      p += pv[r];
      c += cv[r];
    }
  }
  sp[threadIdx.x] = p;
  sc[threadIdx.x] = c;
#pragma unroll
  for (int i = 16; i; i >>= 1) n += __shfl_xor_sync(0xffffffffu, n, i);
  if ((threadIdx.x & 31) == 0) sn[threadIdx.x >> 5] = n;
  __syncthreads();
  if (s == 0) {
    for (int i = 1; i < S; ++i) {
      p += sp[i * W + e];
      c += sc[i * W + e];
    }
  }
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

template <int G, bool VEC>
__global__ void __launch_bounds__(RG_WARPS * 32) router_grad_kernel(const RgArgs a) {
  constexpr int PER = 32 / G;
  __shared__ float sh_d[RG_WARPS * PER][G * RB_N];          // a token's picks' parts; zeros between tokens
  __shared__ unsigned char sh_t[RG_WARPS * PER][G * RB_N];  // which pick has an expert
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % G;
  float* sd = sh_d[warp * PER + lane / G];
  unsigned char* st = sh_t[warp * PER + lane / G];
  float dq[RB_N];
#pragma unroll
  for (int j = 0; j < RB_N; ++j) {
    sd[l + G * j] = 0.f;
    dq[j] = 0.f;
  }
  if (a.counts) {
    int c[RB_N];
    long long all = 0;
#pragma unroll
    for (int j = 0; j < RB_N; ++j) {
      const int e = rb_expert<G, VEC>(j);
      c[j] = e < a.E ? a.counts[e] : 0;
      all += c[j];
    }
#pragma unroll
    for (int s = G / 2; s; s >>= 1) all += __shfl_xor_sync(0xffffffffu, all, s);
    const int n = *a.tokens;
    const float f = all > 0 && n > 0 ? a.weight * (float)a.E / ((float)all * (float)n) : 0.f;
#pragma unroll
    for (int j = 0; j < RB_N; ++j) dq[j] = f * (float)c[j];
  }
  __syncwarp();
  const int step = gridDim.x * RG_WARPS * PER;
  for (int t0 = (blockIdx.x * RG_WARPS + warp) * PER; t0 < a.T; t0 += step) {
    const int t = t0 + lane / G;
    const bool in = t < a.T;
    const float* row = a.logits + (size_t)t * a.E;
    float s[RB_N], rest[RB_N], mx = 0.f, rs = 0.f;
    rb_load<G, VEC>(s, row, a.E, in);
    int id = -1;
    float d = 0.f;
    if (a.dw && in && l < a.k) {
      id = a.inds[(size_t)t * a.k + l];
      d = a.dw[(size_t)t * a.k + l];
    }
    const bool keep = in && (!a.mask || a.mask[t]);
    if (!keep || id >= a.E) id = -1;
    const float x = id >= 0 ? __ldg(row + id) : -INFINITY;
    float total = rb_scores<G>(s, rest, a.score_fn, &mx, &rs);
    rb_again<G, VEC>(s, total, row, a.E, keep && a.counts);
    const bool softmax = a.score_fn == LG_SCORE_SOFTMAX;
    // What goes through the shares: h - sum q h. (A softmax's gradient of weights with norm sums to 0 by itself.)
    const bool through = softmax && a.dw && !a.norm;
    if (a.dw) {
      float unused;
      float p = id < 0 ? 0.f : softmax ? rb_exp(x - mx) * rs : rb_sigmoid(x, &unused);
      if (id >= 0) st[id] = (unsigned char)l;
      if (a.norm) {
        float sum = rb_sum<G>(p);
        const bool faint = id >= 0 && sum < RB_FAINT;
        if (__any_sync(0xffffffffu, faint)) {
          const float m = rb_max<G>(x);
          const float e = id < 0 ? 0.f : rb_exp(x - m), all = rb_sum<G>(e);
          if (faint) {
            p = e;
            sum = all;
          }
        }
        const float top = rb_max<G>(p);
        d -= rb_first<G>(id >= 0 && p == top, d);
        const float dot = rb_sum<G>(id >= 0 ? d * p : 0.f), r = rb_rcp(sum);
        d = (d - dot * r) * (p * r);
      } else if (!softmax) {
        d *= p;
      }
      __syncwarp();
      const bool twice = id >= 0 && st[id] != l;
      if (__any_sync(0xffffffffu, twice)) {  // an expert picked twice: its parts in their order
        for (int j = 0; j < a.k; ++j) {
          if (l == j && id >= 0) sd[id] += d;
          __syncwarp();
        }
      } else if (id >= 0) {
        sd[id] = d;
      }
      __syncwarp();
    }
    const float r = a.counts ? rb_rcp(total) : 1.f;  // softmax: 1
    float h[RB_N];
#pragma unroll
    for (int j = 0; j < RB_N; ++j) {
      const int e = rb_expert<G, VEC>(j);
      h[j] = dq[j] + (through && e < a.E ? sd[e] : 0.f);
    }
    if (a.counts || through) {
      float best = s[0], at = h[0], mean = 0.f;
#pragma unroll
      for (int j = 1; j < RB_N; ++j) {
        at = s[j] > best ? h[j] : at;
        best = fmaxf(best, s[j]);
      }
      const float top = rb_max<G>(best);
      const float ref = rb_first<G>(best == top, at);
#pragma unroll
      for (int j = 0; j < RB_N; ++j) {
        h[j] -= ref;
        mean = fmaf(s[j], h[j], mean);
      }
      mean = rb_sum<G>(mean) * r;
#pragma unroll
      for (int j = 0; j < RB_N; ++j) h[j] -= mean;
    }
#pragma unroll
    for (int j = 0; j < RB_N; ++j) {
      const int e = rb_expert<G, VEC>(j);
      const float part = a.dw && !through && e < a.E ? sd[e] : 0.f;
      const float g = a.counts || through ? fmaf(s[j] * r, h[j], part) : part;
      s[j] = keep ? softmax ? g : rest[j] * g : 0.f;
    }
    if (in) {
      float* out = a.dl + (size_t)t * a.E;
#pragma unroll
      for (int j = 0; j < RB_N; j += VEC ? 4 : 1) {
        const int e = rb_expert<G, VEC>(j);
        if (e >= a.E) continue;
        if (VEC)
          *reinterpret_cast<float4*>(out + e) = make_float4(s[j], s[j + 1], s[j + 2], s[j + 3]);
        else
          out[e] = s[j];
      }
    }
    __syncwarp();
    if (id >= 0) sd[id] = 0.f;
    __syncwarp();
  }
}

// One CTA up to 256 tokens (its 32 warps have two times 32 / G in flight), above that one for every 64.
static int rb_ctas(int T) { return T <= 256 ? 1 : std::min(RB_CTAS, (T + 63) / 64); }

static int rb_check(const char* who, const void* logits, const void* inds, int T, int E, int k, int score_fn) {
  LG_CHECK_ARG(E >= 1 && E <= RB_MAXE, "%s: E=%d not in [1, %d]", who, E, RB_MAXE);
  LG_CHECK_ARG(k >= 1 && k <= 32, "%s: k=%d not in [1, 32]", who, k);
  LG_CHECK_ARG(T >= 0 && T <= (1 << 30), "%s: T=%d", who, T);
  LG_CHECK_ARG(score_fn == LG_SCORE_SIGMOID || score_fn == LG_SCORE_SOFTMAX, "%s: score_fn %d", who, score_fn);
  LG_CHECK_ARG(T == 0 || (logits && inds), "%s: NULL pointer", who);
  LG_CHECK_ARG(aligned(logits, 4), "%s: logits must be 4-byte aligned", who);
  return LG_OK;
}

// Lanes a token: eight scores each, and one pick each.
#define RB_BY_SIZE(E, k, vec, CALL)                      \
  do {                                                   \
    if ((E) <= 64 && (k) <= 8) {                         \
      if (vec) CALL(8, true); else CALL(8, false);       \
    } else if ((E) <= 128 && (k) <= 16) {                \
      if (vec) CALL(16, true); else CALL(16, false);     \
    } else {                                             \
      if (vec) CALL(32, true); else CALL(32, false);     \
    }                                                    \
  } while (0)

}  // namespace lg

using namespace lg;

extern "C" size_t lg_router_balance_workspace_bytes(int T, int E) {
  if (rb_ctas(T) == 1 || E < 1) return 0;
  return align_up((size_t)RB_CTAS * E * 4, 256) + align_up((size_t)RB_CTAS * (E + 1) * 4, 256);
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
  const bool vec = E % 4 == 0 && aligned(logits, 16);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define RB_CALL(G, VEC)                                                                                     \
  router_balance_kernel<G, VEC><<<C, RB_WARPS * 32, 0, st>>>(logits, inds, mask, T, E, k, score_fn, pp, pc, o)
  RB_BY_SIZE(E, k, vec, RB_CALL);
#undef RB_CALL
  LG_LAUNCH_CHECK("router_balance");
  if (C > 1) {
    router_balance_join_kernel<<<1, 1024, 0, st>>>(pp, pc, C, E, o);
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
  const bool vec = E % 4 == 0 && aligned(logits, 16) && aligned(dlogits, 16);
  const int sms = device_sm_count();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define RB_CALL(G, VEC)                                                                                     \
  router_grad_kernel<G, VEC><<<std::max(1, std::min(8 * sms, (T + RG_WARPS * 32 / G - 1) / (RG_WARPS * 32 / G))), \
                               RG_WARPS * 32, 0, st>>>(a)
  RB_BY_SIZE(E, k, vec, RB_CALL);
#undef RB_CALL
  LG_LAUNCH_CHECK("router_grad");
  return LG_OK;
}
