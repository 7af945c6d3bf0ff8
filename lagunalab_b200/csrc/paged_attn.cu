// Attention over a paged bf16 K/V cache: packed prompts (causal, grouped heads, optional sliding
// window) and one-token streams that share a prefix.
//
// For a query q at position p of a sequence (token and head), S = {j : max(0, p - W + 1) <= j <= p}:
//   out = sum_{j in S} softmax_S(scale q . k_j) v_j      (0 where S is empty)
// with one pass over the keys: a running maximum m, l = sum exp(s_j - m), o = sum exp(s_j - m) v_j,
// all in fp32; out = bf16(o / l), then bf16(out * gate) with a gate per (token, head).
#include "paged.cuh"

namespace lg {

static int pa_max_tiles(int kind, int T, int B, int Hq, int Hkv) {
  (void)Hq;
  (void)Hkv;
  return kind == PA_PROMPT ? T / (2 * pa_tq(Hq, Hkv)) + B : B;
}

static PaPlan pa_layout(void* buf, int kind, int T, int B, int Hq, int Hkv) {
  PaPlan p;
  Carver c(buf);
  p.ncta = device_sm_count();
  p.max_tiles = pa_max_tiles(kind, T, B, Hq, Hkv);
  p.head = c.take<PaHead>(1);
  p.start = c.take<PaStart>(p.ncta + 1);
  p.kv = c.take<int>(B);
  p.off = c.take<int>(B + 1);
  p.tiles = c.take<PaTile>(p.max_tiles);
  p.parts = c.take<char>(0);
  p.bytes = align_up(c.used, 256);
  return p;
}

constexpr int PLAN_THREADS = 1024;

__global__ void __launch_bounds__(PLAN_THREADS)
    pa_plan_kernel(const int* cu, const int* kv_len, PaHead h, PaPlan p) {
  __shared__ int wt[32], tot;
  const int tid = threadIdx.x;
  const int tq2 = 2 * pa_tq(h.Hq, h.Hkv);
  int n = 0;
  for (int b0 = 0; b0 < h.B; b0 += PLAN_THREADS) {
    const int b = b0 + tid;
    int v = 0;
    if (b < h.B) {
      p.kv[b] = max(0, kv_len[b]);
      if (h.kind == PA_PROMPT) {
        const int t0 = min(max(cu[b], 0), h.T), t1 = min(max(cu[b + 1], t0), h.T);
        v = (t1 - t0 + tq2 - 1) / tq2;
      } else {
        v = 1;
      }
    }
    const int at = n + block_excl_scan(v, wt, &tot);
    if (b < h.B) p.off[b] = at;
    n += tot;
    __syncthreads();
  }
  n = min(n, p.max_tiles);  // offsets that do not ascend could ask for more
  if (tid == 0) p.off[h.B] = n;
  __syncthreads();
  for (int i = tid; i < n; i += PLAN_THREADS) {
    int lo = 0, hi = h.B - 1;  // the last sequence whose tiles start at or before i
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (p.off[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    const int b = lo;
    PaTile t = {};
    t.row = b;
    if (h.kind == PA_PROMPT) {
      const int t0 = min(max(cu[b], 0), h.T), t1 = min(max(cu[b + 1], t0), h.T);
      const int first = (i - p.off[b]) * tq2;
      t.q0 = t0 + first;
      t.nq = min(tq2, t1 - t0 - first);
      t.pos0 = p.kv[b] - (t1 - t0) + first;
      t.kind = PA_PROMPT;
    } else {
      t.q0 = b;
      t.nq = 1;
      t.pos0 = p.kv[b] - 1;
      t.kind = PA_OWN;
    }
    t.key_end = max(0, t.pos0 + t.nq);
    const int low = h.window ? max(0, t.pos0 - h.window + 1) : 0;
    t.key0 = min(low, t.key_end) / h.R * h.R;
    t.ntile = max(1, (t.key_end - t.key0 + PA_KEYS - 1) / PA_KEYS);
    p.tiles[i] = t;
  }
  if (tid == 0) {
    h.ntile_rows = n;
    *p.head = h;
  }
}

struct PaArgs {
  const __nv_bfloat16 *q, *k, *v, *gate;
  __nv_bfloat16* out;
  const int* table;
  long long q_tok, q_head, pg, hd, rw;  // element strides
  int P, R, M, Hq, Hkv;
  float scale;
  PaPlan plan;
};

// The plain form: one warp per (token, head), four dims a lane, one key at a time.
__global__ void __launch_bounds__(256) pa_simple_kernel(PaArgs a) {
  const PaHead h = *a.plan.head;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = a.Hq / a.Hkv;
  if ((int)blockIdx.x >= h.ntile_rows) return;
  const PaTile t = a.plan.tiles[blockIdx.x];
  for (int r = warp; r < t.nq * G; r += 8) {
    const int tok = t.q0 + r / G, head = blockIdx.y * G + r % G, pos = t.pos0 + r / G;
    const int lo = h.window ? max(0, pos - h.window + 1) : 0;
    float q[4], o[4] = {}, m = -INFINITY, l = 0.f;
    const __nv_bfloat16* qp = a.q + tok * a.q_tok + head * a.q_head + lane * 4;
    for (int d = 0; d < 4; ++d) q[d] = bf2f(qp[d]) * a.scale;
    for (int j = lo; j <= pos; ++j) {
      const int c = j / a.R, pg = c < a.M ? a.table[(long long)t.row * a.M + c] : -1;
      if (pg < 0 || pg >= a.P) {
        l = NAN;
        break;
      }
      const long long at = pg * a.pg + blockIdx.y * a.hd + (j % a.R) * a.rw + lane * 4;
      float s = 0.f;
      for (int d = 0; d < 4; ++d) s += q[d] * bf2f(a.k[at + d]);
      s = warp_sum(s);
      const float mn = fmaxf(m, s), f = __expf(m - mn), e = __expf(s - mn);
      l = l * f + e;
      for (int d = 0; d < 4; ++d) o[d] = o[d] * f + e * bf2f(a.v[at + d]);
      m = mn;
    }
    for (int d = 0; d < 4; ++d) {
      float x = l == 0.f ? 0.f : o[d] / l;
      if (a.gate) x = round_bf16(x) * bf2f(a.gate[(long long)tok * a.Hq + head]);
      a.out[((long long)tok * a.Hq + head) * PA_D + lane * 4 + d] = __float2bfloat16_rn(x);
    }
  }
}

static int plan_check(const char* who, int T, int B, int Hq, int Hkv, int R, int window) {
  LG_CHECK_ARG(T >= 0 && B > 0 && B <= (1 << 20) && T <= (1 << 26), "%s: %d tokens of %d sequences",
               who, T, B);
  LG_CHECK_ARG(Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && Hq / Hkv <= 16 && Hkv <= 1024,
               "%s: %d query heads over %d kv heads (a group of at most 16)", who, Hq, Hkv);
  LG_CHECK_ARG(R == 16 || R == 32 || R == 64 || R == 128, "%s: pages of %d rows (16, 32, 64 or 128)",
               who, R);
  LG_CHECK_ARG(window >= 0, "%s: window %d", who, window);
  return LG_OK;
}

static int plan_run(const char* who, int kind, const int* cu, const int* kv, int B, int T, int Hq,
                    int Hkv, int R, int prefix, int window, void* plan, size_t bytes,
                    void* stream) {
  const PaPlan p = pa_layout(plan, kind, T, B, Hq, Hkv);
  if (!plan || !aligned(plan, 256) || bytes < p.bytes)
    return fail(LG_ERR_WORKSPACE, "%s: the plan buffer needs %zu bytes", who, p.bytes);
  PaHead h = {};
  h.kind = kind;
  h.B = B;
  h.T = T;
  h.Hq = Hq;
  h.Hkv = Hkv;
  h.R = R;
  h.prefix = prefix;
  h.window = window;
  pa_plan_kernel<<<1, PLAN_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(cu, kv, h, p);
  LG_LAUNCH_CHECK("paged_plan");
  return LG_OK;
}

static int attn_run(const char* who, int kind, const void* q, long long q_tok, long long q_head,
                    int T, int Hq, int Hkv, int D, const void* k, const void* v, int P, int R,
                    long long pg, long long hd, long long rw, const int32_t* table, int B, int M,
                    float scale, const void* gate, void* out, void* plan, size_t bytes,
                    void* stream) {
  if (int rc = plan_check(who, T, B, Hq, Hkv, R, 0)) return rc;
  LG_CHECK_ARG(D == PA_D, "%s: head_dim %d (must be %d)", who, D, PA_D);
  LG_CHECK_ARG(P > 0 && M > 0, "%s: %d pages, %d per sequence", who, P, M);
  LG_CHECK_ARG(scale > 0.f && scale < INFINITY, "%s: scale %g must be positive", who, scale);
  if (T == 0) return LG_OK;
  LG_CHECK_ARG(q && k && v && table && out, "%s: NULL pointer", who);
  LG_CHECK_ARG(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(out, 16) &&
                   q_tok % 8 == 0 && q_head % 8 == 0 && pg % 8 == 0 && hd % 8 == 0 && rw % 8 == 0,
               "%s: pointers and strides must be multiples of 16 bytes", who);
  const PaPlan p = pa_layout(plan, kind, T, B, Hq, Hkv);
  if (!plan || !aligned(plan, 256) || bytes < p.bytes)
    return fail(LG_ERR_WORKSPACE, "%s: the plan buffer needs %zu bytes", who, p.bytes);
  PaArgs a;
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.k = static_cast<const __nv_bfloat16*>(k);
  a.v = static_cast<const __nv_bfloat16*>(v);
  a.gate = static_cast<const __nv_bfloat16*>(gate);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.table = table;
  a.q_tok = q_tok;
  a.q_head = q_head;
  a.pg = pg;
  a.hd = hd;
  a.rw = rw;
  a.P = P;
  a.R = R;
  a.M = M;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.scale = scale;
  a.plan = p;
  pa_simple_kernel<<<dim3(p.max_tiles, Hkv), 256, 0, static_cast<cudaStream_t>(stream)>>>(a);
  LG_LAUNCH_CHECK(who);
  return LG_OK;
}

}  // namespace lg

using namespace lg;

extern "C" size_t lg_prompt_plan_bytes(int T, int B, int Hq, int Hkv) {
  if (plan_check("prompt_plan_bytes", T, B, Hq, Hkv, 16, 0)) return 0;
  return pa_layout(nullptr, PA_PROMPT, T, B, Hq, Hkv).bytes;
}

extern "C" size_t lg_stream_plan_bytes(int B, int Hq, int Hkv) {
  if (plan_check("stream_plan_bytes", B, B, Hq, Hkv, 16, 0)) return 0;
  return pa_layout(nullptr, PA_OWN, B, B, Hq, Hkv).bytes;
}

extern "C" int lg_prompt_plan(const int32_t* cu_q, const int32_t* kv_len, int B, int T, int Hq,
                              int Hkv, int page_rows, int window, void* plan, size_t plan_bytes,
                              void* stream) {
  if (int rc = plan_check("prompt_plan", T, B, Hq, Hkv, page_rows, window)) return rc;
  LG_CHECK_ARG(cu_q && kv_len, "prompt_plan: NULL pointer");
  return plan_run("prompt_plan", PA_PROMPT, cu_q, kv_len, B, T, Hq, Hkv, page_rows, 0, window, plan,
                  plan_bytes, stream);
}

extern "C" int lg_stream_plan(const int32_t* kv_len, int B, int Hq, int Hkv, int page_rows,
                              int prefix, int window, void* plan, size_t plan_bytes, void* stream) {
  if (int rc = plan_check("stream_plan", B, B, Hq, Hkv, page_rows, window)) return rc;
  LG_CHECK_ARG(kv_len && prefix >= 0, "stream_plan: NULL pointer or prefix %d", prefix);
  return plan_run("stream_plan", PA_OWN, nullptr, kv_len, B, B, Hq, Hkv, page_rows, prefix, window,
                  plan, plan_bytes, stream);
}

extern "C" int lg_prompt_attention(const void* q, long long q_tok, long long q_head, int T, int Hq,
                                   int Hkv, int D, const void* k_pages, const void* v_pages, int P,
                                   int R, long long page_stride, long long head_stride,
                                   long long row_stride, const int32_t* table, int B, int M,
                                   float scale, const void* gate, void* out, void* plan,
                                   size_t plan_bytes, void* stream) {
  return attn_run("prompt_attention", PA_PROMPT, q, q_tok, q_head, T, Hq, Hkv, D, k_pages, v_pages,
                  P, R, page_stride, head_stride, row_stride, table, B, M, scale, gate, out, plan,
                  plan_bytes, stream);
}

extern "C" int lg_stream_attention(const void* q, long long q_tok, long long q_head, int B, int Hq,
                                   int Hkv, int D, const void* k_pages, const void* v_pages, int P,
                                   int R, long long page_stride, long long head_stride,
                                   long long row_stride, const int32_t* table, int M, float scale,
                                   const void* gate, void* out, void* plan, size_t plan_bytes,
                                   void* stream) {
  return attn_run("stream_attention", PA_OWN, q, q_tok, q_head, B, Hq, Hkv, D, k_pages, v_pages, P,
                  R, page_stride, head_stride, row_stride, table, B, M, scale, gate, out, plan,
                  plan_bytes, stream);
}
