// The attention prologue (prep_core.cuh) of packed tokens of several sequences over a paged cache:
// q/k RMSNorm, RoPE at each token's position, output gate, and the new k and v rows into the pages
// that the table names. One warp per (token, head slot), latency-bound like the one-sequence form;
// the arithmetic is the same function, so a row has the same bits in every kind of cache.
#include <math.h>

#include "prep_core.cuh"

namespace lg {

struct PagedPrep {
  PrepArgs a;  // of one token: qkvg, q_out, gate_out and the caches are moved to the token's
  const int *seq, *pos, *table;
  int T, M, P, R, B;
  long long page;  // elements from one page to the next
};

__global__ void __launch_bounds__(128) attn_prep_pages_kernel(const PagedPrep p) {
  __shared__ uint8_t sb[4][1];  // for quantized caches only
  const int t = blockIdx.x, warp = threadIdx.x >> 5, slot = blockIdx.y * 4 + warp;
  PrepArgs a = p.a;
  const int slots = a.Hq + 2 * a.Hkv;
  if (slot >= slots) return;
  const int gate_w = a.gate_per_head ? a.Hq : a.Hq * a.D;
  a.qkvg += (size_t)t * ((size_t)slots * a.D + gate_w);
  a.q_out += (size_t)t * a.Hq * a.D;
  a.gate_out += (size_t)t * gate_w;
  const int pos = p.pos[t], s = p.seq[t], c = pos / p.R;
  const bool row = pos >= 0 && s >= 0 && s < p.B && c < p.M;
  const int pg = row ? p.table[(size_t)s * p.M + c] : -1;
  a.pos_host = pos;
  if (pg >= 0 && pg < p.P) {
    a.row0 = pos - pos % p.R;  // the page's rows are the cache's
    a.k_cache += pg * p.page;
    a.v_cache += pg * p.page;
  } else {
    if (slot >= a.Hq) return;  // no page: no row
  }
  prep_head(a, 0, slot, true, sb[warp]);
}

}  // namespace lg

using namespace lg;

extern "C" int lg_attn_prep_pages(const void* qkvg, int T, int Hq, int Hkv, int D, const void* qn_w,
                                  const void* kn_w, float eps, float rope_theta,
                                  const int32_t* seq, const int32_t* pos, const int32_t* table,
                                  int B, int M, int P, int R, long long page_stride,
                                  int gate_per_head, void* q_out, void* k_pages, void* v_pages,
                                  void* gate_out, const float* inv_freq, int rot_dims, float mscale,
                                  void* stream) {
  LG_CHECK_ARG((D == 64 || D == 128 || D == 256) && Hq > 0 && Hkv > 0 && T >= 0,
               "attn_prep_pages: head_dim %d (64, 128 or 256)", D);
  LG_CHECK_ARG(B > 0 && M > 0 && P > 0 && R > 0 && page_stride >= (long long)Hkv * R * D,
               "attn_prep_pages: %d sequences of %d pages of %d rows", B, M, R);
  if (T == 0) return LG_OK;
  LG_CHECK_ARG(qkvg && qn_w && kn_w && seq && pos && table && q_out && k_pages && v_pages &&
                   gate_out,
               "attn_prep_pages: NULL pointer");
  PagedPrep p = {};
  if (int rc = prep_extend(&p.a, D, inv_freq, rot_dims, mscale, 0, 0, "attn_prep_pages")) return rc;
  p.a.qkvg = static_cast<const __nv_bfloat16*>(qkvg);
  p.a.qn_w = static_cast<const __nv_bfloat16*>(qn_w);
  p.a.kn_w = static_cast<const __nv_bfloat16*>(kn_w);
  p.a.T = 1;
  p.a.Hq = Hq;
  p.a.Hkv = Hkv;
  p.a.D = D;
  p.a.cap = R;
  p.a.gate_per_head = gate_per_head;
  p.a.eps = eps;
  p.a.log2_theta = log2f(rope_theta);
  p.a.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.a.k_cache = static_cast<__nv_bfloat16*>(k_pages);
  p.a.v_cache = static_cast<__nv_bfloat16*>(v_pages);
  p.a.gate_out = static_cast<__nv_bfloat16*>(gate_out);
  p.seq = seq;
  p.pos = pos;
  p.table = table;
  p.T = T;
  p.M = M;
  p.P = P;
  p.R = R;
  p.B = B;
  p.page = page_stride;
  attn_prep_pages_kernel<<<dim3(T, (Hq + 2 * Hkv + 3) / 4), 128, 0,
                           static_cast<cudaStream_t>(stream)>>>(p);
  LG_LAUNCH_CHECK("attn_prep_pages");
  return LG_OK;
}
