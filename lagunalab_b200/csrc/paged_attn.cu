// Attention over a paged bf16 K/V cache: packed prompts (causal, grouped heads, optional sliding
// window) and one-token streams that share a prefix.
//
// For a query q at position p of a sequence (token and head) and
// S = {j : max(0, p - W + 1) <= j <= p}:
//   out = sum_{j in S} softmax_S(scale q . k_j) v_j      (0 where S is empty)
// with one pass over the keys: a running reference m, l = sum exp(s_j - m),
// o = sum exp(s_j - m) v_j, all in fp32; out = bf16(o / l), then bf16(out * gate) with a gate per
// (token, head).
//
// One kernel serves all of it. A row tile is 128 query rows of one kv head: the G query heads of
// 128 / G tokens (or streams) beside each other, so that grouped heads share every key they read
// and the causal edge costs at most 128 / G keys a tile. Per 128-key tile two products run on the
// tensor cores, S = Q K^T (both operands in shared memory) and O += P V (P from TMEM, where the
// softmax warps put it in bf16 over the scores; V as it lies, keys by head dim).
//   warps 0-3, 4-7  softmax of row tile 0 / 1, a row a thread: scores from TMEM, mask,
//                   exponentials, P into TMEM, and the output at the end
//   warps 8, 11     issue the products of row tile 0 / 1
//   warp 9          TMA: Q, and the pages' rows into a ring of four 32 KB tiles
//   warp 10         clears what a last V tile holds past the last key
// Two row tiles are always at work, so that one's softmax runs under the other's products: two of
// the same head that share each key tile (a pair: 64 KB of keys and values for 256 rows), or, where
// there is one only (streams, short prompts), the same tokens' of two neighbouring heads (a duo),
// or with an odd number of kv heads the one row tile with its even and odd key tiles, joined at
// the end.
//
// The reference m of a row follows the maximum only when that moves by more than 2^8 (the row's sum
// and O are then rescaled): weights up to 2^8 lose nothing in fp32 or bf16, and the common tile
// touches O only through the tensor cores. P is rounded to bf16 (relative 2^-8 a weight at most)
// because the tensor cores take it so; l sums the unrounded weights; O, m and l stay in fp32
// through the join.
//
// What bounds it. A key tile of a pair is 2,048 cycles of products, 2,048 of the special function
// units' exponentials and about 2,300 of the softmax warps' issue; the chain scores -> weights ->
// products of one row tile is 1,420 cycles of softmax alone, 2,200 beside the other's, and 1,024 of
// products, and takes 3,700 with its hand-overs. Measured (B200; calls in a row, in brackets graph
// replays of 10 ms, which end before the power limit acts): one 8,192-token prompt with 32/4 heads
// 585 us (515-547), 940 TFLOP/s of the causal half; 2 x 512 tokens over 33,000 rows 590 us (503-568),
// 900 TFLOP/s, 0.54 of the measured bf16 GEMM rate and 0.65 of the one measured over seconds; 16
// prompts of up to 1,500 tokens 171 us (153-158); 64 streams on an 8,192-row prefix 36 us (32-39), of
// which the join is 5; 64 streams of 8,192 rows each 176 us (6.1 TB/s; pages of 16 rows 203). The plan
// is not in these times. The compiler reports 168 registers and 188 bytes of spill stores a thread.
// The variants below were compared by graph replays.
// Tried without gain: four softmax warpgroups (two threads a row; 560 us for 500), key tiles of 64
// with two score places each (541; a 64-wide product takes as long as a 128-wide one), a part of
// the exponentials as a polynomial on the FMA pipes (1/8: 526, 1/3: 546), the two product warps
// without turns (556), one arrival for all of a tile's weights (519).
#include <algorithm>
#include <atomic>

#include "paged.cuh"
#include "tc_ptx.cuh"
#include "tmap.cuh"

namespace lg {

using namespace tc;

// ---- plan ---------------------------------------------------------------------------------

static int pa_max_tiles(int kind, int T, int B, int Hq, int Hkv) {
  const int tq2 = 2 * pa_tq(Hq, Hkv);
  return kind == PA_PROMPT ? T / tq2 + B : B + (B + tq2 - 1) / tq2;
}

constexpr int JS_PARTS = 192;  // parts that a stream's rows may have: CTAs, and 2

static PaPlan pa_layout(void* buf, int kind, int T, int B, int Hq, int Hkv) {
  PaPlan p;
  Carver c(buf);
  p.ncta = min(device_sm_count(), JS_PARTS - 2);
  p.max_tiles = pa_max_tiles(kind, T, B, Hq, Hkv);
  p.nprefix = kind == PA_PROMPT ? 0 : p.max_tiles - B;
  p.head = c.take<PaHead>(1);
  p.start = c.take<PaStart>(p.ncta + 1);
  p.kv = c.take<int>(B);
  p.off = c.take<int>(B + 1);
  p.tiles = c.take<PaTile>(p.max_tiles);
  // prompts: two slots a CTA (a part that begins its segment, one that does not); streams: the
  // parts in order, segment + CTA
  const size_t wide = kind == PA_PROMPT
                          ? 2 * (size_t)p.ncta
                          : (size_t)p.nprefix * Hkv + p.ncta;
  const size_t own = kind == PA_PROMPT ? 0 : (size_t)B * Hkv + 2 * (size_t)p.ncta;
  p.wide = c.take<float>(wide * pa_slot_floats(PA_WIDE_ROWS));
  p.own = c.take<float>(own * pa_slot_floats(pa_own_rows(Hq, Hkv)));
  p.bytes = align_up(c.used, 256);
  return p;
}

constexpr int PLAN_THREADS = 1024;

__device__ __forceinline__ PaTile pa_stream_tile(const PaHead& h, const PaPlan& p, int i, int tq) {
  PaTile t = {};
  if (i >= p.nprefix) {  // a stream's own keys
    const int b = i - p.nprefix, kv = p.kv[b];
    t.row = t.q0 = b;
    t.nq = 1;
    t.kind = PA_OWN;
    t.key_end = kv;
    t.key0 = min(max(h.prefix, h.window ? kv - h.window : 0), kv);
    t.duo = !(h.Hkv & 1);
    t.w = PA_W_OWN << t.duo;
  } else {  // 2 tq streams against the shared prefix
    t.q0 = i * 2 * tq;
    t.nq = min(2 * tq, h.B - t.q0);
    t.row = t.q0;
    t.kind = PA_PREFIX;
    t.pair = t.nq > tq;
    t.duo = !t.pair && !(h.Hkv & 1);
    int lo = h.prefix, most = -1;
    for (int b = t.q0; b < t.q0 + t.nq; ++b) {
      const int kv = p.kv[b];
      if (kv > most) most = kv, t.row = b;  // the longest stream names the pages
      if (kv > 0) lo = min(lo, h.window ? max(0, kv - h.window) : 0);
    }
    t.key_end = min(h.prefix, max(most, 0));
    t.key0 = min(lo, t.key_end);
    t.w = t.pair || t.duo ? PA_W_TWO : PA_W_ONE;
  }
  return t;
}

// Row tiles, their costs summed, and each CTA's start: one CTA; 4.5 to 7.4 us (one stream; 16 ragged
// prompts), once for all layers of a step with the same heads and window.
__global__ void __launch_bounds__(PLAN_THREADS)
    pa_plan_kernel(const int* cu, const int* kv_len, PaHead h, PaPlan p) {
  __shared__ int wt[32], tot;
  __shared__ long long wsum[32], carry;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int tq = pa_tq(h.Hq, h.Hkv), tq2 = 2 * tq;
  int n = 0;
  for (int b0 = 0; b0 < h.B; b0 += PLAN_THREADS) {
    const int b = b0 + tid;
    int v = 0;
    if (b < h.B) {
      p.kv[b] = max(0, kv_len[b]);
      if (h.kind == PA_PROMPT) {
        const int t0 = min(max(cu[b], 0), h.T), t1 = min(max(cu[b + 1], t0), h.T);
        v = (t1 - t0 + tq2 - 1) / tq2;
      }
    }
    if (h.kind == PA_PROMPT) {
      const int at = n + block_excl_scan(v, wt, &tot);
      if (b < h.B) p.off[b] = at;
      n += tot;
    }
    __syncthreads();
  }
  if (h.kind != PA_PROMPT) n = p.nprefix + h.B;
  n = min(n, p.max_tiles);  // offsets that do not ascend could ask for more
  if (tid == 0) carry = 0;
  __syncthreads();
  for (int i0 = 0; i0 < n; i0 += PLAN_THREADS) {
    const int i = i0 + tid;
    PaTile t = {};
    long long cost = 0;
    if (i < n) {
      if (h.kind == PA_PROMPT) {
        int lo = 0, hi = h.B - 1;  // the last sequence whose tiles start at or before i
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (p.off[mid] <= i) lo = mid;
          else hi = mid - 1;
        }
        const int t0 = min(max(cu[lo], 0), h.T), t1 = min(max(cu[lo + 1], t0), h.T);
        const int first = (i - p.off[lo]) * tq2;
        t.row = lo;
        t.q0 = t0 + first;
        t.nq = min(tq2, t1 - t0 - first);
        t.pos0 = p.kv[lo] - (t1 - t0) + first;
        t.kind = PA_PROMPT;
        t.pair = t.nq > tq;
        t.duo = !t.pair && !(h.Hkv & 1);
        t.key_end = max(0, t.pos0 + t.nq);
        t.key0 = min(h.window ? max(0, t.pos0 - h.window + 1) : 0, t.key_end);
        t.w = t.pair || t.duo ? PA_W_TWO : PA_W_ONE;
      } else {
        t = pa_stream_tile(h, p, i, tq);
      }
      t.key0 = t.key0 / h.R * h.R;
      t.ntile = t.ntile0 = max(1, (t.key_end - t.key0 + PA_KEYS - 1) / PA_KEYS);
      if (t.kind == PA_PROMPT && t.pair)  // the first row tile's tokens see fewer keys
        t.ntile0 = max(1, (max(0, t.pos0 + tq) - t.key0 + PA_KEYS - 1) / PA_KEYS);
      cost = pa_cost(t.ntile, t.w) * pa_segments(t, h.Hkv);
      if (t.kind == PA_PREFIX && h.prefix == 0) cost = 0;  // the tiles are there, no CTA gets one
    }
    long long inc = cost;  // sum of the costs up to this tile's
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    long long base = carry;
    for (int w = 0; w < warp; ++w) base += wsum[w];
    t.before = base + inc - cost;
    if (i < n) p.tiles[i] = t;
    __syncthreads();
    if (tid == PLAN_THREADS - 1) carry = base + inc;
    __syncthreads();
  }
  const long long total = carry;
  const long long chunk = max((long long)PA_MIN_CHUNK, (total + p.ncta - 1) / p.ncta);
  for (int c = tid; c <= p.ncta; c += PLAN_THREADS) {
    PaStart s = {};
    s.tile = n;
    const long long u = c * chunk;
    if (u < total) {
      int lo = 0, hi = n - 1;  // the last tile whose cost begins at or before u
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.tiles[mid].before <= u) lo = mid;
        else hi = mid - 1;
      }
      const PaTile t = p.tiles[lo];
      const long long seg = pa_cost(t.ntile, t.w), r = u - t.before;
      const long long in = r % seg - PA_SEG;  // key tile k begins at PA_SEG + k w of its segment
      s.tile = lo;
      s.head = (int)(r / seg) << t.duo;
      s.t = in <= 0 ? 0 : (int)((in + t.w - 1) / t.w);
      if (s.t >= t.ntile) {
        s.t = 0;
        s.head += 1 << t.duo;
        if (s.head == h.Hkv) s.head = 0, ++s.tile;
      }
      if (s.tile < n) s.rec = p.tiles[s.tile];
    }
    p.start[c] = s;
  }
  if (tid == 0) {
    h.total = total;
    h.chunk = chunk;
    h.ntiles = n;
    h.err = 0;
    *p.head = h;
  }
}

// ---- attention ----------------------------------------------------------------------------

struct PaArgs {
  const __nv_bfloat16* gate;
  __nv_bfloat16* out;
  const int* table;
  int kind, B, T, P, R, M, Hq, Hkv;
  float scale_log2;  // scale * log2(e): exponentials are powers of two
  PaPlan plan;
};

constexpr int PA_THREADS = 384;  // two softmax warpgroups, and one of four single workers
// Registers a thread: 168 at launch (65,536 over 384 threads); 2 * 216 + 72 = 3 * 168.
constexpr int PA_REGS_SOFTMAX = 216, PA_REGS_OTHER = 72;
constexpr int PA_TILE_BYTES = PA_KEYS * PA_D * 2;  // 32 KB: two halves of 64 dims, 128-byte rows
constexpr int PA_HALF = PA_TILE_BYTES / 2;
constexpr int PA_RING = 4;
constexpr int PA_STAGE = 4096;  // output staging of a softmax warp: 32 rows of 128 bytes
constexpr int PA_NBAD = 8;
constexpr size_t PA_SMEM = (2 + PA_RING) * PA_TILE_BYTES + 8 * PA_STAGE + 512 + 2 * PA_ROWS * 8;

// Whether the plan was made for this call's sizes. One that was not (or never made) would send
// reads and writes anywhere.
__device__ __forceinline__ bool pa_fits(const PaArgs& a, const PaHead* h) {
  const int4 x = *reinterpret_cast<const int4*>(&h->kind);
  const int2 y = *reinterpret_cast<const int2*>(&h->Hkv);
  return x.x == a.kind && x.y == a.B && x.z == a.T && x.w == a.Hq && y.x == a.Hkv && y.y == a.R;
}

// The segments of a CTA's share, in order; every warp walks them by itself.
struct PaWalk {
  const PaTile* tiles;
  struct Place {
    int tile, head, t;
  } at, end;
  int t0, t1;
  PaTile rec;
  __device__ explicit PaWalk(const PaPlan& p) : tiles(p.tiles) {
    const PaStart& s = p.start[blockIdx.x];
    const PaStart& e = p.start[blockIdx.x + 1];
    at = {s.tile, s.head, s.t};
    end = {e.tile, e.head, e.t};
    rec = s.rec;
  }
  __device__ bool more() const {
    if (at.tile != end.tile) return at.tile < end.tile;
    return at.head != end.head ? at.head < end.head : at.t < end.t;
  }
  __device__ bool next() {
    if (!more()) return false;
    t0 = at.t;
    t1 = at.tile == end.tile && at.head == end.head ? end.t : rec.ntile;
    return true;
  }
  // The record of the segment after this one: fetched early, for step().
  __device__ PaTile ahead(int Hkv) const {
    return at.head + (1 << rec.duo) == Hkv && at.tile < end.tile ? tiles[at.tile + 1] : rec;
  }
  __device__ void step(int Hkv, const PaTile& then) {
    at.t = 0;
    at.head += 1 << rec.duo;
    if (at.head == Hkv) at.head = 0, ++at.tile;
    rec = then;
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The order of a part's n K and n V tiles in the ring, by place: K0 V0 K1 V1 ... (pair), or
// K0 K1 V0 K2 V1 K3 ...: V tile t as 2 t + 1, K tile t as 2 t.
__device__ __forceinline__ int pa_ring(int place, int n, bool pair) {
  if (pair) return place;
  if (place < 2) return place == 0 ? 0 : n > 1 ? 2 : 1;
  if (place >= 2 * n - 2) return 2 * (place - n) + 1;  // the last two V
  return place & 1 ? place + 1 : place - 1;  // K tile (place + 1) / 2, V tile place / 2 - 1
}

// Whether the part that ends with key tile t1 has keys past the segment's end in its last tile.
__device__ __forceinline__ bool pa_tail(const PaTile& r, int t1) {
  return r.key0 + t1 * PA_KEYS > r.key_end;
}

// Two fp32 values in one 64-bit register: the packed operations issue two lanes' work at once.
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float x, float y) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void f2_get(F2 a, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v));
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
// Bits [lo, hi) of a word.
__device__ __forceinline__ uint32_t key_bits(int lo, int hi) {
  const uint32_t from = lo <= 0 ? ~0u : lo >= 32 ? 0u : ~0u << lo;
  const uint32_t to = hi <= 0 ? 0u : hi >= 32 ? ~0u : ~(~0u << hi);
  return from & to;
}

// bf16 products, each rounded once: with pack2 the two roundings of bf16(bf16(o) * gate).
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// The weights of 32 keys: p = bf16 pairs of 2^(s c - mc), their sum added to sum.
__device__ __forceinline__ void weights32(const float* s, F2 c, F2 mc, uint32_t (&p)[16],
                                          F2 (&sum)[2]) {
#pragma unroll
  for (int x = 0; x < 16; ++x) {
    float e0, e1;
    f2_get(fma2(f2(s[2 * x], s[2 * x + 1]), c, mc), e0, e1);
    e0 = ex2(e0);
    e1 = ex2(e1);
    sum[x & 1] = add2(sum[x & 1], f2(e0, e1));
    p[x] = pack2(e0, e1);
  }
}

// A bounded wait (about two seconds) with one verdict for the whole warp; a failure's code goes to
// *err, which ends the others' waits. Short: a wait stands in many places of the kernel, whose code
// has to stay in the instruction cache.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err, int code) {
  bool got = mbar_try_wait(bar, parity);
  if (!got) {
    const long long t0 = clock64();
#pragma unroll 1
    for (uint32_t n = 1; !got; ++n) {
      got = mbar_try_wait(bar, parity);
      if (!got && (n & 255) == 0 &&
          (*reinterpret_cast<volatile int*>(err) != 0 || clock64() - t0 > 4000000000LL)) {
        atomicCAS(err, 0, code);
        break;
      }
    }
  }
  return __all_sync(0xffffffffu, got);
}

// A warp's one arrival, after its TMEM accesses. (32 lanes that arrive by themselves are 32 updates
// of one word, one after the other.)
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// Named barriers of `n` threads (whole warps). The TMEM accesses before it are ordered before
// those after it.
__device__ __forceinline__ void bar_sync(int id, int n) {
  tc_fence_before();
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory");
  tc_fence_after();
}
__global__ void __launch_bounds__(PA_THREADS, 1)
    pa_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
              const __grid_constant__ CUtensorMap tm_v, const PaArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];  // 1,024: the swizzle's period
  uint8_t* sQ = smem;                       // two row tiles
  uint8_t* sKV = sQ + 2 * PA_TILE_BYTES;    // ring
  uint8_t* sOut = sKV + PA_RING * PA_TILE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(sOut + 8 * PA_STAGE);
  uint64_t* empty = full + PA_RING;
  uint64_t* q_full = empty + PA_RING;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;   // [2] scores of row tile (or half) w
  uint64_t* p_ready = s_full + 2;   // [2][2] the weights of its key tile's halves are in TMEM
  uint64_t* o_full = p_ready + 4;   // [2] its output is complete
  uint64_t* tail = o_full + 2;      // [ring] a last V tile with rows to clear has landed
  uint64_t* done = tail + PA_RING;  // [2]
  uint64_t* turn = done + 2;        // [2] the tensor cores are w's
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(turn + 2);
  volatile int* bad = reinterpret_cast<volatile int*>(tmem_slot + 1);  // [PA_NBAD] per segment
  float2* ml = reinterpret_cast<float2*>(reinterpret_cast<uint8_t*>(full) + 512);  // [2][128]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  PaHead* const head = a.plan.head;
  int* const err = &head->err;
  const int G = a.Hq / a.Hkv, tq = PA_ROWS / G;
  pdl_trigger();  // the joining kernel waits for this one itself
  PaWalk walk(a.plan);
  if (!pa_fits(a, head) || (smem_u32(smem) & 1023)) {  // no work; the loads pass with the walk's
    walk.end = walk.at;
    // not in err, which the waits of later calls look at
    if (threadIdx.x == 0) head->misfit = PA_MISFIT;
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < PA_RING; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 2);  // one arrival of each w's
      mbar_init(tail + i, 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 2);
    for (int w = 0; w < 2; ++w) {
      mbar_init(s_full + w, 1);
      mbar_init(p_ready + 2 * w, 4);  // one arrival a warp
      mbar_init(p_ready + 2 * w + 1, 4);
      mbar_init(o_full + w, 1);
      mbar_init(done + w, 1);
      mbar_init(turn + w, 1);
    }
    mbar_arrive(turn);  // row tile 0 is first
    fence_mbar_init();
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 8) {  // one setmaxnreg for the whole warpgroup
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PA_REGS_OTHER));
    if (warp == 9) {
      // ---- loads: per segment Q, and K and V tiles in the order of use ----
      int rc = 0, seg = 0, nq = 0;  // ring tiles, segments and Q tiles so far
      bool ok = true;
      const int boxes = PA_KEYS / a.R;  // pages a tile; lanes [0, 2 boxes): (page, half)
      const bool mine = lane < 2 * boxes;
      const int half = lane & 1, box = lane >> 1;
      for (; ok && walk.next(); ++seg) {
        const PaTile r = walk.rec, then = walk.ahead(a.Hkv);
        const int n = (walk.t1 - walk.t0) << r.duo;
        const bool clear = pa_tail(r, walk.t1);
        if (lane == 0) bad[seg % PA_NBAD] = 0;
        __syncwarp();
        const int npage = (r.key_end + a.R - 1) / a.R;  // pages the rows need
        const int* row = a.table + (long long)r.row * a.M;
        // The table 32 columns at a time, a column a lane, the next 32 fetched ahead: a key tile's
        // entries lie within one such group or the next.
        const int c0 = r.key0 / a.R + walk.t0 * boxes;
        auto entries = [&](int c) {
          return c + lane < min(npage, a.M) ? __ldg(row + c + lane) : -1;
        };
        int group = 0, cur = entries(c0), nxt = entries(c0 + 32);
#pragma unroll 1
        for (int place = 0; place < 2 * n; ++place) {
          const int slot = rc % PA_RING, x = pa_ring(place, n, r.pair), t = x >> 1 >> r.duo;
          const int col = t * boxes - group + box;  // V tiles trail K tiles by two at most
          const int in_cur = __shfl_sync(0xffffffffu, cur, col & 31);
          const int in_nxt = __shfl_sync(0xffffffffu, nxt, col & 31);
          int page = col < 32 ? in_cur : in_nxt;
          if ((x & 1) && t * boxes - group >= 32) {  // the last use of the older group has gone
            group += 32;
            cur = nxt;
            nxt = entries(c0 + group + 32);
          }
          if (!(ok = warp_wait(empty + slot, ((rc / PA_RING) & 1) ^ 1, err, 1))) break;
          uint64_t* const bar = (clear && place + 1 + r.duo >= 2 * n ? tail : full) + slot;
          if (lane == 0) mbar_arrive_expect_tx(bar, PA_TILE_BYTES);
          if ((unsigned)page >= (unsigned)a.P) {
            page = a.P;  // outside the pool: reads as zeros
            if (mine && c0 + t * boxes + box < npage) bad[seg % PA_NBAD] = 1;
          }
          __syncwarp();
          if (mine)
            tma_load_4d(sKV + slot * PA_TILE_BYTES + half * PA_HALF + box * a.R * 128,
                        x & 1 ? &tm_v : &tm_k, bar, half * 64, 0,
                        walk.at.head + (x >> 1 & r.duo), page);
          ++rc;
          if (place == 0) {
            if (!(ok = warp_wait(q_empty, (seg & 1) ^ 1, err, 2))) break;
            ++nq;
            if (lane == 0) {
              const int halves = r.pair || r.duo ? 4 : 2;
              mbar_arrive_expect_tx(q_full, halves * 128 * G * tq);
              for (int f = 0; f < halves; ++f)
                tma_load_3d(sQ + f * PA_HALF, &tm_q, q_full, (f & 1) * 64,
                            (walk.at.head + (f >> 1 & r.duo)) * G, r.q0 + (f >> 1) * r.pair * tq);
            }
            __syncwarp();
          }
        }
        walk.step(a.Hkv, then);
      }
      // every copy issued has landed before the CTA ends (bounded, also after a failed wait)
      const long long t0 = clock64();
      for (int i = max(0, rc - PA_RING); i < rc; ++i)
        while (!mbar_try_wait(full + i % PA_RING, (i / PA_RING) & 1) &&
               clock64() - t0 < 4000000000LL) {
        }
      while (nq > 0 && !mbar_try_wait(q_full, (nq - 1) & 1) && clock64() - t0 < 4000000000LL) {
      }
    } else if (warp == 8 || warp == 11) {
      // ---- products of row tile (or half of the keys) w: lane 0 issues, the warp stays together
      // so that all operands are uniform. The tensor cores hold two or three products ahead, past
      // that an issue waits for room, and any wait costs 115 cycles or more: so each w has a warp of
      // its own, one's waits pass under the other's products. Both see every tile of the ring go by (a
      // skipped phase of a barrier could not be told from the next); one that w does not use it
      // gives back at once, the others its softmax warps do. ----
      const int w = warp == 11;
      int rc = 0, seg = 0;
      bool ok = true;
      uint32_t p_phase = 0, turn_phase = 0;
      const uint32_t one = lane == 0;
      const uint32_t id_qk = idesc_bf16(PA_ROWS, PA_KEYS);
      const uint32_t id_pv = idesc_bf16(PA_ROWS, PA_D) | IDESC_B_MN;
      const uint32_t q_lo = sw128_lo(smem_u32(sQ)), k_lo = sw128_lo(smem_u32(sKV));
      const uint32_t v_lo = sw128_lo_mn(smem_u32(sKV), PA_HALF);
      const uint32_t tS = tmem + w * 128, tO = tmem + 256 + w * 128;
      for (; ok && walk.next(); ++seg) {
        const PaTile r = walk.rec, then = walk.ahead(a.Hkv);
        const int n = (walk.t1 - walk.t0) << r.duo;
        const int lim = r.pair && w == 0 ? min(n, max(0, r.ntile0 - walk.t0)) : n;
        const int step = r.pair ? 1 : 2, first = r.pair ? 0 : w;
        uint32_t slot = 0;  // the tile at hand, in 16-byte units
        auto qk = [&](int t) {
          const uint32_t q = q_lo + (r.pair || r.duo ? w * (PA_TILE_BYTES >> 4) : 0);
          const uint32_t k = k_lo + slot;
#pragma unroll
          for (int s = 0; s < PA_D / 16; ++s) {
            const uint32_t off = ((s >> 2) * PA_HALF + (s & 3) * 32) >> 4;
            umma_bf16_warp(one, tS, q + off, k + off, SW128_HI, id_qk, s > 0);
          }
          umma_commit_warp(one, s_full + w);
          if (t + step >= lim) umma_commit_warp(one, q_empty);  // the last use of Q
        };
        // The two warps take turns, each with a weights' and a score product: left alone they fall
        // into step, both row tiles' products at once and then both softmaxes.
        auto turn_wait = [&]() {
          ok = ok && warp_wait(turn + w, turn_phase, err, 9);
          turn_phase ^= 1;
        };
        auto turn_pass = [&]() {
          if (ok && lane == 0) mbar_arrive(turn + 1 - w);
        };
        // O += P V, as soon as each half of the weights is there
        auto pv = [&](int t) {
          const uint32_t v = v_lo + slot;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            ok = ok && warp_wait(p_ready + 2 * w + half, p_phase, err, 4);
            if (half == 0) turn_wait();
            if (!ok) return;
            tc_fence_after();
#pragma unroll
            for (int s = 4 * half; s < 4 * half + 4; ++s)
              umma_bf16_ts_warp(one, tO, tS + s * 8, v + s * (2048 >> 4), SW128_HI, id_pv,
                                s > 0 || t != first);
          }
          p_phase ^= 1;
          if (t + step >= lim) umma_commit_warp(one, o_full + w);
        };
        ok = warp_wait(q_full, seg & 1, err, 5);
        tc_fence_after();
        if (ok && first >= lim && lane == 0) mbar_arrive(q_empty);
        const int lead = r.pair ? 1 : 2;
#pragma unroll 1
        for (int place = 0; ok && place < 2 * n; ++place, ++rc) {
          const int x = pa_ring(place, n, r.pair), t = x >> 1, s = rc % PA_RING;
          const bool own = r.pair || (t & 1) == w;
          const bool use = own && t < lim;
          if (!(ok = warp_wait(full + s, (rc / PA_RING) & 1, err, 3))) break;
          if (!use && lane == 0) mbar_arrive(empty + s);
          slot = __shfl_sync(0xffffffffu, (uint32_t)s * (PA_TILE_BYTES >> 4), 0);
          if (x & 1) {
            if (use) pv(t);
            else if (own) turn_wait();
            if (own && t + lead >= n) turn_pass();
          } else {
            if (use) qk(t);
            if (own && t >= lead) turn_pass();
          }
        }
        if (!r.pair && (n & 1) && w == 1) {  // as many turns for both
          turn_wait();
          turn_pass();
        }
        walk.step(a.Hkv, then);
      }
      umma_commit_warp(one, done + w);
      const long long t0 = clock64();
      while (!mbar_try_wait(done + w, 0) && clock64() - t0 < 4000000000LL) {
      }
    } else if (warp == 10) {
      // ---- rows of V past the last key hold anything (also NaN): their weights are 0, they become
      // 0 too. The last V tile of such a segment lands here first and is passed on when clear. ----
      // A barrier a slot: a second such tile may be under way before the first has landed.
      int rc = 0;
      uint32_t phases = 0;
      bool ok = true;
      for (; ok && walk.next();) {
        const PaTile r = walk.rec, then = walk.ahead(a.Hkv);
        rc += 2 * (walk.t1 - walk.t0) << r.duo;
        for (int back = 1 + r.duo; ok && back > 0 && pa_tail(r, walk.t1); --back) {
          const int slot = (rc - back) % PA_RING;  // a part's last tiles in the ring are its last V
          ok = warp_wait(tail + slot, phases >> slot & 1, err, 8);
          phases ^= 1u << slot;
          uint8_t* v = sKV + slot * PA_TILE_BYTES;
          const int keep = max(0, r.key_end - (r.key0 + (walk.t1 - 1) * PA_KEYS));
          for (int x = keep * 8 + lane; ok && x < PA_KEYS * 8; x += 32) {
            *reinterpret_cast<uint4*>(v + x * 16) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(v + PA_HALF + x * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (ok && lane == 0) mbar_arrive(full + slot);
        }
        walk.step(a.Hkv, then);
      }
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PA_REGS_SOFTMAX));
    // ---- softmax: warpgroup w, a row a thread ----
    const int w = warp >> 2, row = threadIdx.x & 127;
    const int quad_bar = 1 + (warp & 3);  // the two warps of the same 32 rows
    const uint32_t quarter = (uint32_t)(warp & 3) << 21;  // lane field: 32 (warp & 3) << 16
    const uint32_t tS = tmem + w * 128 + quarter, tO = tmem + 256 + quarter;
    const float c = a.scale_log2;
    const int prefix = head->prefix, window = head->window;
    uint32_t s_phase = 0, o_phase = 0;
    int seg = 0, rc = 0;
    // After a failed wait a warp arrives at no mbarrier any more (each role has then done a prefix
    // of what it does otherwise, and the others' waits end too); the softmax warps still meet at
    // their named barriers.
    bool ok = true;
    for (; walk.next(); ++seg) {
      const PaTile& r = walk.rec;
      const int n = (walk.t1 - walk.t0) << r.duo;
      const bool halves = !r.pair && !r.duo;  // one row tile, its key tiles in two halves
      // this row's token and the keys [lo, hi) it sees
      const int i = (r.pair ? w * tq : 0) + row / G;
      const bool valid = row < tq * G && i < r.nq;
      int lo = 0, hi = 1 << 30;
      if (valid) {
        const int kv = r.kind == PA_PROMPT ? r.pos0 + i + 1
                       : r.kind == PA_OWN  ? r.key_end
                                           : a.plan.kv[r.q0 + i];
        hi = r.kind == PA_PREFIX ? min(prefix, kv) : kv;
        lo = window ? max(0, kv - window) : 0;
        if (r.kind == PA_OWN) lo = max(lo, prefix);
      }
      const bool active = __any_sync(0xffffffffu, valid);
      const bool whole = walk.t0 == 0 && walk.t1 == r.ntile && (r.kind == PA_PROMPT || prefix == 0);
      const long long at =
          (long long)(r.q0 + i) * a.Hq + (walk.at.head + (w & r.duo)) * G + row % G;
      // fetched now, looked at at the end
      const __nv_bfloat16 gb = valid && whole && a.gate ? a.gate[at] : __float2bfloat16_rn(1.f);
      float m = -INFINITY, l = 0.f;
      const int stride = r.pair ? 1 : 2;
      const int last = r.pair && w == 0 ? min(n, max(0, r.ntile0 - walk.t0)) : n;
      bool any = false;  // this row tile (or half of the keys) has a key tile
      const int last_t = n - 1 - (n - 1 - w & 1);  // half w's last key tile
      int kb = r.key0 + (walk.t0 + (halves ? w : 0)) * PA_KEYS;
      for (int t = r.pair ? 0 : w; t < last; t += stride, kb += (halves ? 2 : 1) * PA_KEYS) {
        ok = ok && warp_wait(s_full + w, s_phase, err, 6);
        s_phase ^= 1;
        tc_fence_after();
        // these scores are there: so the products are through with their K tile and with the V
        // tile of the weights before
        if (ok && (threadIdx.x & 127) == 0) {
          mbar_arrive(empty + (rc + (r.pair ? 2 * t : t < 2 ? t : 2 * t - 1)) % PA_RING);
          if (any) mbar_arrive(empty + (rc + (r.pair ? 2 * t - 1 : 2 * t - 2)) % PA_RING);
        }
        if (active && ok) {
          float s[128];
          tmem_ld128_wait(tS, s);
          if (__any_sync(0xffffffffu, valid && (kb < lo || kb + PA_KEYS > hi))) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t seen = key_bits(lo - kb - 32 * j, hi - kb - 32 * j);
#pragma unroll
              for (int x = 0; x < 32; ++x)
                if (!(seen >> x & 1)) s[32 * j + x] = -INFINITY;
            }
          }
          float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
          for (int j = 4; j < 128; ++j) mx[j & 3] = fmaxf(mx[j & 3], s[j]);
          const float tm = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          const bool move = tm > m && (tm - m) * c > 8.f;  // also from m = -inf
          if (!any) {
            m = tm;
          } else if (__any_sync(0xffffffffu, move)) {
            const float f = move ? (m == -INFINITY ? 0.f : ex2((m - tm) * c)) : 1.f;
            if (move) m = tm;
            l *= f;
#pragma unroll 1
            for (int j = 0; j < PA_D; j += 16) {
              float o[16];
              uint32_t y[16];
              tmem_ld16_wait(tO + w * 128 + j, o);
#pragma unroll
              for (int x = 0; x < 16; ++x) y[x] = __float_as_uint(o[x] * f);
              tmem_st16(tO + w * 128 + j, y);
            }
          }
          const float mc = m == -INFINITY ? 0.f : m * c;
          const F2 c2 = f2(c, c), mc2 = f2(-mc, -mc);
          F2 sum[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t p[16];
            weights32(s + 32 * j, c2, mc2, p, sum);
            tmem_st16(tS + 16 * j, p);
            if (j & 1) {
              tmem_st_wait();
              warp_arrive(p_ready + 2 * w + (j >> 1));
            }
          }
          float l0, l1;
          f2_get(add2(sum[0], sum[1]), l0, l1);
          l += l0 + l1;
        } else if (ok) {
          warp_arrive(p_ready + 2 * w);
          warp_arrive(p_ready + 2 * w + 1);
        }
        any = true;
      }
      const PaTile then = walk.ahead(a.Hkv);
      // ---- output: a pair's row tile, else both halves' sum, 64 columns a thread ----
      if (any) {
        ok = ok && warp_wait(o_full + w, o_phase, err, 7);
        o_phase ^= 1;
        tc_fence_after();
        if (ok && (threadIdx.x & 127) == 0)  // the last V
          mbar_arrive(empty + (rc + (r.pair ? 2 * last - 1 : min(2 * last_t + 2, n + last_t))) %
                                  PA_RING);
      }
      rc += 2 * n;
      if (active) {
        // The flag is this segment's once one of its key tiles has been seen; a half without one
        // is ahead of the loads here and looks after it has met the other half.
        if ((any && bad[seg % PA_NBAD]) || !ok) l = NAN;
        float f0 = 1.f, f1 = 0.f;
        if (halves) {
          ml[w * PA_ROWS + row] = make_float2(m, l);
          bar_sync(quad_bar, 64);
          const float2 x0 = ml[row], x1 = ml[PA_ROWS + row];
          m = fmaxf(x0.x, x1.x);
          f0 = x0.x == -INFINITY ? 0.f : ex2((x0.x - m) * c);
          f1 = n < 2 || x1.x == -INFINITY ? 0.f : ex2((x1.x - m) * c);
          l = x0.y * f0 + x1.y * f1;
          if (bad[seg % PA_NBAD] || !ok) l = NAN;
        }
        int rr = (halves ? 0 : w * PA_ROWS) + row;
        float* slot = nullptr;
        int rows = PA_WIDE_ROWS;
        if (!whole) {
          if (r.kind == PA_PROMPT) {
            slot = a.plan.wide + (2 * blockIdx.x + (walk.t0 == 0)) * pa_slot_floats(rows);
          } else if (r.kind == PA_PREFIX) {
            slot = a.plan.wide + ((size_t)walk.at.tile * a.Hkv + walk.at.head + blockIdx.x) *
                                     pa_slot_floats(rows);
          } else {
            rows = pa_own_rows(a.Hq, a.Hkv);
            rr = row;
            slot = a.plan.own + pa_own_slot(walk.at.tile - a.plan.nprefix,
                                            walk.at.head + (w & r.duo), blockIdx.x, a.Hkv) *
                                    pa_slot_floats(rows);
          }
          if (valid && (!halves || w == 0))
            reinterpret_cast<float2*>(slot)[rr] = make_float2(m, l);
        }
        const uint32_t g2 = __bfloat16_as_ushort(gb) * 0x10001u;  // the gate, twice
        const int row_to = valid ? (int)at : -1;  // rows of out: below 2^31 (checked on the host)
        if (whole) {  // the sum's reciprocal; a row without a key is 0
          const float inv = l == 0.f ? 0.f : 1.f / l;
          f0 *= inv;
          f1 *= inv;
        }
        uint8_t* const stage = sOut + warp * PA_STAGE;
        // Four or two times 32 columns; `part` is opaque so that the loop is not written out for
        // each kind of output (code that is not in the instruction cache took 3 us here). Without a
        // key tile (a pair's first row tile in a late part) there is no O: m = -inf says so.
        int part = !whole;
#pragma unroll 1
        for (int j = halves ? 2 * w : 0; j < (halves ? 2 * w + 2 : any ? 4 : 0); ++j) {
          asm volatile("" : "+r"(part));
          float o[32];
          tmem_ld32_wait(tO + (halves ? 0 : w * 128) + 32 * j, o);
#pragma unroll
          for (int x = 0; x < 32; ++x) o[x] *= f0;
          if (halves) {
            float o1[32];
            tmem_ld32_wait(tO + (n > 1 ? 128 : 0) + 32 * j, o1);  // f1 = 0 without a second half
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = fmaf(o1[x], f1, o[x]);
          }
          if (part) {
            float4* po = reinterpret_cast<float4*>(slot + 2 * rows);
            if (valid)
#pragma unroll
              for (int x = 0; x < 8; ++x)
                po[(8 * j + x) * rows + rr] =
                    make_float4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
            __syncwarp();
            continue;
          }
          // 16-byte chunk k of row `lane` at k ^ (lane & 7): no bank conflicts either way
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t y[4];
#pragma unroll
            for (int x = 0; x < 4; ++x)
              y[x] = mul_bf16x2(pack2(o[8 * k + 2 * x], o[8 * k + 2 * x + 1]), g2);
            *reinterpret_cast<uint4*>(stage + lane * 128 + ((4 * (j & 1) + k) ^ (lane & 7)) * 16) =
                make_uint4(y[0], y[1], y[2], y[3]);
          }
          __syncwarp();
          if (j & 1) {  // 64 columns are there: whole 128-byte lines, 8 lanes a row
            uint4 v[8];
            int to[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int src = 4 * k + (lane >> 3);
              to[k] = __shfl_sync(0xffffffffu, row_to, src);
              v[k] = *reinterpret_cast<const uint4*>(stage + src * 128 +
                                                     ((lane & 7) ^ (src & 7)) * 16);
            }
            __nv_bfloat16* const dst = a.out + 32 * (j - 1) + (lane & 7) * 8;
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (to[k] >= 0) *reinterpret_cast<uint4*>(dst + (long long)to[k] * PA_D) = v[k];
            __syncwarp();
          }
        }
        // neither half's O or ml is overwritten before both have read it
        if (halves) bar_sync(quad_bar, 64);
      }
      walk.step(a.Hkv, then);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(tmem, 512);
}

// The CTAs [c0, c1] whose shares hold key tiles of the segment (tile t, head).
__device__ __forceinline__ void pa_parts(const PaHead& h, const PaTile& t, int head, int* c0,
                                         int* c1) {
  const long long s = t.before + (head >> t.duo) * pa_cost(t.ntile, t.w) + PA_SEG;
  *c0 = (int)(s / h.chunk);
  *c1 = (int)((s + (long long)(t.ntile - 1) * t.w) / h.chunk);
}

// Joins the parts of prompts' split segments: block x looks at the segment that CTA x + 1 begins
// inside of, if CTA x began it; block y takes 32 of its rows, eight lanes a row, so that a row
// leaves as 256 bytes and a slot's column quads are read 64 bytes at a time.
constexpr int JP_ROWS = 32;
__global__ void __launch_bounds__(256) pa_join_prompt_kernel(const PaArgs a) {
  const PaHead h = *a.plan.head;
  const int c = blockIdx.x;
  const bool fits = pa_fits(a, a.plan.head);
  const PaStart st = a.plan.start[c + 1];
  const PaTile& t = st.rec;
  const int G = a.Hq / a.Hkv, tq = PA_ROWS / G;
  const int rr = blockIdx.y * JP_ROWS + (threadIdx.x >> 3), w = rr / PA_ROWS, row = rr % PA_ROWS;
  const int q = (threadIdx.x & 7) * 4;  // the lane's column quads [q, q + 4)
  const int i = w * t.pair * tq + row / G, head = st.head + (w & t.duo);
  int c0, c1;
  pa_parts(h, t, st.head, &c0, &c1);
  // so far the plan was read, now the parts; a CTA without work waits too, or this kernel, and with
  // it what follows, could come before the attention's end
  pdl_wait();
  if (!fits || st.tile >= h.ntiles || st.t == 0 || c0 != c) return;
  if (row >= tq * G || i >= t.nq || w > (t.pair | t.duo)) return;
  const size_t slot = pa_slot_floats(PA_WIDE_ROWS);
  const long long at = (long long)(t.q0 + i) * a.Hq + head * G + row % G;
  const float g = a.gate ? bf2f(a.gate[at]) : 1.f;
  float m = -INFINITY, l = 0.f;
  float o[16] = {};
#pragma unroll 1
  for (int x = c0; x <= c1; ++x) {  // mostly two parts
    const float* p = a.plan.wide + (2 * x + (x == c0)) * slot;
    const float2 ml = reinterpret_cast<const float2*>(p)[rr];
    float4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      v[j] = reinterpret_cast<const float4*>(p + 2 * PA_WIDE_ROWS)[(q + j) * PA_WIDE_ROWS + rr];
    if (ml.x == -INFINITY) {  // no key, and maybe no o; a NaN l stays one
      l += ml.y;
      continue;
    }
    const float mn = fmaxf(m, ml.x);
    const float f = m == -INFINITY ? 0.f : ex2((m - mn) * a.scale_log2);
    const float e = ex2((ml.x - mn) * a.scale_log2);
    m = mn;
    l = l * f + ml.y * e;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      o[4 * j] = o[4 * j] * f + v[j].x * e;
      o[4 * j + 1] = o[4 * j + 1] * f + v[j].y * e;
      o[4 * j + 2] = o[4 * j + 2] * f + v[j].z * e;
      o[4 * j + 3] = o[4 * j + 3] * f + v[j].w * e;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint32_t y[8];
#pragma unroll
  for (int x = 0; x < 8; ++x)
    y[x] = pack2(round_bf16(o[2 * x] * inv) * g, round_bf16(o[2 * x + 1] * inv) * g);
  uint4* dst = reinterpret_cast<uint4*>(a.out + at * PA_D + 4 * q);
  dst[0] = make_uint4(y[0], y[1], y[2], y[3]);
  dst[1] = make_uint4(y[4], y[5], y[6], y[7]);
}

// Joins a stream's parts for one kv head: its share of the prefix's and its own keys'. The parts'
// weights first, all at once, then every element's sum over the parts.
__global__ void __launch_bounds__(256) pa_join_stream_kernel(const PaArgs a) {
  __shared__ float2 ml[JS_PARTS][16];
  __shared__ float inv[16];
  const PaHead h = *a.plan.head;
  const bool fits = pa_fits(a, a.plan.head);
  const int b = blockIdx.x, head = blockIdx.y, G = a.Hq / a.Hkv, tq = PA_ROWS / G;
  const int pi = b / (2 * tq);
  const PaTile own = a.plan.tiles[a.plan.nprefix + b], pre = a.plan.tiles[pi];
  int c0, c1, p0 = 0, p1 = -1, rr = 0, first = head;
  pa_parts(h, own, head, &c0, &c1);
  if (h.prefix) {
    pa_parts(h, pre, head, &p0, &p1);
    const int i = b - pre.q0, w = i / tq;
    rr = pre.duo ? (head & 1) * PA_ROWS + i * G : w * PA_ROWS + (i - w * tq) * G;
    first = head & ~pre.duo;
  }
  pdl_wait();  // as above
  if (!fits) return;
  if (h.prefix == 0 && c0 == c1) return;  // written by the CTA that had it whole
  const int rows = pa_own_rows(a.Hq, a.Hkv), np = p1 - p0 + 1, n = np + c1 - c0 + 1;
  // the prefix's parts, one slot apart, and the own keys', one or two
  const size_t wide_step = pa_slot_floats(PA_WIDE_ROWS), own_step = pa_slot_floats(rows) << own.duo;
  const float* wide = a.plan.wide + ((size_t)pi * a.Hkv + first + p0) * wide_step;
  const float* ow = a.plan.own + pa_own_slot(b, head, c0, a.Hkv) * pa_slot_floats(rows);
  for (int e = threadIdx.x; e < n * G; e += 256) {
    const int x = e / G, g = e % G;
    ml[x][g] = x < np ? reinterpret_cast<const float2*>(wide + x * wide_step)[rr + g]
                      : reinterpret_cast<const float2*>(ow + (x - np) * own_step)[g];
  }
  __syncthreads();
  if (threadIdx.x < G) {
    const int g = threadIdx.x;
    float m = -INFINITY, l = 0.f;
    for (int x = 0; x < n; ++x) m = fmaxf(m, ml[x][g].x);
    for (int x = 0; x < n; ++x) {  // a part without a key has weight 0; a NaN l stays one
      const float f = ml[x][g].x == -INFINITY ? 0.f : ex2((ml[x][g].x - m) * a.scale_log2);
      l += ml[x][g].x == -INFINITY ? ml[x][g].y : ml[x][g].y * f;
      ml[x][g].x = f;
    }
    inv[g] = l == 0.f ? 0.f : 1.f / l;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < G * 32; e += 256) {
    const int g = e % G, q = e / G;  // neighbours take neighbouring rows of one column quad
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    auto sum = [&](const float* p, size_t step, int x0, int x1) {
#pragma unroll 4
      for (int x = x0; x < x1; ++x, p += step) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        const float f = ml[x][g].x;
        o.x = fmaf(v.x, f, o.x);
        o.y = fmaf(v.y, f, o.y);
        o.z = fmaf(v.z, f, o.z);
        o.w = fmaf(v.w, f, o.w);
      }
    };
    sum(wide + 2 * PA_WIDE_ROWS + 4 * (q * PA_WIDE_ROWS + rr + g), wide_step, 0, np);
    sum(ow + 2 * rows + 4 * (q * rows + g), own_step, np, n);
    const long long at = (long long)b * a.Hq + head * G + g;
    const float s = a.gate ? bf2f(a.gate[at]) : 1.f, r = inv[g];
    reinterpret_cast<uint2*>(a.out + at * PA_D)[q] =
        make_uint2(pack2(round_bf16(o.x * r) * s, round_bf16(o.y * r) * s),
                   pack2(round_bf16(o.z * r) * s, round_bf16(o.w * r) * s));
  }
}

// ---- entry points -------------------------------------------------------------------------

static int plan_check(const char* who, int T, int B, int Hq, int Hkv, int R, int window) {
  LG_CHECK_ARG(T >= 0 && B > 0 && B <= (1 << 20) && T <= (1 << 26), "%s: %d tokens of %d sequences",
               who, T, B);
  LG_CHECK_ARG(Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && Hq / Hkv <= 16 && Hkv <= 1024,
               "%s: %d query heads over %d kv heads (a group of at most 16)", who, Hq, Hkv);
  LG_CHECK_ARG(R == 16 || R == 32 || R == 64 || R == 128,
               "%s: pages of %d rows (16, 32, 64 or 128)", who, R);
  LG_CHECK_ARG((long long)T * Hq < (1LL << 31), "%s: %d tokens of %d heads", who, T, Hq);
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

// The kernel's shared memory limit, raised once per device.
static int pa_smem_once() {
  static std::atomic<bool> done[64];
  int dev = 0;
  LG_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 64 && done[dev].load(std::memory_order_relaxed)) return LG_OK;
  LG_CUDA_TRY(cudaFuncSetAttribute(pa_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   (int)PA_SMEM));
  if (dev < 64) done[dev].store(true, std::memory_order_relaxed);
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
  const char* q0 = static_cast<const char*>(q);
  const char* q1 = q0 + 2 * ((T - 1) * std::max(q_tok, 0LL) + (Hq - 1) * std::max(q_head, 0LL) + D);
  const char* o0 = static_cast<const char*>(out);
  LG_CHECK_ARG(o0 >= q1 || q0 >= o0 + 2LL * T * Hq * D,
               "%s: out shares memory with q, which is read until the end", who);
  // a dimension of one element has no stride to speak of
  if (T == 1) q_tok = D;
  if (Hq == 1) q_head = D;
  if (P == 1) pg = D;
  if (Hkv == 1) hd = D;
  // a tensor map's strides: steps of 0 bytes (a broadcast dimension) or back are not among them
  LG_CHECK_ARG(q_tok > 0 && q_head > 0 && pg > 0 && hd > 0 && rw > 0,
               "%s: strides of dimensions of more than one element must be positive", who);
  const int G = Hq / Hkv;
  CUtensorMap tm_q, tm_k, tm_v;
  const uint64_t qd[3] = {(uint64_t)D, (uint64_t)Hq, (uint64_t)T};
  const uint64_t qst[2] = {(uint64_t)q_head * 2, (uint64_t)q_tok * 2};
  const uint32_t qb[3] = {64, (uint32_t)G, (uint32_t)pa_tq(Hq, Hkv)};
  const uint64_t kd[4] = {(uint64_t)D, (uint64_t)R, (uint64_t)Hkv, (uint64_t)P};
  const uint64_t kst[3] = {(uint64_t)rw * 2, (uint64_t)hd * 2, (uint64_t)pg * 2};
  const uint32_t kb[4] = {64, (uint32_t)R, 1, 1};
  if (int rc = make_map_nd(&tm_q, q, 3, qd, qst, qb)) return rc;
  if (int rc = make_map_nd(&tm_k, k, 4, kd, kst, kb)) return rc;
  if (int rc = make_map_nd(&tm_v, v, 4, kd, kst, kb)) return rc;
  PaArgs a;
  a.gate = static_cast<const __nv_bfloat16*>(gate);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.table = table;
  a.kind = kind;
  a.B = B;
  a.T = T;
  a.P = P;
  a.R = R;
  a.M = M;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.plan = p;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int rc = pa_smem_once()) return rc;
  pa_kernel<<<p.ncta, PA_THREADS, PA_SMEM, st>>>(tm_q, tm_k, tm_v, a);
  LG_LAUNCH_CHECK(who);
  // launched early: its CTAs read the plan and wait for the attention's end on the GPU
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (kind == PA_PROMPT) {
    cfg.gridDim = dim3(p.ncta, PA_WIDE_ROWS / JP_ROWS);
    cfg.blockDim = dim3(256);
    LG_CUDA_TRY(cudaLaunchKernelEx(&cfg, pa_join_prompt_kernel, a));
  } else {
    cfg.gridDim = dim3(B, Hkv);
    cfg.blockDim = dim3(256);
    LG_CUDA_TRY(cudaLaunchKernelEx(&cfg, pa_join_stream_kernel, a));
  }
  LG_LAUNCH_CHECK("paged_join");
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

extern "C" int lg_plan_status(const void* plan, int* status) {
  LG_CHECK_ARG(plan && status, "plan_status: NULL pointer");
  PaHead h;
  LG_CUDA_TRY(cudaMemcpy(&h, plan, sizeof(h), cudaMemcpyDeviceToHost));
  *status = h.misfit == PA_MISFIT ? PA_MISFIT : h.err;
  return LG_OK;
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
