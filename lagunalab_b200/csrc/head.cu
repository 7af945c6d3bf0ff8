// The head's cross entropy without its logits, and its gradient.
//
//   z = x W^T (x bf16 [T, H], W bf16 [V, H], or a 4-bit head read as its bf16 weights),
//   lse_t = log sum_v exp z_tv,   loss_t = sum_j w_tj (lse_t - z_t,id_tj)  over the ids in [0, V),
//   dz_tv = g_t (S_t exp(z_tv - lse_t) - sum_{j: id_tj = v} w_tj),   S_t = sum_j w_tj,
//   dx = dz W,   dW = dz^T x.
//
// Four tiled products in one kernel template (hd_kernel): HD_LOSS leaves each 256-column tile's
// maximum and sum of exponentials per token (a second kernel joins them), HD_PROB computes z again
// and leaves dz as bf16 for a piece of the vocabulary, HD_XGRAD and HD_WGRAD take the piece's dz to
// dx (fp32, added over the pieces) and to its rows of dW. Nothing of size [T, V] is kept.
//
// Bound: the tensor cores, and for more than some hundred us the power limit. 8,192 tokens and 100,352 ids of 2,048:
// loss 2.2 ms (1.5 PFLOP/s; tensor pipe 98 % busy), both gradients 7.1 ms (1.4). With few rows the tiles' ends and the
// chain of launches: 301 tokens and 32,003 ids of 1,024, 94 us (31 for dz, 27 dx, 25 dW, the rest sorting and joining).
//
// Roundings: z, the softmax statistics and every sum are fp32. dz is rounded to bf16 (2^-8 relative
// at most) because the tensor cores take bf16 operands. It is kept as dz / c, with c = max |g_t w_tj|, and
// dx and dW are multiplied by c before they are rounded, once, at the end. So the usual g (1/n for every token)
// and weight leave S exp(z - lse) - 1, whose -1 is exact; as -g it was off by up to 2^-8, in all tokens by the
// same, and dx and dW with it. The other errors are independent: sums over the vocabulary or the tokens average them.
// Up to 64 tokens average little (errors up to 1.8 times those of the results' own rounding), and their products cost
// the reading of W: dz is then kept in two rows a token, its rounding and what that left (hd_rest).
// z is the tensor cores' sum, which is cut after each step, but for targets that carry an eighth or more of their
// token's weight: loss and gradient take both their logits from one fp32 sum (hd_dot), since a target's S p - w of
// nearly 0 has all of z's error, and lse's with the other sign: what is left of it is lse's own rounding. For lse
// the logits around one that is a fourth of the softmax are summed again too (hd_join_kernel).
//
// Every mbarrier wait is bounded (tc::mbar_wait). A CTA whose wait ran out writes NaN for what is
// left of its tiles (zeros stay in dz for tokens without a target, and the ids of largest logits have no mark), waits
// (bounded) for its copies and products in flight, frees its TMEM, records its code for lg_head_status and ends.
// Nothing asynchronous outlives the CTA that it writes to: copies, the commits that free a stage, and the epilogue's
// arrivals (remote ones, even where the barrier is the CTA's own) are all waited for at the end of their roles.
#include <math.h>

#include <algorithm>
#include <atomic>

#include "head.cuh"
#include "tmap.cuh"

namespace lg {

using namespace tc;

enum { HD_LOSS = 0, HD_PROB = 1, HD_XGRAD = 2, HD_WGRAD = 3 };

constexpr int HD_BM = 128, HD_BN = 256, HD_BK = 64;
// Warps of the epilogue, from warp 4 on: a thread a row, and two for the halves of its 256 columns where the tile
// leaves as boxes (one: 10,700 cycles a tile of HD_PROB, 5,400 of HD_WGRAD, when 1,024 of a contraction take
// 8,200). HD_LOSS keeps one: each part would double what the join reads.
constexpr int hd_epi(int kind) { return kind == 0 ? 4 : 8; }
constexpr int hd_threads(int kind) { return 128 + 32 * hd_epi(kind); }
constexpr int HD_A_BYTES = HD_BM * HD_BK * 2;  // 16 KB
constexpr int HD_BOX = 64 * HD_BK * 2;  // an MN-major box: 64 K rows of 64 elements
constexpr int HD_RING = 192 << 10;      // stages of A and B
constexpr int HD_OUT = 4096;            // an output box: 32 rows of 128 bytes, swizzled
constexpr size_t HD_SMEM = 1024 + HD_RING + 8 * HD_OUT + 256;

struct HdArgs {
  int M, N;          // rows of the output tile grid, and its columns
  int mt, nt;        // tiles of 128 CG x 256
  int kblocks;       // 64-wide blocks of the contraction
  int splits;        // HD_XGRAD, HD_WGRAD: parts of the contraction, each with a sum of its own
  int b_row0;        // HD_LOSS, HD_PROB: B's first row; HD_XGRAD: B's first row along the contraction
  int v0;            // the piece's first vocabulary id
  int V;
  int K;             // targets a token
  const int* ids;    // [T, K]; K > 1: sorted (with `order`, `start`)
  const float* weights;        // [T, K] or NULL; K > 1: by sorted id, times hd_up
  const unsigned char* order;  // K > 1: [T, K] the caller's index of a sorted id
  const unsigned char* start;  // K > 1: [T, nt_all + 1] first sorted id of each vocabulary tile
  int nt_all;
  // HD_LOSS
  HdParts out;  // a part a tile of 256 ids
  // HD_PROB
  const float* lse;
  const float* g;
  const float2* wsum;  // K > 1: [T] sum (times hd_up) and largest size of the weights that count
  float* scale;        // HD_PROB, HD_WGRAD: c
  const float* again;  // HD_PROB: [T, K] exp(z - lse) - 1 of targets summed again, HD_LIGHT elsewhere
  // not HD_LOSS: bf16 [M, width], HD_XGRAD and parts of HD_WGRAD: fp32 [splits, M, width]
  void* tile_out;
  int width;
  int add;   // HD_XGRAD: 0 for the first piece
  int rest;  // HD_PROB: rows from a token's dz to what its rounding left; 0: that is not kept
};

// K > 1: what a token's weights are multiplied with, and its g divided by, by its largest weight. g / c is at most
// 1 / largest, which overflows below 2^-128.
__device__ __forceinline__ float hd_up(float largest) { return largest < 0x1p-100f ? 0x1p60f : 1.f; }

constexpr float HD_LIGHT = -2.f;  // exp(d) - 1 is never below -1

// v[c], which is gs p, becomes gs p - w; p - 1 = `again` where that is given.
__device__ __forceinline__ void hd_target(float (&v)[32], int c, float w, float gs, float again) {
  const bool light = again == HD_LIGHT;
  const float heavy = fmaf(gs, again, gs - w);
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = i == c ? (light ? v[i] - w : heavy) : v[i];
}

// Sixteen bf16 as one 32-byte store.
__device__ __forceinline__ void hd_store32(__nv_bfloat16* p, const uint32_t* r) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// A unit of work: tile (m, n) of the output, and the part [k0, k1) of the contraction's blocks.
struct HdUnit {
  int m, n, split, k0, k1;
};
template <int KIND>
__device__ __forceinline__ HdUnit hd_unit(const HdArgs& a, int i) {
  HdUnit u;
  if (KIND == HD_LOSS || KIND == HD_PROB) {  // tokens inner: a tile of W serves all of them from L2
    u.n = (unsigned)i / (unsigned)a.mt;
    u.m = i - u.n * a.mt;
    u.split = 0;
  } else {
    const unsigned r = (unsigned)i / (unsigned)a.nt;
    u.n = i - r * a.nt;
    u.split = r / (unsigned)a.mt;
    u.m = r - u.split * a.mt;
  }
  u.k0 = 0;
  u.k1 = a.kblocks;
  if (KIND >= HD_XGRAD && a.splits > 1) {  // at most 2^24 blocks of a contraction times 148 parts
    u.k0 = (unsigned)a.kblocks * u.split / (unsigned)a.splits;
    u.k1 = (unsigned)a.kblocks * (u.split + 1) / (unsigned)a.splits;
  }
  return u;
}

// What an epilogue thread needs of its row, loaded while the tile before is worked on.
struct HdRow {
  int p, p1, next;       // K > 1: sorted ids [p, p1) of the tile; the next id (K == 1: the id, of any tile)
  float w, gs, gg, off;  // its weight; HD_PROB: g S, g, -lse log2(e)
  float again;           // HD_PROB: as in HdArgs
  bool counts;           // the token has a target
};
template <int KIND>
__device__ __forceinline__ HdRow hd_row(const HdArgs& a, const HdUnit& u, int t) {
  HdRow r = {0, 0, -1, 1.f, 0.f, 0.f, 0.f, HD_LIGHT, false};
  if (KIND > HD_PROB || t >= a.M) return r;
  const size_t row_k = (size_t)t * a.K;
  if (KIND == HD_PROB) {
    r.gg = a.g[t];
    if (a.K > 1) {
      const float big = a.wsum[t].y;  // 0: all weights are, and g may be any size above c
      r.gg = big > 0.f ? r.gg / hd_up(big) : r.gg * 0.f;
    }
    r.gg /= *a.scale;
    r.off = -a.lse[t] * HD_LOG2E;
  }
  if (a.K == 1) {
    r.next = a.ids[t];
    if (KIND == HD_PROB) {
      r.counts = r.next >= 0 && r.next < a.V;
      r.gs = a.weights ? a.g[t] * a.weights[t] / *a.scale : r.gg;
      r.again = a.again[t];
    }
  } else {
    const unsigned char* st = a.start + (size_t)t * (a.nt_all + 1);
    const int tile = a.v0 / HD_BN + u.n;
    if (!hd_ok(tile >= 0 && tile < a.nt_all, 1)) return r;
    r.p = st[tile];
    r.p1 = st[tile + 1];
    if (!hd_ok(r.p <= r.p1 && r.p1 <= a.K, 2)) {
      r.p = r.p1 = 0;
      return r;
    }
    if (KIND == HD_PROB) {
      r.counts = st[a.nt_all] > 0;
      r.gs = r.gg * a.wsum[t].x;
    }
    if (r.p < r.p1) {
      r.next = a.ids[row_k + r.p];
      if (KIND == HD_PROB) {
        r.w = a.weights[row_k + r.p];
        r.again = a.again[row_k + r.p];
      }
    }
  }
  return r;
}

// Outputs leave as boxes of 32 rows x 128 bytes: a thread puts its row into shared memory, and the warp stores four
// whole rows of the box at a time (HD_XGRAD: adds them to what earlier pieces left). Stored by the threads themselves,
// a row each, a tile of dW took 8,500 cycles and dx's addition 16 us of 66; stored by TMA, a box waits for
// 2,000 to 5,000 cycles behind the loads that are queued there.
//
// This thread's 128 bytes of a box: rows y ... of the product, `down` further in the output, from its column x (of
// a.width) on.
template <int KIND>
__device__ __forceinline__ void hd_box(const HdArgs& a, uint8_t* box, const uint32_t (&r)[32], int x, int y,
                                       int split, int down = 0) {
  constexpr int PER = KIND == HD_XGRAD ? 4 : 8;  // elements in 16 bytes
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int c = 0; c < 8; ++c)
    *reinterpret_cast<uint4*>(box + lane * 128 + ((c ^ (lane & 7)) << 4)) =
        make_uint4(r[4 * c], r[4 * c + 1], r[4 * c + 2], r[4 * c + 3]);
  __syncwarp();
  const int chunk = lane & 7, col = x + chunk * PER;
  const bool in = col < a.width &&
                  hd_ok(y >= 0 && x >= 0 && split >= 0 && split < a.splits && col + PER <= a.width, 6);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = 4 * i + (lane >> 3);
    const uint4 v = *reinterpret_cast<const uint4*>(box + row * 128 + ((chunk ^ (row & 7)) << 4));
    if (!in || y + row >= a.M) continue;
    if (KIND == HD_XGRAD) {
      float* out = static_cast<float*>(a.tile_out) + ((size_t)split * a.M + y + row) * a.width + col;
      if (a.add)
        red_add_v4_f32(out, __uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
      else
        *reinterpret_cast<uint4*>(out) = v;
    } else {
      *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.tile_out) + (size_t)(down + y + row) * a.width + col) = v;
    }
  }
  __syncwarp();  // the box is free, and a tcgen05.ld of the whole warp may follow
}

// Columns [c0, c1) of one output tile's row t of this thread. `ok` is false after a wait that ran out: NaN is written.
template <int KIND>
__device__ __forceinline__ void hd_epilogue(const HdArgs& a, const HdUnit& u, int t, HdRow row, uint32_t taddr, bool ok,
                                            uint8_t* box, int begin) {
  const int n0 = u.n * HD_BN;  // in the piece (or in H)
  const bool live = t < a.M;
  const int y = t & ~31;
  const float nan = __int_as_float(0x7fffffff);
  constexpr int COLS = HD_BN / (hd_epi(KIND) / 4);
  float v[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = nan;
  if (KIND == HD_LOSS) {
    const int ntile = a.v0 / HD_BN + u.n;
    const size_t row_k = (size_t)t * a.K;
    float mx = -INFINITY, sum = 0.f, best = 0.f;  // best: of the 32 ids that hold the maximum
    int arg = 0, at = 0;
#pragma unroll 1
    for (int c = 0; c < COLS; c += 32) {
      const int id0 = a.v0 + n0 + c;  // vocabulary ids
      if (id0 >= a.V) break;
      __syncwarp();
      if (ok) tmem_ld32_wait(taddr + c, v);
      if (id0 + 32 > a.V) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = id0 + i < a.V ? v[i] : -INFINITY;
      }
      while ((unsigned)row.next - (unsigned)id0 < 32u) {
        const float z = hd_pick(v, row.next - id0);
        if (a.K == 1) {
          if (hd_ok(t < a.M, 4)) a.out.ztgt[t] = z;
          break;
        }
        if (!hd_ok(row.p < a.K && t < a.M && a.order[row_k + row.p] < a.K, 3)) break;
        a.out.ztgt[row_k + a.order[row_k + row.p]] = z;
        row.next = ++row.p < row.p1 ? a.ids[row_k + row.p] : -1;
      }
      float cm = v[0];
#pragma unroll
      for (int i = 1; i < 32; ++i) cm = fmaxf(cm, v[i]);
      const bool higher = cm > mx;
      if (higher) {
        if (a.out.top) {
          int first = 0;
#pragma unroll
          for (int i = 31; i >= 0; --i) first = v[i] == cm ? i : first;
          arg = id0 + first;
        }
        sum *= hd_ex2((mx - cm) * HD_LOG2E);  // mx = -inf: sum is 0
        mx = cm;
      }
      const float off = mx == -INFINITY ? 0.f : -mx * HD_LOG2E;
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        s0 += hd_ex2(fmaf(v[i], HD_LOG2E, off));
        s1 += hd_ex2(fmaf(v[i + 1], HD_LOG2E, off));
      }
      sum += s0 + s1;
      best = higher ? s0 + s1 : best;
      at = higher ? c : at;
    }
    if (live) {
      if (hd_ok(ntile < a.nt_all && ntile >= 0, 5))
        a.out.part[(size_t)t * a.nt_all + ntile] =
            make_float4(mx, ok ? sum : nan, best, __int_as_float(a.v0 + n0 + at));
      if (a.out.top) a.out.top[(size_t)t * a.nt_all + ntile] = arg;
    }
  } else if (KIND == HD_XGRAD || (KIND == HD_WGRAD && a.splits > 1)) {
#pragma unroll 1
    for (int c = begin; c < begin + COLS && n0 + c < a.width; c += 32) {
      __syncwarp();
      if (ok) tmem_ld32_wait(taddr + c, v);
      uint32_t r[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(v[i]);
      hd_box<HD_XGRAD>(a, box, r, n0 + c, y, u.split);
    }
  } else {
    const float scale = KIND == HD_WGRAD ? *a.scale : 1.f;
#pragma unroll 1
    for (int c = begin; c < begin + COLS && n0 + c < a.width; c += 64) {
      const HdRow start = row;
#pragma unroll 1
      for (int left = 0; left <= (KIND == HD_PROB && a.rest ? 1 : 0); ++left) {
        if (KIND == HD_PROB) row = start;
        uint32_t r[32];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          __syncwarp();
          if (ok) tmem_ld32_wait(taddr + c + 32 * h, v);
          if (KIND == HD_PROB) {
            const int id0 = a.v0 + n0 + c + 32 * h;
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = ok ? row.gs * hd_ex2(fmaf(v[i], HD_LOG2E, row.off)) : nan;
            // K > 1: of the tile's ids in order, those of the other half of the columns only pass by
            while (a.K > 1 ? row.next >= 0 && row.next < id0 + 32 : (unsigned)row.next - (unsigned)id0 < 32u) {
              if (a.K == 1) {
                hd_target(v, row.next - id0, row.gs, row.gs, row.again);
                break;
              }
              if (row.next >= id0) hd_target(v, row.next - id0, row.gg * row.w, row.gs, row.again);
              const size_t at = (size_t)t * a.K + ++row.p;
              row.next = -1;
              if (row.p < row.p1) {
                row.next = a.ids[at];
                row.w = a.weights[at];
                row.again = a.again[at];
              }
            }
            if (!row.counts) {  // a token without a target: nothing of it, whatever its row holds
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = 0.f;
            }
          }
          if (KIND == HD_WGRAD) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] *= scale;
          }
          if (KIND == HD_PROB && left) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] -= __bfloat162float(__float2bfloat16_rn(v[i]));
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) r[16 * h + i] = hd_pack(v[2 * i], v[2 * i + 1]);
        }
        __syncwarp();
        hd_box<KIND>(a, box, r, n0 + c, y, 0, left * a.rest);
      }
    }
  }
}

// D[M, N] = A B^T over tiles of 128 CG x 256. A and B are K-major ([rows, contraction]) or MN-major
// ([contraction, rows]): HD_LOSS, HD_PROB: x and W, both K-major; HD_XGRAD: dz K-major, W MN-major;
// HD_WGRAD: dz and x, both MN-major. Warp 0: TMA; warp 1: products into one of two TMEM tiles;
// warps 4 to 7 (11): the finished tile's rows, one a thread, while the next one's products run.
//
// CG = 2: a pair of CTAs shares a tile, each loads its 128 rows of A and half of B, and the leader issues for
// both. Per 64 of the contraction an SM then loads 32 KB instead of 48 in 512 cycles of products: one CTA alone
// waits for L2 (60 bytes a cycle; 204 cycles a product instead of 128).
template <int KIND, int CG>
__global__ void __launch_bounds__(hd_threads(KIND), 1)
    hd_kernel(const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mb,
              const HdArgs a) {
  constexpr bool A_MN = KIND == HD_WGRAD, B_MN = KIND == HD_XGRAD || KIND == HD_WGRAD;
  constexpr int B_ROWS = HD_BN / CG;  // of B in this CTA
  constexpr int STAGE = HD_A_BYTES + B_ROWS * HD_BK * 2;
  constexpr int STAGES = HD_RING / STAGE;
  extern __shared__ uint8_t hd_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)hd_smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + HD_RING + 8 * HD_OUT);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;  // [2]
  uint64_t* acc_empty = acc_full + 2;   // [2]
  uint64_t* done = acc_empty + 2;
  uint32_t* tmem_base = reinterpret_cast<uint32_t*>(done + 1);
  int* err = reinterpret_cast<int*>(tmem_base + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CG == 2 ? (int)cluster_rank() : 0;
  const int first = blockIdx.x / CG, step = gridDim.x / CG;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full + i, 1);
      mbar_init(acc_empty + i, hd_epi(KIND) * CG);
    }
    mbar_init(done, 1);
    err[0] = err[1] = err[2] = 0;  // of all roles; of the copies' end; of the products' end
    fence_mbar_init();
    prefetch_tmap(&ma);
    prefetch_tmap(&mb);
  }
  if (warp == 2) {
    if (CG == 2) {
      tmem_alloc_pair(tmem_base, 512);
    } else {
      tmem_alloc(tmem_base, 512);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();  // the other CTA's barriers are ready
  tc_fence_after();
  const uint32_t tmem = *tmem_base;
  const int units = a.mt * a.nt * a.splits;

  if (warp == 0) {
    if (elect_one()) {
      int st = 0, used = 0;  // used: stages that hold a copy in this or an earlier turn
      uint32_t ph = 0;
      bool ok = true;
      for (int i = first; i < units && ok; i += step) {
        const HdUnit u = hd_unit<KIND>(a, i);
        const int ar = (u.m * CG + rank) * HD_BM, br = u.n * HD_BN + rank * B_ROWS;
        for (int kb = u.k0; kb < u.k1; ++kb) {
          if (!mbar_wait(empty + st, ph ^ 1, err, 1)) {
            ok = false;
            break;
          }
          if (!hd_ok(st >= 0 && st < STAGES && kb >= 0 && kb < a.kblocks && ar >= 0 && br >= 0 && u.m < a.mt &&
                         u.n < a.nt && u.split < a.splits,
                     7)) {
            ok = false;
            break;
          }
          uint8_t* sa = smem + st * STAGE;
          uint8_t* sb = sa + HD_A_BYTES;
          const int k = kb * HD_BK;
          // Both CTAs' copies complete on the leader's barrier, which expects the bytes of both.
          if (rank == 0) mbar_arrive_expect_tx(full + st, CG * STAGE);
          const uint32_t bar = CG == 2 ? mapa(full + st, 0) : smem_u32(full + st);
          const auto load = [&](void* dst, const CUtensorMap* m, int x, int y) {
            if (CG == 2)
              tma_load_2d_pair(dst, m, bar, x, y);
            else
              tma_load_2d(dst, m, full + st, x, y);
          };
          if (A_MN) {
#pragma unroll
            for (int j = 0; j < HD_BM / 64; ++j) load(sa + j * HD_BOX, &ma, ar + j * 64, k);
          } else {
            load(sa, &ma, k, ar);
          }
          if (B_MN) {
#pragma unroll
            for (int j = 0; j < B_ROWS / 64; ++j)
              load(sb + j * HD_BOX, &mb, br + j * 64, (KIND == HD_XGRAD ? a.b_row0 : 0) + k);
          } else {
            load(sb, &mb, k, a.b_row0 + br);
          }
          if (used < STAGES) ++used;
          if (++st == STAGES) {
            st = 0;
            ph ^= 1;
          }
        }
      }
      // Before the CTA ends, the products have freed the last `used` stages, oldest first: both CTAs' copies into them
      // have then landed, and the commits' arrivals are here. Where products are missing after a wait that ran out,
      // 0.2 s pass instead, for the copies in flight to land (those of rank 1 arrive at the leader's barrier).
      for (int j = used; j > 0; --j) {
        const int s = (st - j + STAGES) % STAGES;
        const uint32_t p = s < st ? ph : ph ^ 1;
        mbar_wait(empty + s, p, err + 1, 2, 400000000LL);
      }
    }
    __syncwarp();
  } else if (warp == 1 && rank == 0) {
    if (elect_one()) {
      constexpr uint32_t idesc = idesc_bf16(HD_BM * CG, HD_BN) | (A_MN ? 1u << 15 : 0u) |
                                 (B_MN ? IDESC_B_MN : 0u);
      const uint64_t hi = (uint64_t)SW128_HI << 32;
      const auto commit = [](uint64_t* bar) {
        if (CG == 2)
          umma_commit_pair(bar);
        else
          umma_commit(bar);
      };
      int st = 0, n = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int i = first; i < units && ok; i += step, ++n) {
        const HdUnit u = hd_unit<KIND>(a, i);
        const int acc = n & 1;
        if (!mbar_wait(acc_empty + acc, ((n >> 1) & 1) ^ 1, err, 3)) break;
        tc_fence_after();
        for (int kb = u.k0; kb < u.k1; ++kb) {
          if (!mbar_wait(full + st, ph, err, 4)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (!hd_ok((tmem & 0x1ff) == 0 && st < STAGES, 8)) {
            ok = false;
            break;
          }
          const uint32_t sa = smem_u32(smem + st * STAGE), sb = sa + HD_A_BYTES;
          const uint32_t da = A_MN ? sw128_lo_mn(sa, HD_BOX) : sw128_lo(sa);
          const uint32_t db = B_MN ? sw128_lo_mn(sb, HD_BOX) : sw128_lo(sb);
#pragma unroll
          for (int k = 0; k < HD_BK / 16; ++k) {  // 16 along K: 32 bytes, or two groups of 8 rows
            const uint64_t ad = hi | (da + k * (A_MN ? 128 : 2)), bd = hi | (db + k * (B_MN ? 128 : 2));
            if (CG == 2)
              umma_bf16_pair(tmem + acc * HD_BN, ad, bd, idesc, kb > u.k0 || k > 0);
            else
              umma_bf16(tmem + acc * HD_BN, ad, bd, idesc, kb > u.k0 || k > 0);
          }
          commit(empty + st);
          if (++st == STAGES) {
            st = 0;
            ph ^= 1;
          }
        }
        if (ok) commit(acc_full + acc);
      }
      commit(done);
      // The epilogue's arrivals for the last two tiles, which nothing else waits for.
      for (int j = min(n, 2); j > 0; --j)
        mbar_wait(acc_empty + ((n - j) & 1), ((n - j) >> 1) & 1, err, 7, 400000000LL);
    }
    __syncwarp();
  } else if (warp >= 4) {
    const int q = warp & 3, begin = warp < 8 ? 0 : HD_BN / 2;
    uint8_t* box = smem + HD_RING + (warp - 4) * HD_OUT;
    bool ok = true;
    int n = 0;
    const auto row_of = [&](const HdUnit& u) { return (u.m * CG + rank) * HD_BM + q * 32 + lane; };
    HdUnit u = hd_unit<KIND>(a, first);
    HdRow row = first < units ? hd_row<KIND>(a, u, row_of(u)) : HdRow{};
    for (int i = first; i < units; i += step, ++n) {
      const HdUnit un = hd_unit<KIND>(a, i + step);
      HdRow next = {};
      if (i + step < units) next = hd_row<KIND>(a, un, row_of(un));
      const int acc = n & 1;
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(acc_full + acc, (n >> 1) & 1, err, 5));
      tc_fence_after();
      hd_epilogue<KIND>(a, u, row_of(u), row, tmem + acc * HD_BN + ((uint32_t)(q * 32) << 16), ok, box, begin);
      u = un;
      row = next;
      tc_fence_before();
      __syncwarp();
      if (ok && lane == 0) {
        // The tile has been read (each tcgen05.ld waited for); what was stored meanwhile is nobody's here. (Arriving
        // before the last box is stored gains nothing.)
        mbar_arrive_cluster_relaxed(mapa(acc_empty + acc, 0));
      }
    }
  }
  // The products have ended before their TMEM goes.
  if (warp == 2) {
    mbar_wait(done, 0, err + 2, 6, 8000000000LL);
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();  // nothing of the pair's reaches a CTA that has ended
  tc_fence_after();
  if (warp == 2) {
    if (CG == 2)
      tmem_dealloc_pair(tmem, 512);
    else
      tmem_dealloc(tmem, 512);
  }
  if (threadIdx.x == 0 && (err[0] || err[1] || err[2])) hd_record(1 + KIND, err[0] ? err[0] : err[1] ? err[1] : err[2]);
}

// The eight weights of a word, in their order, from the bf16 bits of scale and bias.
__device__ __forceinline__ void hd_unpack(uint32_t q, uint16_t scale, uint16_t bias, uint32_t* r) {
  const uint32_t s2 = scale | (uint32_t)scale << 16, b2 = bias | (uint32_t)bias << 16;
  uint32_t v[4];
  if (q4_fast(s2))
    q4_word(q, s2, b2, v);
  else
    q4_word_any(q, s2, b2, v);
  r[0] = __byte_perm(v[0], v[1], 0x5410);
  r[1] = __byte_perm(v[2], v[3], 0x5410);
  r[2] = __byte_perm(v[0], v[1], 0x7632);
  r[3] = __byte_perm(v[2], v[3], 0x7632);
}

// ---- small kernels ------------------------------------------------------------------------------

// K > 1: a warp sorts a token's ids (those in [0, V), ascending, equal ones in their order) with each one's
// weight and place in the caller's list, the first of each vocabulary tile, and the weights' sum.
__global__ void __launch_bounds__(256) hd_sort_kernel(const int* __restrict__ ids,
                                                      const float* __restrict__ weights, int T, int K,
                                                      int V, int nt, int* __restrict__ sorted,
                                                      unsigned char* __restrict__ order,
                                                      float* __restrict__ sorted_w,
                                                      unsigned char* __restrict__ start,
                                                      float2* __restrict__ wsum) {
  __shared__ int sh[8][2 * HD_MAXK];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x * 8 + warp;
  if (t >= T) return;
  int* row = sh[warp];
  float sum = 0.f, big = 0.f;
  for (int j = lane; j < HD_MAXK; j += 32) {
    const int id = j < K ? ids[(size_t)t * K + j] : -1;
    const bool in = id >= 0 && id < V;
    row[j] = in ? id : 0x7fffffff;
    if (in) {
      const float w = weights ? weights[(size_t)t * K + j] : 1.f;
      sum += w;
      big = fmaxf(big, fabsf(w));
    }
  }
  sum = warp_sum(sum);
  big = warp_max(big);
  const float times = hd_up(big);
  __syncwarp();
  int* up = sh[warp] + HD_MAXK;  // ascending
  up[lane] = up[lane + 32] = 0x7fffffff;
  __syncwarp();
#pragma unroll 1
  for (int j = lane; j < K; j += 32) {
    const int id = row[j];
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < K; ++i) rank += row[i] < id || (row[i] == id && i < j);
    if (!hd_ok(rank >= 0 && rank < K, 9)) continue;
    up[rank] = id;
    sorted[(size_t)t * K + rank] = id;
    order[(size_t)t * K + rank] = (unsigned char)j;
    sorted_w[(size_t)t * K + rank] = (weights ? weights[(size_t)t * K + j] : 1.f) * times;
  }
  __syncwarp();
  for (int n = lane; n <= nt; n += 32) {  // ids below the tile's first; n = nt: all that count
    const int lim = n == nt ? V : n * HD_BN;
    int c = 0;
#pragma unroll
    for (int b = HD_MAXK / 2; b; b >>= 1)
      if (up[c + b - 1] < lim) c += b;
    if (up[c] < lim) ++c;
    start[(size_t)t * (nt + 1) + n] = (unsigned char)c;
  }
  if (lane == 0) wsum[t] = make_float2(sum * times, big);
}

// Of hd_join_kernel. Few tokens: twice as many, for the 32 ids around a large logit (37 tokens, 4-bit: 16.4 us against
// 11.2 where a token has one, 7 where none has); many: 2,048 tokens' loss takes 632 us with 256, 625 with 128.
constexpr int HJ_THREADS = 256;
static int hj_threads(bool few) { return few ? HJ_THREADS : HJ_THREADS / 2; }

// sum_h x_h W_vh by a warp, in fp32 with each sum rounded to nearest; the same bits for every U.
template <bool QUANT, int U>
__device__ __forceinline__ float hd_dot(const HdHead& w, const __nv_bfloat16* x, int H, int v) {
  const int lane = threadIdx.x & 31;
  float s = 0.f;
  for (int c0 = lane * 8; c0 < H; c0 += U * 256) {  // U chunks' loads before their sums
    uint4 xv[U], wv[U];
    uint32_t q[U];
    uint16_t sc[U], bi[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * 256;
      xv[u] = wv[u] = make_uint4(0, 0, 0, 0);
      q[u] = 0;
      sc[u] = bi[u] = 0;
      if (c < H) {
        xv[u] = *reinterpret_cast<const uint4*>(x + c);
        if (QUANT) {
          q[u] = static_cast<const uint32_t*>(w.w)[(size_t)v * (H / 8) + c / 8];
          sc[u] = reinterpret_cast<const uint16_t*>(w.scales)[(size_t)v * (H / 64) + c / 64];
          bi[u] = reinterpret_cast<const uint16_t*>(w.biases)[(size_t)v * (H / 64) + c / 64];
        } else {
          wv[u] = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(w.w) + (size_t)v * w.ld + c);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t xs[4] = {xv[u].x, xv[u].y, xv[u].z, xv[u].w};
      uint32_t ws[4] = {wv[u].x, wv[u].y, wv[u].z, wv[u].w};
      if (QUANT) hd_unpack(q[u], sc[u], bi[u], ws);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s = fmaf(__uint_as_float(xs[i] << 16), __uint_as_float(ws[i] << 16), s);
        s = fmaf(__uint_as_float(xs[i] & 0xffff0000u), __uint_as_float(ws[i] & 0xffff0000u), s);
      }
    }
  }
  return warp_sum(s);
}

// hd_dot of N rows from v on (below V; the others give -inf), two chunks of each in flight: each row's sum goes in
// hd_dot's order, to the same bits.
template <bool QUANT, int N>
__device__ __forceinline__ void hd_dots(const HdHead& w, const __nv_bfloat16* x, int H, int v, int V, float (&out)[N]) {
  constexpr int U = 2;
  const int lane = threadIdx.x & 31;
  float s[N] = {};
  for (int c0 = lane * 8; c0 < H; c0 += U * 256) {
    uint4 xv[U], wv[U][QUANT ? 1 : N];
    uint32_t q[U][QUANT ? N : 1];
    uint16_t sc[U][QUANT ? N : 1], bi[U][QUANT ? N : 1];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * 256;
      xv[u] = make_uint4(0, 0, 0, 0);
      if (c < H) xv[u] = *reinterpret_cast<const uint4*>(x + c);
#pragma unroll
      for (int r = 0; r < N; ++r) {
        const bool in = c < H && v + r < V;
        const size_t row = v + r;
        if (QUANT) {
          q[u][r] = 0;
          sc[u][r] = bi[u][r] = 0;
          if (in) {
            q[u][r] = static_cast<const uint32_t*>(w.w)[row * (H / 8) + c / 8];
            sc[u][r] = reinterpret_cast<const uint16_t*>(w.scales)[row * (H / 64) + c / 64];
            bi[u][r] = reinterpret_cast<const uint16_t*>(w.biases)[row * (H / 64) + c / 64];
          }
        } else {
          wv[u][r] = make_uint4(0, 0, 0, 0);
          if (in) wv[u][r] = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(w.w) + row * w.ld + c);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t xs[4] = {xv[u].x, xv[u].y, xv[u].z, xv[u].w};
#pragma unroll
      for (int r = 0; r < N; ++r) {
        uint32_t ws[4];
        if (QUANT) {
          hd_unpack(q[u][r], sc[u][r], bi[u][r], ws);
        } else {
          ws[0] = wv[u][r].x;
          ws[1] = wv[u][r].y;
          ws[2] = wv[u][r].z;
          ws[3] = wv[u][r].w;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[r] = fmaf(__uint_as_float(xs[i] << 16), __uint_as_float(ws[i] << 16), s[r]);
          s[r] = fmaf(__uint_as_float(xs[i] & 0xffff0000u), __uint_as_float(ws[i] & 0xffff0000u), s[r]);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < N; ++r) out[r] = v + r < V ? warp_sum(s[r]) : -INFINITY;
}

// Of a warp's targets, two a lane (id -1: none): those with an eighth or more of all weights, eight ids at most. None
// where all weights are 0.
__device__ __forceinline__ unsigned long long hd_heavy(const int (&id)[2], const float (&wt)[2]) {
  const float all = warp_sum(fabsf(wt[0]) + fabsf(wt[1]));
  unsigned long long heavy = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    heavy |= (unsigned long long)__ballot_sync(0xffffffffu, id[i] >= 0 && all > 0.f && 8.f * fabsf(wt[i]) >= all)
             << (32 * i);
  return heavy;
}
// The targets that hold id v.
__device__ __forceinline__ unsigned long long hd_same(const int (&id)[2], int v) {
  return __ballot_sync(0xffffffffu, id[0] == v) |
         (unsigned long long)__ballot_sync(0xffffffffu, id[1] == v) << 32;
}

// HdParts of two parts, the first before the second; arg: the maximum's lowest id.
struct HdStat {
  float mx, sum;
  int arg;
  float best;
  int at;
};
__device__ __forceinline__ HdStat hd_merge(const HdStat& a, const HdStat& b) {
  HdStat r;
  r.mx = fmaxf(a.mx, b.mx);
  const float ea = a.mx == r.mx ? 1.f : hd_ex2((a.mx - r.mx) * HD_LOG2E);
  const float eb = b.mx == r.mx ? 1.f : hd_ex2((b.mx - r.mx) * HD_LOG2E);
  r.sum = a.sum * ea + b.sum * eb;
  r.arg = b.mx > a.mx || (b.mx == a.mx && b.arg < a.arg) ? b.arg : a.arg;
  r.best = fmaxf(a.best * ea, b.best * eb);
  r.at = b.best * eb > a.best * ea ? b.at : a.at;
  return r;
}

// A CTA joins a token's parts (maximum, sum of exponentials, the maximum's id): lse, the loss, the id of the
// largest logit.
//
// The tensor cores' accumulators are cut, not rounded, after each step: a logit of 11 that H = 2048 like-signed
// products make is 1e-5 too small, more than all other errors together (loss off by 1.5e-6 in the 2-norm
// against 64 bits, 3e-7 with an fp32 product). The logits of targets with an eighth or more of the token's
// weight, eight at most, are therefore summed again here, in fp32 rounded to nearest, and take their first
// value's place in lse too. A warp sums one target's; all work side by side. So are, for lse's
// sake, the 32 ids around a logit that has a fourth of the softmax or more, unless a target among them is nearly all of
// it: lse of a token without a target was off by up to 2.3e-6 of itself.
template <bool QUANT>
__global__ void __launch_bounds__(HJ_THREADS) hd_join_kernel(HdParts in, const __nv_bfloat16* __restrict__ x,
                                                             long long ldx, int H, HdHead w,
                                                             const int* __restrict__ ids,
                                                             const float* __restrict__ weights, int K, int V,
                                                             float* __restrict__ loss,
                                                             float* __restrict__ lse_out,
                                                             int* __restrict__ top) {
  const int warps = blockDim.x >> 5;
  __shared__ HdStat sh[HJ_THREADS / 32];
  __shared__ float sh_dot[HD_MAXK], sh_near[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x;
  const int parts = in.parts;
  // the targets: two a lane, the same in every warp
  int id[2];
  float wt[2], z[2];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int j = lane + 32 * i;
    id[i] = j < K ? ids[(size_t)t * K + j] : -1;
    bad = bad || id[i] >= V;
    if (id[i] >= V) id[i] = -1;
    wt[i] = id[i] < 0 ? 0.f : weights ? weights[(size_t)t * K + j] : 1.f;
    z[i] = id[i] < 0 ? 0.f : in.ztgt[(size_t)t * K + j];
  }
  const float4* row = in.part + (size_t)t * parts;
  HdStat st = {-INFINITY, 0.f, 0x7fffffff, 0.f, 0};
#pragma unroll 4
  for (int n = threadIdx.x; n < parts; n += blockDim.x) {
    const float4 v = row[n];
    st = hd_merge(st, {v.x, v.y, top ? in.top[(size_t)t * parts + n] : 0, v.z, __float_as_int(v.w)});
  }
  // The list of heavy targets, an id once: every warp has it, and sums its share.
  unsigned long long todo = hd_heavy(id, wt);
  const unsigned long long heavy = todo;
  int n = 0;
  while (todo) {
    const int j = __ffsll(todo) - 1;
    const int v = __shfl_sync(0xffffffffu, j < 32 ? id[0] : id[1], j & 31);
    if (!hd_ok(v >= 0 && v < V && n < HD_MAXK, 10)) break;
    if (n % warps == warp) {
      const float d = hd_dot<QUANT, 4>(w, x + (size_t)t * ldx, H, v);
      if (lane == 0) sh_dot[n] = d;
    }
    ++n;
    todo &= ~hd_same(id, v);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const HdStat p = {__shfl_xor_sync(0xffffffffu, st.mx, o), __shfl_xor_sync(0xffffffffu, st.sum, o),
                      __shfl_xor_sync(0xffffffffu, st.arg, o), __shfl_xor_sync(0xffffffffu, st.best, o),
                      __shfl_xor_sync(0xffffffffu, st.at, o)};
    st = (lane & o) ? hd_merge(p, st) : hd_merge(st, p);
  }
  if (lane == 0) sh[warp] = st;
  __syncthreads();
  st = sh[0];
  for (int i = 1; i < warps; ++i) st = hd_merge(st, sh[i]);
  // The same decision in every thread.
  bool near = in.maxima ? st.sum <= 4.f && st.best > 0.f : st.best > 0.f && 4.f * st.best >= st.sum;
  if (near) {
    float known = 0.f;
    for (todo = heavy; todo;) {
      const int j = __ffsll(todo) - 1;
      const int v = __shfl_sync(0xffffffffu, j < 32 ? id[0] : id[1], j & 31);
      const float was = __shfl_sync(0xffffffffu, j < 32 ? z[0] : z[1], j & 31);
      if ((unsigned)v - (unsigned)st.at < 32u) known += hd_ex2((was - st.mx) * HD_LOG2E);
      todo &= ~hd_same(id, v);
    }
    near = known < 0.875f * st.best;
  }
  if (near) {
    constexpr int N = 4;
    for (int i = warp * N; i < 32; i += warps * N) {
      float d[N];
      hd_dots<QUANT, N>(w, x + (size_t)t * ldx, H, hd_ok(st.at >= 0, 13) ? st.at + i : V, V, d);
#pragma unroll
      for (int r = 0; r < N; ++r)
        if (lane == 0) sh_near[i + r] = d[r];
    }
    __syncthreads();
  }
  if (warp) return;
  if (near) {
    st.sum += warp_sum(hd_ex2((sh_near[lane] - st.mx) * HD_LOG2E)) - st.best;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (id[i] >= 0 && (unsigned)id[i] - (unsigned)st.at < 32u) z[i] = sh_near[id[i] - st.at];
  }
  todo = heavy;
  for (n = 0; todo; ++n) {
    const int j = __ffsll(todo) - 1;
    const int v = __shfl_sync(0xffffffffu, j < 32 ? id[0] : id[1], j & 31);
    const float was = __shfl_sync(0xffffffffu, j < 32 ? z[0] : z[1], j & 31), now = sh_dot[n];
    if (!near || (unsigned)v - (unsigned)st.at >= 32u)
      st.sum += hd_ex2((now - st.mx) * HD_LOG2E) - hd_ex2(fmaf(was, HD_LOG2E, -st.mx * HD_LOG2E));
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (id[i] == v) z[i] = now;  // every place of the list that names it
    todo &= ~hd_same(id, v);
  }
  // Neither loss nor what is taken off above has the roundings of large logits: the loss does not go through lse, and a
  // term of the sum is taken off as it was put on (its argument's rounding is 2^-24 of the logit).
  const float log_sum = logf(st.sum), lse = st.mx + log_sum;
  float l = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (id[i] >= 0) l += wt[i] * ((st.mx - z[i]) + log_sum);
  l = warp_sum(l);
  bad = __any_sync(0xffffffffu, bad);
  if (lane == 0) {
    loss[t] = bad ? __int_as_float(0x7fffffff) : l;
    lse_out[t] = lse;
    if (top) top[t] = st.arg == 0x7fffffff ? 0 : st.arg;
  }
}

// What HD_PROB needs besides z, by blocks of 256 threads of a kernel that runs before the products anyway: block 0
// finds c, the largest |g_t w_tj| that counts (1 if there is none above 0, or an infinite one), in 3 us; the others
// (hd_again) sum heavy targets' logits again.
struct HdScale {
  const int* ids;
  const float *g, *weights;
  const unsigned char* start;  // K > 1: as in HdArgs
  const float2* wsum;
  float* scale;  // NULL: not asked for
  int T, V, nt;
  // hd_again
  const __nv_bfloat16* x;
  long long ldx;
  int H, K;
  HdHead w;
  const float* lse;
  float* again;

  __host__ __device__ int warps() const { return K > 1 ? 4 : 1; }  // a token
  __host__ __device__ int blocks() const { return scale ? 1 + (T + 8 / warps() - 1) / (8 / warps()) : 0; }
};
__device__ __forceinline__ bool hd_counts(const HdScale& a, int t) {
  return a.start ? a.start[(size_t)t * (a.nt + 1) + a.nt] > 0 : a.ids[t] >= 0 && a.ids[t] < a.V;
}
__device__ __forceinline__ void hd_scale(const HdScale& a) {
  __shared__ float sh[8];
  float big = 0.f;
#pragma unroll 4
  for (int t = threadIdx.x; t < a.T; t += 256) {
    const float w = a.start ? a.wsum[t].y : a.weights ? a.weights[t] : 1.f;
    if (hd_counts(a, t)) big = fmaxf(big, fabsf(a.g[t] * w));
  }
  big = warp_max(big);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = big;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) big = fmaxf(big, sh[i]);
    *a.scale = big > 0.f && big < INFINITY ? big : 1.f;
  }
}

// exp(z - lse) - 1 of a token's heavy targets, at the first of an id's places in order. The targets are those of
// hd_join_kernel to the bit: the sum of weights is taken in the caller's order in both. Its warps take the targets in
// turn (301 tokens of 5 targets, both gradients: 92.5 us with one warp a token, 90 with four).
template <bool QUANT>
__device__ __forceinline__ void hd_again(const HdScale& a, int block) {
  const int lane = threadIdx.x & 31, warps = a.warps(), part = (threadIdx.x >> 5) % warps;
  const int t = block * (8 / warps) + (threadIdx.x >> 5) / warps;
  if (t >= a.T) return;
  const size_t row = (size_t)t * a.K;
  int id[2];
  float wt[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int j = lane + 32 * i;
    id[i] = j < a.K ? a.ids[row + j] : -1;
    if (id[i] >= a.V) id[i] = -1;
    wt[i] = id[i] < 0 ? 0.f : a.weights ? a.weights[row + j] : 1.f;
  }
  const float lse = a.lse[t];
  unsigned long long heavy = 0;  // places in order
  int turn = 0;
  for (unsigned long long todo = hd_heavy(id, wt); todo; ++turn) {
    const int j = __ffsll(todo) - 1;
    const int v = __shfl_sync(0xffffffffu, j < 32 ? id[0] : id[1], j & 31);
    int place = 0;  // ids that come before
#pragma unroll
    for (int i = 0; i < 2; ++i) place += __popc(__ballot_sync(0xffffffffu, id[i] >= 0 && id[i] < v));
    if (!hd_ok(v >= 0 && v < a.V && place >= 0 && place < a.K, 11)) break;
    heavy |= 1ull << place;
    if (turn % warps == part) {
      const float d = expm1f(hd_dot<QUANT, QUANT ? 2 : 4>(a.w, a.x + (size_t)t * a.ldx, a.H, v) - lse);
      if (lane == 0) a.again[row + place] = d;
    }
    todo &= ~hd_same(id, v);
  }
  if (part == 0) {
    for (int j = lane; j < a.K; j += 32)
      if (!(heavy >> j & 1)) a.again[row + j] = HD_LIGHT;
  }
}

// Blocks [0, a.blocks()): as HdScale says. The others, for dW: x with the rows of tokens without a target at 0, so
// that dW has nothing of them (0 * NaN is NaN); `rest` rows further once more, for the second rows of dz.
__global__ void __launch_bounds__(256) hd_rows_kernel(const __nv_bfloat16* __restrict__ x, long long ldx, int H,
                                                      const HdScale a, int rest, __nv_bfloat16* __restrict__ out) {
  const int first = a.blocks();
  if ((int)blockIdx.x < first) {
    if (blockIdx.x == 0)
      hd_scale(a);
    else
      hd_again<false>(a, blockIdx.x - 1);
    return;
  }
  const int per = H / 8;
  const long long n = (long long)a.T * per;
  for (long long i = (blockIdx.x - first) * 256LL + threadIdx.x; i < n; i += (gridDim.x - first) * 256LL) {
    const int t = (int)(i / per), c = (int)(i % per) * 8;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (!hd_ok(t >= 0 && t < a.T && c + 8 <= H, 12)) continue;
    if (hd_counts(a, t)) v = *reinterpret_cast<const uint4*>(x + (size_t)t * ldx + c);
    *reinterpret_cast<uint4*>(out + (size_t)t * H + c) = v;
    if (rest) *reinterpret_cast<uint4*>(out + (size_t)(rest + t) * H + c) = v;
  }
}

// Rows of a 4-bit group-64 head as bf16: bf16(scale * code + bias), two words a thread: a warp writes 1 KB in one
// store (four words a thread with 16-byte stores: 3 TB/s written instead of 4.3). Blocks [0, a.blocks()): as HdScale
// says; they take two chunks of hd_dot at a time, which leaves 48 registers.
__global__ void __launch_bounds__(256, 5) hd_dequant_kernel(const uint2* __restrict__ q,
                                                            const uint16_t* __restrict__ s,
                                                            const uint16_t* __restrict__ b, long long n,
                                                            const HdScale a, __nv_bfloat16* __restrict__ out) {
  const int first = a.blocks();  // of the blocks that unpack
  if ((int)blockIdx.x < first) {
    if (blockIdx.x == 0)
      hd_scale(a);
    else
      hd_again<true>(a, blockIdx.x - 1);
    return;
  }
  constexpr int U = 4;
  const long long step = (gridDim.x - first) * 256LL;
  for (long long i0 = (blockIdx.x - first) * 256LL + threadIdx.x; i0 < n; i0 += U * step) {
    uint2 w[U];
    uint16_t sc[U], bi[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long i = i0 + u * step;
      if (i < n) {
        w[u] = q[i];
        sc[u] = s[i >> 2];
        bi[u] = b[i >> 2];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long i = i0 + u * step;
      if (i >= n) break;
      uint32_t r[8];
      hd_unpack(w[u].x, sc[u], bi[u], r);
      hd_unpack(w[u].y, sc[u], bi[u], r + 4);
      hd_store32(out + 16 * i, r);
    }
  }
}

// dx (dW) = c times the sum of its parts, in their order, rounded once.
__global__ void __launch_bounds__(256) hd_sum_kernel(const float* __restrict__ parts, int n,
                                                     long long size, const float* __restrict__ scale,
                                                     __nv_bfloat16* __restrict__ out) {
  const float c = *scale;
  const long long q = size / 4;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < q; i += gridDim.x * 256LL) {
    float4 s = reinterpret_cast<const float4*>(parts)[i];
    for (int j = 1; j < n; ++j) {
      const float4 v = reinterpret_cast<const float4*>(parts + j * size)[i];
      s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
    }
    *reinterpret_cast<uint2*>(out + 4 * i) = make_uint2(hd_pack(c * s.x, c * s.y), hd_pack(c * s.z, c * s.w));
  }
}

// ---- host ---------------------------------------------------------------------------------------

// dz of a piece (8,192 tokens, dx and dW of 100,352 ids: 7.25 ms with 256 MB, 7.10 with 512, 7.53 with 128).
constexpr long long HD_DZ_BYTES = 512LL << 20;
// bf16 rows of a piece of a 4-bit head: 100,352 ids of 2,048 are one. Pieces that stay in L2 are no faster, even for
// few tokens: the launches cost more (37 tokens, dx of 100,352 ids: 388 us with 32 MB, 276 with 64, 234 with 256, 229
// with 512).
constexpr long long HD_WQ_BYTES = 512LL << 20;

// Rows of dz that hold what the rounding of T tokens' rows left. Up to 64 tokens: both are one tile of rows of dx's
// product (100,352 ids of 2,048: dx of 37 tokens 155 us instead of 145, of 128 tokens it would be 176 instead of 157).
static int hd_rest(int T) { return T <= HD_BM / 2 ? T : 0; }

static int hd_cg(int rows) { return rows > HD_BM ? 2 : 1; }
static long long hd_rounds(long long units, int cg) {
  const int slots = device_sm_count() / cg;
  return (units + slots - 1) / slots;
}

// Vocabulary ids a piece: a multiple of 256, within the bytes above, such that the tiles of its products fill the
// SMs in few whole rounds (8,192 tokens, dx and dW of 100,352 ids: 6.26 to 6.62 ms; as many ids as fit 6.63 to 6.84,
// even pieces 6.52 to 6.67). Costs in blocks of 64 of a contraction; a launch costs about 15.
static int hd_piece(int T, int H, int V, bool quant, bool grad, bool dw) {
  const long long all = ((long long)V + HD_BN - 1) / HD_BN;
  long long most = all;
  if (grad) most = std::min(most, HD_DZ_BYTES / (2LL * T * HD_BN));
  if (quant) most = std::min(most, HD_WQ_BYTES / (2LL * H * HD_BN));
  most = std::max(most, 1LL);
  if (most == all) return (int)(all * HD_BN);
  const int cg = hd_cg(T);
  const long long mt = (T + HD_BM * cg - 1) / (HD_BM * cg), nt = (H + HD_BN - 1) / HD_BN;
  const long long kh = (H + HD_BK - 1) / HD_BK, kt = (T + HD_BK - 1) / HD_BK;
  const auto cost = [&](long long n) {
    long long c = 15 * (1 + (quant ? 1 : 0) + (grad ? 1 : 0) + (dw ? 1 : 0)) + kh * hd_rounds(mt * n, cg);
    if (dw) c += kt * hd_rounds(nt * n, 2);
    return c;
  };
  long long best = most, best_cost = -1;
  for (long long n = most; n >= 1 && 2 * n >= most; --n) {
    const long long last = all % n, c = all / n * cost(n) + (last ? cost(last) : 0);
    if (best_cost < 0 || c < best_cost) {
      best = n;
      best_cost = c;
    }
  }
  return (int)(best * HD_BN);
}

// Parts of dx's contraction, so that the tiles fill the SMs in whole rounds: the fewest whose last round is within
// 6 % of full, or the best of up to 8 rounds' worth; each part keeps at least 8 blocks of 64.
static int hd_splits(int T, int H, int piece) {
  const int cg = hd_cg(T), slots = device_sm_count() / cg;
  const int tiles = ((T + HD_BM * cg - 1) / (HD_BM * cg)) * ((H + HD_BN - 1) / HD_BN);
  const int most = std::max(1, std::min(piece / (8 * HD_BK), std::max(8, slots / tiles)));
  int best = 1;
  double best_fill = 0;
  for (int s = 1; s <= most; ++s) {
    const long long units = (long long)tiles * s, rounds = (units + slots - 1) / slots;
    const double fill = (double)units / (double)(rounds * slots);
    if (fill > best_fill + 0.02) {
      best_fill = fill;
      best = s;
    }
    if (best_fill > 0.94) break;
  }
  return best;
}

// Parts of dW's contraction, the tokens: where its tiles fill less than half the SMs, as many as fit, of at least 8
// blocks of 64 each (8,192 tokens, 512 ids of 256: 65 us with one part, 36 with 16; 4,757 tokens, 380 ids of 136: 52
// and 36). Not below 40 blocks: the join costs as much (2,048 tokens, 4,000 ids of 256: 39 and 38 us, with a launch
// more).
static int hd_wsplits(int T, int H, int rows) {
  const int cg = hd_cg(rows);
  const long long tiles = (((long long)rows + HD_BM * cg - 1) / (HD_BM * cg)) * ((H + HD_BN - 1) / HD_BN);
  if (T < 40 * HD_BK) return 1;
  const long long fit = device_sm_count() / cg / tiles;
  return (int)std::max(1LL, std::min<long long>(fit, T / (8 * HD_BK)));
}

// The 4-bit loss of few tokens: straight from the codes (head_q4.cu), or by the products over unpacked weights. The
// first takes time by the passes (of up to 128 tokens) and their blocks of 32 tokens, the second by the bytes to
// unpack. Both, us, as measured over V = 6,264 and 77,689, H = 64 to 2,048; of 77,689 ids (codes against products):
//   tokens   H = 64     512        1,024       2,048
//   32       15 : 20    18 : 41    25 : 74     41 : 141
//   128      33 : 20    35 : 38    39 : 72     55 : 142
//   256      58 : 27    64 : 46    71 : 75     100 : 144
//   384      84 : 41    92 : 59    104 : 91    143 : 177
// and of 6,264 ids 24 : 25 for 128 tokens of 2,048, 59 : 26 for 384.
static bool hd_few(int T, int H, int V) {
  if (T > HQ_PASSES * HQ_MAXT) return false;
  if (T <= 32) return true;
  const int passes = (T + HQ_MAXT - 1) / HQ_MAXT, n = (T + passes - 1) / passes, blocks = (n + 31) / 32;
  const double ids = V * 1e-3;
  const double codes = 3 + passes * (7 + 0.04 * n + 0.0026 * H + ids * (0.052 * blocks + 0.00011 * H));
  const double products = 11 + 0.0017 * H + ids * (0.11 * ((T + HD_BM - 1) / HD_BM) + 0.00076 * H);
  return codes < products;
}

struct HdWork {
  HdParts out;
  __nv_bfloat16* xp;  // few tokens and 4 bits: x in the order of a word's codes, ids by target
  int* idt;
  int* sorted;
  unsigned char *order, *start;
  float* sorted_w;
  float2* wsum;
  float *scale, *again;
  __nv_bfloat16 *wq, *dz, *xz;
  float *dx, *dw;  // fp32 parts (dw: NULL where it has one)
  size_t bytes;
  int piece, nt, splits, wsplits;
};

static HdWork hd_carve(void* base, int T, int H, int V, int K, bool quant, bool few, bool grad, bool dx,
                       bool dw, bool top) {
  HdWork w = {};
  Carver c(base);
  w.nt = (V + HD_BN - 1) / HD_BN;
  w.piece = hd_piece(grad ? T + hd_rest(T) : T, H, V, quant, grad, dw);
  if (!grad) {
    w.out.parts = few ? hq_parts(V) : w.nt;
    w.out.maxima = !few;
    w.out.part = c.take<float4>((size_t)T * w.out.parts);
    if (top) w.out.top = c.take<int>((size_t)T * w.out.parts);
    w.out.ztgt = c.take<float>((size_t)T * K);
    if (few) {
      w.xp = c.take<__nv_bfloat16>((size_t)T * H);
      w.idt = c.take<int>((size_t)HQ_PASSES * HQ_MAXT * K);
      w.bytes = align_up(c.used, 256);
      return w;
    }
  }
  if (K > 1) {
    w.sorted = c.take<int>((size_t)T * K);
    w.order = c.take<unsigned char>((size_t)T * K);
    w.sorted_w = c.take<float>((size_t)T * K);
    w.start = c.take<unsigned char>((size_t)T * (w.nt + 1));
    w.wsum = c.take<float2>(T);
  }
  if (quant) w.wq = c.take<__nv_bfloat16>((size_t)std::min(w.piece, V) * H);
  if (grad) {
    w.scale = c.take<float>(1);
    w.again = c.take<float>((size_t)T * K);
    const int rows = T + hd_rest(T);
    w.dz = c.take<__nv_bfloat16>((size_t)rows * w.piece);
    if (dw) {
      w.xz = c.take<__nv_bfloat16>((size_t)rows * H);
      w.wsplits = hd_wsplits(rows, H, std::min(w.piece, V));
      if (w.wsplits > 1) w.dw = c.take<float>((size_t)w.wsplits * std::min(w.piece, V) * H);
    }
    if (dx) {
      w.splits = hd_splits(rows, H, std::min(w.piece, V));
      w.dx = c.take<float>((size_t)w.splits * rows * H);
    }
  }
  w.bytes = align_up(c.used, 256);
  return w;
}

#define HD_TRY(expr)           \
  do {                         \
    const int rc_ = (expr);    \
    if (rc_ != LG_OK) return rc_; \
  } while (0)

template <int KIND, int CG>
static int hd_launch_as(const CUtensorMap& ma, const CUtensorMap& mb, const HdArgs& a, cudaStream_t st) {
  static std::atomic<bool> done[64];
  int dev = 0;
  LG_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= 64 || !done[dev].load(std::memory_order_relaxed)) {
    LG_CUDA_TRY(cudaFuncSetAttribute(hd_kernel<KIND, CG>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)HD_SMEM));
    if (dev < 64) done[dev].store(true, std::memory_order_relaxed);
  }
  const long long units = (long long)a.mt * a.nt * a.splits;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = CG * (int)std::max(1LL, std::min<long long>(units, device_sm_count() / CG));
  cfg.blockDim = hd_threads(KIND);
  cfg.dynamicSmemBytes = HD_SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CG;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  LG_CUDA_TRY(cudaLaunchKernelEx(&cfg, hd_kernel<KIND, CG>, ma, mb, a));
  LG_LAUNCH_CHECK("head");
  return LG_OK;
}

// Operands of a product: [contraction, rows] (mn) or [rows, contraction] matrices of bf16.
struct HdOperand {
  const void* p;
  long long inner, rows, ld;
};

// One CTA a tile where the output has no more than 128 rows, else a pair.
//
// Every kernel of a call starts when the one before has ended. (Starting the products under the small kernels before
// them, by programmatic serialization, took 1 to 2.5 us less a call: 301 tokens of 5 targets 95.5 against 98 us. It is
// not worth the reasoning that it needs: CTAs of 225 KB that wait on an SM for a kernel whose CTAs need SMs.)
template <int KIND>
static int hd_launch(const HdOperand& a, const HdOperand& b, HdArgs g, cudaStream_t st) {
  constexpr bool A_MN = KIND == HD_WGRAD, B_MN = KIND == HD_XGRAD || KIND == HD_WGRAD;
  const int cg = hd_cg(g.M);
  g.mt = (g.M + HD_BM * cg - 1) / (HD_BM * cg);
  g.nt = (g.N + HD_BN - 1) / HD_BN;
  CUtensorMap ma, mb;
  HD_TRY(make_map_2d(&ma, a.p, true, a.inner, a.rows, (uint64_t)a.ld * 2, 64, A_MN ? HD_BK : HD_BM, 128));
  HD_TRY(make_map_2d(&mb, b.p, true, b.inner, b.rows, (uint64_t)b.ld * 2, 64, B_MN ? HD_BK : HD_BN / cg, 128));
  return cg == 2 ? hd_launch_as<KIND, 2>(ma, mb, g, st) : hd_launch_as<KIND, 1>(ma, mb, g, st);
}

static int hd_check(const char* who, const void* x, long long ldx, int T, int H, const void* w,
                    long long ldw, const void* ws, const void* wb, int V, const int* ids, int K) {
  // tokens rounded up to whole tiles stay below 2^31
  LG_CHECK_ARG(T >= 0 && T < 0x7fffffff - 1024 && V >= 1 && V <= (1 << 30), "%s: T=%d V=%d", who, T, V);
  LG_CHECK_ARG(K >= 1 && K <= HD_MAXK, "%s: K=%d targets not in [1, %d]", who, K, HD_MAXK);
  LG_CHECK_ARG((ws == nullptr) == (wb == nullptr), "%s: scales and biases go together", who);
  const int unit = ws ? 64 : 8;
  LG_CHECK_ARG(H >= unit && H <= (1 << 20) && H % unit == 0, "%s: H=%d is not a multiple of %d", who, H, unit);
  LG_CHECK_ARG(w && (T == 0 || (x && ids)), "%s: NULL pointer", who);
  LG_CHECK_ARG(aligned(x, 16) && aligned(w, 16) && aligned(ws, 2) && aligned(wb, 2),
               "%s: x and the weights must be 16-byte aligned", who);
  LG_CHECK_ARG(ldx >= H && ldx % 8 == 0 && ldx < (1LL << 38), "%s: x's row stride %lld", who, ldx);
  LG_CHECK_ARG(ws ? ldw == H : ldw >= H && ldw % 8 == 0 && ldw < (1LL << 38),
               "%s: the weights' row stride %lld", who, ldw);
  LG_CHECK_ARG((long long)((T + HD_BM - 1) / HD_BM) * ((V + HD_BN - 1) / HD_BN) < (1LL << 30),
               "%s: T=%d times V=%d is too large", who, T, V);
  return LG_OK;
}

static int hd_blocks(long long n) { return (int)std::min<long long>((n + 255) / 256, 148 * 16); }

// The piece's bf16 weights, and c if it is asked for.
static int hd_weights(const void* w, const void* ws, const void* wb, int H, int v0, int rows,
                      const HdWork& k, const HdScale& scale, cudaStream_t st) {
  if (!ws) return LG_OK;
  const long long n = (long long)rows * (H / 16);
  const size_t at = (size_t)v0 * (H / 16);
  hd_dequant_kernel<<<hd_blocks(n) + scale.blocks(), 256, 0, st>>>(
      static_cast<const uint2*>(w) + at, static_cast<const uint16_t*>(ws) + at / 4,
      static_cast<const uint16_t*>(wb) + at / 4, n, scale, k.wq);
  LG_LAUNCH_CHECK("head_dequant");
  return LG_OK;
}

static int hd_join_parts(const float* parts, int n, long long size, const float* scale, void* out, cudaStream_t st) {
  hd_sum_kernel<<<hd_blocks(size / 4), 256, 0, st>>>(parts, n, size, scale, static_cast<__nv_bfloat16*>(out));
  LG_LAUNCH_CHECK("head_sum");
  return LG_OK;
}

static int hd_sort(const int* ids, const float* weights, int T, int K, int V, const HdWork& k,
                   cudaStream_t st) {
  if (K == 1) return LG_OK;
  hd_sort_kernel<<<(T + 7) / 8, 256, 0, st>>>(ids, weights, T, K, V, k.nt, k.sorted, k.order, k.sorted_w, k.start,
                                              k.wsum);
  LG_LAUNCH_CHECK("head_sort");
  return LG_OK;
}

static HdArgs hd_args(int T, int V, int K, const int* ids, const float* weights, const HdWork& k) {
  HdArgs a = {};
  a.V = V;
  a.K = K;
  a.ids = K > 1 ? k.sorted : ids;
  a.weights = K > 1 ? k.sorted_w : weights;
  a.order = k.order;
  a.start = k.start;
  a.nt_all = k.nt;
  a.splits = 1;
  a.M = T;
  return a;
}

}  // namespace lg

using namespace lg;

extern "C" size_t lg_head_loss_workspace_bytes(int T, int H, int V, int K, int bits, int top) {
  if (T < 1 || H < 8 || V < 1 || K < 1) return 256;
  const bool quant = bits == 4;
  return hd_carve(nullptr, T, H, V, K, quant, quant && hd_few(T, H, V), false, false, false, top != 0).bytes;
}

extern "C" size_t lg_head_loss_grad_workspace_bytes(int T, int H, int V, int K, int bits, int dx, int dw) {
  if (T < 1 || H < 8 || V < 1 || K < 1) return 256;
  return hd_carve(nullptr, T, H, V, K, bits == 4, false, true, dx != 0, dw != 0, false).bytes;
}

extern "C" int lg_head_status(int* status, int reset) {
  LG_CHECK_ARG(status, "head_status: NULL pointer");
  int here = 0, q4 = 0;
  LG_CUDA_TRY(cudaMemcpyFromSymbol(&here, hd_status_word, sizeof(int)));
  HD_TRY(hq_status(&q4, reset));
  if (reset) {
    const int zero = 0;
    LG_CUDA_TRY(cudaMemcpyToSymbol(hd_status_word, &zero, sizeof(int)));
  }
  *status = here ? here : q4;
  return LG_OK;
}

extern "C" int lg_head_loss(const void* x, long long ldx, int T, int H, const void* w, long long ldw,
                            const void* w_scales, const void* w_biases, int V, const int32_t* ids,
                            const float* weights, int K, float* loss, float* lse, int32_t* top,
                            void* workspace, size_t workspace_bytes, void* stream) {
  HD_TRY(hd_check("head_loss", x, ldx, T, H, w, ldw, w_scales, w_biases, V, ids, K));
  if (T == 0) return LG_OK;
  LG_CHECK_ARG(loss && lse, "head_loss: NULL output");
  const bool quant = w_scales != nullptr;
  const HdHead head = {w, static_cast<const __nv_bfloat16*>(w_scales),
                       static_cast<const __nv_bfloat16*>(w_biases), ldw};
  const __nv_bfloat16* xb = static_cast<const __nv_bfloat16*>(x);
  const bool few = quant && hd_few(T, H, V);
  const HdWork k = hd_carve(workspace, T, H, V, K, quant, few, false, false, false, top != nullptr);
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < k.bytes)
    return fail(LG_ERR_WORKSPACE, "head_loss: workspace of %zu bytes, need %zu", workspace_bytes, k.bytes);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (few) {
    const int passes = (T + HQ_MAXT - 1) / HQ_MAXT;
    for (int i = 0; i < passes; ++i) {  // even shares: a pass's time goes by its blocks of 32 tokens
      const int t0 = (int)((long long)T * i / passes), n = (int)((long long)T * (i + 1) / passes) - t0;
      HdParts out = k.out;
      out.part += (size_t)t0 * out.parts;
      if (out.top) out.top += (size_t)t0 * out.parts;
      out.ztgt += (size_t)t0 * K;
      HD_TRY(hq_loss_parts(xb + (size_t)t0 * ldx, ldx, n, H, head, V, ids + (size_t)t0 * K, K, k.xp + (size_t)t0 * H,
                           k.idt + (size_t)i * HQ_MAXT * K, out, st));
    }
  } else {
    HD_TRY(hd_sort(ids, weights, T, K, V, k, st));
    HdArgs a = hd_args(T, V, K, ids, weights, k);
    a.kblocks = (H + HD_BK - 1) / HD_BK;
    a.out = k.out;
    for (int v0 = 0; v0 < V; v0 += k.piece) {
      const int n = std::min(k.piece, V - v0);
      HD_TRY(hd_weights(w, w_scales, w_biases, H, v0, n, k, {}, st));
      a.N = n;
      a.v0 = v0;
      a.b_row0 = quant ? 0 : v0;
      const HdOperand mw = quant ? HdOperand{k.wq, H, n, H} : HdOperand{w, H, V, ldw};
      HD_TRY(hd_launch<HD_LOSS>({x, H, T, ldx}, mw, a, st));
    }
  }
  const auto join = quant ? hd_join_kernel<true> : hd_join_kernel<false>;
  join<<<T, hj_threads(few), 0, st>>>(k.out, xb, ldx, H, head, ids, weights, K, V, loss, lse, top);
  LG_LAUNCH_CHECK("head_join");
  return LG_OK;
}

extern "C" int lg_head_loss_grad(const void* x, long long ldx, int T, int H, const void* w, long long ldw,
                                 const void* w_scales, const void* w_biases, int V, const int32_t* ids,
                                 const float* weights, int K, const float* lse, const float* g, void* dx,
                                 void* dw, void* workspace, size_t workspace_bytes, void* stream) {
  HD_TRY(hd_check("head_loss_grad", x, ldx, T, H, w, ldw, w_scales, w_biases, V, ids, K));
  const bool quant = w_scales != nullptr;
  LG_CHECK_ARG(T == 0 || dx || dw, "head_loss_grad: neither dx nor dw is asked for");
  LG_CHECK_ARG(!(dw && quant), "head_loss_grad: a 4-bit head has no gradient");
  LG_CHECK_ARG(aligned(dx, 16) && aligned(dw, 16), "head_loss_grad: outputs must be 16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T == 0) {
    if (dw) LG_CUDA_TRY(cudaMemsetAsync(dw, 0, (size_t)V * H * 2, st));
    return LG_OK;
  }
  LG_CHECK_ARG(lse && g, "head_loss_grad: NULL pointer");
  const HdWork k = hd_carve(workspace, T, H, V, K, quant, false, true, dx != nullptr, dw != nullptr, false);
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < k.bytes)
    return fail(LG_ERR_WORKSPACE, "head_loss_grad: workspace of %zu bytes, need %zu", workspace_bytes,
                k.bytes);
  HD_TRY(hd_sort(ids, weights, T, K, V, k, st));
  const HdHead head = {w, static_cast<const __nv_bfloat16*>(w_scales),
                       static_cast<const __nv_bfloat16*>(w_biases), ldw};
  const HdScale scale = {ids, g, weights, k.start, k.wsum, k.scale, T, V, k.nt,
                         static_cast<const __nv_bfloat16*>(x), ldx, H, K, head, lse, k.again};
  if (!quant) {
    hd_rows_kernel<<<scale.blocks() + (dw ? hd_blocks((long long)T * (H / 8)) : 0), 256, 0, st>>>(
        static_cast<const __nv_bfloat16*>(x), ldx, H, scale, hd_rest(T), k.xz);
    LG_LAUNCH_CHECK("head_rows");
  }
  const int rest = hd_rest(T), rows = T + rest;
  for (int v0 = 0; v0 < V; v0 += k.piece) {
    const int n = std::min(k.piece, V - v0);
    HD_TRY(hd_weights(w, w_scales, w_biases, H, v0, n, k, v0 == 0 ? scale : HdScale{}, st));
    const HdOperand mw = quant ? HdOperand{k.wq, H, n, H} : HdOperand{w, H, V, ldw};
    HdArgs a = hd_args(T, V, K, ids, weights, k);
    a.v0 = v0;
    a.b_row0 = quant ? 0 : v0;
    a.N = n;
    a.kblocks = (H + HD_BK - 1) / HD_BK;
    a.lse = lse;
    a.g = g;
    a.wsum = k.wsum;
    a.scale = k.scale;
    a.again = k.again;
    const int ldz = (n + 63) / 64 * 64;
    a.tile_out = k.dz;
    a.width = ldz;
    a.rest = rest;
    HD_TRY(hd_launch<HD_PROB>({x, H, T, ldx}, mw, a, st));
    const HdOperand mz = {k.dz, n, rows, ldz};
    if (dx) {
      HdArgs b = a;
      b.M = rows;
      b.N = H;
      b.kblocks = (n + HD_BK - 1) / HD_BK;
      b.splits = std::min(k.splits, b.kblocks);
      b.add = v0 > 0;
      b.tile_out = k.dx;
      b.width = H;
      HD_TRY(hd_launch<HD_XGRAD>(mz, mw, b, st));
    }
    if (dw) {
      HdArgs b = a;
      b.M = n;
      b.N = H;
      b.kblocks = (rows + HD_BK - 1) / HD_BK;
      b.splits = k.wsplits;
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(dw) + (size_t)v0 * H;
      b.tile_out = k.wsplits > 1 ? static_cast<void*>(k.dw) : out;
      b.width = H;
      HD_TRY(hd_launch<HD_WGRAD>(mz, {k.xz, H, rows, H}, b, st));
      if (k.wsplits > 1) HD_TRY(hd_join_parts(k.dw, k.wsplits, (long long)n * H, k.scale, out, st));
    }
  }
  if (dx) {
    // The last piece may have fewer parts than the first; later parts then kept the earlier sums.
    const int parts = std::min(k.splits, (std::min(k.piece, V) + HD_BK - 1) / HD_BK) * (rest ? 2 : 1);
    HD_TRY(hd_join_parts(k.dx, parts, (long long)T * H, k.scale, dx, st));
  }
  return LG_OK;
}
