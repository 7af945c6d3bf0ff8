// The head's loss for few tokens (up to 128) from 4-bit weights that never become bf16 in memory.
//
// z^T = W x^T in tiles of 128 vocabulary ids (the rows, M) by the tokens (the columns, N = T rounded up to 16):
// the weights are the product's A operand, taken from TMEM, where the warps that unpack them write them; x is B.
// So few tokens cost few columns, and an unpacked weight crosses neither memory nor shared memory.
//
//   warp 0       TMA: packed words (32 rows x 256 codes a box, 128-byte swizzle)
//   warp 2       TMA: x, 128 columns a slot
//   warps 4-19   unpack: a row a thread, 128 codes a turn (two quantization groups), four groups of four warps in
//                turns; tcgen05.st of 32 columns a group. Scales and biases come by plain loads a turn ahead: as
//                TMA boxes (16 bytes of a row) they were a quarter of all rows that TMA moved, and waited for
//   warp 1       four products (M 128, N, K 16) a 64-wide block into one of two accumulators
//   warps 20-23  per tile and token the sum of exponentials over the warp's 32 rows, which lie across its lanes: a
//                transposing reduction (31 shuffles for 32 columns) leaves token i with lane i. The exponentials are
//                taken from a reference per token, the maximum of the warp's first tile, until one lies 2^90 above
//                it; then (and always where the maximum's id is asked for) the maximum is reduced like the sum
//
// Unpacking: q4_word (head.cuh); a warp that holds a scale it does not take unpacks by q4_word_any.
//
// K order: one LOP3 splits a word into the pairs (0,4), (1,5), (2,6), (3,7); x is copied in that order first
// (hq_order_kernel), so that no code is moved.
//
// Each CTA has 1/148 of the blocks of 32 ids. HBM needs 0.56 bytes a weight. 37 tokens, 100,352 ids of 2,048: 48 us a
// call with the order and the join (40 this kernel: 116 MB, 2.9 TB/s). No pipe is near its limit then (HBM 31 %, an
// instruction issued in 54 % of the cycles, a third of those unpacking at nine a word, the tensor pipe busy in 24 %):
// the roles wait for one another. A part of it: 21 or 22 blocks a CTA are six tiles of four, 5.3 of them full.
#include <math.h>

#include <algorithm>
#include <atomic>

#include "head.cuh"
#include "tmap.cuh"

namespace lg {

using namespace tc;

constexpr int HQ_UNPACK = 16;  // warps
constexpr int HQ_THREADS = (8 + HQ_UNPACK) * 32;
constexpr int HQ_BLOCK = 32;               // ids a block: a warp's TMEM lanes
constexpr int HQ_W_BYTES = 4 * 32 * 128;   // a stage of packed words, two turns': 128 rows x 256 codes
constexpr float HQ_FAR = 90.f;             // of exponents of 2: 100,000 terms of 2^90 are below 2^127
constexpr int HQ_SMEM_MAX = 224 << 10;

struct HqArgs {
  int T, N, V, K;
  int kb;       // 64-wide blocks of H
  int blocks;   // blocks of 32 ids
  int ws;        // stages of packed words: even
  bool pairs;    // two groups' scales are one aligned load
  const uint16_t *scales, *biases;
  const int* ids;  // [K][32 NT], -1 past T
  HdParts out;
};

// Slots of unpacked weights and x, 128 columns each: 64 columns of TMEM beside two accumulators of 32 NT. At least 4
// (four groups of warps write side by side).
template <int NT>
constexpr int HQ_SLOTS = NT == 4 ? 4 : 6;

// A[tmem] B[smem]: M 128 x N x 16.
__device__ __forceinline__ void hq_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

__device__ __forceinline__ void hq_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,"
      "%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// Over the warp's lanes: lane i ends with op over all lanes of v[i].
template <typename Op>
__device__ __forceinline__ float hq_across(float (&v)[32], Op op) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float send = up ? v[i] : v[i + o], keep = up ? v[i + o] : v[i];
      v[i] = op(keep, __shfl_xor_sync(0xffffffffu, send, o));
    }
  }
  return v[0];
}

template <int NT>  // blocks of 32 tokens
__global__ void __launch_bounds__(HQ_THREADS, 1)
    hq_kernel(const __grid_constant__ CUtensorMap mw, const __grid_constant__ CUtensorMap mw4,
              const __grid_constant__ CUtensorMap mx, const HqArgs a) {
  constexpr int AS = HQ_SLOTS<NT>;
  extern __shared__ uint8_t hq_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)hq_raw + 1023) & ~(uintptr_t)1023);
  const int x_bytes = a.N * 128;  // 64 columns of x
  uint8_t* sm_w = smem;
  uint8_t* sm_x = sm_w + a.ws * HQ_W_BYTES;
  float* sm_m = reinterpret_cast<float*>(sm_x + 2 * AS * x_bytes);
  float* sm_sum = sm_m + 4 * 32 * NT;
  int* sm_top = reinterpret_cast<int*>(sm_sum + 4 * 32 * NT);
  float* sm_ref = reinterpret_cast<float*>(sm_top + 4 * 32 * NT);
  float* sm_best = sm_ref + 4 * 32 * NT;
  int* sm_at = reinterpret_cast<int*>(sm_best + 4 * 32 * NT);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm_at + 4 * 32 * NT);
  uint64_t *w_full = bars, *w_empty = bars + 8, *full = bars + 16, *empty = bars + 24;
  uint64_t *acc_full = bars + 32, *acc_empty = bars + 34;
  uint64_t* done = bars + 36;
  uint32_t* tmem_base = reinterpret_cast<uint32_t*>(bars + 37);
  int* err = reinterpret_cast<int*>(tmem_base + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // uniform, and known to be
  const int b0 = (int)((long long)a.blocks * blockIdx.x / gridDim.x);
  const int b1 = (int)((long long)a.blocks * (blockIdx.x + 1) / gridDim.x);
  const int tiles = (b1 - b0 + 3) / 4;
  const int turns = (a.kb + 1) / 2;  // of 128 codes (the last perhaps 64), a tile
  const int stages = (turns + 1) / 2;  // of packed words, a tile

  if (threadIdx.x == 0) {
    for (int i = 0; i < a.ws; ++i) {
      mbar_init(w_full + i, 1);
      mbar_init(w_empty + i, 8);  // the two groups of its turns
    }
    for (int i = 0; i < AS; ++i) {
      mbar_init(full + i, 5);  // x's copy and four warps
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full + i, 1);
      mbar_init(acc_empty + i, 4);
    }
    mbar_init(done, 1);
    for (int i = 0; i < 4; ++i) err[i] = 0;  // of all roles; of the two copies' ends; of the products' end
    fence_mbar_init();
    prefetch_tmap(&mw);
    prefetch_tmap(&mw4);
    prefetch_tmap(&mx);
  }
  if (warp == 3) {
    tmem_alloc(tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_base;        // accumulators: columns [0, 64 NT)
  const uint32_t tmem_a = tmem + 64 * NT;  // weights: 64 columns a slot

  if (warp == 0) {
    if (elect_one()) {
      int st = 0, used = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int i = 0; i < tiles && ok; ++i) {
        const int row = (b0 + 4 * i) * HQ_BLOCK, nb = min(4, b1 - b0 - 4 * i);
        for (int k = 0; k < stages; ++k) {
          if (!mbar_wait(w_empty + st, ph ^ 1, err, 2)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(w_full + st, nb * 4096);
          if (nb == 4) {
            tma_load_2d(sm_w + st * HQ_W_BYTES, &mw4, w_full + st, k * 32, row);
          } else {
            for (int j = 0; j < nb; ++j)
              tma_load_2d(sm_w + st * HQ_W_BYTES + j * 4096, &mw, w_full + st, k * 32, row + j * HQ_BLOCK);
          }
          if (used < a.ws) ++used;
          if (++st == a.ws) {
            st = 0;
            ph ^= 1;
          }
        }
      }
      // Every copy has landed before the CTA ends.
      for (int j = used; j > 0; --j) {
        const int s = (st - j + a.ws) % a.ws;
        mbar_wait(w_full + s, s < st ? ph : ph ^ 1, err + 1, 2, 400000000LL);
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    if (elect_one()) {
      int st = 0, used = 0;
      uint32_t ph = 0;
      bool ok = true;
#pragma unroll 1
      for (int i = 0; i < tiles && ok; ++i) {
#pragma unroll 1
        for (int k = 0; k < a.kb; k += 2) {
          if (!mbar_wait(empty + st, ph ^ 1, err, 3)) {
            ok = false;
            break;
          }
          // both 64s of the turn: [2][N][64] (the second of an odd H / 64 lies past H: zeros)
          mbar_arrive_expect_tx(full + st, 2 * x_bytes);
          tma_load_3d(sm_x + 2 * st * x_bytes, &mx, full + st, 0, 0, k);
          if (used < AS) ++used;
          if (++st == AS) {
            st = 0;
            ph ^= 1;
          }
        }
      }
      // The products have freed the last slots before the CTA ends: their copies have landed, the commits have
      // arrived. (After a wait that ran out, 0.2 s pass for the copies.)
      for (int j = used; j > 0; --j) {
        const int s = (st - j + AS) % AS;
        mbar_wait(empty + s, s < st ? ph : ph ^ 1, err + 2, 3, 400000000LL);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // The whole warp goes through the loop and one lane issues: counters and descriptors then stay in uniform
    // registers. With a lane's own loop each product's operands were moved there first, and this warp, which has
    // a sixth of its scheduler's issue slots beside the unpacking ones, was what all others waited for.
    const uint32_t idesc = idesc_bf16(128, a.N);
    const uint64_t hi = (uint64_t)SW128_HI << 32;
    const uint32_t xd = sw128_lo(smem_u32(sm_x)), step = x_bytes >> 4;
    int slot = 0;
    uint32_t ph = 0;
    bool ok = true;
#pragma unroll 1
    for (int i = 0; i < tiles && ok; ++i) {
      const int acc = i & 1;
      ok = __all_sync(0xffffffffu, mbar_wait(acc_empty + acc, ((i >> 1) & 1) ^ 1, err, 4));
      if (!ok) break;
      const uint32_t d = tmem + acc * 32 * NT;
#pragma unroll 1
      for (int k = 0; k < a.kb; k += 2) {
        ok = __all_sync(0xffffffffu, mbar_wait(full + slot, ph, err, 5));
        if (!ok) break;
        tc_fence_after();
        const uint32_t da = tmem_a + slot * 64, db = xd + 2 * slot * step;
        if (elect_one()) {
#pragma unroll
          for (int j = 0; j < 4; ++j) hq_mma(d, da + j * 8, hi | (db + j * 2), idesc, k > 0 || j > 0);
          if (k + 1 < a.kb) {
#pragma unroll
            for (int j = 0; j < 4; ++j) hq_mma(d, da + 32 + j * 8, hi | (db + step + j * 2), idesc, 1);
          }
          umma_commit(empty + slot);
        }
        __syncwarp();
        if (++slot == AS) {
          slot = 0;
          ph ^= 1;
        }
      }
      if (ok && elect_one()) umma_commit(acc_full + acc);
      __syncwarp();
    }
    if (elect_one()) umma_commit(done);
    __syncwarp();
  } else if (warp >= 4 && warp < 4 + HQ_UNPACK) {
    // Stage s holds two turns, of groups 2 s % 4 and the next one (a tile's last stage may have one turn: its second
    // group unpacks nothing). The number of stages is even, so that a stage is always the same groups': nobody looks at
    // the barrier of another's, two phases early or late, where the parity is the same. The slots' barriers have no
    // such case as long as a group waits for one of every four turns, or of as many as there are slots: the products
    // end in order, so that the turn two rounds before the one waited for has then ended. A group without a turn
    // therefore waits as the next turn's group does.
    const int q = warp & 3, group = (warp >> 2) & 3, half = group & 1;
    const int r = q * 32 + lane;
    const uint32_t lanes = (uint32_t)(q * 32) << 16;
    int i = 0, st = group >> 1;  // tile, stage in it
    while (st >= stages) st -= stages, ++i;
    int ws = group >> 1;
    uint32_t wph = 0;
    bool ok = true;
    // Scales and biases of this row's two groups in turn 2 st + half of tile i.
    const auto scales = [&](int i, int st, uint32_t& sw, uint32_t& bw) {
      const int blk = b0 + 4 * i + q, row = blk * HQ_BLOCK + lane, k = 2 * (2 * st + half);
      sw = bw = 0;
      if (blk < b1 && row < a.V && k < a.kb) {
        const size_t at = (size_t)row * a.kb + k;
        if (!hd_ok(row >= 0 && k >= 0 && k < a.kb, 21)) return;
        if (a.pairs) {
          sw = __ldg(reinterpret_cast<const uint32_t*>(a.scales + at));
          bw = __ldg(reinterpret_cast<const uint32_t*>(a.biases + at));
        } else {
          const int two = k + 1 < a.kb;
          sw = __ldg(a.scales + at) | (uint32_t)__ldg(a.scales + at + two) << 16;
          bw = __ldg(a.biases + at) | (uint32_t)__ldg(a.biases + at + two) << 16;
        }
      }
    };
    uint32_t next_s = 0, next_b = 0;
    if (i < tiles) scales(i, st, next_s, next_b);
    while (i < tiles) {
      const bool mine = q < b1 - b0 - 4 * i;
      const int k2 = 2 * st + half;
      const uint32_t sw = next_s, bw = next_b;
      int ni = i, ns = st + 2;
      while (ns >= stages) ns -= stages, ++ni;
      if (ni < tiles) scales(ni, ns, next_s, next_b);
      ok = __all_sync(0xffffffffu, mbar_wait(w_full + ws, wph, err, 7));
      if (!ok) break;
      const unsigned n = i * turns + min(k2, turns), turn = n / AS;
      const int slot = n - turn * AS;
      if (k2 == turns) {
        ok = __all_sync(0xffffffffu, mbar_wait(empty + slot, (turn & 1) ^ 1, err, 8));
        if (!ok) break;
      } else {
        {
          const bool two = 2 * k2 + 1 < a.kb;
          const bool fast = __all_sync(0xffffffffu, !mine || q4_fast(sw));
          if (!hd_ok(ws >= 0 && ws < a.ws && slot >= 0 && slot < AS && (tmem & 0x1ff) == 0, 22)) {
            ok = false;
            break;
          }
          const uint8_t* row = sm_w + ws * HQ_W_BYTES + r * 128;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h == 1 && !two) break;
            const int c = half * 4 + h * 2;  // 16-byte chunks of the row's 128
            const uint4 w0 = *reinterpret_cast<const uint4*>(row + ((c ^ (lane & 7)) << 4));
            const uint4 w1 = *reinterpret_cast<const uint4*>(row + (((c + 1) ^ (lane & 7)) << 4));
            const uint32_t w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
            const uint32_t s2 = __byte_perm(sw, 0, h ? 0x3232 : 0x1010), b2 = __byte_perm(bw, 0, h ? 0x3232 : 0x1010);
            uint32_t v[32];
            if (fast) {
#pragma unroll
              for (int j = 0; j < 8; ++j) q4_word(w[j], s2, b2, v + 4 * j);
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j) q4_word_any(w[j], s2, b2, v + 4 * j);
            }
            if (h == 0) {
              ok = __all_sync(0xffffffffu, mbar_wait(empty + slot, (turn & 1) ^ 1, err, 8));
              if (!ok) break;
              tc_fence_after();
            }
            if (mine) hq_st32(tmem_a + slot * 64 + h * 32 + lanes, v);
          }
          if (!ok) break;
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(full + slot);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(w_empty + ws);
      if ((ws += 2) >= a.ws) {
        ws -= a.ws;
        wph ^= 1;
      }
      i = ni;
      st = ns;
    }
  } else if (warp >= 4 + HQ_UNPACK) {
    const int q = warp & 3;
    const float nan = __int_as_float(0x7fffffff);
    float mx[NT], sum[NT];  // of token c * 32 + lane: the reference (its maximum so far, or that of some tile), the sum
    int top[NT];
    float* ref = sm_ref + q * 32 * NT;  // -reference * log2(e) of each token; -inf past T: their columns hold anything
    float* best = sm_best + q * 32 * NT;  // the largest sum of one block's exponentials, and the block
    int* best_at = sm_at + q * 32 * NT;
#pragma unroll
    for (int c = 0; c < NT; ++c) {
      mx[c] = -INFINITY;
      sum[c] = 0.f;
      top[c] = 0x7fffffff;
      ref[c * 32 + lane] = -INFINITY;
      best[c * 32 + lane] = 0.f;
      best_at[c * 32 + lane] = 0;
    }
    bool ok = true;
    for (int i = 0; i < tiles && ok; ++i) {
      const int acc = i & 1;
      ok = __all_sync(0xffffffffu, mbar_wait(acc_full + acc, (i >> 1) & 1, err, 9));
      if (!ok) break;
      tc_fence_after();
      const int blk = b0 + 4 * i + q;
      if (blk < b1) {
        const int id0 = blk * HQ_BLOCK;  // this warp's ids: id0 + lane
        const bool in = id0 + lane < a.V;
#pragma unroll
        for (int c = 0; c < NT; ++c) {
          float v[32];
          const auto load = [&](float (&v)[32]) {
            __syncwarp();
            tmem_ld32_wait(tmem + acc * 32 * NT + c * 32 + ((uint32_t)(q * 32) << 16), v);
            if (!in) {
#pragma unroll
              for (int b = 0; b < 32; ++b) v[b] = -INFINITY;
            }
          };
          load(v);
#pragma unroll 4
          for (int j = 0; j < a.K; ++j) {
            const int id = a.ids[j * 32 * NT + c * 32 + lane];
            unsigned hit = __ballot_sync(0xffffffffu, (unsigned)id - (unsigned)id0 < 32u);
            while (hit) {  // token c * 32 + b has its target in lane id - id0
              const int b = __ffs(hit) - 1;
              hit &= hit - 1;
              const int at = __shfl_sync(0xffffffffu, id, b) - id0;
              if (lane == at && hd_ok(c * 32 + b < a.T, 20))
                a.out.ztgt[(size_t)(c * 32 + b) * a.K + j] = hd_pick(v, b);
            }
          }
          const bool live = c * 32 + lane < a.T;
          float far = 0.f;
          const auto exponents = [&]() {
            far = -INFINITY;
#pragma unroll
            for (int b = 0; b < 32; b += 4) {
              const float4 o = *reinterpret_cast<const float4*>(ref + c * 32 + b);
              v[b] = fmaf(v[b], HD_LOG2E, o.x);
              v[b + 1] = fmaf(v[b + 1], HD_LOG2E, o.y);
              v[b + 2] = fmaf(v[b + 2], HD_LOG2E, o.z);
              v[b + 3] = fmaf(v[b + 3], HD_LOG2E, o.w);
              far = fmaxf(far, fmaxf(fmaxf(v[b], v[b + 1]), fmaxf(v[b + 2], v[b + 3])));
            }
          };
          bool anew = a.out.top || __any_sync(0xffffffffu, live && mx[c] == -INFINITY);
          if (!anew) {
            exponents();
            anew = __any_sync(0xffffffffu, far > HQ_FAR);
            if (anew) load(v);
          }
          if (anew) {
            const float cm = hq_across(v, [](float x, float y) { return fmaxf(x, y); });
            load(v);  // the logits again, in the reduction's registers
            if (a.out.top) {
              int arg = 0;
#pragma unroll
              for (int b = 0; b < 32; ++b) {
                const unsigned hit = __ballot_sync(0xffffffffu, v[b] == __shfl_sync(0xffffffffu, cm, b));
                if (lane == b && hit) arg = __ffs(hit) - 1;
              }
              if (cm > mx[c]) top[c] = id0 + arg;
            }
            if (cm > mx[c]) {
              const float down = hd_ex2((mx[c] - cm) * HD_LOG2E);  // mx = -inf: sum is 0 (or NaN)
              sum[c] *= down;
              best[c * 32 + lane] *= down;
              mx[c] = cm;
            }
            if (live) ref[c * 32 + lane] = mx[c] == -INFINITY ? 0.f : -mx[c] * HD_LOG2E;
            __syncwarp();
            exponents();
          }
#pragma unroll
          for (int b = 0; b < 32; ++b) v[b] = hd_ex2(v[b]);
          const float block = hq_across(v, [](float x, float y) { return x + y; });
          sum[c] += block;
          if (block > best[c * 32 + lane]) {
            best[c * 32 + lane] = block;
            best_at[c * 32 + lane] = id0;
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty + acc);
    }
#pragma unroll
    for (int c = 0; c < NT; ++c) {
      sm_m[q * 32 * NT + c * 32 + lane] = mx[c];
      sm_sum[q * 32 * NT + c * 32 + lane] = ok ? sum[c] : nan;
      sm_top[q * 32 * NT + c * 32 + lane] = top[c];
    }
  }
  if (warp == 3) {
    mbar_wait(done, 0, err + 3, 10, 8000000000LL);
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 3) tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0 && (err[0] || err[1] || err[2] || err[3]))
    hd_record(5, err[0] ? err[0] : err[1] ? err[1] : err[2] ? err[2] : err[3]);
  // The four warps' parts, in their order.
  if (threadIdx.x < a.T) {
    const int t = threadIdx.x;
    float mx = -INFINITY, sum = 0.f, best = 0.f;
    int top = 0x7fffffff, at = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float m = sm_m[q * 32 * NT + t], s = sm_sum[q * 32 * NT + t];
      const int p = sm_top[q * 32 * NT + t];
      float b = sm_best[q * 32 * NT + t];
      if (m > mx) {
        const float down = hd_ex2((mx - m) * HD_LOG2E);
        sum = sum * down + s;
        best *= down;
        mx = m;
        top = p;
      } else {
        const float down = m == -INFINITY ? 1.f : hd_ex2((m - mx) * HD_LOG2E);
        sum += s * down;
        b *= down;
        if (m == mx && p < top) top = p;
      }
      if (b > best) {
        best = b;
        at = sm_at[q * 32 * NT + t];
      }
    }
    if (hd_ok(blockIdx.x < a.out.parts, 23))
      a.out.part[(size_t)t * a.out.parts + blockIdx.x] = make_float4(mx, sum, best, __int_as_float(at));
    if (a.out.top) a.out.top[(size_t)t * a.out.parts + blockIdx.x] = top;
  }
}

// x with every eight columns in the order 0, 4, 1, 5, 2, 6, 3, 7, and the ids by target [K][nt] (-1 past T).
__global__ void __launch_bounds__(256) hq_order_kernel(const __nv_bfloat16* __restrict__ x, long long ldx, int n,
                                                       int per, __nv_bfloat16* __restrict__ out,
                                                       const int* __restrict__ ids, int T, int K, int nt,
                                                       int* __restrict__ idt) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < K * nt) {
    const int t = i % nt, j = i / nt;
    idt[i] = t < T ? ids[(size_t)t * K + j] : -1;
  }
  if (i >= n) return;
  const int t = i / per, c = i % per;
  const uint4 v = *reinterpret_cast<const uint4*>(x + (size_t)t * ldx + 8 * c);
  reinterpret_cast<uint4*>(out)[i] =
      make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                 __byte_perm(v.y, v.w, 0x7632));
}

static int hq_nt(int T) { return T <= 32 ? 1 : T <= 64 ? 2 : 4; }

// Sizes and the stages that fit; returns the bytes of shared memory (at most 128 tokens: 64 KB of stages and 128 of x
// always do).
static size_t hq_layout(int T, int H, HqArgs* a) {
  const int NT = hq_nt(T);
  a->N = (T + 15) / 16 * 16;
  a->kb = H / 64;
  const int slots = NT == 4 ? HQ_SLOTS<4> : HQ_SLOTS<1>;
  const size_t fixed = 1024 + (size_t)24 * 32 * NT * 4 + 38 * 8 + 32 + (size_t)2 * slots * a->N * 128;
  for (a->ws = 8; a->ws > 4 && fixed + (size_t)a->ws * HQ_W_BYTES > HQ_SMEM_MAX; a->ws -= 2) {
  }
  return fixed + (size_t)a->ws * HQ_W_BYTES;
}

int hq_status(int* status, int reset) {
  LG_CUDA_TRY(cudaMemcpyFromSymbol(status, hd_status_word, sizeof(int)));
  const int zero = 0;
  if (reset) LG_CUDA_TRY(cudaMemcpyToSymbol(hd_status_word, &zero, sizeof(int)));
  return LG_OK;
}

int hq_parts(int V) { return std::min(device_sm_count(), (V + HQ_BLOCK - 1) / HQ_BLOCK); }

template <int NT>
static int hq_launch(const CUtensorMap (&m)[3], const HqArgs& a, int grid, size_t smem, cudaStream_t st) {
  static std::atomic<bool> done[64];
  int dev = 0;
  LG_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= 64 || !done[dev].load(std::memory_order_relaxed)) {
    LG_CUDA_TRY(cudaFuncSetAttribute(hq_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, HQ_SMEM_MAX));
    if (dev < 64) done[dev].store(true, std::memory_order_relaxed);
  }
  hq_kernel<NT><<<grid, HQ_THREADS, smem, st>>>(m[0], m[1], m[2], a);
  LG_LAUNCH_CHECK("head_q4");
  return LG_OK;
}

int hq_loss_parts(const __nv_bfloat16* x, long long ldx, int T, int H, const HdHead& w, int V, const int* ids,
                  int K, __nv_bfloat16* xp, int* idt, const HdParts& out, cudaStream_t st) {
  HqArgs a = {};
  const size_t smem = hq_layout(T, H, &a);
  a.T = T;
  a.V = V;
  a.K = K;
  a.blocks = (V + HQ_BLOCK - 1) / HQ_BLOCK;
  a.ids = idt;
  a.scales = reinterpret_cast<const uint16_t*>(w.scales);
  a.biases = reinterpret_cast<const uint16_t*>(w.biases);
  a.pairs = a.kb % 2 == 0 && aligned(w.scales, 4) && aligned(w.biases, 4);
  a.out = out;
  const int n = T * (H / 8);
  const int nt = 32 * hq_nt(T);
  hq_order_kernel<<<(std::max(n, K * nt) + 255) / 256, 256, 0, st>>>(x, ldx, n, H / 8, xp, ids, T, K, nt, idt);
  LG_LAUNCH_CHECK("head_order");
  CUtensorMap m[3];
  int rc = make_map_2d(&m[0], w.w, false, H / 8, V, (uint64_t)H / 2, 32, 32, 128);
  if (rc == LG_OK) rc = make_map_2d(&m[1], w.w, false, H / 8, V, (uint64_t)H / 2, 32, 128, 128);
  const uint64_t dims[3] = {64, (uint64_t)T, (uint64_t)H / 64}, strides[2] = {(uint64_t)H * 2, 128};
  const uint32_t box[3] = {64, (uint32_t)a.N, 2};
  if (rc == LG_OK) rc = make_map_nd(&m[2], xp, 3, dims, strides, box);
  if (rc != LG_OK) return rc;
  const int grid = out.parts;
  return T <= 32 ? hq_launch<1>(m, a, grid, smem, st)
         : T <= 64 ? hq_launch<2>(m, a, grid, smem, st)
                   : hq_launch<4>(m, a, grid, smem, st);
}

}  // namespace lg
