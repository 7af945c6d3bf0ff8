// What the head's kernels share (head.cu, head_q4.cu).
#pragma once

#include "common.cuh"
#include "tc_ptx.cuh"

namespace lg {

constexpr int HD_MAXK = 64;  // targets a token
constexpr float HD_LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float hd_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// v[c] with a runtime c, by selects (registers have no index).
__device__ __forceinline__ float hd_pick(const float (&v)[32], int c) {
  float r = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) r = i == c ? v[i] : r;
  return r;
}
__device__ __forceinline__ uint32_t hd_pack(float a, float b) {
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

// The head as the caller has it: bf16 rows `ld` apart, or (scales not NULL) 4-bit words.
struct HdHead {
  const void* w;
  const __nv_bfloat16 *scales, *biases;
  long long ld;
};

// Where the parts of a loss go before they are joined: per token `parts` pairs (maximum, sum of
// exponentials from it), the ids of the maxima (or NULL), and the targets' logits.
struct HdParts {
  float2* part;  // [T, parts]
  int* top;      // [T, parts]
  float* ztgt;   // [T, K]
  int parts;
};

// head_q4.cu: the loss's parts from a 4-bit head for few tokens, without the bf16 weights in memory. xp: T H
// bf16, idt: HQ_MAXT K ints of workspace.
constexpr int HQ_MAXT = 128;
bool hq_takes(int T, int H, int V, int K, const HdHead& w);
int hq_parts(int V);
int hq_loss_parts(const __nv_bfloat16* x, long long ldx, int T, int H, const HdHead& w, int V, const int* ids,
                  int K, __nv_bfloat16* xp, int* idt, const HdParts& out, cudaStream_t st);

}  // namespace lg
