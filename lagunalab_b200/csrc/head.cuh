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

// Unpacking a word of eight 4-bit codes to bf16(scale * code + bias) in one rounding, as the pairs (0,4), (1,5),
// (2,6), (3,7); s2, b2: scale and bias twice.
//
// The 16 bits of a pair's half that hold a code c, all else masked away, are the bf16 number c 2^-133 (codes in bits
// 0-3) or c 2^-129 (bits 4-7): below the exponent 2 a bf16's bits count units of 2^-133. A packed fma with
// scale 2^133 or scale 2^129 and the bias is the result: a shift, four LOP3 and four fma a word. That takes scales
// in [2^-126, 2^-5) (q4_fast); any other: 128 + c put together, 128 taken off, 15 instructions a word.
__device__ __forceinline__ uint32_t q4_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ bool q4_fast(uint32_t s2) {  // both halves' exponents in [1, 121]
  const uint32_t e = s2 & 0x7F807F80u;
  return (((e + 0x43004300u) | (e - 0x00800080u)) & 0x80008000u) == 0;
}
__device__ __forceinline__ void q4_word(uint32_t w, uint32_t s2, uint32_t b2, uint32_t* v) {
  const uint32_t lo = s2 + 0x42804280u, hi = s2 + 0x40804080u;  // * 2^133, * 2^129
  const uint32_t u = w >> 8;
  v[0] = q4_fma(w & 0x000F000Fu, lo, b2);
  v[1] = q4_fma(w & 0x00F000F0u, hi, b2);
  v[2] = q4_fma(u & 0x000F000Fu, lo, b2);
  v[3] = q4_fma(u & 0x00F000F0u, hi, b2);
}
__device__ __forceinline__ void q4_word_any(uint32_t w, uint32_t s2, uint32_t b2, uint32_t* v) {
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    uint32_t c;
    asm("{\n\t"
        "lop3.b32 %0, %1, 0x000F000F, 0x43004300, 0xEA;\n\t"
        "sub.rn.bf16x2 %0, %0, %2;\n\t}"
        : "=r"(c)
        : "r"(w >> (4 * p)), "r"(0x43004300u));
    v[p] = q4_fma(c, s2, b2);
  }
}

// The head as the caller has it: bf16 rows `ld` apart, or (scales not NULL) 4-bit words.
struct HdHead {
  const void* w;
  const __nv_bfloat16 *scales, *biases;
  long long ld;
};

// Where the parts of a loss go before they are joined: per token `parts` times (maximum or another reference, sum of
// exponentials from it, the share of that sum which the heaviest 32 ids have, the first of these), the ids of the
// maxima (or NULL), and the targets' logits.
struct HdParts {
  float4* part;  // [T, parts]
  int* top;      // [T, parts]
  float* ztgt;   // [T, K]
  int parts;
  bool maxima;  // the references are the maxima
};

// The first wait of a source file's kernels that ran out: kernel << 8 | code of the wait (lg_head_status).
static __device__ int hd_status_word;
__device__ __forceinline__ void hd_record(int kernel, int code) { atomicCAS(&hd_status_word, 0, kernel << 8 | code); }

// An index that the kernels' own arithmetic keeps in bounds: where it is not, the access is left out and its site
// recorded as kernel 6. The kernels stay in this form: it is the one that long runs were made with.
__device__ __forceinline__ bool hd_ok(bool in, int site) {
  if (!in) hd_record(6, site);
  return in;
}

// head_q4.cu: the loss's parts from a 4-bit head for few tokens, without the bf16 weights in memory: up to HQ_MAXT
// tokens a pass over the weights. xp: T H bf16, idt: HQ_MAXT K ints of workspace. Taken for up to
// HQ_PASSES passes, where that is faster than the products of head.cu over unpacked weights.
constexpr int HQ_MAXT = 128, HQ_PASSES = 3;
int hq_parts(int V);
int hq_status(int* status, int reset);
int hq_loss_parts(const __nv_bfloat16* x, long long ldx, int T, int H, const HdHead& w, int V, const int* ids,
                  int K, __nv_bfloat16* xp, int* idt, const HdParts& out, cudaStream_t st);

}  // namespace lg
