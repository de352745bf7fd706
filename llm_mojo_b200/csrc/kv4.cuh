// The 4-bit key/value cache: its layout and the conversions of its two formats.
//
// Codes are e2m1, two to a byte, the first value in the low nibble; every 16 values along the head share an e4m3 scale; all keys share one
// power of two and all values another.  value = e2m1 * e4m3 * 2^exp: at most 2 x 4 significant bits, exact in bf16, and without the power of
// two (0 or 2^-10 .. 2688) exact in f16 as well.  A row (one token, one head) with a non-finite key or value is kept with all scales NaN in both.
#pragma once
#include "common.cuh"

struct Kv4Desc {
  uint8_t *kc, *ks, *vc, *vs;
  long long code_layer, code_slot, scale_layer, scale_slot;     // strides in bytes; heads, tokens and values lie densely
  int layers, slots, heads, capacity, head_size, k_exp, v_exp, pad;
};
static_assert(sizeof(Kv4Desc) == 96, "the Python side (ops/kv4.py) lays it out alike; a change counts as one of the arguments (LLMB_ABI)");

namespace kv4 {
constexpr int PAGE = 64;
constexpr int BLOCK = 16;                                       // values that share a scale

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }        // -126 <= e <= 127

// two values to e2m1, ties to even, saturating: lo in the low nibble
__device__ __forceinline__ uint32_t e2m1x2(float lo, float hi) {
  uint32_t q;
  asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %1, %2;\n\tcvt.u32.u8 %0, t;\n\t}" : "=r"(q) : "f"(hi), "f"(lo));
  return q;
}
// two e2m1 values of a byte (0 .. 255) as f16x2, the low nibble in the low half
__device__ __forceinline__ uint32_t e2m1x2_f16x2(uint32_t byte) {
  uint32_t h;
  asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(h) : "r"(byte));
  return h;
}
// e4m3 of v >= 0, ties to even, saturating at 448
__device__ __forceinline__ uint32_t e4m3(float v) {
  uint16_t q;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(q) : "f"(0.f), "f"(v));
  return q & 0xff;
}
// two e4m3 values of 16 bits as f16x2
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint32_t two) {
  uint32_t h;
  asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(h) : "r"(two));
  return h;
}
__device__ __forceinline__ float2 f16x2_f32(uint32_t h) {
  float2 f;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(f.x), "=f"(f.y) : "r"(h));
  return f;
}
__device__ __forceinline__ float e4m3_f32(uint32_t byte) { return f16x2_f32(e4m3x2_f16x2(byte)).x; }
}  // namespace kv4

// One call of the attention over a cache.
struct Kv4Attn {
  Kv4Desc d;
  void* out; const void* q;
  const int *lens, *counts, *pages;
  int layer, n, group, splits;
  float scale_log2;
  long long qb, qt, qh, ob, ot, oh;                    // element strides
  int* status;
  bool q_vec, o_vec;                                   // rows of q can be read 16 bytes at a time, those of out written four values at a time
};

// Many rows, on the tcgen05 kernel (bf16, heads of 64): attention_kv4_prompt.cu
int kv4_attention_prompt(const Kv4Attn& p, cudaStream_t st);
