// What the kernels over a paged cache in 8 bits share: where a block's bytes are, and
// e4m3 numbers.
//
// Keys lie in rows of a token, as a contraction over channels takes them; values in runs
// of 32 tokens of a channel, as a contraction over tokens does.  Bytes of a row or run are
// in the order that the kernels want them in shared memory, where whole blocks arrive as
// they are:
//   * a key row's 16-byte pieces turn with the token, which is the 128-byte (head_dim 64:
//     64-byte) swizzle that tcgen05 reads operands in, and keeps eight rows' pieces apart
//     in banks;
//   * a value run has for each of the four threads of an mma.sync column the tokens that
//     follow each other in its operand registers, side by side.
#pragma once

#include "paged_common.cuh"

namespace kivi {

__host__ __device__ __forceinline__ int key8_offset(int t, int d, int D) {           // t: token of the page
    const int turn = D % 128 == 0 ? t & 7 : D == 64 ? (t >> 1) & 3 : 0;
    return t * D + (((d >> 4) ^ turn) << 4) + (d & 15);
}
__host__ __device__ __forceinline__ int value8_run(int G) { return G % 32 == 0 ? 32 : 16; }
__host__ __device__ __forceinline__ int value8_place(int u, int run) {               // u: token of the run
    return ((u >> 1) & 3) * (run / 4) + (u >> 4) * 4 + ((u >> 3) & 1) * 2 + (u & 1);
}
__host__ __device__ __forceinline__ int value8_offset(int t, int d, int D, int run) { return (t / run * D + d) * run + value8_place(t % run, run); }

constexpr float kPerLargest = 1.0f / 448.0f, kLeastScale = 1e-30f;          // (448: the largest e4m3 number)

#ifdef __CUDACC__

// two numbers to e4m3, the first in the low byte; beyond the largest: the largest
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
    uint16_t y;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(y) : "f"(hi), "f"(lo));
    return y;
}
// two e4m3 numbers as fp16, which holds them exactly
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t two) {
    uint32_t y;
    asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(y) : "r"(two));
    return y;
}
// a word's four numbers, two and two
__device__ __forceinline__ void e4m3x4_to_half2(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ float half_lo(uint32_t h) {
    float y;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.f32.f16 %0, a;\n\t}" : "=f"(y) : "r"(h));
    return y;
}
__device__ __forceinline__ float half_hi(uint32_t h) {
    float y;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.f32.f16 %0, b;\n\t}" : "=f"(y) : "r"(h));
    return y;
}
// a word's four numbers
__device__ __forceinline__ float4 e4m3x4(uint32_t w) {
    uint32_t a, b;
    e4m3x4_to_half2(w, a, b);
    return make_float4(half_lo(a), half_hi(a), half_lo(b), half_hi(b));
}

__device__ __forceinline__ void settle_paged8(kivi_paged8_layer& L, kivi_paged_batch& b) {
    L.k_codes = settled(L.k_codes); L.k_scales = settled(L.k_scales);
    L.v_codes = settled(L.v_codes); L.v_scales = settled(L.v_scales);
    L.k_res = settled(L.k_res); L.v_res = settled(L.v_res);
    b.page_table = settled(b.page_table); b.slots = settled(b.slots);
    b.seq_lens = settled(b.seq_lens); b.cu_new = settled(b.cu_new);
}

#endif

// ---- host side -------------------------------------------------------------------
int validate_paged8(const kivi_paged8_layer* L);
int validate_batch8(const kivi_paged8_layer* L, const kivi_paged_batch* b);

}  // namespace kivi
