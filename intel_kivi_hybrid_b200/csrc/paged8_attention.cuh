// Arguments that the attention kernels over a paged cache in 8 bits share, and what a row sees.
#pragma once

#include "paged8.cuh"
#include "paged_attention.cuh"

namespace kivi {

struct Paged8Attn {
    kivi_paged8_layer L;
    kivi_paged_batch b;
    kivi_rows q, k, v, out;
    kivi_score_rules rules;
    int q_dtype, out_dtype, n_rep, vec;
    float scale;                 // of q k
    int pieces, chunk;           // a block's tiles of tokens are cut into pieces of `chunk` (no block has more than `pieces`)
    float *part_o, *part_ml;     // [block][KV head][piece][row]: unnormalised output, (maximum, sum) in powers of two
    int* notes;                  // of CTAs to the fold (attn_paged8_decode.cu)
};

// The tiles of T tokens that rows at places p_lo .. p_hi of a sequence of `total` tokens see something of: those of
// the prefix and those from the first row's window on, without what lies between.
struct Span {
    int n, n1, gap;              // tiles; tile v is token tile v for v < n1, else v + gap
    __host__ __device__ __forceinline__ int tile(int v) const { return v < n1 ? v : v + gap; }
};
__host__ __device__ __forceinline__ Span span_of(int T, int total, int p_lo, int p_hi, int window, int prefix) {
    const int P = prefix < 0 ? 0 : prefix < total ? prefix : total, end = p_hi + 1 > P ? p_hi + 1 : P;
    const int from = window > 0 && p_lo >= window ? p_lo - window + 1 : 0;
    Span s{(end + T - 1) / T, 0, 0};
    if (from > P) {
        s.n1 = (P + T - 1) / T;
        const int second = from / T > s.n1 ? from / T : s.n1;
        s.gap = second - s.n1;
        s.n -= s.gap;
    }
    return s;
}
// first token of a row's window (the row is at place p)
__host__ __device__ __forceinline__ int window_from(int p, int window) { return window > 0 && p >= window ? p - window + 1 : 0; }

// cap * tanh(z) where exponentials are cheaper than tanhf.  Up to |z| = kTanhNear z times an even polynomial, fitted (tanh z to
// 1.2e-6 of itself, in fp32); beyond by tanh z = 1 - 2 / (1 + e^(2z)), which near 0 would be off by 2^-23 of the cap, whatever
// the score.
constexpr float kTanhNear = 0.8f;
constexpr float kSmallCap = 256.0f;                      // up to it the latter does for all scores: off by 2^-13 at the most
constexpr float kTanh1 = 0.9999990463256836f, kTanh3 = -0.33325737714767456f, kTanh5 = 0.13233496248722076f, kTanh7 = -0.04925421252846718f, kTanh9 = 0.012158339843153954f;

#ifdef __CUDACC__
__device__ __forceinline__ int prefix_of(const kivi_score_rules& r, int s, int total) {
    const int p = r.prefix ? r.prefix[s] : 0;
    return p < 0 ? 0 : p < total ? p : total;
}
__device__ __forceinline__ void settle_args(Paged8Attn& a) {
    settle_paged8(a.L, a.b);
    a.q.data = settled(a.q.data); a.k.data = settled(a.k.data); a.v.data = settled(a.v.data);
    a.rules.slopes = settled(a.rules.slopes); a.rules.prefix = settled(a.rules.prefix);
    a.part_o = settled(a.part_o); a.part_ml = settled(a.part_ml); a.notes = settled(a.notes);
}
#endif

}  // namespace kivi
