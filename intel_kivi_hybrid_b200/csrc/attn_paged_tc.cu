// Attention of a step's rows over a paged cache on the 5th-generation tensor cores:
// head_dim 64 and 128, groups of 32 tokens, bf16 rows.
//
//   S = Q K^T,  P = 2^(S c - m),  O = O + P V,  out = O / sum P
//
// over tiles of 128 tokens, for two blocks of 128 rows at a time ((new token, query head)
// pairs of one sequence and KV head: all heads of a group share the tile).  Codes become
// numbers once per tile and serve 256 rows.  A CTA that has one block only gives it to both
// groups of softmax warps, one for the even tiles and one for the odd.  Roles of the 19 warps:
//   0-3, 4-7   a thread per row of the first / second block: running maximum and sum,
//              weights, rescaling, output
//   8-11       K of a tile: codes, scales and zeros (of the window and the new tokens: rows)
//              become fp16 numbers in shared memory, two stages; a warp has a group of tokens
//   12-15      V, likewise
//   16         one thread issues the MMAs: S of a block while the other block's weights
//              are made; P comes from tensor memory, where it takes the place of S
//   17         one thread brings codes, scales and zeros of the tiles to come to shared
//              memory with bulk copies, two tiles ahead (loads into registers half a tile
//              ahead left every second tile waiting for its slowest warp)
//   18         finds the largest factor of the tiles of codes, ahead of those who need it
//
// Operands are fp16 numbers with powers of two taken out: a row of Q and a tile of K by
// their own largest, V by the largest that the CTA has met so far (when it grows, O is
// rescaled as for a new maximum).  The largest is between 2^13 and 2^14, so whatever is
// within 2^-27 of it keeps 11 bits: a window's bf16 numbers are not rounded, weights at 2^-11, a
// group's scales and zeros at 2^-11 too (the same way for its 32 tokens) and what a code stands for
// once more.  Codes count from 1, and z + s stands where z would, since those are smaller than c s and
// z where numbers lie on both sides of 0 (from 0: 389 us where the 512 rows below take 391, and the error
// after this 0.0020).  bf16 operands would round at 2^-8, which is what the output itself is rounded at
// (measured: 0.0018 of the output's 2-norm off 64 bits where its own rounding is 0.0017).
// Sums, maxima and O are fp32.  One power of two for all the tokens of a tile is no good where a row
// does not see, or gives no weight to, a token that is far larger than the others: the rows of a CTA
// that has met a value of 2^16 or more, an infinity or a NaN are computed on the CUDA cores in fp32
// by a launch behind this one (attn_paged.cu; the 512 rows below take 5.7 ms if all are; a fallback
// within this kernel cost every call 8 %).  Below that, other tokens are exact to 2^-22.
//
// Codes to fp16: a 2-bit field and the exponent of 1024 make the number 1024 + c 4^n, of
// which 1024 + 4^n is taken off exactly; (c - 1) 4^n (s / 4^n) + (z + s) is one fused operation
// for two numbers.  3.3 instructions for two elements, where fp32 takes five and a conversion.
//
// Per tile and SM: 2048 cycles of MMA for 256 rows, 2048 of exponentials (16 a cycle); measured
// 5500.  A block's chain is what bounds it: maximum 630-1000, weights 2800 while the other block
// makes its own, then 1400 until P V and the next scores are done.  One block: 4300, of which the
// conversion of a tile takes 2800-3100 (bf16, 32k tokens).
// 512 rows of 4 heads per KV head over 32k tokens, 8 KV heads: 391 us, 708 TFLOP/s; 4 x 2048 over
// 16k 3142 us; 16 x 5 tokens over 4k 76 us; a prompt of 4 x 2048 440 us.  The roles share an
// instruction cache, so bodies are small: with the MMAs of a tile and four tokens of a key quad side
// by side 403 us where this form had 391, 3280 (3246), 90 (78), with the conversions' channels unrolled
// too 423, 3393, 99; but weights by 32 columns 426, 3440 (81) and values a token at a time 394, 3271, 88.
// Lost: two threads to a row that meet for its maximum (406, 3323, 101 with one group of softmax
// warps for one block); scores in halves of 64 tokens,
// so that the next half's are made meanwhile (471, 3753: twice the dependent MMAs in a row);
// maxima of the halves one after the other, without a pass for them (439, 3594: spills).  608 threads
// leave a thread 96 registers (room is given by four warps), too few for the 128 scores of its row, so
// each score is read twice; registers have not been moved from the other roles to the softmax warps.
#include "paged_attention.cuh"
#include "tcgen05.cuh"

#include <cuda_fp16.h>

namespace kivi {
namespace {

__device__ int g_fault = 0;

constexpr int kN = 128;                                  // tokens of a tile
constexpr int kM = 128;                                  // rows of a block
constexpr int kSoftmaxWarps = 8, kTileWarps = 4;        // (four for keys, four for values)
constexpr int kMmaWarp = kSoftmaxWarps + 2 * kTileWarps, kCopyWarp = kMmaWarp + 1, kTopWarp = kMmaWarp + 2, kThreads = (kTopWarp + 1) * 32;
constexpr int kRing = 8;                                 // exponents of so many tiles are kept (they are found up to five tiles ahead of the rows)
constexpr float kGrowth = 8.0f;                          // weights up to 2^8 are let stand before the maximum moves

__device__ __forceinline__ uint32_t hadd2(uint32_t a, uint32_t b) {
    const __half2 r = __hadd2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&c));
    return *reinterpret_cast<const uint32_t*>(&r);
}
constexpr uint32_t k1024 = 0x64006400u, kMinus1024 = 0xe400e400u;        // (neighbours are 1 apart: bits of 1024 + n are 0x6400 + n)

// The power of two that takes a largest magnitude (its bits) to 2^13 .. 2^14, kept where
// it and its inverse are normal numbers; nothing (or infinity) is left as it is.
__device__ __forceinline__ int exponent_of(uint32_t bits) { return (int)(bits >> 23); }
constexpr int kRough = 127 + 16;                         // (biased exponent)
__device__ __forceinline__ int shift_of(int e) {         // biased exponent -> power to multiply with
    if (e == 0 || e == 255) return 0;
    const int s = 127 + 13 - e;
    return s < -110 ? -110 : s > 110 ? 110 : s;
}
__device__ __forceinline__ float pow2i(int s) { return __uint_as_float((uint32_t)(127 + s) << 23); }
template <int D> struct Shared {
    static constexpr int kBlocks = D / 64;               // blocks of 64 channels, 128 bytes a row
    static constexpr uint32_t kTileBytes = kBlocks * kN * 128;
    static constexpr uint32_t q = 0, k = 2 * kTileBytes, v = k + 2 * kTileBytes, raw = v + 2 * kTileBytes;
    // codes, scales and zeros of a tile's K or V as they lie in the pages; K of two tiles, then V
    static constexpr uint32_t kCodes = 32 * D / 4, kFactors = D * 4;            // bytes of a group
    static constexpr uint32_t raw_s = 4 * kCodes, raw_z = raw_s + 4 * kFactors, kRawBytes = raw_z + 4 * kFactors;
    static constexpr uint32_t bars = raw + 4 * kRawBytes;
    static constexpr uint32_t bytes = bars + 2048 + 1024;            // (the tiles start on a boundary of 1024)
};
struct Misc {                                            // behind the tiles
    uint64_t q_full, full[2][2], empty[2][2], s_full[2], p_full[2][2], o_done;       // full, empty: [K, V][stage]
    uint64_t raw_full[2][2], raw_empty[2][2], ready[2][2];
    uint64_t v_known[4];                                 // v_top of tile j, at j % 4
    uint32_t tmem;
    int place[2];
    int k_top[kRing], v_top[kRing];                      // biased exponents of tile j's largest at j % kRing
    int rough;                                           // a value has been met that the tiles' operands are no good for
    uint32_t top[2][2][kTileWarps];                      // [tile parity][K, V][warp]
};

// Bits of the largest magnitude among z and z + 3 s of a group's factors (D of each): what
// codes stand for lies between.
template <int D>
__device__ __forceinline__ uint32_t group_top(uint32_t factors, int lane) {
    uint32_t top = 0u;                                   // (as bits: a NaN is the largest)
    auto bits = [](float x) { return __float_as_uint(fabsf(x)); };
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
        const float2 s = lds_float2(factors + Shared<D>::raw_s + (64 * i + 2 * lane) * 4), z = lds_float2(factors + Shared<D>::raw_z + (64 * i + 2 * lane) * 4);
        top = max(top, max(bits(z.x), bits(fmaf(3.0f, s.x, z.x))));
        top = max(top, max(bits(z.y), bits(fmaf(3.0f, s.y, z.y))));
    }
    return top;
}
// columns from `seen` on count for nothing
__device__ __forceinline__ void hide(uint32_t (&v)[32], int seen) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = i < seen ? v[i] : 0xff800000u;
}
template <int D>
__global__ void __launch_bounds__(kThreads, 1)
paged_attention_tc_kernel(PagedAttnArgs A) {
    constexpr int G = 32;
    using S = Shared<D>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    Misc& misc = *reinterpret_cast<Misc*>(smem + S::bars);
    static_assert(sizeof(Misc) <= 2048, "behind the tiles");
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const uint32_t base = smem_u32(smem);

    stream_order();
    settle_args(A);
    const kivi_paged_layer& L = A.L;
    const int R = L.residual_cap, H = L.num_kv_heads, h = blockIdx.y, n_rep = A.n_rep;
    if (blockIdx.x + blockIdx.y + blockIdx.z == 0) report_left_out(L, A.b, &g_fault);
    // the last blocks of a sequence see most: they start first
    const int item = (int)(gridDim.x - 1 - blockIdx.x);
    if (warp == 0) {
        const ItemPlace p = find_item(item, A.b.num_seqs, [&](int i) {
            PagedSeq q;
            load_seq(L, A.b, i, q);
            return (int)(((int64_t)q.n * n_rep + 2 * kM - 1) / (2 * kM));
        });
        if (lane == 0) { misc.place[0] = p.s; misc.place[1] = p.sub; misc.rough = 0; }
    }
    __syncthreads();
    const int s = misc.place[0];
    if (s >= A.b.num_seqs) return;
    PagedSeq q;
    load_seq(L, A.b, s, q);
    const int rows = q.n * n_rep, row_first = misc.place[1] * 2 * kM;
    const int n_rows = rows - row_first < 2 * kM ? rows - row_first : 2 * kM;
    const int n_sub = n_rows > kM ? 2 : 1;
    // One block of rows: both groups of softmax warps have it, one the even tiles and one the odd, each with
    // scores, weights, sums and output of its own; they are joined at the end.
    const bool turns = n_sub == 1;
    const int inside = min(quant_of(q.held + q.n, G, R), q.held);
    const int keys = q.held + (row_first + n_rows - 1) / n_rep + 1;
    const int t_begin = blockIdx.z * A.chunk;            // (a multiple of kN)
    if (t_begin >= keys) return;
    const int t_end = min(t_begin + A.chunk, keys), n_tiles = (t_end - t_begin + kN - 1) / kN;
    const bool whole = t_end == keys && blockIdx.z == 0;

    auto bar = [&](const uint64_t& b) { return smem_u32(&b); };
    if (warp == kMmaWarp) {
        if (elect_one()) {
            mbar_init(bar(misc.q_full), kM * n_sub);
            for (int i = 0; i < 2; ++i) {
                for (int x = 0; x < 2; ++x) {
                    mbar_init(bar(misc.full[x][i]), kTileWarps); mbar_init(bar(misc.empty[x][i]), 1);
                    mbar_init(bar(misc.ready[x][i]), 1); mbar_init(bar(misc.raw_full[x][i]), 1); mbar_init(bar(misc.raw_empty[x][i]), kTileWarps);
                }
                mbar_init(bar(misc.s_full[i]), 1); mbar_init(bar(misc.p_full[i][0]), kM); mbar_init(bar(misc.p_full[i][1]), kM);
            }
            for (int i = 0; i < 4; ++i) mbar_init(bar(misc.v_known[i]), 1);
            mbar_init(bar(misc.o_done), 1);
            mbar_init_fence();
        }
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&misc.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = misc.tmem;
    // A wait that runs out is reported and ends the block's work: every role comes to the
    // barrier at the end by waits that are bounded, too.
    auto wait = [&](const uint64_t& b, int phase) {
        if (mbar_sleep(bar(b), (uint32_t)phase & 1u)) return true;
        atomicOr(&g_fault, 1);
        return false;
    };
    auto wait_warp = [&](const uint64_t& b, int phase) { return __all_sync(0xffffffffu, wait(b, phase)) != 0; };

    if (warp < kSoftmaxWarps) {
        // ---------------- rows ----------------
        const int t = warp >> 2, r = tid & (kM - 1);
        if (t < n_sub || turns) {
            const int in_cta = (turns ? 0 : t * kM) + r, row = row_first + in_cta;
            const bool there = in_cta < n_rows;
            const int token = there ? row / n_rep : 0, head = h * n_rep + (there ? row % n_rep : 0);
            // the row of Q: its largest to 2^13 .. 2^14
            int q_shift = 0;
            {
                const __nv_bfloat16* from = reinterpret_cast<const __nv_bfloat16*>(A.q.data) + ((int64_t)q.row0 + token) * A.q.row_stride + (int64_t)head * A.q.head_stride;
                uint32_t top = 0u;
                for (int d = 0; there && d < D; d += 8) {
                    uint4 x;
                    if (A.vec) x = *reinterpret_cast<const uint4*>(from + d);
                    else {
                        const uint16_t* u = reinterpret_cast<const uint16_t*>(from + d);
                        x = make_uint4(u[0] | (uint32_t)u[1] << 16, u[2] | (uint32_t)u[3] << 16, u[4] | (uint32_t)u[5] << 16, u[6] | (uint32_t)u[7] << 16);
                    }
                    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {                 // (the largest finite one)
                        const uint32_t lo = (w[i] << 16) & 0x7fffffffu, hi = w[i] & 0x7fff0000u;
                        top = max(top, max(lo < 0x7f800000u ? lo : 0u, hi < 0x7f800000u ? hi : 0u));
                    }
                }
                q_shift = shift_of(exponent_of(top));
                const float f = pow2i(q_shift);
#pragma unroll 1
                for (int d = 0; d < D && t < n_sub; d += 8) {
                    uint32_t w[4] = {0u, 0u, 0u, 0u};
                    if (there) {
                        const uint16_t* u = reinterpret_cast<const uint16_t*>(from + d);
                        uint4 x;
                        if (A.vec) x = *reinterpret_cast<const uint4*>(from + d);
                        else x = make_uint4(u[0] | (uint32_t)u[1] << 16, u[2] | (uint32_t)u[3] << 16, u[4] | (uint32_t)u[5] << 16, u[6] | (uint32_t)u[7] << 16);
                        const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[i] = pack_half(__uint_as_float(y[i] << 16) * f, __uint_as_float(y[i] & 0xffff0000u) * f);
                    }
                    *reinterpret_cast<uint4*>(smem + S::q + t * S::kTileBytes + (d / 64) * (kM * 128) + swizzled(r, (d % 64) / 8)) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            fence_async();
            if (t < n_sub) arrive(bar(misc.q_full));

            const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16, s_at = tmem + lanes + t * kN, o_at = tmem + lanes + 2 * kN + t * D;
            const int last = there ? q.held + token : 0x3fffffff;    // last token that the row sees (a row that is not there is in nobody's way)
            float m = -INFINITY, l = 0.0f;
            int v_shift = 0;
            const float scale = A.scale_log2;
            bool ok = true;
            const int first = turns ? t : 0, step = turns ? 2 : 1;
            for (int j = first; j < n_tiles; j += step) {
                const int turn = turns ? j >> 1 : j;
                // (given up: on to the end without waiting; the groups meet at a barrier there)
                if (ok) ok = wait_warp(misc.s_full[t], turn);
                fence_after();
                const int t0 = t_begin + j * kN;
                const int k_shift = shift_of(misc.k_top[j % kRing]);
                // S is 2^(q_shift + k_shift) times the score
                const float c = fmaxf(scale * pow2i(-q_shift) * pow2i(-k_shift), 1.0e-37f);      // (not 0: hidden columns are -inf)
                const int seen = min(last, t_end - 1) - t0 + 1;      // columns that count
                // (loops of one body: the roles share an instruction cache, unrolled ones cost 15 % of the call)
                float top = -INFINITY;
#pragma unroll 1
                for (int x = 0; x < kN; x += 32) {
                    uint32_t v[32];
                    tmem_load32(s_at + x, v);
                    tmem_wait_load();
                    if (__any_sync(0xffffffffu, seen < x + 32)) hide(v, seen - x);
#pragma unroll
                    for (int i = 0; i < 32; i += 2) top = fmaxf(top, fmaxf(__uint_as_float(v[i]), __uint_as_float(v[i + 1])));
                }
                top *= c;
                // (V of tile j + 2 is not made before this tile's weights are contracted, so the barrier's phase is this tile's)
                if (ok) ok = wait_warp(misc.v_known[j % 4], j >> 2);
                const int v_new = shift_of(misc.v_top[j % kRing]);
                const bool grows = top > m + kGrowth;                // (from -inf: whenever there is a maximum)
                if (__any_sync(0xffffffffu, grows) || (j > first && v_new != v_shift)) {
                    const float m_new = fmaxf(m, top);
                    const float alpha = m == -INFINITY ? 0.0f : ex2(m - m_new);
                    m = m_new;
                    l *= alpha;
                    if (j > first) {
                        const float f = (m == -INFINITY ? 1.0f : alpha) * pow2i(max(v_new - v_shift, -126));
#pragma unroll 1
                        for (int x = 0; x < D; x += 16) {
                            uint32_t o[16];
                            tmem_load16(o_at + x, o);
                            tmem_wait_load();
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            tmem_store16(o_at + x, o);
                        }
                    }
                }
                v_shift = v_new;
                const float base_m = m == -INFINITY ? 0.0f : m;
                float2 sum = make_float2(0.0f, 0.0f);
                // Weights: columns 64 .. 127 become columns 64 .. 95 and are contracted while 0 .. 63 become columns 0 .. 31.
#pragma unroll 1
                for (int half = 1; half >= 0; --half) {
                    const int x = 64 * half;
                    uint32_t v[2][32];
                    tmem_load32(s_at + x, v[0]);
                    tmem_load32(s_at + x + 32, v[1]);
                    tmem_wait_load();
                    if (__any_sync(0xffffffffu, seen < x + 64)) { hide(v[0], seen - x); hide(v[1], seen - x - 32); }
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        uint32_t p[16];
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const float2 e = fma2(make_float2(__uint_as_float(v[k][i]), __uint_as_float(v[k][i + 1])), both(c), both(-base_m));
                            const float2 w = make_float2(ex2(e.x), ex2(e.y));
                            sum = add2(sum, w);
                            p[i / 2] = pack_half(w.x, w.y);
                        }
                        tmem_store16(s_at + x + 16 * k, p);
                    }
                    tmem_wait_store();
                    fence_before();
                    arrive(bar(misc.p_full[t][half]));
                }
                l += sum.x + sum.y;
            }
            if (ok) ok = wait_warp(misc.o_done, 0);
            {
                fence_after();
                const bool rough = *const_cast<volatile int*>(&misc.rough) != 0;         // (computed by another launch, and `out` may be `q`)
                float f = pow2i(-v_shift), other = 0.0f;
                float* const odd_o = reinterpret_cast<float*>(smem + S::k) + r;           // [channel][row]: the odd tiles' output
                if (turns && n_tiles > 1) {
                    float* const odd_ml = reinterpret_cast<float*>(smem + S::q) + r;
                    if (t == 1) {
                        odd_ml[0] = m; odd_ml[kM] = l;
#pragma unroll 1
                        for (int x = 0; x < D; x += 16) {
                            uint32_t o[16];
                            tmem_load16(o_at + x, o);
                            tmem_wait_load();
#pragma unroll
                            for (int i = 0; i < 16; ++i) odd_o[(x + i) * kM] = __uint_as_float(o[i]) * f;
                        }
                    }
                    asm volatile("bar.sync 3, %0;" ::"n"(2 * kM) : "memory");
                    if (t == 0) {
                        const float m_odd = odd_ml[0], m_new = fmaxf(m, m_odd), b = m_new == -INFINITY ? 0.0f : m_new, mine = ex2(m - b);
                        other = ex2(m_odd - b);
                        l = l * mine + odd_ml[kM] * other;
                        f *= mine;
                        m = m_new;
                    }
                }
                const bool writes = there && !rough && t < n_sub;
                const float by = whole ? 1.0f / l : 1.0f;
                const int64_t at = ((int64_t)q.row0 + token) * A.out.row_stride + (int64_t)head * A.out.head_stride;
                const int64_t part = (((int64_t)item * H + h) * A.pieces + blockIdx.z) * (2 * kM) + in_cta;
#pragma unroll 1
                for (int x = 0; x < D; x += 16) {
                    uint32_t o[16];
                    tmem_load16(o_at + x, o);
                    tmem_wait_load();
                    if (!writes) continue;
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        float y_[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            y_[e] = __uint_as_float(o[i + e]) * f;
                            if (turns && n_tiles > 1) y_[e] = fmaf(odd_o[(x + i + e) * kM], other, y_[e]);
                        }
                        const float4 y = make_float4(y_[0] * by, y_[1] * by, y_[2] * by, y_[3] * by);
                        if (whole) store_quad(A.out.data, A.out_dtype, at + x + i, y);
                        else *reinterpret_cast<float4*>(A.part_o + part * D + x + i) = y;
                    }
                }
                if (!whole && writes) *reinterpret_cast<float2*>(A.part_ml + 2 * part) = make_float2(m, l);
                fence_before();
            }
        }
    } else if (warp < kMmaWarp) {
        // ---------------- tiles ----------------
        const bool of_keys = warp < kSoftmaxWarps + kTileWarps;
        const int x_ = of_keys ? 0 : 1, g = (warp - kSoftmaxWarps) & 3;          // group of the tile
        const __nv_bfloat16* const ring = reinterpret_cast<const __nv_bfloat16*>(of_keys ? L.k_res : L.v_res) + ((int64_t)q.slot * H + h) * R * D;
        const kivi_rows& fresh = of_keys ? A.k : A.v;
        const __nv_bfloat16* const rows_new = reinterpret_cast<const __nv_bfloat16*>(fresh.data) + (int64_t)h * fresh.head_stride;
        // Rows as they are (window, new tokens): lane = (16-byte piece of 64 channels, token of four).
        const int p8 = lane & 7, sub = lane >> 3;
        auto row_at = [&](int t) {                                   // token t >= inside
            return t < q.held ? ring + (int64_t)ring_slot(t, A.b.ring_shift, R) * D : rows_new + ((int64_t)q.row0 + t - q.held) * fresh.row_stride;
        };
        auto row8 = [&](int t, int ch) {                             // its eight channels; behind the piece's end zeros
            if (t >= t_end) return make_uint4(0u, 0u, 0u, 0u);
            const __nv_bfloat16* from = row_at(t) + ch;
            if (t < q.held || A.vec) return *reinterpret_cast<const uint4*>(from);
            const uint16_t* u = reinterpret_cast<const uint16_t*>(from);
            return make_uint4(u[0] | (uint32_t)u[1] << 16, u[2] | (uint32_t)u[3] << 16, u[4] | (uint32_t)u[5] << 16, u[6] | (uint32_t)u[7] << 16);
        };
        auto half8 = [&](const uint4& x, float f) {
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
            uint32_t y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = pack_half(__uint_as_float(w[i] << 16) * f, __uint_as_float(w[i] & 0xffff0000u) * f);
            return make_uint4(y[0], y[1], y[2], y[3]);
        };
        auto top8 = [&](const uint4& x) {                            // largest magnitudes of the even and the odd channels, as bf16 bits
            return __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu), __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
        };
        auto place = [&](uint32_t to, int hw, int r) { return to + hw * (kN * 128) + r * 128 + ((p8 ^ (r & 7)) << 4); };

        // Keys of a packed group.  (c, m) = lane & 7: channels 64 hw + 16 c + 8 m .. + 7, which are two
        // words of a token quad 16 bytes apart (kblock_offset); quads jq, jq + 4 with jq = lane >> 3.
        auto convert_keys = [&](uint32_t raw, uint32_t to, float f) {
            const int c = lane & 3, m = lane >> 2 & 1, jq = lane >> 3;
            const uint32_t ch = 16 * c + 8 * m;
#pragma unroll 1
            for (int hw = 0; hw < D / 64; ++hw) {
                uint32_t s2[4], z2[4], x[2][4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t af = raw + g * S::kFactors + (64 * hw + ch + 4 * i) * 4;
                    const float4 sc = lds_float4(af + S::raw_s), ze = lds_float4(af + S::raw_z);
                    const float4 sf = make_float4(sc.x * f, sc.y * f, sc.z * f, sc.w * f);
                    s2[2 * i] = pack_half(sf.x, sf.y); s2[2 * i + 1] = pack_half(sf.z, sf.w);
                    z2[2 * i] = pack_half(fmaf(ze.x, f, sf.x), fmaf(ze.y, f, sf.y)); z2[2 * i + 1] = pack_half(fmaf(ze.z, f, sf.z), fmaf(ze.w, f, sf.w));
                    // bytes of two channels, 16 bits apart
                    const uint32_t at = raw + g * S::kCodes + hw * 512 + (jq + 4 * i) * 64 + 32 * m + 4 * c;
                    const uint32_t a = lds_u32(at), b = lds_u32(at + 16);
                    x[i][0] = __byte_perm(a, 0u, 0x4140); x[i][1] = __byte_perm(a, 0u, 0x4342);
                    x[i][2] = __byte_perm(b, 0u, 0x4140); x[i][3] = __byte_perm(b, 0u, 0x4342);
                }
                uint32_t one = kMinus1024 + 0x00010001u, mask = 0x00030003u;        // -(1024 + 4^n), and the codes' places
#pragma unroll 1
                for (int n = 0; n < 4; ++n, one = 4u * one - 3u * kMinus1024, mask <<= 2) {
                    const uint32_t turn = to + (4 * jq + n) * 128 + (((2 * c + m) ^ ((4 * jq + n) & 7)) << 4);      // piece of the row, swizzled
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t y[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[e] = hfma2(hadd2((x[i][e] & mask) | k1024, one), s2[e], z2[e]);
                        sts128(turn + hw * (kN * 128) + i * (16 * 128), y[0], y[1], y[2], y[3]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) s2[e] = hmul2(s2[e], 0x34003400u);        // a quarter
                }
            }
        };
        // Values of a packed group.  r = lane & 3, vg = lane >> 2 & 1: channels 64 p + 32 vg + 8 r .. + 7;
        // tokens 16 kap + 4 c + n with c = lane >> 3.  D = 128: word (gd, kap, r, c) of the codes holds the
        // four tokens n in its bytes (kivi_common.cuh); D = 64: 16 bytes a token.
        auto convert_values = [&](uint32_t raw, uint32_t to, float f) {
            const int r = lane & 3, vg = lane >> 2 & 1, c = lane >> 3;
            const uint32_t piece = (4 * vg + r) ^ (4 * (c & 1));
#pragma unroll 1
            for (int pk = 0; pk < 2 * (D / 64); ++pk) {
                const int p = pk >> 1, kap = pk & 1;
                uint32_t w[2];
                if constexpr (D == 128) {
                    const uint32_t at = raw + g * S::kCodes + ((2 * p + vg) * 64 + 32 * kap + 8 * r + c) * 4;
                    w[0] = lds_u32(at); w[1] = lds_u32(at + 16);
                } else {
                    w[0] = w[1] = 0u;
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const uint32_t b = lds_u16(raw + g * S::kCodes + (16 * kap + 4 * c + n) * 16 + 8 * vg + 2 * r);
                        w[0] |= (b & 255u) << (8 * n); w[1] |= (b >> 8) << (8 * n);
                    }
                }
                // factors of tokens 16 kap + 4 c + n: rows 4 n + c (kivi_common.cuh), or as they come
                const uint32_t at = raw + g * S::kFactors + (D == 128 ? (16 * kap + c) * 16 + (2 * p + vg) * 4 : (16 * kap + 4 * c) * 8 + vg * 4);
                const uint32_t out = to + p * (kN * 128) + (4 * c + 16 * kap) * 128;
                float sc[4], ze[4];
#pragma unroll
                for (int n = 0; n < 4; ++n) { sc[n] = lds_float(at + S::raw_s + n * (D == 128 ? 64 : 8)); ze[n] = lds_float(at + S::raw_z + n * (D == 128 ? 64 : 8)); }
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const float s1 = sc[n] * f, z1 = fmaf(ze[n], f, s1);
                    const uint32_t s_lo = pack_half(s1, 0.25f * s1), s_hi = hmul2(s_lo, 0x2c002c00u) /* a sixteenth */, z = pack_half(z1, z1);
                    uint32_t y[4];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t b = __byte_perm(w[e], 0u, 0x4040 + 0x0101 * n);      // byte n in both halves
                        y[2 * e] = hfma2(hadd2((b & 0x000c0003u) | k1024, kMinus1024 + 0x00040001u), s_lo, z);
                        y[2 * e + 1] = hfma2(hadd2((b & 0x00c00030u) | k1024, kMinus1024 + 0x00400010u), s_hi, z);
                    }
                    sts128(out + n * 128 + ((piece ^ n) << 4), y[0], y[1], y[2], y[3]);
                }
            }
        };

        int v_top = 0;                                               // biased exponent of the largest value so far
        bool ok = true;
#pragma unroll 1
        for (int j = 0; j < n_tiles; ++j) {
            const int tile0 = t_begin + j * kN, t0 = tile0 + G * g, st = j & 1;
            const bool packed = t0 < inside;                         // (a group with any token in pages has all 32 there)
            const uint32_t raw = base + S::raw + (2 * x_ + st) * S::kRawBytes;
            const uint32_t to = base + (of_keys ? S::k : S::v) + st * S::kTileBytes + (uint32_t)(G * g) * 128u;
            // (given up: on to the end without waiting, the other warps wait at the barrier below)
            int e_top;
            if (tile0 + kN - G < inside) {                           // four packed groups: the power of two is known
                if (ok) ok = wait_warp(misc.ready[x_][st], j >> 1);
                e_top = (of_keys ? misc.k_top : misc.v_top)[j % kRing];
                if (ok && j >= 2) ok = wait_warp(misc.empty[x_][st], (j >> 1) - 1);
            } else {
                // rows go to their place as they are, which finds the largest, and are converted there
                if (ok && j >= 2) ok = wait_warp(misc.empty[x_][st], (j >> 1) - 1);
                uint32_t top = 0u;
                if (packed) {
                    if (ok) ok = wait_warp(misc.raw_full[x_][st], j >> 1);
                    top = group_top<D>(raw + g * S::kFactors, lane);
                } else {
                    uint32_t pair = 0u;
                    // All of a lane's copies are on their way at once, and it reads them back itself (loads of four
                    // through registers: 4 x 2048 tokens of a prompt 521 us, of eight 463, so 440).
#pragma unroll 1
                    for (int i = 0; i < 8 * (D / 64); ++i) {
                        const int r = sub + 4 * (i & 7), t = t0 + r, ch = 64 * (i >> 3) + 8 * p8;
                        const uint32_t at = place(to, i >> 3, r);
                        if (t >= q.held && !A.vec) {
                            const uint4 x = row8(t, ch);
                            sts128(at, x.x, x.y, x.z, x.w);
                        } else {
                            copy16(at, row_at(min(t, t_end - 1)) + ch, t < t_end);
                        }
                    }
                    copies_wait();
#pragma unroll 1
                    for (int i = 0; i < 8 * (D / 64); i += 4) {
                        uint4 x[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = lds_uint4(place(to, i >> 3, sub + 4 * ((i + e) & 7)));
#pragma unroll
                        for (int e = 0; e < 4; ++e) pair = __vmaxu2(pair, top8(x[e]));
                    }
                    top = max(pair << 16, pair & 0xffff0000u);
                }
                top = __reduce_max_sync(0xffffffffu, top);
                if (lane == 0) misc.top[st][x_][g] = top;
                asm volatile("bar.sync %0, %1;" ::"r"(1 + x_), "n"(32 * kTileWarps) : "memory");
                e_top = exponent_of(__reduce_max_sync(0xffffffffu, misc.top[st][x_][lane & 3]));
                if (!of_keys) e_top = max(e_top, v_top);
                if (g == 0 && lane == 0) {
                    (of_keys ? misc.k_top : misc.v_top)[j % kRing] = e_top;
                    if (e_top >= kRough) misc.rough = 1;
                    if (!of_keys) arrive(bar(misc.v_known[j % 4]));
                }
            }
            v_top = e_top;
            const float f = pow2i(shift_of(e_top));
            if (packed) {
                if (of_keys) convert_keys(raw, to, f);
                else convert_values(raw, to, f);
                if (t0 + G > inside) {
                    // the step's own tokens of this group are served as they are, not from the page
                    __syncwarp();
#pragma unroll 1
                    for (int i = 0; i < 8 * (D / 64); ++i) {
                        const int r = sub + 4 * (i & 7);
                        if (t0 + r < inside) continue;
                        uint4 x = row8(t0 + r, 64 * (i >> 3) + 8 * p8);
                        const uint32_t pair = top8(x);               // (what the page stands for is as large, or the rows are not those appended)
                        if (exponent_of(max(pair << 16, pair & 0xffff0000u)) > e_top + 1) misc.rough = 1;
                        x = half8(x, f);
                        sts128(place(to, i >> 3, r), x.x, x.y, x.z, x.w);
                    }
                }
            } else {
#pragma unroll 1
                for (int i = 0; i < 2 * (D / 64); ++i) {
                    uint4 x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = lds_uint4(place(to, i >> 1, sub + 4 * (4 * (i & 1) + e)));
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[e] = half8(x[e], f);
                        sts128(place(to, i >> 1, sub + 4 * (4 * (i & 1) + e)), x[e].x, x[e].y, x[e].z, x[e].w);
                    }
                }
            }
            fence_async();
            __syncwarp();
            if (lane == 0) {
                arrive(bar(misc.raw_empty[x_][st]));
                arrive(bar(misc.full[x_][st]));
            }
        }
    } else if (warp == kTopWarp) {
        // ---------------- the largest of a tile of codes ----------------
        uint32_t v_top = 0u;
        bool ok = true;
#pragma unroll 1
        for (int j = 0; j < n_tiles && t_begin + j * kN + kN - G < inside; ++j) {
#pragma unroll 1
            for (int x = 0; x < 2; ++x) {
                if (ok) ok = wait_warp(misc.raw_full[x][j & 1], j >> 1);
                uint32_t top = 0u;
                const uint32_t raw = base + S::raw + (2 * x + (j & 1)) * S::kRawBytes;
#pragma unroll
                for (int i = 0; i < kN / G; ++i) top = max(top, group_top<D>(raw + i * S::kFactors, lane));
                top = __reduce_max_sync(0xffffffffu, top);
                if (x) top = v_top = max(v_top, top);
                if (lane == 0) {
                    (x ? misc.v_top : misc.k_top)[j % kRing] = exponent_of(top);
                    if (exponent_of(top) >= kRough) misc.rough = 1;
                    arrive(bar(misc.ready[x][j & 1]));
                    if (x) arrive(bar(misc.v_known[j % 4]));
                }
            }
        }
    } else if (warp == kCopyWarp) {
        // ---------------- copies ----------------
        if (elect_one()) {
            const uint64_t policy = l2_stream_policy();
            const int gpp = L.page_tokens / G;
            int page = t_begin / L.page_tokens, group = t_begin % L.page_tokens / G;
            bool ok = true;
            int sent = 0;
            for (int j = 0; ok && j < n_tiles; ++j) {
                const int t0 = t_begin + j * kN, st = j & 1;
                const int n = min(max((inside - t0 + G - 1) / G, 0), kN / G);        // groups of the tile with a token in pages
                if (n == 0) break;
                int next_page = page, next_group = group;
                for (int x = 0; ok && x < 2; ++x) {                          // (keys do not wait for the values' buffer)
                    if (j >= 2 && !wait(misc.raw_empty[x][st], (j >> 1) - 1)) { ok = false; break; }
                    const uint32_t to = base + S::raw + (2 * x + st) * S::kRawBytes, b = bar(misc.raw_full[x][st]);
                    mbar_expect_tx(b, n * (S::kCodes + 2 * S::kFactors));
                    next_page = page; next_group = group;
                    for (int i = 0; i < n;) {                                // runs of groups that lie in one page
                        const int id = q.pages[next_page], run = min(n - i, gpp - next_group);
                        const bool there = (unsigned)id < (unsigned)L.num_pages;
                        if (!there) atomicOr(&g_fault, kPagedFault);
                        const int64_t at = ((int64_t)(there ? id : 0) * H + h) * gpp + next_group;
                        bulk_g2s(to + i * S::kCodes, (x ? L.v_codes : L.k_codes) + at * S::kCodes, run * S::kCodes, b, policy);
                        bulk_g2s(to + S::raw_s + i * S::kFactors, (x ? L.v_scales : L.k_scales) + at * D, run * S::kFactors, b, policy);
                        bulk_g2s(to + S::raw_z + i * S::kFactors, (x ? L.v_zeros : L.k_zeros) + at * D, run * S::kFactors, b, policy);
                        i += run;
                        next_group += run;
                        if (next_group == gpp) { next_group = 0; ++next_page; }
                    }
                }
                page = next_page; group = next_group;
                if (ok) sent = j + 1;
            }
            // no copy is under way when the block ends
            for (int j = max(sent - 2, 0); j < sent; ++j) { wait(misc.raw_full[0][j & 1], j >> 1); wait(misc.raw_full[1][j & 1], j >> 1); }
        }
    } else if (elect_one()) {
        // ---------------- MMAs ----------------
        constexpr uint32_t kQK = mma_shape(kM, kN, false), kPV = mma_shape(kM, D, true);
        auto scores = [&](int t, int st) {
            const uint32_t rows_at = base + S::q + (turns ? 0 : t) * S::kTileBytes;
#pragma unroll 1
            for (int i = 0; i < D / 16; ++i) {
                const uint32_t off = (uint32_t)(i / 4) * (kM * 128) + (i % 4) * 32;
                mma_ss(tmem + t * kN, smem_desc(rows_at + off, 16, 1024), smem_desc(base + S::k + st * S::kTileBytes + off, 16, 1024), kQK, i > 0);
            }
            mma_commit(bar(misc.s_full[t]));
        };
        // weights of block t in turn n times values of stage st
        auto contract = [&](int t, int st, int n) {
            for (int half = 1; half >= 0; --half) {
                if (!wait(misc.p_full[t][half], n)) return false;
                fence_after();
#pragma unroll 1
                for (int i = 0; i < kN / 32; ++i)
                    mma_ts(tmem + 2 * kN + t * D, tmem + t * kN + 64 * half + 8 * i, smem_desc(base + S::v + st * S::kTileBytes + (4 * half + i) * 2048, kN * 128, 1024), kPV,
                           n > 0 || half == 0 || i > 0);
            }
            return true;
        };
        bool ok = wait(misc.q_full, 0);
        if (turns) {
            // tile j is block j % 2's, in stage j % 2: scores of the next tile are there before this one's weights are
            for (int j = 0; ok && j < n_tiles + 2; ++j) {
                const int t = j & 1;
                if (j >= 2) {
                    ok = wait(misc.full[1][t], (j - 2) >> 1) && contract(t, t, (j - 2) >> 1);
                    if (!ok) break;
                    mma_commit(bar(misc.empty[1][t]));
                }
                if (j < n_tiles) {
                    ok = wait(misc.full[0][t], j >> 1);
                    if (!ok) break;
                    fence_after();
                    scores(t, t);
                    mma_commit(bar(misc.empty[0][t]));
                }
            }
            if (ok) mma_commit(bar(misc.o_done));
            ok = false;                                  // (done)
        }
        ok = ok && wait(misc.full[0][0], 0);
        if (ok) {
            fence_after();
            for (int t = 0; t < n_sub; ++t) scores(t, 0);
            mma_commit(bar(misc.empty[0][0]));
            for (int j = 0; ok && j < n_tiles; ++j) {
                const int st = j & 1;
                const bool more = j + 1 < n_tiles;
                if (!wait(misc.full[1][st], j >> 1)) { ok = false; break; }
                for (int t = 0; t < n_sub; ++t) {
                    ok = contract(t, st, j);
                    if (t == 0 && more && ok) ok = wait(misc.full[0][st ^ 1], (j + 1) >> 1);
                    if (!ok) break;
                    if (more) scores(t, st ^ 1);
                }
                if (!ok) break;
                mma_commit(bar(misc.empty[1][st]));
                if (more) mma_commit(bar(misc.empty[0][st ^ 1]));
            }
            if (ok) mma_commit(bar(misc.o_done));
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    if (tid == 0) A.rough[((int64_t)item * H + h) * A.pieces + blockIdx.z] = misc.rough;
}

}  // namespace

// Whatever the decode kernel does not take.  head_dim 64, few rows, here and with eight rows a CTA on the CUDA
// cores: 1 x 712 tokens, 12 heads 25.6 and 24.6 us; 8 x 4 heads, one token over 1 x 4k 33 and 57, 1 x 32k 51 and
// 104, 16 x 4k 68 and 158, 64 x 2k 154 and 311, 64 x 8k 423 and 1169; two tokens over 1 x 4k 33 and 45.
bool paged_tc_serves(const kivi_paged_layer* L, int q_dtype) {
    return (L->head_dim == 128 || L->head_dim == 64) && L->group_size == 32 && L->res_dtype == KIVI_BF16 && q_dtype == KIVI_BF16;
}

int run_paged_tc(const PagedAttnArgs& a, int blocks, cudaStream_t st) {
    auto go = [&](auto* kernel, uint32_t smem) {
        KIVI_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        KIVI_CUDA_OK(launch(kernel, dim3((unsigned)blocks, (unsigned)a.L.num_kv_heads, (unsigned)a.pieces), kThreads, smem, st, true, a));
        return KIVI_OK;
    };
    return a.L.head_dim == 128 ? go(paged_attention_tc_kernel<128>, Shared<128>::bytes) : go(paged_attention_tc_kernel<64>, Shared<64>::bytes);
}

int paged_tc_fault_word(int* out) {
    KIVI_CUDA_OK(cudaMemcpyFromSymbol(out, g_fault, sizeof(int)));
    return KIVI_OK;
}
int paged_tc_fault_clear() {
    const int zero = 0;
    KIVI_CUDA_OK(cudaMemcpyToSymbol(g_fault, &zero, sizeof(int)));
    return KIVI_OK;
}

}  // namespace kivi
