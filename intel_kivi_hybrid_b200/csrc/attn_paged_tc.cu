// Attention of a step's rows over a paged cache on the 5th-generation tensor cores:
// head_dim 64 and 128, groups of 32 tokens, bf16 rows.
//
//   S = Q K^T,  P = 2^(S c - m),  O = O + P V,  out = O / sum P
//
// over tiles of 128 tokens, for two blocks of 128 rows at a time ((new token, query head)
// pairs of one sequence and KV head: all heads of a group share the tile).  Codes become
// numbers once per tile and serve 256 rows.  Roles of the 17 warps:
//   0-3, 4-7   one thread per row of the first / second block: running maximum and sum,
//              weights, rescaling, output
//   8-15       fetch codes, scales and zeros (window and new tokens: rows) and write the
//              tile's K and V to shared memory, two stages each
//   16         one thread issues the MMAs: S of a block while the other block's weights
//              are made; P comes from tensor memory, where it takes the place of S
//
// Operands are fp16 numbers with powers of two taken out: a row of Q and a tile of K by
// their own largest, V by the largest that the CTA has met so far (when it grows, O is
// rescaled as for a new maximum).  The largest is between 2^13 and 2^14, so whatever is
// within 2^-27 of it keeps 11 bits: the dequantized numbers and the weights are rounded at
// 2^-12, a window's bf16 numbers not at all.  bf16 operands would round at 2^-9, which is what the
// output itself is rounded at (measured: error 1.0 of the output's own rounding, not 2).
// Sums, maxima and O are fp32.  A row that sees a value that is not finite comes out as NaN; one
// that does not see it is not touched by it.
//
// Codes to fp16: a 2-bit field and the exponent of 1024 make the number 1024 + c 4^n, of
// which 1024 is taken off exactly; c 4^n (s / 4^n) + z is one fused operation for two
// numbers.  3.3 instructions for two elements, where fp32 takes five and a conversion.
//
// Per tile and SM: 2048 cycles of MMA for 256 rows, 2048 of exponentials (16 a cycle),
// about 500 issue cycles of conversion and 800 of softmax arithmetic on each quarter.
#include "async_copy.cuh"
#include "paged_attention.cuh"

#include <cuda_fp16.h>

namespace kivi {
namespace {

__device__ int g_fault = 0;

constexpr int kN = 128;                                  // tokens of a tile
constexpr int kM = 128;                                  // rows of a block
constexpr int kSoftmaxWarps = 8, kProducerWarps = 8, kThreads = (kSoftmaxWarps + kProducerWarps + 1) * 32;
constexpr int kProducers = kProducerWarps * 32;
constexpr int kRing = 4;                                 // factors of so many tiles are kept
constexpr float kGrowth = 8.0f;                          // weights up to 2^8 are let stand before the maximum moves

// ---- tensor core ----------------------------------------------------------------
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead_bytes, uint32_t stride_bytes) {
    return (uint64_t)((addr & 0x3ffffu) >> 4) | (uint64_t)((lead_bytes >> 4) & 0x3fffu) << 16 | (uint64_t)((stride_bytes >> 4) & 0x3fffu) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;        // 128-byte swizzle
}
__host__ __device__ constexpr uint32_t mma_shape(int m, int n, bool b_by_columns) {
    return 1u << 4 /* fp32 sums */ | (b_by_columns ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;      // (fp16 operands: 0)
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(shape), "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t shape, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(shape), "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

#define R8(a, i) "=r"(a[i]), "=r"(a[i + 1]), "=r"(a[i + 2]), "=r"(a[i + 3]), "=r"(a[i + 4]), "=r"(a[i + 5]), "=r"(a[i + 6]), "=r"(a[i + 7])
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : R8(r, 0), R8(r, 8), R8(r, 16), R8(r, 24) : "r"(addr) : "memory");
}
#undef R8
#define R8(a, i) "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3]), "r"(a[i + 4]), "r"(a[i + 5]), "r"(a[i + 6]), "r"(a[i + 7])
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(addr), R8(r, 0), R8(r, 8), R8(r, 16), R8(r, 24) : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(addr), R8(r, 0), R8(r, 8) : "memory");
}
#undef R8
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    uint32_t y;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
    return y;
}
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
constexpr uint32_t k1024 = 0x64006400u, kMinus1024 = 0xe400e400u;

// The power of two that takes a largest magnitude (its bits) to 2^13 .. 2^14, kept where
// it and its inverse are normal numbers; nothing (or infinity) is left as it is.
__device__ __forceinline__ int exponent_of(uint32_t bits) { return (int)(bits >> 23); }
__device__ __forceinline__ int shift_of(int e) {         // biased exponent -> power to multiply with
    if (e == 0 || e == 255) return 0;
    const int s = 127 + 13 - e;
    return s < -110 ? -110 : s > 110 ? 110 : s;
}
__device__ __forceinline__ float pow2i(int s) { return __uint_as_float((uint32_t)(127 + s) << 23); }
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// of finite numbers only
__device__ __forceinline__ uint32_t finite_magnitude(float x) { const uint32_t b = magnitude(x); return b < 0x7f800000u ? b : 0u; }

template <int D> struct Shared {
    static constexpr int kBlocks = D / 64;               // blocks of 64 channels, 128 bytes a row
    static constexpr uint32_t kTileBytes = kBlocks * kN * 128;
    static constexpr uint32_t q = 0, k = 2 * kTileBytes, v = k + 2 * kTileBytes, bars = v + 2 * kTileBytes;
    static constexpr uint32_t bytes = bars + 1024 + 1024;            // (the tiles start on a boundary of 1024)
};
// byte of (row, 16-byte piece of a 128-byte row) of a block with the 128-byte swizzle
__device__ __forceinline__ uint32_t swizzled(int row, int piece) { return (uint32_t)row * 128u + (uint32_t)((piece ^ (row & 7)) << 4); }

struct Misc {                                            // behind the tiles
    uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_done;
    uint32_t tmem;
    int place[2];
    int k_shift[kRing], v_shift[kRing];                  // of tile j at j % kRing
    uint32_t odd[kRing][4];                              // tokens of the tile whose values are not all finite
    uint32_t top[2][2][kProducerWarps];                  // [tile parity][K, V][warp]
};

// What a producer thread holds of a packed group of 32 tokens on its way to shared memory.
// Keys: (c, m) = lane & 7, token quads 2*jq, 2*jq+1 with jq = lane >> 3; the warp has the
// group and the block of 64 channels: channels 64*hw + 16*c + 8*m .. +7.
// Values: r2 = lane & 3, gd & 1 = lane >> 2 & 1, c = lane >> 3; the warp has the group and gd >> 1:
// channels 32*gd + 8*r2 .. +7 of tokens 16*kap + 4*c + n.
struct RawK { uint32_t w[4]; float4 s[2], z[2]; };
struct RawV { uint32_t w[2][2]; float s[2][4], z[2][4]; };

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
paged_attention_tc_kernel(PagedAttnArgs A) {
    constexpr int G = 32;
    using S = Shared<D>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    Misc& misc = *reinterpret_cast<Misc*>(smem + S::bars);
    static_assert(sizeof(Misc) <= 1024, "behind the tiles");
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
        if (lane == 0) { misc.place[0] = p.s; misc.place[1] = p.sub; }
    }
    __syncthreads();
    const int s = misc.place[0];
    if (s >= A.b.num_seqs) return;
    PagedSeq q;
    load_seq(L, A.b, s, q);
    const int rows = q.n * n_rep, row_first = misc.place[1] * 2 * kM;
    const int n_rows = rows - row_first < 2 * kM ? rows - row_first : 2 * kM;
    const int n_sub = n_rows > kM ? 2 : 1;
    const int inside = min(quant_of(q.held + q.n, G, R), q.held);
    const int keys = q.held + (row_first + n_rows - 1) / n_rep + 1;
    const int t_begin = blockIdx.z * A.chunk;            // (a multiple of kN)
    if (t_begin >= keys) return;
    const int t_end = min(t_begin + A.chunk, keys), n_tiles = (t_end - t_begin + kN - 1) / kN;
    const bool whole = t_end == keys && blockIdx.z == 0;

    auto bar = [&](const uint64_t& b) { return smem_u32(&b); };
    if (warp == 16) {
        if (elect_one()) {
            mbar_init(bar(misc.q_full), kM * n_sub);
            for (int i = 0; i < 2; ++i) {
                mbar_init(bar(misc.k_full[i]), kProducerWarps); mbar_init(bar(misc.k_empty[i]), 1);
                mbar_init(bar(misc.v_full[i]), kProducerWarps); mbar_init(bar(misc.v_empty[i]), 1);
                mbar_init(bar(misc.s_full[i]), 1); mbar_init(bar(misc.p_full[i]), kM);
            }
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
        if (mbar_wait(bar(b), (uint32_t)phase & 1u)) return true;
        atomicOr(&g_fault, 1);
        return false;
    };
    auto wait_warp = [&](const uint64_t& b, int phase) { return __all_sync(0xffffffffu, wait(b, phase)) != 0; };

    if (warp < kSoftmaxWarps) {
        // ---------------- rows ----------------
        const int t = warp >> 2, r = tid & (kM - 1);
        if (t < n_sub) {
            const int row = row_first + t * kM + r;
            const bool there = t * kM + r < n_rows;
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
                    for (int i = 0; i < 4; ++i) top = max(top, max(finite_magnitude(__uint_as_float(w[i] << 16)), finite_magnitude(__uint_as_float(w[i] & 0xffff0000u))));
                }
                q_shift = shift_of(exponent_of(top));
                const float f = pow2i(q_shift);
#pragma unroll
                for (int d = 0; d < D; d += 8) {
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
            arrive(bar(misc.q_full));

            const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16, s_at = tmem + lanes + t * kN, o_at = tmem + lanes + 2 * kN + t * D;
            const int last = there ? q.held + token : -1;            // last token that the row sees
            float m = -INFINITY, l = 0.0f;
            int v_shift = 0;
            const float scale = A.scale_log2;
            bool ok = true;
            for (int j = 0; j < n_tiles; ++j) {
                if (!wait_warp(misc.s_full[t], j)) { ok = false; break; }
                fence_after();
                const int t0 = t_begin + j * kN;
                const int k_shift = misc.k_shift[j % kRing], v_new = misc.v_shift[j % kRing];
                // S is 2^(q_shift + k_shift) times the score
                const float c = scale * pow2i(-q_shift) * pow2i(-k_shift);
                const int seen = min(last, t_end - 1) - t0 + 1;      // columns that count
                float top = -INFINITY;
#pragma unroll 1
                for (int x = 0; x < kN; x += 32) {
                    uint32_t v[32];
                    tmem_load32(s_at + x, v);
                    tmem_wait_load();
                    if (__all_sync(0xffffffffu, seen >= x + 32)) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) top = fmaxf(top, __uint_as_float(v[i]));
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) top = fmaxf(top, x + i < seen ? __uint_as_float(v[i]) : -INFINITY);
                    }
                }
                top *= c;
                const bool grows = top > m + kGrowth;                // (from -inf: whenever there is a maximum)
                if (__any_sync(0xffffffffu, grows) || (j > 0 && v_new != v_shift)) {
                    const float m_new = fmaxf(m, top);
                    const float alpha = m == -INFINITY ? 0.0f : ex2(m - m_new);
                    m = m_new;
                    l *= alpha;
                    if (j > 0) {
                        const float f = (m == -INFINITY ? 1.0f : alpha) * pow2i(max(v_new - v_shift, -126));
#pragma unroll 1
                        for (int x = 0; x < D; x += 32) {
                            uint32_t v[32];
                            tmem_load32(o_at + x, v);
                            tmem_wait_load();
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
                            tmem_store32(o_at + x, v);
                        }
                    }
                }
                v_shift = v_new;
                if (t0 + kN > inside) {                              // a tile that holds rows as they are
                    const uint32_t* odd = misc.odd[j % kRing];
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const int in_word = min(max(seen - 32 * w, 0), 32);
                        if (odd[w] & (in_word >= 32 ? 0xffffffffu : (1u << in_word) - 1u)) l = __uint_as_float(0x7fc00000u);
                    }
                }
                const float base_m = m == -INFINITY ? 0.0f : m;
#pragma unroll 1
                for (int x = 0; x < kN; x += 32) {
                    uint32_t v[32], p[16];
                    tmem_load32(s_at + x, v);
                    tmem_wait_load();
                    const bool all = __all_sync(0xffffffffu, seen >= x + 32);
                    float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        float a = ex2(fmaf(__uint_as_float(v[i]), c, -base_m)), b = ex2(fmaf(__uint_as_float(v[i + 1]), c, -base_m));
                        if (!all) {
                            a = x + i < seen ? a : 0.0f;
                            b = x + i + 1 < seen ? b : 0.0f;
                        }
                        sum0 += a; sum1 += b;
                        p[i / 2] = pack_half(a, b);
                    }
                    l += sum0 + sum1;
                    tmem_store16(s_at + x / 2, p);                   // over columns that have been read
                }
                tmem_wait_store();
                fence_before();
                arrive(bar(misc.p_full[t]));
            }
            if (ok && wait_warp(misc.o_done, 0)) {
                fence_after();
                const float f = pow2i(-v_shift);
                const float by = whole ? f / l : f;
                const int64_t at = ((int64_t)q.row0 + token) * A.out.row_stride + (int64_t)head * A.out.head_stride;
                const int64_t part = (((int64_t)item * H + h) * A.pieces + blockIdx.z) * (2 * kM) + t * kM + r;
#pragma unroll 1
                for (int x = 0; x < D; x += 32) {
                    uint32_t v[32];
                    tmem_load32(o_at + x, v);
                    tmem_wait_load();
                    if (!there) continue;
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 o = make_float4(__uint_as_float(v[i]) * by, __uint_as_float(v[i + 1]) * by, __uint_as_float(v[i + 2]) * by, __uint_as_float(v[i + 3]) * by);
                        if (whole) store_quad(A.out.data, A.out_dtype, at + x + i, o);
                        else *reinterpret_cast<float4*>(A.part_o + part * D + x + i) = o;
                    }
                }
                if (!whole && there) *reinterpret_cast<float2*>(A.part_ml + 2 * part) = make_float2(m, l);
                fence_before();
            }
        }
    } else if (warp < kSoftmaxWarps + kProducerWarps) {
        // ---------------- tiles ----------------
        const int pw = warp - kSoftmaxWarps;
        const int g = pw >> 1;                                       // group of the tile: two warps each
        const int part = pw & 1;                                     // D = 128: block of 64 channels; D = 64: half of the token quads
        const int kc = lane & 3, km = lane >> 2 & 1, jq = lane >> 3;
        const int k_ch = (D == 128 ? 64 * part : 0) + 16 * kc + 8 * km;                      // keys: first of 8 channels
        const int k_j0 = D == 128 ? 2 * jq : jq + 4 * part;          // token quads k_j0 .. of the group
        const int vr = lane & 3, vg = lane >> 2 & 1, vc = lane >> 3;
        const int v_gd = (D == 128 ? 2 * part : 0) + vg, v_ch = 32 * v_gd + 8 * vr;          // values
        const int64_t groups_per_page = L.page_tokens / G;
        const __nv_bfloat16* const k_ring = reinterpret_cast<const __nv_bfloat16*>(L.k_res) + ((int64_t)q.slot * H + h) * R * D;
        const __nv_bfloat16* const v_ring = reinterpret_cast<const __nv_bfloat16*>(L.v_res) + ((int64_t)q.slot * H + h) * R * D;
        const __nv_bfloat16* const k_new = reinterpret_cast<const __nv_bfloat16*>(A.k.data) + (int64_t)h * A.k.head_stride;
        const __nv_bfloat16* const v_new = reinterpret_cast<const __nv_bfloat16*>(A.v.data) + (int64_t)h * A.v.head_stride;
        auto group_at = [&](int t) { return ((int64_t)page_of(L, q, t, &g_fault) * H + h) * groups_per_page + t % L.page_tokens / G; };
        auto packed = [&](int t0) { return t0 + G <= inside && t0 < t_end; };

        RawK rk;
        RawV rv;
        auto fetch_k = [&](int64_t at) {
            const uint8_t* codes = L.k_codes + at * (D * G / 4) + (D == 128 ? part * 512 : 0) + 32 * km + 4 * kc;
#pragma unroll
            for (int i = 0; i < (D == 128 ? 2 : 1); ++i) {
                rk.w[2 * i] = __ldg(reinterpret_cast<const uint32_t*>(codes + (k_j0 + i) * 64));
                rk.w[2 * i + 1] = __ldg(reinterpret_cast<const uint32_t*>(codes + (k_j0 + i) * 64 + 16));
            }
            const float* s = L.k_scales + at * D + k_ch;
            const float* z = L.k_zeros + at * D + k_ch;
#pragma unroll
            for (int i = 0; i < 2; ++i) { rk.s[i] = __ldg(reinterpret_cast<const float4*>(s) + i); rk.z[i] = __ldg(reinterpret_cast<const float4*>(z) + i); }
        };
        // values of D = 128: word (gd, kap, r, c) holds tokens 16 kap + 4 c + n in its bytes; D = 64: rows of 16 bytes a token
        auto fetch_v = [&](int64_t at) {
            if constexpr (D == 128) {
                const uint32_t* codes = reinterpret_cast<const uint32_t*>(L.v_codes + at * 1024) + v_gd * 64 + 8 * vr + vc;
#pragma unroll
                for (int kap = 0; kap < 2; ++kap) {
                    rv.w[kap][0] = __ldg(codes + 32 * kap); rv.w[kap][1] = __ldg(codes + 32 * kap + 4);
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const int64_t f = at * 128 + (16 * kap + 4 * n + vc) * 4 + v_gd;
                        rv.s[kap][n] = __ldg(L.v_scales + f); rv.z[kap][n] = __ldg(L.v_zeros + f);
                    }
                }
            } else {                                                 // tokens 16 part + 4 vc + n, 16 bits of the row each
                uint32_t b[4];
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const int tok = 16 * part + 4 * vc + n;
                    b[n] = __ldg(reinterpret_cast<const uint16_t*>(L.v_codes + at * 512 + tok * 16) + 4 * vg + vr);
                    rv.s[0][n] = __ldg(L.v_scales + at * 64 + tok * 2 + v_gd); rv.z[0][n] = __ldg(L.v_zeros + at * 64 + tok * 2 + v_gd);
                }
                rv.w[0][0] = (b[0] & 255u) | (b[1] & 255u) << 8 | (b[2] & 255u) << 16 | b[3] << 24;
                rv.w[0][1] = b[0] >> 8 | (b[1] >> 8) << 8 | (b[2] >> 8) << 16 | (b[3] >> 8) << 24;
            }
        };
        constexpr int kKaps = D == 128 ? 2 : 1, kQuads = D == 128 ? 2 : 1;
        // rows as they are: eight channels of token t; tokens behind the piece's end are zeros
        auto row8 = [&](bool of_keys, int t, int ch, float (&y)[8]) {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = 0.0f;
            if (t >= t_end) return;
            if (t < inside) {                                        // a token of a group that is not whole here
                const int64_t at = group_at(t);
                const int tt = t % G;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (of_keys) {
                        const uint32_t b = L.k_codes[at * (D * G / 4) + kblock_offset(ch + i, tt >> 2, G / 4, 64)];
                        y[i] = fmaf((float)((b >> (2 * (tt & 3))) & 3u), L.k_scales[at * D + ch + i], L.k_zeros[at * D + ch + i]);
                    } else {
                        const uint32_t b = L.v_codes[at * (D * G / 4) + vcode_offset(tt, (ch + i) / 4, D, G)];
                        const int64_t f = at * D + vmeta_index(tt, ch / G, D, G);
                        y[i] = fmaf((float)((b >> (2 * (i & 3))) & 3u), L.v_scales[f], L.v_zeros[f]);
                    }
                }
                return;
            }
            const __nv_bfloat16* from = t < q.held ? (of_keys ? k_ring : v_ring) + (int64_t)ring_slot(t, A.b.ring_shift, R) * D + ch
                                                   : (of_keys ? k_new + ((int64_t)q.row0 + t - q.held) * A.k.row_stride : v_new + ((int64_t)q.row0 + t - q.held) * A.v.row_stride) + ch;
            if (t < q.held || A.vec) {
                const uint4 x = *reinterpret_cast<const uint4*>(from);
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) { y[2 * i] = __uint_as_float(w[i] << 16); y[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = __bfloat162float(from[i]);
            }
        };
        auto top8 = [&](const float (&y)[8], uint32_t top, bool& finite) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                finite = finite && magnitude(y[i]) < 0x7f800000u;
                top = max(top, finite_magnitude(y[i]));
            }
            return top;
        };
        auto half8 = [&](const float (&y)[8], float f) {
            return make_uint4(pack_half(y[0] * f, y[1] * f), pack_half(y[2] * f, y[3] * f), pack_half(y[4] * f, y[5] * f), pack_half(y[6] * f, y[7] * f));
        };
        // tokens of the thread in a group of rows as they are: keys 4 * (k_j0 + i) + n, values 16 * kap + 4 * vc + n
        auto v_token = [&](int kap, int n) { return (D == 128 ? 16 * kap : 16 * part) + 4 * vc + n; };

        int v_run = 0;                                               // biased exponent of the largest value so far
        bool is_packed = packed(t_begin + G * g);
        if (is_packed) { const int64_t at = group_at(t_begin + G * g); fetch_k(at); fetch_v(at); }
        bool ok = true;
        for (int j = 0; j < n_tiles; ++j) {
            const int t0 = t_begin + j * kN + G * g, st = j & 1;
            // ---- largest of the tile ----
            uint32_t k_top = 0u, v_top = 0u, odd = 0u;
            if (is_packed) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float sv[4] = {rk.s[i].x, rk.s[i].y, rk.s[i].z, rk.s[i].w}, zv[4] = {rk.z[i].x, rk.z[i].y, rk.z[i].z, rk.z[i].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) k_top = max(k_top, max(finite_magnitude(zv[e]), finite_magnitude(fmaf(3.0f, sv[e], zv[e]))));
                }
#pragma unroll
                for (int kap = 0; kap < kKaps; ++kap)
#pragma unroll
                    for (int n = 0; n < 4; ++n) v_top = max(v_top, max(finite_magnitude(rv.z[kap][n]), finite_magnitude(fmaf(3.0f, rv.s[kap][n], rv.z[kap][n]))));
            } else {
                bool none = true;
#pragma unroll 1
                for (int i = 0; i < 4 * kQuads; ++i) {
                    float y[8];
                    row8(true, t0 + 4 * k_j0 + i, k_ch, y);
                    k_top = top8(y, k_top, none);
                }
#pragma unroll 1
                for (int i = 0; i < 4 * kKaps; ++i) {
                    bool finite = true;
                    const int tok = v_token(i >> 2, i & 3);
                    float y[8];
                    row8(false, t0 + tok, v_ch, y);
                    v_top = top8(y, v_top, finite);
                    if (!finite) odd |= 1u << tok;
                }
                odd = __reduce_or_sync(0xffffffffu, odd);
            }
            k_top = __reduce_max_sync(0xffffffffu, k_top);
            v_top = __reduce_max_sync(0xffffffffu, v_top);
            if (lane == 0) {
                misc.top[st][0][pw] = k_top;
                misc.top[st][1][pw] = v_top;
                if (part == 0) misc.odd[j % kRing][g] = 0u;
            }
            asm volatile("bar.sync 1, %0;" ::"n"(kProducers) : "memory");
            if (lane == 0 && odd) atomicOr(&misc.odd[j % kRing][g], odd);
            uint32_t kt = 0u, vt = 0u;
#pragma unroll
            for (int w = 0; w < kProducerWarps; ++w) { kt = max(kt, misc.top[st][0][w]); vt = max(vt, misc.top[st][1][w]); }
            const int k_shift = shift_of(exponent_of(kt));
            v_run = max(v_run, exponent_of(vt));
            const int v_shift = shift_of(v_run);
            if (pw == 0 && lane == 0) { misc.k_shift[j % kRing] = k_shift; misc.v_shift[j % kRing] = v_shift; }

            // ---- keys ----
            if (ok && j >= 2) ok = wait_warp(misc.k_empty[st], (j >> 1) - 1);        // (given up: on to the end, the other warps wait at the barrier above)
            uint8_t* const kt_s = smem + S::k + st * S::kTileBytes + (D == 128 ? part * (kN * 128) : 0);
            const float kf = pow2i(k_shift);
            const int k_piece = 2 * kc + km;
            const int next = t0 + kN;
            const bool next_packed = j + 1 < n_tiles && packed(next);
            const int64_t next_at = next_packed ? group_at(next) : 0;
            if (is_packed) {
                uint32_t s2[4], z2[4];
                s2[0] = pack_half(rk.s[0].x * kf, rk.s[0].y * kf); s2[1] = pack_half(rk.s[0].z * kf, rk.s[0].w * kf);
                s2[2] = pack_half(rk.s[1].x * kf, rk.s[1].y * kf); s2[3] = pack_half(rk.s[1].z * kf, rk.s[1].w * kf);
                z2[0] = pack_half(rk.z[0].x * kf, rk.z[0].y * kf); z2[1] = pack_half(rk.z[0].z * kf, rk.z[0].w * kf);
                z2[2] = pack_half(rk.z[1].x * kf, rk.z[1].y * kf); z2[3] = pack_half(rk.z[1].z * kf, rk.z[1].w * kf);
                uint32_t x[kQuads][4];                               // bytes of two channels, 16 bits apart
#pragma unroll
                for (int i = 0; i < kQuads; ++i) {
                    x[i][0] = __byte_perm(rk.w[2 * i], 0u, 0x4140); x[i][1] = __byte_perm(rk.w[2 * i], 0u, 0x4342);
                    x[i][2] = __byte_perm(rk.w[2 * i + 1], 0u, 0x4140); x[i][3] = __byte_perm(rk.w[2 * i + 1], 0u, 0x4342);
                }
                if (next_packed) fetch_k(next_at);
#pragma unroll
                for (int n = 0; n < 4; ++n) {
#pragma unroll
                    for (int i = 0; i < kQuads; ++i) {
                        uint32_t y[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[e] = hfma2(hadd2((x[i][e] & (0x00030003u << (2 * n))) | k1024, kMinus1024), s2[e], z2[e]);
                        *reinterpret_cast<uint4*>(kt_s + swizzled(G * g + 4 * (k_j0 + i) + n, k_piece)) = make_uint4(y[0], y[1], y[2], y[3]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) s2[e] = hmul2(s2[e], 0x34003400u);        // a quarter
                }
            } else {
                if (next_packed) fetch_k(next_at);
#pragma unroll 1
                for (int i = 0; i < 4 * kQuads; ++i) {
                    const int tok = 4 * k_j0 + i;
                    float y[8];
                    row8(true, t0 + tok, k_ch, y);
                    *reinterpret_cast<uint4*>(kt_s + swizzled(G * g + tok, k_piece)) = half8(y, kf);
                }
            }
            fence_async();
            __syncwarp();
            if (lane == 0) arrive(bar(misc.k_full[st]));

            // ---- values ----
            if (ok && j >= 2) ok = wait_warp(misc.v_empty[st], (j >> 1) - 1);
            uint8_t* const vt_s = smem + S::v + st * S::kTileBytes + (v_ch / 64) * (kN * 128);
            const float vf = pow2i(v_shift);
            const int v_piece = (v_ch % 64) / 8;
            if (is_packed) {
                uint32_t w[kKaps][2];
                float sv[kKaps][4], zv[kKaps][4];
#pragma unroll
                for (int kap = 0; kap < kKaps; ++kap) {
                    w[kap][0] = rv.w[kap][0]; w[kap][1] = rv.w[kap][1];
#pragma unroll
                    for (int n = 0; n < 4; ++n) { sv[kap][n] = rv.s[kap][n] * vf; zv[kap][n] = rv.z[kap][n] * vf; }
                }
                if (next_packed) fetch_v(next_at);
#pragma unroll
                for (int kap = 0; kap < kKaps; ++kap)
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const uint32_t s_lo = pack_half(sv[kap][n], 0.25f * sv[kap][n]), s_hi = hmul2(s_lo, 0x2c002c00u) /* a sixteenth */, z = pack_half(zv[kap][n], zv[kap][n]);
                        uint32_t y[4];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t b = __byte_perm(w[kap][e], 0u, 0x4040 + 0x0101 * n);      // byte n in both halves
                            y[2 * e] = hfma2(hadd2((b & 0x000c0003u) | k1024, kMinus1024), s_lo, z);
                            y[2 * e + 1] = hfma2(hadd2((b & 0x00c00030u) | k1024, kMinus1024), s_hi, z);
                        }
                        *reinterpret_cast<uint4*>(vt_s + swizzled(G * g + v_token(kap, n), v_piece)) = make_uint4(y[0], y[1], y[2], y[3]);
                    }
            } else {
                if (next_packed) fetch_v(next_at);
#pragma unroll 1
                for (int i = 0; i < 4 * kKaps; ++i) {
                    const int tok = v_token(i >> 2, i & 3);
                    float y[8];
                    row8(false, t0 + tok, v_ch, y);
                    bool finite = true;
                    top8(y, 0u, finite);                             // (not finite: the rows that see it are told by `odd`)
                    *reinterpret_cast<uint4*>(vt_s + swizzled(G * g + tok, v_piece)) = finite ? half8(y, vf) : make_uint4(0u, 0u, 0u, 0u);
                }
            }
            fence_async();
            __syncwarp();
            if (lane == 0) arrive(bar(misc.v_full[st]));
            is_packed = next_packed;
        }
    } else if (elect_one()) {
        // ---------------- MMAs ----------------
        constexpr uint32_t kQK = mma_shape(kM, kN, false), kPV = mma_shape(kM, D, true);
        auto scores = [&](int t, int st) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                const uint32_t off = (uint32_t)(i / 4) * (kM * 128) + (i % 4) * 32;
                mma_ss(tmem + t * kN, smem_desc(base + S::q + t * S::kTileBytes + off, 16, 1024), smem_desc(base + S::k + st * S::kTileBytes + off, 16, 1024), kQK, i > 0);
            }
            mma_commit(bar(misc.s_full[t]));
        };
        bool ok = wait(misc.q_full, 0) && wait(misc.k_full[0], 0);
        if (ok) {
            fence_after();
            for (int t = 0; t < n_sub; ++t) scores(t, 0);
            mma_commit(bar(misc.k_empty[0]));
            for (int j = 0; ok && j < n_tiles; ++j) {
                const int st = j & 1;
                const bool more = j + 1 < n_tiles;
                if (!wait(misc.v_full[st], j >> 1) || (more && !wait(misc.k_full[st ^ 1], (j + 1) >> 1))) { ok = false; break; }
                for (int t = 0; t < n_sub; ++t) {
                    if (!wait(misc.p_full[t], j)) { ok = false; break; }
                    fence_after();
#pragma unroll
                    for (int i = 0; i < kN / 16; ++i)
                        mma_ts(tmem + 2 * kN + t * D, tmem + t * kN + 8 * i, smem_desc(base + S::v + st * S::kTileBytes + i * 2048, kN * 128, 1024), kPV, j > 0 || i > 0);
                    if (more) scores(t, st ^ 1);
                }
                if (!ok) break;
                mma_commit(bar(misc.v_empty[st]));
                if (more) mma_commit(bar(misc.k_empty[st ^ 1]));
            }
            if (ok) mma_commit(bar(misc.o_done));
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 16) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

}  // namespace

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
