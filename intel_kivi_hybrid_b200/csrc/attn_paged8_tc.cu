// Attention of a step's rows over a paged cache in 8 bits on the 5th-generation tensor cores:
// head_dim 64 and 128, blocks of whole 32 tokens, bf16 rows.
//
//   S = Q K^T,  P = 2^(rules(S) - m),  O = O + P V,  out = O / sum P
//
// over tiles of 128 tokens, for two blocks of 128 rows at a time ((new token, query head)
// pairs of one sequence and KV head: all heads of a group share the tile).  Roles of the 16
// warps:
//   0-3, 4-7   a thread per row of the first / second block: maximum, weights, running sum,
//              rescaling, output
//   8-11       values of a tile of pages become fp16 numbers in shared memory; those of the
//              window and the new tokens are brought as they are
//   12         one thread issues the MMAs: S of a block while the other block's weights are
//              made; P comes from tensor memory, where it takes the place of S
//   13         one thread brings the bytes of the pages to shared memory with bulk copies
//   14, 15     keys of the window and the new tokens, as they are
//
// Keys of a page are operands as they lie: S is two MMAs of kind f8f6f4, a row of Q less a
// power of two being the sum of two e4m3 numbers (a bf16 number is, as far as 2^-9 of the
// row's largest; what is smaller is off by 2^-17 of it).  They take as long as one of fp16 operands
// would, without a conversion of K, the shared memory it takes and its traffic there.  A block's key scale multiplies S.
// Values are fp16, which e4m3 numbers are exactly, with P in fp16: a weight times its value
// scale less the power of two of the largest such product that the row has met, so that neither
// a row's own range nor what other rows see takes its bits.  Two terms of e4m3 would do for P's bits, not for its range.
// Window and new tokens are bf16 operands as they are, Q and P then too: Q is written again
// when the pages are done.  Keys of a page are there codes times their scale's power of two, and its rest multiplies S; where only
// some of a group's tokens come from the page, the others' scores are divided by that rest (keys rounded to bf16 instead: 0.0027 off
// 64 bits where the output's rounding is 0.0017), and the page's values are held the same way, their rest in the weights.  P is rounded
// at 2^-8 there, at 2^-11 over pages: bf16 for the values' range (0.0019 to 0.0022 off 64 bits where most of the weight lies on such
// rows).  A value that is not finite would reach all rows of a tile through weights of 0: it is left out there, and added to the
// outputs of the rows that see it.
//
// Per tile and SM: 2048 cycles of MMA for 256 rows, 2048 of exponentials (16 a cycle).
#include "paged8_attention.cuh"
#include "tcgen05.cuh"

#include <type_traits>

namespace kivi {
namespace {

__device__ int g_fault = 0;

constexpr int kN = 128;                                  // tokens of a tile
constexpr int kM = 128;                                  // rows of a block
constexpr int kG = 32;                                   // tokens that share their scales
constexpr int kThreads = 512, kStageWarp = 8, kMmaWarp = 12, kCopyWarp = 13, kKeyWarp = 14;
constexpr int kRing = 8;                                 // scales of so many tiles are kept
// Who says of each tile that its keys' stage may be filled again: the MMAs, the values' warps, each of the two keys' warps,
// and the copies (in tiles of rows the first keys' warp for them).  A barrier tells a phase from the next one only, so whoever
// waits for it has a part in each of its phases and cannot be overtaken by two.
constexpr int kStageUsers = 5;
constexpr float kGrowth = 8.0f;                          // weights up to 2^8 are let stand before the maximum moves
constexpr float kHeadroom = 8.0f, kSlack = 6.0f;         // products of weight and scale: up to 2^8, or 2^14 before their reference moves

template <int D> struct Shared {
    static constexpr uint32_t kRow = D == 128 ? 128 : 64;            // bytes of a row of e4m3 operands
    static constexpr uint32_t kF8 = kM * kRow;                       // bytes of 128 such rows
    static constexpr uint32_t kTile = kN * D * 2;                    // of 128 rows of 16-bit operands
    static constexpr uint32_t q = 0, a = 2 * kTile, v = a + 2 * kTile;            // a: keys (and the bytes of the values behind them), two stages
    static constexpr uint32_t raw_v = kN * D;                        // in a stage
    static constexpr uint32_t bars = v + 2 * kTile;
    static constexpr uint32_t bytes = bars + 2048 + 1024;            // (the tiles start on a boundary of 1024)
};

struct Misc {                                            // behind the tiles
    uint64_t q_full, q_again[2], k_full[2], a_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2][2], o_done;
    uint32_t tmem;
    int place[2];
    int odd;                                             // a value that is not finite has been met
    float4 k_scale[kRing], v_scale[kRing];               // of tile j's four groups at j % kRing; values': their log2
    float v_rest;                                        // of the group that is partly in its page: its values' scale over their power of two
};

__device__ __forceinline__ float2 ex2x2(float2 x) { return make_float2(ex2(x.x), ex2(x.y)); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t y;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
    return y;
}
__device__ __forceinline__ float log2_of(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pow2i(int s) { return __uint_as_float((uint32_t)(127 + max(-126, min(127, s))) << 23); }

// a scale as a power of two and the rest, 1 to 2
__device__ __forceinline__ float power_of(float x) { return __uint_as_float(__float_as_uint(x) & 0x7f800000u); }
__device__ __forceinline__ float rest_of(float x) { return __uint_as_float((__float_as_uint(x) & 0x7fffffu) | 0x3f800000u); }

// cap * tanh(z)
__device__ __forceinline__ float2 capped_near(float2 z, float cap) {
    const float2 s = mul2(z, z);
    float2 p = fma2(s, both(kTanh9), both(kTanh7));
    p = fma2(p, s, both(kTanh5));
    p = fma2(p, s, both(kTanh3));
    p = fma2(p, s, both(kTanh1));
    return mul2(mul2(p, z), both(cap));
}
__device__ __forceinline__ float capped_far(float z, float cap) {
    const float e = z * 2.8853900817779268f;
    return cap - __fdividef(2.0f * cap, 1.0f + ex2(e > 120.0f ? 120.0f : e));
}

// What is done to scores: nothing, slopes alone, a cap up to kSmallCap and not far above sm_scale, any cap (both of them with
// slopes or without).
enum { kNoRules, kSlopes, kSmallCaps, kAnyCaps };

template <int D, int RULES>
__global__ void __launch_bounds__(kThreads, 1)
paged8_tc_kernel(Paged8Attn A) {
    using S = Shared<D>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    Misc& misc = *reinterpret_cast<Misc*>(smem + S::bars);
    static_assert(sizeof(Misc) <= 2048, "behind the tiles");
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const uint32_t base = smem_u32(smem);

    stream_order();
    settle_args(A);
    const kivi_paged8_layer& L = A.L;
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
        if (lane == 0) { misc.place[0] = p.s; misc.place[1] = p.sub; misc.odd = 0; }
    }
    __syncthreads();
    const int s = misc.place[0];
    if (s >= A.b.num_seqs) return;
    PagedSeq q;
    load_seq(L, A.b, s, q);
    const int rows = q.n * n_rep, row_first = misc.place[1] * 2 * kM, total = q.held + q.n;
    const int n_rows = min(rows - row_first, 2 * kM), n_sub = n_rows > kM ? 2 : 1;
    const int inside = min(quant_of(total, L.group_size, R), q.held), window = A.rules.window, prefix = prefix_of(A.rules, s, total);
    const int p_lo = q.held + row_first / n_rep, p_hi = q.held + (row_first + n_rows - 1) / n_rep;
    const Span span = span_of(kN, total, p_lo, p_hi, window, prefix);
    const int v_begin = blockIdx.z * A.chunk;
    if (v_begin >= span.n) return;
    const int n_tiles = min(A.chunk, span.n - v_begin);
    const bool whole = span.n <= A.chunk;
    auto tile_start = [&](int j) { return span.tile(v_begin + j) * kN; };
    // the first n_packed tiles come from pages alone
    int n_packed = 0;
    {
        const int full = inside / kN;                    // token tiles
        n_packed = min(span.n1, full) + max(0, full - (span.n1 + span.gap)) - v_begin;
        n_packed = max(0, min(n_packed, n_tiles));
    }

    auto bar = [&](const uint64_t& b) { return smem_u32(&b); };
    if (warp == kMmaWarp) {
        if (elect_one()) {
            mbar_init(bar(misc.q_full), kM * n_sub);
            for (int i = 0; i < 2; ++i) {
                mbar_init(bar(misc.q_again[i]), kM);
                mbar_init(bar(misc.k_full[i]), 1); mbar_init(bar(misc.a_empty[i]), kStageUsers);
                mbar_init(bar(misc.v_full[i]), 1); mbar_init(bar(misc.v_empty[i]), 1);
                mbar_init(bar(misc.s_full[i]), 1); mbar_init(bar(misc.p_full[i][0]), kM); mbar_init(bar(misc.p_full[i][1]), kM);
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
        if (mbar_sleep(bar(b), (uint32_t)phase & 1u)) return true;
        atomicOr(&g_fault, 1);
        return false;
    };
    auto wait_warp = [&](const uint64_t& b, int phase) { return __all_sync(0xffffffffu, wait(b, phase)) != 0; };

    if (warp < kStageWarp) {
        // ---------------- rows ----------------
        const int t = warp >> 2, r = tid & (kM - 1);
        if (t < n_sub) {
            const int in_cta = t * kM + r, row = row_first + in_cta;
            const bool there = in_cta < n_rows;
            // (a row that is not there sees what the block's first one sees, and is not written)
            const int token = (there ? row : row_first) / n_rep, head = h * n_rep + (there ? row : row_first) % n_rep, place = q.held + token, from = window_from(place, window);
            const __nv_bfloat16* const q_row = reinterpret_cast<const __nv_bfloat16*>(A.q.data) + ((int64_t)q.row0 + token) * A.q.row_stride + (int64_t)head * A.q.head_stride;
            auto q8 = [&](int d) {                       // eight channels as they lie
                if (A.vec) return *reinterpret_cast<const uint4*>(q_row + d);
                const uint16_t* u = reinterpret_cast<const uint16_t*>(q_row + d);
                return make_uint4(u[0] | (uint32_t)u[1] << 16, u[2] | (uint32_t)u[3] << 16, u[4] | (uint32_t)u[5] << 16, u[6] | (uint32_t)u[7] << 16);
            };
            uint8_t* const q_at = smem + S::q + t * S::kTile;
            auto q_as_bf16 = [&] {
#pragma unroll 1
                for (int d = 0; d < D; d += 8) *reinterpret_cast<uint4*>(q_at + (d / 64) * (kM * 128) + swizzled(r, (d % 64) / 8)) = q8(d);
            };
            int q_shift = 0;
            if (n_packed > 0) {
                uint32_t top = 0u;
#pragma unroll 1
                for (int d = 0; d < D; d += 8) {
                    const uint4 x = q8(d);
                    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {        // (the largest finite one)
                        const uint32_t lo = (w[i] << 16) & 0x7fffffffu, hi = w[i] & 0x7fff0000u;
                        top = max(top, max(lo < 0x7f800000u ? lo : 0u, hi < 0x7f800000u ? hi : 0u));
                    }
                }
                const int e = (int)(top >> 23);
                q_shift = min(126, 127 + 7 - e);          // to 2^7 .. 2^8 (what is below 2^-119 as far as a power of two goes)
                const float f = pow2i(q_shift);
#pragma unroll 1
                for (int d = 0; d < D; d += 16) {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint4 x = q8(d + 8 * i);
                        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float a = __uint_as_float(w[k] << 16) * f, b = __uint_as_float(w[k] & 0xffff0000u) * f;
                            uint32_t first = to_e4m3x2(a, b);
                            const uint32_t half = e4m3x2_to_half2(first);
                            const uint32_t rest = to_e4m3x2(a - half_lo(half), b - half_hi(half));
                            if (!(fabsf(a) <= 448.0f)) first |= 0x7fu;                // (infinite: not a number)
                            if (!(fabsf(b) <= 448.0f)) first |= 0x7f00u;
                            const int at = 2 * i + (k >> 1), sh = 16 * (k & 1);
                            hi[at] = sh ? hi[at] | first << 16 : first;
                            lo[at] = sh ? lo[at] | rest << 16 : rest;
                        }
                    }
                    const uint32_t piece = D == 128 ? (uint32_t)(d / 16) ^ (r & 7) : (uint32_t)(d / 16) ^ ((r >> 1) & 3), at = (uint32_t)r * S::kRow + piece * 16;
                    *reinterpret_cast<uint4*>(q_at + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    *reinterpret_cast<uint4*>(q_at + S::kF8 + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
            } else {
                q_as_bf16();
            }
            fence_async();
            arrive(bar(misc.q_full));

            const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16, s_at = tmem + lanes + t * kN, o_at = tmem + lanes + 2 * kN + t * D;
            constexpr float kLog2e = 1.4426950408889634f;
            auto factor = [](float scale, float to) { return fmaxf(scale * to, 1.2e-38f); };         // (not 0: hidden columns are -inf)
            const bool capped = RULES >= kSmallCaps && A.rules.softcap > 0.0f, biased = RULES != kNoRules && A.rules.slopes != nullptr;
            const float cap = A.rules.softcap * kLog2e, slope = biased && there ? A.rules.slopes[head] * kLog2e : 0.0f;
            // (Any cap: to scores first, then over the cap: the two at once may be below what fp32 holds.)
            const float to_x = RULES == kAnyCaps ? A.scale : capped ? A.scale / A.rules.softcap : A.scale * kLog2e, inv_cap = RULES == kAnyCaps ? 1.0f / A.rules.softcap : 1.0f;
            float m = -INFINITY, ref = -1.0e30f, l = 0.0f, base_m = 0.0f, up = 0.0f;         // ref: the largest maximum plus value scale, so far; up: log2 of what brings weights times scales to O's scale
            bool ok = true, low = false;                 // low: a row of the warp has `up` below -60
            for (int j = 0; j < n_tiles; ++j) {
                // (given up: on to the end without waiting)
                if (ok) ok = wait_warp(misc.s_full[t], j);
                fence_after();
                const int t0 = tile_start(j);
                const bool packed = j < n_packed;
                const float* const k_scales = reinterpret_cast<const float*>(&misc.k_scale[j % kRing]);
                const float* const v_scales = reinterpret_cast<const float*>(&misc.v_scale[j % kRing]);
                const float to_c = to_x * (packed ? pow2i(-q_shift) : 1.0f);
                // columns that the row sees: below `near`, and lo .. hi
                const int near = prefix - t0, lo = from - t0, hi = place - t0;
                const bool edge = __any_sync(0xffffffffu, near < kN && (lo > 0 || hi < kN - 1));
                // a group of which the first columns alone come from its page: the others' scores are divided by what multiplies it
                const int cut = inside - t0;
                const bool cuts = cut > 0 && cut < kN && cut % kG != 0;
                if (cuts) {
                    const float inv = __fdividef(1.0f, k_scales[cut / kG]);
#pragma unroll 1
                    for (int x = cut / kG * kG; x < cut / kG * kG + kG; x += 16) {
                        uint32_t o[16];
                        tmem_load16(s_at + x, o);
                        tmem_wait_load();
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (x + i >= cut) o[i] = __float_as_uint(__uint_as_float(o[i]) * inv);
                        tmem_store16(s_at + x, o);
                    }
                    tmem_wait_store();
                }
                float top_all = -INFINITY, most = -INFINITY;         // most: with the value scales
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
                    uint32_t v[2][32];
                    tmem_load32(s_at + 64 * half, v[0]);
                    tmem_load32(s_at + 64 * half + 32, v[1]);
                    const float c[2] = {factor(k_scales[2 * half], to_c), factor(k_scales[2 * half + 1], to_c)};
                    tmem_wait_load();
                    auto at2 = [&](int g, int i) { return make_float2(__uint_as_float(v[g][i]), __uint_as_float(v[g][i + 1])); };
                    auto put2 = [&](int g, int i, float2 x) { v[g][i] = __float_as_uint(x.x); v[g][i + 1] = __float_as_uint(x.y); };
                    if constexpr (RULES != kNoRules) {
                        if (capped) {
                            float far = 0.0f;
#pragma unroll
                            for (int g = 0; g < 2; ++g)
#pragma unroll
                                for (int i = 0; i < 32; i += 2) {
                                    float2 z = mul2(at2(g, i), both(c[g]));
                                    if constexpr (RULES == kAnyCaps) z = mul2(z, both(inv_cap));
                                    far = fmaxf(far, fmaxf(fabsf(z.x), fabsf(z.y)));
                                    put2(g, i, z);
                                }
                            if (__any_sync(0xffffffffu, far > kTanhNear)) {
                                if constexpr (RULES != kAnyCaps) {
#pragma unroll
                                    for (int g = 0; g < 2; ++g)
#pragma unroll
                                        for (int i = 0; i < 32; ++i) v[g][i] = __float_as_uint(capped_far(__uint_as_float(v[g][i]), cap));
                                } else {                 // (what is near 0 is not to pay for what is far)
#pragma unroll
                                    for (int g = 0; g < 2; ++g)
#pragma unroll
                                        for (int i = 0; i < 32; i += 2) {
                                            const float2 z = at2(g, i), y = capped_near(z, cap);
                                            put2(g, i, make_float2(fabsf(z.x) <= kTanhNear ? y.x : capped_far(z.x, cap), fabsf(z.y) <= kTanhNear ? y.y : capped_far(z.y, cap)));
                                        }
                                }
                            } else {
#pragma unroll
                                for (int g = 0; g < 2; ++g)
#pragma unroll
                                    for (int i = 0; i < 32; i += 2) put2(g, i, capped_near(at2(g, i), cap));
                            }
                        }
                        if (biased) {
                            const float2 on = both(2.0f * slope);
#pragma unroll
                            for (int g = 0; g < 2; ++g) {
                                const float start = slope * (float)(t0 + 64 * half + kG * g - place);
                                float2 b = make_float2(start, start + slope);
#pragma unroll
                                for (int i = 0; i < 32; i += 2) {
                                    put2(g, i, capped ? add2(at2(g, i), b) : fma2(at2(g, i), both(c[g]), b));
                                    b = add2(b, on);
                                }
                            }
                        }
                    }
                    if (edge) {
                        const int a = near - 64 * half, b = lo - 64 * half, e = hi - 64 * half;
#pragma unroll
                        for (int i = 0; i < 64; ++i)
                            if (!(i < a || (i >= b && i <= e))) v[i / 32][i % 32] = 0xff800000u;
                    }
                    if (RULES != kNoRules || edge)              // (read again below)
#pragma unroll
                        for (int g = 0; g < 2; ++g)
#pragma unroll
                            for (int i = 0; i < 32; i += 16) tmem_store16(s_at + 64 * half + kG * g + i, reinterpret_cast<const uint32_t(&)[16]>(v[g][i]));
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        float x = -INFINITY, y = -INFINITY;
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            x = fmaxf(x, fmaxf(__uint_as_float(v[g][i]), __uint_as_float(v[g][i + 1])));
                            y = fmaxf(y, fmaxf(__uint_as_float(v[g][i + 2]), __uint_as_float(v[g][i + 3])));
                        }
                        x = fmaxf(x, y) * (RULES != kNoRules ? 1.0f : c[g]);
                        top_all = fmaxf(top_all, x);
                        most = fmaxf(most, x + v_scales[2 * half + g]);
                    }
                }
                if (RULES != kNoRules || edge) tmem_wait_store();
                if (__any_sync(0xffffffffu, top_all > m + kGrowth || most > ref + kSlack)) {
                    if (top_all > m + kGrowth) {         // (from -inf: whenever there is a maximum)
                        l *= m == -INFINITY ? 0.0f : ex2(m - top_all);
                        m = top_all;
                        base_m = m;
                    }
                    const bool grows = most > ref + kSlack;
                    if (__any_sync(0xffffffffu, grows)) {
                        const float f = grows ? ex2(ref - most) : 1.0f;
                        if (grows) ref = most;
                        if (j > 0) {
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
                    up = fminf(base_m - ref + kHeadroom, 126.0f);
                    low = __any_sync(0xffffffffu, up < -60.0f);
                }
                auto weights = [&](auto as_half) {
#pragma unroll 1
                    for (int half = 0; half < 2; ++half) {
                        uint32_t v[2][32];
                        tmem_load32(s_at + 64 * half, v[0]);
                        tmem_load32(s_at + 64 * half + 32, v[1]);
                        const float c[2] = {RULES != kNoRules ? 1.0f : factor(k_scales[2 * half], to_c), RULES != kNoRules ? 1.0f : factor(k_scales[2 * half + 1], to_c)};
                        // weights times value scales, on O's scale: 2^(lift) p.  (Below 2^-60 they are 0 as fp16 whatever they are, and bf16 ones are not made here.)
                        // (Tiles of rows have scales of 1 here.  Read all the same where there are no rules: 380 us, 390 without, for 512 rows over
                        // 32k; prompts of 2 x 4001 with a cap 642, 653 with.)
                        constexpr bool kScaled = decltype(as_half)::value || RULES == kNoRules;
                        const float lift[2] = {fmaxf(kScaled ? v_scales[2 * half] + up : up, -60.0f), fmaxf(kScaled ? v_scales[2 * half + 1] + up : up, -60.0f)};
                        tmem_wait_load();
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            uint32_t p[16];
                            const float2 off = both(lift[g] - base_m);
                            float2 part = make_float2(0.0f, 0.0f);
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                const float2 w = ex2x2(fma2(make_float2(__uint_as_float(v[g][i]), __uint_as_float(v[g][i + 1])), both(c[g]), off));
                                part = add2(part, w);
                                p[i / 2] = decltype(as_half)::value ? pack_half(w.x, w.y) : pack_bf16(w.x, w.y);
                            }
                            l = fmaf(part.x + part.y, ex2(-lift[g]), l);
                            tmem_store16(s_at + 32 * half + 16 * g, p);
                        }
                        tmem_wait_store();
                        fence_before();
                        arrive(bar(misc.p_full[t][half]));
                    }
                };
                // The same for tiles of rows that are rare: with tokens of pages, of which a group that is partly there wants the rest of its
                // values' scale; and beside values so much larger that weights on O's scale are below 2^-60, which bf16 holds as well as 1.
                auto weights_rare = [&] {
#pragma unroll 1
                    for (int x = 0; x < kN; x += 16) {
                        const int g = x / kG, edge = cuts && g == cut / kG ? cut - x : 0;            // columns before it have the rest
                        uint32_t v[16], p[8];
                        tmem_load16(s_at + x, v);
                        const float c = RULES != kNoRules ? 1.0f : factor(k_scales[g], to_c), f = ex2(fminf(fmaxf(v_scales[g] + up, -126.0f), 126.0f)), f_cut = f * misc.v_rest;
                        tmem_wait_load();
                        float part = 0.0f;
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            const float w0 = ex2(fmaf(__uint_as_float(v[i]), c, -base_m)), w1 = ex2(fmaf(__uint_as_float(v[i + 1]), c, -base_m));
                            part += w0 + w1;
                            p[i / 2] = pack_bf16(w0 * (i < edge ? f_cut : f), w1 * (i + 1 < edge ? f_cut : f));
                        }
                        l += part;
                        tmem_store8(s_at + x / 2, p);
                        if (x % 64 == 48) {
                            tmem_wait_store();
                            fence_before();
                            arrive(bar(misc.p_full[t][x / 64]));
                        }
                    }
                };
                if (packed) {
                    weights(std::true_type{});
                } else {
                    if (t0 < inside || low) weights_rare();
                    else weights(std::false_type{});
                }
                if (j + 1 == n_packed && j + 1 < n_tiles) {
                    // (S of this tile is there, so Q has been read)
                    q_as_bf16();
                    fence_async();
                    arrive(bar(misc.q_again[t]));
                }
            }
            if (ok) ok = wait_warp(misc.o_done, 0);
            fence_after();
            {
                const bool odd = *const_cast<volatile int*>(&misc.odd) != 0;
                // O is 2^(kHeadroom - ref) times the sum of weights in powers of two from 0
                const float f = m == -INFINITY ? 0.0f : ex2(fmaxf(ref - m - kHeadroom, -126.0f)), by = f * (whole ? 1.0f / l : 1.0f);      // (a row sees itself: l > 0)
                const int64_t at = ((int64_t)q.row0 + token) * A.out.row_stride + (int64_t)head * A.out.head_stride;
                const int64_t part = (((int64_t)item * H + h) * A.pieces + blockIdx.z) * (2 * kM) + in_cta;
#pragma unroll 1
                for (int x = 0; x < D; x += 16) {
                    uint32_t o[16];
                    tmem_load16(o_at + x, o);
                    tmem_wait_load();
                    if (!there) continue;
                    float y[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) y[i] = __uint_as_float(o[i]) * by;
                    if (odd) {
                        const __nv_bfloat16* const ring = reinterpret_cast<const __nv_bfloat16*>(L.v_res) + ((int64_t)q.slot * H + h) * R * D;
                        for (int j = n_packed; j < n_tiles; ++j)
                            for (int tok = max(tile_start(j), inside); tok < min(tile_start(j) + kN, total); ++tok) {
                                if (!(tok < prefix || (tok >= from && tok <= place))) continue;
                                const __nv_bfloat16* from_row = tok < q.held ? ring + (int64_t)ring_slot(tok, 0, R) * D
                                    : reinterpret_cast<const __nv_bfloat16*>(A.v.data) + ((int64_t)q.row0 + tok - q.held) * A.v.row_stride + (int64_t)h * A.v.head_stride;
#pragma unroll
                                for (int i = 0; i < 16; ++i) {
                                    const float z = __bfloat162float(from_row[x + i]);
                                    if (!(fabsf(z) <= 3.4e38f)) y[i] += z;
                                }
                            }
                    }
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const float4 z = make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]);
                        if (whole) store_quad(A.out.data, A.out_dtype, at + x + i, z);
                        else *reinterpret_cast<float4*>(A.part_o + part * D + x + i) = z;
                    }
                }
                if (!whole && there) *reinterpret_cast<float2*>(A.part_ml + 2 * part) = make_float2(m, l);
            }
            fence_before();
        }
    } else {
        auto scale_at = [&](int tok) {                   // of a token in pages
            const int64_t unit = (int64_t)page_of(L, q, tok, &g_fault) * H + h;
            return unit * (L.page_tokens / L.group_size) + tok % L.page_tokens / L.group_size;
        };
        // Keys or values of tokens first .. first + 31 to rows at .. of a tile of 64-channel halves, by a warp.
        auto group_of_rows = [&](bool of_keys, int first, int at, uint32_t to) {
            constexpr int kPieces = D / 8, kStep = 32 / kPieces;             // 16-byte pieces of a row; rows that a warp takes at a time
            const int p = lane % kPieces, r0 = lane / kPieces;
            auto place_of = [&](int r) { return to + (uint32_t)(p >> 3) * (kN * 128) + swizzled(at + r, p & 7); };
            const kivi_rows& fresh = of_keys ? A.k : A.v;
            const __nv_bfloat16* const fresh0 = reinterpret_cast<const __nv_bfloat16*>(fresh.data) + (int64_t)q.row0 * fresh.row_stride + (int64_t)h * fresh.head_stride + 8 * p;
            if (first < inside) {
                const int64_t unit = (int64_t)page_of(L, q, first, &g_fault) * H + h;
                const int in_page = first % L.page_tokens;
                const uint8_t* const codes = (of_keys ? L.k_codes : L.v_codes) + unit * L.page_tokens * D;
                // codes times their scale's power of two, which bf16 holds exactly: q k then fits where the formula's does
                const float f = of_keys ? power_of(L.k_scales[scale_at(first)]) : first + kG <= inside ? 1.0f : power_of(L.v_scales[scale_at(first)]);
#pragma unroll 1
                for (int r = r0; r < kG && first + r < inside; r += kStep) {
                    uint32_t b[2] = {0u, 0u}, w[4];
                    if (of_keys) {
                        const uint2 x = *reinterpret_cast<const uint2*>(codes + key8_offset(in_page + r, 8 * p, D));
                        b[0] = x.x; b[1] = x.y;
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) b[e >> 2] |= (uint32_t)codes[value8_offset(in_page + r, 8 * p + e, D, 32)] << (8 * (e & 3));
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float4 x = e4m3x4(b[e]);
                        w[2 * e] = pack_bf16(x.x * f, x.y * f); w[2 * e + 1] = pack_bf16(x.z * f, x.w * f);
                    }
                    sts128(place_of(r), w[0], w[1], w[2], w[3]);
                }
                if (first + kG <= inside) return;
            }
            // all of a lane's copies are on their way at once
            if (first >= q.held && first + kG <= total && A.vec) {
                const __nv_bfloat16* from = fresh0 + (int64_t)(first - q.held + r0) * fresh.row_stride;
                const int64_t step = kStep * fresh.row_stride;
#pragma unroll 4
                for (int r = r0; r < kG; r += kStep, from += step) copy16(place_of(r), from, true);
            } else {
                const __nv_bfloat16* const ring = reinterpret_cast<const __nv_bfloat16*>(of_keys ? L.k_res : L.v_res) + ((int64_t)q.slot * H + h) * R * D + 8 * p;
#pragma unroll 1
                for (int r = r0; r < kG; r += kStep) {
                    const int tok = first + r;
                    if (tok < inside) continue;
                    const bool held = tok < q.held, in = tok < total;
                    const __nv_bfloat16* const from = held ? ring + (int64_t)ring_slot(tok, 0, R) * D : fresh0 + (int64_t)(in ? tok - q.held : 0) * fresh.row_stride;
                    if (held || A.vec) { copy16(place_of(r), from, in); continue; }
                    const uint16_t* u = reinterpret_cast<const uint16_t*>(from);
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = in ? u[2 * e] | (uint32_t)u[2 * e + 1] << 16 : 0u;
                    sts128(place_of(r), w[0], w[1], w[2], w[3]);
                }
            }
            copies_wait();
            if (of_keys) return;
            // a lane looks its values over
#pragma unroll 4
            for (int r = r0; r < kG; r += kStep) {
                const uint4 x = lds_uint4(place_of(r));
                uint32_t w[4] = {x.x, x.y, x.z, x.w};
                bool bad = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if ((w[e] & 0x7f80u) == 0x7f80u) { w[e] &= 0xffff0000u; bad = true; }
                    if ((w[e] & 0x7f800000u) == 0x7f800000u) { w[e] &= 0xffffu; bad = true; }
                }
                if (bad) { misc.odd = 1; sts128(place_of(r), w[0], w[1], w[2], w[3]); }
            }
        };
        if (warp < kMmaWarp) {
            // ---------------- values; tiles of rows ----------------
            // (whoever has given up a wait says no more that anything is done: the others give up in their turn)
            const int i128 = tid & 127, g = warp - kStageWarp;
            auto meet = [&] { asm volatile("bar.sync 1, 128;" ::: "memory"); };
            bool ok = true;
#pragma unroll 1
            for (int j = 0; j < n_tiles; ++j) {
                const int st = j & 1, t0 = tile_start(j);
                const uint32_t a_at = base + S::a + st * S::kTile, v_at = base + S::v + st * S::kTile;
                if (j < n_packed) {
                    if (ok) ok = wait_warp(misc.k_full[st], j >> 1);
                    if (ok && j >= 2) ok = wait_warp(misc.v_empty[st], (j >> 1) - 1);
                    // a lane has 32 tokens of a channel: 32 bytes to 64, in the order of the tokens
#pragma unroll 1
                    for (int i = i128; i < 4 * D; i += 128) {
                        const int run = i / D, d = i % D;
                        const uint32_t raw = a_at + S::raw_v + (uint32_t)i * 32u;
                        const uint4 x = lds_uint4(raw), y = lds_uint4(raw + 16);
                        const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};       // [quarter][sixteen]
                        const uint32_t to = v_at + (run >> 1) * (D * 128) + (uint32_t)d * 128u;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {    // eight tokens: sixteen k / 2, its half k % 2
                            uint32_t z[4];
#pragma unroll
                            for (int u = 0; u < 4; ++u) z[u] = e4m3x2_to_half2(k & 1 ? w[2 * u + (k >> 1)] >> 16 : w[2 * u + (k >> 1)] & 0xffffu);
                            sts128(to + (((4 * (run & 1) + k) ^ (d & 7)) << 4), z[0], z[1], z[2], z[3]);
                        }
                    }
                    fence_async();
                    meet();
                    if (ok && i128 == 0) { arrive(bar(misc.a_empty[st])); arrive(bar(misc.v_full[st])); }
                } else {
                    if (ok && j >= 2) ok = wait_warp(misc.a_empty[st], (j >> 1) - 1) && wait_warp(misc.v_empty[st], (j >> 1) - 1);
                    group_of_rows(false, t0 + kG * g, kG * g, v_at);
                    fence_async();
                    meet();
                    // (nothing of these values lies in the keys' stage)
                    if (ok && i128 == 0) { arrive(bar(misc.a_empty[st])); arrive(bar(misc.v_full[st])); }
                }
            }
        } else if (warp >= kKeyWarp) {
            // ---------------- keys of tiles of rows, and all their scales ----------------
            bool ok = true;
#pragma unroll 1
            for (int j = 0; j < n_tiles; ++j) {
                const int st = j & 1, t0 = tile_start(j);
                // (every phase is waited for in its turn, the pages' tiles' too)
                if (ok && j >= 2) ok = wait_warp(misc.a_empty[st], (j >> 1) - 1);
                if (j < n_packed) {
                    if (ok && lane == 0) arrive(bar(misc.a_empty[st]));
                    continue;
                }
#pragma unroll 1
                for (int g = 2 * (warp - kKeyWarp); g < 2 * (warp - kKeyWarp) + 2; ++g) {
                    const int first = t0 + kG * g;
                    group_of_rows(true, first, kG * g, base + S::a + st * S::kTile);
                    if (lane == 0) {
                        float ks = 1.0f, vs = 1.0f;
                        if (first < inside) {
                            const int64_t f = scale_at(first);
                            ks = rest_of(L.k_scales[f]);
                            if (first + kG <= inside) vs = L.v_scales[f];
                            else misc.v_rest = rest_of(L.v_scales[f]);
                        }
                        reinterpret_cast<float*>(&misc.k_scale[j % kRing])[g] = ks;
                        reinterpret_cast<float*>(&misc.v_scale[j % kRing])[g] = log2_of(vs);
                    }
                }
                fence_async();
                asm volatile("bar.sync 2, 64;" ::: "memory");
                if (ok && lane == 0) arrive(bar(misc.a_empty[st]));
                if (ok && tid == 32 * kKeyWarp) {
                    arrive(bar(misc.a_empty[st]));       // (in place of the copies)
                    arrive(bar(misc.k_full[st]));
                }
            }
        } else if (warp == kCopyWarp) {
            // ---------------- copies ----------------
            if (elect_one()) {
                const uint64_t policy = l2_stream_policy();
                bool ok = true;
                int sent = 0;
                for (int j = 0; ok && j < n_packed; ++j) {
                    const int t0 = tile_start(j), st = j & 1;
                    if (j >= 2 && !wait(misc.a_empty[st], (j >> 1) - 1)) { ok = false; break; }
                    const uint32_t to = base + S::a + st * S::kTile, b = bar(misc.k_full[st]);
                    float ks[4], vs[4];
                    int64_t at[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int tok = t0 + kG * i;
                        const int64_t unit = (int64_t)page_of(L, q, tok, &g_fault) * H + h;
                        const int in_page = tok % L.page_tokens;
                        at[i] = (unit * L.page_tokens + in_page) * D;
                        const int64_t f = unit * (L.page_tokens / L.group_size) + in_page / L.group_size;
                        ks[i] = L.k_scales[f]; vs[i] = L.v_scales[f];
                    }
                    misc.k_scale[j % kRing] = make_float4(ks[0], ks[1], ks[2], ks[3]);
                    misc.v_scale[j % kRing] = make_float4(log2_of(vs[0]), log2_of(vs[1]), log2_of(vs[2]), log2_of(vs[3]));
                    mbar_expect_tx(b, 2 * kN * D);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        bulk_g2s(to + i * (kG * D), L.k_codes + at[i], kG * D, b, policy);
                        bulk_g2s(to + S::raw_v + i * (kG * D), L.v_codes + at[i], kG * D, b, policy);
                    }
                    if (j < n_packed - 2) arrive(bar(misc.a_empty[st]));
                    sent = j + 1;
                }
                // no copy is under way when the block ends (and nobody fills the last two stages again before this has been seen)
                for (int j = max(sent - 2, 0); j < sent; ++j)
                    if (wait(misc.k_full[j & 1], j >> 1) && ok) arrive(bar(misc.a_empty[j & 1]));
            }
        } else if (warp == kMmaWarp) {
            // ---------------- MMAs ----------------
            // The whole warp goes through the steps and one lane issues, with operands that are the same in all lanes and
            // offsets that are constants.  What a tile waits for is the MMAs themselves: 64 cycles for one of 16 (fp8: 32) channels
            // or tokens alone, 76 to 100 beside the other warps' traffic in shared memory.
            constexpr uint32_t kF8 = mma_shape(kM, kN, false), kPages = mma_shape(kM, D, false), kBf16 = mma_shape(kM, kN, false, 1u), kRowsV = mma_shape(kM, D, true, 1u);
            constexpr uint32_t kSwizzle = D == 128 ? 2u : 4u;
            const uint32_t base_u = __shfl_sync(0xffffffffu, base, 0), tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
            auto scores = [&](int t, int j) {
                const uint32_t q_at = base_u + S::q + t * S::kTile, k_at = base_u + S::a + (j & 1) * S::kTile, to = tmem_u + t * kN;
                if (j < n_packed) {
                    const uint64_t qd = smem_desc(q_at, 16, 8 * S::kRow, kSwizzle), kd = smem_desc(k_at, 16, 8 * S::kRow, kSwizzle);
                    if (elect_one()) {
#pragma unroll
                        for (int i = 0; i < 2 * (D / 32); ++i)
                            mma_f8_ss(to, qd + ((i / (D / 32)) * S::kF8 + (i % (D / 32)) * 32u) / 16u, kd + (i % (D / 32)) * 2u, kF8, i > 0);
                        mma_commit(bar(misc.s_full[t]));
                    }
                } else {
                    const uint64_t qd = smem_desc(q_at, 16, 1024), kd = smem_desc(k_at, 16, 1024);
                    if (elect_one()) {
#pragma unroll
                        for (int i = 0; i < D / 16; ++i) {
                            const uint32_t off = ((uint32_t)(i / 4) * (kM * 128) + (i % 4) * 32) / 16;
                            mma_ss(to, qd + off, kd + off, kBf16, i > 0);
                        }
                        mma_commit(bar(misc.s_full[t]));
                    }
                }
                __syncwarp();
            };
            // weights of block t of tile j times its values
            auto contract = [&](int t, int j) {
                const uint32_t v_at = base_u + S::v + (j & 1) * S::kTile, to = tmem_u + 2 * kN + t * D, p_at = tmem_u + t * kN;
                const bool packed = j < n_packed;
                const uint64_t vd = packed ? smem_desc(v_at, 16, 1024) : smem_desc(v_at, kN * 128, 1024);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if (!wait_warp(misc.p_full[t][half], j)) return false;
                    fence_after();
                    if (packed) {
                        if (elect_one()) {
#pragma unroll
                            for (int i = 0; i < kN / 32; ++i) mma_ts(to, p_at + 32 * half + 8 * i, vd + (half * (D * 128) + i * 32) / 16, kPages, j > 0 || half > 0 || i > 0);
                        }
                    } else if (elect_one()) {
#pragma unroll
                        for (int i = 0; i < kN / 32; ++i) mma_ts(to, p_at + 32 * half + 8 * i, vd + (4 * half + i) * 128, kRowsV, j > 0 || half > 0 || i > 0);
                    }
                    __syncwarp();
                }
                return true;
            };
            auto commit = [&](const uint64_t& b) {
                if (elect_one()) mma_commit(bar(b));
                __syncwarp();
            };
            bool ok = wait_warp(misc.q_full, 0) && wait_warp(misc.k_full[0], 0);
            if (ok) {
                fence_after();
                for (int t = 0; t < n_sub; ++t) scores(t, 0);
                commit(misc.a_empty[0]);
                for (int j = 0; ok && j < n_tiles; ++j) {
                    const int st = j & 1;
                    const bool more = j + 1 < n_tiles, turns = more && j + 1 == n_packed;
                    if (!wait_warp(misc.v_full[st], j >> 1)) { ok = false; break; }
                    for (int t = 0; t < n_sub; ++t) {
                        ok = contract(t, j);
                        if (t == 0 && more && ok) ok = wait_warp(misc.k_full[st ^ 1], (j + 1) >> 1);
                        if (turns && ok) ok = wait_warp(misc.q_again[t], 0);
                        if (!ok) break;
                        fence_after();
                        if (more) scores(t, j + 1);
                    }
                    if (!ok) break;
                    if (elect_one()) {
                        mma_commit(bar(misc.v_empty[st]));
                        if (more) mma_commit(bar(misc.a_empty[st ^ 1]));
                    }
                    __syncwarp();
                }
                if (ok) commit(misc.o_done);
            }
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

}  // namespace

bool paged8_tc_serves(const kivi_paged8_layer* L, int q_dtype) {
    return (L->head_dim == 128 || L->head_dim == 64) && L->group_size % kG == 0 && L->res_dtype == KIVI_BF16 && q_dtype == KIVI_BF16;
}

int run_paged8_tc(const Paged8Attn& a, int blocks, cudaStream_t st) {
    auto go = [&](auto* kernel, uint32_t smem) {
        KIVI_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        KIVI_CUDA_OK(launch(kernel, dim3((unsigned)blocks, (unsigned)a.L.num_kv_heads, (unsigned)a.pieces), kThreads, smem, st, true, a));
        return KIVI_OK;
    };
    auto go_rules = [&](auto d) {
        constexpr int D = decltype(d)::value;
        if (a.rules.softcap > kSmallCap || a.scale < 1e-28f * a.rules.softcap) return go(paged8_tc_kernel<D, kAnyCaps>, Shared<D>::bytes);
        if (a.rules.softcap > 0.0f) return go(paged8_tc_kernel<D, kSmallCaps>, Shared<D>::bytes);
        return a.rules.slopes != nullptr ? go(paged8_tc_kernel<D, kSlopes>, Shared<D>::bytes) : go(paged8_tc_kernel<D, kNoRules>, Shared<D>::bytes);
    };
    return a.L.head_dim == 128 ? go_rules(std::integral_constant<int, 128>{}) : go_rules(std::integral_constant<int, 64>{});
}

int paged8_tc_fault_word(int* out) {
    KIVI_CUDA_OK(cudaMemcpyFromSymbol(out, g_fault, sizeof(int)));
    return KIVI_OK;
}
int paged8_tc_fault_clear() {
    const int zero = 0;
    KIVI_CUDA_OK(cudaMemcpyToSymbol(g_fault, &zero, sizeof(int)));
    return KIVI_OK;
}

}  // namespace kivi
