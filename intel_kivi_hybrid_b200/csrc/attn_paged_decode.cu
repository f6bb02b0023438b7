// Attention of a few rows per sequence over a paged cache: single tokens, a handful of
// speculative ones.  head_dim 128, groups of 32 tokens.
//
// The arithmetic is that of the decode kernel over contiguous stores (attn_mma.cu): codes
// are contracted as bytes on the integer tensor cores, a CTA serves four rows ((new token,
// query head) pairs here).  What differs is where things are: a warp's token groups lie in
// pages, so each pair of groups is one run of copies or two; a sequence's length comes from
// device memory, so the grid is what the host's bounds allow and CTAs behind a sequence's
// end leave at once; and the tokens that are not packed -- window, the step's own, and up to 31
// of a group that the step's append has just moved to pages together with new tokens -- are
// a CTA's work of their own, with fp32 FMAs and the causal limit of each row.
//
// All rows see all whole packed groups.  Partials: the window's in slot 0, pieces behind it;
// a second kernel folds them.
//
// Bound as the contiguous kernel is: HBM and issue slots at length, latency with few tokens.
// 12 rows at most: a block of four rows costs what it costs there (510 instructions of a warp
// per group), the tensor-core kernel with 256 rows (attn_paged_tc.cu) the same for all.
#include "attn_mma_core.cuh"
#include "paged_attention.cuh"

namespace kivi {
namespace {

__device__ int g_fault = 0;

constexpr int kRows = 4;                                 // rows of a CTA

// ---- the tokens that are not packed ----------------------------------------------
// Running maximum, sum and output of the warp over tokens [t_begin, t_end), 32 a pass and
// kWarps warps side by side; row(t, value) gives the row of token t, last[h] the last token
// that row h sees.  lane = (4 tokens, quarter of the channels) for q.k, 4 channels for p.v.
template <typename T, typename Row>
__device__ __forceinline__ void window_part(const Row& row, int t_begin, int t_end, const int (&last)[kRows], const float* q_s, int lane, int warp,
                                            float (&m)[kRows], float (&l)[kRows], float (&o)[kRows][4]) {
    const int cq = lane & 3, tl = lane >> 2;
    for (int t0 = t_begin + 32 * warp; t0 < t_end; t0 += 32 * kWarps) {
        float acc[4][kRows];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int t = t0 + tl + 8 * j;
            const T* k = row(t < t_end ? t : t0, false) + 32 * cq;
#pragma unroll
            for (int h = 0; h < kRows; ++h) acc[j][h] = 0.0f;
#pragma unroll 2
            for (int c = 0; c < 4; ++c) {
                float kv[8];
                RowVec<T>::load8(k + 8 * c, kv);
#pragma unroll
                for (int h = 0; h < kRows; ++h) {
                    const float4 qa = *reinterpret_cast<const float4*>(q_s + h * kD + 32 * cq + 8 * c), qb = *reinterpret_cast<const float4*>(q_s + h * kD + 32 * cq + 8 * c + 4);
                    float a = acc[j][h];
                    a = fmaf(kv[0], qa.x, a); a = fmaf(kv[1], qa.y, a); a = fmaf(kv[2], qa.z, a); a = fmaf(kv[3], qa.w, a);
                    a = fmaf(kv[4], qb.x, a); a = fmaf(kv[5], qb.y, a); a = fmaf(kv[6], qb.z, a); a = fmaf(kv[7], qb.w, a);
                    acc[j][h] = a;
                }
            }
        }
        float p[4][kRows];
#pragma unroll
        for (int h = 0; h < kRows; ++h) {
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float sc = acc[j][h];
                sc += __shfl_xor_sync(0xffffffffu, sc, 1);
                sc += __shfl_xor_sync(0xffffffffu, sc, 2);
                const int t = t0 + tl + 8 * j;
                acc[j][h] = t < t_end && t <= last[h] ? sc : -INFINITY;
                mx = fmaxf(mx, acc[j][h]);
            }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float m_new = fmaxf(m[h], mx), base = m_new == -INFINITY ? 0.0f : m_new;
            const float alpha = ex2(m[h] - base);
            m[h] = m_new;
            float ps = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) { p[j][h] = ex2(acc[j][h] - base); ps += p[j][h]; }
            // the four lanes of a token quad hold the same p: count it once
            l[h] = l[h] * alpha + (cq == 0 ? ps : 0.0f);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[h][i] *= alpha;
        }
        const int ntok = t_end - t0 < 32 ? t_end - t0 : 32;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll 1
            for (int tk = 0; tk < 8 && 8 * j + tk < ntok; tk += 4) {
                float vv[4][4];
#pragma unroll
                for (int e = 0; e < 4; ++e) RowVec<T>::load4(row(t0 + min(8 * j + tk + e, ntok - 1), true) + 4 * lane, vv[e]);
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int h = 0; h < kRows; ++h) {
                        const float ph = __shfl_sync(0xffffffffu, p[j][h], 4 * (tk + e));
                        // (a token that the row does not see may hold anything, infinities and NaN too)
                        const bool seen = 8 * j + tk + e < ntok && t0 + 8 * j + tk + e <= last[h];
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[h][i] = fmaf(ph, seen ? vv[e][i] : 0.0f, o[h][i]);
                    }
            }
        }
    }
}

// grid = (row blocks of all sequences, KV heads, pieces + 1): the pieces of the packed
// groups first, the window (short) last.  WIDE: fp32 queries, operands long enough for fp32
// accuracy.  ONE: one row.
template <typename T, bool WIDE, bool ONE>
__global__ void __launch_bounds__(kWarps * 32, 3)
paged_decode_kernel(PagedAttnArgs A, int blocks_per_seq, int gps) {
    extern __shared__ __align__(128) uint8_t smem_raw[];
    uint8_t* const stage_mem = smem_raw;                                          // [kWarps][kStages][kStageBytes]
    uint8_t* const scratch_mem = smem_raw + kWarps * kStages * kStageBytes;       // [kWarps][kScratchBytes]
    uint64_t* const bars = reinterpret_cast<uint64_t*>(scratch_mem + kWarps * kScratchBytes);
    float* const ml_s = reinterpret_cast<float*>(bars + kWarps * kStages);        // [kWarps][4][2]
    float* const q_s = ml_s + kWarps * 4 * 2;                                     // [4][128] queries times scale * log2(e), absent rows zero

    cudaTriggerProgrammaticLaunchCompletion();           // (the fold behind this grid waits for its end)
    stream_order();
    settle_args(A);
    const kivi_paged_layer& L = A.L;
    const int H = L.num_kv_heads, R = L.residual_cap, n_rep = A.n_rep, h = blockIdx.y;
    const int s = (int)blockIdx.x / blocks_per_seq, row_first = ((int)blockIdx.x - s * blocks_per_seq) * kRows;
    const bool is_window = blockIdx.z == gridDim.z - 1;
    PagedSeq q;
    if (!load_seq(L, A.b, s, q) && is_window && h == 0 && row_first == 0 && threadIdx.x == 0) atomicOr(&g_fault, kPagedFault);
    const int n_rows = min(q.n * n_rep - row_first, kRows);
    if (n_rows <= 0) return;
    const int inside = min(quant_of(q.held + q.n, kG, R), q.held);
    const int n_groups = inside / kG;                    // whole groups that every row sees
    const int piece = blockIdx.z;
    const int g_begin = piece * gps;
    if (!is_window && g_begin >= n_groups) return;
    const int n_my_groups = is_window ? 0 : min(gps, n_groups - g_begin);

    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);
    const int gid = lane >> 2, tig = lane & 3;
    uint8_t* const wstage = stage_mem + warp * kStages * kStageBytes;
    float* const fo = reinterpret_cast<float*>(wstage);                           // [4][128] once the ring is idle
    const int n_chunks = (n_my_groups + kGPS - 1) / kGPS;
    const int my_n = n_chunks > warp ? (n_chunks - warp + kWarps - 1) / kWarps : 0;
    const uint32_t bar0 = smem_u32(bars + warp * kStages), stage0 = smem_u32(wstage);
    const int gpp = L.page_tokens / kG;
    if (!is_window) {
        if (elect_one()) {
#pragma unroll
            for (int i = 0; i < kStages; ++i) mbar_init(bar0 + 8 * i, 1);
            mbar_init_fence();
        }
        __syncwarp();
    }
    const uint64_t policy = l2_stream_policy();
    // Chunk c of the warp: groups g_begin + (warp + kWarps c) kGPS and the next, wherever their pages are.
    auto place = [&](int g) {
        const int page = q.pages[g / gpp];
        const bool there = (unsigned)page < (unsigned)L.num_pages;
        if (!there) atomicOr(&g_fault, kPagedFault);
        return ((int64_t)(there ? page : 0) * H + h) * gpp + g % gpp;
    };
    auto issue = [&](int c) {
        const int goff = (warp + kWarps * c) * kGPS;
        const int ng = min(n_my_groups - goff, kGPS);
        const int st = c % kStages;
        const uint32_t bar = bar0 + 8 * st, dst = stage0 + st * kStageBytes;
        if (elect_one()) {
            const int64_t a = place(g_begin + goff), b = ng > 1 ? place(g_begin + goff + 1) : a + 1;
            mbar_expect_tx(bar, ng * kGroupBytes);
            auto copy = [&](uint32_t at, int64_t g, uint32_t n) {                 // n groups side by side, group `at` of the stage first
                bulk_g2s(dst + at * 1024, L.k_codes + g * 1024, n * 1024, bar, policy);
                bulk_g2s(dst + kGPS * 1024 + at * 512, L.k_scales + g * 128, n * 512, bar, policy);
                bulk_g2s(dst + kGPS * 1536 + at * 512, L.k_zeros + g * 128, n * 512, bar, policy);
                bulk_g2s(dst + kGPS * 2048 + at * 1024, L.v_codes + g * 1024, n * 1024, bar, policy);
                bulk_g2s(dst + kGPS * 3 * 1024 + at * 512, L.v_scales + g * 128, n * 512, bar, policy);
                bulk_g2s(dst + kGPS * 3584 + at * 512, L.v_zeros + g * 128, n * 512, bar, policy);
            };
            if (b == a + 1) copy(0, a, ng);
            else { copy(0, a, 1); copy(1, b, 1); }
        }
        __syncwarp();
    };
    for (int c = 0; c < kStages && c < my_n; ++c) issue(c);

    // the rows' queries
    for (int i = threadIdx.x; i < kRows * kD / 4; i += kWarps * 32) {
        const int r = i >> 5, d = (i & 31) * 4, row = row_first + r;
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (r < n_rows) {
            const int64_t at = ((int64_t)q.row0 + row / n_rep) * A.q.row_stride + (int64_t)(h * n_rep + row % n_rep) * A.q.head_stride + d;
            if (WIDE) RowVec<float>::load4(reinterpret_cast<const float*>(A.q.data) + at, x);
            else RowVec<__nv_bfloat16>::load4(reinterpret_cast<const __nv_bfloat16*>(A.q.data) + at, x);
        }
        *reinterpret_cast<float4*>(q_s + r * kD + d) = make_float4(x[0] * A.scale_log2, x[1] * A.scale_log2, x[2] * A.scale_log2, x[3] * A.scale_log2);
    }
    __syncthreads();

    if (is_window) {
        float m[kRows], l[kRows], o[kRows][4];
        int last[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            m[r] = -INFINITY; l[r] = 0.0f;
            last[r] = r < n_rows ? q.held + (row_first + r) / n_rep : -1;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[r][i] = 0.0f;
        }
        // tokens of a group that left together with new ones: from its page to shared memory, fp32
        const int loose = inside - n_groups * kG;
        if (loose > 0) {
            float* const k_s = reinterpret_cast<float*>(stage_mem);               // [31][128], then the values
            float* const v_s = k_s + kG * kD;
            const int64_t g = place(n_groups);
            for (int i = threadIdx.x; i < loose * (kD / 4); i += kWarps * 32) {
                const int t = i >> 5, d = (i & 31) * 4;
                const uint32_t w = *reinterpret_cast<const uint32_t*>(L.k_codes + g * 1024 + kblock_offset(d, t >> 2, 8, 64));
                const uint32_t c = L.v_codes[g * 1024 + vcode_offset(t, d / 4, kD, kG)];
                const int64_t f = g * kD + vmeta_index(t, d / kG, kD, kG);
                const float vs = L.v_scales[f], vz = L.v_zeros[f];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    k_s[t * kD + d + e] = fmaf((float)((w >> (8 * e + 2 * (t & 3))) & 3u), L.k_scales[g * kD + d + e], L.k_zeros[g * kD + d + e]);
                    v_s[t * kD + d + e] = fmaf((float)((c >> (2 * e)) & 3u), vs, vz);
                }
            }
            __syncthreads();
            window_part<float>([&](int t, bool value) { return (value ? v_s : k_s) + (t - n_groups * kG) * kD; }, n_groups * kG, inside, last, q_s, lane, warp, m, l, o);
            __syncthreads();                             // the buffers take the outputs
        }
        const T* const k_ring = reinterpret_cast<const T*>(L.k_res) + ((int64_t)q.slot * H + h) * R * kD;
        const T* const v_ring = reinterpret_cast<const T*>(L.v_res) + ((int64_t)q.slot * H + h) * R * kD;
        const int t_end = min(q.held + (row_first + n_rows - 1) / n_rep + 1, q.held + q.n);
        window_part<T>([&](int t, bool value) {
            if (t < q.held) return (value ? v_ring : k_ring) + (int64_t)ring_slot(t, A.b.ring_shift, R) * kD;
            const kivi_rows& r = value ? A.v : A.k;
            return reinterpret_cast<const T*>(r.data) + ((int64_t)q.row0 + t - q.held) * r.row_stride + (int64_t)h * r.head_stride;
        }, inside, t_end, last, q_s, lane, warp, m, l, o);
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], off);
        if (lane < kRows) {
            float mr = m[0], lr = l[0];
#pragma unroll
            for (int r = 1; r < kRows; ++r)
                if (lane == r) { mr = m[r]; lr = l[r]; }
            ml_s[(warp * 4 + lane) * 2] = mr; ml_s[(warp * 4 + lane) * 2 + 1] = lr;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            float M = -INFINITY;
#pragma unroll
            for (int w2 = 0; w2 < kWarps; ++w2) M = fmaxf(M, ml_s[(w2 * 4 + r) * 2]);
            const float f = m[r] == -INFINITY ? 0.0f : ex2(m[r] - M);
            *reinterpret_cast<float4*>(fo + r * kD + 4 * lane) = make_float4(f * o[r][0], f * o[r][1], f * o[r][2], f * o[r][3]);
        }
    } else {
        std::conditional_t<ONE, OneView, LaneView> v;
        v.gid = gid; v.tig = tig; v.lane = lane;
        uint8_t* const scratch = scratch_mem + warp * kScratchBytes;
        v.scratch = smem_u32(scratch);
        // row `lane & 15` of matrix `lane >> 4`
        v.k_rows = v.scratch + 1024 * (lane >> 4) + 512 * (lane & 1) + 16 * ((lane >> 1) & 7);
        v.v_rows = v.scratch + 256 * (lane >> 4) + 16 * (lane & 15);
        // contraction index of the token whose scales are row `lane`
        const int kap = gid >> 2, k = 4 * tig + (gid & 3);
        v.v_write = v.scratch + 16 * k + 8 * (kap ^ (k >> 3));
        v.v_first = 32 * (tig >> 1);
        if constexpr (ONE) {
            v.p_write = v.scratch + 128 * (tig & 1) + 4 * (16 * kap + (gid & 3));
        } else {
            v.p_even = v.scratch + 16 * (16 * kap + (gid & 3)) + 64 * kap + 4 * tig;
            v.p_odd = v.scratch + 16 * (16 * kap + (gid & 3)) + 64 * (1 - kap) + 4 * tig;
            v.p_read = v.scratch + 16 * p_row(lane);
            v.rest_rows = 128 * (lane >> 4) + 512 * (lane & 1) + 16 * ((lane >> 1) & 7);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) asm volatile("mov.b32 %0, %1;" : "=r"(v.start[i]) : "n"(kTwo23Bits));
        load_queries<float>(q_s, kRows, 1.0f, v);
        if constexpr (WIDE) {
#pragma unroll
            for (int i = 0; i < 4; ++i) asm volatile("mov.b32 %0, %1;" : "=r"(v.ones[i]) : "n"(kOnes));
            v.q_zero = reinterpret_cast<const float4*>(q_s) + 32 * tig;
        }
        std::conditional_t<ONE, OneState, WarpState> st;
        clear(st);
        bool ok = true;
        int c = 0;
        for (; c < my_n; ++c) {
            const int i = c % kStages;
            if (!__all_sync(0xffffffffu, mbar_wait(bar0 + 8 * i, (uint32_t)(c / kStages) & 1u))) { ok = false; break; }
            const int goff = (warp + kWarps * c) * kGPS;
            const uint8_t* sb = wstage + i * kStageBytes;
            if (n_my_groups - goff >= 2) process_groups<2, WIDE>(sb, v, scratch, st);
            else process_groups<1, WIDE>(sb, v, scratch, st);
            __syncwarp();
            if (c + kStages < my_n) issue(c + kStages);
        }
        if (!ok) {
            // A copy did not land within the bound: the others in flight get a second bounded wait
            // before the ring is reused, then the partial is reported empty.
            if (lane == 0) atomicOr(&g_fault, 1);
            for (int i = c; i < c + kStages && i < my_n; ++i) mbar_wait(bar0 + 8 * (i % kStages), (uint32_t)(i / kStages) & 1u);
            clear(st);
        }
        fold_lanes<ONE>(v, st, scratch, fo, ml_s, warp);
    }
    __syncthreads();

    // ---- the CTA's partial: warps added in warp order ------------------------------
    const int64_t base = (((int64_t)blockIdx.x * H + h) * A.pieces + (is_window ? 0 : 1 + piece)) * kRows;
    for (int i = threadIdx.x; i < n_rows * kD / 4; i += kWarps * 32) {
        const int r = i >> 5, d = (i & 31) * 4;
        float4 a = *reinterpret_cast<const float4*>(stage_mem + (r * kD + d) * 4);
#pragma unroll
        for (int w2 = 1; w2 < kWarps; ++w2) {
            const float4 b = *reinterpret_cast<const float4*>(stage_mem + w2 * kStages * kStageBytes + (r * kD + d) * 4);
            a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
        }
        *reinterpret_cast<float4*>(A.part_o + (base + r) * kD + d) = a;
    }
    if ((int)threadIdx.x < n_rows) {
        const int r = threadIdx.x;
        float M = -INFINITY, ls = 0.0f;
        for (int w2 = 0; w2 < kWarps; ++w2) M = fmaxf(M, ml_s[(w2 * 4 + r) * 2]);
        for (int w2 = 0; w2 < kWarps; ++w2) {
            const float mw = ml_s[(w2 * 4 + r) * 2];
            ls += ml_s[(w2 * 4 + r) * 2 + 1] * (mw == -INFINITY ? 0.0f : ex2(mw - M));       // (no maximum: 0, or NaN where NaN is all that was seen)
        }
        *reinterpret_cast<float2*>(A.part_ml + 2 * (base + r)) = make_float2(M, ls);
    }
}

// grid = (row blocks of all sequences, KV heads); 128 threads have a quad of channels of a
// row each, with many pieces several such teams share them.
constexpr int kTeam = kRows * kD / 4;
__global__ void __launch_bounds__(8 * kTeam)
paged_decode_merge_kernel(PagedAttnArgs A, int blocks_per_seq, int gps) {
    __shared__ float4 out_s[7][kTeam];
    __shared__ float2 ml_s[7][kTeam];
    stream_order();
    settle_args(A);
    const kivi_paged_layer& L = A.L;
    const int n_rep = A.n_rep, h = blockIdx.y, team = threadIdx.x / kTeam, teams = blockDim.x / kTeam, me = threadIdx.x % kTeam;
    const int s = (int)blockIdx.x / blocks_per_seq, row_first = ((int)blockIdx.x - s * blocks_per_seq) * kRows;
    PagedSeq q;
    load_seq(L, A.b, s, q);
    if (row_first >= q.n * n_rep) return;
    const int r = me >> 5, d = (me & 31) * 4, row = row_first + r;
    const int n_groups = min(quant_of(q.held + q.n, kG, L.residual_cap), q.held) / kG;
    const int n = row < q.n * n_rep ? 1 + (n_groups + gps - 1) / gps : 0;
    const int64_t base = ((int64_t)blockIdx.x * L.num_kv_heads + h) * A.pieces;
    float M = -INFINITY, sum = 0.0f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float2 ml, float4 v) {
        if (ml.x == -INFINITY && ml.y == 0.0f) return;
        const float top = fmaxf(M, ml.x), w0 = ex2(M - top), w1 = ex2(ml.x - top);
        M = top;
        sum = fmaf(w0, sum, w1 * ml.y);
        a.x = fmaf(w0, a.x, w1 * v.x); a.y = fmaf(w0, a.y, w1 * v.y); a.z = fmaf(w0, a.z, w1 * v.z); a.w = fmaf(w0, a.w, w1 * v.w);
    };
#pragma unroll 4
    for (int p = team; p < n; p += teams)
        add(*reinterpret_cast<const float2*>(A.part_ml + 2 * ((base + p) * kRows + r)), *reinterpret_cast<const float4*>(A.part_o + ((base + p) * kRows + r) * kD + d));
    if (teams > 1) {
        if (team) { out_s[team - 1][me] = a; ml_s[team - 1][me] = make_float2(M, sum); }
        __syncthreads();
        if (team) return;
        for (int t = 0; t < teams - 1; ++t) add(ml_s[t][me], out_s[t][me]);
    }
    if (n == 0) return;
    const float inv = 1.0f / sum;
    const int64_t at = ((int64_t)q.row0 + row / n_rep) * A.out.row_stride + (int64_t)(h * n_rep + row % n_rep) * A.out.head_stride;
    store_quad(A.out.data, A.out_dtype, at + d, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
}

constexpr size_t kSmemBytes = (size_t)kWarps * (kStages * kStageBytes + kScratchBytes) + kWarps * kStages * 8 + kWarps * 4 * 2 * 4 + kRows * kD * 4;
static_assert(kWarps * kStages * kStageBytes >= 2 * kG * kD * 4, "the window's CTA keeps the tokens of one group there");

}  // namespace

bool paged_decode_serves(const kivi_paged_layer* L, int q_dtype, int64_t max_rows) {
    // Three blocks of rows (3 tokens, 4 query heads per KV head, 8 KV heads), here and with 256 rows on the
    // 5th-generation tensor cores: 16 sequences x 4k 80 and 80 us, 64 x 2k 176 and 201, 1 x 32k 33 and 52;
    // four blocks: 103 and 83, 229 and 203, 46 and 52.
    // (bf16 windows with fp32 queries and the other way round go to the general kernel)
    return L->head_dim == kD && L->group_size == kG && q_dtype == L->res_dtype && max_rows <= 12;
}

// Row blocks of a sequence, packed groups a piece and pieces, in whole rounds of the CTA's
// warps (eight groups, 1.4 us).  Rounds of CTAs on the GPU times rounds of a piece, two more
// for a CTA's start and end, and what a piece costs in the fold; but no piece above a sixth
// of a GPU's share where that is long, since sequences shorter than the longest leave theirs
// unused (64 ragged sequences up to 32k: 280 us).
void paged_decode_plan(const kivi_paged_layer* L, const kivi_paged_batch* b, int n_rep, int* blocks_per_seq, int* gps, int* pieces) {
    constexpr int kRound = kWarps * kGPS;
    *blocks_per_seq = (b->max_new * n_rep + kRows - 1) / kRows;
    const int64_t groups = quant_of(b->max_len, kG, L->residual_cap) / kG, units = (int64_t)b->num_seqs * *blocks_per_seq * L->num_kv_heads;
    const int64_t slots = 3 * (int64_t)num_sms(), share = (units * groups + slots - 1) / slots;
    const int64_t longest = share / 6 > 96 ? share / 6 : 96;
    double best = 1e30;
    int64_t per = kRound;
    for (int64_t k = 1; k * kRound < longest + kRound && k <= 4096; ++k) {
        const int64_t n = (groups + k * kRound - 1) / (k * kRound);
        if (n > 255 && k < 4096) continue;
        const double cost = (double)((units * n + slots - 1) / slots) * (double)(k + 2) + 0.05 * (double)n;
        if (cost < best) { best = cost; per = k * kRound; }
    }
    while ((groups + per - 1) / per > 255) per += kRound;
    *gps = (int)per;
    *pieces = 1 + (int)((groups + per - 1) / per);
}

int run_paged_decode(const PagedAttnArgs& a, int blocks_per_seq, int gps, cudaStream_t st) {
    auto* const kernel = a.q_dtype == KIVI_F32 ? paged_decode_kernel<float, true, false>
                       : a.b.max_new * a.n_rep == 1 ? paged_decode_kernel<__nv_bfloat16, false, true> : paged_decode_kernel<__nv_bfloat16, false, false>;
    KIVI_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes));
    const dim3 grid((unsigned)(a.b.num_seqs * blocks_per_seq), (unsigned)a.L.num_kv_heads, (unsigned)a.pieces);
    KIVI_CUDA_OK(launch(kernel, grid, kWarps * 32, kSmemBytes, st, true, a, blocks_per_seq, gps));
    const int teams = a.pieces > 32 ? 8 : a.pieces > 8 ? 4 : 1;
    KIVI_CUDA_OK(launch(paged_decode_merge_kernel, dim3(grid.x, grid.y), (unsigned)(kTeam * teams), 0, st, true, a, blocks_per_seq, gps));
    return KIVI_OK;
}

int paged_decode_fault_word(int* out) {
    KIVI_CUDA_OK(cudaMemcpyFromSymbol(out, g_fault, sizeof(int)));
    return KIVI_OK;
}
int paged_decode_fault_clear() {
    const int zero = 0;
    KIVI_CUDA_OK(cudaMemcpyToSymbol(g_fault, &zero, sizeof(int)));
    return KIVI_OK;
}

}  // namespace kivi
