// Attention of a few rows over a paged cache in 8 bits: head_dim 64 and 128, blocks of whole
// 32 tokens, queries of the window's type.
//
//   S = Q K^T,  P = 2^(rules(S) - m),  O = O + P V,  out = O / sum P
//
// by mma.sync m16n8k16 for sixteen rows ((new token, query head) pairs of one sequence and
// KV head), 32 tokens of a page to a warp at a time.  What bounds it is the page's bytes:
// a 32-token tile is 4 KB of keys and 4 KB of values (head_dim 128), 128 conversions
// and 64 MMAs of a warp (twice the MMAs for fp32 rows), a quarter of the time its bytes take.
//
// Work is dealt out evenly whatever the sequences' lengths: the tiles of all (sequence, KV
// head, block of rows) units lie one after the other, the window and the step's own tokens
// as a few tiles more, and CTA c has positions c per .. (c + 1) per - 1 of that line,
// with `per` from the lengths in device memory.  A unit in one CTA is finished there; of the others
// a CTA has two at most, its first and its last, whose partials it leaves in slots 2c and
// 2c + 1 for a second kernel.  Nothing depends on the order in which CTAs run.
//
// A warp has a ring of stages that bulk copies fill, its lane issues them; the four warps
// take tiles in turn and meet at a unit's end.
//
// Numbers: e4m3 codes are exact as fp16.  A row of bf16 queries is exact as fp16 after a power
// of two, but for what is below 2^-27 of its largest; fp32 rows are two fp16 numbers (22 bits).  A block's key scale
// multiplies the scores, its value scale the weights, which are fp16 (bf16 rows: rounded at
// 2^-12 of themselves, where the output is rounded at 2^-9) or two of them, less the power of
// two of the largest value scale so far.  Window and own tokens are contracted as bf16 numbers, exact for
// bf16 rows (weights at 2^-9 there: bf16 reaches as far as the values do); fp32 ones as three, the six products that matter.  Sums are fp32.
#include "async_copy.cuh"
#include "paged8_attention.cuh"

#include <type_traits>

namespace kivi {
namespace {

__device__ int g_fault = 0;

constexpr int kWarps = 4, kThreads = kWarps * 32, kStages = 2;
constexpr int kRows = 16, kTile = 32;                    // rows of a unit, tokens of a tile
constexpr int kPerSm = 2;                                // CTAs
constexpr int kLeast = 8;                                // tiles of a CTA
constexpr float kGrowth = 8.0f;                          // weights up to 2^8 are let stand before the maximum moves
constexpr int kHeadroom = 5;                             // value scales are brought to 2^5 .. 2^6: weights stay below 2^14

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
    uint32_t y;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
    return y;
}
__device__ __forceinline__ uint32_t bf16x2_of(float lo, float hi) {
    uint32_t y;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
    return y;
}
__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// what is left of two numbers after their first term
__device__ __forceinline__ uint32_t half2_rest(float lo, float hi, uint32_t first) { return half2_of(lo - half_lo(first), hi - half_hi(first)); }
// two numbers as N bf16 terms
template <int N> __device__ __forceinline__ void bf16_terms(float lo, float hi, uint32_t (&w)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        w[i] = bf16x2_of(lo, hi);
        lo -= bf_lo(w[i]); hi -= bf_hi(w[i]);
    }
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void ldmatrix_trans(uint32_t at, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ float pow2i(int s) { return __uint_as_float((uint32_t)(127 + max(-126, min(127, s))) << 23); }

// ---- the line of work ---------------------------------------------------------------
struct SeqWork {
    PagedSeq q;
    int total, inside, prefix, rows, blocks;             // rows of the step, blocks of kRows of them
    int tiles, tail;                                     // of a unit: packed tiles, and positions that the other tokens count for
    Span span;
    __device__ __forceinline__ int cost() const { return tiles + tail; }
};
template <bool F32>
__device__ __forceinline__ bool seq_work(const Paged8Attn& A, int s, SeqWork& w) {
    const kivi_paged8_layer& L = A.L;
    if (!load_seq(L, A.b, s, w.q) || w.q.n == 0) { w.blocks = w.tiles = w.tail = 0; return false; }
    w.rows = w.q.n * A.n_rep;
    w.blocks = (w.rows + kRows - 1) / kRows;
    w.total = w.q.held + w.q.n;
    w.inside = min(quant_of(w.total, L.group_size, L.residual_cap), w.q.held);
    w.prefix = prefix_of(A.rules, s, w.total);
    w.span = span_of(kTile, w.total, w.q.held, w.total - 1, A.rules.window, w.prefix);
    const int packed = (w.inside + kTile - 1) / kTile;
    w.tiles = min(w.span.n1, packed) + max(0, packed - (w.span.n1 + w.span.gap));
    w.tail = 1 + (w.total - w.inside) * (F32 ? 4 : 2) / kTile;
    return true;
}

struct Line { int64_t cost; int64_t before; int first; };         // all positions; those before sequence `first`, which has position `at`

// Called by the whole CTA: the line's length, and which sequence has position at(length).
template <bool F32, typename At>
__device__ __forceinline__ Line find_line(const Paged8Attn& A, int64_t* scratch /* [kWarps + 2] shared */, const At& at) {
    const int n = A.b.num_seqs, H = A.L.num_kv_heads, per = (n + kThreads - 1) / kThreads;
    int64_t mine = 0;
    for (int i = 0; i < per; ++i) {
        const int s = threadIdx.x * per + i;
        SeqWork w;
        if (s < n && seq_work<F32>(A, s, w)) mine += (int64_t)H * w.blocks * w.cost();
    }
    // sums of what comes before each thread's sequences
    int64_t sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int64_t up = __shfl_up_sync(0xffffffffu, sum, o);
        if ((threadIdx.x & 31) >= o) sum += up;
    }
    if ((threadIdx.x & 31) == 31) scratch[threadIdx.x >> 5] = sum;
    if (threadIdx.x == 0) scratch[kWarps] = -1;
    __syncthreads();
    int64_t before = sum - mine, total = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
        if (i < (int)threadIdx.x >> 5) before += scratch[i];
        total += scratch[i];
    }
    const int64_t want = at(total);
    if (want >= before && want < before + mine) {
        for (int i = 0; i < per; ++i) {
            const int s = threadIdx.x * per + i;
            SeqWork w;
            const int64_t c = s < n && seq_work<F32>(A, s, w) ? (int64_t)H * w.blocks * w.cost() : 0;
            if (want < before + c) { scratch[kWarps] = s; scratch[kWarps + 1] = before; break; }
            before += c;
        }
    }
    __syncthreads();
    return {total, scratch[kWarps + 1], (int)scratch[kWarps]};
}
__host__ __device__ __forceinline__ int64_t per_cta(int64_t cost, int ctas) {
    const int64_t per = (cost + ctas - 1) / ctas;
    return per < kLeast ? kLeast : per;
}

// The CTA's segments, one after the other.
template <bool F32>
struct Walk {
    SeqWork w;
    int64_t at, end, off;                                // next position, the CTA's end, the sequence's first position
    int s, h, rb;                                        // of the segment
    int64_t unit;                                        // its unit's first position
    int a, b;                                            // its positions within the unit

    __device__ __forceinline__ bool next(const Paged8Attn& A) {
        while (at < end) {
            const int64_t size = (int64_t)A.L.num_kv_heads * w.blocks * w.cost();
            if (at >= off + size) {
                off += size;
                if (++s >= A.b.num_seqs) return false;
                seq_work<F32>(A, s, w);
                continue;
            }
            const int c = w.cost();
            const int64_t u = (at - off) / c;
            h = (int)(u / w.blocks); rb = (int)(u % w.blocks);
            unit = off + u * c;
            a = (int)(at - unit);
            b = (int)min((int64_t)c, end - unit);
            at = unit + b;
            if (a <= w.tiles) return true;               // (behind the tail's first position there is nothing to do)
        }
        return false;
    }
    __device__ __forceinline__ int tiles_end() const { return min(b, w.tiles); }
    __device__ __forceinline__ bool has_tail() const { return a <= w.tiles && w.tiles < b; }
};

template <int D> struct Layout {
    static constexpr int kPart = kTile * D;              // bytes of a tile's keys, or values
    static constexpr int kQ = D + 4, kO = D + 8;         // floats of a row
    static constexpr int kVStage = 16 * D * 2;           // bytes: values of sixteen tokens as bf16
    static constexpr int ring = 0, fold = ring + kWarps * kStages * 2 * kPart;
    static constexpr int kFold = 2 * kRows * kO * 4 > kWarps * kVStage ? 2 * kRows * kO * 4 : kWarps * kVStage;
    static constexpr int q = fold + kFold, ml = q + kRows * kQ * 4, scratch = ml + 2 * kRows * 8, bars = scratch + (kWarps + 2) * 8;
    static constexpr int bytes = bars + kWarps * kStages * 8;
};

template <int D, bool F32, bool RULES>
__global__ void __launch_bounds__(kThreads, kPerSm)
paged8_decode_kernel(Paged8Attn A) {
    using S = Layout<D>;
    constexpr int kSteps = D / 16, kChan = D / 4;        // MMAs along the channels; channels of a lane's keys
    constexpr int kTerms = F32 ? 2 : 1, kBf = F32 ? 3 : 1;
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), g = lane >> 2, t = lane & 3;
    stream_order();
    settle_args(A);
    cudaTriggerProgrammaticLaunchCompletion();           // (the fold's few blocks wait for this kernel's end)
    const kivi_paged8_layer& L = A.L;
    const int G = L.group_size, R = L.residual_cap, H = L.num_kv_heads, n_rep = A.n_rep, window = A.rules.window;
    if (blockIdx.x == 0) report_left_out(L, A.b, &g_fault);
    float* const q_s = reinterpret_cast<float*>(smem + S::q);
    float* const fold_s = reinterpret_cast<float*>(smem + S::fold);
    float* const ml_s = reinterpret_cast<float*>(smem + S::ml);
    const uint32_t ring = smem_u32(smem + S::ring) + warp * (kStages * 2 * S::kPart), v_stage = smem_u32(smem + S::fold) + warp * S::kVStage;
    const uint32_t bars = smem_u32(smem + S::bars) + warp * (kStages * 8);
    if (lane == 0) {
        for (int i = 0; i < kStages; ++i) mbar_init(bars + 8 * i, 1);
        mbar_init_fence();
    }
    const Line line = find_line<F32>(A, reinterpret_cast<int64_t*>(smem + S::scratch), [&](int64_t cost) { return per_cta(cost, gridDim.x) * blockIdx.x; });
    if (line.first < 0) return;
    const int64_t per = per_cta(line.cost, gridDim.x);
    Walk<F32> walk, ahead;                               // what is computed, and what is copied
    walk.s = line.first; walk.off = line.before;
    walk.at = per * blockIdx.x; walk.end = min(walk.at + per, line.cost);
    seq_work<F32>(A, walk.s, walk.w);
    ahead = walk;
    const uint64_t policy = l2_stream_policy();

    // ---- copies: the warp's next tile into a stage; its scales come along in registers
    bool more = ahead.next(A);
    int av = more ? ahead.a + warp : 0, issued = 0;
    float2 scales[kStages];
#pragma unroll
    for (int i = 0; i < kStages; ++i) scales[i] = make_float2(0.f, 0.f);
    auto settle_next = [&] {                             // on to the warp's next tile
        while (more && av >= ahead.tiles_end()) {
            more = ahead.next(A);
            if (more) av = ahead.a + warp;
        }
    };
    settle_next();
    int next_page = 0;
    auto look_up = [&] { if (more) next_page = ahead.w.q.pages[ahead.w.span.tile(av) * kTile / L.page_tokens]; };
    look_up();
    auto issue = [&](int stage, float2& sc) {
        if (!more) return;
        const int t0 = ahead.w.span.tile(av) * kTile, in_page = t0 % L.page_tokens;
        const bool there = (unsigned)next_page < (unsigned)L.num_pages;
        if (!there) atomicOr(&g_fault, kPagedFault);
        const int64_t unit = (int64_t)(there ? next_page : 0) * H + ahead.h;
        const int64_t at = (unit * L.page_tokens + in_page) * D, f = unit * (L.page_tokens / G) + in_page / G;
        if (lane == 0) {
            const uint32_t to = ring + stage * (2 * S::kPart), b = bars + 8 * stage;
            mbar_expect_tx(b, 2 * S::kPart);
            bulk_g2s(to, L.k_codes + at, S::kPart, b, policy);
            bulk_g2s(to + S::kPart, L.v_codes + at, S::kPart, b, policy);
        }
        sc = make_float2(L.k_scales[f], L.v_scales[f]);
        ++issued;
        av += kWarps;
        settle_next();
        look_up();
    };
#pragma unroll
    for (int i = 0; i < kStages; ++i) issue(i, scales[i]);
    int taken = 0;
    bool ok = true;

    while (walk.next(A)) {
        const PagedSeq& q = walk.w.q;
        const int h = walk.h, row_first = walk.rb * kRows, n_rows = min(kRows, walk.w.rows - row_first), inside = walk.w.inside, prefix = walk.w.prefix;
        // ---- the unit's queries
        __syncthreads();                                 // (the unit before is folded)
        for (int i = tid; i < kRows * (D / 4); i += kThreads) {
            const int r = i / (D / 4), d = 4 * (i % (D / 4)), row = row_first + r;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < n_rows) x = load4_as(A.q, F32 ? KIVI_F32 : KIVI_BF16, (int64_t)q.row0 + row / n_rep, h * n_rep + row % n_rep, d, A.vec != 0);
            *reinterpret_cast<float4*>(q_s + r * S::kQ + d) = x;
        }
        __syncthreads();
        // A lane has channels kChan t .. of rows g and g + 8, four to an MMA; keys lie the same way.
        uint32_t qa[kTerms][kSteps][4];
        float unscale[2];                                // of a contracted score, and to powers of two where nothing else is done to it
        {
            int shift[2];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                float top = 0.0f;
                for (int c = 0; c < kChan; c += 4) {
                    const float4 x = *reinterpret_cast<const float4*>(q_s + (g + 8 * hf) * S::kQ + kChan * t + c);
                    top = fmaxf(fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(x.z), fabsf(x.w)));
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int e = (int)(__float_as_uint(top) >> 23);
                shift[hf] = e == 0 || e == 255 ? 0 : max(-110, min(110, 127 + 13 - e));       // largest to 2^13 .. 2^14
                unscale[hf] = A.scale * pow2i(-shift[hf]) * (RULES ? 1.0f : 1.4426950408889634f);
            }
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const float f = pow2i(shift[hf]);
                    float4 x = *reinterpret_cast<const float4*>(q_s + (g + 8 * hf) * S::kQ + kChan * t + 4 * i);
                    x = make_float4(x.x * f, x.y * f, x.z * f, x.w * f);
                    qa[0][i][hf] = half2_of(x.x, x.y);
                    qa[0][i][2 + hf] = half2_of(x.z, x.w);
                    if constexpr (F32) {
                        qa[kTerms - 1][i][hf] = half2_rest(x.x, x.y, qa[0][i][hf]);
                        qa[kTerms - 1][i][2 + hf] = half2_rest(x.z, x.w, qa[0][i][2 + hf]);
                    }
                }
        }
        int place[2], from[2];
        float slope[2];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            const int r = g + 8 * hf, row = row_first + r;
            // (a row that is not there sees what the first one sees, and is not written)
            place[hf] = q.held + (r < n_rows ? row : row_first) / n_rep;
            from[hf] = window_from(place[hf], window);
            slope[hf] = RULES && A.rules.slopes && r < n_rows ? A.rules.slopes[h * n_rep + row % n_rep] : 0.0f;
        }
        const int from_most = window_from(q.held + (row_first + n_rows - 1) / n_rep, window);
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, o[D / 8][4];
        int v_exp = -1000;                               // O is 2^(kHeadroom - v_exp) times what it stands for
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[c][e] = 0.0f;
        auto rescale = [&](float f0, float f1) {
#pragma unroll
            for (int c = 0; c < D / 8; ++c) { o[c][0] *= f0; o[c][1] *= f0; o[c][2] *= f1; o[c][3] *= f1; }
        };
        auto reach = [&](int e) {                        // value scales up to 2^(e + 1)
            if (e > v_exp) {
                if (v_exp != -1000) { const float f = pow2i(v_exp - e); rescale(f, f); }
                v_exp = e;
            }
        };
        // Scores x[n] (tokens t0 + 8 n + 2 t and the next, rows g and g + 8), in powers of two or (RULES) as contracted
        // and scaled, to weights.  hidden(token, hf): the row does not see it.
        auto weights = [&](auto& x, int t0, bool some_hidden, auto&& hidden) {
            constexpr int N = sizeof(x) / sizeof(x[0]);
            if constexpr (RULES) {
                const bool capped = A.rules.softcap > 0.0f;
                const float cap = A.rules.softcap, inv_cap = capped ? 2.0f * 1.4426950408889634f / cap : 0.0f;
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float y = x[n][e];
                        // tanh(z) = 1 - 2 / (1 + e^(2z))
                        if (capped) y = F32 ? cap * tanhf(y / cap) : cap - __fdividef(2.0f * cap, 1.0f + ex2(y * inv_cap > 120.0f ? 120.0f : y * inv_cap));
                        y = fmaf(slope[e >> 1], (float)(t0 + 8 * n + 2 * t + (e & 1) - place[e >> 1]), y);
                        x[n][e] = y * 1.4426950408889634f;
                    }
            }
            if (some_hidden) {
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (hidden(t0 + 8 * n + 2 * t + (e & 1), e >> 1)) x[n][e] = -INFINITY;
            }
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int n = 0; n < N; ++n) {
                top[0] = fmaxf(top[0], fmaxf(x[n][0], x[n][1]));
                top[1] = fmaxf(top[1], fmaxf(x[n][2], x[n][3]));
            }
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                top[hf] = fmaxf(top[hf], __shfl_xor_sync(0xffffffffu, top[hf], 1));
                top[hf] = fmaxf(top[hf], __shfl_xor_sync(0xffffffffu, top[hf], 2));
            }
            if (__any_sync(0xffffffffu, top[0] > m[0] + kGrowth || top[1] > m[1] + kGrowth)) {
                float f[2];
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const float m_new = fmaxf(m[hf], top[hf]);
                    f[hf] = m[hf] == -INFINITY ? 0.0f : ex2(m[hf] - m_new);
                    m[hf] = m_new;
                    l[hf] *= f[hf];
                }
                rescale(f[0], f[1]);
            }
            const float base[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[n][e] = F32 ? exp2f(x[n][e] - base[e >> 1]) : ex2(x[n][e] - base[e >> 1]);
#pragma unroll
            for (int n = 0; n < N; ++n) { l[0] += x[n][0] + x[n][1]; l[1] += x[n][2] + x[n][3]; }
        };

        // ---- tiles of pages
        for (int v = walk.a + warp; v < walk.tiles_end(); v += kWarps) {
            const int stage = taken % kStages, t0 = walk.w.span.tile(v) * kTile;
            const float2 sc = stage ? scales[kStages - 1] : scales[0];
            static_assert(kStages == 2, "scales of a stage are picked by hand");
            if (ok && !mbar_wait(bars + 8 * stage, (uint32_t)(taken / kStages) & 1u)) { atomicOr(&g_fault, 1); ok = false; }
            ok = __all_sync(0xffffffffu, ok);
            const uint32_t keys = ring + stage * (2 * S::kPart), values = keys + S::kPart;
            float x[4][4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.0f;
#pragma unroll
                for (int p = 0; p < kChan / 16; ++p) {
                    const int piece = D == 128 ? (2 * t + p) ^ g : t ^ (g >> 1 & 3);
                    const uint4 k = lds128(keys + (8 * n + g) * D + 16 * piece);
                    const uint32_t w[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t b0 = e4m3x2_to_half2(w[i] & 0xffffu), b1 = e4m3x2_to_half2(w[i] >> 16);
#pragma unroll
                        for (int term = kTerms - 1; term >= 0; --term) mma_f16(x[n], qa[term][4 * p + i], b0, b1);
                    }
                }
            }
            const float u0 = unscale[0] * sc.x, u1 = unscale[1] * sc.x;
#pragma unroll
            for (int n = 0; n < 4; ++n) { x[n][0] *= u0; x[n][1] *= u0; x[n][2] *= u1; x[n][3] *= u1; }
            // (a page's tokens come before every row)
            const bool edge = t0 + kTile > inside || (t0 < from_most && t0 + kTile > prefix);
            weights(x, t0, edge, [&](int tok, int hf) { return tok >= inside || (tok < from[hf] && tok >= prefix); });
            const int e = (int)(__float_as_uint(sc.y) >> 23) - 127;
            reach(e);
            const float f = sc.y * pow2i(kHeadroom - v_exp);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                uint32_t pa[kTerms][4];
#pragma unroll
                for (int e2 = 0; e2 < 4; ++e2) {         // (row g, g + 8, then the next eight tokens)
                    const float lo = x[2 * i + (e2 >> 1)][2 * (e2 & 1)] * f, hi = x[2 * i + (e2 >> 1)][2 * (e2 & 1) + 1] * f;
                    pa[0][e2] = half2_of(lo, hi);
                    if constexpr (F32) pa[kTerms - 1][e2] = half2_rest(lo, hi, pa[0][e2]);
                }
#pragma unroll
                for (int e2 = 0; e2 < 2; ++e2) {
                    // (kept as they were rounded)
                    x[2 * i + e2][0] = __uint_as_float(pa[0][2 * e2]); x[2 * i + e2][1] = __uint_as_float(pa[0][2 * e2 + 1]);
                    if constexpr (F32) { x[2 * i + e2][2] = __uint_as_float(pa[kTerms - 1][2 * e2]); x[2 * i + e2][3] = __uint_as_float(pa[kTerms - 1][2 * e2 + 1]); }
                }
            }
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                const uint2 w = lds64(values + (8 * c + g) * kTile + 8 * t);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t y = i ? w.y : w.x, b0 = e4m3x2_to_half2(y & 0xffffu), b1 = e4m3x2_to_half2(y >> 16);
#pragma unroll
                    for (int term = kTerms - 1; term >= 0; --term) {
                        const uint32_t pa[4] = {__float_as_uint(x[2 * i][2 * term]), __float_as_uint(x[2 * i][2 * term + 1]),
                                                __float_as_uint(x[2 * i + 1][2 * term]), __float_as_uint(x[2 * i + 1][2 * term + 1])};
                        mma_f16(o[c], pa, b0, b1);
                    }
                }
            }
            __syncwarp();                                // (the stage has been read)
            ++taken;
            if (stage) issue(kStages - 1, scales[kStages - 1]);
            else issue(0, scales[0]);
        }

        // ---- the window and the step's own tokens, sixteen at a time
        if (walk.has_tail()) {
            using T = typename std::conditional<F32, float, __nv_bfloat16>::type;
            const T* const k_ring = reinterpret_cast<const T*>(L.k_res) + ((int64_t)q.slot * H + h) * R * D;
            const T* const v_ring = reinterpret_cast<const T*>(L.v_res) + ((int64_t)q.slot * H + h) * R * D;
            auto row_at = [&](int tok, bool of_keys) -> const T* {
                if (tok < q.held) return (of_keys ? k_ring : v_ring) + (int64_t)ring_slot(tok, 0, R) * D;
                const kivi_rows& r = of_keys ? A.k : A.v;
                return reinterpret_cast<const T*>(r.data) + ((int64_t)q.row0 + min(tok, walk.w.total - 1) - q.held) * r.row_stride + (int64_t)h * r.head_stride;
            };
            for (int t0 = inside + 16 * warp; t0 < walk.w.total; t0 += 16 * kWarps) {
                float x[2][4];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.0f;
                    const int tok = t0 + 8 * n + g;
                    const T* const from_row = row_at(tok, true) + kChan * t;
                    const bool vec = tok < q.held || A.vec;
                    float4 kx[kChan / 4];
#pragma unroll
                    for (int i = 0; i < kChan / 4; ++i) kx[i] = load4(from_row + 4 * i, vec);
#pragma unroll
                    for (int i = 0; i < kSteps; ++i) {
                        uint32_t qb[kBf][4], b0[kBf], b1[kBf];
                        bf16_terms(kx[i].x, kx[i].y, b0);
                        bf16_terms(kx[i].z, kx[i].w, b1);
#pragma unroll
                        for (int hf = 0; hf < 2; ++hf) {
                            const float4 y = *reinterpret_cast<const float4*>(q_s + (g + 8 * hf) * S::kQ + kChan * t + 4 * i);
                            uint32_t lo[kBf], hi[kBf];
                            bf16_terms(y.x, y.y, lo);
                            bf16_terms(y.z, y.w, hi);
#pragma unroll
                            for (int term = 0; term < kBf; ++term) { qb[term][hf] = lo[term]; qb[term][2 + hf] = hi[term]; }
                        }
#pragma unroll
                        for (int sum = kBf - 1; sum >= 0; --sum)                 // products of like size together, the small ones first
#pragma unroll
                            for (int a = 0; a <= sum; ++a) mma_bf16(x[n], qb[a], b0[sum - a], b1[sum - a]);
                    }
                }
                const float u = A.scale * (RULES ? 1.0f : 1.4426950408889634f);
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[n][e] *= u;
                auto hidden = [&](int tok, int hf) { return tok >= walk.w.total || ((tok > place[hf] || tok < from[hf]) && tok >= prefix); };
                weights(x, t0, true, hidden);
                reach(0);
                const float f = pow2i(kHeadroom - v_exp);
                uint32_t pb[kBf][4];
#pragma unroll
                for (int e2 = 0; e2 < 4; ++e2) {
                    uint32_t terms[kBf];
                    bf16_terms(x[e2 >> 1][2 * (e2 & 1)] * f, x[e2 >> 1][2 * (e2 & 1) + 1] * f, terms);
#pragma unroll
                    for (int term = 0; term < kBf; ++term) pb[term][e2] = terms[term];
                }
                // Values go through shared memory, a term at a time.  One that is not finite would reach rows that do not
                // see it through weights of 0: it is left out there, and added to the rows that do.
                bool odd = false;
#pragma unroll
                for (int term = 0; term < kBf; ++term) {
                    __syncwarp();
                    for (int i = lane; i < 16 * (D / 8); i += 32) {
                        const int j = i / (D / 8), p = i % (D / 8), tok = t0 + j;
                        const T* const from_row = row_at(tok, false) + 8 * p;
                        const bool vec = tok < q.held || A.vec;
                        float4 y[2] = {load4(from_row, vec), load4(from_row + 4, vec)};
                        uint32_t w[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            float a = k & 1 ? y[k >> 1].z : y[k >> 1].x, b = k & 1 ? y[k >> 1].w : y[k >> 1].y;
                            if (!(fabsf(a) <= 3.4028234e38f)) { odd = true; a = 0.0f; }
                            if (!(fabsf(b) <= 3.4028234e38f)) { odd = true; b = 0.0f; }
                            uint32_t terms[kBf];
                            bf16_terms(a, b, terms);
                            w[k] = tok < walk.w.total ? terms[term] : 0u;
                        }
                        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(v_stage + j * (2 * D) + ((p ^ (j & 7)) << 4)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                    }
                    __syncwarp();
#pragma unroll
                    for (int c = 0; c < D / 8; c += 2) {
                        uint32_t r[4];
                        const int j = (lane & 7) + (lane & 8), p = c + (lane >> 4);
                        ldmatrix_trans(v_stage + j * (2 * D) + ((p ^ (j & 7)) << 4), r);
#pragma unroll
                        for (int a = kBf - 1 - term; a >= 0; --a) {
                            mma_bf16(o[c], pb[a], r[0], r[1]);
                            mma_bf16(o[c + 1], pb[a], r[2], r[3]);
                        }
                    }
                }
                if (__any_sync(0xffffffffu, odd)) {
                    for (int j = 0; j < 16; ++j) {
                        const int tok = t0 + j;
                        if (tok >= walk.w.total) break;
                        const T* const from_row = row_at(tok, false);
#pragma unroll
                        for (int c = 0; c < D / 8; ++c)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float y = (float)from_row[8 * c + 2 * t + (e & 1)];
                                if (!(fabsf(y) <= 3.4028234e38f) && !hidden(tok, e >> 1)) o[c][e] += y;
                            }
                    }
                }
            }
        }

        // ---- the warps meet
        {
            const float f = pow2i(v_exp == -1000 ? 0 : v_exp - kHeadroom);
            rescale(f, f);
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 1);
                l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 2);
            }
            auto leave = [&](int buf) {
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const int r = g + 8 * hf;
                    if (r >= n_rows) continue;
                    if (t == 0) *reinterpret_cast<float2*>(ml_s + (buf * kRows + r) * 2) = make_float2(m[hf], l[hf]);
#pragma unroll
                    for (int c = 0; c < D / 8; ++c)
                        *reinterpret_cast<float2*>(fold_s + (buf * kRows + r) * S::kO + 8 * c + 2 * t) = make_float2(o[c][2 * hf], o[c][2 * hf + 1]);
                }
            };
            auto take = [&](int buf) {
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const int r = g + 8 * hf;
                    if (r >= n_rows) continue;
                    const float2 ml = *reinterpret_cast<const float2*>(ml_s + (buf * kRows + r) * 2);
                    const float M = fmaxf(m[hf], ml.x), b = M == -INFINITY ? 0.0f : M;
                    const float mine = F32 ? exp2f(m[hf] - b) : ex2(m[hf] - b), other = F32 ? exp2f(ml.x - b) : ex2(ml.x - b);
                    m[hf] = M;
                    l[hf] = l[hf] * mine + ml.y * other;
#pragma unroll
                    for (int c = 0; c < D / 8; ++c) {
                        const float2 y = *reinterpret_cast<const float2*>(fold_s + (buf * kRows + r) * S::kO + 8 * c + 2 * t);
                        o[c][2 * hf] = fmaf(y.x, other, o[c][2 * hf] * mine);
                        o[c][2 * hf + 1] = fmaf(y.y, other, o[c][2 * hf + 1] * mine);
                    }
                }
            };
            __syncthreads();                             // (values of the tail have been read)
            if (warp >= 2) leave(warp - 2);
            __syncthreads();
            if (warp < 2) take(warp);
            __syncthreads();
            if (warp == 1) leave(0);
            __syncthreads();
            if (warp == 0) {
                take(0);
                // the CTAs that have something of the unit
                const int64_t c0 = walk.unit / per, c1 = (walk.unit + walk.w.tiles) / per;
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const int r = g + 8 * hf, row = row_first + r;
                    if (r >= n_rows) continue;
                    if (c0 == c1) {
                        const float inv = 1.0f / l[hf];  // (a row sees itself: l > 0)
                        const int64_t at = ((int64_t)q.row0 + row / n_rep) * A.out.row_stride + (int64_t)(h * n_rep + row % n_rep) * A.out.head_stride;
#pragma unroll
                        for (int c = 0; c < D / 8; ++c) {
                            const int64_t i = at + 8 * c + 2 * t;
                            const float a = o[c][2 * hf] * inv, b = o[c][2 * hf + 1] * inv;
                            if (A.out_dtype == KIVI_BF16) {
                                __nv_bfloat16* to = reinterpret_cast<__nv_bfloat16*>(A.out.data) + i;
                                if ((reinterpret_cast<uintptr_t>(to) & 3u) == 0) *reinterpret_cast<uint32_t*>(to) = bf16x2_of(a, b);
                                else { to[0] = __float2bfloat16_rn(a); to[1] = __float2bfloat16_rn(b); }
                            } else {
                                float* to = reinterpret_cast<float*>(A.out.data) + i;
                                to[0] = a; to[1] = b;
                            }
                        }
                    } else {
                        const int64_t slot = 2 * (int64_t)blockIdx.x + (c0 == (int64_t)blockIdx.x ? 1 : 0), part = slot * kRows + r;
                        if (t == 0) *reinterpret_cast<float2*>(A.part_ml + 2 * part) = make_float2(m[hf], l[hf]);
#pragma unroll
                        for (int c = 0; c < D / 8; ++c) *reinterpret_cast<float2*>(A.part_o + part * D + 8 * c + 2 * t) = make_float2(o[c][2 * hf], o[c][2 * hf + 1]);
                    }
                }
            }
        }
    }
    // (a stage that a wait has given up on is not left to the next block's shared memory)
    for (; taken < issued; ++taken) mbar_wait(bars + 8 * (taken % kStages), (uint32_t)(taken / kStages) & 1u);
}

// Folds the units that lie across a CTA's end.  Block c has the unit that position c per lies in, if it is the first
// such end there; a thread a quad of channels of a row.
template <bool F32>
__global__ void __launch_bounds__(kThreads)
paged8_fold_kernel(Paged8Attn A, int ctas) {
    __shared__ int64_t scratch[kWarps + 2];
    stream_order();
    settle_args(A);
    const int c = blockIdx.x + 1, D = A.L.head_dim, n_rep = A.n_rep;
    const Line line = find_line<F32>(A, scratch, [&](int64_t cost) { return per_cta(cost, ctas) * c; });
    if (line.first < 0) return;
    const int64_t per = per_cta(line.cost, ctas), at = per * c;
    SeqWork w;
    seq_work<F32>(A, line.first, w);
    const int64_t u = (at - line.before) / w.cost(), unit = line.before + u * w.cost();
    const int64_t c0 = unit / per, c1 = (unit + w.tiles) / per;
    if (unit == at || c0 != c - 1 || c1 == c0) return;
    const int h = (int)(u / w.blocks), row_first = (int)(u % w.blocks) * kRows, n_rows = min(kRows, w.rows - row_first), quads = D / 4;
    for (int i = threadIdx.x; i < n_rows * quads; i += kThreads) {
        const int r = i / quads, d = 4 * (i % quads);
        auto part = [&](int64_t k) { return (2 * k + (k == c0 ? 1 : 0)) * kRows + r; };
        float M = -INFINITY, sum = 0.0f;
#pragma unroll 4
        for (int64_t k = c0; k <= c1; ++k) M = fmaxf(M, A.part_ml[2 * part(k)]);
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int64_t k = c0; k <= c1; ++k) {
            const float2 ml = *reinterpret_cast<const float2*>(A.part_ml + 2 * part(k));
            const float4 v = *reinterpret_cast<const float4*>(A.part_o + part(k) * D + d);
            const float f = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - M);         // (nothing of it is seen: O is 0)
            sum = fmaf(f, ml.y, sum);
            a.x = fmaf(f, v.x, a.x); a.y = fmaf(f, v.y, a.y); a.z = fmaf(f, v.z, a.z); a.w = fmaf(f, v.w, a.w);
        }
        const float inv = 1.0f / sum;
        const int row = row_first + r;
        const int64_t to = ((int64_t)w.q.row0 + row / n_rep) * A.out.row_stride + (int64_t)(h * n_rep + row % n_rep) * A.out.head_stride;
        store_quad(A.out.data, A.out_dtype, to + d, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
    }
}

template <int D, bool F32, bool RULES>
int go(const Paged8Attn& a, int ctas, cudaStream_t st) {
    auto* const kernel = paged8_decode_kernel<D, F32, RULES>;
    KIVI_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::bytes));
    KIVI_CUDA_OK(launch(kernel, dim3((unsigned)ctas), kThreads, Layout<D>::bytes, st, true, a));
    KIVI_CUDA_OK(launch(paged8_fold_kernel<F32>, dim3((unsigned)(ctas - 1)), kThreads, 0, st, true, a, ctas));
    return KIVI_OK;
}

}  // namespace

bool paged8_decode_serves(const kivi_paged8_layer* L, int q_dtype, int64_t max_rows) {
    return (L->head_dim == 64 || L->head_dim == 128) && L->group_size % 32 == 0 && q_dtype == L->res_dtype && max_rows <= 64;
}
int paged8_decode_ctas() { return kPerSm * num_sms(); }
size_t paged8_decode_parts() { return (size_t)paged8_decode_ctas() * 2 * kRows; }          // rows of partials

int run_paged8_decode(const Paged8Attn& a, cudaStream_t st) {
    const bool f32 = a.q_dtype == KIVI_F32, rules = a.rules.softcap > 0.0f || a.rules.slopes != nullptr;
    const int n = paged8_decode_ctas();
    if (a.L.head_dim == 64) return f32 ? (rules ? go<64, true, true>(a, n, st) : go<64, true, false>(a, n, st)) : (rules ? go<64, false, true>(a, n, st) : go<64, false, false>(a, n, st));
    return f32 ? (rules ? go<128, true, true>(a, n, st) : go<128, true, false>(a, n, st)) : (rules ? go<128, false, true>(a, n, st) : go<128, false, false>(a, n, st));
}

int paged8_decode_fault_word(int* out) {
    KIVI_CUDA_OK(cudaMemcpyFromSymbol(out, g_fault, sizeof(int)));
    return KIVI_OK;
}
int paged8_decode_fault_clear() {
    const int zero = 0;
    KIVI_CUDA_OK(cudaMemcpyToSymbol(g_fault, &zero, sizeof(int)));
    return KIVI_OK;
}

}  // namespace kivi
