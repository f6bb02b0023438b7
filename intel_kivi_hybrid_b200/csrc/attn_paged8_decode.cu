// Attention of a few rows over a paged cache in 8 bits, head_dim 64 and 128.
//
//   S = Q K^T,  P = 2^(rules(S) - m),  O = O + P V,  out = O / sum P
//
// Work is dealt out evenly whatever the sequences' lengths: the 32-token tiles of all (sequence, KV
// head, block of rows) units lie one after the other, the window and the step's own tokens
// as a few tiles more, and CTA c has positions c per .. (c + 1) per - 1 of that line,
// with `per` from the lengths in device memory.  A unit in one CTA is finished there; of the others
// a CTA has two at most, its first and its last, whose partials it leaves in slots 2c and
// 2c + 1 for a second kernel.  Nothing depends on the order in which CTAs run.
//
// paged8_decode_kernel: bf16, blocks of whole 32 tokens.  mma.sync m16n8k16, 32 tokens of a page to a warp
// at a time; tokens (and channels of V) are the sixteen rows of an MMA, the (new token, query head) pairs of one
// sequence and KV head its eight columns, up to three times eight to a unit: with the pairs as rows a single token of
// four heads took twice the MMAs and the registers (64 ragged sequences up to 32k 555 us, 385 to 406 now).  Weights change places with
// movmatrix in between.  A tile is 4 KB of keys and 4 KB of values (head_dim 128), 128 conversions and 32 MMAs of a warp,
// less than its bytes take.  A warp has a ring of stages that bulk copies fill, its first lane issues them; the warps take
// tiles in turn and meet at a unit's end.
//
// Numbers: e4m3 codes are exact as fp16.  A row of bf16 queries is exact as fp16 after a power
// of two, but for what is below 2^-27 of its largest.  A block's key scale multiplies the scores, its value scale the weights,
// which are fp16 (rounded at 2^-11 of themselves, where a bf16 output is rounded at 2^-8), less the power of
// two of the largest such product that the row has met.  Window and own tokens are contracted as the bf16 numbers they are
// (weights at 2^-8 there: bf16 reaches as far as the values do).  Sums are fp32.
//
// paged8_lanes_kernel: fp32 and mixed types, and blocks of 16: CUDA cores, fp32 throughout (below).
#include "async_copy.cuh"
#include "paged8_attention.cuh"

namespace kivi {
namespace {

__device__ int g_fault = 0;

constexpr int kStages = 2;
constexpr int kTile = 32;                                // tokens of a tile
constexpr int kPerSm = 2;                                // CTAs
constexpr int kNote = 8;                                 // numbers of a CTA's note to the fold: CTAs behind it that have some of the unit, row0, head, first row, rows
constexpr int kLeast = 8;                                // tiles of a CTA
constexpr float kGrowth = 8.0f;                          // weights up to 2^8 are let stand before the maximum moves
constexpr float kHeadroom = 8.0f, kSlack = 6.0f;         // products of weight and scale: up to 2^8, or 2^14 before their reference moves

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
// four neighbouring numbers as they lie
__device__ __forceinline__ uint2 quad_of(const __nv_bfloat16* p, bool vec) {
    if (vec) return *reinterpret_cast<const uint2*>(p);
    const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
    return make_uint2(u[0] | (uint32_t)u[1] << 16, u[2] | (uint32_t)u[3] << 16);
}
// bf16 numbers that are not finite become 0
__device__ __forceinline__ uint32_t finite_pair(uint32_t w, bool& odd) {
    if ((w & 0x7f80u) == 0x7f80u) { w &= 0xffff0000u; odd = true; }
    if ((w & 0x7f800000u) == 0x7f800000u) { w &= 0xffffu; odd = true; }
    return w;
}
__device__ __forceinline__ void copy8(uint32_t to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
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
// an 8 x 8 matrix of 16-bit numbers, a row to four lanes, with rows and columns in each other's place
__device__ __forceinline__ uint32_t turned(uint32_t w) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(w));
    return y;
}
// cap * tanh z of a score y = cap z
__device__ __forceinline__ float capped_far(float z2, float cap) {           // z2: 2 z log2(e)
    return cap - __fdividef(2.0f * cap, 1.0f + ex2(z2 > 120.0f ? 120.0f : z2));
}
__device__ __forceinline__ float capped(float y, float cap, float inv_cap) {
    const float z = y * inv_cap, s = z * z, far = capped_far(z * (2.0f * 1.4426950408889634f), cap);
    return fabsf(z) <= kTanhNear ? y * fmaf(fmaf(fmaf(fmaf(kTanh9, s, kTanh7), s, kTanh5), s, kTanh3), s, kTanh1) : far;
}
__device__ __forceinline__ float pow2i(int s) { return __uint_as_float((uint32_t)(127 + max(-126, min(127, s))) << 23); }

// ---- the line of work ---------------------------------------------------------------
struct SeqWork {
    PagedSeq q;
    int total, inside, prefix, rows, blocks;             // rows of the step, units' blocks of them
    int tiles, tail;                                     // of a unit: packed tiles, and positions that the other tokens count for
    Span span;
    __device__ __forceinline__ int cost() const { return tiles + tail; }
};
__device__ __forceinline__ bool seq_work(const Paged8Attn& A, int unit_rows, int s, SeqWork& w) {
    const kivi_paged8_layer& L = A.L;
    if (!load_seq(L, A.b, s, w.q) || w.q.n == 0) { w.blocks = w.tiles = w.tail = 0; return false; }
    w.rows = w.q.n * A.n_rep;
    w.blocks = (w.rows + unit_rows - 1) / unit_rows;
    w.total = w.q.held + w.q.n;
    w.inside = min(quant_of(w.total, L.group_size, L.residual_cap), w.q.held);
    w.prefix = prefix_of(A.rules, s, w.total);
    w.span = span_of(kTile, w.total, w.q.held, w.total - 1, A.rules.window, w.prefix);
    const int packed = (w.inside + kTile - 1) / kTile;
    w.tiles = min(w.span.n1, packed) + max(0, packed - (w.span.n1 + w.span.gap));
    w.tail = 1 + (w.total - w.inside) * elem_size(L.res_dtype) / kTile;
    return true;
}

struct Line { int64_t cost, before; int first; };        // all positions; those before sequence `first`

// Called by the whole CTA: the line's length, and which sequence has position at(length) (-1: none), which comes to `found`.
template <int kWarps, typename At>
__device__ __forceinline__ Line find_line(const Paged8Attn& A, int unit_rows, int64_t* scratch /* [kWarps + 2] shared */, SeqWork& found /* shared */, const At& at) {
    constexpr int kThreads = 32 * kWarps;
    const int n = A.b.num_seqs, H = A.L.num_kv_heads, per = (n + kThreads - 1) / kThreads;
    SeqWork w;
    int64_t mine = 0;
    for (int i = 0; i < per; ++i) {
        const int s = threadIdx.x * per + i;
        if (s < n && seq_work(A, unit_rows, s, w)) mine += (int64_t)H * w.blocks * w.cost();
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
            if (per > 1 && (s >= n || !seq_work(A, unit_rows, s, w))) continue;
            const int64_t c = (int64_t)H * w.blocks * w.cost();
            if (want < before + c) { scratch[kWarps] = s; scratch[kWarps + 1] = before; found = w; break; }
            before += c;
        }
    }
    __syncthreads();
    return {total, scratch[kWarps + 1], (int)scratch[kWarps]};
}
__host__ __device__ __forceinline__ int64_t per_cta(int64_t cost, int ctas, int least) {
    const int64_t per = (cost + ctas - 1) / ctas;
    return per < least ? least : per;
}

// The CTA's segments, one after the other.  (In shared memory: as registers two of them were 60 of a thread's.)
struct Walk {
    SeqWork w;
    int64_t at, end, off;                                // next position, the CTA's end, the sequence's first position
    int s, h, rb;                                        // of the segment
    int64_t unit;                                        // its unit's first position
    int a, b;                                            // its positions within the unit

    __device__ __forceinline__ bool next(const Paged8Attn& A, int unit_rows) {
        while (at < end) {
            const int64_t size = (int64_t)A.L.num_kv_heads * w.blocks * w.cost();
            if (at >= off + size) {
                off += size;
                if (++s >= A.b.num_seqs) return false;
                seq_work(A, unit_rows, s, w);
                continue;
            }
            const int c = w.cost();
            const uint64_t x = (uint64_t)(at - off);
            const uint32_t u = x >> 32 ? (uint32_t)(x / (uint32_t)c) : (uint32_t)x / (uint32_t)c;        // (a sequence's units are fewer than 2^32)
            h = (int)(u / (uint32_t)w.blocks); rb = (int)(u % (uint32_t)w.blocks);
            unit = off + (int64_t)u * c;
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

// Warps of a CTA, two CTAs to an SM: what registers and shared memory hold (64 ragged sequences up to 32k with
// four: 488 us).
constexpr int warps_of(int nb) { return nb == 1 ? 6 : 4; }
template <int D, int NB> struct Layout {
    static constexpr int kRows = 8 * NB, kWarps = warps_of(NB), kHalf = kWarps / 2;
    static constexpr int kPart = kTile * D;              // bytes of a tile's keys, or values
    static constexpr int kQ = D + 8, kO = D + 4;         // bf16 numbers, floats of a row
    static constexpr int kVStage = 8 * D * 2;            // bytes: values of eight tokens as bf16
    static constexpr int ring = 0, fold = ring + kWarps * kStages * 2 * kPart;
    static constexpr int kFold = kHalf * kRows * kO * 4 > kWarps * kVStage ? kHalf * kRows * kO * 4 : kWarps * kVStage;
    static constexpr int q = fold + kFold, ml = q + kRows * kQ * 2, scratch = ml + kHalf * kRows * 8, walks = scratch + (kWarps + 2) * 8;
    static constexpr int bars = walks + (kWarps + 1) * (int)sizeof(Walk);
    static constexpr int bytes = bars + kWarps * kStages * 16;
};

// What is done to scores: nothing, rules with a small cap or none, rules with any cap (16 x 8192, 5 tokens, cap 50: 101 us
// as a small cap, 108 as any).
enum { kNoRules, kRules, kAnyCap };

template <int D, int NB, int RULES>
__global__ void __launch_bounds__(32 * warps_of(NB), kPerSm)
paged8_decode_kernel(Paged8Attn A) {
    using S = Layout<D, NB>;
    constexpr int kWarps = S::kWarps, kThreads = 32 * kWarps, kRows = S::kRows, kSteps = D / 16, kChan = D / 4;        // MMAs along the channels; channels of a lane's keys
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), g = lane >> 2, t = lane & 3;
    stream_order();
    settle_args(A);
    cudaTriggerProgrammaticLaunchCompletion();           // (the fold's few blocks wait for this kernel's end)
    const kivi_paged8_layer& L = A.L;
    const int R = L.residual_cap, H = L.num_kv_heads, n_rep = A.n_rep, window = A.rules.window;
    if (blockIdx.x == 0) report_left_out(L, A.b, &g_fault);
    __nv_bfloat16* const q_s = reinterpret_cast<__nv_bfloat16*>(smem + S::q);
    float* const fold_s = reinterpret_cast<float*>(smem + S::fold);
    float* const ml_s = reinterpret_cast<float*>(smem + S::ml);
    const uint32_t ring = smem_u32(smem + S::ring) + warp * (kStages * 2 * S::kPart), v_stage = smem_u32(smem + S::fold) + warp * S::kVStage;
    const uint32_t bars = smem_u32(smem + S::bars) + warp * (kStages * 16);          // of a stage: keys, values
    if (lane == 0) {
        for (int i = 0; i < 2 * kStages; ++i) mbar_init(bars + 8 * i, 1);
        mbar_init_fence();
    }
    Walk& walk = *reinterpret_cast<Walk*>(smem + S::walks);                 // what is computed
    Walk& ahead = (&walk)[1 + warp];                                         // what the warp copies: its first lane's
    int* const note = A.notes + kNote * (int)blockIdx.x;
    const Line line = find_line<kWarps>(A, kRows, reinterpret_cast<int64_t*>(smem + S::scratch), walk.w, [&](int64_t cost) { return per_cta(cost, gridDim.x, kLeast) * blockIdx.x; });
    if (tid == 0) note[0] = 0;                           // (nothing of this CTA's is to be folded, so far)
    if (line.first < 0) return;
    const int64_t per = per_cta(line.cost, gridDim.x, kLeast);
    if (tid == 0) {
        walk.s = line.first; walk.off = line.before;
        walk.at = per * blockIdx.x; walk.end = min(walk.at + per, line.cost);
    }
    __syncthreads();
    if (lane == 0) ahead = walk;
    const uint64_t policy = l2_stream_policy();

    // ---- copies, all of them the first lane's: the warp's next tile into a stage
    const int per_page = L.page_tokens / kTile, per_block = L.group_size / kTile;            // tiles
    const uint32_t block_of = (1u << 20) / per_block + 1;                                    // tile of a page / per_block, for up to 2^15 tiles
    int av = 0, a_end = 0, n1 = 0, a_head = 0, page = 0, in_page = 0, next_page = 0, issued = 0;         // the tile; its place among the sequence's pages
    const int32_t* a_pages = nullptr;
    bool more = true;
    float2 scales[kStages];
    int64_t v_from[kStages];
#pragma unroll
    for (int i = 0; i < kStages; ++i) { scales[i] = make_float2(0.f, 0.f); v_from[i] = -1; }
    auto settle_next = [&] {                             // on to the warp's next tile
        if (av < a_end && !(av >= n1 && av - kWarps < n1)) {
            in_page += kWarps;
            while (in_page >= per_page) { in_page -= per_page; ++page; }
        } else {
            while (av >= a_end) {
                more = ahead.next(A, kRows);
                if (!more) return;
                av = ahead.a + warp;
                a_end = ahead.tiles_end();
                n1 = ahead.w.span.n1; a_head = ahead.h; a_pages = ahead.w.q.pages;
            }
            const int tile = ahead.w.span.tile(av);
            page = tile / per_page;
            in_page = tile - page * per_page;
        }
        next_page = a_pages[page];
    };
    // Keys of the next tile, when the ones before them have been contracted; its values follow when theirs have.
    auto issue_keys = [&](int stage, float2& sc, int64_t& values) {
        values = -1;
        if (!more) return;
        const bool there = (unsigned)next_page < (unsigned)L.num_pages;
        if (!there) atomicOr(&g_fault, kPagedFault);
        const int64_t unit = (there ? next_page : 0) * (int64_t)H + a_head;
        const int64_t f = unit * (uint32_t)(L.page_tokens / L.group_size) + (uint32_t)(((uint64_t)(uint32_t)in_page * block_of) >> 20);
        values = (unit * per_page + in_page) * S::kPart;
        mbar_expect_tx(bars + 16 * stage, S::kPart);
        bulk_g2s(ring + stage * (2 * S::kPart), L.k_codes + values, S::kPart, bars + 16 * stage, policy);
        sc = make_float2(L.k_scales[f], L.v_scales[f]);
        ++issued;
        av += kWarps;
        settle_next();
    };
    auto issue_values = [&](int stage, int64_t from) {
        if (from < 0) return;
        mbar_expect_tx(bars + 16 * stage + 8, S::kPart);
        bulk_g2s(ring + stage * (2 * S::kPart) + S::kPart, L.v_codes + from, S::kPart, bars + 16 * stage + 8, policy);
    };
    int taken = 0;
    bool ok = true, started = false;

    for (;;) {
        __syncthreads();                                 // (the unit before is folded)
        if (tid == 0 && !walk.next(A, kRows)) walk.h = -1;
        __syncthreads();
        if (walk.h < 0) break;
        const PagedSeq& q = walk.w.q;
        const int h = walk.h, row_first = walk.rb * kRows, n_rows = min(kRows, walk.w.rows - row_first), inside = walk.w.inside, prefix = walk.w.prefix;
        // ---- the unit's queries
        for (int i = tid; i < kRows * (D / 4); i += kThreads) {
            const int r = i / (D / 4), d = 4 * (i % (D / 4)), row = row_first + r;
            const __nv_bfloat16* const from_row = reinterpret_cast<const __nv_bfloat16*>(A.q.data) + ((int64_t)q.row0 + row / n_rep) * A.q.row_stride + (int64_t)(h * n_rep + row % n_rep) * A.q.head_stride + d;
            if (r >= n_rows || !A.vec) *reinterpret_cast<uint2*>(q_s + r * S::kQ + d) = r < n_rows ? quad_of(from_row, false) : make_uint2(0u, 0u);
            else copy8(smem_u32(q_s + r * S::kQ + d), from_row);
        }
        if (!started && lane == 0) {
            settle_next();
#pragma unroll
            for (int i = 0; i < kStages; ++i) { issue_keys(i, scales[i], v_from[i]); issue_values(i, v_from[i]); }
        }
        started = true;
        __syncwarp();
        const int total = walk.w.total;
        const __nv_bfloat16* const k_ring = reinterpret_cast<const __nv_bfloat16*>(L.k_res) + ((int64_t)q.slot * H + h) * R * D;
        const __nv_bfloat16* const v_ring = reinterpret_cast<const __nv_bfloat16*>(L.v_res) + ((int64_t)q.slot * H + h) * R * D;
        auto row_at = [&](int tok, bool of_keys) -> const __nv_bfloat16* {
            if (tok < q.held) return (of_keys ? k_ring : v_ring) + (int64_t)ring_slot(tok, 0, R) * D;
            const kivi_rows& r = of_keys ? A.k : A.v;
            return reinterpret_cast<const __nv_bfloat16*>(r.data) + ((int64_t)q.row0 + min(tok, total - 1) - q.held) * r.row_stride + (int64_t)h * r.head_stride;
        };
        if (walk.has_tail())                             // the rows that come last are on their way to L2 meanwhile
            for (int t0 = inside + 16 * warp; t0 < total; t0 += 16 * kWarps)
#pragma unroll
                for (int i = 0; i < D / 64; ++i) {
                    const char* const at = reinterpret_cast<const char*>(row_at(t0 + (lane & 15), lane < 16)) + 128 * i;
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
                }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();
        // As an operand a lane has channels kChan t .. of row 8 b + g, four to an MMA; keys lie the same way.
        uint32_t qb[NB][kSteps][2];
        float unscale[NB][2];                            // of a contracted score of rows 8 b + 2 t and the next, and to powers of two where nothing else is done to it
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float top = 0.0f;
            for (int c = 0; c < kChan; c += 4) {
                const float4 x = load4(q_s + (8 * b + g) * S::kQ + kChan * t + c, true);
                const float y[4] = {fabsf(x.x), fabsf(x.y), fabsf(x.z), fabsf(x.w)};
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, y[i] <= 3.4e38f ? y[i] : 0.0f);         // (the largest finite one)
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = (int)(__float_as_uint(top) >> 23), shift = min(126, 127 + 13 - e);             // largest to 2^13 .. 2^14 (what is below 2^-113 as far as a power of two goes)
            const float f = pow2i(shift);
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                float4 x = load4(q_s + (8 * b + g) * S::kQ + kChan * t + 4 * i, true);
                x = make_float4(x.x * f, x.y * f, x.z * f, x.w * f);
                qb[b][i][0] = half2_of(x.x, x.y);
                qb[b][i][1] = half2_of(x.z, x.w);
            }
#pragma unroll
            for (int e2 = 0; e2 < 2; ++e2)
                unscale[b][e2] = A.scale * pow2i(-__shfl_sync(0xffffffffu, shift, 4 * (2 * t + e2))) * (RULES ? 1.0f : 1.4426950408889634f);
        }
        int place[NB][2], from[NB][2];
        float slope[NB][2];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = 8 * b + 2 * t + e, row = row_first + r;
                // (a row that is not there sees what the first one sees, and is not written)
                place[b][e] = q.held + (r < n_rows ? row : row_first) / n_rep;
                from[b][e] = window_from(place[b][e], window);
                slope[b][e] = RULES && A.rules.slopes && r < n_rows ? A.rules.slopes[h * n_rep + row % n_rep] : 0.0f;
            }
        const int from_most = window_from(q.held + (row_first + n_rows - 1) / n_rep, window);
        // o[c][b]: channels 16 c + g and + 8 of rows 8 b + 2 t and the next
        float m[NB][2], l[NB][2], ref[NB][2], o[D / 16][NB][4];           // ref: the largest score plus value scale so far; O is 2^(kHeadroom - ref) times what it stands for
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) { m[b][e] = -INFINITY; l[b][e] = 0.0f; ref[b][e] = -1.0e30f; }
#pragma unroll
        for (int c = 0; c < D / 16; ++c)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[c][b][e] = 0.0f;
        auto rescale = [&](int b, float f0, float f1) {
#pragma unroll
            for (int c = 0; c < D / 16; ++c) { o[c][b][0] *= f0; o[c][b][1] *= f1; o[c][b][2] *= f0; o[c][b][3] *= f1; }
        };
        // Scores x[n][b] (tokens t0 + 16 n + g and + 8, rows 8 b + 2 t and the next) to weights; u: what makes powers of two
        // of them (RULES: scores).  hidden(token, b, e): the row does not see it.  lift: their value scale's power of two, rounded
        // up.  up: what weights times the value scale are multiplied with to be on O's scale.
        auto weights = [&](auto& x, const float (&u)[NB][2], int t0, bool some_hidden, auto&& hidden, float lift, float (&up)[NB][2]) {
            constexpr int N = sizeof(x) / sizeof(x[0]);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if constexpr (RULES) {
                    const float cap = A.rules.softcap;
                    if constexpr (RULES == kAnyCap) {
                        const float inv_cap = 1.0f / cap;
#pragma unroll
                        for (int n = 0; n < N; ++n)
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[n][b][e] = capped(x[n][b][e] * u[b][e & 1], cap, inv_cap);
                    }
                    const bool small_cap = RULES == kRules && cap > 0.0f;
                    const float to_z2 = small_cap ? 2.0f * 1.4426950408889634f / cap : 0.0f;
#pragma unroll
                    for (int n = 0; n < N; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float y = x[n][b][e];
                            if (RULES == kRules) y *= u[b][e & 1];
                            if (small_cap) y = capped_far(y * to_z2, cap);
                            y = fmaf(slope[b][e & 1], (float)(t0 + 16 * n + g + 8 * (e >> 1) - place[b][e & 1]), y);
                            x[n][b][e] = y * 1.4426950408889634f;
                        }
                }
                if (some_hidden) {
#pragma unroll
                    for (int n = 0; n < N; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (hidden(t0 + 16 * n + g + 8 * (e >> 1), b, e & 1)) x[n][b][e] = -INFINITY;
                }
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    top[0] = fmaxf(top[0], fmaxf(x[n][b][0], x[n][b][2]));
                    top[1] = fmaxf(top[1], fmaxf(x[n][b][1], x[n][b][3]));
                }
                float base[2], by[2];
                bool grows = false;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 4));
                    top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 8));
                    top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 16));
                    by[e] = RULES ? 1.0f : u[b][e];
                    top[e] *= by[e];
                    if (top[e] > m[b][e] + kGrowth) {    // (from -inf: whenever there is a maximum)
                        l[b][e] *= m[b][e] == -INFINITY ? 0.0f : ex2(m[b][e] - top[e]);
                        m[b][e] = top[e];
                    }
                    base[e] = m[b][e] == -INFINITY ? 0.0f : m[b][e];
                    top[e] += lift;
                    grows |= top[e] > ref[b][e] + kSlack;
                }
                if (__any_sync(0xffffffffu, grows)) {
                    float f[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const bool grow = top[e] > ref[b][e];
                        f[e] = grow ? ex2(ref[b][e] - top[e]) : 1.0f;
                        if (grow) ref[b][e] = top[e];
                    }
                    rescale(b, f[0], f[1]);
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) up[b][e] = ex2(fminf(base[e] - ref[b][e] + kHeadroom, 126.0f));
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[n][b][e] = ex2(fmaf(x[n][b][e], by[e & 1], -base[e & 1]));
                        l[b][e & 1] += x[n][b][e];
                    }
            }
        };

        // ---- tiles of pages
        const Span span = walk.w.span;
        const int v_end = walk.tiles_end();
        for (int v = walk.a + warp; v < v_end; v += kWarps) {
            const int stage = taken % kStages, t0 = span.tile(v) * kTile;
            float2 sc = stage ? scales[kStages - 1] : scales[0];
            sc.x = __shfl_sync(0xffffffffu, sc.x, 0); sc.y = __shfl_sync(0xffffffffu, sc.y, 0);
            static_assert(kStages == 2, "scales of a stage are picked by hand");
            const uint32_t phase = (uint32_t)(taken / kStages) & 1u;
            if (ok && !mbar_wait(bars + 16 * stage, phase)) { atomicOr(&g_fault, 1); ok = false; }
            ok = __all_sync(0xffffffffu, ok);
            const uint32_t keys = ring + stage * (2 * S::kPart), values = keys + S::kPart;
            float x[2][NB][4], x2[2][NB][4];             // (two sums each: an MMA waits for the one before it)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[n][b][e] = x2[n][b][e] = 0.0f;
#pragma unroll
            for (int p = 0; p < kChan / 16; ++p)
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int piece = D == 128 ? (2 * t + p) ^ g : t ^ (g >> 1 & 3);
                    const uint4 k0 = lds128(keys + (16 * n + g) * D + 16 * piece), k1 = lds128(keys + (16 * n + 8 + g) * D + 16 * piece);
                    const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t a[4];
                        e4m3x4_to_half2(w0[i], a[0], a[2]);
                        e4m3x4_to_half2(w1[i], a[1], a[3]);
#pragma unroll
                        for (int b = 0; b < NB; ++b)
                            mma_f16(i & 1 ? x2[n][b] : x[n][b], a, qb[b][4 * p + i][0], qb[b][4 * p + i][1]);
                    }
                }
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[n][b][e] += x2[n][b][e];
            __syncwarp();                                // (the keys have been read)
            if (lane == 0) {
                if (stage) issue_keys(kStages - 1, scales[kStages - 1], v_from[kStages - 1]);
                else issue_keys(0, scales[0], v_from[0]);
            }
            __syncwarp();
            float u[NB][2], f[NB][2];
#pragma unroll
            for (int b = 0; b < NB; ++b) { u[b][0] = fmaxf(unscale[b][0] * sc.x, 1.0e-37f); u[b][1] = fmaxf(unscale[b][1] * sc.x, 1.0e-37f); }      // (not 0: hidden scores are -inf)
            // (a page's tokens come before every row)
            const bool edge = t0 + kTile > inside || (t0 < from_most && t0 + kTile > prefix);
            weights(x, u, t0, edge, [&](int tok, int b, int e) { return tok >= inside || (tok < from[b][e] && tok >= prefix); },
                    (float)((int)(__float_as_uint(sc.y) >> 23) - 126), f);
            // weights as the other operand: rows and tokens change places eight by eight
            uint32_t pb[NB][2][2];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                f[b][0] = fminf(f[b][0] * sc.y, 1.0e37f);
                f[b][1] = fminf(f[b][1] * sc.y, 1.0e37f);
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float lo = x[n][b][2 * e] * f[b][0], hi = x[n][b][2 * e + 1] * f[b][1];
                        pb[b][n][e] = turned(half2_of(lo, hi));
                    }
            }
            if (ok && !mbar_wait(bars + 16 * stage + 8, phase)) { atomicOr(&g_fault, 1); ok = false; }
            ok = __all_sync(0xffffffffu, ok);
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
                const uint2 w0 = lds64(values + (16 * c + g) * kTile + 8 * t), w1 = lds64(values + (16 * c + 8 + g) * kTile + 8 * t);
                uint32_t a[2][4];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    e4m3x4_to_half2(n ? w0.y : w0.x, a[n][0], a[n][2]);
                    e4m3x4_to_half2(n ? w1.y : w1.x, a[n][1], a[n][3]);
                }
#pragma unroll
                for (int b = 0; b < NB; ++b) {
#pragma unroll
                    for (int n = 0; n < 2; ++n) mma_f16(o[c][b], a[n], pb[b][n][0], pb[b][n][1]);
                }
            }
            __syncwarp();                                // (the values have been read)
            ++taken;
            if (lane == 0) issue_values(stage, stage ? v_from[kStages - 1] : v_from[0]);
            __syncwarp();
        }

        // ---- the window and the step's own tokens, sixteen at a time
        if (walk.has_tail()) {
            float one[NB][2];
#pragma unroll
            for (int b = 0; b < NB; ++b) one[b][0] = one[b][1] = A.scale * (RULES ? 1.0f : 1.4426950408889634f);
            for (int t0 = inside + 16 * warp; t0 < total; t0 += 16 * kWarps) {
                float x[1][NB][4];
#pragma unroll
                for (int b = 0; b < NB; ++b) x[0][b][0] = x[0][b][1] = x[0][b][2] = x[0][b][3] = 0.0f;
                const __nv_bfloat16* const row0 = row_at(t0 + g, true) + kChan * t;
                const __nv_bfloat16* const row1 = row_at(t0 + 8 + g, true) + kChan * t;
                const bool vec0 = t0 + g < q.held || A.vec, vec1 = t0 + 8 + g < q.held || A.vec;
                uint2 k0[kSteps], k1[kSteps], vw[2][D / 32][2];          // (all on their way together)
#pragma unroll
                for (int i = 0; i < kSteps; ++i) { k0[i] = quad_of(row0 + 4 * i, vec0); k1[i] = quad_of(row1 + 4 * i, vec1); }
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        const int tok = t0 + 8 * half + (32 * i + lane) / (D / 8);
                        const __nv_bfloat16* const from_row = row_at(tok, false) + 8 * (lane % (D / 8));
                        const bool vec = tok < q.held || A.vec;
                        vw[half][i][0] = quad_of(from_row, vec); vw[half][i][1] = quad_of(from_row + 4, vec);
                    }
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    const uint32_t a[4] = {k0[i].x, k1[i].x, k0[i].y, k1[i].y};
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const uint2 y = *reinterpret_cast<const uint2*>(q_s + (8 * b + g) * S::kQ + kChan * t + 4 * i);
                        mma_bf16(x[0][b], a, y.x, y.y);
                    }
                }
                auto hidden = [&](int tok, int b, int e) { return tok >= total || ((tok > place[b][e] || tok < from[b][e]) && tok >= prefix); };
                float f[NB][2];
                weights(x, one, t0, true, hidden, 1.0f, f);
                uint32_t pb[NB][2];
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 2; ++e) pb[b][e] = turned(bf16x2_of(x[0][b][2 * e] * f[b][0], x[0][b][2 * e + 1] * f[b][1]));
                // Values go through shared memory, eight tokens at a time.  One that is not finite would reach rows that do not
                // see it through weights of 0: it is left out there, and added to the rows that do.
                bool odd = false;
                uint32_t a[D / 16][4];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        const int j = (32 * i + lane) / (D / 8), p = lane % (D / 8), tok = t0 + 8 * half + j;
                        const uint2 lo = vw[half][i][0], hi = vw[half][i][1];
                        const bool there = tok < total;
                        const uint32_t w[4] = {there ? finite_pair(lo.x, odd) : 0u, there ? finite_pair(lo.y, odd) : 0u, there ? finite_pair(hi.x, odd) : 0u, there ? finite_pair(hi.y, odd) : 0u};
                        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(v_stage + j * (2 * D) + ((p ^ j) << 4)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                    }
                    __syncwarp();
#pragma unroll
                    for (int c = 0; c < D / 16; c += 2) {
                        uint32_t r[4];
                        const int j = lane & 7, p = 2 * c + (lane >> 3);
                        ldmatrix_trans(v_stage + j * (2 * D) + ((p ^ j) << 4), r);
                        a[c][2 * half] = r[0]; a[c][2 * half + 1] = r[1];
                        a[c + 1][2 * half] = r[2]; a[c + 1][2 * half + 1] = r[3];
                    }
                }
#pragma unroll
                for (int c = 0; c < D / 16; ++c)
#pragma unroll
                    for (int b = 0; b < NB; ++b) mma_bf16(o[c][b], a[c], pb[b][0], pb[b][1]);
                if (__any_sync(0xffffffffu, odd)) {
#pragma unroll 1
                    for (int j = 0; j < 16 && t0 + j < total; ++j) {
                        const __nv_bfloat16* const from_row = row_at(t0 + j, false);
#pragma unroll
                        for (int c = 0; c < D / 16; ++c)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float y = __bfloat162float(from_row[16 * c + 8 * (e >> 1) + g]);
                                if (fabsf(y) <= 3.4028234e38f) continue;
#pragma unroll
                                for (int b = 0; b < NB; ++b)
                                    if (!hidden(t0 + j, b, e & 1)) o[c][b][e] += y;
                            }
                    }
                }
            }
        }

        // ---- the warps meet
        {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                // (weights in powers of two from the maximum; nothing seen: 0)
                float f[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    f[e] = m[b][e] == -INFINITY ? 0.0f : ex2(fmaxf(ref[b][e] - m[b][e] - kHeadroom, -126.0f));
                    l[b][e] += __shfl_xor_sync(0xffffffffu, l[b][e], 4);
                    l[b][e] += __shfl_xor_sync(0xffffffffu, l[b][e], 8);
                    l[b][e] += __shfl_xor_sync(0xffffffffu, l[b][e], 16);
                }
                rescale(b, f[0], f[1]);
            }
            auto leave = [&](int buf) {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int r = 8 * b + 2 * t + e;
                        if (r >= n_rows) continue;
                        if (g == 0) *reinterpret_cast<float2*>(ml_s + (buf * kRows + r) * 2) = make_float2(m[b][e], l[b][e]);
#pragma unroll
                        for (int c = 0; c < D / 16; ++c) {
                            fold_s[(buf * kRows + r) * S::kO + 16 * c + g] = o[c][b][e];
                            fold_s[(buf * kRows + r) * S::kO + 16 * c + 8 + g] = o[c][b][2 + e];
                        }
                    }
            };
            auto take = [&](int buf) {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int r = 8 * b + 2 * t + e;
                        if (r >= n_rows) continue;
                        const float2 ml = *reinterpret_cast<const float2*>(ml_s + (buf * kRows + r) * 2);
                        const float M = fmaxf(m[b][e], ml.x), from_0 = M == -INFINITY ? 0.0f : M, mine = ex2(m[b][e] - from_0), other = ex2(ml.x - from_0);
                        m[b][e] = M;
                        l[b][e] = l[b][e] * mine + ml.y * other;
#pragma unroll
                        for (int c = 0; c < D / 16; ++c) {
                            o[c][b][e] = fmaf(fold_s[(buf * kRows + r) * S::kO + 16 * c + g], other, o[c][b][e] * mine);
                            o[c][b][2 + e] = fmaf(fold_s[(buf * kRows + r) * S::kO + 16 * c + 8 + g], other, o[c][b][2 + e] * mine);
                        }
                    }
            };
            __syncthreads();                             // (values of the tail have been read)
            if (warp >= S::kHalf) leave(warp - S::kHalf);
            __syncthreads();
            if (warp < S::kHalf) take(warp);
            __syncthreads();
            if (warp > 0 && warp < S::kHalf) leave(warp);
            __syncthreads();
            if (warp == 0) {
#pragma unroll 1
                for (int i = 1; i < S::kHalf; ++i) take(i);
                leave(0);
            }
            __syncthreads();
            // the CTAs that have something of the unit
            const int64_t c0 = walk.unit / per, c1 = (walk.unit + walk.w.tiles) / per;
            const int64_t slot = 2 * (int64_t)blockIdx.x + (c0 == (int64_t)blockIdx.x ? 1 : 0);
            if (tid == 0 && c0 != c1 && c0 == (int64_t)blockIdx.x) {
                note[1] = q.row0; note[2] = h; note[3] = row_first; note[4] = n_rows;
                note[0] = (int)(c1 - c0);
            }
            for (int i = tid; i < n_rows * (D / 4); i += kThreads) {
                const int r = i / (D / 4), d = 4 * (i % (D / 4)), row = row_first + r;
                const float4 y = *reinterpret_cast<const float4*>(fold_s + r * S::kO + d);
                const float2 ml = *reinterpret_cast<const float2*>(ml_s + r * 2);
                if (c0 == c1) {
                    const float inv = 1.0f / ml.y;       // (a row sees itself: the sum is above 0)
                    const int64_t at = ((int64_t)q.row0 + row / n_rep) * A.out.row_stride + (int64_t)(h * n_rep + row % n_rep) * A.out.head_stride;
                    store_quad(A.out.data, A.out_dtype, at + d, make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
                } else {
                    const int64_t part = slot * kRows + r;
                    if (d == 0) *reinterpret_cast<float2*>(A.part_ml + 2 * part) = ml;
                    *reinterpret_cast<float4*>(A.part_o + part * D + d) = y;
                }
            }
        }
    }
    // (a stage that a wait has given up on is not left to the next block's shared memory)
    for (; lane == 0 && taken < issued; ++taken)
        for (int i = 0; i < 2; ++i) mbar_wait(bars + 16 * (taken % kStages) + 8 * i, (uint32_t)(taken / kStages) & 1u);
}

// ---- up to four rows on the CUDA cores ---------------------------------------------------------
// The same line of work for long sequences that the tensor cores do not take: fp32 rows (an MMA truncates what it adds: 1.1e-6 off
// 64 bits where fp32 sums are 3e-7), mixed types, blocks of 16 tokens.  A lane has sixteen channels of a
// token's key, a warp reads 512 bytes in a row, a token's lanes add up their parts.  Of the values a lane has sixteen tokens
// of a channel; the two lanes of a channel add up at a unit's end.  Keys of the next tile are on their way while values are weighed,
// and the other way round, 4 KB of each a warp.  A row or two to a unit: with four, queries, sums and bytes do not
// fit into 255 registers (16 x 8192 tokens, 8 x 4 heads of 128, fp32: 489 us, 450 as two units of two that find the bytes in L2).
// Bound by issue: 16 bytes are 16 FMAs a row and 12 conversions (28 x 14650 tokens, 4 heads, fp32: 278 us for 431 MB, 1.55 TB/s; the general
// kernel 1090).
constexpr int kLaneWarps = 4;
template <int D, int NR> struct LaneLayout {
    static constexpr int kO = D + 4;                     // floats of a row
    static constexpr int p = 0, q = p + kLaneWarps * NR * 32 * 4, fold = q + NR * kO * 4, ml = fold + kLaneWarps * NR * kO * 4, scratch = ml + kLaneWarps * NR * 8;
    static constexpr int walks = scratch + (kLaneWarps + 2) * 8, bytes = walks + (int)sizeof(Walk);
};

template <typename T, int D, int NR>
__global__ void __launch_bounds__(32 * kLaneWarps, 2)
paged8_lanes_kernel(Paged8Attn A) {
    using S = LaneLayout<D, NR>;
    constexpr int kWarps = kLaneWarps, kThreads = 32 * kWarps, kPieces = D / 16, kSteps = D / 16, kTokens = 32 / kPieces;      // tokens of a step's keys
    __shared__ __align__(16) uint8_t smem[S::bytes];
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    stream_order();
    settle_args(A);
    cudaTriggerProgrammaticLaunchCompletion();           // (the fold's few blocks wait for this kernel's end)
    const kivi_paged8_layer& L = A.L;
    const int G = L.group_size, R = L.residual_cap, H = L.num_kv_heads, n_rep = A.n_rep, window = A.rules.window, run = value8_run(G);
    if (blockIdx.x == 0) report_left_out(L, A.b, &g_fault);
    float* const p_s = reinterpret_cast<float*>(smem + S::p) + warp * NR * 32;           // [row][place of a token among the value bytes]
    float* const q_s = reinterpret_cast<float*>(smem + S::q);
    float* const fold_s = reinterpret_cast<float*>(smem + S::fold);
    float2* const ml_s = reinterpret_cast<float2*>(smem + S::ml);
    Walk& walk = *reinterpret_cast<Walk*>(smem + S::walks);
    int* const note = A.notes + kNote * (int)blockIdx.x;
    const Line line = find_line<kWarps>(A, NR, reinterpret_cast<int64_t*>(smem + S::scratch), walk.w, [&](int64_t cost) { return per_cta(cost, gridDim.x, kWarps) * blockIdx.x; });
    if (tid == 0) note[0] = 0;                           // (nothing of this CTA's is to be folded, so far)
    if (line.first < 0) return;
    const int64_t per = per_cta(line.cost, gridDim.x, kWarps);
    if (tid == 0) {
        walk.s = line.first; walk.off = line.before;
        walk.at = per * blockIdx.x; walk.end = min(walk.at + per, line.cost);
    }
    // a lane's part of a tile: channels 16 piece .. of tokens kTokens i + first_token; sixteen tokens of channels 16 i + channel
    const int piece = lane % kPieces, first_token = lane / kPieces;
    const int part = run == 32 ? lane & 1 : lane >> 4, channel = run == 32 ? lane >> 1 : lane & 15;
    const bool capped = A.rules.softcap > 0.0f;
    constexpr float kLog2e = 1.4426950408889634f;

    for (;;) {
        __syncthreads();                                 // (the unit before is folded)
        if (tid == 0 && !walk.next(A, NR)) walk.h = -1;
        __syncthreads();
        if (walk.h < 0) break;
        const PagedSeq q = walk.w.q;
        const int h = walk.h, row_first = walk.rb * NR, n_rows = min(NR, walk.w.rows - row_first), inside = walk.w.inside, prefix = walk.w.prefix, total = walk.w.total;
        const Span span = walk.w.span;
        const int v_end = walk.tiles_end(), v_begin = walk.a;
        const bool has_tail = walk.has_tail();
        for (int i = tid; i < NR * (D / 4); i += kThreads) {
            const int r = i / (D / 4), d = 4 * (i % (D / 4)), row = row_first + r;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < n_rows) x = load4_as(A.q, A.q_dtype, (int64_t)q.row0 + row / n_rep, h * n_rep + row % n_rep, d, A.vec != 0);
            *reinterpret_cast<float4*>(q_s + r * S::kO + d) = x;
        }
        __syncthreads();
        int place[NR], from[NR];
        float slope[NR], m[NR], l[NR], o[NR][kSteps];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const int row = row_first + r;
            // (a row that is not there sees what the first one sees, and is not written)
            place[r] = q.held + (r < n_rows ? row : row_first) / n_rep;
            from[r] = window_from(place[r], window);
            slope[r] = A.rules.slopes && r < n_rows ? A.rules.slopes[h * n_rep + row % n_rep] : 0.0f;
            m[r] = -INFINITY; l[r] = 0.0f;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) o[r][i] = 0.0f;
        }
        // a contracted score as the rules leave it
        auto ruled = [&](float x, int r, int tok) {
            x *= A.scale;
            if (capped) x = A.rules.softcap * tanhf(x / A.rules.softcap);
            return fmaf(slope[r], (float)(tok - place[r]), x);
        };
        auto hidden = [&](int tok, int r) { return tok >= total || ((tok > place[r] || tok < from[r]) && tok >= prefix); };
        auto move = [&](int r, float top) {              // to a larger maximum; what that leaves of the sums so far
            if (top <= m[r]) return 1.0f;
            const float f = m[r] == -INFINITY ? 0.0f : exp2f((m[r] - top) * kLog2e);
            m[r] = top;
            l[r] *= f;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) o[r][i] *= f;
            return f;
        };

        // ---- tiles of pages
        float2 scale_next[2];
        auto look_up = [&](int v) {                      // the scales of a tile's sixteens (pages and blocks are whole sixteens)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int t = span.tile(v) * kTile + 16 * i;
                scale_next[i] = make_float2(0.0f, 0.0f);
                if (t >= inside) continue;
                const int64_t f = ((int64_t)page_of(L, q, t, &g_fault) * H + h) * (L.page_tokens / G) + t % L.page_tokens / G;
                scale_next[i] = make_float2(L.k_scales[f], L.v_scales[f]);
            }
        };
        uint4 kx[kSteps], vx[kSteps];
        float2 scale[2];
        auto load_tile = [&](int v, bool of_keys) {
            const int t0 = span.tile(v) * kTile;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                // keys: token kTokens i + first_token; values: the run that has the lane's part
                const int t = of_keys ? t0 + kTokens * i + first_token : t0 + (run == 32 ? 0 : 16 * part);
                const int sixteen = t & ~15;
                uint4 x = make_uint4(0u, 0u, 0u, 0u);
                if (sixteen < inside) {
                    const int64_t base = ((int64_t)page_of(L, q, sixteen, &g_fault) * H + h) * L.page_tokens * D;
                    const int in_page = t % L.page_tokens;
                    x = of_keys ? *reinterpret_cast<const uint4*>(L.k_codes + base + key8_offset(in_page, 16 * piece, D))
                                : *reinterpret_cast<const uint4*>(L.v_codes + base + (int64_t)in_page * D + (16 * i + channel) * run + (run == 32 ? 16 * part : 0));
                }
                (of_keys ? kx : vx)[i] = x;
            }
        };
        int v = v_begin + warp;
        if (v < v_end) { load_tile(v, true); load_tile(v, false); look_up(v); }
        for (; v < v_end; v += kWarps) {
            const int t0 = span.tile(v) * kTile;
            scale[0] = scale_next[0]; scale[1] = scale_next[1];
            float x[NR][kSteps];
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const uint32_t w[4] = {kx[i].x, kx[i].y, kx[i].z, kx[i].w};
                float k[16];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float4 y = e4m3x4(w[e]);
                    k[4 * e] = y.x; k[4 * e + 1] = y.y; k[4 * e + 2] = y.z; k[4 * e + 3] = y.w;
                }
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const float4 y = *reinterpret_cast<const float4*>(q_s + r * S::kO + 16 * piece + e);
                        sum = fmaf(k[e], y.x, fmaf(k[e + 1], y.y, fmaf(k[e + 2], y.z, fmaf(k[e + 3], y.w, sum))));
                    }
                    x[r][i] = sum;
                }
            }
            if (v + kWarps < v_end) { load_tile(v + kWarps, true); look_up(v + kWarps); }
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
#pragma unroll
                    for (int b = 1; b < kPieces; b *= 2) x[r][i] += __shfl_xor_sync(0xffffffffu, x[r][i], b);
                    const int u = kTokens * i + first_token, tok = t0 + u;
                    x[r][i] = ruled(x[r][i] * (u < 16 ? scale[0].x : scale[1].x), r, tok);
                    if (tok >= inside || (tok < from[r] && tok >= prefix)) x[r][i] = -INFINITY;      // (a page's tokens come before every row)
                    top = fmaxf(top, x[r][i]);
                }
#pragma unroll
                for (int b = kPieces; b < 32; b *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, b));
                move(r, top);
                const float base = m[r] == -INFINITY ? 0.0f : m[r];
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    const int u = kTokens * i + first_token;
                    const float p = exp2f((x[r][i] - base) * kLog2e);
                    if (piece == 0) {
                        l[r] += p;
                        p_s[r * 32 + (run == 32 ? value8_place(u, 32) : (u & 16) + value8_place(u & 15, 16))] = p;
                    }
                }
            }
            __syncwarp();
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                float w[16];
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const float4 y = *reinterpret_cast<const float4*>(p_s + r * 32 + 16 * part + e);
                    w[e] = y.x; w[e + 1] = y.y; w[e + 2] = y.z; w[e + 3] = y.w;
                }
                const float by = run == 32 ? scale[0].y : part ? scale[1].y : scale[0].y;
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    const uint32_t c[4] = {vx[i].x, vx[i].y, vx[i].z, vx[i].w};
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float4 y = e4m3x4(c[e]);
                        sum = fmaf(w[4 * e], y.x, fmaf(w[4 * e + 1], y.y, fmaf(w[4 * e + 2], y.z, fmaf(w[4 * e + 3], y.w, sum))));
                    }
                    o[r][i] = fmaf(sum, by, o[r][i]);
                }
            }
            if (v + kWarps < v_end) load_tile(v + kWarps, false);
            __syncwarp();                                // (weights have been read)
        }

        // ---- the window and the step's own tokens, eight at a time: a lane has D / 32 channels of each
        float l_tail[NR], o_tail[NR][D / 32];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            l_tail[r] = 0.0f;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) o_tail[r][c] = 0.0f;
        }
        if (has_tail) {
            constexpr int kC = D / 32, kAt = 8;
            const T* const k_ring = reinterpret_cast<const T*>(L.k_res) + ((int64_t)q.slot * H + h) * R * D;
            const T* const v_ring = reinterpret_cast<const T*>(L.v_res) + ((int64_t)q.slot * H + h) * R * D;
            auto row_at = [&](int tok, bool of_keys) -> const T* {
                if (tok < q.held) return (of_keys ? k_ring : v_ring) + (int64_t)ring_slot(tok, 0, R) * D;
                const kivi_rows& r = of_keys ? A.k : A.v;
                return reinterpret_cast<const T*>(r.data) + ((int64_t)q.row0 + min(tok, total - 1) - q.held) * r.row_stride + (int64_t)h * r.head_stride;
            };
            for (int t0 = inside + kAt * warp; t0 < total; t0 += kAt * kWarps) {
                float k[kAt][kC], y[kAt][kC];
#pragma unroll
                for (int j = 0; j < kAt; ++j) {
                    const T* const kr = row_at(t0 + j, true) + lane;
                    const T* const vr = row_at(t0 + j, false) + lane;
#pragma unroll
                    for (int c = 0; c < kC; ++c) { k[j][c] = (float)kr[32 * c]; y[j][c] = (float)vr[32 * c]; }
                }
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    float x[kAt], top = -INFINITY;
#pragma unroll
                    for (int j = 0; j < kAt; ++j) {
                        x[j] = 0.0f;
#pragma unroll
                        for (int c = 0; c < kC; ++c) x[j] = fmaf(k[j][c], q_s[r * S::kO + 32 * c + lane], x[j]);
#pragma unroll
                        for (int b = 1; b < 32; b *= 2) x[j] += __shfl_xor_sync(0xffffffffu, x[j], b);
                        x[j] = hidden(t0 + j, r) ? -INFINITY : ruled(x[j], r, t0 + j);
                        top = fmaxf(top, x[j]);
                    }
                    const float f = move(r, top), base = m[r] == -INFINITY ? 0.0f : m[r];
                    l_tail[r] *= f;
#pragma unroll
                    for (int c = 0; c < kC; ++c) o_tail[r][c] *= f;
#pragma unroll
                    for (int j = 0; j < kAt; ++j) {
                        const float p = exp2f((x[j] - base) * kLog2e);
                        l_tail[r] += p;
                        // (a token that the row does not see may hold anything, infinities and NaN too)
                        const bool seen = !hidden(t0 + j, r);
#pragma unroll
                        for (int c = 0; c < kC; ++c) o_tail[r][c] = fmaf(p, seen ? y[j][c] : 0.0f, o_tail[r][c]);
                    }
                }
            }
        }

        // ---- the warps meet: each leaves its rows, all of them add up
#pragma unroll
        for (int r = 0; r < NR; ++r) {
#pragma unroll
            for (int b = kPieces; b < 32; b *= 2) l[r] += __shfl_xor_sync(0xffffffffu, l[r], b);
            l[r] = __shfl_sync(0xffffffffu, l[r], 0) + l_tail[r];
            float* const mine = fold_s + (warp * NR + r) * S::kO;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                o[r][i] += __shfl_xor_sync(0xffffffffu, o[r][i], run == 32 ? 1 : 16);
                if (part == 0) mine[16 * i + channel] = o[r][i];
            }
            __syncwarp();
#pragma unroll
            for (int c = 0; c < D / 32; ++c) mine[32 * c + lane] += o_tail[r][c];
            if (lane == 0) ml_s[warp * NR + r] = make_float2(m[r] * kLog2e, l[r]);          // (partials: in powers of two)
        }
        __syncthreads();
        // the CTAs that have something of the unit
        const int64_t c0 = walk.unit / per, c1 = (walk.unit + walk.w.tiles) / per;
        const int64_t slot = 2 * (int64_t)blockIdx.x + (c0 == (int64_t)blockIdx.x ? 1 : 0);
        if (tid == 0 && c0 != c1 && c0 == (int64_t)blockIdx.x) {
            note[1] = q.row0; note[2] = h; note[3] = row_first; note[4] = n_rows;
            note[0] = (int)(c1 - c0);
        }
        for (int i = tid; i < n_rows * (D / 4); i += kThreads) {
            const int r = i / (D / 4), d = 4 * (i % (D / 4)), row = row_first + r;
            float M = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ml_s[w * NR + r].x);
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float2 ml = ml_s[w * NR + r];
                const float4 y = *reinterpret_cast<const float4*>(fold_s + (w * NR + r) * S::kO + d);
                const float f = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - M);
                if (ml.x == -INFINITY && ml.y == 0.0f) continue;      // (nothing of it is seen)
                sum = fmaf(f, ml.y, sum);
                a.x = fmaf(f, y.x, a.x); a.y = fmaf(f, y.y, a.y); a.z = fmaf(f, y.z, a.z); a.w = fmaf(f, y.w, a.w);
            }
            if (c0 == c1) {
                const float inv = 1.0f / sum;            // (a row sees itself: the sum is above 0)
                const int64_t at = ((int64_t)q.row0 + row / n_rep) * A.out.row_stride + (int64_t)(h * n_rep + row % n_rep) * A.out.head_stride;
                store_quad(A.out.data, A.out_dtype, at + d, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
            } else {
                const int64_t partial = slot * NR + r;
                if (d == 0) *reinterpret_cast<float2*>(A.part_ml + 2 * partial) = make_float2(M, sum);
                *reinterpret_cast<float4*>(A.part_o + partial * D + d) = a;
            }
        }
    }
}

// Folds the units that lie across a CTA's end: block c the one that CTA c has left a note of.  A thread has a quad
// of channels of a row.
__global__ void __launch_bounds__(128)
paged8_fold_kernel(Paged8Attn A, int unit_rows) {
    stream_order();
    settle_args(A);
    const int c = blockIdx.x, D = A.L.head_dim, n_rep = A.n_rep, quads = D / 4;
    const int* const note = A.notes + kNote * c;
    const int more = note[0];
    if (more <= 0) return;
    const int row0 = note[1], h = note[2], row_first = note[3], n_rows = note[4];
    for (int i = threadIdx.x; i < n_rows * quads; i += 128) {
        const int r = i / quads, d = 4 * (i % quads);
        auto part = [&](int k) { return (int64_t)(2 * (c + k) + (k == 0 ? 1 : 0)) * unit_rows + r; };
        float M = -INFINITY, sum = 0.0f;
#pragma unroll 4
        for (int k = 0; k <= more; ++k) M = fmaxf(M, A.part_ml[2 * part(k)]);
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int k = 0; k <= more; ++k) {
            const float2 ml = *reinterpret_cast<const float2*>(A.part_ml + 2 * part(k));
            const float4 v = *reinterpret_cast<const float4*>(A.part_o + part(k) * D + d);
            const float f = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - M);         // (nothing of it is seen: O is 0)
            sum = fmaf(f, ml.y, sum);
            a.x = fmaf(f, v.x, a.x); a.y = fmaf(f, v.y, a.y); a.z = fmaf(f, v.z, a.z); a.w = fmaf(f, v.w, a.w);
        }
        const float inv = 1.0f / sum;
        const int row = row_first + r;
        const int64_t to = ((int64_t)row0 + row / n_rep) * A.out.row_stride + (int64_t)(h * n_rep + row % n_rep) * A.out.head_stride;
        store_quad(A.out.data, A.out_dtype, to + d, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
    }
}

// kMostRows: all of a sequence's rows in one unit.  Beyond it its bytes are read again for every 24 rows: 16 x 8192, 8 x 4 heads, bf16, 130 us
// for 24 rows where the tensor-core kernel takes 190, 194 against 188 for 32, 286 against 249 for 64; 64 x 2048 204 against 264, then 362 against
// 266.  (One sequence of 32768: 60 against 69 for 8 rows, 89 and 124 against 69 for 16 and 24.)
constexpr int kMostBlocks = 3, kMostRows = 8 * kMostBlocks, kLaneRows = 2, kMostLaneRows = 4;

// Blocks of eight rows of a unit: all of a sequence's rows in one unit where registers hold them, so that its bytes are
// read once.
int unit_blocks(int64_t max_rows) {
    const int64_t need = (max_rows + 7) / 8;
    return need <= kMostBlocks ? (int)need : kMostBlocks;
}

template <int D, int NB, int RULES>
int go(const Paged8Attn& a, cudaStream_t st) {
    constexpr int kSmem = Layout<D, NB>::bytes;
    auto* const kernel = paged8_decode_kernel<D, NB, RULES>;
    const int ctas = kPerSm * num_sms();
    KIVI_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    KIVI_CUDA_OK(launch(kernel, dim3((unsigned)ctas), 32 * warps_of(NB), kSmem, st, true, a));
    KIVI_CUDA_OK(launch(paged8_fold_kernel, dim3((unsigned)(ctas - 1)), 128, 0, st, true, a, 8 * NB));
    return KIVI_OK;
}
template <int D, int NB>
int go(const Paged8Attn& a, cudaStream_t st) {
    if (a.rules.softcap > kSmallCap) return go<D, NB, kAnyCap>(a, st);
    return a.rules.softcap > 0.0f || a.rules.slopes != nullptr ? go<D, NB, kRules>(a, st) : go<D, NB, kNoRules>(a, st);
}

}  // namespace

static bool on_tensor_cores(const kivi_paged8_layer* L, int q_dtype) { return L->group_size % kTile == 0 && q_dtype == KIVI_BF16 && L->res_dtype == KIVI_BF16; }
bool paged8_decode_serves(const kivi_paged8_layer* L, const kivi_paged_batch* b, int q_dtype, int n_rep, int window) {
    if (L->head_dim != 64 && L->head_dim != 128) return false;
    const int64_t rows = (int64_t)b->max_new * n_rep;
    if (on_tensor_cores(L, q_dtype)) return rows <= kMostRows;
    // Lanes: fp32, 16 sequences of 8192 tokens, 8 heads of 128: 241 us against 790 of the general kernel for two rows, 450 against 790 for four (4
    // heads, eight rows: 452 against 347); one sequence of 2048, 12 heads of 64: 31 against 34; four of 712 29 against 26 (a second
    // launch); four of 2048 with four rows 66 against 60.
    const int len = window > 0 && window < b->max_len ? window : b->max_len;
    return rows <= kMostLaneRows && len >= (rows <= kLaneRows ? 2048 : 4096);
}
int paged8_decode_notes() { return kPerSm * num_sms() * kNote; }           // whole numbers behind the partials
size_t paged8_decode_parts(int64_t max_rows) { return (size_t)kPerSm * num_sms() * 2 * 8 * unit_blocks(max_rows); }          // rows of partials

namespace {
template <typename T, int D, int NR> int go_lanes(const Paged8Attn& a, cudaStream_t st) {
    const int ctas = kPerSm * num_sms();
    KIVI_CUDA_OK(launch(paged8_lanes_kernel<T, D, NR>, dim3((unsigned)ctas), 32 * kLaneWarps, 0, st, true, a));
    KIVI_CUDA_OK(launch(paged8_fold_kernel, dim3((unsigned)(ctas - 1)), 128, 0, st, true, a, NR));
    return KIVI_OK;
}
template <typename T, int D> int go_lanes(const Paged8Attn& a, cudaStream_t st) {
    return (int64_t)a.b.max_new * a.n_rep == 1 ? go_lanes<T, D, 1>(a, st) : go_lanes<T, D, kLaneRows>(a, st);
}
}  // namespace

int run_paged8_decode(const Paged8Attn& a, cudaStream_t st) {
    if (!on_tensor_cores(&a.L, a.q_dtype)) {
        if (a.L.res_dtype == KIVI_F32) return a.L.head_dim == 64 ? go_lanes<float, 64>(a, st) : go_lanes<float, 128>(a, st);
        return a.L.head_dim == 64 ? go_lanes<__nv_bfloat16, 64>(a, st) : go_lanes<__nv_bfloat16, 128>(a, st);
    }
    const int nb = unit_blocks((int64_t)a.b.max_new * a.n_rep);
    if (a.L.head_dim == 64) return nb == 1 ? go<64, 1>(a, st) : nb == 2 ? go<64, 2>(a, st) : go<64, 3>(a, st);
    return nb == 1 ? go<128, 1>(a, st) : nb == 2 ? go<128, 2>(a, st) : go<128, 3>(a, st);
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
