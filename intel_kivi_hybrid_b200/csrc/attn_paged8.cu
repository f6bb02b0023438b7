// Attention of a step's rows over a paged cache in 8 bits, on the CUDA cores: every shape
// the cache takes, fp32 accuracy.
//
//   x = rules(q k),  out = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m)   over the tokens a row sees
//
// The rows of one sequence and KV head -- (new token, query head) pairs, n_rep heads side
// by side -- are cut into blocks of RT; a CTA takes a block and a piece of the tokens that
// any of them sees, 64 at a time: turned into numbers in shared memory or copied from the
// window or the step's own rows, scored, folded into running maxima and sums, and contracted
// with the values.  A thread has RPT rows and four tokens of the scores, RPT rows and D/16
// channels of the output; the 16 threads of a row are half a warp, so weights change hands
// without a block barrier.
//
// Bound by the FMA pipe with 64 rows (4 x 160 tokens of GPT-2-small over 512 53 us; weights of tokens beside values that are not
// finite are selected token by token, in all tiles of rows that cost 59), by shared memory with few: bytes loaded a tile ahead into
// registers changed nothing (16 x 8192 tokens, 8 x 4 heads, fp32: 753 us, 792; up to four rows of long sequences go elsewhere).
#include "paged8_attention.cuh"

#include <type_traits>

namespace kivi {
namespace {

__device__ int g_fault = 0;

constexpr int kTile = 64;                                // tokens in shared memory at a time

// DT: head_dim 64 or 128, or 256 for any up to that.
template <int RPT, int TY, int DT>
__global__ void __launch_bounds__(TY * 16)
paged8_attention_kernel(Paged8Attn A) {
    constexpr int RT = RPT * TY, kThreads = TY * 16, NC = DT / 64;       // NC: quads of channels a thread has
    extern __shared__ __align__(16) float smem_f[];
    __shared__ int place_s[2], in_page_s[2][kTile / 16];
    __shared__ int64_t unit_s[2][kTile / 16];            // of a tile's sixteens: page and head
    __shared__ float2 scales_s[2][kTile / 16];
    __shared__ int odd_s[2];                             // the tile has a value that is not finite
    stream_order();
    settle_args(A);
    const kivi_paged8_layer& L = A.L;
    const int D = DT == 256 ? L.head_dim : DT, G = L.group_size, R = L.residual_cap, H = L.num_kv_heads, S = D + 4, run = value8_run(G);
    float* const q_s = smem_f;                           // [RT][S]
    float* const k_s = q_s + RT * S;                     // [kTile][S]
    float* const v_s = k_s + kTile * S;                  // [kTile][S]
    float* const p_s = v_s + kTile * S;                  // [RT][kTile + 4]
    const int h = blockIdx.y, tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int64_t unit = (int64_t)blockIdx.x * H + h;
    if (blockIdx.x + blockIdx.y + blockIdx.z == 0) report_left_out(L, A.b, &g_fault);
    if (tid < 32) {
        const ItemPlace p = find_item(blockIdx.x, A.b.num_seqs, [&](int i) {
            PagedSeq q;
            load_seq(L, A.b, i, q);
            return (int)(((int64_t)q.n * A.n_rep + RT - 1) / RT);
        });
        if (tid == 0) { place_s[0] = p.s; place_s[1] = p.sub; }
    }
    __syncthreads();
    const int s = place_s[0];
    if (s >= A.b.num_seqs) return;
    PagedSeq q;
    load_seq(L, A.b, s, q);                              // (sequences left out have no items)
    const int n_rep = A.n_rep, rows = q.n * n_rep, row_first = place_s[1] * RT;
    const int n_rows = rows - row_first < RT ? rows - row_first : RT, total = q.held + q.n;
    const int inside = min(quant_of(total, G, R), q.held);               // tokens read from pages
    const int window = A.rules.window, prefix = prefix_of(A.rules, s, total);
    const Span span = span_of(kTile, total, q.held + row_first / n_rep, q.held + (row_first + n_rows - 1) / n_rep, window, prefix);
    const int v_begin = blockIdx.z * A.chunk;
    if (v_begin >= span.n) return;
    const int v_end = min(v_begin + A.chunk, span.n);
    const bool whole = span.n <= A.chunk;                // the only piece of this block
    const bool vec = A.vec != 0;

    // where a tile's sixteens are, looked up a tile ahead (blocks are whole sixteens)
    auto look_up = [&](int v, int buf) {
        if (tid >= kTile / 16 || v >= v_end) return;
        const int t = span.tile(v) * kTile + 16 * tid;
        if (t >= inside) return;
        const int page = t / L.page_tokens, in_page = t - page * L.page_tokens;
        const int64_t u = (int64_t)page_of(L, q, t, &g_fault) * H + h, at = u * (L.page_tokens / G) + in_page / G;
        unit_s[buf][tid] = u;
        in_page_s[buf][tid] = in_page;
        scales_s[buf][tid] = make_float2(L.k_scales[at], L.v_scales[at]);
    };
    look_up(v_begin, 0);
    if (tid < 2) odd_s[tid] = 0;
    for (int i = tid; i < RT * (D / 4); i += kThreads) {
        const int r = i / (D / 4), d = 4 * (i % (D / 4));
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < n_rows) {
            const int row = row_first + r;
            x = load4_as(A.q, A.q_dtype, (int64_t)q.row0 + row / n_rep, h * n_rep + row % n_rep, d, vec);
        }
        *reinterpret_cast<float4*>(q_s + r * S + d) = x;
    }
    // Scores are kept as they are contracted where nothing is done to them, else as the rules leave them: differences to
    // the maximum are then rounded at their own size.
    const bool capped = A.rules.softcap > 0.0f, plain = !capped && A.rules.slopes == nullptr;
    const float to_log2 = (plain ? A.scale : 1.0f) * 1.4426950408889634f;
    const float inv_cap = capped ? 1.0f / A.rules.softcap : 0.0f;
    float m[RPT], l[RPT], o[RPT][4 * NC], slope[RPT];
    int place[RPT], from[RPT];                           // of the row, and of its window's first token
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        m[i] = -INFINITY; l[i] = 0.0f;
        const int r = ty * RPT + i, row = row_first + r;
        place[i] = r < n_rows ? q.held + row / n_rep : -1;
        from[i] = window_from(place[i], window);
        slope[i] = r < n_rows && A.rules.slopes ? A.rules.slopes[h * n_rep + row % n_rep] : 0.0f;
#pragma unroll
        for (int c = 0; c < 4 * NC; ++c) o[i][c] = 0.0f;
    }
    auto sees = [&](int i, int t) { return (t <= place[i] && t >= from[i]) || (t < prefix && place[i] >= 0); };
    int buf = 0;
    for (int v = v_begin; v < v_end; ++v, buf ^= 1) {
        const int t0 = span.tile(v) * kTile;
        __syncthreads();                                 // the tile before has been read, this one's places are known
        // four tokens that share a word of a value run, of four channels
#pragma unroll 2
        for (int i = tid; i < kTile / 4 * (D / 4); i += kThreads) {
            const int set = i / (D / 4), d = 4 * (i % (D / 4)), six = set >> 2, j0 = 16 * six + 2 * (set & 3);
            const int at_j[4] = {j0, j0 + 1, j0 + 8, j0 + 9};
            float4 k[4], x[4];
            if (t0 + 16 * six < inside) {
                const int in_page = in_page_s[buf][six];
                const uint8_t* const kc = L.k_codes + unit_s[buf][six] * L.page_tokens * D;
                const uint8_t* const vc = L.v_codes + unit_s[buf][six] * L.page_tokens * D;
                const float2 sc = scales_s[buf][six];
                uint32_t kw[4], vw[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    kw[e] = *reinterpret_cast<const uint32_t*>(kc + key8_offset(in_page + at_j[e] - 16 * six, d, D));
                    vw[e] = *reinterpret_cast<const uint32_t*>(vc + value8_offset(in_page + 2 * (set & 3), d + e, D, run));
                }
                float y[4][4];                           // [channel][token]
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float4 a = e4m3x4(kw[e]), b = e4m3x4(vw[e]);
                    k[e] = make_float4(a.x * sc.x, a.y * sc.x, a.z * sc.x, a.w * sc.x);
                    y[e][0] = b.x * sc.y; y[e][1] = b.y * sc.y; y[e][2] = b.z * sc.y; y[e][3] = b.w * sc.y;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = make_float4(y[0][e], y[1][e], y[2][e], y[3][e]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int t = t0 + at_j[e];
                if (t >= inside) {
                    k[e] = x[e] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (t < q.held) {
                        const int64_t at = (((int64_t)q.slot * H + h) * R + ring_slot(t, 0, R)) * D + d;
                        k[e] = L.res_dtype == KIVI_BF16 ? load4(reinterpret_cast<const __nv_bfloat16*>(L.k_res) + at, true) : load4(reinterpret_cast<const float*>(L.k_res) + at, true);
                        x[e] = L.res_dtype == KIVI_BF16 ? load4(reinterpret_cast<const __nv_bfloat16*>(L.v_res) + at, true) : load4(reinterpret_cast<const float*>(L.v_res) + at, true);
                    } else if (t < total) {
                        k[e] = load4_as(A.k, L.res_dtype, (int64_t)q.row0 + (t - q.held), h, d, vec);
                        x[e] = load4_as(A.v, L.res_dtype, (int64_t)q.row0 + (t - q.held), h, d, vec);
                    }
                    // (the sum of the magnitudes is not finite where one of them is not, or all are near the largest number)
                    if (!(fabsf(x[e].x) + fabsf(x[e].y) + fabsf(x[e].z) + fabsf(x[e].w) <= 3.4028234e38f)) odd_s[buf] = 1;
                }
                *reinterpret_cast<float4*>(k_s + at_j[e] * S + d) = k[e];
                *reinterpret_cast<float4*>(v_s + at_j[e] * S + d) = x[e];
            }
        }
        look_up(v + 1, buf ^ 1);
        __syncthreads();
        const bool odd = odd_s[buf] != 0;
        if (tid == 0) odd_s[buf ^ 1] = 0;                // (the next tile's is written behind the next barrier)
        float sc[RPT][4];
#pragma unroll
        for (int i = 0; i < RPT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[i][j] = 0.0f;
        // sixteen channels by themselves and then to the sum, which is rounded a sixteenth as often
        for (int d0 = 0; d0 < D; d0 += 16) {
            float part[RPT][4];
#pragma unroll
            for (int i = 0; i < RPT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) part[i][j] = 0.0f;
#pragma unroll
            for (int d = d0; d < d0 + 16; d += 4) {
                float4 a[RPT], b[4];
#pragma unroll
                for (int i = 0; i < RPT; ++i) a[i] = *reinterpret_cast<const float4*>(q_s + (ty * RPT + i) * S + d);
#pragma unroll
                for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const float4*>(k_s + (tx + 16 * j) * S + d);
#pragma unroll
                for (int i = 0; i < RPT; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        part[i][j] = fmaf(a[i].x, b[j].x, fmaf(a[i].y, b[j].y, fmaf(a[i].z, b[j].z, fmaf(a[i].w, b[j].w, part[i][j]))));
            }
#pragma unroll
            for (int i = 0; i < RPT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) sc[i][j] += part[i][j];
        }
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int t = t0 + tx + 16 * j;
                if (!plain) {
                    sc[i][j] = capped ? A.rules.softcap * tanhf(sc[i][j] * A.scale * inv_cap) : sc[i][j] * A.scale;
                    sc[i][j] = fmaf(slope[i], (float)(t - place[i]), sc[i][j]);
                }
                if (!sees(i, t)) sc[i][j] = -INFINITY;
                mx = fmaxf(mx, sc[i][j]);
            }
#pragma unroll
            for (int x = 1; x < 16; x *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
            const float m_new = fmaxf(m[i], mx), base = m_new == -INFINITY ? 0.0f : m_new;
            const float alpha = exp2f((m[i] - base) * to_log2);      // 0 while there is no maximum
            m[i] = m_new;
            l[i] *= alpha;
#pragma unroll
            for (int c = 0; c < 4 * NC; ++c) o[i][c] *= alpha;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = exp2f((sc[i][j] - base) * to_log2);
                l[i] += p;
                p_s[(ty * RPT + i) * (kTile + 4) + tx + 16 * j] = p;
            }
        }
        __syncwarp();
        // (a token that a row does not see may hold anything, infinities and NaN too: its weight is 0, which does not do then)
        auto weigh = [&](auto masked) {
#pragma unroll 2
            for (int j = 0; j < kTile; j += 4) {
                float4 p[RPT];
#pragma unroll
                for (int i = 0; i < RPT; ++i) p[i] = *reinterpret_cast<const float4*>(p_s + (ty * RPT + i) * (kTile + 4) + j);
#pragma unroll
                for (int jj = 0; jj < 4; ++jj)
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        const int d = 4 * tx + 64 * c;
                        if (DT == 256 && d >= D) break;
                        const float4 x = *reinterpret_cast<const float4*>(v_s + (j + jj) * S + d);
#pragma unroll
                        for (int i = 0; i < RPT; ++i) {
                            const float w = jj == 0 ? p[i].x : jj == 1 ? p[i].y : jj == 2 ? p[i].z : p[i].w;
                            const bool seen = !decltype(masked)::value || sees(i, t0 + j + jj);
                            o[i][4 * c] = fmaf(w, seen ? x.x : 0.0f, o[i][4 * c]); o[i][4 * c + 1] = fmaf(w, seen ? x.y : 0.0f, o[i][4 * c + 1]);
                            o[i][4 * c + 2] = fmaf(w, seen ? x.z : 0.0f, o[i][4 * c + 2]); o[i][4 * c + 3] = fmaf(w, seen ? x.w : 0.0f, o[i][4 * c + 3]);
                        }
                    }
            }
        };
        if (odd) weigh(std::true_type{});
        else weigh(std::false_type{});
        __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
#pragma unroll
        for (int x = 1; x < 16; x *= 2) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
        const int r = ty * RPT + i, row = row_first + r;
        if (r >= n_rows) continue;
        if (whole) {
            const float inv = 1.0f / l[i];               // (a row sees itself: l > 0)
            const int64_t at = ((int64_t)q.row0 + row / n_rep) * A.out.row_stride + (int64_t)(h * n_rep + row % n_rep) * A.out.head_stride;
#pragma unroll
            for (int c = 0; c < NC; ++c)
                if (4 * tx + 64 * c < D)
                    store_quad(A.out.data, A.out_dtype, at + 4 * tx + 64 * c, make_float4(o[i][4 * c] * inv, o[i][4 * c + 1] * inv, o[i][4 * c + 2] * inv, o[i][4 * c + 3] * inv));
        } else {
            const int64_t part = (unit * A.pieces + blockIdx.z) * RT + r;
            if (tx == 0) *reinterpret_cast<float2*>(A.part_ml + 2 * part) = make_float2(m[i] * to_log2, l[i]);
#pragma unroll
            for (int c = 0; c < NC; ++c)
                if (4 * tx + 64 * c < D)
                    *reinterpret_cast<float4*>(A.part_o + part * D + 4 * tx + 64 * c) = make_float4(o[i][4 * c], o[i][4 * c + 1], o[i][4 * c + 2], o[i][4 * c + 3]);
        }
    }
}

// Folds the pieces of a block's rows, a thread per quad of channels of a row.
// grid = (blocks, KV heads, slices of kFoldRows rows).  RT: rows of a block, T: tokens of a tile.
constexpr int kFoldRows = 8;
__global__ void __launch_bounds__(256)
paged8_merge_kernel(Paged8Attn A, int RT, int T) {
    __shared__ int place_s[2];
    stream_order();
    settle_args(A);
    const kivi_paged8_layer& L = A.L;
    const int D = L.head_dim, H = L.num_kv_heads, h = blockIdx.y, n_rep = A.n_rep;
    if (threadIdx.x < 32) {
        const ItemPlace p = find_item(blockIdx.x, A.b.num_seqs, [&](int i) {
            PagedSeq q;
            load_seq(L, A.b, i, q);
            return (int)(((int64_t)q.n * n_rep + RT - 1) / RT);
        });
        if (threadIdx.x == 0) { place_s[0] = p.s; place_s[1] = p.sub; }
    }
    __syncthreads();
    const int s = place_s[0];
    if (s >= A.b.num_seqs) return;
    PagedSeq q;
    load_seq(L, A.b, s, q);
    const int rows = q.n * n_rep, row_first = place_s[1] * RT, total = q.held + q.n;
    const int n_rows = rows - row_first < RT ? rows - row_first : RT;
    const Span span = span_of(T, total, q.held + row_first / n_rep, q.held + (row_first + n_rows - 1) / n_rep, A.rules.window, prefix_of(A.rules, s, total));
    const int n_pieces = (span.n + A.chunk - 1) / A.chunk;
    if (n_pieces <= 1) return;
    const int quads = D / 4;
    const int64_t part0 = ((int64_t)blockIdx.x * H + h) * A.pieces;
    for (int i = threadIdx.x; i < kFoldRows * quads; i += 256) {
        const int r = blockIdx.z * kFoldRows + i / quads, d = 4 * (i % quads);
        if (r >= n_rows) break;
        float M = -INFINITY, sum = 0.0f;
        for (int p = 0; p < n_pieces; ++p) M = fmaxf(M, A.part_ml[2 * ((part0 + p) * RT + r)]);
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int p = 0; p < n_pieces; ++p) {
            const float2 ml = *reinterpret_cast<const float2*>(A.part_ml + 2 * ((part0 + p) * RT + r));
            if (ml.x == -INFINITY && ml.y == 0.0f) continue;         // a piece that the row sees nothing of (of what it sees, NaN may be all)
            const float w = exp2f(ml.x - M);
            const float4 v = *reinterpret_cast<const float4*>(A.part_o + ((part0 + p) * RT + r) * D + d);
            sum = fmaf(w, ml.y, sum);
            a.x = fmaf(w, v.x, a.x); a.y = fmaf(w, v.y, a.y); a.z = fmaf(w, v.z, a.z); a.w = fmaf(w, v.w, a.w);
        }
        const float inv = 1.0f / sum;
        const int row = row_first + r;
        const int64_t at = ((int64_t)q.row0 + row / n_rep) * A.out.row_stride + (int64_t)(h * n_rep + row % n_rep) * A.out.head_stride;
        store_quad(A.out.data, A.out_dtype, at + d, make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv));
    }
}

constexpr size_t general_bytes(int rows, int D) { return ((size_t)(rows + 2 * kTile) * (D + 4) + (size_t)rows * (kTile + 4)) * 4; }

template <int RPT, int TY, int DT>
int run_general(const Paged8Attn& a, int blocks, cudaStream_t st) {
    auto* const kernel = paged8_attention_kernel<RPT, TY, DT>;
    // (the limit is the kernel's, not the call's: what every call sets is the most that one needs)
    constexpr size_t most = general_bytes(RPT * TY, DT);
    static_assert(most <= 227 * 1024, "shared memory of a CTA");
    if (most > 48 * 1024) KIVI_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
    const size_t smem = general_bytes(RPT * TY, a.L.head_dim);
    KIVI_CUDA_OK(launch(kernel, dim3((unsigned)blocks, (unsigned)a.L.num_kv_heads, (unsigned)a.pieces), TY * 16, smem, st, true, a));
    return KIVI_OK;
}

}  // namespace

int paged8_attention_fault_word(int* out) {
    KIVI_CUDA_OK(cudaMemcpyFromSymbol(out, g_fault, sizeof(int)));
    return KIVI_OK;
}
int paged8_attention_fault_clear() {
    const int zero = 0;
    KIVI_CUDA_OK(cudaMemcpyToSymbol(g_fault, &zero, sizeof(int)));
    return KIVI_OK;
}

bool paged8_decode_serves(const kivi_paged8_layer* L, const kivi_paged_batch* b, int q_dtype, int n_rep, int window);
size_t paged8_decode_parts(int64_t max_rows);
int paged8_decode_notes();
int run_paged8_decode(const Paged8Attn& a, cudaStream_t st);
bool paged8_tc_serves(const kivi_paged8_layer* L, int q_dtype);
int run_paged8_tc(const Paged8Attn& a, int blocks, cudaStream_t st);

// ---- the cut of a call -----------------------------------------------------------
// Rows per block, blocks (at most: what the host knows are bounds) and pieces of the tiles that a block sees.
enum class Paged8Kernel { kDecode, kTensor, kGeneral };
constexpr int kTensorRows = 256, kTensorTile = 128;      // of a CTA on the tensor cores
struct Paged8Plan { Paged8Kernel kernel; int rows, blocks, pieces, chunk; };

static Paged8Plan plan_paged8(const kivi_paged8_layer* L, const kivi_paged_batch* b, int q_dtype, int n_rep, const kivi_score_rules& rules) {
    Paged8Plan p{};
    const int64_t rows = (int64_t)b->max_new * n_rep;
    if (paged8_decode_serves(L, b, q_dtype, n_rep, rules.window)) {
        p.kernel = Paged8Kernel::kDecode;
        p.rows = 1;
        p.blocks = (int)paged8_decode_parts(rows);
        p.pieces = 1;
        return p;
    }
    auto blocks_of = [&](int block_rows) {
        const int64_t blocks = (int64_t)b->total_new * n_rep / block_rows + b->num_seqs;
        return (int)(blocks < (1 << 30) ? blocks : (1 << 30));
    };
    // tiles of T tokens that a block sees (how long prefixes are the host does not know)
    auto tiles_of = [&](int T, int block_rows) {
        const int64_t all = ((int64_t)b->max_len + T - 1) / T, near = ((int64_t)rules.window + block_rows / n_rep + 1 + 2 * T) / T;
        return rules.window > 0 && rules.prefix == nullptr && near < all ? near : all;
    };
    if (paged8_tc_serves(L, q_dtype)) {
        p.kernel = Paged8Kernel::kTensor;
        p.rows = kTensorRows;
        p.blocks = blocks_of(p.rows);
        // One CTA per SM: the fewest rounds of the shortest pieces, each with the start and
        // end of a CTA on top (about four tiles).
        const int tiles = (int)tiles_of(kTensorTile, p.rows), most = tiles < 64 ? tiles : 64;
        const int64_t units = (int64_t)p.blocks * L->num_kv_heads;
        int64_t best = INT64_MAX;
        for (int n = 1; n <= most; ++n) {
            const int per = (tiles + n - 1) / n;
            const int64_t cost = ((units * n + num_sms() - 1) / num_sms()) * (per + 4);
            if (cost < best) { best = cost; p.chunk = per; p.pieces = (tiles + per - 1) / per; }
        }
        return p;
    }
    p.kernel = Paged8Kernel::kGeneral;
    // Blocks of 8 rows against blocks of 64, fp32: 16 x 1000, 8 heads of 128, 93 us against 218 for 8 rows, 206 against 220 for 16, 222 against 222
    // for 24, 371 against 228 for 32; 4 x 1000, 12 heads of 64, 36 against 67, 48 against 67, 52 against 69, 62 against 69.
    p.rows = rows <= 24 ? 8 : 64;
    p.blocks = blocks_of(p.rows);
    const int64_t tiles = tiles_of(kTile, p.rows);
    // as many pieces as give every SM four CTAs
    int64_t want = (4 * (int64_t)num_sms() + p.blocks * (int64_t)L->num_kv_heads - 1) / (p.blocks * (int64_t)L->num_kv_heads);
    if (want > tiles) want = tiles;
    if (want > 256) want = 256;
    if (want < 1) want = 1;
    p.chunk = (int)((tiles + want - 1) / want);
    p.pieces = (int)((tiles + p.chunk - 1) / p.chunk);
    return p;
}

}  // namespace kivi

using namespace kivi;

static int check_attention8(const kivi_paged8_layer* L, const kivi_paged_batch* b, int q_dtype, int n_rep, const kivi_score_rules* rules) {
    if (int rc = validate_paged8(L)) return rc;
    if (int rc = validate_batch8(L, b)) return rc;
    KIVI_REQUIRE(n_rep >= 1 && n_rep <= 1024, "n_rep (%d) outside 1..1024", n_rep);
    KIVI_REQUIRE((int64_t)b->max_new * n_rep <= (1 << 30), "max_new * n_rep must be at most 2^30");
    KIVI_REQUIRE(q_dtype == KIVI_F32 || q_dtype == KIVI_BF16, "q dtype must be KIVI_F32 or KIVI_BF16");
    if (rules != nullptr) KIVI_REQUIRE(rules->softcap <= 0.0f || (rules->softcap >= 1e-10f && rules->softcap <= 1e10f), "softcap (%g) outside 1e-10..1e10", (double)rules->softcap);
    if (rules != nullptr) KIVI_REQUIRE(rules->softcap == rules->softcap, "softcap is not a number");
    return KIVI_OK;
}

static size_t plan_bytes(const kivi_paged8_layer* L, const Paged8Plan& p) {
    if (p.kernel == Paged8Kernel::kDecode) return ((size_t)p.blocks * (L->head_dim + 2) + paged8_decode_notes()) * 4;
    return p.pieces > 1 ? (size_t)p.blocks * L->num_kv_heads * p.pieces * p.rows * (L->head_dim + 2) * 4 : 0;
}

extern "C" size_t kivi_paged8_attention_workspace(const kivi_paged8_layer* L, const kivi_paged_batch* b, int q_dtype, int n_rep, const kivi_score_rules* rules) {
    if (check_attention8(L, b, q_dtype, n_rep, rules) != KIVI_OK || b->max_new == 0) return 0;
    return plan_bytes(L, plan_paged8(L, b, q_dtype, n_rep, rules ? *rules : kivi_score_rules{}));
}

extern "C" int kivi_paged8_attention(const kivi_paged8_layer* L, const kivi_paged_batch* b, const kivi_rows* q,
                                     int q_dtype, const kivi_rows* new_k, const kivi_rows* new_v, const kivi_rows* out,
                                     int out_dtype, int n_rep, float sm_scale, const kivi_score_rules* rules, void* workspace,
                                     size_t workspace_bytes, void* stream) {
    if (int rc = check_attention8(L, b, q_dtype, n_rep, rules)) return rc;
    KIVI_REQUIRE(out_dtype == KIVI_F32 || out_dtype == KIVI_BF16, "out dtype must be KIVI_F32 or KIVI_BF16");
    for (const kivi_rows* r : {q, new_k, new_v, out}) {
        KIVI_REQUIRE(r != nullptr && r->data != nullptr, "q, new_k, new_v or out is null");
        KIVI_REQUIRE(r->row_stride >= 0 && r->head_stride >= 0, "q, new_k, new_v or out has a negative stride");
    }
    if (int rc = validate_in_place(out, "out", q, "q", b->total_new, L->num_kv_heads * n_rep, out_dtype == q_dtype)) return rc;
    KIVI_REQUIRE(!(sm_scale > 1e10f), "sm_scale (%g) is above 1e10", (double)sm_scale);
    if (b->max_new == 0) { note_launches(0); return KIVI_OK; }
    const int D = L->head_dim;
    Paged8Attn a{};
    a.rules = rules ? *rules : kivi_score_rules{};
    const Paged8Plan p = plan_paged8(L, b, q_dtype, n_rep, a.rules);
    const size_t need = plan_bytes(L, p);
    KIVI_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), "workspace too small: %zu bytes given, %zu needed", workspace_bytes, need);
    KIVI_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "workspace must be 16-byte aligned");
    auto grid4 = [](const kivi_rows& r, int dtype) {
        return reinterpret_cast<uintptr_t>(r.data) % (4 * elem_size(dtype)) == 0 && r.row_stride % 4 == 0 && r.head_stride % 4 == 0;
    };
    a.L = *L; a.b = *b; a.q = *q; a.k = *new_k; a.v = *new_v; a.out = *out;
    a.q_dtype = q_dtype; a.out_dtype = out_dtype; a.n_rep = n_rep;
    a.scale = sm_scale > 0.0f ? sm_scale : 1.0f / sqrtf((float)D);
    a.pieces = p.pieces; a.chunk = p.chunk;
    a.part_o = reinterpret_cast<float*>(workspace);
    a.part_ml = a.part_o + (p.kernel == Paged8Kernel::kDecode ? (size_t)p.blocks : (size_t)p.blocks * L->num_kv_heads * p.pieces * p.rows) * D;
    a.vec = grid4(*q, q_dtype) && grid4(*new_k, L->res_dtype) && grid4(*new_v, L->res_dtype);
    cudaStream_t st = (cudaStream_t)stream;
    if (p.kernel == Paged8Kernel::kDecode) {
        a.notes = reinterpret_cast<int*>(a.part_ml + (size_t)p.blocks * 2);
        if (int rc = run_paged8_decode(a, st)) return rc;
        note_launches(2);
        return KIVI_OK;
    }
    int rc, tile = kTile;
    if (p.kernel == Paged8Kernel::kTensor) {
        auto aligned = [](const kivi_rows& r) { return (reinterpret_cast<uintptr_t>(r.data) & 15u) == 0 && r.row_stride % 8 == 0 && r.head_stride % 8 == 0; };
        a.vec = aligned(*q) && aligned(*new_k) && aligned(*new_v);
        tile = kTensorTile;
        rc = run_paged8_tc(a, p.blocks, st);
    } else if (p.rows == 8) rc = D == 64 ? run_general<1, 8, 64>(a, p.blocks, st) : D == 128 ? run_general<1, 8, 128>(a, p.blocks, st) : run_general<1, 8, 256>(a, p.blocks, st);
    else rc = D == 64 ? run_general<4, 16, 64>(a, p.blocks, st) : D == 128 ? run_general<4, 16, 128>(a, p.blocks, st) : run_general<4, 16, 256>(a, p.blocks, st);
    if (rc) return rc;
    int launches = 1;
    if (p.pieces > 1) {
        KIVI_CUDA_OK(launch(paged8_merge_kernel, dim3((unsigned)p.blocks, (unsigned)L->num_kv_heads, (unsigned)((p.rows + kFoldRows - 1) / kFoldRows)), 256, 0, st, true, a, p.rows, tile));
        ++launches;
    }
    note_launches(launches);
    return KIVI_OK;
}
