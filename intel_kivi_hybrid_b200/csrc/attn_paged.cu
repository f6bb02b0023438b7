// Attention of a step's rows over a paged cache, on the CUDA cores: every shape the cache
// takes, fp32 accuracy.
//
// The rows of one sequence and KV head -- (new token, query head) pairs, n_rep heads side
// by side -- are cut into blocks of RT; a CTA takes a block and a piece of the sequence's
// tokens, 64 at a time: dequantized into shared memory (code * scale + zero in one
// rounding) or copied from the window or the step's own rows, scored, folded into running
// maxima and sums, and contracted with the values.  A thread has RPT rows and four tokens
// of the scores, RPT rows and D/16 channels of the output; the 16 threads of a row are half
// a warp, so weights change hands without a block barrier.
// Row i of a sequence sees its tokens 0 .. held + i; blocks stop at their last row's.
//
// Bound by the FMA pipe with 64 rows, by the latency of a tile's loads with few.  Where a tile's
// tokens are is looked up a tile ahead, and a thread has the loads of four quads of channels on
// their way: GPT-2-small in fp32, one token over 712 23.5 -> 14.3 us, 4 x 160 over 512 49 -> 43.
#include "paged_common.cuh"
#include "paged_attention.cuh"

#include <type_traits>

namespace kivi {
namespace {

__device__ int g_fault = 0;

constexpr int kTile = 64;                                // tokens in shared memory at a time
constexpr int kAtOnce = 4;
constexpr int kTensorRows = 256;                         // of a CTA on the tensor cores

// DT: head_dim 64 or 128, or 256 for any up to that.
// AGAIN: the same for the pieces of the tensor-core kernel's blocks (256 rows) that it has flagged, in place
// of what it would have written; four CTAs to such a piece.
template <int RPT, int TY, int DT, bool AGAIN = false>
__global__ void __launch_bounds__(TY * 16)
paged_attention_kernel(PagedAttnArgs A) {
    constexpr int RT = RPT * TY, kThreads = TY * 16, NC = DT / 64;       // NC: quads of channels a thread has
    extern __shared__ __align__(16) float smem_f[];
    __shared__ int place_s[2], in_group[2][kTile];
    __shared__ int64_t at_s[2][kTile];                   // of a tile's tokens: group of the pages, or element of the window, or row
    stream_order();
    settle_args(A);
    const kivi_paged_layer& L = A.L;
    const int D = DT == 256 ? L.head_dim : DT, G = L.group_size, R = L.residual_cap, H = L.num_kv_heads, S = D + 4, Q = G / 4, W = D < 64 ? D : 64;
    float* const q_s = smem_f;                           // [RT][S]
    float* const k_s = q_s + RT * S;                     // [kTile][S]
    float* const v_s = k_s + kTile * S;                  // [kTile][S]
    float* const p_s = v_s + kTile * S;                  // [RT][kTile + 4]
    const int h = blockIdx.y, tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    constexpr int BT = AGAIN ? kTensorRows : RT;         // rows of a block
    const int block = AGAIN ? blockIdx.x / (BT / RT) : blockIdx.x, row_in_block = AGAIN ? blockIdx.x % (BT / RT) * RT : 0;
    const int64_t unit = (int64_t)block * H + h;
    // (a block that no sequence has may hold any flag, and is not found below)
    if (AGAIN && A.rough[unit * A.pieces + blockIdx.z] == 0) return;
    if (!AGAIN && blockIdx.x + blockIdx.y + blockIdx.z == 0) report_left_out(L, A.b, &g_fault);
    if (tid < 32) {
        const ItemPlace p = find_item(block, A.b.num_seqs, [&](int i) {
            PagedSeq q;
            load_seq(L, A.b, i, q);
            return (int)(((int64_t)q.n * A.n_rep + BT - 1) / BT);
        });
        if (tid == 0) { place_s[0] = p.s; place_s[1] = p.sub; }
    }
    __syncthreads();
    const int s = place_s[0];
    if (s >= A.b.num_seqs) return;
    PagedSeq q;
    load_seq(L, A.b, s, q);                              // (sequences left out have no items)
    const int n_rep = A.n_rep, rows = q.n * n_rep, row_first = place_s[1] * BT + row_in_block;
    const int n_rows = rows - row_first < RT ? rows - row_first : RT;
    if (AGAIN && n_rows <= 0) return;
    const int inside = min(quant_of(q.held + q.n, G, R), q.held);        // tokens read from pages
    const int last_row = min(place_s[1] * BT + BT, rows) - 1;
    const int keys = q.held + last_row / n_rep + 1;      // tokens the block's last row sees
    const int t_begin = blockIdx.z * A.chunk;
    if (t_begin >= keys) return;
    const int t_end = min(t_begin + A.chunk, keys);
    const bool whole = t_end == keys && blockIdx.z == 0;                 // the only piece of this block
    const bool vec = A.vec != 0;

    // where a tile's tokens are, looked up a tile ahead: one division and one look at the page table a token
    auto look_up = [&](int t0, int buf) {
        const int t = t0 + tid;
        if (tid >= kTile || t >= t_end) return;
        int64_t at;
        int tt = 0;
        if (t < inside) {
            const int page = t / L.page_tokens, in_page = t - page * L.page_tokens;
            at = ((int64_t)page_of(L, q, t, &g_fault) * H + h) * (L.page_tokens / G) + in_page / G;
            tt = in_page % G;
        } else if (t < q.held) {
            at = (((int64_t)q.slot * H + h) * R + ring_slot(t, A.b.ring_shift, R)) * D;
        } else {
            at = (int64_t)q.row0 + (t - q.held);
        }
        at_s[buf][tid] = at;
        in_group[buf][tid] = tt;
    };
    look_up(t_begin, 0);
    for (int i = tid; i < RT * (D / 4); i += kThreads) {
        const int r = i / (D / 4), d = 4 * (i % (D / 4));
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < n_rows) {
            const int row = row_first + r;
            x = load4_as(A.q, A.q_dtype, (int64_t)q.row0 + row / n_rep, h * n_rep + row % n_rep, d, vec);
        }
        *reinterpret_cast<float4*>(q_s + r * S + d) = x;
    }
    float m[RPT], l[RPT], o[RPT][4 * NC];
    int last[RPT];                                       // last token that the row sees
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        m[i] = -INFINITY; l[i] = 0.0f;
        const int r = ty * RPT + i;
        last[i] = r < n_rows ? q.held + (row_first + r) / n_rep : -1;
#pragma unroll
        for (int c = 0; c < 4 * NC; ++c) o[i][c] = 0.0f;
    }
    int buf = 0;
    for (int t0 = t_begin; t0 < t_end; t0 += kTile, buf ^= 1) {
        __syncthreads();                                 // the tile before has been read, this one's places are known
        const int64_t* const at = at_s[buf];
        if (t0 + kTile <= inside && kTile * (DT == 256 ? 0 : DT / 4) % (kAtOnce * kThreads) == 0 && DT != 256) {
            // all in pages: the loads of kAtOnce quads of channels are on their way together
            for (int i0 = tid; i0 < kTile * (D / 4); i0 += kAtOnce * kThreads) {
                uint32_t w[kAtOnce], c[kAtOnce];
                float4 ks[kAtOnce], kz[kAtOnce];
                float vs[kAtOnce], vz[kAtOnce];
#pragma unroll
                for (int u = 0; u < kAtOnce; ++u) {
                    const int i = i0 + u * kThreads, j = i / (D / 4), d = 4 * (i % (D / 4)), tt = in_group[buf][j];
                    const int64_t g = at[j], x = g * D + vmeta_index(tt, d / G, D, G);
                    w[u] = *reinterpret_cast<const uint32_t*>(L.k_codes + g * (D * Q) + kblock_offset(d, tt >> 2, Q, W));
                    c[u] = L.v_codes[g * (D * Q) + vcode_offset(tt, d / 4, D, G)];
                    ks[u] = *reinterpret_cast<const float4*>(L.k_scales + g * D + d); kz[u] = *reinterpret_cast<const float4*>(L.k_zeros + g * D + d);
                    vs[u] = L.v_scales[x]; vz[u] = L.v_zeros[x];
                }
#pragma unroll
                for (int u = 0; u < kAtOnce; ++u) {
                    const int i = i0 + u * kThreads, j = i / (D / 4), d = 4 * (i % (D / 4)), sh = 2 * (in_group[buf][j] & 3);
                    *reinterpret_cast<float4*>(k_s + j * S + d) =
                        make_float4(fmaf((float)((w[u] >> sh) & 3u), ks[u].x, kz[u].x), fmaf((float)((w[u] >> (sh + 8)) & 3u), ks[u].y, kz[u].y),
                                    fmaf((float)((w[u] >> (sh + 16)) & 3u), ks[u].z, kz[u].z), fmaf((float)((w[u] >> (sh + 24)) & 3u), ks[u].w, kz[u].w));
                    *reinterpret_cast<float4*>(v_s + j * S + d) = make_float4(fmaf((float)(c[u] & 3u), vs[u], vz[u]), fmaf((float)((c[u] >> 2) & 3u), vs[u], vz[u]),
                                                                              fmaf((float)((c[u] >> 4) & 3u), vs[u], vz[u]), fmaf((float)(c[u] >> 6), vs[u], vz[u]));
                }
            }
        } else {
#pragma unroll 4
            for (int i = tid; i < kTile * (D / 4); i += kThreads) {
                const int j = i / (D / 4), d = 4 * (i % (D / 4)), t = t0 + j;
                float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
                if (t < inside) {
                    const int tt = in_group[buf][j];
                    k = packed_key4(L, at[j], tt, d);
                    v = packed_value4(L, at[j], tt, d);
                } else if (t < q.held) {
                    k = L.res_dtype == KIVI_BF16 ? load4(reinterpret_cast<const __nv_bfloat16*>(L.k_res) + at[j] + d, true) : load4(reinterpret_cast<const float*>(L.k_res) + at[j] + d, true);
                    v = L.res_dtype == KIVI_BF16 ? load4(reinterpret_cast<const __nv_bfloat16*>(L.v_res) + at[j] + d, true) : load4(reinterpret_cast<const float*>(L.v_res) + at[j] + d, true);
                } else if (t < t_end) {
                    k = load4_as(A.k, L.res_dtype, at[j], h, d, vec);
                    v = load4_as(A.v, L.res_dtype, at[j], h, d, vec);
                }
                *reinterpret_cast<float4*>(k_s + j * S + d) = k;
                *reinterpret_cast<float4*>(v_s + j * S + d) = v;
            }
        }
        look_up(t0 + kTile, buf ^ 1);
        __syncthreads();
        float sc[RPT][4];
#pragma unroll
        for (int i = 0; i < RPT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[i][j] = 0.0f;
        // Sixteen channels by themselves and then to the sum, which is rounded a sixteenth as often
        // (12 heads of 64 over 712 tokens, 2-norm error 8.7e-7 without, 4.9e-7 with; the same time).
        for (int d0 = 0; d0 < D; d0 += 16) {
            float part[RPT][4];
#pragma unroll
            for (int i = 0; i < RPT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) part[i][j] = 0.0f;
#pragma unroll
            for (int d = d0; d < d0 + 16; d += 4) {
                if (DT == 256 && d >= D) break;
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
                if (t > last[i] || t >= t_end) sc[i][j] = -INFINITY;
                mx = fmaxf(mx, sc[i][j]);
            }
#pragma unroll
            for (int x = 1; x < 16; x *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
            const float m_new = fmaxf(m[i], mx), base = m_new == -INFINITY ? 0.0f : m_new;
            const float alpha = exp2f((m[i] - base) * A.scale_log2);      // 0 while there is no maximum
            m[i] = m_new;
            l[i] *= alpha;
#pragma unroll
            for (int c = 0; c < 4 * NC; ++c) o[i][c] *= alpha;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = exp2f((sc[i][j] - base) * A.scale_log2);      // (the difference is rounded at its own size, not at the scores')
                l[i] += p;
                p_s[(ty * RPT + i) * (kTile + 4) + tx + 16 * j] = p;
            }
        }
        __syncwarp();
        // (a token that a row does not see may hold anything, infinities and NaN too: only among the step's own)
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
                        const float4 v = *reinterpret_cast<const float4*>(v_s + (j + jj) * S + d);
#pragma unroll
                        for (int i = 0; i < RPT; ++i) {
                            const float w = jj == 0 ? p[i].x : jj == 1 ? p[i].y : jj == 2 ? p[i].z : p[i].w;
                            const bool seen = !decltype(masked)::value || t0 + j + jj <= last[i];
                            o[i][4 * c] = fmaf(w, seen ? v.x : 0.0f, o[i][4 * c]); o[i][4 * c + 1] = fmaf(w, seen ? v.y : 0.0f, o[i][4 * c + 1]);
                            o[i][4 * c + 2] = fmaf(w, seen ? v.z : 0.0f, o[i][4 * c + 2]); o[i][4 * c + 3] = fmaf(w, seen ? v.w : 0.0f, o[i][4 * c + 3]);
                        }
                    }
            }
        };
        if (t0 + kTile > q.held) weigh(std::true_type{});
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
            const int64_t part = (unit * A.pieces + blockIdx.z) * BT + row_in_block + r;
            if (tx == 0) *reinterpret_cast<float2*>(A.part_ml + 2 * part) = make_float2(m[i] * A.scale_log2, l[i]);
#pragma unroll
            for (int c = 0; c < NC; ++c)
                if (4 * tx + 64 * c < D)
                    *reinterpret_cast<float4*>(A.part_o + part * D + 4 * tx + 64 * c) = make_float4(o[i][4 * c], o[i][4 * c + 1], o[i][4 * c + 2], o[i][4 * c + 3]);
        }
    }
}

// Folds the pieces of a block's rows, a thread per quad of channels of a row.
// grid = (blocks, KV heads, slices of kFoldRows rows).
constexpr int kFoldRows = 8;
__global__ void __launch_bounds__(256)
paged_merge_kernel(PagedAttnArgs A, int RT) {
    __shared__ int place_s[2];
    stream_order();
    settle_args(A);
    const kivi_paged_layer& L = A.L;
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
    const int rows = q.n * n_rep, row_first = place_s[1] * RT;
    const int n_rows = rows - row_first < RT ? rows - row_first : RT;
    const int keys = q.held + (row_first + n_rows - 1) / n_rep + 1, n_pieces = (keys + A.chunk - 1) / A.chunk;
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
            if (ml.x == -INFINITY && ml.y == 0.0f) continue;         // a piece behind the row's own token (of what it sees, NaN may be all)
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
int run_general(const PagedAttnArgs& a, int blocks, cudaStream_t st) {
    auto* const kernel = paged_attention_kernel<RPT, TY, DT>;
    // (the limit is the kernel's, not the call's: what every call sets is the most that one needs)
    constexpr size_t most = general_bytes(RPT * TY, DT);
    if (most > 48 * 1024) KIVI_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
    const size_t smem = general_bytes(RPT * TY, a.L.head_dim);
    KIVI_CUDA_OK(launch(kernel, dim3((unsigned)blocks, (unsigned)a.L.num_kv_heads, (unsigned)a.pieces), TY * 16, smem, st, true, a));
    return KIVI_OK;
}

// what the tensor cores have flagged (rows of 64 by CTAs that see in one load that there is nothing to do)
template <int DT>
int run_again(const PagedAttnArgs& a, int blocks, cudaStream_t st) {
    auto* const kernel = paged_attention_kernel<4, 16, DT, true>;
    constexpr size_t smem = general_bytes(64, DT);
    KIVI_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    KIVI_CUDA_OK(launch(kernel, dim3((unsigned)blocks * (kTensorRows / 64), (unsigned)a.L.num_kv_heads, (unsigned)a.pieces), 256, smem, st, true, a));
    return KIVI_OK;
}

}  // namespace

int paged_attention_fault_word(int* out) {
    KIVI_CUDA_OK(cudaMemcpyFromSymbol(out, g_fault, sizeof(int)));
    return KIVI_OK;
}
int paged_attention_fault_clear() {
    const int zero = 0;
    KIVI_CUDA_OK(cudaMemcpyToSymbol(g_fault, &zero, sizeof(int)));
    return KIVI_OK;
}

bool paged_tc_serves(const kivi_paged_layer* L, int q_dtype);
int run_paged_tc(const PagedAttnArgs& a, int blocks, cudaStream_t st);

bool paged_decode_serves(const kivi_paged_layer* L, int q_dtype, int64_t max_rows);
void paged_decode_plan(const kivi_paged_layer* L, const kivi_paged_batch* b, int n_rep, int* blocks_per_seq, int* gps, int* pieces);
int run_paged_decode(const PagedAttnArgs& a, int blocks_per_seq, int gps, cudaStream_t st);

// ---- the cut of a call -----------------------------------------------------------
// Rows per block, blocks (at most: what the host knows are bounds) and pieces of the
// sequences' tokens.
enum class PagedKernel { kDecode, kTensor, kGeneral };
struct PagedPlan { PagedKernel kernel; int rows, blocks, pieces, chunk; };          // (decode: chunk is groups of tokens, blocks a sequence's times sequences)

static PagedPlan plan_paged(const kivi_paged_layer* L, const kivi_paged_batch* b, int q_dtype, int n_rep, bool vec) {
    PagedPlan p;
    const int64_t rows = (int64_t)b->max_new * n_rep;
    if (vec && paged_decode_serves(L, q_dtype, rows)) {
        p.kernel = PagedKernel::kDecode;
        p.rows = 4;
        paged_decode_plan(L, b, n_rep, &p.blocks, &p.chunk, &p.pieces);
        p.blocks *= b->num_seqs;
        return p;
    }
    p.kernel = paged_tc_serves(L, q_dtype) ? PagedKernel::kTensor : PagedKernel::kGeneral;
    if (p.kernel == PagedKernel::kTensor) {
        p.rows = kTensorRows;
        const int64_t blocks = (int64_t)b->total_new * n_rep / p.rows + b->num_seqs;
        p.blocks = (int)(blocks < (1 << 30) ? blocks : (1 << 30));
        // One CTA per SM: the fewest rounds of the shortest pieces, each with the start and
        // end of a CTA on top (about four tiles).
        const int tiles = (b->max_len + 127) / 128, most = tiles < 64 ? tiles : 64;
        const int64_t units = (int64_t)p.blocks * L->num_kv_heads;
        int64_t best = INT64_MAX;
        for (int n = 1; n <= most; ++n) {
            const int per = (tiles + n - 1) / n;
            const int64_t cost = ((units * n + num_sms() - 1) / num_sms()) * (per + 4);
            if (cost < best) { best = cost; p.chunk = per * 128; p.pieces = (tiles + per - 1) / per; }
        }
        return p;
    }
    p.rows = rows <= 8 ? 8 : 64;
    const int64_t blocks = ((int64_t)b->total_new * n_rep) / p.rows + b->num_seqs;
    p.blocks = (int)(blocks < (1 << 30) ? blocks : (1 << 30));
    const int tiles = (b->max_len + kTile - 1) / kTile;
    // as many pieces as give every SM four CTAs
    int64_t want = (4 * (int64_t)num_sms() + p.blocks * (int64_t)L->num_kv_heads - 1) / (p.blocks * (int64_t)L->num_kv_heads);
    if (want > tiles) want = tiles;
    if (want > 256) want = 256;
    if (want < 1) want = 1;
    const int per = (int)((tiles + want - 1) / want);
    p.chunk = per * kTile;
    p.pieces = (tiles + per - 1) / per;
    return p;
}

}  // namespace kivi

using namespace kivi;

static int check_attention(const kivi_paged_layer* L, const kivi_paged_batch* b, int q_dtype, int n_rep) {
    if (int rc = validate_paged(L)) return rc;
    if (int rc = validate_batch(L, b)) return rc;
    KIVI_REQUIRE(n_rep >= 1 && n_rep <= 1024, "n_rep (%d) outside 1..1024", n_rep);
    KIVI_REQUIRE((int64_t)b->max_new * n_rep <= (1 << 30), "max_new * n_rep must be at most 2^30");
    KIVI_REQUIRE(q_dtype == KIVI_F32 || q_dtype == KIVI_BF16, "q dtype must be KIVI_F32 or KIVI_BF16");
    return KIVI_OK;
}

static size_t plan_bytes(const kivi_paged_layer* L, const PagedPlan& p) {
    const size_t parts = (size_t)p.blocks * L->num_kv_heads * p.pieces;
    return (p.pieces > 1 || p.kernel == PagedKernel::kDecode ? parts * p.rows * (L->head_dim + 2) * 4 : 0) + (p.kernel == PagedKernel::kTensor ? parts * 4 : 0);
}

// (enough for rows on 16-byte boundaries, and for others, which the decode kernel does not take)
extern "C" size_t kivi_paged_attention_workspace(const kivi_paged_layer* L, const kivi_paged_batch* b, int q_dtype, int n_rep) {
    if (check_attention(L, b, q_dtype, n_rep) != KIVI_OK || b->max_new == 0) return 0;
    const size_t on = plan_bytes(L, plan_paged(L, b, q_dtype, n_rep, true)), off = plan_bytes(L, plan_paged(L, b, q_dtype, n_rep, false));
    return on > off ? on : off;
}

extern "C" int kivi_paged_attention(const kivi_paged_layer* L, const kivi_paged_batch* b, const kivi_rows* q,
                                    int q_dtype, const kivi_rows* new_k, const kivi_rows* new_v, const kivi_rows* out,
                                    int out_dtype, int n_rep, float sm_scale, void* workspace, size_t workspace_bytes,
                                    void* stream) {
    if (int rc = check_attention(L, b, q_dtype, n_rep)) return rc;
    KIVI_REQUIRE(out_dtype == KIVI_F32 || out_dtype == KIVI_BF16, "out dtype must be KIVI_F32 or KIVI_BF16");
    for (const kivi_rows* r : {q, new_k, new_v, out}) {
        KIVI_REQUIRE(r != nullptr && r->data != nullptr, "q, new_k, new_v or out is null");
        KIVI_REQUIRE(r->row_stride >= 0 && r->head_stride >= 0, "q, new_k, new_v or out has a negative stride");
    }
    if (int rc = validate_in_place(out, "out", q, "q", b->total_new, L->num_kv_heads * n_rep, out_dtype == q_dtype)) return rc;
    if (b->max_new == 0) { note_launches(0); return KIVI_OK; }
    const int D = L->head_dim;
    // rows on 16-byte boundaries
    auto aligned = [](const kivi_rows& r, int dtype) {
        const int n = 16 / elem_size(dtype);
        return (reinterpret_cast<uintptr_t>(r.data) & 15u) == 0 && r.row_stride % n == 0 && r.head_stride % n == 0;
    };
    const bool vec16 = aligned(*q, q_dtype) && aligned(*new_k, L->res_dtype) && aligned(*new_v, L->res_dtype);
    const PagedPlan p = plan_paged(L, b, q_dtype, n_rep, vec16);
    const size_t need = plan_bytes(L, p);
    KIVI_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), "workspace too small: %zu bytes given, %zu needed", workspace_bytes, need);
    KIVI_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "workspace must be 16-byte aligned");
    if (sm_scale <= 0.0f) sm_scale = 1.0f / sqrtf((float)D);
    auto grid4 = [](const kivi_rows& r, int dtype) {
        return reinterpret_cast<uintptr_t>(r.data) % (4 * elem_size(dtype)) == 0 && r.row_stride % 4 == 0 && r.head_stride % 4 == 0;
    };
    PagedAttnArgs a{};
    a.L = *L; a.b = *b; a.q = *q; a.k = *new_k; a.v = *new_v; a.out = *out;
    a.q_dtype = q_dtype; a.out_dtype = out_dtype; a.n_rep = n_rep; a.scale_log2 = sm_scale * 1.4426950408889634f;
    a.pieces = p.pieces; a.chunk = p.chunk;
    a.part_o = reinterpret_cast<float*>(workspace);
    a.part_ml = a.part_o + (size_t)p.blocks * L->num_kv_heads * p.pieces * p.rows * D;
    a.vec = grid4(*q, q_dtype) && grid4(*new_k, L->res_dtype) && grid4(*new_v, L->res_dtype);
    cudaStream_t st = (cudaStream_t)stream;
    int rc;
    if (p.kernel == PagedKernel::kDecode) {
        if (int rc2 = run_paged_decode(a, p.blocks / b->num_seqs, p.chunk, st)) return rc2;
        note_launches(2);
        return KIVI_OK;
    }
    if (p.kernel == PagedKernel::kTensor) {
        a.vec = vec16;
        a.rough = reinterpret_cast<int*>(static_cast<char*>(workspace) + need) - (size_t)p.blocks * L->num_kv_heads * p.pieces;
        rc = run_paged_tc(a, p.blocks, st);
        if (!rc) rc = D == 64 ? run_again<64>(a, p.blocks, st) : run_again<128>(a, p.blocks, st);
    } else if (p.rows == 8) rc = D == 64 ? run_general<1, 8, 64>(a, p.blocks, st) : D == 128 ? run_general<1, 8, 128>(a, p.blocks, st) : run_general<1, 8, 256>(a, p.blocks, st);
    else rc = D == 64 ? run_general<4, 16, 64>(a, p.blocks, st) : D == 128 ? run_general<4, 16, 128>(a, p.blocks, st) : run_general<4, 16, 256>(a, p.blocks, st);
    if (rc) return rc;
    int launches = p.kernel == PagedKernel::kTensor ? 2 : 1;
    if (p.pieces > 1) {
        KIVI_CUDA_OK(launch(paged_merge_kernel, dim3((unsigned)p.blocks, (unsigned)L->num_kv_heads, (unsigned)((p.rows + kFoldRows - 1) / kFoldRows)), 256, 0, st, true, a, p.rows));
        ++launches;
    }
    note_launches(launches);
    return KIVI_OK;
}
