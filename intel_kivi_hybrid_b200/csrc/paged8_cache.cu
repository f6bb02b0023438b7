// Paged cache in 8 bits: append with the rotation on the way, dense read-back.
//
// One launch per append, two kinds of CTAs:
//   * for each KV head and each block of G tokens that leaves for its page: a CTA finds the
//     block's largest key and value and rounds the block.  One for each sequence at least
//     has what stays: the tokens that go to the window.  A slot of the window is overwritten
//     by the CTA that has read it (a block that starts in the window has whole slots), so
//     nothing is ordered between CTAs; each new row is read, turned and written by one thread,
//     so that k_out may be new_k itself;
//   * behind them, rows of queries that are turned.
//
// A thread has two 8-channel vectors of a token's key, which hold each other's partners
// where halves are paired, and the same channels of its value.  Where a block is no more
// than a unit a thread (32 x 128), its numbers stay in registers from the search for the
// largest to the rounding; else they are read again, new keys from where the thread itself
// has written them.  Value codes go through shared memory, where they change from rows to
// runs of tokens (rows of 36 bytes: of 32, eight lanes meet in a bank).
//
// Bound by memory: bf16, D = 128, G = 32 moves 2 bytes per element of the rows in and out
// and 1 per element that leaves.  What it takes beyond that is latency, so CTAs an SM count: 4 x 2048 tokens
// of 8 and 32 heads, three axes, 123 us with the 100 registers that a thread would like, 74 with the 64 that leave room
// for four CTAs and with a row's angles in shared memory for all of its heads (2 x 5003 fp32: 180, 135 with three).
// One token of 64 sequences: launch and latency.
#include <float.h>

#include "paged8.cuh"

namespace kivi {
namespace {

__device__ int g_fault = 0;

constexpr int kThreads = 256;
constexpr int kTurnUnits = 8;                            // pairs of vectors of queries that a thread turns, about
constexpr int kMostTurnRows = 8;                         // rows of a CTA, whose angles are in shared memory

struct Append8Args {
    kivi_paged8_layer L;
    kivi_paged_batch b;
    kivi_rows k, v, q, q_out, k_out;
    kivi_rotary rot;
    int n_rep, items_vary, items, turn_rows;
};

template <typename T> __device__ __forceinline__ T* row_of(const kivi_rows& r, int64_t row, int head) {
    return reinterpret_cast<T*>(r.data) + row * r.row_stride + (int64_t)head * r.head_stride;
}

// eight neighbouring channels
template <bool VEC> __device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
    if constexpr (VEC) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = p[i];
    }
}
template <bool VEC> __device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
    if constexpr (VEC) {
        reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = x[i];
    }
}
template <bool VEC> __device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&x)[8]) {
    if constexpr (VEC) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __bfloat162float(p[i]);
    }
}
template <bool VEC> __device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
    if constexpr (VEC) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 t = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&t);
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = __float2bfloat16_rn(x[i]);
    }
}
template <typename T> __device__ __forceinline__ float rounded(float x) {
    if constexpr (sizeof(T) == 2) return __bfloat162float(__float2bfloat16_rn(x));
    else return x;
}

// ---- the turning of a row ----------------------------------------------------------
// D/16 units of two vectors: unit u < dim/16 of paired halves has 8u and 8u + dim/2, any
// other has 16u and 16u + 8.
__device__ __forceinline__ void places(const kivi_rotary& r, int u, int& d, int& e) {
    if (r.table != nullptr && !r.interleaved && u < r.dim / 16) { d = 8 * u; e = d + r.dim / 2; }
    else { d = 16 * u; e = d + 8; }
}
__device__ __forceinline__ int axis_row(const kivi_rotary& r, int pair, int64_t row, int64_t rows) {
    const int axis = r.pair_axis[pair];
    const bool there = (unsigned)axis < (unsigned)r.num_axes;
    const int pos = r.positions[(there ? axis : 0) * rows + row];
    const bool in = (unsigned)pos < (unsigned)r.rows;
    if (!there || !in) atomicOr(&g_fault, kPagedFault);
    return in ? pos : 0;
}
// cosines and sines of pairs p0 .. p0 + N - 1 (those that there are) of a token: at place t of its sequence, in row
// `row` of the step's `rows`
template <int N>
__device__ __forceinline__ void angles(const kivi_rotary& r, int t, int64_t row, int64_t rows, int p0, float (&c)[N], float (&s)[N]) {
    const int half = r.dim / 2;
    if (r.positions == nullptr) {
        const float* at = r.table + (int64_t)t * r.dim + p0;
        if (p0 + N <= half && ((reinterpret_cast<uintptr_t>(at) | (half * 4)) & 15u) == 0) {
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const float4 a = *reinterpret_cast<const float4*>(at + i), b = *reinterpret_cast<const float4*>(at + half + i);
                c[i] = a.x; c[i + 1] = a.y; c[i + 2] = a.z; c[i + 3] = a.w;
                s[i] = b.x; s[i + 1] = b.y; s[i + 2] = b.z; s[i + 3] = b.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) { const bool in = p0 + i < half; c[i] = in ? at[i] : 1.0f; s[i] = in ? at[half + i] : 0.0f; }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            c[i] = 1.0f; s[i] = 0.0f;
            if (p0 + i < half) {
                const float* at = r.table + (int64_t)axis_row(r, p0 + i, row, rows) * r.dim + p0 + i;
                c[i] = at[0]; s[i] = at[half];
            }
        }
    }
}
template <typename T> __device__ __forceinline__ void turn_pair(float c, float s, float& a, float& b) {
    const float t = a;
    a = rounded<T>(__fsub_rn(__fmul_rn(t, c), __fmul_rn(b, s)));
    b = rounded<T>(__fadd_rn(__fmul_rn(b, c), __fmul_rn(t, s)));
}
template <typename T>
__device__ __forceinline__ void turn_unit(const kivi_rotary& r, int u, int t, int64_t row, int64_t rows, float (&x)[8], float (&y)[8]) {
    if (r.table == nullptr) return;
    if (!r.interleaved) {
        if (u >= r.dim / 16) return;
        float c[8], s[8];
        angles(r, t, row, rows, 8 * u, c, s);
#pragma unroll
        for (int i = 0; i < 8; ++i) turn_pair<T>(c[i], s[i], x[i], y[i]);
    } else {
        float c[4], s[4];
        const int p = 8 * u;
        if (2 * p < r.dim) {
            angles(r, t, row, rows, p, c, s);
#pragma unroll
            for (int i = 0; i < 4; ++i) if (p + i < r.dim / 2) turn_pair<T>(c[i], s[i], x[2 * i], x[2 * i + 1]);
        }
        if (2 * p + 8 < r.dim) {
            angles(r, t, row, rows, p + 4, c, s);
#pragma unroll
            for (int i = 0; i < 4; ++i) if (p + 4 + i < r.dim / 2) turn_pair<T>(c[i], s[i], y[2 * i], y[2 * i + 1]);
        }
    }
}

// ---- rounding a block ----------------------------------------------------------------
__device__ __forceinline__ float finite_size(float x) {
    const float a = fabsf(x);
    return a <= FLT_MAX ? a : 0.0f;                      // (NaN: 0)
}
__device__ __forceinline__ float largest(float top, const float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, finite_size(x[i]));
    return top;
}
__device__ __forceinline__ float code_input(float x, float inv) { return x == x ? __fmul_rn(x, inv) : 0.0f; }
__device__ __forceinline__ uint2 codes8(const float (&x)[8], float inv) {
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = to_e4m3x2(code_input(x[2 * i], inv), code_input(x[2 * i + 1], inv));
    return make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
}

// ONE: a unit for a thread, whose numbers stay in registers.
template <typename T, bool VEC, bool ONE>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 4 : 3)
paged8_append_kernel(Append8Args A) {
    extern __shared__ __align__(16) uint8_t v_block[];   // [G / run][D][run + 4]
    __shared__ int place_s[2];
    __shared__ float top_s[2][kThreads / 32];
    stream_order();
    settle_paged8(A.L, A.b);
    A.k.data = settled(A.k.data); A.v.data = settled(A.v.data); A.q.data = settled(A.q.data);
    A.rot.table = settled(A.rot.table); A.rot.positions = settled(A.rot.positions); A.rot.pair_axis = settled(A.rot.pair_axis);
    const kivi_paged8_layer& L = A.L;
    const int D = L.head_dim, G = L.group_size, R = L.residual_cap, H = L.num_kv_heads, units = D / 16, tid = threadIdx.x;
    const int64_t rows_all = A.b.total_new;

    if ((int64_t)blockIdx.x >= (int64_t)A.items * H) {
        // ---------------- queries ----------------
        const int row0 = (int)(blockIdx.x - (int64_t)A.items * H) * A.turn_rows, heads = H * A.n_rep;
        float* const turn_s = reinterpret_cast<float*>(v_block);             // [turn_rows][dim]: a row's cosines and sines, for all its heads
        __shared__ int token_s[kMostTurnRows];
        if (tid < A.turn_rows) {
            const int row = row0 + tid;
            // the last sequence that starts at or before the row (none of a sequence that is left out)
            int lo = 0, hi = A.b.num_seqs;
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (A.b.cu_new[mid] <= row) lo = mid;
                else hi = mid;
            }
            PagedSeq q;
            const bool ok = load_seq(L, A.b, lo, q) && row >= q.row0 && row - q.row0 < q.n;
            token_s[tid] = ok ? q.held + (row - q.row0) : -1;
        }
        __syncthreads();
        const int dim = A.rot.dim, half = dim / 2;
        for (int i = tid; i < A.turn_rows * half; i += kThreads) {
            const int r = i / half, pair = i % half, t = token_s[r];
            if (t < 0) continue;
            const float* const at = A.rot.table + (int64_t)(A.rot.positions ? axis_row(A.rot, pair, row0 + r, rows_all) : t) * dim + pair;
            turn_s[r * dim + pair] = at[0];
            turn_s[r * dim + half + pair] = at[half];
        }
        __syncthreads();
        kivi_rotary staged = A.rot;                      // (row r of the block's own table)
        staged.table = turn_s;
        staged.positions = nullptr;
#pragma unroll 2
        for (int i = tid; i < A.turn_rows * heads * units; i += kThreads) {
            const int u = i % units, head = i / units % heads, r = i / units / heads;
            if (token_s[r] < 0) continue;
            int d, e;
            float x[8], y[8];
            places(A.rot, u, d, e);
            const T* from = row_of<const T>(A.q, row0 + r, head);
            load8<VEC>(from + d, x); load8<VEC>(from + e, y);
            turn_unit<T>(staged, u, r, 0, 0, x, y);
            T* to = row_of<T>(A.q_out, row0 + r, head);
            store8<VEC>(to + d, x); store8<VEC>(to + e, y);
        }
        return;
    }

    // sequence s has an item for each block that starts in the window (one at least) and one for
    // each whole block of new tokens
    auto fresh_blocks = [&](const PagedSeq& q) {
        const int first = (q.held + G - 1) / G * G, out = quant_of(q.held + q.n, G, R);
        return out > first ? (out - first) / G : 0;
    };
    auto window_blocks = [&](const PagedSeq& q) {
        const int first = (q.held + G - 1) / G * G, in = quant_of(q.held, G, R), out = quant_of(q.held + q.n, G, R);
        return max(1, (min(out, first) - in) / G);
    };
    const int item = (int)(blockIdx.x / (unsigned)H), h = (int)(blockIdx.x % (unsigned)H);
    int s = item, sub = 0;
    if (A.items_vary) {
        if (tid < 32) {
            const ItemPlace p = find_item(item, A.b.num_seqs, [&](int i) {
                PagedSeq q;
                load_seq(L, A.b, i, q);
                return window_blocks(q) + fresh_blocks(q);
            });
            if (tid == 0) { place_s[0] = p.s; place_s[1] = p.sub; }
        }
        __syncthreads();
        s = place_s[0]; sub = place_s[1];
    }
    if (blockIdx.x == 0) report_left_out(L, A.b, &g_fault);
    if (s >= A.b.num_seqs) return;
    PagedSeq q;
    if (!load_seq(L, A.b, s, q) || q.n == 0) return;

    const int64_t ring0 = ((int64_t)q.slot * H + h) * R;
    T* const k_ring = reinterpret_cast<T*>(L.k_res) + ring0 * D;
    T* const v_ring = reinterpret_cast<T*>(L.v_res) + ring0 * D;

    // A new token's unit, its key turned and written out.
    auto fresh_unit = [&](int t, int u, int d, int e, float (&x)[8], float (&y)[8], float (&vx)[8], float (&vy)[8]) {
        const int64_t row = (int64_t)q.row0 + (t - q.held);
        const T* k = row_of<const T>(A.k, row, h);
        const T* v = row_of<const T>(A.v, row, h);
        load8<VEC>(k + d, x); load8<VEC>(k + e, y);
        load8<VEC>(v + d, vx); load8<VEC>(v + e, vy);
        if (A.rot.table != nullptr) {
            turn_unit<T>(A.rot, u, t, row, rows_all, x, y);
            T* to = row_of<T>(A.k_out, row, h);
            store8<VEC>(to + d, x); store8<VEC>(to + e, y);
        }
    };
    auto held_unit = [&](int t, int d, int e, float (&x)[8], float (&y)[8], float (&vx)[8], float (&vy)[8]) {
        const int64_t at = (int64_t)ring_slot(t, 0, R) * D;
        load8<true>(k_ring + at + d, x); load8<true>(k_ring + at + e, y);
        load8<true>(v_ring + at + d, vx); load8<true>(v_ring + at + e, vy);
    };
    // the block of tokens t0 .. t0 + G - 1 to its page
    auto to_page = [&](int t0) {
        const int run = value8_run(G), pitch = run + 4, total = G * units;
        float k_top = 0.0f, v_top = 0.0f;
        float x[8], y[8], vx[8], vy[8];
        auto fetch = [&](int i, bool again) {
            const int t = t0 + i / units, u = i % units;
            int d, e;
            places(A.rot, u, d, e);
            if (t < q.held) held_unit(t, d, e, x, y, vx, vy);
            else if (!again) fresh_unit(t, u, d, e, x, y, vx, vy);
            else {
                const int64_t row = (int64_t)q.row0 + (t - q.held);
                const T* k = A.rot.table != nullptr ? row_of<T>(A.k_out, row, h) : row_of<T>(A.k, row, h);      // (what this thread has written)
                const T* v = row_of<const T>(A.v, row, h);
                load8<VEC>(k + d, x); load8<VEC>(k + e, y);
                load8<VEC>(v + d, vx); load8<VEC>(v + e, vy);
            }
        };
        for (int i = tid; i < total; i += kThreads) {
            fetch(i, false);
            k_top = largest(largest(k_top, x), y);
            v_top = largest(largest(v_top, vx), vy);
            if (ONE) break;
        }
        // (magnitudes order as their bits)
        k_top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(k_top)));
        v_top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v_top)));
        if ((tid & 31) == 0) { top_s[0][tid >> 5] = k_top; top_s[1][tid >> 5] = v_top; }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) { k_top = fmaxf(k_top, top_s[0][w]); v_top = fmaxf(v_top, top_s[1][w]); }
        const float k_scale = fmaxf(__fmul_rn(k_top, kPerLargest), kLeastScale), v_scale = fmaxf(__fmul_rn(v_top, kPerLargest), kLeastScale);
        const float k_inv = __frcp_rn(k_scale), v_inv = __frcp_rn(v_scale);

        const int page = q.pages[t0 / L.page_tokens], in_page = t0 % L.page_tokens;
        const bool there = (unsigned)page < (unsigned)L.num_pages;
        if (!there && tid == 0) atomicOr(&g_fault, kPagedFault);
        const int64_t unit = (int64_t)(there ? page : 0) * H + h;
        uint8_t* const k_codes = L.k_codes + unit * L.page_tokens * D;
        for (int i = tid; i < total; i += kThreads) {
            if (!ONE) fetch(i, true);
            const int j = i / units;
            int d, e;
            places(A.rot, i % units, d, e);
            if (there) {
                *reinterpret_cast<uint2*>(k_codes + key8_offset(in_page + j, d, D)) = codes8(x, k_inv);
                *reinterpret_cast<uint2*>(k_codes + key8_offset(in_page + j, e, D)) = codes8(y, k_inv);
            }
            const uint2 a = codes8(vx, v_inv), b = codes8(vy, v_inv);
            uint8_t* const to = v_block + (j / run * D) * pitch + value8_place(j % run, run);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                to[(d + c) * pitch] = (uint8_t)((c < 4 ? a.x : a.y) >> (8 * (c & 3)));
                to[(e + c) * pitch] = (uint8_t)((c < 4 ? b.x : b.y) >> (8 * (c & 3)));
            }
            if (ONE) break;
        }
        __syncthreads();
        if (there) {
            const int words = run / 4;
            uint32_t* const v_codes = reinterpret_cast<uint32_t*>(L.v_codes + (unit * L.page_tokens + in_page) * D);
            for (int i = tid; i < G * D / 4; i += kThreads) v_codes[i] = reinterpret_cast<const uint32_t*>(v_block)[i / words * (words + 1) + i % words];
            if (tid == 0) {
                const int64_t at = unit * (L.page_tokens / G) + in_page / G;
                L.k_scales[at] = k_scale;
                L.v_scales[at] = v_scale;
            }
        }
    };

    const int end = q.held + q.n, out = quant_of(end, G, R);
    const int first = (q.held + G - 1) / G * G, n_fresh = fresh_blocks(q);
    const int in = quant_of(q.held, G, R), n_window = window_blocks(q);
    if (sub >= n_window) {
        to_page(first + (sub - n_window) * G);
        return;
    }
    const int t0 = in + sub * G;
    if (t0 < min(out, first)) to_page(t0);               // (its last barrier is behind the last read of the window)
    // what no other CTA has: the tokens before the first whole new block and those behind the last
    const int lo = n_fresh ? first : end, hi = n_fresh ? first + n_fresh * G : end;
    const int rest = (lo - q.held) + (end - hi), leaving = min(out, q.held);
    for (int i = tid; i < rest * units; i += kThreads) {
        const int u = i % units, j = i / units, t = j < lo - q.held ? q.held + j : hi + (j - (lo - q.held));
        if (t < out) continue;                           // (left with the block that starts in the window: that CTA's)
        // the token of the window that had the slot, if it leaves, says whose it is
        const int had = in + (t - in) % R;
        if ((had < leaving ? (had - in) / G : t % n_window) != sub) continue;
        int d, e;
        float x[8], y[8], vx[8], vy[8];
        places(A.rot, u, d, e);
        fresh_unit(t, u, d, e, x, y, vx, vy);
        const int64_t at = (int64_t)ring_slot(t, 0, R) * D;
        store8<true>(k_ring + at + d, x); store8<true>(k_ring + at + e, y);
        store8<true>(v_ring + at + d, vx); store8<true>(v_ring + at + e, vy);
    }
}

// Four tokens, those that share a word of a value run, of four channels a thread; neighbouring
// threads take neighbouring channels, so a row leaves in whole lines.  Bound by its writes.
// grid = (pieces of rows, KV heads, sequences).  DT: head_dim, 0: as the layer says.
template <typename T, int DT>
__global__ void __launch_bounds__(256)
paged8_read_kernel(kivi_paged8_layer L, kivi_paged_batch b, const int32_t* starts, float* __restrict__ k_out, float* __restrict__ v_out) {
    stream_order();
    settle_paged8(L, b);
    starts = settled(starts);
    const int s = blockIdx.z, h = blockIdx.y, D = DT ? DT : L.head_dim, G = L.group_size, R = L.residual_cap, H = L.num_kv_heads, quads = D / 4;
    const int r0 = b.cu_new[s], r1 = b.cu_new[s + 1], held = b.seq_lens[s], start = starts[s], slot = b.slots[s];
    const int n = r1 - r0;
    if (r0 < 0 || n < 0 || r1 > b.total_new || n > b.max_new || held < 0 || held > b.max_len || start < 0 || start > held - n || slot < 0 || slot >= L.num_slots) {
        if (threadIdx.x == 0) atomicOr(&g_fault, kPagedFault);
        return;
    }
    if (n == 0) return;
    PagedSeq q{held, n, r0, slot, b.page_table + (int64_t)s * b.table_width};
    const int out = quant_of(held, G, R), run = value8_run(G);
    const int first = start / 16, sets = ((start + n + 15) / 16 - first) * 4;       // sets of four tokens
    for (int64_t i = blockIdx.x * 256 + threadIdx.x; i < (int64_t)sets * quads; i += (int64_t)gridDim.x * 256) {
        const int set = (int)(i / quads), d = 4 * (int)(i % quads), t0 = 16 * (first + set / 4) + 2 * (set & 3);
        const int token[4] = {t0, t0 + 1, t0 + 8, t0 + 9};
        float4 k[4], v[4];
        if (t0 < out) {                                  // (blocks are whole sixteens)
            const int64_t unit = (int64_t)page_of(L, q, t0, &g_fault) * H + h;
            const int in_page = t0 % L.page_tokens;
            const uint8_t* const kc = L.k_codes + unit * L.page_tokens * D;
            const uint8_t* const vc = L.v_codes + unit * L.page_tokens * D;
            const int64_t at = unit * (L.page_tokens / G) + in_page / G;
            const float ks = L.k_scales[at], vs = L.v_scales[at];
            uint32_t kw[4], vw[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                kw[e] = *reinterpret_cast<const uint32_t*>(kc + key8_offset(in_page + token[e] - t0, d, D));
                vw[e] = *reinterpret_cast<const uint32_t*>(vc + value8_offset(in_page, d + e, D, run));
            }
            float vx[4][4];                              // [channel][token]
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float4 x = e4m3x4(kw[e]), y = e4m3x4(vw[e]);
                k[e] = make_float4(x.x * ks, x.y * ks, x.z * ks, x.w * ks);
                vx[e][0] = y.x * vs; vx[e][1] = y.y * vs; vx[e][2] = y.z * vs; vx[e][3] = y.w * vs;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = make_float4(vx[0][e], vx[1][e], vx[2][e], vx[3][e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t at = (((int64_t)slot * H + h) * R + ring_slot(min(token[e], held - 1), 0, R)) * D + d;
                const T* kr = reinterpret_cast<const T*>(L.k_res) + at;
                const T* vr = reinterpret_cast<const T*>(L.v_res) + at;
                k[e] = make_float4((float)kr[0], (float)kr[1], (float)kr[2], (float)kr[3]);
                v[e] = make_float4((float)vr[0], (float)vr[1], (float)vr[2], (float)vr[3]);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int t = token[e];
            if (t < start || t >= start + n) continue;
            const int64_t to = (((int64_t)r0 + (t - start)) * H + h) * D + d;
            store_quad(k_out, KIVI_F32, to, k[e]);
            store_quad(v_out, KIVI_F32, to, v[e]);
        }
    }
}

}  // namespace

int validate_paged8(const kivi_paged8_layer* L) {
    KIVI_REQUIRE(L != nullptr, "layer is null");
    KIVI_REQUIRE(L->num_pages > 0 && L->num_kv_heads > 0 && L->num_slots > 0, "num_pages, num_kv_heads and num_slots must be positive");
    KIVI_REQUIRE(L->group_size >= 16 && L->group_size <= 256 && L->group_size % 16 == 0, "group_size (%d) must be a multiple of 16 up to 256", L->group_size);
    KIVI_REQUIRE(L->head_dim >= 16 && L->head_dim <= 256 && L->head_dim % 16 == 0, "head_dim (%d) must be a multiple of 16 up to 256", L->head_dim);
    KIVI_REQUIRE(L->page_tokens > 0 && L->page_tokens % L->group_size == 0, "page_tokens (%d) must be a multiple of group_size (%d)", L->page_tokens, L->group_size);
    KIVI_REQUIRE(L->page_tokens <= (1 << 20), "page_tokens (%d) must be at most 2^20", L->page_tokens);
    KIVI_REQUIRE(L->residual_cap >= L->group_size, "residual_cap (%d) must be at least group_size (%d)", L->residual_cap, L->group_size);
    KIVI_REQUIRE(L->num_kv_heads <= 65535, "num_kv_heads (%d) must be at most 65535", L->num_kv_heads);
    KIVI_REQUIRE(L->res_dtype == KIVI_F32 || L->res_dtype == KIVI_BF16, "res_dtype must be KIVI_F32 or KIVI_BF16");
    KIVI_REQUIRE(L->k_codes && L->k_scales && L->v_codes && L->v_scales && L->k_res && L->v_res, "a pointer of the layer is null");
    auto off = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; };
    KIVI_REQUIRE(!off(L->k_codes) && !off(L->k_scales) && !off(L->v_codes) && !off(L->v_scales) && !off(L->k_res) && !off(L->v_res),
                 "the arrays of a paged layer must start on 16-byte boundaries");
    return KIVI_OK;
}

int validate_batch8(const kivi_paged8_layer* L, const kivi_paged_batch* b) {
    kivi_paged_layer sizes{};
    sizes.group_size = L->group_size; sizes.residual_cap = L->residual_cap; sizes.page_tokens = L->page_tokens;
    if (int rc = validate_batch(&sizes, b)) return rc;
    KIVI_REQUIRE(b->ring_shift == 0, "ring_shift must be 0 for a cache in 8 bits");
    return KIVI_OK;
}

int paged8_cache_fault_word(int* out) {
    KIVI_CUDA_OK(cudaMemcpyFromSymbol(out, g_fault, sizeof(int)));
    return KIVI_OK;
}
int paged8_cache_fault_clear() {
    const int zero = 0;
    KIVI_CUDA_OK(cudaMemcpyToSymbol(g_fault, &zero, sizeof(int)));
    return KIVI_OK;
}

namespace {
int check_rows(const kivi_rows* r, const char* name) {
    KIVI_REQUIRE(r != nullptr && r->data != nullptr, "%s is null", name);
    KIVI_REQUIRE(r->row_stride >= 0 && r->head_stride >= 0, "%s has a negative stride", name);
    return KIVI_OK;
}
bool on_grid(const kivi_rows& r, int esz) {              // vectors of eight channels
    const int n = 16 / esz;
    return (reinterpret_cast<uintptr_t>(r.data) & 15u) == 0 && r.row_stride % n == 0 && r.head_stride % n == 0;
}
using AppendKernel = void (*)(Append8Args);
template <typename T> AppendKernel append_kernel(bool vec, bool one) {
    if (vec) return one ? paged8_append_kernel<T, true, true> : paged8_append_kernel<T, true, false>;
    return one ? paged8_append_kernel<T, false, true> : paged8_append_kernel<T, false, false>;
}
}  // namespace
}  // namespace kivi

using namespace kivi;

extern "C" int kivi_paged8_append(const kivi_paged8_layer* layer, const kivi_paged_batch* batch,
                                  const kivi_rows* new_k, const kivi_rows* new_v, const kivi_rotary* rotary,
                                  const kivi_rows* q, int n_rep, const kivi_rows* q_out, const kivi_rows* k_out, void* stream) {
    if (int rc = validate_paged8(layer)) return rc;
    if (int rc = validate_batch8(layer, batch)) return rc;
    const int D = layer->head_dim, G = layer->group_size, H = layer->num_kv_heads, esz = elem_size(layer->res_dtype);
    if (int rc = check_rows(new_k, "new_k")) return rc;
    if (int rc = check_rows(new_v, "new_v")) return rc;
    const bool turns = rotary != nullptr && rotary->table != nullptr, queries = q != nullptr && q->data != nullptr;
    if (turns) {
        KIVI_REQUIRE(rotary->dim > 0 && rotary->dim <= D && rotary->dim % 2 == 0, "rotary_dim (%d) must be even and at most head_dim (%d)", rotary->dim, D);
        KIVI_REQUIRE(rotary->interleaved || rotary->dim % 16 == 0, "rotary_dim (%d) must be a multiple of 16 where channels half of it apart are paired", rotary->dim);
        KIVI_REQUIRE((rotary->positions != nullptr) == (rotary->pair_axis != nullptr), "positions and pair_axis are given together or not at all");
        if (rotary->positions != nullptr) {
            KIVI_REQUIRE(rotary->num_axes >= 1, "positions need an axis");
            KIVI_REQUIRE(rotary->rows >= 1, "rotary holds no positions");
        } else {
            KIVI_REQUIRE(rotary->rows >= batch->max_len, "rotary holds %d positions, max_len is %d", rotary->rows, batch->max_len);
        }
        if (int rc = check_rows(k_out, "k_out")) return rc;
        if (int rc = validate_in_place(k_out, "k_out", new_k, "new_k", batch->total_new, H, true)) return rc;
        if (queries) {
            KIVI_REQUIRE(n_rep >= 1 && n_rep <= 1024, "n_rep (%d) outside 1..1024", n_rep);
            if (int rc = check_rows(q_out, "q_out")) return rc;
            if (int rc = validate_in_place(q_out, "q_out", q, "q", batch->total_new, H * n_rep, true)) return rc;
        }
    } else {
        KIVI_REQUIRE(!queries, "queries are only taken together with rotary");
        KIVI_REQUIRE(k_out == nullptr || k_out->data == nullptr, "k_out is only written together with rotary");
    }
    if (batch->max_new == 0) { note_launches(0); return KIVI_OK; }
    Append8Args a{};
    a.L = *layer; a.b = *batch; a.k = *new_k; a.v = *new_v; a.n_rep = n_rep;
    if (turns) { a.rot = *rotary; a.k_out = *k_out; }
    if (queries) { a.q = *q; a.q_out = *q_out; }
    const bool vec = on_grid(a.k, esz) && on_grid(a.v, esz) && on_grid(a.k_out, esz) && on_grid(a.q, esz) && on_grid(a.q_out, esz);
    // a step of one token moves at most the block that it completes
    a.items_vary = batch->max_new > 1;
    const int64_t window_items = a.items_vary ? (layer->residual_cap - 1) / G + 1 : 1;
    const int64_t items = (int64_t)batch->num_seqs * window_items + batch->total_new / G, units = D / 16;
    int64_t turn_blocks = 0;
    a.turn_rows = 1;
    if (queries) {
        const int64_t per_row = (int64_t)H * n_rep * units;
        while (a.turn_rows < kMostTurnRows && (a.turn_rows + 1) * per_row <= kThreads * kTurnUnits && (int64_t)batch->total_new > (int64_t)a.turn_rows * num_sms()) ++a.turn_rows;
        turn_blocks = ((int64_t)batch->total_new + a.turn_rows - 1) / a.turn_rows;
    }
    KIVI_REQUIRE(items * H + turn_blocks <= 0x7fffffff, "too many blocks in one step");
    a.items = (int)items;
    const int run = value8_run(G);
    size_t smem = (size_t)G / run * D * (run + 4);               // (80 KB at the most)
    if (queries && smem < (size_t)a.turn_rows * rotary->dim * 4) smem = (size_t)a.turn_rows * rotary->dim * 4;
    auto* const kernel = layer->res_dtype == KIVI_BF16 ? append_kernel<__nv_bfloat16>(vec, G * units <= kThreads) : append_kernel<float>(vec, G * units <= kThreads);
    constexpr int kMostSmem = 256 / 16 * 256 * 20;               // (the limit is the kernel's, not the call's: two calls at once set the same)
    if (smem > 48 * 1024) KIVI_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem));
    KIVI_CUDA_OK(launch(kernel, dim3((unsigned)(items * H + turn_blocks)), kThreads, smem, (cudaStream_t)stream, true, a));
    note_launches(1);
    return KIVI_OK;
}

extern "C" int kivi_paged8_read(const kivi_paged8_layer* layer, const kivi_paged_batch* batch, const int32_t* starts,
                                float* k_out, float* v_out, void* stream) {
    if (int rc = validate_paged8(layer)) return rc;
    if (int rc = validate_batch8(layer, batch)) return rc;
    KIVI_REQUIRE(starts != nullptr && k_out != nullptr && v_out != nullptr, "starts, k_out or v_out is null");
    if (batch->max_new == 0) { note_launches(0); return KIVI_OK; }
    int64_t pieces = ((((int64_t)batch->max_new + 30) / 16 * 4) * (layer->head_dim / 4) + 255) / 256;        // (sixteens of tokens that the rows touch)
    if (pieces > 4096) pieces = 4096;
    const bool bf16 = layer->res_dtype == KIVI_BF16;
    auto* const kernel = layer->head_dim == 128 ? (bf16 ? paged8_read_kernel<__nv_bfloat16, 128> : paged8_read_kernel<float, 128>)
                       : layer->head_dim == 64 ? (bf16 ? paged8_read_kernel<__nv_bfloat16, 64> : paged8_read_kernel<float, 64>)
                                               : (bf16 ? paged8_read_kernel<__nv_bfloat16, 0> : paged8_read_kernel<float, 0>);
    KIVI_CUDA_OK(launch(kernel, dim3((unsigned)pieces, (unsigned)layer->num_kv_heads, (unsigned)batch->num_seqs), 256, 0, (cudaStream_t)stream, true,
                        *layer, *batch, starts, k_out, v_out));
    note_launches(1);
    return KIVI_OK;
}
