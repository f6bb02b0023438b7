// Paged cache: append with the position rotation on the way, dense read-back.
//
// One launch per append.  A sequence's new tokens are dealt out to CTAs so that nothing
// is ordered between them:
//   * one CTA per KV head and group that starts in the window (one at least) quantizes it.
//     Then it writes to the window those tokens that stay and whose slots its own tokens had,
//     so that a slot is overwritten by the CTA that has read it, and the turned keys of its own
//     new tokens, whose rows may be overwritten by them; what stays and meets no token that
//     leaves is dealt out in turn;
//   * one CTA per whole group of new tokens and KV head quantizes that group.
// Every CTA also turns the keys it has and, in steps of a few tokens, the queries of its KV
// head; in longer steps the queries are a streaming kernel of their own (in the same CTAs
// they took 160 registers: 4 x 2048 tokens 189 us, 100 apart).
//
// Bound by memory: bf16, D = 128, G = 32 moves 2.1 bytes per element of the rows in and
// out and 0.5 per flushed element; the smallest call (one token) is launch and latency.
// A thread takes two 16-byte vectors of a token's key and of its value at a time.
#include "paged_common.cuh"

namespace kivi {
namespace {

__device__ int g_fault = 0;

struct Rotary {
    const float* table;      // [rows][dim]: dim/2 cosines, dim/2 sines; nullptr: rows are taken as they are
    int dim, interleaved;
};

// N neighbouring channels of a row; VEC: they lie on the grid of such vectors.
template <typename T, int N, bool VEC> struct Channels;
template <int N, bool VEC> struct Channels<float, N, VEC> {
    __device__ static void load(const float* p, float (&x)[N]) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < N; i += 4) { const float4 v = *reinterpret_cast<const float4*>(p + i); x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w; }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = p[i];
        }
    }
    __device__ static void store(float* p, const float (&x)[N]) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) p[i] = x[i];
        }
    }
    __device__ static float round(float x) { return x; }
};
template <int N, bool VEC> struct Channels<__nv_bfloat16, N, VEC> {
    __device__ static void widen(uint32_t w, float& a, float& b) { a = __uint_as_float(w << 16); b = __uint_as_float(w & 0xffff0000u); }
    __device__ static uint32_t narrow(float a, float b) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    __device__ static void load(const __nv_bfloat16* p, float (&x)[N]) {
        if constexpr (VEC && N == 8) {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            widen(v.x, x[0], x[1]); widen(v.y, x[2], x[3]); widen(v.z, x[4], x[5]); widen(v.w, x[6], x[7]);
        } else if constexpr (VEC) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            widen(v.x, x[0], x[1]); widen(v.y, x[2], x[3]);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = __bfloat162float(p[i]);
        }
    }
    __device__ static void store(__nv_bfloat16* p, const float (&x)[N]) {
        if constexpr (VEC && N == 8) *reinterpret_cast<uint4*>(p) = make_uint4(narrow(x[0], x[1]), narrow(x[2], x[3]), narrow(x[4], x[5]), narrow(x[6], x[7]));
        else if constexpr (VEC) *reinterpret_cast<uint2*>(p) = make_uint2(narrow(x[0], x[1]), narrow(x[2], x[3]));
        else {
#pragma unroll
            for (int i = 0; i < N; ++i) p[i] = __float2bfloat16_rn(x[i]);
        }
    }
    __device__ static float round(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }
};

struct AppendArgs {
    kivi_paged_layer L;
    kivi_paged_batch b;
    kivi_rows k, v, q, q_out, k_out;
    Rotary rotary;
    int n_rep, items_vary;
};

template <typename T> __device__ __forceinline__ T* row_of(const kivi_rows& r, int64_t row, int head) {
    return reinterpret_cast<T*>(r.data) + row * r.row_stride + (int64_t)head * r.head_stride;
}

constexpr int kThreads = 128;
template <typename T> constexpr int kPad = 16 / sizeof(T);                // rows of a tile start 16 bytes apart in bank space

// Codes of a tile in shared memory, tile[t][D + pad], for the group's place in a page.
template <typename T, bool HALF_EVEN>
__device__ __forceinline__ void quantize_keys_tile(const T* tile, uint8_t* block, int D, int G, float* scales, float* zeros) {
    const int Q = G / 4, W = D < 64 ? D : 64, S = D + kPad<T>;
    for (int d = threadIdx.x; d < D; d += kThreads) {
        float mn = 1e30f, mx = -1e30f;
#pragma unroll 8
        for (int t = 0; t < G; ++t) { const float x = (float)tile[t * S + d]; mn = fminf(mn, x); mx = fmaxf(mx, x); }
        const float scale = group_scale(mn, mx), rcp = group_rcp(scale);
        scales[d] = scale;
        zeros[d] = mn;
#pragma unroll 2
        for (int j = 0; j < Q; ++j) {
            float m[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) m[i] = code_magic<HALF_EVEN>((float)tile[(4 * j + i) * S + d], mn, scale, rcp);
            block[kblock_offset(d, j, Q, W)] = (uint8_t)pack4_magic(m[0], m[1], m[2], m[3]);
        }
    }
}
template <typename T, bool HALF_EVEN>
__device__ __forceinline__ void quantize_values_tile(const T* tile, uint8_t* block, float* factors, int D, int G) {
    const int S = D + kPad<T>, ng = D / G;
    for (int i = threadIdx.x; i < G * ng; i += kThreads) {
        const int t = i % G, gd = i / G;                 // (tokens on neighbouring threads: rows are four banks apart)
        const T* x = tile + t * S + gd * G;
        float mn = 1e30f, mx = -1e30f;
#pragma unroll 4
        for (int c = 0; c < G; c += 4) {
            float v[4];
            Channels<T, 4, true>::load(x + c, v);
            mn = fminf(fminf(mn, v[0]), fminf(v[1], fminf(v[2], v[3])));
            mx = fmaxf(fmaxf(mx, v[0]), fmaxf(v[1], fmaxf(v[2], v[3])));
        }
        const float scale = group_scale(mn, mx), rcp = group_rcp(scale);
        const int at = (int)vmeta_index(t, gd, D, G);
        factors[at] = scale;
        factors[D + at] = mn;
#pragma unroll 2
        for (int c = 0; c < G; c += 4) {
            float v[4];
            Channels<T, 4, true>::load(x + c, v);
            block[vcode_offset(t, (gd * G + c) / 4, D, G)] =
                (uint8_t)pack4_magic(code_magic<HALF_EVEN>(v[0], mn, scale, rcp), code_magic<HALF_EVEN>(v[1], mn, scale, rcp),
                                     code_magic<HALF_EVEN>(v[2], mn, scale, rcp), code_magic<HALF_EVEN>(v[3], mn, scale, rcp));
        }
    }
}

// The turning of a row, in units of two vectors of N channels.
template <typename T, int N, bool VEC>
struct Turn {
    using C = Channels<T, N, VEC>;
    const Rotary rot;
    const int D;
    struct Angles { float c[N], s[N], c2[N / 2], s2[N / 2]; };

    __device__ __forceinline__ bool halves() const { return rot.table != nullptr && !rot.interleaved; }
    __device__ __forceinline__ int pairs() const { return halves() ? rot.dim / 2 / N : 0; }
    __device__ __forceinline__ int units() const { return pairs() + (D - 2 * N * pairs() + 2 * N - 1) / (2 * N); }
    // vectors d and e (-1: none) of unit u
    __device__ __forceinline__ void places(int u, int& d, int& e) const {
        if (u < pairs()) { d = N * u; e = d + rot.dim / 2; }
        else { d = 2 * N * u; e = d + N < D ? d + N : -1; }
    }
    // cosines and sines for the unit's vectors: halves share theirs
    __device__ __forceinline__ void angles(int t, int u, int d, int e, Angles& a) const {
        if (rot.table == nullptr) return;
        const int half = rot.dim / 2;
        const float* row = rot.table + (int64_t)t * rot.dim;
        if (halves()) {
            if (u < pairs()) { Channels<float, N, VEC>::load(row + d, a.c); Channels<float, N, VEC>::load(row + half + d, a.s); }
        } else {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                const int p = d / 2 + i, r = e / 2 + i;
                a.c[i] = p < half ? row[p] : 1.0f; a.s[i] = p < half ? row[half + p] : 0.0f;
                a.c2[i] = e >= 0 && r < half ? row[r] : 1.0f; a.s2[i] = e >= 0 && r < half ? row[half + r] : 0.0f;
            }
        }
    }
    __device__ __forceinline__ static void pair(float c, float s, float& p, float& r) {
        const float t = p;
        p = C::round(__fsub_rn(__fmul_rn(t, c), __fmul_rn(r, s)));
        r = C::round(__fadd_rn(__fmul_rn(r, c), __fmul_rn(t, s)));
    }
    __device__ __forceinline__ void turn(int u, int d, int e, const Angles& a, float (&x)[N], float (&y)[N]) const {
        if (rot.table == nullptr) return;
        if (halves()) {
            if (u < pairs()) {
#pragma unroll
                for (int i = 0; i < N; ++i) pair(a.c[i], a.s[i], x[i], y[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                if (d + 2 * i < rot.dim) pair(a.c[i], a.s[i], x[2 * i], x[2 * i + 1]);
                if (e >= 0 && e + 2 * i < rot.dim) pair(a.c2[i], a.s2[i], y[2 * i], y[2 * i + 1]);
            }
        }
    }
};

// N: channels of a vector (16 bytes, or 4 channels for shapes that those do not divide); a
// thread has two of them of a row, which hold each other's partners where halves are
// paired.  QUERIES: a step shorter than a group, whose queries are turned here.
// DT, GT: head_dim and group size where they are constants, the shape the decode kernels take too (0: as the
// layer says): 4 x 2048 tokens 100 -> 92 us with turn and read-back, 2 x 5003 in fp32 213 -> 195, 64 single
// tokens 15.0 -> 13.2.  (Registers for six or eight CTAs an SM: 89 us, 195, 13.8 and 14.8.)
template <typename T, int N, bool VEC, bool HALF_EVEN, bool QUERIES, int DT = 0, int GT = 0>
__global__ void __launch_bounds__(kThreads)
paged_append_kernel(AppendArgs A) {
    using C = Channels<T, N, VEC>;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int place_s[2];
    stream_order();
    settle_paged(A.L, A.b);
    A.k.data = settled(A.k.data); A.v.data = settled(A.v.data); A.q.data = settled(A.q.data);
    A.rotary.table = settled(A.rotary.table);
    const kivi_paged_layer& L = A.L;
    const int D = DT ? DT : L.head_dim, G = GT ? GT : L.group_size, R = L.residual_cap, H = L.num_kv_heads, S = D + kPad<T>;
    T* const k_tile = reinterpret_cast<T*>(smem);                         // [G][D + pad]
    T* const v_tile = k_tile + G * S;
    float* const factors = reinterpret_cast<float*>(v_tile + G * S);      // [2][D]
    uint8_t* const k_block = reinterpret_cast<uint8_t*>(factors + 2 * D); // [D * G / 4]
    uint8_t* const v_block = k_block + D * G / 4;
    const int h = blockIdx.y;

    // sequence s has an item for each group that starts in the window (one at least) and one for
    // each whole group of new tokens
    auto fresh_groups = [&](const PagedSeq& q) {
        const int first = (q.held + G - 1) / G * G, out = quant_of(q.held + q.n, G, R);
        return out > first ? (out - first) / G : 0;
    };
    auto window_groups = [&](const PagedSeq& q) {
        const int first = (q.held + G - 1) / G * G, in = quant_of(q.held, G, R), out = quant_of(q.held + q.n, G, R);
        return max(1, (min(out, first) - in) / G);
    };
    int s = blockIdx.x, sub = 0;
    if (A.items_vary) {
        if (threadIdx.x < 32) {
            const ItemPlace p = find_item(blockIdx.x, A.b.num_seqs, [&](int i) {
                PagedSeq q;
                load_seq(L, A.b, i, q);
                return window_groups(q) + fresh_groups(q);
            });
            if (threadIdx.x == 0) { place_s[0] = p.s; place_s[1] = p.sub; }
        }
        __syncthreads();
        s = place_s[0]; sub = place_s[1];
    }
    if (s >= A.b.num_seqs) return;
    PagedSeq q;
    if (!load_seq(L, A.b, s, q)) { if (threadIdx.x == 0) atomicOr(&g_fault, kPagedFault); return; }
    if (q.n == 0) return;

    const Turn<T, N, VEC> by{A.rotary, D};
    const int units = by.units();
    auto load2 = [&](const T* row, int d, int e, float (&x)[N], float (&y)[N]) {
        C::load(row + d, x);
        if (e >= 0) C::load(row + e, y);
        else {
#pragma unroll
            for (int i = 0; i < N; ++i) y[i] = 0.0f;
        }
    };
    auto store2 = [&](T* row, int d, int e, const float (&x)[N], const float (&y)[N]) {
        C::store(row + d, x);
        if (e >= 0) C::store(row + e, y);
    };
    auto tile2 = [&](T* row, int d, int e, const float (&x)[N], const float (&y)[N]) {
        Channels<T, N, true>::store(row + d, x);
        if (e >= 0) Channels<T, N, true>::store(row + e, y);
    };
    const int64_t ring0 = ((int64_t)q.slot * H + h) * R;
    T* const k_ring = reinterpret_cast<T*>(L.k_res) + ring0 * D;
    T* const v_ring = reinterpret_cast<T*>(L.v_res) + ring0 * D;

    // One unit of a new token: its turned key to a tile, the window and k_out, its value likewise.
    auto fresh_unit = [&](int t, int u, T* kt, T* vt, bool to_ring, bool out) {
        const int64_t row = (int64_t)q.row0 + (t - q.held);
        int d, e;
        by.places(u, d, e);
        typename Turn<T, N, VEC>::Angles a;
        float x[N], y[N], vx[N], vy[N];
        by.angles(t, u, d, e, a);
        load2(row_of<const T>(A.k, row, h), d, e, x, y);
        if (vt || to_ring) load2(row_of<const T>(A.v, row, h), d, e, vx, vy);
        by.turn(u, d, e, a, x, y);
        if (out && A.k_out.data) store2(row_of<T>(A.k_out, row, h), d, e, x, y);
        if (kt) { tile2(kt, d, e, x, y); tile2(vt, d, e, vx, vy); }
        if (to_ring) {
            const int64_t at = (int64_t)ring_slot(t, A.b.ring_shift, R) * D;
            Channels<T, N, VEC>::store(k_ring + at + d, x); Channels<T, N, VEC>::store(v_ring + at + d, vx);
            if (e >= 0) { Channels<T, N, VEC>::store(k_ring + at + e, y); Channels<T, N, VEC>::store(v_ring + at + e, vy); }
        }
    };
    // the group in the tiles to its page
    auto flush_tiles = [&](int t0) {
        const int page = q.pages[t0 / L.page_tokens];
        const bool ok = (unsigned)page < (unsigned)L.num_pages;
        if (!ok && threadIdx.x == 0) atomicOr(&g_fault, kPagedFault);
        const int64_t g = ((int64_t)(ok ? page : 0) * H + h) * (L.page_tokens / G) + t0 % L.page_tokens / G;
        __syncthreads();
        if (!ok) return;
        quantize_keys_tile<T, HALF_EVEN>(k_tile, k_block, D, G, L.k_scales + g * D, L.k_zeros + g * D);
        quantize_values_tile<T, HALF_EVEN>(v_tile, v_block, factors, D, G);
        __syncthreads();
        const int words = D * G / 16;
        for (int i = threadIdx.x; i < words; i += kThreads) {
            reinterpret_cast<uint32_t*>(L.k_codes + g * (D * G / 4))[i] = reinterpret_cast<const uint32_t*>(k_block)[i];
            reinterpret_cast<uint32_t*>(L.v_codes + g * (D * G / 4))[i] = reinterpret_cast<const uint32_t*>(v_block)[i];
        }
        for (int i = threadIdx.x; i < D; i += kThreads) { L.v_scales[g * D + i] = factors[i]; L.v_zeros[g * D + i] = factors[D + i]; }
    };

    const int end = q.held + q.n, out = quant_of(end, G, R);
    const int first = (q.held + G - 1) / G * G, n_fresh = fresh_groups(q);
    const int in = quant_of(q.held, G, R), n_window = window_groups(q);
    if (sub >= n_window) {
        const int t0 = first + (sub - n_window) * G;
#pragma unroll 1
        for (int i = threadIdx.x; i < G * units; i += kThreads) {
            const int j = i / units;
            fresh_unit(t0 + j, i % units, k_tile + j * S, v_tile + j * S, false, true);
        }
        flush_tiles(t0);
        return;
    }
    const int t0 = in + sub * G;
    if (t0 < min(out, first)) {
        for (int i = threadIdx.x; i < G * units; i += kThreads) {
            const int j = i / units, t = t0 + j, u = i % units;
            if (t < q.held) {
                int d, e;
                float x[N], y[N], vx[N], vy[N];
                by.places(u, d, e);
                const int64_t at = (int64_t)ring_slot(t, A.b.ring_shift, R) * D;
                load2(k_ring + at, d, e, x, y);
                load2(v_ring + at, d, e, vx, vy);
                tile2(k_tile + j * S, d, e, x, y);
                tile2(v_tile + j * S, d, e, vx, vy);
            } else {
                fresh_unit(t, u, k_tile + j * S, v_tile + j * S, false, false);
            }
        }
        flush_tiles(t0);
        __syncthreads();
    }
    // what no other CTA has: the tokens before the first whole new group and those behind the last
    const int lo = n_fresh ? first : end, hi = n_fresh ? first + n_fresh * G : end;
    const int rest = (lo - q.held) + (end - hi), leaving = min(out, q.held);
    const int slots = QUERIES ? 1 + A.n_rep : 1;         // key and value, then the query heads: a thread's work each
    for (int i = threadIdx.x; i < rest * units * slots; i += kThreads) {
        const int u = i % units, slot = i / units % slots, j = i / units / slots, t = j < lo - q.held ? q.held + j : hi + (j - (lo - q.held));
        // A token that stays: the token of the window that had the slot, if it leaves, says whose it is.  One that
        // leaves with a group of the window is that group's CTA's, which has read its row (k_out may be new_k).
        const int had = in + (t - in) % R;
        const int whose = t < min(out, first) ? (t - in) / G : t >= out && had < leaving ? (had - in) / G : t % n_window;
        if (whose != sub) continue;
        if (!QUERIES || slot == 0) {
            fresh_unit(t, u, nullptr, nullptr, t >= out, true);
        } else {
            const int64_t row = (int64_t)q.row0 + (t - q.held);
            const int head = h * A.n_rep + slot - 1;
            int d, e;
            float x[N], y[N];
            typename Turn<T, N, VEC>::Angles a;
            by.places(u, d, e);
            load2(row_of<const T>(A.q, row, head), d, e, x, y);
            by.angles(t, u, d, e, a);
            by.turn(u, d, e, a, x, y);
            store2(row_of<T>(A.q_out, row, head), d, e, x, y);
        }
    }
}

// Queries of a long step, two vectors a thread and pass; the rows of a block find their
// sequences first.  Bound by memory.
constexpr int kTurnRows = 8;
template <typename T, int N, bool VEC>
__global__ void __launch_bounds__(256)
paged_turn_kernel(AppendArgs A) {
    using C = Channels<T, N, VEC>;
    __shared__ int token_s[kTurnRows];
    stream_order();
    settle_paged(A.L, A.b);
    A.q.data = settled(A.q.data);
    A.rotary.table = settled(A.rotary.table);
    const Turn<T, N, VEC> by{A.rotary, A.L.head_dim};
    const int row0 = blockIdx.x * kTurnRows, units = by.units(), heads = A.L.num_kv_heads * A.n_rep;
    if (threadIdx.x < kTurnRows) {
        const int row = row0 + threadIdx.x;
        // the last sequence that starts at or before the row (none of a sequence that is left out)
        int lo = 0, hi = A.b.num_seqs;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (A.b.cu_new[mid] <= row) lo = mid;
            else hi = mid;
        }
        PagedSeq q;
        const bool ok = load_seq(A.L, A.b, lo, q) && row >= q.row0 && row - q.row0 < q.n;
        token_s[threadIdx.x] = ok ? q.held + (row - q.row0) : -1;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kTurnRows * heads * units; i += 256) {
        const int u = i % units, head = i / units % heads, r = i / units / heads, t = token_s[r];
        if (t < 0) continue;
        int d, e;
        float x[N], y[N];
        typename Turn<T, N, VEC>::Angles a;
        by.places(u, d, e);
        const T* from = row_of<const T>(A.q, row0 + r, head);
        C::load(from + d, x);
        if (e >= 0) C::load(from + e, y);
        by.angles(t, u, d, e, a);
        by.turn(u, d, e, a, x, y);
        T* to = row_of<T>(A.q_out, row0 + r, head);
        C::store(to + d, x);
        if (e >= 0) C::store(to + e, y);
    }
}

// Four channels of keys and values of four tokens per thread, which a word of key codes
// holds; neighbouring threads take neighbouring channels, so a row leaves in whole lines.
// Bound by its writes.  grid = (pieces of rows, KV heads, sequences).  DT, GT: head_dim and group size,
// 0: as the layer says.
template <typename T, int DT, int GT>
__global__ void __launch_bounds__(256)
paged_read_kernel(kivi_paged_layer L, kivi_paged_batch b, const int32_t* starts, float* __restrict__ k_out, float* __restrict__ v_out) {
    stream_order();
    settle_paged(L, b);
    starts = settled(starts);
    const int s = blockIdx.z, h = blockIdx.y, D = DT ? DT : L.head_dim, G = GT ? GT : L.group_size, R = L.residual_cap, H = L.num_kv_heads, quads = D / 4;
    const int r0 = b.cu_new[s], r1 = b.cu_new[s + 1], held = b.seq_lens[s], start = starts[s], slot = b.slots[s];
    const int n = r1 - r0;
    if (r0 < 0 || n < 0 || r1 > b.total_new || n > b.max_new || held < 0 || held > b.max_len || start < 0 || start > held - n || slot < 0 || slot >= L.num_slots) {
        if (threadIdx.x == 0) atomicOr(&g_fault, kPagedFault);
        return;
    }
    if (n == 0) return;
    PagedSeq q{held, n, r0, slot, b.page_table + (int64_t)s * b.table_width};
    const int out = quant_of(held, G, R), Q = G / 4, W = D < 64 ? D : 64, gpp = L.page_tokens / G;
    const int first = start / 4, blocks = (start + n + 3) / 4 - first;            // quads of tokens
    for (int64_t i = blockIdx.x * 256 + threadIdx.x; i < (int64_t)blocks * quads; i += (int64_t)gridDim.x * 256) {
        const int t0 = 4 * (first + (int)(i / quads)), d = 4 * (int)(i % quads);
        float4 k[4], v[4];
        if (t0 < out) {                                  // (groups are whole quads)
            const int64_t g = ((int64_t)page_of(L, q, t0, &g_fault) * H + h) * gpp + t0 % L.page_tokens / G;
            const int tt = t0 % G;
            const uint32_t w = *reinterpret_cast<const uint32_t*>(L.k_codes + g * (D * Q) + kblock_offset(d, tt >> 2, Q, W));
            const float4 ks = *reinterpret_cast<const float4*>(L.k_scales + g * D + d), kz = *reinterpret_cast<const float4*>(L.k_zeros + g * D + d);
            uint32_t c[4];
            float vs[4], vz[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                c[e] = L.v_codes[g * (D * Q) + vcode_offset(tt + e, d / 4, D, G)];
                const int64_t at = g * D + vmeta_index(tt + e, d / G, D, G);
                vs[e] = L.v_scales[at]; vz[e] = L.v_zeros[at];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t x = w >> (2 * e);
                k[e] = make_float4(dequant((float)(x & 3u), ks.x, kz.x), dequant((float)((x >> 8) & 3u), ks.y, kz.y),
                                   dequant((float)((x >> 16) & 3u), ks.z, kz.z), dequant((float)((x >> 24) & 3u), ks.w, kz.w));
                v[e] = make_float4(dequant((float)(c[e] & 3u), vs[e], vz[e]), dequant((float)((c[e] >> 2) & 3u), vs[e], vz[e]),
                                   dequant((float)((c[e] >> 4) & 3u), vs[e], vz[e]), dequant((float)(c[e] >> 6), vs[e], vz[e]));
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t at = (((int64_t)slot * H + h) * R + ring_slot(min(t0 + e, held - 1), b.ring_shift, R)) * D + d;
                float x[4];
                Channels<T, 4, true>::load(reinterpret_cast<const T*>(L.k_res) + at, x);
                k[e] = make_float4(x[0], x[1], x[2], x[3]);
                Channels<T, 4, true>::load(reinterpret_cast<const T*>(L.v_res) + at, x);
                v[e] = make_float4(x[0], x[1], x[2], x[3]);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int t = t0 + e;
            if (t < start || t >= start + n) continue;
            const int64_t to = (((int64_t)r0 + (t - start)) * H + h) * D + d;
            store_quad(k_out, KIVI_F32, to, k[e]);
            store_quad(v_out, KIVI_F32, to, v[e]);
        }
    }
}

}  // namespace

int validate_paged(const kivi_paged_layer* L) {
    KIVI_REQUIRE(L != nullptr, "layer is null");
    KIVI_REQUIRE(L->num_pages > 0 && L->num_kv_heads > 0 && L->num_slots > 0, "num_pages, num_kv_heads and num_slots must be positive");
    KIVI_REQUIRE(L->group_size >= 4 && L->group_size % 4 == 0, "group_size (%d) must be >= 4 and divisible by 4", L->group_size);
    KIVI_REQUIRE(L->head_dim > 0 && L->head_dim % L->group_size == 0, "head_dim (%d) must be divisible by group_size (%d)", L->head_dim, L->group_size);
    KIVI_REQUIRE(L->head_dim <= 256 && (L->head_dim <= 64 || L->head_dim % 64 == 0), "head_dim (%d) must be <= 64 or a multiple of 64 up to 256", L->head_dim);
    KIVI_REQUIRE(L->page_tokens > 0 && L->page_tokens % L->group_size == 0, "page_tokens (%d) must be a multiple of group_size (%d)", L->page_tokens, L->group_size);
    KIVI_REQUIRE(L->residual_cap >= L->group_size, "residual_cap (%d) must be at least group_size (%d)", L->residual_cap, L->group_size);
    KIVI_REQUIRE(L->num_kv_heads <= 65535, "num_kv_heads (%d) must be at most 65535", L->num_kv_heads);
    KIVI_REQUIRE(L->res_dtype == KIVI_F32 || L->res_dtype == KIVI_BF16, "res_dtype must be KIVI_F32 or KIVI_BF16");
    KIVI_REQUIRE(L->k_codes && L->k_scales && L->k_zeros && L->v_codes && L->v_scales && L->v_zeros && L->k_res && L->v_res, "a pointer of the layer is null");
    auto off = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; };
    KIVI_REQUIRE(!off(L->k_codes) && !off(L->k_scales) && !off(L->k_zeros) && !off(L->v_codes) && !off(L->v_scales) && !off(L->v_zeros) && !off(L->k_res) && !off(L->v_res),
                 "the arrays of a paged layer must start on 16-byte boundaries");
    return KIVI_OK;
}

int validate_batch(const kivi_paged_layer* L, const kivi_paged_batch* b) {
    KIVI_REQUIRE(b != nullptr, "batch is null");
    KIVI_REQUIRE(b->num_seqs > 0 && b->num_seqs <= 65535, "num_seqs (%d) outside 1..65535", b->num_seqs);
    KIVI_REQUIRE(b->table_width > 0, "table_width must be positive");
    KIVI_REQUIRE(b->page_table && b->slots && b->seq_lens && b->cu_new, "an array of the batch is null");
    KIVI_REQUIRE(b->total_new >= 0 && b->max_new >= 0 && b->max_new <= b->total_new, "max_new (%d) must be between 0 and total_new (%d)", b->max_new, b->total_new);
    // (2^30: sums of two positions, and positions rounded up to a tile, stay in 32 bits)
    KIVI_REQUIRE(b->max_len >= b->max_new && b->max_len <= (1 << 30), "max_len (%d) must be between max_new (%d) and 2^30", b->max_len, b->max_new);
    KIVI_REQUIRE(b->total_new <= (1 << 30), "total_new (%d) must be at most 2^30", b->total_new);
    KIVI_REQUIRE(b->ring_shift >= 0 && b->ring_shift < L->residual_cap, "ring_shift (%d) outside 0..%d", b->ring_shift, L->residual_cap - 1);
    KIVI_REQUIRE(quant_of(b->max_len, L->group_size, L->residual_cap) <= (int64_t)b->table_width * L->page_tokens,
                 "a sequence of max_len (%d) tokens does not fit the page table (%d pages of %d tokens)", b->max_len, b->table_width, L->page_tokens);
    return KIVI_OK;
}

int validate_in_place(const kivi_rows* to, const char* to_name, const kivi_rows* from, const char* from_name, int rows, int heads, bool same_type) {
    KIVI_REQUIRE(to->data != from->data || (same_type && (rows <= 1 || to->row_stride == from->row_stride) && (heads <= 1 || to->head_stride == from->head_stride)),
                 "%s starts where %s does but is laid out differently", to_name, from_name);
    return KIVI_OK;
}

int paged_cache_fault_word(int* out) {
    KIVI_CUDA_OK(cudaMemcpyFromSymbol(out, g_fault, sizeof(int)));
    return KIVI_OK;
}
int paged_cache_fault_clear() {
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
// vectors of n channels lie on their own grid
bool on_grid(const kivi_rows& r, int esz, int n) {
    return (reinterpret_cast<uintptr_t>(r.data) % (n * esz)) == 0 && r.row_stride % n == 0 && r.head_stride % n == 0;
}
using AppendKernel = void (*)(AppendArgs);
template <typename T>
AppendKernel turn_kernel(bool wide, bool vec) {
    constexpr int N = 16 / sizeof(T);
    return wide ? paged_turn_kernel<T, N, true> : vec ? paged_turn_kernel<T, 4, true> : paged_turn_kernel<T, 4, false>;
}
template <typename T, bool QUERIES>
AppendKernel append_kernel(bool wide, bool vec, bool even, bool fixed) {
    constexpr int N = 16 / sizeof(T);
    if (wide && fixed) return even ? paged_append_kernel<T, N, true, true, QUERIES, 128, 32> : paged_append_kernel<T, N, true, false, QUERIES, 128, 32>;
    if (wide) return even ? paged_append_kernel<T, N, true, true, QUERIES> : paged_append_kernel<T, N, true, false, QUERIES>;
    if (vec) return even ? paged_append_kernel<T, 4, true, true, QUERIES> : paged_append_kernel<T, 4, true, false, QUERIES>;
    return even ? paged_append_kernel<T, 4, false, true, QUERIES> : paged_append_kernel<T, 4, false, false, QUERIES>;
}

}  // namespace
}  // namespace kivi

using namespace kivi;

extern "C" int kivi_paged_append(const kivi_paged_layer* layer, const kivi_paged_batch* batch,
                                 const kivi_rows* new_k, const kivi_rows* new_v, const float* rotary, int rotary_rows,
                                 int rotary_dim, int interleaved, const kivi_rows* q, int n_rep, const kivi_rows* q_out,
                                 const kivi_rows* k_out, int rounding, void* stream) {
    if (int rc = validate_paged(layer)) return rc;
    if (int rc = validate_batch(layer, batch)) return rc;
    const int D = layer->head_dim, G = layer->group_size, esz = elem_size(layer->res_dtype);
    if (int rc = check_rows(new_k, "new_k")) return rc;
    if (int rc = check_rows(new_v, "new_v")) return rc;
    KIVI_REQUIRE(rounding == KIVI_ROUND_HALF_AWAY || rounding == KIVI_ROUND_HALF_EVEN, "rounding must be KIVI_ROUND_HALF_AWAY or KIVI_ROUND_HALF_EVEN");
    const bool queries = q != nullptr && q->data != nullptr;
    if (rotary != nullptr) {
        KIVI_REQUIRE(rotary_dim > 0 && rotary_dim <= D && rotary_dim % 2 == 0, "rotary_dim (%d) must be even and at most head_dim (%d)", rotary_dim, D);
        KIVI_REQUIRE(interleaved || rotary_dim % 8 == 0, "rotary_dim (%d) must be a multiple of 8 where channels half of it apart are paired", rotary_dim);
        KIVI_REQUIRE(rotary_rows >= batch->max_len, "rotary holds %d positions, max_len is %d", rotary_rows, batch->max_len);
        if (int rc = check_rows(k_out, "k_out")) return rc;
        if (int rc = validate_in_place(k_out, "k_out", new_k, "new_k", batch->total_new, layer->num_kv_heads, true)) return rc;
        if (queries) {
            KIVI_REQUIRE(n_rep >= 1, "n_rep (%d) must be positive", n_rep);
            if (int rc = check_rows(q_out, "q_out")) return rc;
            if (int rc = validate_in_place(q_out, "q_out", q, "q", batch->total_new, layer->num_kv_heads * n_rep, true)) return rc;
        }
    } else {
        KIVI_REQUIRE(!queries, "queries are only taken together with rotary");
        KIVI_REQUIRE(k_out == nullptr || k_out->data == nullptr, "k_out is only written together with rotary");
    }
    const size_t smem = 2 * (size_t)G * (D * esz + 16) + 2 * D * 4 + (size_t)D * G / 2;
    constexpr size_t kMostSmem = 220 * 1024;
    if (smem > kMostSmem) {
        set_error("a group of %d tokens of head_dim %d does not fit shared memory", G, D);
        return KIVI_ERR_UNSUPPORTED;
    }
    if (batch->max_new == 0) { note_launches(0); return KIVI_OK; }
    AppendArgs a{};
    a.L = *layer; a.b = *batch; a.k = *new_k; a.v = *new_v; a.n_rep = n_rep;
    a.rotary = {rotary, rotary ? rotary_dim : 0, interleaved ? 1 : 0};
    if (rotary) a.k_out = *k_out;
    if (queries) { a.q = *q; a.q_out = *q_out; }
    auto grid = [&](int n) {
        const bool table = rotary == nullptr || ((reinterpret_cast<uintptr_t>(rotary) & 15u) == 0 && rotary_dim % 4 == 0 && (interleaved || rotary_dim % (2 * n) == 0));
        return D % n == 0 && table && on_grid(a.k, esz, n) && on_grid(a.v, esz, n) && on_grid(a.k_out, esz, n) && on_grid(a.q, esz, n) && on_grid(a.q_out, esz, n);
    };
    const bool bf16 = layer->res_dtype == KIVI_BF16, wide = bf16 ? grid(8) : grid(4), vec = grid(4);
    cudaStream_t st = (cudaStream_t)stream;
    int launches = 1;
    // queries of more than a group of tokens: by themselves
    if (queries && batch->max_new >= G) {
        auto* const turn = bf16 ? turn_kernel<__nv_bfloat16>(wide, vec) : turn_kernel<float>(wide, vec);
        KIVI_CUDA_OK(launch(turn, dim3((unsigned)((batch->total_new + kTurnRows - 1) / kTurnRows)), 256, 0, st, true, a));
        a.q = a.q_out = kivi_rows{};
        ++launches;
    }
    // a step of one token moves at most the group that it completes
    a.items_vary = batch->max_new > 1;
    const int64_t window_items = a.items_vary ? (layer->residual_cap - 1) / G + 1 : 1;
    const int64_t items = (int64_t)batch->num_seqs * window_items + batch->total_new / G;
    KIVI_REQUIRE(items <= 0x7fffffff, "too many groups in one step");
    const bool even = rounding == KIVI_ROUND_HALF_EVEN, fixed = D == 128 && G == 32;
    auto* const kernel = bf16 ? (a.q.data ? append_kernel<__nv_bfloat16, true>(wide, vec, even, fixed) : append_kernel<__nv_bfloat16, false>(wide, vec, even, fixed))
                              : (a.q.data ? append_kernel<float, true>(wide, vec, even, fixed) : append_kernel<float, false>(wide, vec, even, fixed));
    // (the limit is the kernel's, not the call's: two calls at once set the same)
    if (smem > 48 * 1024) KIVI_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostSmem));
    KIVI_CUDA_OK(launch(kernel, dim3((unsigned)items, (unsigned)layer->num_kv_heads), kThreads, smem, st, true, a));
    note_launches(launches);
    return KIVI_OK;
}

extern "C" int kivi_paged_read(const kivi_paged_layer* layer, const kivi_paged_batch* batch, const int32_t* starts,
                               float* k_out, float* v_out, void* stream) {
    if (int rc = validate_paged(layer)) return rc;
    if (int rc = validate_batch(layer, batch)) return rc;
    KIVI_REQUIRE(starts != nullptr && k_out != nullptr && v_out != nullptr, "starts, k_out or v_out is null");
    if (batch->max_new == 0) { note_launches(0); return KIVI_OK; }
    int64_t pieces = (((int64_t)batch->max_new + 6) / 4 * (layer->head_dim / 4) + 255) / 256;        // (quads of tokens that the rows touch)
    if (pieces > 4096) pieces = 4096;
    const bool fixed = layer->head_dim == 128 && layer->group_size == 32, bf16 = layer->res_dtype == KIVI_BF16;
    auto* const kernel = fixed ? (bf16 ? paged_read_kernel<__nv_bfloat16, 128, 32> : paged_read_kernel<float, 128, 32>)
                               : (bf16 ? paged_read_kernel<__nv_bfloat16, 0, 0> : paged_read_kernel<float, 0, 0>);
    KIVI_CUDA_OK(launch(kernel, dim3((unsigned)pieces, (unsigned)layer->num_kv_heads, (unsigned)batch->num_seqs), 256, 0, (cudaStream_t)stream, true,
                        *layer, *batch, starts, k_out, v_out));
    note_launches(1);
    return KIVI_OK;
}
