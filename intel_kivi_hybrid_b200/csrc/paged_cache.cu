// Paged cache: append with the position rotation on the way, dense read-back.
//
// One launch per append.  A sequence's new tokens are dealt out to CTAs so that nothing
// is ordered between them:
//   * one CTA per (sequence, KV head) takes the groups that start in the window, then
//     writes what stays to the window -- a slot it overwrites is one of a token it has
//     moved out before, so the order holds inside the CTA;
//   * one CTA per whole group of new tokens and KV head quantizes that group.
// Every CTA also turns the rows it has (keys, and the queries of its KV head), so the
// step's tensors are read once.
//
// Bound by memory: bf16, D = 128, G = 32 moves 2.1 bytes per element of the rows in and
// out and 0.5 per flushed element; the smallest call (one token) is launch and latency.
#include "paged_common.cuh"

namespace kivi {
namespace {

__device__ int g_fault = 0;

struct Rotary {
    const float* table;      // [rows][dim]: dim/2 cosines, dim/2 sines; nullptr: rows are taken as they are
    int dim, interleaved;
};

template <typename T> struct Quad;
template <> struct Quad<float> {
    __device__ static void load(const float* p, float (&x)[4], bool vec) {
        if (vec) { const float4 v = *reinterpret_cast<const float4*>(p); x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w; }
        else { x[0] = p[0]; x[1] = p[1]; x[2] = p[2]; x[3] = p[3]; }
    }
    __device__ static void store(float* p, const float (&x)[4], bool vec) {
        if (vec) *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
        else { p[0] = x[0]; p[1] = x[1]; p[2] = x[2]; p[3] = x[3]; }
    }
    __device__ static float round(float x) { return x; }
};
template <> struct Quad<__nv_bfloat16> {
    __device__ static void load(const __nv_bfloat16* p, float (&x)[4], bool vec) {
        if (vec) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            x[0] = __uint_as_float(v.x << 16); x[1] = __uint_as_float(v.x & 0xffff0000u);
            x[2] = __uint_as_float(v.y << 16); x[3] = __uint_as_float(v.y & 0xffff0000u);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = __bfloat162float(p[i]);
        }
    }
    __device__ static void store(__nv_bfloat16* p, const float (&x)[4], bool vec) {
        if (vec) {
            const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
            *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = __float2bfloat16_rn(x[i]);
        }
    }
    __device__ static float round(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }
};

// Rows of one head that a CTA turns: `from` and `to` may be the same memory, so a row is
// turned by one thread per pair of quads that exchange values.
// A unit of work is 8 channels: quads d and e that hold each other's partners (halves), or
// two quads of whole pairs (interleaved, or behind the rotated channels).
template <typename T>
struct Turn {
    const Rotary r;
    const int D;
    const bool vec;                                      // rows lie on the grid of a quad
    // unit u of D/8 (the last may hold one quad only where D % 8 == 4)
    __device__ __forceinline__ bool halves() const { return r.table != nullptr && !r.interleaved && r.dim % 8 == 0; }
    __device__ __forceinline__ int units() const { return (D + 7) / 8; }
    __device__ __forceinline__ void places(int u, int& d, int& e) const {
        const int pairs = halves() ? r.dim / 8 : 0;
        if (u < pairs) { d = 4 * u; e = 4 * u + r.dim / 2; }
        else { d = 8 * u; e = 8 * u + 4 < D ? 8 * u + 4 : -1; }
    }
    // the unit's values turned to the angles of `angle` (a row of the table) and rounded to T
    __device__ __forceinline__ void load(const T* row, const float* angle, int d, int e, float (&x)[4], float (&y)[4]) const {
        Quad<T>::load(row + d, x, vec);
        if (e >= 0) Quad<T>::load(row + e, y, vec);
        else { y[0] = y[1] = y[2] = y[3] = 0.0f; }
        if (r.table == nullptr) return;
        const int h = r.dim / 2;
        if (halves()) {
            if (d < h) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float c = angle[d + i], s = angle[h + d + i], a = x[i], b = y[i];
                    x[i] = Quad<T>::round(__fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s)));
                    y[i] = Quad<T>::round(__fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s)));
                }
            }
            return;
        }
        // interleaved (halves of other sizes are refused by the host)
        turn_pairs(angle, d, x);
        if (e >= 0) turn_pairs(angle, e, y);
    }
    __device__ __forceinline__ void turn_pairs(const float* angle, int d, float (&x)[4]) const {
        const int h = r.dim / 2;
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            if (d + i >= r.dim) break;
            const float c = angle[(d + i) / 2], s = angle[h + (d + i) / 2], a = x[i], b = x[i + 1];
            x[i] = Quad<T>::round(__fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s)));
            x[i + 1] = Quad<T>::round(__fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s)));
        }
    }
};

struct AppendArgs {
    kivi_paged_layer L;
    kivi_paged_batch b;
    kivi_rows k, v, q, q_out, k_out;
    Rotary rotary;
    int n_rep, vec;
};

template <typename T> __device__ __forceinline__ const T* row_of(const kivi_rows& r, int64_t row, int head) {
    return reinterpret_cast<const T*>(r.data) + row * r.row_stride + (int64_t)head * r.head_stride;
}

constexpr int kThreads = 128;

// Codes of the tile in shared memory, tile[t][D + 4], to the group's place in a page.
template <bool HALF_EVEN>
__device__ __forceinline__ void quantize_keys_tile(const float* tile, uint8_t* block, int D, int G, uint8_t* codes, float* scales, float* zeros) {
    const int Q = G / 4, W = D < 64 ? D : 64, S = D + 4;
    for (int d = threadIdx.x; d < D; d += kThreads) {
        float mn = 1e30f, mx = -1e30f;
        for (int t = 0; t < G; ++t) { const float x = tile[t * S + d]; mn = fminf(mn, x); mx = fmaxf(mx, x); }
        const float scale = group_scale(mn, mx), rcp = group_rcp(scale);
        scales[d] = scale;
        zeros[d] = mn;
        for (int j = 0; j < Q; ++j) {
            float m[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) m[i] = code_magic<HALF_EVEN>(tile[(4 * j + i) * S + d], mn, scale, rcp);
            block[kblock_offset(d, j, Q, W)] = (uint8_t)pack4_magic(m[0], m[1], m[2], m[3]);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < D * Q / 4; i += kThreads) reinterpret_cast<uint32_t*>(codes)[i] = reinterpret_cast<const uint32_t*>(block)[i];
}
template <bool HALF_EVEN>
__device__ __forceinline__ void quantize_values_tile(const float* tile, uint8_t* block, float* factors, int D, int G, uint8_t* codes, float* scales, float* zeros) {
    const int S = D + 4, ng = D / G;
    for (int i = threadIdx.x; i < G * ng; i += kThreads) {
        const int t = i % G, gd = i / G;                 // (tokens on neighbouring threads: rows are four banks apart)
        const float* x = tile + t * S + gd * G;
        float mn = 1e30f, mx = -1e30f;
        for (int c = 0; c < G; c += 4) {
            const float4 v = *reinterpret_cast<const float4*>(x + c);
            mn = fminf(fminf(mn, v.x), fminf(v.y, fminf(v.z, v.w)));
            mx = fmaxf(fmaxf(mx, v.x), fmaxf(v.y, fmaxf(v.z, v.w)));
        }
        const float scale = group_scale(mn, mx), rcp = group_rcp(scale);
        const int at = (int)vmeta_index(t, gd, D, G);
        factors[at] = scale;
        factors[D + at] = mn;
        for (int c = 0; c < G; c += 4) {
            const float4 v = *reinterpret_cast<const float4*>(x + c);
            block[vcode_offset(t, (gd * G + c) / 4, D, G)] =
                (uint8_t)pack4_magic(code_magic<HALF_EVEN>(v.x, mn, scale, rcp), code_magic<HALF_EVEN>(v.y, mn, scale, rcp),
                                     code_magic<HALF_EVEN>(v.z, mn, scale, rcp), code_magic<HALF_EVEN>(v.w, mn, scale, rcp));
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < D * G / 16; i += kThreads) reinterpret_cast<uint32_t*>(codes)[i] = reinterpret_cast<const uint32_t*>(block)[i];
    for (int i = threadIdx.x; i < D; i += kThreads) { scales[i] = factors[i]; zeros[i] = factors[D + i]; }
}

template <typename T, bool HALF_EVEN>
__global__ void __launch_bounds__(kThreads)
paged_append_kernel(AppendArgs A) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int place_s[2];
    stream_order();
    settle_paged(A.L, A.b);
    A.k.data = settled(A.k.data); A.v.data = settled(A.v.data); A.q.data = settled(A.q.data);
    A.rotary.table = settled(A.rotary.table);
    const kivi_paged_layer& L = A.L;
    const int D = L.head_dim, G = L.group_size, R = L.residual_cap, H = L.num_kv_heads, S = D + 4;
    float* const tile = reinterpret_cast<float*>(smem);                   // [G][D + 4]
    float* const factors = tile + G * S;                                  // [2][D]
    uint8_t* const block = reinterpret_cast<uint8_t*>(factors + 2 * D);   // [D * G / 4]
    const int h = blockIdx.y;

    // sequence s has one item for its window and one for each whole group of new tokens
    auto fresh_groups = [&](const PagedSeq& q) {
        const int first = (q.held + G - 1) / G * G, out = quant_of(q.held + q.n, G, R);
        return out > first ? (out - first) / G : 0;
    };
    int s = blockIdx.x, sub = 0;
    if (A.b.max_new >= G) {
        if (threadIdx.x < 32) {
            const ItemPlace p = find_item(blockIdx.x, A.b.num_seqs, [&](int i) {
                PagedSeq q;
                load_seq(L, A.b, i, q);
                return 1 + fresh_groups(q);
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

    const Turn<T> plain{{nullptr, 0, 0}, D, A.vec != 0}, turn{A.rotary, D, A.vec != 0};
    const int units = turn.units();
    auto angle_of = [&](int t) { return A.rotary.table + (int64_t)t * A.rotary.dim; };
    const int64_t ring0 = ((int64_t)q.slot * H + h) * R;
    T* const k_ring = reinterpret_cast<T*>(L.k_res) + ring0 * D;
    T* const v_ring = reinterpret_cast<T*>(L.v_res) + ring0 * D;
    auto row = [&](int t) { return (int64_t)q.row0 + (t - q.held); };

    // one group of tokens t0 .. t0 + G - 1 to its page; its new tokens come from the step's rows, where `write` turned keys go out too
    auto flush = [&](int t0, bool write) {
        const int page = q.pages[t0 / L.page_tokens];
        const bool ok = (unsigned)page < (unsigned)L.num_pages;
        if (!ok && threadIdx.x == 0) atomicOr(&g_fault, kPagedFault);
        const int gpp = L.page_tokens / G;
        const int64_t g = ((int64_t)(ok ? page : 0) * H + h) * gpp + t0 % L.page_tokens / G;
        for (int pass = 0; pass < 2; ++pass) {
            __syncthreads();
            for (int i = threadIdx.x; i < G * units; i += kThreads) {
                const int t = t0 + i / units;
                int d, e;
                float x[4], y[4];
                const bool fresh = t >= q.held, keys = pass == 0;
                const Turn<T>& by = keys && fresh ? turn : plain;
                turn.places(i % units, d, e);
                const T* from = fresh ? row_of<T>(keys ? A.k : A.v, row(t), h) : (keys ? k_ring : v_ring) + (int64_t)ring_slot(t, A.b.ring_shift, R) * D;
                by.load(from, by.r.table ? angle_of(t) : nullptr, d, e, x, y);
                if (keys && fresh && write && A.k_out.data) {
                    T* to = const_cast<T*>(row_of<T>(A.k_out, row(t), h));
                    Quad<T>::store(to + d, x, A.vec);
                    if (e >= 0) Quad<T>::store(to + e, y, A.vec);
                }
                float* const to = tile + (t - t0) * S;
                *reinterpret_cast<float4*>(to + d) = make_float4(x[0], x[1], x[2], x[3]);
                if (e >= 0) *reinterpret_cast<float4*>(to + e) = make_float4(y[0], y[1], y[2], y[3]);
            }
            __syncthreads();
            if (!ok) continue;
            if (pass == 0) quantize_keys_tile<HALF_EVEN>(tile, block, D, G, L.k_codes + g * (D * G / 4), L.k_scales + g * D, L.k_zeros + g * D);
            else quantize_values_tile<HALF_EVEN>(tile, block, factors, D, G, L.v_codes + g * (D * G / 4), L.v_scales + g * D, L.v_zeros + g * D);
        }
    };
    // queries of this KV head, tokens lo .. hi - 1
    auto turn_queries = [&](int lo, int hi) {
        if (A.q.data == nullptr) return;
        const int per = A.n_rep * units;
        for (int i = threadIdx.x; i < (hi - lo) * per; i += kThreads) {
            const int t = lo + i / per, r = i % per / units;
            int d, e;
            float x[4], y[4];
            turn.places(i % units, d, e);
            turn.load(row_of<T>(A.q, row(t), h * A.n_rep + r), angle_of(t), d, e, x, y);
            T* to = const_cast<T*>(row_of<T>(A.q_out, row(t), h * A.n_rep + r));
            Quad<T>::store(to + d, x, A.vec);
            if (e >= 0) Quad<T>::store(to + e, y, A.vec);
        }
    };

    const int end = q.held + q.n, out = quant_of(end, G, R);
    const int first = (q.held + G - 1) / G * G, n_fresh = fresh_groups(q);
    if (sub > 0) {
        const int t0 = first + (sub - 1) * G;
        flush(t0, true);
        turn_queries(t0, t0 + G);
        return;
    }
    for (int t0 = quant_of(q.held, G, R); t0 < (out < first ? out : first); t0 += G) flush(t0, false);
    __syncthreads();
    // what no other CTA has: the tokens before the first whole new group and those behind the last
    const int lo = n_fresh ? first : end, hi = n_fresh ? first + n_fresh * G : end;
    const int rest = (lo - q.held) + (end - hi);
    for (int i = threadIdx.x; i < rest * units; i += kThreads) {
        const int j = i / units, t = j < lo - q.held ? q.held + j : hi + (j - (lo - q.held));
        int d, e;
        float x[4], y[4];
        turn.places(i % units, d, e);
        turn.load(row_of<T>(A.k, row(t), h), A.rotary.table ? angle_of(t) : nullptr, d, e, x, y);
        if (A.k_out.data) {
            T* to = const_cast<T*>(row_of<T>(A.k_out, row(t), h));
            Quad<T>::store(to + d, x, A.vec);
            if (e >= 0) Quad<T>::store(to + e, y, A.vec);
        }
        if (t < out) continue;
        const int64_t at = (int64_t)ring_slot(t, A.b.ring_shift, R) * D;
        Quad<T>::store(k_ring + at + d, x, A.vec);
        if (e >= 0) Quad<T>::store(k_ring + at + e, y, A.vec);
        plain.load(row_of<T>(A.v, row(t), h), nullptr, d, e, x, y);
        Quad<T>::store(v_ring + at + d, x, A.vec);
        if (e >= 0) Quad<T>::store(v_ring + at + e, y, A.vec);
    }
    turn_queries(q.held, lo);
    turn_queries(hi, end);
}

// Four channels of keys and of values of one token per thread; neighbouring threads take
// neighbouring channels, so a row leaves in whole lines.  Bound by its writes.
// grid = (pieces of rows, KV heads, sequences).
template <typename T>
__global__ void __launch_bounds__(256)
paged_read_kernel(kivi_paged_layer L, kivi_paged_batch b, const int32_t* starts, float* __restrict__ k_out, float* __restrict__ v_out) {
    stream_order();
    settle_paged(L, b);
    starts = settled(starts);
    const int s = blockIdx.z, h = blockIdx.y, D = L.head_dim, G = L.group_size, R = L.residual_cap, H = L.num_kv_heads, quads = D / 4;
    const int r0 = b.cu_new[s], r1 = b.cu_new[s + 1], held = b.seq_lens[s], start = starts[s], slot = b.slots[s];
    const int n = r1 - r0;
    if (r0 < 0 || n < 0 || r1 > b.total_new || n > b.max_new || held < 0 || held > b.max_len || start < 0 || start > held - n || slot < 0 || slot >= L.num_slots) {
        if (threadIdx.x == 0) atomicOr(&g_fault, kPagedFault);
        return;
    }
    PagedSeq q{held, n, r0, slot, b.page_table + (int64_t)s * b.table_width};
    const int out = quant_of(held, G, R), Q = G / 4, W = D < 64 ? D : 64;
    for (int64_t i = blockIdx.x * 256 + threadIdx.x; i < (int64_t)n * quads; i += (int64_t)gridDim.x * 256) {
        const int t = start + (int)(i / quads), d = 4 * (int)(i % quads);
        float4 k, v;
        if (t < out) {
            const int page = page_of(L, q, t, &g_fault), gpp = L.page_tokens / G;
            const int64_t g = ((int64_t)page * H + h) * gpp + t % L.page_tokens / G;
            const int tt = t % G;
            const uint32_t w = *reinterpret_cast<const uint32_t*>(L.k_codes + g * (D * Q) + kblock_offset(d, tt >> 2, Q, W));
            const float4 ks = *reinterpret_cast<const float4*>(L.k_scales + g * D + d), kz = *reinterpret_cast<const float4*>(L.k_zeros + g * D + d);
            const int sh = 2 * (tt & 3);
            k = make_float4(dequant((float)((w >> sh) & 3u), ks.x, kz.x), dequant((float)((w >> (sh + 8)) & 3u), ks.y, kz.y),
                            dequant((float)((w >> (sh + 16)) & 3u), ks.z, kz.z), dequant((float)((w >> (sh + 24)) & 3u), ks.w, kz.w));
            const uint32_t c = L.v_codes[g * (D * Q) + vcode_offset(tt, d / 4, D, G)];
            const int64_t at = g * D + vmeta_index(tt, d / G, D, G);
            const float vs = L.v_scales[at], vz = L.v_zeros[at];
            v = make_float4(dequant((float)(c & 3u), vs, vz), dequant((float)((c >> 2) & 3u), vs, vz),
                            dequant((float)((c >> 4) & 3u), vs, vz), dequant((float)(c >> 6), vs, vz));
        } else {
            const int64_t at = (((int64_t)slot * H + h) * R + ring_slot(t, b.ring_shift, R)) * D + d;
            float x[4];
            Quad<T>::load(reinterpret_cast<const T*>(L.k_res) + at, x, false);
            k = make_float4(x[0], x[1], x[2], x[3]);
            Quad<T>::load(reinterpret_cast<const T*>(L.v_res) + at, x, false);
            v = make_float4(x[0], x[1], x[2], x[3]);
        }
        const int64_t to = (((int64_t)r0 + i / quads) * H + h) * D + d;
        store_quad(k_out, KIVI_F32, to, k);
        store_quad(v_out, KIVI_F32, to, v);
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

int check_rows(const kivi_rows* r, const char* name, int head_dim) {
    KIVI_REQUIRE(r != nullptr && r->data != nullptr, "%s is null", name);
    KIVI_REQUIRE(r->row_stride >= 0 && r->head_stride >= 0, "%s has a negative stride", name);
    (void)head_dim;
    return KIVI_OK;
}
bool on_grid(const kivi_rows& r, int esz) {
    return (reinterpret_cast<uintptr_t>(r.data) % (4 * esz)) == 0 && r.row_stride % 4 == 0 && r.head_stride % 4 == 0;
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
    if (int rc = check_rows(new_k, "new_k", D)) return rc;
    if (int rc = check_rows(new_v, "new_v", D)) return rc;
    KIVI_REQUIRE(rounding == KIVI_ROUND_HALF_AWAY || rounding == KIVI_ROUND_HALF_EVEN, "rounding must be KIVI_ROUND_HALF_AWAY or KIVI_ROUND_HALF_EVEN");
    const bool queries = q != nullptr && q->data != nullptr;
    if (rotary != nullptr) {
        KIVI_REQUIRE(rotary_dim > 0 && rotary_dim <= D && rotary_dim % 2 == 0, "rotary_dim (%d) must be even and at most head_dim (%d)", rotary_dim, D);
        KIVI_REQUIRE(interleaved || rotary_dim % 8 == 0, "rotary_dim (%d) must be a multiple of 8 where channels half of it apart are paired", rotary_dim);
        KIVI_REQUIRE(rotary_rows >= batch->max_len, "rotary holds %d positions, max_len is %d", rotary_rows, batch->max_len);
        if (int rc = check_rows(k_out, "k_out", D)) return rc;
        if (queries) {
            KIVI_REQUIRE(n_rep >= 1, "n_rep (%d) must be positive", n_rep);
            if (int rc = check_rows(q_out, "q_out", D)) return rc;
        }
    } else {
        KIVI_REQUIRE(!queries, "queries are only taken together with rotary");
        KIVI_REQUIRE(k_out == nullptr || k_out->data == nullptr, "k_out is only written together with rotary");
    }
    const size_t smem = (size_t)G * (D + 4) * 4 + 2 * D * 4 + (size_t)D * G / 4;
    if (smem > 220 * 1024) {
        set_error("a group of %d tokens of head_dim %d does not fit shared memory", G, D);
        return KIVI_ERR_UNSUPPORTED;
    }
    if (batch->max_new == 0) { note_launches(0); return KIVI_OK; }
    AppendArgs a{};
    a.L = *layer; a.b = *batch; a.k = *new_k; a.v = *new_v; a.n_rep = n_rep;
    a.rotary = {rotary, rotary ? rotary_dim : 0, interleaved ? 1 : 0};
    if (rotary) a.k_out = *k_out;
    if (queries) { a.q = *q; a.q_out = *q_out; }
    a.vec = on_grid(a.k, esz) && on_grid(a.v, esz) && on_grid(a.k_out, esz) && on_grid(a.q, esz) && on_grid(a.q_out, esz);
    const int64_t items = batch->max_new >= G ? (int64_t)batch->num_seqs + batch->total_new / G : batch->num_seqs;
    KIVI_REQUIRE(items <= 0x7fffffff, "too many groups in one step");
    auto* const kernel = layer->res_dtype == KIVI_BF16
        ? (rounding == KIVI_ROUND_HALF_EVEN ? paged_append_kernel<__nv_bfloat16, true> : paged_append_kernel<__nv_bfloat16, false>)
        : (rounding == KIVI_ROUND_HALF_EVEN ? paged_append_kernel<float, true> : paged_append_kernel<float, false>);
    if (smem > 48 * 1024) KIVI_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    KIVI_CUDA_OK(launch(kernel, dim3((unsigned)items, (unsigned)layer->num_kv_heads), kThreads, smem, (cudaStream_t)stream, true, a));
    note_launches(1);
    return KIVI_OK;
}

extern "C" int kivi_paged_read(const kivi_paged_layer* layer, const kivi_paged_batch* batch, const int32_t* starts,
                               float* k_out, float* v_out, void* stream) {
    if (int rc = validate_paged(layer)) return rc;
    if (int rc = validate_batch(layer, batch)) return rc;
    KIVI_REQUIRE(starts != nullptr && k_out != nullptr && v_out != nullptr, "starts, k_out or v_out is null");
    if (batch->max_new == 0) { note_launches(0); return KIVI_OK; }
    int64_t pieces = ((int64_t)batch->max_new * (layer->head_dim / 4) + 255) / 256;
    if (pieces > 4096) pieces = 4096;
    auto* const kernel = layer->res_dtype == KIVI_BF16 ? paged_read_kernel<__nv_bfloat16> : paged_read_kernel<float>;
    KIVI_CUDA_OK(launch(kernel, dim3((unsigned)pieces, (unsigned)layer->num_kv_heads, (unsigned)batch->num_seqs), 256, 0, (cudaStream_t)stream, true,
                        *layer, *batch, starts, k_out, v_out));
    note_launches(1);
    return KIVI_OK;
}
