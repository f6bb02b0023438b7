// Next-token choice under temperature, top-k, top-p and min-p of each row, from given
// random numbers.
//
// m_i = exp((x_i - max) / temperature) needs no normalisation: every cut compares masses
// with masses.  A CTA walks its row up to four times, each from L2:
//   1. the largest entry and its first index;
//   2. (top-k or top-p) entries per bin of 1/256 octave of mass, 32 octaves: the counts give
//      the bin that the k-th largest is in, and bound the mass above any bin to 0.15 %, which
//      leaves a few bins that the nucleus can end in;
//   3. exact masses: all of them, those above the open bins, and a list of the entries in
//      the open bins, on which both cuts are then found, 32 keys at a time (a warp each; keys, so
//      that ties stay together);
//   4. sums of the kept masses over runs of the row, and the run, piece and entry at which
//      the sum passes uniform * all.
// Where a list does not fit (thousands of equal logits at a cut, as bf16 has them) the row is
// walked again, up to four times, each of which cuts the open keys into 256 ranges.  Lists
// come in any order and ranges add by atomics: what is summed there are whole numbers (2^-46
// of the largest mass at 50257 entries), so that the same inputs give the same id.
//
// Masses: 2^(k/32) from a table in fp64 and a correction below 2^-6 of it in fp32 (good to
// 2^-29 of the mass); the exponent (x - max) log2(e) 32 / T is a product of two-term fp32 numbers,
// good to 1e-10.  fp64 takes one addition per entry.
// Bound by latency: 4 walks of 2-3 us, 13 barriers.
#include "kivi_common.cuh"

namespace kivi {
namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32;
static_assert(kWarps == 32, "a warp looks after 32 warps' results, and fills a row of the table");
constexpr int kBins = 8192;                              // of 1/256 octave; the last holds what is below 2^-32
constexpr int kPerThread = kBins / kThreads;
constexpr int kListK = 2048, kListP = 4096;              // entries at the k-th largest, at the end of the nucleus
constexpr float kSlack = 0.0016f;                        // 2^(0.5/256) - 1 and roundings: how far a bin's mass is off its centre's

// order-preserving map float -> uint32; NaN counts as -inf, the zeros are one
__device__ __forceinline__ uint32_t ordered_key(float x) {
    if (x != x) x = -INFINITY;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_to_float(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

struct FilterArgs {
    const float *uniforms, *temperature, *top_p, *min_p;
    const int32_t* top_k;
};

struct Shared {
    uint32_t bins[kBins];
    uint32_t list_k[kListK], list_p[kListP];
    unsigned long long mass_p[kListP];                   // in whole units
    uint32_t table_hi[32][32], table_lo[32][32];         // words of 2^(i/32), a column for each lane: no two lanes meet in a bank
    double sum[kWarps];
    unsigned long long range[256], open_base;
    uint32_t flag[2][kWarps];
    uint32_t open_lo, open_hi;
    int draw_lo, draw_hi;
    float part[kWarps];
    int count[kWarps];
    uint32_t key[kWarps];
    int first, bin_k, need, zone_lo, zone_hi, n_k, n_p, pick, last;
    float mass_k[2], tail;
    uint32_t cut;
};

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
// Sums over the block of three numbers of each thread, through 24 KB of shared memory: three
// warps add them up (32 warps that shuffle share one pipe: 2500 cycles for a sum).
__device__ __forceinline__ void block_sums(double a, double b, double c, double* scratch, double* out) {
    scratch[threadIdx.x] = a;
    scratch[kThreads + threadIdx.x] = b;
    scratch[2 * kThreads + threadIdx.x] = c;
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp < 3) {
        double x[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int i = 0; i < kThreads / 32; ++i) x[i & 3] += scratch[warp * kThreads + 32 * i + lane];
        const double sum = warp_sum((x[0] + x[1]) + (x[2] + x[3]));
        if (lane == 0) out[warp] = sum;
    }
    __syncthreads();
}

// The entries of an aligned 16 bytes
template <typename T> struct Granule;
template <> struct Granule<float> {
    static constexpr int kSize = 4;
    __device__ static void get(const uint4& v, float (&x)[4]) {
        x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
    }
};
template <> struct Granule<__nv_bfloat16> {
    static constexpr int kSize = 8;
    __device__ static void get(const uint4& v, float (&x)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
};
// f(x, index) for entries [lo, hi) of a row, by `n` threads of which this is number `me`:
// 16 bytes at a time, four in flight, the ends one by one.
template <typename T, typename F>
__device__ __forceinline__ void walk(const T* row, int lo, int hi, int me, int n, const F& f) {
    constexpr int kSize = Granule<T>::kSize;
    const int off = (int)((reinterpret_cast<uintptr_t>(row + lo) & 15u) / sizeof(T));
    int body = lo + (off ? kSize - off : 0);             // first entry on a 16-byte boundary
    if (body > hi) body = hi;
    const int granules = (hi - body) / kSize, tail = body + granules * kSize;
    for (int i = lo + me; i < body; i += n) f((float)row[i], i);
    const uint4* g = reinterpret_cast<const uint4*>(row + body);
    for (int i = me; i < granules; i += 4 * n) {
        uint4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j * n < granules) v[j] = g[i + j * n];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j * n < granules) {
                float x[kSize];
                Granule<T>::get(v[j], x);
#pragma unroll
                for (int e = 0; e < kSize; ++e) f(x[e], body + (i + j * n) * kSize + e);
            }
    }
    for (int i = tail + me; i < hi; i += n) f((float)row[i], i);
}

// Masses relative to the row's largest entry.
struct Masses {
    float largest, c_hi, c_lo;                           // 32 log2(e) / T in two terms
    bool only_largest;                                   // an infinite largest, or a temperature that leaves nothing else
    const Shared* s;

    // mass = hi + lo; false: none
    __device__ __forceinline__ bool get(float x, double& hi, float& lo) const {
        hi = 0.0; lo = 0.0f;
        if (only_largest) {
            if (x == largest) hi = 1.0;
            return x == largest;
        }
        const float d = __fsub_rn(x, largest);
        const float p = __fmul_rn(d, c_hi);
        if (!(p > -31000.0f)) return false;              // below 2^-968, -inf or NaN
        // d = x - largest to the last bit: what the subtraction rounded away
        const float b = __fsub_rn(x, d), lost = __fadd_rn(__fsub_rn(x, __fadd_rn(d, b)), __fsub_rn(b, largest));
        const float t = __fadd_rn(p, 12582912.0f), whole = __fsub_rn(t, 12582912.0f);        // (1.5 * 2^23: rounds to a whole number)
        const int k = __float_as_int(t) - 0x4b400000, n = k >> 5;
        const float r = __fsub_rn(p, whole) + (__fmaf_rn(d, c_hi, -p) + __fmaf_rn(d, c_lo, __fmul_rn(lost, c_hi)));
        const uint32_t w1 = s->table_hi[k & 31][threadIdx.x & 31], w0 = s->table_lo[k & 31][threadIdx.x & 31];
        hi = __hiloint2double((int)w1 + (n << 20), (int)w0);
        const float u = r * 0.02166084939249829f;        // ln 2 / 32
        const float e = u * fmaf(u, fmaf(u, fmaf(u, 0.041666667f, 0.16666667f), 0.5f), 1.0f);       // 2^(r/32) - 1 to u^5 / 120 = 1e-12
        // (a mass below 2^-120 needs no correction)
        lo = n > -120 ? e * __uint_as_float(((__funnelshift_l(w0, w1, 3) & 0x7fffffu) | 0x3f800000u) + (uint32_t)(n * (1 << 23))) : 0.0f;
        return true;
    }
    // bin of an entry, falling with it; -1 for one that can have no mass (-inf, NaN)
    __device__ __forceinline__ int bin(float x) const {
        const float p = __fmul_rn(__fmul_rn(__fsub_rn(largest, x), c_hi), 8.0f);
        return p < (float)(kBins - 1) ? __float_as_int(__fadd_rn(p, 12582912.0f)) - 0x4b400000 : x > -INFINITY ? kBins - 1 : -1;
    }
};

// sums of two terms, folded once at the end
struct Sum {
    double hi = 0.0;
    float lo = 0.0f;
    __device__ __forceinline__ void add(double h, float l) { hi += h; lo += l; }
    __device__ __forceinline__ double value() const { return hi + (double)lo; }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
sample_filtered_kernel(const T* logits, int vocab, int64_t row_stride, FilterArgs f, int64_t* __restrict__ ids) {
    extern __shared__ __align__(16) unsigned char smem[];
    Shared& s = *reinterpret_cast<Shared*>(smem);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.x;
    {
        const double t = exp2((double)warp * (1.0 / 32.0));
        s.table_hi[warp][lane] = (uint32_t)__double2hiint(t);
        s.table_lo[warp][lane] = (uint32_t)__double2loint(t);
    }
    if (tid == 0) { s.first = 0x7fffffff; s.bin_k = kBins; s.need = 0; s.zone_lo = kBins; s.zone_hi = -1; s.n_k = 0; s.n_p = 0; s.pick = 0x7fffffff; s.last = -1; }
    for (int i = tid; i < kBins; i += kThreads) s.bins[i] = 0u;
    stream_order();
    const T* const row = settled(logits) + (int64_t)b * row_stride;
    const float u = settled(f.uniforms)[b], temperature = f.temperature ? settled(f.temperature)[b] : 1.0f;
    const float top_p = f.top_p ? settled(f.top_p)[b] : 1.0f, min_p = f.min_p ? settled(f.min_p)[b] : 0.0f;
    const int top_k = f.top_k ? settled(f.top_k)[b] : 0;
    // whole units of mass: a row's sum stays below 2^62
    const double unit = (double)(1ll << (__clz(vocab) + 30 < 50 ? __clz(vocab) + 30 : 50));
    auto units = [&](double mass) { return (unsigned long long)__double2ll_rn(mass * unit); };
    const bool cut_k = top_k > 0 && top_k < vocab, cut_p = top_p < 1.0f;

    // ---- 1. the largest and its first index ----
    float best = -INFINITY;
    int at = 0x7fffffff;
    walk(row, 0, vocab, tid, kThreads, [&](float x, int i) {
        if (x > best || (x == best && i < at)) { best = x; at = i; }
    });
    const uint32_t mine = ordered_key(best), warp_best = __reduce_max_sync(0xffffffffu, mine);
    if (lane == 0) s.key[warp] = warp_best;
    __syncthreads();
    const uint32_t top = __reduce_max_sync(0xffffffffu, s.key[lane]);
    if (mine == top) atomicMin(&s.first, at);
    __syncthreads();
    const float largest = key_to_float(top);
    if (!(temperature > 0.0f) || largest == -INFINITY) {
        if (tid == 0) ids[b] = largest == -INFINITY ? 0 : s.first;
        return;
    }
    Masses m;
    m.largest = largest;
    const double c = 32.0 * 1.4426950408889634 / (double)temperature;
    m.c_hi = (float)c;
    m.c_lo = (float)(c - (double)m.c_hi);
    m.only_largest = largest == INFINITY || temperature < 1e-30f;
    m.s = &s;

    uint32_t cut = 0u;                                   // least key that is kept
    if ((cut_k || cut_p) && !m.only_largest) {
        // ---- 2. entries per bin ----
        walk(row, 0, vocab, tid, kThreads, [&](float x, int) {
            const int bin = m.bin(x);
            if (bin >= 0) atomicAdd(&s.bins[bin], 1u);
        });
        __syncthreads();
        int count[kPerThread], n = 0;
        float mass = 0.0f;                               // of the thread's bins, by their centres
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            const int bin = tid * kPerThread + i;
            count[i] = (int)s.bins[bin];
            n += count[i];
            mass += (float)count[i] * exp2f((float)-bin * (1.0f / 256.0f));
        }
        int n_upto = n;
        float m_upto = mass;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int x = __shfl_up_sync(0xffffffffu, n_upto, o);
            const float y = __shfl_up_sync(0xffffffffu, m_upto, o);
            if (lane >= o) { n_upto += x; m_upto += y; }
        }
        if (lane == 31) { s.count[warp] = n_upto; s.part[warp] = m_upto; }
        if (tid == kThreads - 1) s.tail = (float)count[kPerThread - 1] * exp2f(-(kBins - 1) / 256.0f);        // (anything down to nothing)
        __syncthreads();
        float all = 0.0f, all_most = 0.0f;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) { n_upto += s.count[w]; m_upto += s.part[w]; }
            all += s.part[w];
        }
        if (cut_k) {
            int upto = n_upto - n;
            float above = m_upto - mass;
#pragma unroll
            for (int i = 0; i < kPerThread; ++i) {
                const float w = exp2f((float)-(tid * kPerThread + i) * (1.0f / 256.0f));
                if (upto < top_k && upto + count[i] >= top_k) { s.bin_k = tid * kPerThread + i; s.need = top_k - upto; s.mass_k[0] = above + (float)(top_k - upto) * w; s.mass_k[1] = above + (float)count[i] * w; }
                upto += count[i];
                above += (float)count[i] * w;
            }
            __syncthreads();
        }
        // what the top-k cut leaves: ties with the k-th stay, up to the whole of its bin (fewer than top_k
        // entries with a mass: no cut)
        all_most = s.bin_k < kBins ? s.mass_k[1] : all;
        if (s.bin_k < kBins) all = s.mass_k[0];
        const int bin_k = s.bin_k;
        if (cut_p) {
            // mass above an entry of a bin: between that above the bin and that up to its end; a float's
            // worth of doubt on sums of thousands of terms is inside the slack
            const float lo = top_p * (all - s.tail) * (1.0f - kSlack), hi = top_p * all_most * (1.0f + kSlack);
            float above = m_upto - mass;
#pragma unroll
            for (int i = 0; i < kPerThread; ++i) {
                const int bin = tid * kPerThread + i;
                const float upto = above + (float)count[i] * exp2f((float)-bin * (1.0f / 256.0f));
                if (count[i] > 0 && bin <= bin_k) {
                    const bool stays = upto * (1.0f + kSlack) < lo && bin < kBins - 1, goes = above * (1.0f - kSlack) >= hi;
                    if (!stays && !goes) { atomicMin(&s.zone_lo, bin); atomicMax(&s.zone_hi, bin); }
                }
                above = upto;
            }
        }
        __syncthreads();
        const int zone_lo = s.zone_lo, zone_hi = s.zone_hi;
        // ---- 3. exact masses ----
        Sum in, over;                                    // bins before bin_k; of those, before the zone
        walk(row, 0, vocab, tid, kThreads, [&](float x, int) {
            const int bin = m.bin(x);
            if (bin < 0 || bin > bin_k) return;
            const bool at_k = bin == bin_k, at_p = bin >= zone_lo && bin <= zone_hi;
            if (at_k) { const int j = atomicAdd(&s.n_k, 1); if (j < kListK) s.list_k[j] = ordered_key(x); }
            if (!cut_p) return;
            double h;
            float l;
            m.get(x, h, l);
            if (!at_k) in.add(h, l);
            if (at_p) { const int j = atomicAdd(&s.n_p, 1); if (j < kListP) { s.list_p[j] = ordered_key(x); s.mass_p[j] = units(h + (double)l); } }
            else if (bin < zone_lo) over.add(h, l);
        });
        __syncthreads();
        const int n_k = s.n_k, n_p = s.n_p;
        // The largest key for which holds(key), asked of whole warps, is true; it falls from true to
        // false between lo and hi (0 if it is nowhere true).  32 keys at a time.
        auto search = [&](uint32_t lo, uint32_t hi, auto&& holds) {
            uint32_t found = 0u;
            int buf = 0;
            for (int shift = hi > lo ? (31 - __clz(hi - lo)) / 5 * 5 : 0; shift >= 0; shift -= 5, buf ^= 1) {
                const uint32_t off = (uint32_t)warp << shift;
                const bool yes = (off >> shift) == (uint32_t)warp && off <= hi - lo && holds(lo + off);
                if (lane == 0) s.flag[buf][warp] = yes;
                __syncthreads();
                const unsigned all_yes = __ballot_sync(0xffffffffu, s.flag[buf][lane] != 0u);
                if (!all_yes) return found;
                found = lo + ((uint32_t)(31 - __clz(all_yes)) << shift);
                lo = found;
                hi = min(hi, lo + ((1u << shift) - 1u));
            }
            return found;
        };
        auto ends = [&](const uint32_t* list, int n, uint32_t& lo, uint32_t& hi) {
            lo = 0xffffffffu; hi = 0u;
            for (int i = lane; i < n; i += 32) { lo = min(lo, list[i]); hi = max(hi, list[i]); }
            lo = __reduce_min_sync(0xffffffffu, lo);
            hi = __reduce_max_sync(0xffffffffu, hi);
        };
        // The same over the row: amount(x, key) of the keys in lo .. hi, 256 ranges of keys at a time;
        // the largest key at which what is at or above it reaches `most` (in the amount's units).
        auto search_row = [&](uint32_t lo, uint32_t hi, unsigned long long most, auto&& amount) {
            if (tid == 0) { s.open_lo = lo; s.open_hi = hi; s.open_base = 0; }
            for (;;) {
                __syncthreads();
                lo = s.open_lo; hi = s.open_hi;
                if (tid < 256) s.range[tid] = 0;
                __syncthreads();
                const int bits = 32 - __clz(hi - lo), shift = hi > lo && bits > 8 ? bits - 8 : 0;
                walk(row, 0, vocab, tid, kThreads, [&](float x, int) {
                    const uint32_t key = ordered_key(x);
                    if (key < lo || key > hi) return;
                    const unsigned long long a = amount(x);
                    if (a) atomicAdd(&s.range[(key - lo) >> shift], a);
                });
                __syncthreads();
                if (tid == 0) {
                    unsigned long long upto = s.open_base;
                    int i = 255;
                    for (; i >= 0; --i) {
                        if (upto + s.range[i] >= most) break;
                        upto += s.range[i];
                    }
                    s.open_base = upto;
                    if (i < 0) { s.open_lo = 1u; s.open_hi = 0u; }               // nowhere
                    else { s.open_lo = lo + ((uint32_t)i << shift); s.open_hi = min(hi, s.open_lo + ((1u << shift) - 1u)); }
                }
                __syncthreads();
                if (s.open_lo > s.open_hi) return 0u;
                if (shift == 0) return s.open_lo;
            }
        };
        if (cut_k && bin_k < kBins) {
            if (n_k <= kListK) {
                uint32_t lo, hi;
                ends(s.list_k, n_k, lo, hi);
                const int need = s.need;
                cut = search(lo, hi, [&](uint32_t key) {
                    int c1 = 0;
                    for (int i = lane; i < n_k; i += 32) c1 += s.list_k[i] >= key;
                    return __reduce_add_sync(0xffffffffu, c1) >= need;
                });
            } else {
                cut = search_row(0u, 0xffffffffu, (unsigned long long)top_k, [&](float) { return 1ull; });
            }
        }
        if (cut_p) {
            // the whole mass: bins before bin_k and what of that bin stays
            // (whole units below 2^53 of the list: exact in any order)
            double rest = 0.0;
            auto add_rest = [&](float x) { double h; float l; m.get(x, h, l); rest += (double)units(h + (double)l); };
            if (bin_k < kBins) {
                if (n_k <= kListK) {
                    for (int i = tid; i < n_k; i += kThreads)
                        if (s.list_k[i] >= cut) add_rest(key_to_float(s.list_k[i]));
                } else {
                    walk(row, 0, vocab, tid, kThreads, [&](float x, int) { if (m.bin(x) == bin_k && ordered_key(x) >= cut) add_rest(x); });
                }
            }
            __syncthreads();
            block_sums(in.value(), over.value(), rest, reinterpret_cast<double*>(s.bins), s.sum);
            double most = (double)top_p * (s.sum[0] + s.sum[2] / unit);
            // (the least key above which there is less than top_p is the largest one at or above which there is no less)
            most = (most - s.sum[1]) * unit;
            uint32_t key = top;                          // (top_p <= 0: the largest alone)
            if (most > 0.0) {
                const unsigned long long most_u = (unsigned long long)__double2ll_ru(most);
                if (n_p <= kListP) {
                    uint32_t lo, hi;
                    ends(s.list_p, n_p, lo, hi);
                    lo = max(lo, cut);                   // (the list may hold what the top-k cut took)
                    key = lo > hi ? 0u : search(lo, hi, [&](uint32_t probe) {
                        unsigned long long x = 0;
                        for (int i = lane; i < n_p; i += 32) x += s.list_p[i] >= probe ? s.mass_p[i] : 0ull;
                        // (21 bits at a time: reductions of 32-bit numbers)
                        const unsigned long long a = __reduce_add_sync(0xffffffffu, (uint32_t)x & 0x1fffffu), b = __reduce_add_sync(0xffffffffu, (uint32_t)(x >> 21) & 0x1fffffu),
                                                 c = __reduce_add_sync(0xffffffffu, (uint32_t)(x >> 42));
                        return a + (b << 21) + (c << 42) >= most_u;
                    });
                } else {
                    key = search_row(max(cut, 1u), top, most_u, [&](float x) {
                        const int bin = m.bin(x);
                        if (bin < zone_lo || bin > zone_hi) return 0ull;
                        double h;
                        float l;
                        m.get(x, h, l);
                        return units(h + (double)l);
                    });
                }
            }
            cut = max(cut, min(key, top));
        }
    }
    // ---- 4. the draw ----
    const float cut_x = cut ? key_to_float(cut) : -INFINITY;
    auto kept = [&](float x, double& h, float& l) {
        if (!(x >= cut_x) || !m.get(x, h, l)) return false;
        return x == largest || !(min_p > 0.0f) || h + (double)l >= (double)min_p;
    };
    // sum of the entries [lo, hi) by this warp
    auto run_sum = [&](int lo, int hi) {
        Sum x;
        walk(row, lo, hi, lane, 32, [&](float v, int) {
            double h;
            float l;
            if (kept(v, h, l)) x.add(h, l);
        });
        return warp_sum(x.value());
    };
    int lo = 0, hi = vocab;
    double before = 0.0, target = 0.0;
    for (int level = 0; level < 2; ++level) {
        // the run of 32 that the sum passes the target in; the last with a mass where roundings leave none
        const int per = (hi - lo + kWarps - 1) / kWarps;
        const int a = min(lo + warp * per, hi), z = min(a + per, hi);
        const double sum = run_sum(a, z);
        __syncthreads();
        if (lane == 0) s.sum[warp] = sum;
        __syncthreads();
        if (warp == 0) {
            double upto = s.sum[lane];
            const bool some = upto > 0.0;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const double x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += x;
            }
            if (level == 0) target = (double)u * __shfl_sync(0xffffffffu, upto, 31);
            const unsigned passes = __ballot_sync(0xffffffffu, some && before + upto > target), holds = __ballot_sync(0xffffffffu, some);
            const int w = passes ? __ffs(passes) - 1 : 31 - __clz(holds);
            before += __shfl_sync(0xffffffffu, upto, w) - s.sum[w];
            if (lane == 0) { s.draw_lo = min(lo + w * per, hi); s.draw_hi = min(min(lo + w * per, hi) + per, hi); }
        }
        __syncthreads();
        lo = s.draw_lo;
        hi = s.draw_hi;
    }
    if (warp == 0) {
        int pick = -1, last = -1;
        for (int i0 = lo; i0 < hi && pick < 0; i0 += 32) {
            const int i = i0 + lane;
            double h = 0.0;
            float l = 0.0f;
            const bool stays = i < hi && kept((float)row[i], h, l);
            double upto = stays ? h + (double)l : 0.0;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const double x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += x;
            }
            const unsigned passes = __ballot_sync(0xffffffffu, stays && before + upto > target), holds = __ballot_sync(0xffffffffu, stays);
            if (passes) pick = i0 + __ffs(passes) - 1;
            if (holds) last = i0 + 31 - __clz(holds);
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (lane == 0) ids[b] = pick >= 0 ? pick : last;
    }
}

}  // namespace
}  // namespace kivi

using namespace kivi;

extern "C" int kivi_sample_filtered(const void* logits, int dtype, int batch, int vocab, int64_t row_stride,
                                    const float* uniforms, const float* temperature, const int32_t* top_k,
                                    const float* top_p, const float* min_p, int64_t* ids_out, void* stream) {
    KIVI_REQUIRE(logits != nullptr && uniforms != nullptr && ids_out != nullptr, "logits, uniforms or ids_out is null");
    KIVI_REQUIRE(dtype == KIVI_F32 || dtype == KIVI_BF16, "logits dtype must be KIVI_F32 or KIVI_BF16");
    KIVI_REQUIRE(batch > 0 && vocab > 0 && (row_stride >= vocab || row_stride == 0), "batch (%d) and vocab (%d) must be positive, row_stride >= vocab or 0", batch, vocab);
    // (indices step past the end of a row)
    KIVI_REQUIRE(vocab <= (1 << 30), "vocab (%d) must be at most 2^30", vocab);
    const FilterArgs f{uniforms, temperature, top_p, min_p, top_k};
    auto go = [&](auto* kernel, auto* x) {
        KIVI_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared)));
        KIVI_CUDA_OK(launch(kernel, dim3((unsigned)batch), kThreads, sizeof(Shared), (cudaStream_t)stream, true, x, vocab, row_stride, f, ids_out));
        note_launches(1);
        return KIVI_OK;
    };
    return dtype == KIVI_BF16 ? go(sample_filtered_kernel<__nv_bfloat16>, reinterpret_cast<const __nv_bfloat16*>(logits))
                              : go(sample_filtered_kernel<float>, reinterpret_cast<const float*>(logits));
}
