// Next-token choice under temperature, top-k, top-p and min-p of each row, from given
// random numbers.
//
// m_i = exp((x_i - max) / temperature) needs no normalisation: every cut compares masses
// with masses.  A CTA (or a few, of a long row) walks its row up to four times, each from L2:
//   1. the largest entry and its first index;
//   2. (top-k or top-p) entries per bin of 1/256 octave of mass, 32 octaves: the counts give
//      the bin that the k-th largest is in, and bound the mass above any bin to 0.15 %, which
//      leaves a few bins that the nucleus can end in;
//   3. exact masses: all of them, those above the open bins, and a list of the entries in
//      the open bins, on which both cuts are then found, 256 ranges of keys at a time (keys, so
//      that ties stay together).  A warp has a run of the row, so this walk also gives the runs'
//      sums of what is kept for certain; the list adds its own.  What belongs where is told by
//      thresholds on the logits, looked up once: bins, and the masses that min_p leaves, fall with them;
//   4. the run, the piece of it and the entry at which the sum passes uniform * all.  Only where
//      there was no third walk (no cut but min_p, or min_p above them) is the row walked for the sums.
// Where a list does not fit (thousands of equal logits at a cut, as bf16 has them) the row is
// walked again, up to four times, each of which cuts the open keys into 256 ranges.  Lists
// come in any order and ranges add by atomics: what is summed there are whole numbers (2^-46
// of the largest mass at 50257 entries), so that the same inputs give the same id.
//
// Masses: 2^(k/32) from a table in fp64, times 1 and a correction below 2^-6 in fp32 (good to
// 2^-29).  The exponent x c - L, c = 32 log2(e) / T, is taken with L on a grid on
// which L and the whole number k add exactly, so one fused operation leaves its fraction.
//
// Bound by issue slots where rows are long, most of them the third walk's (130000 bf16 logits in
// one CTA: 140000 cycles a row, of them maximum 11000, bins 23000-31000, third walk 75000), else by
// latency: fourteen barriers up to the exact masses, seven to nine for each list that is searched, five
// for the draw, and what hangs on them.  50257 fp32 logits: one row 29 us, 128 rows
// of all filters 33; 64 rows of 130000 bf16 60.  Integer instructions take two slots, so
// masses use few of them (two-word masses by bit operations: 92 us).
#include "kivi_common.cuh"

#include <cooperative_groups.h>
#include <type_traits>

namespace cg = cooperative_groups;

namespace kivi {
namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32;
static_assert(kWarps == 32, "a warp looks after 32 warps' results, and fills a row of the table");
// CTAs of a row (a cluster), and the entries that one is worth: adding up the bins of the others and
// five barriers cost about what 20000 entries take.  us with one, two, four and eight CTAs, top-p: 16 x 130000
// bf16 60 46 37 69 (16 clusters of eight do not all find room), 64 x 130000 81 60, 64 x 50257 fp32 42 37,
// 16 x 50257 35 33 32 63, 1 x 50257 28 29 30 36, 8 x 16000 19 23 24.
constexpr int kMaxCtas = 4, kLeast = 25000;
constexpr int kBins = 8192;                              // of 1/256 octave; the last holds what is below 2^-32
constexpr int kPerThread = kBins / kThreads;
constexpr int kListK = 2048, kListP = 8192;              // entries at the k-th largest, at the end of the nucleus
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

struct Entry { uint32_t key; int index; };
struct Shared {
    uint32_t bins[kBins];
    Entry list_k[kListK], list_p[kListP];
    unsigned long long mass_p[kListP];                   // in whole units
    uint2 table[32][32];                                 // 2^(i/32), less the constant of power(); a column for each lane: no two lanes meet in a bank
    double sum[kWarps], runs[kWarps];
    uint32_t range[256][3], run_units[kMaxCtas * kWarps][3];         // whole units in three parts of 18 bits
    // from all CTAs of the row (the last three: to the first one)
    uint32_t peer_key[kMaxCtas];
    int peer_first[kMaxCtas];
    double all_runs[kMaxCtas * kWarps], sum_in[kMaxCtas], sum_over[kMaxCtas];
    unsigned long long wide_range[256], open_base;
    uint32_t open_lo, open_hi;
    int draw_lo, draw_hi, draw_run;
    float part[kWarps];
    int count[kWarps];
    uint32_t key[kWarps];
    int first, bin_k, need, zone_lo, zone_hi, n_k, n_p;
    float mass_k[2], tail;
    uint32_t over_key, zone_key, in_key, k_key, min_key;
};
// (a list's units: 8192 times 2^18 stays in 32 bits)
__device__ __forceinline__ void add_units(uint32_t (&to)[3], unsigned long long x) {
    atomicAdd(&to[0], (uint32_t)x & 0x3ffffu);
    if (x >> 18) atomicAdd(&to[1], (uint32_t)(x >> 18) & 0x3ffffu);
    if (x >> 36) atomicAdd(&to[2], (uint32_t)(x >> 36));
}
__device__ __forceinline__ unsigned long long units_of(const uint32_t (&x)[3]) {
    return x[0] + ((unsigned long long)x[1] << 18) + ((unsigned long long)x[2] << 36);
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
// Sums over the block of two numbers of each thread, and of the second over each warp, through
// 16 KB of shared memory: three warps add them up (32 warps that shuffle share one pipe: 2500 cycles
// for a sum).
__device__ __forceinline__ void block_sums(double a, double b, double* scratch, double* out, double* runs) {
    scratch[threadIdx.x] = a;
    scratch[kThreads + threadIdx.x] = b;
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp < 3) {
        double x[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int i = 0; i < kWarps; ++i) x[i & 3] += scratch[warp == 2 ? kThreads + 32 * lane + ((i + lane) & 31) : warp * kThreads + 32 * i + lane];
        const double sum = (x[0] + x[1]) + (x[2] + x[3]);
        if (warp == 2) runs[lane] = sum;
        else {
            const double all = warp_sum(sum);
            if (lane == 0) out[warp] = all;
        }
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
// 16 bytes at a time, the ends one by one.  kAtOnce: granules whose code is laid out side by side; four are in flight.
template <typename T, int kAtOnce = 4, typename F>
__device__ __forceinline__ void walk(const T* row, int lo, int hi, int me, int n, const F& f) {
    constexpr int kSize = Granule<T>::kSize;
    const int off = (int)((reinterpret_cast<uintptr_t>(row + lo) & 15u) / sizeof(T));
    int body = lo + (off ? kSize - off : 0);             // first entry on a 16-byte boundary
    if (body > hi) body = hi;
    const int granules = (hi - body) / kSize, tail = body + granules * kSize;
    const uint4* g = reinterpret_cast<const uint4*>(row + body);
    auto entries = [&](const uint4& v, int at) {
        float x[kSize];
        Granule<T>::get(v, x);
#pragma unroll
        for (int e = 0; e < kSize; ++e) f(x[e], body + at * kSize + e);
    };
    if constexpr (kAtOnce == 1) {
        // the ends, and granules of which the next two are on their way
#pragma unroll 1
        for (int i = me; i < (body - lo) + (hi - tail); i += n) { const int at = i < body - lo ? lo + i : tail + (i - (body - lo)); f((float)row[at], at); }
        uint4 v = make_uint4(0u, 0u, 0u, 0u), v1 = v, v2 = v;
        if (me < granules) v = g[me];
        if (me + n < granules) v1 = g[me + n];
        if (me + 2 * n < granules) v2 = g[me + 2 * n];
#pragma unroll 1
        for (int i = me; i < granules; i += n) {
            uint4 v3 = v;
            if (i + 3 * n < granules) v3 = g[i + 3 * n];
            entries(v, i);
            v = v1; v1 = v2; v2 = v3;
        }
    } else {
        for (int i = lo + me; i < body; i += n) f((float)row[i], i);
        for (int i = me; i < granules; i += 4 * n) {
            uint4 v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j * n < granules) v[j] = g[i + j * n];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j * n < granules) entries(v[j], i + j * n);
        }
        for (int i = tail + me; i < hi; i += n) f((float)row[i], i);
    }
}

// Masses relative to the row's largest entry.
struct Masses {
    float largest, half_largest, c_hi, c_lo;             // 32 log2(e) / T in two terms
    float l_hi, l_lo;                                    // the largest times that: on a grid, and the rest
    float lowest;                                        // about 2^-940 of the largest's mass
    bool only_largest;                                   // an infinite largest, or a temperature that leaves nothing else
    bool narrow;                                         // |l_hi| below 2^18: the grid is 2^-5 or finer
    bool bounded;                                        // narrow, and `lowest` is a number (not at temperatures of 2^115 and more)
    const Shared* s;

    __device__ __forceinline__ void set(float top, float temperature) {
        largest = top;
        half_largest = 0.5f * top;
        const double c = 32.0 * 1.4426950408889634 / (double)temperature, l = (double)top * c;
        c_hi = (float)c;
        c_lo = (float)(c - (double)c_hi);
        only_largest = largest == INFINITY || temperature < 1e-30f;
        narrow = fabs(l) < 262144.0;
        // l + whole numbers down to -31000, in 24 bits: steps of 2^-8 up to 2^16, of 2^-5 up to 2^18 + 31000
        const double steps = fabs(l) < 32768.0 ? 256.0 : 32.0, grid = rint(l * steps) / steps;
        l_hi = (float)grid;
        l_lo = (float)(l - grid);
        lowest = top - 30000.0f / c_hi;
        bounded = narrow && lowest > -INFINITY;
    }
    // 2^((k + r) / 32), t = k + 1.5 * 2^23.  Few instructions of the integer pipe, which bounds the third walk.
    __device__ __forceinline__ double power(float t, float r) const {
        const uint32_t b = __float_as_uint(t), i = b & 31u;          // (the constant's low bits are 0)
        const uint2 w = s->table[i][threadIdx.x & 31];
        const double at = __hiloint2double((int)((b - i) * 32768u + w.y), (int)w.x);
        const float u = r * 0.02166084939249829f;        // ln 2 / 32
        const float e = u * fmaf(u, fmaf(u, fmaf(u, 0.041666667f, 0.16666667f), 0.5f), 1.0f);       // 2^(r/32) - 1 to u^5 / 120 = 2e-12
        return fma(at, (double)e, at);
    }
    __device__ __forceinline__ double narrow_power(float x, float p) const {
        const float t = __fadd_rn(p, 12582912.0f), whole = __fsub_rn(t, 12582912.0f);        // (1.5 * 2^23: rounds to a whole number)
        return power(t, __fadd_rn(__fmaf_rn(x, c_hi, -__fadd_rn(l_hi, whole)), __fmaf_rn(x, c_lo, -l_lo)));
    }
    // 0: none (2^-968 and less, -inf, NaN)
    __device__ __forceinline__ double get(float x) const {
        if (only_largest) return x == largest ? 1.0 : 0.0;
        if (narrow) {
            const float p = __fmaf_rn(x, c_hi, -l_hi);
            return p > -31000.0f ? narrow_power(x, p) : 0.0;
        }
        const float d = __fsub_rn(x, largest), p = __fmul_rn(d, c_hi);
        if (!(p > -31000.0f)) return 0.0;
        // d = x - largest to the last bit: what the subtraction rounded away
        const float b = __fsub_rn(x, d), lost = __fadd_rn(__fsub_rn(x, __fadd_rn(d, b)), __fsub_rn(b, largest));
        const float t = __fadd_rn(p, 12582912.0f);
        return power(t, __fsub_rn(p, __fsub_rn(t, 12582912.0f)) + (__fmaf_rn(d, c_hi, -p) + __fmaf_rn(d, c_lo, __fmul_rn(lost, c_hi))));
    }
    // The same for sums, where what has no mass may count as 2^-938 (kBounded: `bounded` and not `only_largest`).
    template <bool kBounded>
    __device__ __forceinline__ double get_any(float x) const {
        if constexpr (kBounded) { x = fmaxf(x, lowest); return narrow_power(x, __fmaf_rn(x, c_hi, -l_hi)); }
        else return get(x);
    }
    // bin of an entry, falling with it; -1 for one that can have no mass (-inf, NaN).  (Half the difference: the
    // whole may be above fp32's largest number.)
    __device__ __forceinline__ int bin(float x) const {
        const float p = __fmul_rn(__fmul_rn(__fmaf_rn(-0.5f, x, half_largest), c_hi), 16.0f);
        return p < (float)(kBins - 1) ? __float_as_int(__fadd_rn(p, 12582912.0f)) - 0x4b400000 : x > -INFINITY ? kBins - 1 : -1;
    }
};

// kMany: a cluster of CTAs has a row.  Each walks its part; bins are added up by all, lists and sums go
// to the first, which ends the draw.  What the CTAs decide on (bins, thresholds) is the same in all.
template <typename T, bool kMany>
__global__ void __launch_bounds__(kThreads, 1)
sample_filtered_kernel(const T* logits, int vocab, int64_t row_stride, FilterArgs f, int64_t* __restrict__ ids) {
    extern __shared__ __align__(16) unsigned char smem[];
    Shared& s = *reinterpret_cast<Shared*>(smem);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const cg::cluster_group cluster = cg::this_cluster();
    const int ctas = kMany ? (int)cluster.num_blocks() : 1, rank = kMany ? (int)cluster.block_rank() : 0, b = (int)blockIdx.x / ctas;
    Shared& lead = kMany ? *cluster.map_shared_rank(&s, 0) : s;
    auto sync_row = [&] { if constexpr (kMany) cluster.sync(); else __syncthreads(); };
    {
        const double t = exp2((double)warp * (1.0 / 32.0));
        s.table[warp][lane] = make_uint2((uint32_t)__double2loint(t), (uint32_t)__double2hiint(t) - 0x4b400000u * 32768u);
    }
    if (tid == 0) { s.first = 0x7fffffff; s.bin_k = kBins; s.need = 0; s.zone_lo = kBins; s.zone_hi = -1; s.n_k = 0; s.n_p = 0; s.min_key = 0u; }
    if (tid < 3 * kMaxCtas * kWarps) s.run_units[tid / 3][tid % 3] = 0u;
    for (int i = tid; i < kBins; i += kThreads) s.bins[i] = 0u;
    stream_order();
    if constexpr (kMany) cluster.sync();                 // (all are there, and their shared memory is laid out)
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
    const int n_runs = ctas * kWarps, run = (vocab + n_runs - 1) / n_runs;          // a warp's part of the row
    const int part_lo = min(rank * kWarps * run, vocab), part_hi = min(part_lo + kWarps * run, vocab);
    walk(row, part_lo, part_hi, tid, kThreads, [&](float x, int i) {
        if (x > best || (x == best && i < at)) { best = x; at = i; }
    });
    const uint32_t mine = ordered_key(best), warp_best = __reduce_max_sync(0xffffffffu, mine);
    if (lane == 0) s.key[warp] = warp_best;
    __syncthreads();
    uint32_t top = __reduce_max_sync(0xffffffffu, s.key[lane]);
    if (mine == top) atomicMin(&s.first, at);
    __syncthreads();
    int first = s.first;
    if constexpr (kMany) {
        if (tid < ctas) {
            Shared& to = *cluster.map_shared_rank(&s, tid);
            to.peer_key[rank] = top;
            to.peer_first[rank] = first;
        }
        cluster.sync();
        for (int c = 0; c < ctas; ++c) top = max(top, s.peer_key[c]);
        first = 0x7fffffff;
        for (int c = 0; c < ctas; ++c)
            if (s.peer_key[c] == top) first = min(first, s.peer_first[c]);
    }
    const float largest = key_to_float(top);
    if (!(temperature > 0.0f) || largest == -INFINITY) {
        if (tid == 0 && rank == 0) ids[b] = largest == -INFINITY ? 0 : first;
        return;
    }
    Masses m;
    m.s = &s;
    m.set(largest, temperature);
    // The least key, of those of finite logits up to the largest, for which holds(x) is true; it is true from there on
    // (where it is not even true of the largest: one above that).  By a warp, 32 keys at a time.
    auto least = [&](auto&& holds) {
        uint32_t lo = 0x00800000u, hi = top;
        if (!holds(largest)) return top + 1u;
        while (lo < hi) {                                // (true at hi)
            const uint32_t step = (hi - lo) / 32u + 1u, key = lo + (uint32_t)lane * step;
            const unsigned yes = __ballot_sync(0xffffffffu, key >= hi || holds(key_to_float(key)));
            const int f = yes ? __ffs(yes) - 1 : 32;     // (the keys of all lanes lie below hi or hold)
            hi = f < 32 ? min(hi, lo + (uint32_t)f * step) : hi;
            if (f > 0) lo = lo + (uint32_t)(f - 1) * step + 1u;
            if (f == 0) hi = lo;
        }
        return hi;
    };

    uint32_t cut = 0u;                                   // least key that is kept
    bool sums_known = false, alone = !kMany;             // alone: the others have left
    if (cut_p && top_p <= 0.0f && !m.only_largest) cut = top;
    else if ((cut_k || cut_p) && !m.only_largest) {
        // ---- 2. entries per bin ----
        uint32_t far = 0u;                               // (entries of the last bin would all meet in one place)
        walk<T, 4>(row, part_lo, part_hi, tid, kThreads, [&](float x, int) {
            const int bin = m.bin(x);
            if (bin == kBins - 1) ++far;
            else if (bin >= 0) atomicAdd(&s.bins[bin], 1u);
        });
        far = __reduce_add_sync(0xffffffffu, far);
        if (lane == 0 && far) atomicAdd(&s.bins[kBins - 1], far);
        sync_row();
        int count[kPerThread], n = 0;
        float mass = 0.0f;                               // of the thread's bins, by their centres
        const float first_w = exp2f((float)-(tid * kPerThread) * (1.0f / 256.0f));
        auto weight = [&](int i) { return first_w * (float)(1.0 - 0.0027076062 * i + 0.0000036655656 * i * i); };        // 2^(-i/256), i < 8, to 2^-19
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) count[i] = (int)s.bins[tid * kPerThread + i];
        if constexpr (kMany) {
            for (int c = 1; c < ctas; ++c) {
                const uint4* other = reinterpret_cast<const uint4*>(cluster.map_shared_rank(&s, (rank + c) % ctas)->bins + tid * kPerThread);
                const uint4 x = other[0], y = other[1];
                count[0] += x.x; count[1] += x.y; count[2] += x.z; count[3] += x.w;
                count[4] += y.x; count[5] += y.y; count[6] += y.z; count[7] += y.w;
            }
            cluster.sync();                              // (the bins become scratch)
        }
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            n += count[i];
            mass += (float)count[i] * weight(i);
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
        if (tid == kThreads - 1) s.tail = (float)count[kPerThread - 1] * weight(kPerThread - 1);        // (anything down to nothing)
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
                const float w = weight(i);
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
                const float upto = above + (float)count[i] * weight(i);
                if (count[i] > 0 && bin <= bin_k) {
                    const bool stays = upto * (1.0f + kSlack) < lo && bin < kBins - 1, goes = above * (1.0f - kSlack) >= hi;
                    if (!stays && !goes) { atomicMin(&s.zone_lo, bin); atomicMax(&s.zone_hi, bin); }
                }
                above = upto;
            }
        }
        __syncthreads();
        int zone_lo = s.zone_lo, zone_hi = s.zone_hi;
        if (cut_p && zone_lo > zone_hi) { zone_lo = 0; zone_hi = min(bin_k, kBins - 1); }        // (never: a nucleus ends somewhere)
        // thresholds: entries above the zone, of it, before the k-th largest's bin, of it; what min_p leaves
        if (warp < 5) {
            uint32_t key;
            if (warp == 0) key = least([&](float x) { return m.bin(x) < (cut_p ? zone_lo : bin_k); });
            else if (warp == 1) key = least([&](float x) { return m.bin(x) <= zone_hi; });
            else if (warp == 2) key = least([&](float x) { return m.bin(x) < bin_k; });
            else if (warp == 3) key = least([&](float x) { return m.bin(x) <= bin_k; });
            else key = min_p > 0.0f ? min(top, least([&](float x) { return m.get(x) >= (double)min_p; })) : 0u;
            if (lane == 0) (&s.over_key)[warp] = key;
        }
        __syncthreads();
        const uint32_t over_key = s.over_key;
        if (s.min_key < over_key) {                      // (else it lies above both cuts)
        // ---- 3. exact masses ----
        // (one above the largest finite number's key is that of +infinity; what counts as 2^-938 for want of a
        // mass is in no run's sum, or a draw of 0 would end in a run of such entries)
        const float over_x = fmaxf(key_to_float(over_key), m.lowest), zone_x = cut_p ? key_to_float(s.zone_key) : INFINITY, in_x = key_to_float(s.in_key), k_x = key_to_float(s.k_key);
        double in = 0.0, over = 0.0;                     // before the k-th largest's bin; above the zone
        auto put = [&](float x, int i) {
            const int j = atomicAdd(&lead.n_p, 1);
            if (j < kListP) { lead.list_p[j] = {ordered_key(x), i}; lead.mass_p[j] = units(m.get(x)); }
        };
        auto third = [&](auto bounded) {
            walk<T, 1>(row, min(part_lo + warp * run, part_hi), min(part_lo + warp * run + run, part_hi), lane, 32, [&](float x, int i) {
                if (cut_k && !(x >= in_x)) {
                    if (x >= k_x) {                      // of the k-th largest's bin
                        const int j = atomicAdd(&lead.n_k, 1);
                        if (j < kListK) lead.list_k[j] = {ordered_key(x), i};
                        if (x < over_x && x >= zone_x) put(x, i);
                    }
                    return;
                }
                const double mass = m.template get_any<decltype(bounded)::value>(x);
                in += mass;
                if (x >= over_x) over += mass;
                if (x < over_x && x >= zone_x) put(x, i);
            });
        };
        if (m.bounded) third(std::true_type{});
        else third(std::false_type{});
        __syncthreads();
        block_sums(in, over, reinterpret_cast<double*>(s.bins), s.sum, s.runs);
        if (tid < kWarps) lead.all_runs[rank * kWarps + tid] = s.runs[tid];
        if (tid == 0) { lead.sum_in[rank] = s.sum[0]; lead.sum_over[rank] = s.sum[1]; }
        sync_row();
        if (rank != 0) return;
        alone = true;
        double all_in = 0.0, all_over = 0.0;
        for (int c = 0; c < ctas; ++c) { all_in += s.sum_in[c]; all_over += s.sum_over[c]; }
        const int n_k = s.n_k, n_p = s.n_p;
        // The largest key at which the amounts of a list's entries at or above it reach `most` (0: nowhere),
        // among keys from `floor` on: 256 ranges of keys at a time.
        auto search = [&](const Entry* list, int n, uint32_t floor, unsigned long long most, auto&& amount) {
            uint32_t lo = 0xffffffffu, hi = 0u;
            for (int i = tid; i < n; i += kThreads) { lo = min(lo, list[i].key); hi = max(hi, list[i].key); }
            lo = __reduce_min_sync(0xffffffffu, lo);
            hi = __reduce_max_sync(0xffffffffu, hi);
            __syncthreads();
            if (lane == 0) { s.key[warp] = lo; s.count[warp] = (int)hi; }
            __syncthreads();
            lo = max(floor, __reduce_min_sync(0xffffffffu, s.key[lane]));
            hi = __reduce_max_sync(0xffffffffu, (uint32_t)s.count[lane]);
            unsigned long long above = 0;                // at the keys behind hi
            while (lo <= hi) {
                if (tid < 256) { s.range[tid][0] = 0u; s.range[tid][1] = 0u; s.range[tid][2] = 0u; }
                __syncthreads();
                const int bits = 32 - __clz(hi - lo), shift = hi > lo && bits > 8 ? bits - 8 : 0;
                for (int i = tid; i < n; i += kThreads)
                    if (list[i].key >= lo && list[i].key <= hi) add_units(s.range[(list[i].key - lo) >> shift], amount(i));
                __syncthreads();
                if (warp == 0) {                         // lane 0 has the highest eight ranges
                    unsigned long long x[8], sum = above;
                    unsigned long long mine = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) { x[i] = units_of(s.range[255 - 8 * lane - i]); mine += x[i]; }
                    unsigned long long upto = mine;
#pragma unroll
                    for (int o = 1; o < 32; o *= 2) {
                        const unsigned long long y = __shfl_up_sync(0xffffffffu, upto, o);
                        if (lane >= o) upto += y;
                    }
                    sum += upto - mine;
                    int at_range = -1;
                    unsigned long long base = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (at_range < 0 && sum + x[i] >= most) { at_range = 255 - 8 * lane - i; base = sum; }
                        sum += x[i];
                    }
                    const unsigned some = __ballot_sync(0xffffffffu, at_range >= 0);
                    if (some == 0u) { if (lane == 0) { s.open_lo = 1u; s.open_hi = 0u; } }
                    else if (lane == __ffs(some) - 1) {
                        s.open_lo = lo + ((uint32_t)at_range << shift);
                        s.open_hi = min(hi, s.open_lo + ((1u << shift) - 1u));
                        s.open_base = base;
                    }
                }
                __syncthreads();
                lo = s.open_lo; hi = s.open_hi; above = s.open_base;
                if (shift == 0 && lo <= hi) return lo;
                __syncthreads();
            }
            return 0u;
        };
        // The same over the row: amount(x, key) of the keys in lo .. hi, 256 ranges of keys at a time;
        // the largest key at which what is at or above it reaches `most` (in the amount's units).
        auto search_row = [&](uint32_t lo, uint32_t hi, unsigned long long most, auto&& amount) {
            if (tid == 0) { s.open_lo = lo; s.open_hi = hi; s.open_base = 0; }
            for (;;) {
                __syncthreads();
                lo = s.open_lo; hi = s.open_hi;
                if (tid < 256) s.wide_range[tid] = 0;
                __syncthreads();
                const int bits = 32 - __clz(hi - lo), shift = hi > lo && bits > 8 ? bits - 8 : 0;
                walk(row, 0, vocab, tid, kThreads, [&](float x, int) {
                    const uint32_t key = ordered_key(x);
                    if (key < lo || key > hi) return;
                    const unsigned long long a = amount(x);
                    if (a) atomicAdd(&s.wide_range[(key - lo) >> shift], a);
                });
                __syncthreads();
                if (tid == 0) {
                    unsigned long long upto = s.open_base;
                    int i = 255;
                    for (; i >= 0; --i) {
                        if (upto + s.wide_range[i] >= most) break;
                        upto += s.wide_range[i];
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
                cut = search(s.list_k, n_k, 0u, (unsigned long long)s.need, [](int) { return 1ull; });
            } else {
                cut = search_row(0u, 0xffffffffu, (unsigned long long)top_k, [&](float) { return 1ull; });
            }
        }
        if (cut_p) {
            // the whole mass: bins before bin_k and what of that bin stays
            // (whole units below 2^53 of the list: exact in any order)
            double rest = 0.0;
            auto add_rest = [&](float x) { rest += (double)units(m.get(x)); };
            if (bin_k < kBins) {
                if (n_k <= kListK) {
                    for (int i = tid; i < n_k; i += kThreads)
                        if (s.list_k[i].key >= cut) add_rest(key_to_float(s.list_k[i].key));
                } else {
                    walk(row, 0, vocab, tid, kThreads, [&](float x, int) { if (m.bin(x) == bin_k && ordered_key(x) >= cut) add_rest(x); });
                }
            }
            if (bin_k < kBins) {
                __syncthreads();
                block_sums(rest, 0.0, reinterpret_cast<double*>(s.bins), s.sum, s.runs);
                all_in += s.sum[0] / unit;
            }
            // (the least key above which there is less than top_p is the largest one at or above which there is no less)
            const double most = ((double)top_p * all_in - all_over) * unit;
            uint32_t key = top;                          // (never: what is above the zone is less)
            if (most > 0.0) {
                const unsigned long long most_u = (unsigned long long)__double2ll_ru(most);
                if (n_p <= kListP) {
                    // (the list may hold what the top-k cut took)
                    key = search(s.list_p, n_p, cut, most_u, [&](int i) { return s.mass_p[i]; });
                    sums_known = key != 0u;
                } else {
                    key = search_row(max(cut, 1u), top, most_u, [&](float x) {
                        const int bin = m.bin(x);
                        if (bin < zone_lo || bin > zone_hi) return 0ull;
                        return units(m.get(x));
                    });
                }
            }
            cut = max(cut, min(key, top));
        } else {
            sums_known = bin_k >= kBins || n_k <= kListK;
        }
        cut = max(cut, s.min_key);
        if (sums_known) {                                // what is kept of the list, to its runs
            const int n = cut_p ? n_p : bin_k < kBins ? n_k : 0;
            for (int i = tid; i < n; i += kThreads) {
                const Entry e = cut_p ? s.list_p[i] : s.list_k[i];
                if (e.key < cut) continue;
                add_units(s.run_units[e.index / run], cut_p ? s.mass_p[i] : units(m.get(key_to_float(e.key))));
            }
            __syncthreads();
            if (tid < n_runs) s.all_runs[tid] += (double)units_of(s.run_units[tid]) / unit;
            __syncthreads();
        }
        }
        cut = max(cut, s.min_key);
    } else if (min_p > 0.0f && !m.only_largest) {
        if (warp == 0) {
            const uint32_t key = min(top, least([&](float x) { return m.get(x) >= (double)min_p; }));
            if (lane == 0) s.min_key = key;
        }
        __syncthreads();
        cut = s.min_key;
    }
    // ---- 4. the draw ----
    const float cut_x = cut ? key_to_float(cut) : -INFINITY;
    // sum of the entries [lo, hi) by this warp
    auto run_sum = [&](int lo, int hi) {
        double x = 0.0;
        walk<T, 1>(row, lo, hi, lane, 32, [&](float v, int) { if (v >= cut_x) x += m.get(v); });
        return warp_sum(x);
    };
    if (!sums_known) {
        // (a list that did not fit: the first CTA does the others' runs too)
        for (int c = alone ? 0 : rank; c < (alone ? ctas : rank + 1); ++c) {
            const int a = min((c * kWarps + warp) * run, vocab);
            const double sum = run_sum(a, min(a + run, vocab));
            if (lane == 0) lead.all_runs[c * kWarps + warp] = sum;
        }
        if (alone) __syncthreads();
        else sync_row();
        if (rank != 0) return;
    }
    // The run that the sum passes the target in, then the piece of it; the last with a mass where roundings
    // leave none.  (before, target: the first warp's)
    double before = 0.0, target = 0.0;
    int lo, hi;
    if (warp == 0) {
        double mine = 0.0;
        for (int c = 0; c < ctas; ++c) mine += s.all_runs[lane * ctas + c];
        double upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const double x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        target = (double)u * __shfl_sync(0xffffffffu, upto, 31);
        const unsigned passes = __ballot_sync(0xffffffffu, mine > 0.0 && upto > target), holds = __ballot_sync(0xffffffffu, mine > 0.0);
        const int w = passes ? __ffs(passes) - 1 : max(31 - __clz(holds), 0);        // (never nothing: the largest is kept)
        double at_run = __shfl_sync(0xffffffffu, upto - mine, w);
        int pick = w * ctas;
        for (int c = 0; c < ctas; ++c) {                 // (all lanes the same)
            const double x = s.all_runs[w * ctas + c];
            if (!(x > 0.0)) continue;
            pick = w * ctas + c;
            before = at_run;
            if (at_run + x > target) break;
            at_run += x;
        }
        if (lane == 0) s.draw_run = pick;
    }
    __syncthreads();
    lo = min(s.draw_run * run, vocab);
    hi = min(lo + run, vocab);
    {
        const int per = (hi - lo + kWarps - 1) / kWarps;
        const int a = min(lo + warp * per, hi), z = min(a + per, hi);
        const double sum = run_sum(a, z);
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
            const unsigned passes = __ballot_sync(0xffffffffu, some && before + upto > target), holds = __ballot_sync(0xffffffffu, some);
            const int w = passes ? __ffs(passes) - 1 : max(31 - __clz(holds), 0);
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
            const float x = i < hi ? (float)row[i] : -INFINITY;
            double upto = x >= cut_x ? m.get(x) : 0.0;
            const bool stays = upto > 0.0;
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
        if (lane == 0) ids[b] = pick >= 0 ? pick : max(last, 0);
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
    // As many CTAs to a row as the GPU has to spare, each with its share of entries.
    int ctas = 1;
    while (ctas < kMaxCtas && (int64_t)batch * ctas * 2 <= num_sms() && vocab / (ctas * 2) >= kLeast) ctas *= 2;
    auto go = [&](auto* kernel, auto* x) {
        KIVI_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared)));
        KIVI_CUDA_OK(launch_cluster(kernel, ctas > 1 ? ctas : 0, dim3((unsigned)batch * (unsigned)ctas), kThreads, sizeof(Shared), (cudaStream_t)stream, true, x, vocab, row_stride, f, ids_out));
        note_launches(1);
        return KIVI_OK;
    };
    auto of = [&](auto many) {
        constexpr bool kMany = decltype(many)::value;
        return dtype == KIVI_BF16 ? go(sample_filtered_kernel<__nv_bfloat16, kMany>, reinterpret_cast<const __nv_bfloat16*>(logits))
                                  : go(sample_filtered_kernel<float, kMany>, reinterpret_cast<const float*>(logits));
    };
    return ctas > 1 ? of(std::true_type{}) : of(std::false_type{});
}
