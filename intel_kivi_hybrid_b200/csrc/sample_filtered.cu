// Next-token choice under temperature, top-k, top-p and min-p of each row, from given
// random numbers.
//
// m_i = exp((x_i - max) / temperature) needs no normalisation: every cut compares masses
// with masses.  The k-th largest logit is found by bisection on the bits of an
// order-preserving integer (counts), the nucleus likewise (fp64 sums of the masses above a
// candidate), and the draw walks the kept masses in index order.  No sum goes through
// atomics, so the same inputs give the same id.
#include "kivi_common.cuh"

namespace kivi {
namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32;

// order-preserving map float -> uint32; NaN counts as -inf
__device__ __forceinline__ uint32_t ordered_key(float x) {
    if (x != x) x = -INFINITY;
    const uint32_t b = __float_as_uint(x);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

template <typename T> __device__ __forceinline__ float entry(const T* row, int i) { return (float)row[i]; }

__device__ __forceinline__ double block_sum(double x, double* s) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = x;
    __syncthreads();
    double sum = 0.0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += s[w];
    return sum;
}
__device__ __forceinline__ int block_count(int x, int* s) {
    x = __reduce_add_sync(0xffffffffu, x);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = x;
    __syncthreads();
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += s[w];
    return sum;
}

struct FilterArgs {
    const float *uniforms, *temperature, *top_p, *min_p;
    const int32_t* top_k;
};

template <typename T>
__global__ void __launch_bounds__(kThreads)
sample_filtered_kernel(const T* logits, int vocab, int64_t row_stride, FilterArgs f, int64_t* __restrict__ ids) {
    __shared__ double sum_s[kWarps];
    __shared__ int int_s[kWarps];
    __shared__ uint32_t key_s[kWarps];
    __shared__ int pick_s;
    stream_order();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.x;
    const T* const row = settled(logits) + (int64_t)b * row_stride;
    const float u = settled(f.uniforms)[b], temperature = f.temperature ? settled(f.temperature)[b] : 1.0f;
    const float top_p = f.top_p ? settled(f.top_p)[b] : 1.0f, min_p = f.min_p ? settled(f.min_p)[b] : 0.0f;
    const int top_k = f.top_k ? settled(f.top_k)[b] : 0;
    if (tid == 0) pick_s = 0x7fffffff;

    // the largest and its first index
    uint32_t best = 0u;
    int at = 0x7fffffff;
    for (int64_t i = tid; i < vocab; i += kThreads) {
        const uint32_t k = ordered_key(entry(row, (int)i));
        if (k > best) { best = k; at = (int)i; }
    }
    const uint32_t warp_best = __reduce_max_sync(0xffffffffu, best);
    if (lane == 0) key_s[warp] = warp_best;
    __syncthreads();
    uint32_t top = 0u;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = max(top, key_s[w]);
    if (best == top) atomicMin(&pick_s, at);
    __syncthreads();
    const int first = pick_s;
    const float largest = __uint_as_float((top & 0x80000000u) ? (top & 0x7fffffffu) : ~top);
    if (!(temperature > 0.0f) || largest == -INFINITY) {
        if (tid == 0) ids[b] = largest == -INFINITY ? 0 : first;
        return;
    }
    auto mass = [&](float x) {
        if (x == largest) return 1.0;
        if (!(x > -INFINITY) || largest == INFINITY) return 0.0;
        return exp(((double)x - (double)largest) / (double)temperature);
    };

    uint32_t cut = 0u;                                   // least key that is kept
    if (top_k > 0 && top_k < vocab) {
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t probe = cut | (1u << bit);
            int n = 0;
            for (int64_t i = tid; i < vocab; i += kThreads) n += ordered_key(entry(row, (int)i)) >= probe;
            if (block_count(n, int_s) >= top_k) cut = probe;
        }
    }
    if (top_p < 1.0f) {
        auto above = [&](uint32_t key, bool equal) {     // mass of the entries above a key
            double sum = 0.0;
            for (int64_t i = tid; i < vocab; i += kThreads) {
                const float x = entry(row, (int)i);
                const uint32_t k = ordered_key(x);
                if (k > key || (equal && k == key)) sum += mass(x);
            }
            return block_sum(sum, sum_s);
        };
        const double most = (double)top_p * above(cut, true);
        uint32_t c = 0u;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t probe = c + ((1u << bit) - 1u);
            if (!(above(probe, false) < most)) c += 1u << bit;
        }
        cut = max(cut, min(c, top));
    }
    auto kept = [&](float x) {
        const double m = ordered_key(x) >= cut ? mass(x) : 0.0;
        return m >= (double)min_p || x == largest ? m : 0.0;
    };
    // the draw: a thread sums a run of neighbouring entries
    const int64_t per = ((int64_t)vocab + kThreads - 1) / kThreads, lo = tid * per, hi = lo + per < vocab ? lo + per : vocab;
    double mine = 0.0;
    for (int64_t i = lo; i < hi; ++i) mine += kept(entry(row, (int)i));
    double upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const double x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    __syncthreads();
    if (lane == 31) sum_s[warp] = upto;
    if (tid == 0) { pick_s = 0x7fffffff; int_s[0] = -1; }
    __syncthreads();
    double before = 0.0, all = 0.0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) { if (w < warp) before += sum_s[w]; all += sum_s[w]; }
    const double target = (double)u * all;
    before += upto - mine;
    if (mine > 0.0) {
        double sum = before;
        int last = -1;
        for (int64_t i = lo; i < hi; ++i) {
            const double m = kept(entry(row, (int)i));
            if (m > 0.0) last = (int)i;
            sum += m;
            if (m > 0.0 && sum > target) { atomicMin(&pick_s, (int)i); break; }
        }
        atomicMax(&int_s[0], last);                      // (a number that is no less than one takes the last kept entry)
    }
    __syncthreads();
    if (tid == 0) ids[b] = pick_s != 0x7fffffff ? pick_s : int_s[0];
}

}  // namespace
}  // namespace kivi

using namespace kivi;

extern "C" int kivi_sample_filtered(const void* logits, int dtype, int batch, int vocab, int64_t row_stride,
                                    const float* uniforms, const float* temperature, const int32_t* top_k,
                                    const float* top_p, const float* min_p, int64_t* ids_out, void* stream) {
    KIVI_REQUIRE(logits != nullptr && uniforms != nullptr && ids_out != nullptr, "logits, uniforms or ids_out is null");
    KIVI_REQUIRE(dtype == KIVI_F32 || dtype == KIVI_BF16, "logits dtype must be KIVI_F32 or KIVI_BF16");
    KIVI_REQUIRE(batch > 0 && vocab > 0 && row_stride >= vocab, "batch (%d), vocab (%d) and row_stride must be positive, row_stride >= vocab", batch, vocab);
    const FilterArgs f{uniforms, temperature, top_p, min_p, top_k};
    if (dtype == KIVI_BF16)
        KIVI_CUDA_OK(launch(sample_filtered_kernel<__nv_bfloat16>, dim3((unsigned)batch), kThreads, 0, (cudaStream_t)stream, true,
                            reinterpret_cast<const __nv_bfloat16*>(logits), vocab, row_stride, f, ids_out));
    else
        KIVI_CUDA_OK(launch(sample_filtered_kernel<float>, dim3((unsigned)batch), kThreads, 0, (cudaStream_t)stream, true,
                            reinterpret_cast<const float*>(logits), vocab, row_stride, f, ids_out));
    note_launches(1);
    return KIVI_OK;
}
