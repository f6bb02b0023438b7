// Penalties for tokens that a row has had, biases and masks on its logits.
//
//   x = had ? (x > 0 ? x / r : x r) : x,   x -= f * times said,   x -= p if said,
//   x += bias,   x = -inf where the mask has no bit
//
// A CTA takes a stretch of a row that its threads hold in registers, 16-byte vectors on the
// row's own grid (rows of 50257 numbers start anywhere).  What the row has had is counted
// in shared memory, a word for each entry of the stretch: every CTA of a row reads all of
// the row's list and keeps what falls into its stretch.  Counts are whole numbers and the
// last bias is found by its place, so the order in which threads come changes nothing.
//
// Bound by memory for many rows, by latency for one: bounds of the lists, tokens, counts,
// one after the other, with the logits on their way meanwhile.  Long stretches read the lists
// less often, short ones give one row to more SMs (stretch_threads).
#include "kivi_common.cuh"

namespace kivi {
namespace {

__device__ int g_fault = 0;
constexpr int kListFault = 4;                            // bit of the device fault word: arrays that contradict each other
constexpr int kVectors = 4;                              // of a thread

struct LogitArgs {
    const void* in;
    void* out;
    int batch, vocab;
    int64_t in_stride, out_stride;
    kivi_logit_rules r;
};

template <typename T> struct Pack;
template <> struct Pack<float> {
    static constexpr int N = 4;
    __device__ static void load(const float* p, float (&x)[4]) { const float4 v = *reinterpret_cast<const float4*>(p); x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w; }
    __device__ static void store(float* p, const float (&x)[4]) { *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]); }
};
template <> struct Pack<__nv_bfloat16> {
    static constexpr int N = 8;
    __device__ static void load(const __nv_bfloat16* p, float (&x)[8]) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
    __device__ static void store(__nv_bfloat16* p, const float (&x)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 t = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&t);
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
};
__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// the part of a list that is a row's; bounds that the array does not have: nothing
__device__ __forceinline__ int2 list_of(const int32_t* cu, int row, int total) {
    const int lo = cu[row], hi = cu[row + 1];
    if (lo < 0 || hi < lo || hi > total) {
        if (threadIdx.x == 0 && blockIdx.x == 0) atomicOr(&g_fault, kListFault);
        return make_int2(0, 0);
    }
    return make_int2(lo, hi);
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS)
adjust_logits_kernel(LogitArgs A) {
    constexpr int N = Pack<T>::N, kEntries = THREADS * kVectors * N;
    extern __shared__ __align__(16) uint32_t word_s[];   // [kEntries]
    stream_order();
    const kivi_logit_rules& r = A.r;
    const int row = blockIdx.y, tid = threadIdx.x;
    const T* const in = settled(reinterpret_cast<const T*>(A.in)) + (int64_t)row * A.in_stride;
    T* const out = reinterpret_cast<T*>(A.out) + (int64_t)row * A.out_stride;
    // entry `first` is the stretch's first; vectors lie on 16-byte boundaries of the row
    const int before = (int)(reinterpret_cast<uintptr_t>(in) / sizeof(T)) & (N - 1);
    const int64_t first = (int64_t)blockIdx.x * kEntries - before;
    if (first >= A.vocab) return;
    const bool apart = ((reinterpret_cast<uintptr_t>(out) / sizeof(T)) & (N - 1)) != (unsigned)before;        // (out's vectors lie elsewhere)
    float x[kVectors][N];
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
        const int64_t i = first + (v * THREADS + tid) * N;
        if (i >= 0 && i + N <= A.vocab) Pack<T>::load(in + i, x[v]);
        else {
#pragma unroll
            for (int e = 0; e < N; ++e) x[v][e] = i + e >= 0 && i + e < A.vocab ? as_float(in[i + e]) : 0.0f;
        }
    }
    auto clear = [&] {
#pragma unroll
        for (int i = 0; i < kEntries; i += 4 * THREADS) *reinterpret_cast<uint4*>(word_s + i + 4 * tid) = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
    };
    // a list's ids that lie in the stretch
    auto scan = [&](const int64_t* ids, int2 list, auto&& take) {
        for (int i0 = list.x; i0 < list.y; i0 += 4 * THREADS) {
            int64_t id[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) { const int i = i0 + u * THREADS + tid; id[u] = i < list.y && i >= i0 ? ids[i] : -1; }
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (id[u] >= 0 && id[u] < A.vocab && id[u] >= first && id[u] < first + kEntries) take((int)(id[u] - first), i0 + u * THREADS + tid);
        }
        __syncthreads();
    };
    auto each = [&](auto&& f) {
#pragma unroll
        for (int v = 0; v < kVectors; ++v)
#pragma unroll
            for (int e = 0; e < N; e += 4) {
                const uint4 w = *reinterpret_cast<const uint4*>(word_s + (v * THREADS + tid) * N + e);
                if ((w.x | w.y | w.z | w.w) == 0u) continue;
                if (w.x) f(x[v][e], w.x);
                if (w.y) f(x[v][e + 1], w.y);
                if (w.z) f(x[v][e + 2], w.z);
                if (w.w) f(x[v][e + 3], w.w);
            }
    };
    if (r.tokens != nullptr) {
        const int2 list = list_of(settled(r.cu_tokens), row, r.num_tokens);
        const int given = r.prompt_lens ? max(0, settled(r.prompt_lens)[row]) : 0;
        const float rep = r.repetition ? settled(r.repetition)[row] : 1.0f, freq = r.frequency ? settled(r.frequency)[row] : 0.0f, pres = r.presence ? settled(r.presence)[row] : 0.0f;
        clear();
        scan(settled(r.tokens), list, [&](int at, int i) {
            if (i - list.x < given) atomicOr(word_s + at, 0x80000000u);
            else atomicAdd(word_s + at, 1u);
        });
        each([&](float& y, uint32_t w) {
            if (rep != 1.0f) y = y > 0.0f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
            const uint32_t said = w & 0x7fffffffu;
            if (said) y = __fsub_rn(__fsub_rn(y, __fmul_rn(freq, (float)said)), pres);
        });
    }
    if (r.bias_ids != nullptr) {
        const int2 list = list_of(settled(r.cu_bias), row, r.num_bias);
        const float* const bias = settled(r.bias);
        __syncthreads();                                 // (the counts have been read)
        clear();
        scan(settled(r.bias_ids), list, [&](int at, int i) { atomicMax(word_s + at, (uint32_t)i + 1u); });
        each([&](float& y, uint32_t w) { y = __fadd_rn(y, bias[w - 1u]); });
    }
    if (r.allowed != nullptr) {
        int m = r.allowed_rows ? settled(r.allowed_rows)[row] : row;
        if (m >= r.num_masks) {
            if (tid == 0 && blockIdx.x == 0) atomicOr(&g_fault, kListFault);
            m = -1;
        }
        if (m >= 0) {
            const uint32_t* const mask = reinterpret_cast<const uint32_t*>(settled(r.allowed)) + m * r.mask_stride;
            const int last_word = (A.vocab - 1) >> 5;
#pragma unroll
            for (int v = 0; v < kVectors; ++v) {
                const int64_t i = first + (v * THREADS + tid) * N;
                if (i + N <= 0 || i >= A.vocab) continue;
                const int w = (int)(i >> 5);             // (a vector that begins before the row: word -1, which is not read)
                const uint32_t lo = w >= 0 ? mask[w] : 0u, hi = ((i + N - 1) >> 5) > w && w < last_word ? mask[w + 1] : 0u;
                const uint32_t bits = __funnelshift_r(lo, hi, (uint32_t)(i & 31));
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (!((bits >> e) & 1u)) x[v][e] = -INFINITY;
            }
        }
    }
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
        const int64_t i = first + (v * THREADS + tid) * N;
        if (!apart && i >= 0 && i + N <= A.vocab) Pack<T>::store(out + i, x[v]);
        else {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (i + e >= 0 && i + e < A.vocab) put(out + i + e, x[v][e]);
        }
    }
}

template <typename T, int THREADS>
int run_adjust(const LogitArgs& a, cudaStream_t st) {
    constexpr int kEntries = THREADS * kVectors * Pack<T>::N, kSmem = kEntries * 4;
    auto* const kernel = adjust_logits_kernel<T, THREADS>;
    if (kSmem > 48 * 1024) KIVI_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    const int64_t stretches = ((int64_t)a.vocab + Pack<T>::N - 1 + kEntries - 1) / kEntries;          // (a row may begin N - 1 entries into its first vector)
    const bool lists = a.r.tokens != nullptr || a.r.bias_ids != nullptr;
    KIVI_CUDA_OK(launch(kernel, dim3((unsigned)stretches, (unsigned)a.batch), THREADS, lists ? kSmem : 0, st, true, a));
    return KIVI_OK;
}

// Threads of a CTA: as many as still leave two CTAs to an SM.
template <typename T> int stretch_threads(const LogitArgs& a) {
    int threads = 512;
    while (threads > 128 && (int64_t)a.batch * ((a.vocab + threads * kVectors * Pack<T>::N - 1) / (threads * kVectors * Pack<T>::N)) < 2 * num_sms()) threads /= 2;
    return threads;
}
template <typename T> int adjust(const LogitArgs& a, cudaStream_t st) {
    const int threads = stretch_threads<T>(a);
    return threads == 512 ? run_adjust<T, 512>(a, st) : threads == 256 ? run_adjust<T, 256>(a, st) : run_adjust<T, 128>(a, st);
}

}  // namespace

int logit_rules_fault_word(int* out) {
    KIVI_CUDA_OK(cudaMemcpyFromSymbol(out, g_fault, sizeof(int)));
    return KIVI_OK;
}
int logit_rules_fault_clear() {
    const int zero = 0;
    KIVI_CUDA_OK(cudaMemcpyToSymbol(g_fault, &zero, sizeof(int)));
    return KIVI_OK;
}

}  // namespace kivi

using namespace kivi;

extern "C" int kivi_adjust_logits(const void* logits, int dtype, int batch, int vocab, int64_t row_stride, const kivi_logit_rules* rules,
                                  void* out, int64_t out_stride, void* stream) {
    KIVI_REQUIRE(dtype == KIVI_F32 || dtype == KIVI_BF16, "dtype must be KIVI_F32 or KIVI_BF16");
    KIVI_REQUIRE(batch >= 0 && batch <= 65535, "batch (%d) outside 0..65535", batch);
    KIVI_REQUIRE(vocab > 0 && vocab <= 0x7fff0000, "vocab (%d) outside 1..2^31-2^16", vocab);
    KIVI_REQUIRE(rules != nullptr, "rules is null");
    if (batch == 0) { note_launches(0); return KIVI_OK; }
    KIVI_REQUIRE(logits != nullptr && out != nullptr, "logits or out is null");
    KIVI_REQUIRE(reinterpret_cast<uintptr_t>(logits) % elem_size(dtype) == 0 && reinterpret_cast<uintptr_t>(out) % elem_size(dtype) == 0, "logits or out is not on its type's boundary");
    KIVI_REQUIRE(batch == 1 || row_stride == 0 || row_stride >= vocab, "rows of logits overlap");
    KIVI_REQUIRE(batch == 1 || out_stride >= vocab, "rows of out overlap");
    KIVI_REQUIRE(out != logits || batch == 1 || row_stride == out_stride, "out starts where logits does but is laid out differently");
    KIVI_REQUIRE(rules->tokens == nullptr || (rules->cu_tokens != nullptr && rules->num_tokens >= 0), "tokens need cu_tokens");
    KIVI_REQUIRE(rules->tokens != nullptr || (!rules->prompt_lens && !rules->repetition && !rules->frequency && !rules->presence), "penalties need tokens");
    KIVI_REQUIRE(rules->bias_ids == nullptr || (rules->bias != nullptr && rules->cu_bias != nullptr && rules->num_bias >= 0), "bias_ids need bias and cu_bias");
    KIVI_REQUIRE(rules->allowed != nullptr || rules->allowed_rows == nullptr, "allowed_rows need allowed");
    if (rules->allowed != nullptr) {
        KIVI_REQUIRE(rules->mask_stride >= ((int64_t)vocab + 31) / 32, "a mask of %lld words does not hold %d bits", (long long)rules->mask_stride, vocab);
        KIVI_REQUIRE(rules->num_masks >= 1, "allowed holds no mask");
        KIVI_REQUIRE(rules->allowed_rows != nullptr || rules->num_masks >= batch, "allowed holds %d masks for %d rows", rules->num_masks, batch);
    }
    LogitArgs a{logits, out, batch, vocab, row_stride, out_stride, *rules};
    if (int rc = dtype == KIVI_BF16 ? adjust<__nv_bfloat16>(a, (cudaStream_t)stream) : adjust<float>(a, (cudaStream_t)stream)) return rc;
    note_launches(1);
    return KIVI_OK;
}
