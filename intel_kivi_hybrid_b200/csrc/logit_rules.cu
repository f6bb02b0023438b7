// Penalties for tokens that a row has had, biases and masks on its logits.
//
//   x = had ? (x > 0 ? x / r : x r) : x,   x -= f * times said,   x -= p if said,
//   x += bias,   x = -inf where the mask has no bit
//
// A CTA takes a stretch of a row, 16-byte vectors on the row's own grid (rows of 50257 numbers
// start anywhere): copies it to `out`, with -inf where the mask says so, and then writes the
// entries that a list speaks of once more.  What the row has had is counted in shared memory, 16 bits
// for each entry of the stretch, and 16 for the last bias's place in its list: every CTA of a row reads all of
// the row's lists and keeps what falls into its stretch.  Rows with longer lists have 32 bits, for
// half of the stretch at a time.  Of an entry's several mentions the first that comes writes it, all the same number,
// and of several biases the last: counts are whole numbers, so the order in which threads come changes nothing.
//
// Bound by memory without lists, by latency with them: bounds of the lists, ids, counts, ids again, logits, one
// after the other, so that what counts is how many CTAs an SM holds.  128 x 130000 bf16 with lists of 2100 and of 150:
// 66 us with the stretch in registers and every word looked over, 55 with words of 32 bits, 64 with the lists shared
// out over a cluster that counts in each other's shared memory.
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

template <typename T> constexpr int kPack = 16 / sizeof(T);              // numbers of a vector
__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
// a vector's numbers without a bit become -inf
template <typename T> __device__ __forceinline__ uint4 masked(uint4 v, uint32_t bits) {
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            if (!(bits >> i & 1u)) w[i] = 0xff800000u;
        } else {
            if (!(bits >> (2 * i) & 1u)) w[i] = (w[i] & 0xffff0000u) | 0xff80u;
            if (!(bits >> (2 * i + 1) & 1u)) w[i] = (w[i] & 0xffffu) | 0xff800000u;
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// the part of a list that is a row's; bounds that the array does not have: nothing
__device__ __forceinline__ int2 list_of(const int32_t* cu, int row, int total) {
    const int lo = cu[row], hi = cu[row + 1];
    if (lo < 0 || hi < lo || hi > total) {
        if (threadIdx.x == 0 && blockIdx.x == 0) atomicOr(&g_fault, kListFault);
        return make_int2(0, 0);
    }
    return make_int2(lo, hi);
}

// Counters of 16 or 32 bits.
struct Counters {
    uint8_t* at;
    bool wide;
    __device__ uint32_t given() const { return wide ? 0x80000000u : 0x8000u; }   // had in the prompt
    __device__ uint32_t taken() const { return wide ? 0x40000000u : 0x4000u; }   // written; below: times said
    __device__ uint32_t get(int i) const { return wide ? reinterpret_cast<const uint32_t*>(at)[i] : reinterpret_cast<const uint16_t*>(at)[i]; }
    __device__ uint32_t put(int i, uint32_t bits, bool add) const {              // what was there before
        uint32_t* const word = reinterpret_cast<uint32_t*>(at) + (wide ? i : i >> 1);
        const int shift = wide ? 0 : 16 * (i & 1);
        const uint32_t was = (add ? atomicAdd(word, bits << shift) : atomicOr(word, bits << shift)) >> shift;
        return wide ? was : was & 0xffffu;
    }
    __device__ void most(int i, uint32_t place) const {
        if (wide) { atomicMax(reinterpret_cast<uint32_t*>(at) + i, place); return; }
        unsigned short* const half = reinterpret_cast<unsigned short*>(at) + i;
        unsigned short was = *half;
        while (was < place) {
            const unsigned short now = atomicCAS(half, was, (unsigned short)place);
            if (now == was) break;
            was = now;
        }
    }
};
constexpr int kNarrowTokens = 0x3fff, kNarrowBiases = 0xfffe;

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1536 / THREADS)
adjust_logits_kernel(LogitArgs A) {
    constexpr int N = kPack<T>, kEntries = THREADS * kVectors * N;
    extern __shared__ __align__(16) uint8_t counters[];  // 2 * kEntries bytes where there are tokens, then as many where there are biases
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
    const bool tokens = r.tokens != nullptr, biases = r.bias_ids != nullptr, copies = out != in || r.allowed != nullptr;
    uint4 x[kVectors];
    if (copies)
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            const int64_t i = first + (v * THREADS + tid) * N;
            x[v] = i >= 0 && i + N <= A.vocab ? *reinterpret_cast<const uint4*>(in + i) : make_uint4(0u, 0u, 0u, 0u);
        }
    const int2 said = tokens ? list_of(settled(r.cu_tokens), row, r.num_tokens) : make_int2(0, 0), given = biases ? list_of(settled(r.cu_bias), row, r.num_bias) : make_int2(0, 0);
    int m = -1;
    if (r.allowed != nullptr) {
        m = r.allowed_rows ? settled(r.allowed_rows)[row] : row;
        if (m >= r.num_masks) {
            if (tid == 0 && blockIdx.x == 0) atomicOr(&g_fault, kListFault);
            m = -1;
        }
    }
    const uint32_t* const mask = m >= 0 ? reinterpret_cast<const uint32_t*>(settled(r.allowed)) + m * r.mask_stride : nullptr;
    const int prompt = tokens && r.prompt_lens ? max(0, settled(r.prompt_lens)[row]) : 0;
    const float rep = tokens && r.repetition ? settled(r.repetition)[row] : 1.0f, freq = tokens && r.frequency ? settled(r.frequency)[row] : 0.0f,
                pres = tokens && r.presence ? settled(r.presence)[row] : 0.0f;
    const float* const bias = settled(r.bias);
    auto copy = [&] {
#pragma unroll
        for (int v = 0; v < kVectors; ++v) {
            const int64_t i = first + (v * THREADS + tid) * N;
            if (i + N <= 0 || i >= A.vocab) continue;
            uint32_t bits = 0xffffffffu;
            if (mask != nullptr) {
                const int w = (int)(i >> 5);             // (a vector that begins before the row: word -1, which is not read)
                const uint32_t lo = w >= 0 ? mask[w] : 0u, hi = ((i + N - 1) >> 5) > w && w < (A.vocab - 1) >> 5 ? mask[w + 1] : 0u;
                bits = __funnelshift_r(lo, hi, (uint32_t)(i & 31));
            }
            if (i >= 0 && i + N <= A.vocab) {
                const uint4 y = masked<T>(x[v], bits);
                if (!apart) *reinterpret_cast<uint4*>(out + i) = y;
                else {
#pragma unroll
                    for (int e = 0; e < N; ++e) out[i + e] = reinterpret_cast<const T*>(&y)[e];
                }
            } else {
                for (int e = 0; e < N; ++e)
                    if (i + e >= 0 && i + e < A.vocab) {
                        if (bits >> e & 1u) out[i + e] = in[i + e];
                        else put(out + i + e, -INFINITY);
                    }
            }
        }
    };
    if (!tokens && !biases) {                            // (in place and without a mask there is nothing to do, and nothing has been loaded)
        if (copies) copy();
        return;
    }
    const bool wide = said.y - said.x > kNarrowTokens || given.y - given.x > kNarrowBiases;
    const int part = wide ? kEntries / 2 : kEntries;
    const Counters had{counters, wide}, last{counters + (tokens ? 2 * kEntries : 0), wide};
    {
#pragma unroll 1
        for (int64_t from = first; from < first + kEntries && from < A.vocab; from += part) {
            // a list's ids that lie in the part
            auto scan = [&](const int64_t* ids, int2 list, auto&& take) {
                for (int64_t i0 = list.x; i0 < list.y; i0 += 4 * THREADS) {
                    int64_t id[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) { const int64_t i = i0 + u * THREADS + tid; id[u] = i < list.y ? ids[i] : -1; }
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        if (id[u] >= 0 && id[u] < A.vocab && id[u] >= from && id[u] < from + part) take(id[u], (int)(i0 + u * THREADS) + tid);
                }
            };
            if (from != first) __syncthreads();
            for (int i = 16 * tid; i < (tokens + biases) * 2 * kEntries; i += 16 * THREADS) *reinterpret_cast<uint4*>(counters + i) = make_uint4(0u, 0u, 0u, 0u);
            __syncthreads();
            scan(settled(r.tokens), said, [&](int64_t id, int i) {
                const bool was_given = i - said.x < prompt;
                had.put((int)(id - from), was_given ? had.given() : 1u, !was_given);
            });
            scan(settled(r.bias_ids), given, [&](int64_t id, int i) { last.most((int)(id - from), (uint32_t)(i - given.x) + 1u); });
            if (copies && from == first) copy();
            __syncthreads();
            auto write = [&](int64_t id, uint32_t word, uint32_t place) {
                if (mask != nullptr && !(mask[id >> 5] >> (id & 31) & 1u)) return;
                float y = as_float(in[id]);
                if (word) {
                    if (rep != 1.0f) y = y > 0.0f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
                    const uint32_t n = word & (had.taken() - 1u);
                    if (n) y = __fsub_rn(__fsub_rn(y, __fmul_rn(freq, (float)n)), pres);
                }
                if (place) y = __fadd_rn(y, bias[given.x + (int)place - 1]);
                put(out + id, y);
            };
            scan(settled(r.tokens), said, [&](int64_t id, int) {
                const uint32_t word = had.put((int)(id - from), had.taken(), false);
                if (!(word & had.taken())) write(id, word, biases ? last.get((int)(id - from)) : 0u);
            });
            scan(settled(r.bias_ids), given, [&](int64_t id, int i) {
                const uint32_t place = (uint32_t)(i - given.x) + 1u;
                if (last.get((int)(id - from)) == place && (!tokens || had.get((int)(id - from)) == 0u)) write(id, 0u, place);
            });
        }
    }
}

template <typename T, int THREADS>
int run_adjust(const LogitArgs& a, cudaStream_t st) {
    constexpr int kEntries = THREADS * kVectors * kPack<T>, kMostSmem = kEntries * 4;
    auto* const kernel = adjust_logits_kernel<T, THREADS>;
    if (kMostSmem > 48 * 1024) KIVI_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem));
    const int64_t stretches = ((int64_t)a.vocab + kPack<T> - 1 + kEntries - 1) / kEntries;          // (a row may begin N - 1 entries into its first vector)
    const int lists = (a.r.tokens != nullptr) + (a.r.bias_ids != nullptr);
    KIVI_CUDA_OK(launch(kernel, dim3((unsigned)stretches, (unsigned)a.batch), THREADS, (size_t)lists * 2 * kEntries, st, true, a));
    return KIVI_OK;
}

// Threads of a CTA: 512 where that leaves two CTAs to an SM, else 128.
template <typename T> int adjust(const LogitArgs& a, cudaStream_t st) {
    constexpr int kEntries = 512 * kVectors * kPack<T>;
    return (int64_t)a.batch * ((a.vocab + kEntries - 1) / kEntries) >= 2 * num_sms() ? run_adjust<T, 512>(a, st) : run_adjust<T, 128>(a, st);
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
    KIVI_REQUIRE(rules->num_tokens < (1 << 30), "tokens holds %d ids, 2^30 or more", rules->num_tokens);
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
