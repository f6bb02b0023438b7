// Fused decode attention over the packed KIVI cache: tensor-core kernel for
// head_dim 128, group_size 32, up to 8 query heads per KV head in blocks of
// four per CTA (sm_100a).
//
// Decode attention over 2-bit codes is instruction-bound before it is HBM-bound:
// one quantized (token, kv_head) is 128 bytes of HBM but 256 codes that each
// feed 4 query heads.  The GQA query-group tile therefore runs on the tensor
// cores (mma.sync m16n8k32, bytes in, exact 32-bit integer sums) with the codes as
// one operand, and everything that depends on scales and zeros is folded into the
// small operand, a fixed-point number cut into bytes:
//
//   q.k   score[t,h] = sum_d (q[h,d]*s[g,d]) * c[d,t]  +  sum_d q[h,d]*z[g,d]
//         A = codes of 16 tokens x 32 channels; a byte of four codes is an operand as
//         it lies, and so is what three masks leave of it (below); B = q*s in 22 bits
//         and a sign of the largest of the group and head, three bytes and a constant (16
//         columns = 4 heads x 4 bytes); the zero term is an fp32 dot product.
//   p.v   out[h,d]   = sum_t (p[h,t]*s[t,gd]) * c[t,d]  +  sum_t p[h,t]*z[t,gd]
//         A = codes of 16 channels x 32 tokens, same encoding; B = p*s in 16 bits of
//         the largest of the stage's tokens, of the same head and channel group (8 columns =
//         4 heads x 2 bytes); the zero term accumulates in fp32.
//   What shares a largest value ends in the same sums: scores of one group, outputs of one
//   channel group.  One for the whole stage cost those beside a louder neighbour their bits
//   (channel groups 32 times apart: 2.9e-3 of the quiet one's largest output, now 1e-4).
//   Two to four times as many warp reductions for that: 64 units x 32k 57.1 -> 60.5 us, 128 x 4k
//   21.8 -> 22.2, one head 32 x 8k 11.7 -> 11.9.
//   Infinities, NaN and negative value scales take an fp32 form of their own.
//
// Bytes instead of fp16 (codes as subnormals, q*s in two parts): 16 codes cost three
// ALU operations instead of nine, and every MMA contracts twice as many.  512 units x
// 32k tokens at boost clocks 416 -> 368 us (5.9 TB/s, 0.90 of a plain copy), under the power
// cap 484 -> 435 (0.76); 32 x 128k 129 -> 117, 128 x 4k 25.1 -> 23.7, and the error against the
// fp32 kernel falls to a seventh.  A group of 32 tokens takes about 510 instructions of a
// warp, 24 of them MMAs.
//
// Data movement: every warp streams its own token groups from HBM into a
// private shared-memory ring with bulk asynchronous copies (cp.async.bulk,
// completion on an mbarrier), two groups (8 KB) per stage, and masks codes in
// registers.  The small operands are made where their scales are read without
// repetition (a lane takes four channels, or one token, for all four heads) and
// travel through 2 KB of shared memory per warp to where the MMA wants them
// (ldmatrix with byte transposition).  Nothing dequantized is ever written anywhere.
// The residual ring (full precision) is handled by extra CTAs with fp32 FMAs.
//
// Every wait on an mbarrier is bounded; on expiry the warp raises the device
// fault word, stops consuming and its partial is written as "empty".
#include "attn_mma_core.cuh"
#include "cluster_fold.cuh"

#include <atomic>

namespace kivi {
namespace {

__device__ int g_fault_word = 0;

// grid = units * head blocks * (nq_splits + n_res_splits) CTAs in one dimension
// (head blocks = ceil(n_rep / 4): a CTA serves up to four query heads); block =
// kWarps warps.  The first units*nq_splits CTAs are the quantized pieces, unit by unit:
// piece i of a unit covers token groups [i*gps, min((i+1)*gps, n_groups)).  The
// units*n_res_splits CTAs of the residual ring come last: they are short, so
// the long CTAs start first and the short ones fill the end of the grid
// (measured against ring CTAs first: 3.5 % faster at batch 64 x 32k, 7 % at
// batch 16 x 4k).  Partial slots: quantized piece i -> i, residual part r ->
// nq_splits + r.
//
// Shared memory: [kWarps][kStages][kStageBytes] stage rings | [kWarps][kScratchBytes]
// (in ring CTAs the first holds the queries, [4][128] fp32 times sm_scale*log2(e), absent
// rows zero) | mbarriers | (max, sum) of the warps.  When a warp is done, its ring doubles
// as the [4][128] buffer its scaled output goes to; the CTA then adds the warps'
// buffers in warp order (deterministic) and writes one partial.
//
// ONE: one query head per KV head.  WIDE: operands long enough for fp32 accuracy.
// FOLD: the CTAs of a unit and head block are a cluster and fold their partials
// themselves (a template, so that the wide grids keep their registers).
template <bool FOLD, bool WIDE, bool ONE>
__global__ void __launch_bounds__(kWarps * 32, 3)
attn_mma_kernel(kivi_layer L, int64_t quant_len, int res_start, int res_len,
                const void* q, int q_dtype,
                float scale_log2, int n_rep, int gps, int nq_splits, int n_res_splits, int res_chunk,
                float* __restrict__ part_o, float* __restrict__ part_ml, ClusterOut direct) {
    extern __shared__ __align__(128) uint8_t smem_raw[];
    uint8_t* stage_mem = smem_raw;                                               // [kWarps][kStages][kStageBytes]
    uint8_t* scratch_mem = smem_raw + kWarps * kStages * kStageBytes;            // [kWarps][kScratchBytes]
    float* q_s = reinterpret_cast<float*>(scratch_mem);                          // [4][128], ring CTAs
    uint64_t* bars = reinterpret_cast<uint64_t*>(scratch_mem + kWarps * kScratchBytes);   // [kWarps][kStages]
    float* ml_s = reinterpret_cast<float*>(bars + kWarps * kStages);             // [kWarps][4][2]
    float* const zero_s = ml_s + kWarps * 4 * 2;                                 // WIDE: [4][128] queries for the zero term

    // With a fold kernel behind this one, its few small blocks may become resident from
    // here on (it waits for this grid's end).  Without (FOLD), what comes next can be
    // another attention call, whose blocks would take places beside this one's while
    // other SMs stay empty: let in before the fold in the cluster (cluster_fold.cuh).
    if constexpr (!FOLD) cudaTriggerProgrammaticLaunchCompletion();
    stream_order();
    q = settled(q);
    settle_layer(L);

    // grid order: all quantized pieces (unit-major), then all residual-ring CTAs --
    // the long CTAs start first, the short ones fill the end
    // With more than four query heads per KV head a unit is served by two CTAs per
    // piece, one per block of four heads (they run side by side, so the second
    // read of the piece mostly comes from L2).
    const int head_blocks = (n_rep + 3) >> 2;
    const int n_quant_ctas = (int)L.num_units * head_blocks * nq_splits;
    // When the partials are folded inside clusters (FOLD), the CTAs of a unit and
    // head block lie side by side instead: pieces, then ring parts.
    const int n_all = nq_splits + n_res_splits;
    const int in_row = (int)blockIdx.x % n_all;
    const bool is_res = FOLD ? in_row >= nq_splits : (int)blockIdx.x >= n_quant_ctas;
    const int rel = is_res ? (int)blockIdx.x - n_quant_ctas : (int)blockIdx.x;
    const int per_unit = is_res ? n_res_splits : nq_splits;
    const int uv = FOLD ? (int)blockIdx.x / n_all : rel / per_unit;
    const int sub = FOLD ? (is_res ? in_row - nq_splits : in_row) : rel - uv * per_unit;
    const int u = uv / head_blocks, head0 = 4 * (uv - u * head_blocks);
    const int n_heads = n_rep - head0 < 4 ? n_rep - head0 : 4;       // heads of this CTA: head0 .. head0 + n_heads - 1
    const int n_splits_total = nq_splits + n_res_splits;
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);      // (known to be the same for all lanes)
    const int gid = lane >> 2, tig = lane & 3;
    uint8_t* wstage = stage_mem + warp * kStages * kStageBytes;
    float* fo = reinterpret_cast<float*>(wstage);                               // [4][128] once the ring is idle
    const int slot = is_res ? nq_splits + sub : sub;

    // ---- quantized split: start the copies before anything else ----------------
    const int64_t n_groups = quant_len / kG;
    const int64_t g_begin = is_res ? 0 : (int64_t)slot * gps;
    int64_t g_end = is_res ? 0 : g_begin + gps;
    if (g_end > n_groups) g_end = n_groups;
    const int n_my_groups = (int)(g_end - g_begin);
    const int n_chunks = (n_my_groups + kGPS - 1) / kGPS;
    const int my_n = n_chunks > warp ? (n_chunks - warp + kWarps - 1) / kWarps : 0;
    const uint32_t bar0 = smem_u32(bars + warp * kStages);
    const uint32_t stage0 = smem_u32(wstage);
    // The six pieces of a chunk (key codes, scales, zeros, value codes, scales, zeros) are
    // contiguous runs of 1024 or 512 bytes per token group.  One elected lane issues them
    // from addresses that are the same for the whole warp (a bulk copy takes its operands
    // from uniform registers: six lanes with an address each cost a loop of some 70
    // instructions).  Chunk c of this warp starts at group g_begin + (warp + kWarps*c)*kGPS.
    if (!is_res) {
        if (elect_one()) {
#pragma unroll
            for (int s = 0; s < kStages; ++s) mbar_init(bar0 + 8 * s, 1);
            mbar_init_fence();
        }
        __syncwarp();
    }
    const uint64_t policy = l2_stream_policy();
    const int64_t gw0 = (int64_t)u * (L.max_tokens / kG) + g_begin + (int64_t)warp * kGPS;
    auto issue = [&](int c) {                 // all lanes call it
        const int goff = (warp + kWarps * c) * kGPS;             // groups from g_begin
        const uint32_t ng = (n_my_groups - goff) < kGPS ? (n_my_groups - goff) : kGPS;
        const int s = c % kStages;
        const uint32_t bar = bar0 + 8 * s, dst = stage0 + s * kStageBytes;
        const int64_t g = gw0 + (int64_t)c * (kWarps * kGPS);
        if (elect_one()) {
            mbar_expect_tx(bar, ng * kGroupBytes);
            bulk_g2s(dst, L.k_codes + g * 1024, ng * 1024, bar, policy);
            bulk_g2s(dst + kGPS * 1024, L.k_scales + g * 128, ng * 512, bar, policy);
            bulk_g2s(dst + kGPS * 1536, L.k_zeros + g * 128, ng * 512, bar, policy);
            bulk_g2s(dst + kGPS * 2048, L.v_codes + g * 1024, ng * 1024, bar, policy);
            bulk_g2s(dst + kGPS * 3 * 1024, L.v_scales + g * 128, ng * 512, bar, policy);
            bulk_g2s(dst + kGPS * 3584, L.v_zeros + g * 128, ng * 512, bar, policy);
        }
        __syncwarp();
    };
    for (int c = 0; c < kStages && c < my_n; ++c) issue(c);

    const int64_t q_row = (int64_t)u * n_rep + head0;
    auto stage_queries = [&](float* dst) {                               // [4][128], pre-scaled (absent heads: zeros)
        for (int i = threadIdx.x; i < kD; i += blockDim.x) {
            float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if ((i >> 5) < n_heads) {
                if (q_dtype == KIVI_BF16) RowVec<__nv_bfloat16>::load4(reinterpret_cast<const __nv_bfloat16*>(q) + q_row * kD + 4 * i, t);
                else RowVec<float>::load4(reinterpret_cast<const float*>(q) + q_row * kD + 4 * i, t);
            }
            *reinterpret_cast<float4*>(dst + 4 * i) = make_float4(scale_log2 * t[0], scale_log2 * t[1], scale_log2 * t[2], scale_log2 * t[3]);
        }
    };
    if (is_res) {
        // ---------------- residual ring ----------------
        stage_queries(q_s);
        __syncthreads();
        const int rs = sub;
        const int t_begin = rs * res_chunk;
        const int t_end = t_begin + res_chunk < res_len ? t_begin + res_chunk : res_len;
        float m[4], l[4], o[4][4];
        if (L.res_dtype == KIVI_BF16)
            residual_part<__nv_bfloat16>(reinterpret_cast<const __nv_bfloat16*>(L.k_res) + (int64_t)u * L.residual_cap * kD,
                                         reinterpret_cast<const __nv_bfloat16*>(L.v_res) + (int64_t)u * L.residual_cap * kD,
                                         L.residual_cap, res_start, res_len, t_begin, t_end, q_s, lane, warp, m, l, o);
        else
            residual_part<float>(reinterpret_cast<const float*>(L.k_res) + (int64_t)u * L.residual_cap * kD,
                                 reinterpret_cast<const float*>(L.v_res) + (int64_t)u * L.residual_cap * kD,
                                 L.residual_cap, res_start, res_len, t_begin, t_end, q_s, lane, warp, m, l, o);
        if (lane < 4) {
            // lane h publishes head h (m and l are warp-uniform after the reductions)
            float mh = m[0], lh = l[0];
            if (lane == 1) { mh = m[1]; lh = l[1]; }
            if (lane == 2) { mh = m[2]; lh = l[2]; }
            if (lane == 3) { mh = m[3]; lh = l[3]; }
            ml_s[(warp * 4 + lane) * 2] = mh; ml_s[(warp * 4 + lane) * 2 + 1] = lh;
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            float M = -INFINITY;
#pragma unroll
            for (int w2 = 0; w2 < kWarps; ++w2) M = fmaxf(M, ml_s[(w2 * 4 + h) * 2]);
            const float f = (m[h] == -INFINITY) ? 0.0f : ex2(m[h] - M);
            *reinterpret_cast<float4*>(fo + h * kD + 4 * lane) = make_float4(f * o[h][0], f * o[h][1], f * o[h][2], f * o[h][3]);
        }
    } else {
        // ---------------- quantized history ----------------
        std::conditional_t<ONE, OneView, LaneView> v;
        v.gid = gid; v.tig = tig; v.lane = lane;
        uint8_t* scratch = scratch_mem + warp * kScratchBytes;
        v.scratch = smem_u32(scratch);
        // row `lane & 15` of matrix `lane >> 4`
        v.k_rows = v.scratch + 1024 * (lane >> 4) + 512 * (lane & 1) + 16 * ((lane >> 1) & 7);
        v.v_rows = v.scratch + 256 * (lane >> 4) + 16 * (lane & 15);
        // contraction index of the token whose scales are row `lane`
        const int kap = gid >> 2, k = 4 * tig + (gid & 3);
        v.v_write = v.scratch + 16 * k + 8 * (kap ^ (k >> 3));
        v.v_first = 32 * (tig >> 1);
        if constexpr (ONE) {
            v.p_write = v.scratch + 128 * (tig & 1) + 4 * (16 * kap + (gid & 3));
        } else {
            v.p_even = v.scratch + 16 * (16 * kap + (gid & 3)) + 64 * kap + 4 * tig;
            v.p_odd = v.scratch + 16 * (16 * kap + (gid & 3)) + 64 * (1 - kap) + 4 * tig;
            v.p_read = v.scratch + 16 * p_row(lane);
            v.rest_rows = 128 * (lane >> 4) + 512 * (lane & 1) + 16 * ((lane >> 1) & 7);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) asm volatile("mov.b32 %0, %1;" : "=r"(v.start[i]) : "n"(kTwo23Bits));
        if (q_dtype == KIVI_BF16) load_queries(reinterpret_cast<const __nv_bfloat16*>(q) + q_row * kD, n_heads, scale_log2, v);
        else load_queries(reinterpret_cast<const float*>(q) + q_row * kD, n_heads, scale_log2, v);

        if constexpr (WIDE) {
#pragma unroll
            for (int i = 0; i < 4; ++i) asm volatile("mov.b32 %0, %1;" : "=r"(v.ones[i]) : "n"(kOnes));
            v.q_zero = reinterpret_cast<const float4*>(zero_s) + 32 * tig;
            stage_queries(zero_s);
            __syncthreads();
        }

        std::conditional_t<ONE, OneState, WarpState> st;
        clear(st);

        bool ok = true;
        int c = 0;
        for (; c < my_n; ++c) {
            const int s = c % kStages;
            if (!__all_sync(0xffffffffu, mbar_wait(bar0 + 8 * s, (uint32_t)(c / kStages) & 1u))) { ok = false; break; }
            const int goff = (warp + kWarps * c) * kGPS;
            const uint8_t* sb = wstage + s * kStageBytes;
            if (n_my_groups - goff >= 2) process_groups<2, WIDE>(sb, v, scratch, st);
            else process_groups<1, WIDE>(sb, v, scratch, st);
            __syncwarp();
            if (c + kStages < my_n) issue(c + kStages);
        }
        if (!ok) {
            // A copy did not land within the bound.  The copies still in flight
            // target this warp's ring: give each of them (chunks c .. c+kStages-1,
            // those that were issued) a second bounded wait on its own phase
            // before the ring is reused, then report an empty partial.
            if (lane == 0) atomicExch(&g_fault_word, 1);
            for (int i = c; i < c + kStages && i < my_n; ++i)
                mbar_wait(bar0 + 8 * (i % kStages), (uint32_t)(i / kStages) & 1u);
            clear(st);
        }

        fold_lanes<ONE>(v, st, scratch, fo, ml_s, warp);
    }
    __syncthreads();

    // ---- the CTA's partial: warps added in warp order ------------------------------
    // (for the fold inside a cluster it stays in shared memory, behind the first warp's buffer)
    const int64_t pbase = ((int64_t)u * n_splits_total + slot) * n_rep + head0;
    float* const cta_o = reinterpret_cast<float*>(stage_mem) + 4 * kD;
    for (int i = threadIdx.x; i < kD; i += blockDim.x) {
        const int h = i >> 5, cc = (i & 31) * 4;
        if (h < n_heads) {
            float4 a = *reinterpret_cast<const float4*>(stage_mem + h * kD * 4 + cc * 4);
#pragma unroll
            for (int w2 = 1; w2 < kWarps; ++w2) {
                const float4 b = *reinterpret_cast<const float4*>(stage_mem + w2 * kStages * kStageBytes + h * kD * 4 + cc * 4);
                a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
            }
            *reinterpret_cast<float4*>(FOLD ? cta_o + h * kD + cc : part_o + (pbase + h) * kD + cc) = a;
        }
    }
    float* const ml_out = FOLD ? cta_o + 4 * kD : part_ml + pbase * 2;
    if (threadIdx.x < n_heads) {
        const int h = threadIdx.x;
        float Mh = -INFINITY, ls = 0.0f;
        for (int w2 = 0; w2 < kWarps; ++w2) Mh = fmaxf(Mh, ml_s[(w2 * 4 + h) * 2]);
        for (int w2 = 0; w2 < kWarps; ++w2) {
            const float mw = ml_s[(w2 * 4 + h) * 2];
            if (mw != -INFINITY) ls += ml_s[(w2 * 4 + h) * 2 + 1] * ex2(mw - Mh);
        }
        ml_out[h * 2] = Mh;
        ml_out[h * 2 + 1] = ls;
    }
    if constexpr (FOLD) cluster_fold(cta_o, ml_out, n_heads, kD, (int64_t)u * n_rep + head0, direct);
}

constexpr size_t kSmemBytes = (size_t)kWarps * (kStages * kStageBytes + kScratchBytes) + kWarps * kStages * 8 + kWarps * 4 * 2 * 4;
constexpr size_t kSmemBytesWide = kSmemBytes + 4 * kD * 4;
static_assert(kScratchBytes >= 4 * kD * 4, "ring CTAs keep the queries in the first warp's scratch");
static_assert(kStages * kStageBytes >= 2 * 4 * kD * 4 + 32, "a warp's ring doubles as its [4][128] fold buffer, the first also holds the CTA's partial");
static_assert(kWarps * 32 >= 32, "at least one warp");

}  // namespace

bool attn_mma_supported(const kivi_layer* L, int n_rep, const void* q) {
    auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
    return L->head_dim == kD && L->group_size == kG && n_rep >= 1 && n_rep <= 8 && al(q) &&
           al(L->k_res) && al(L->v_res) && al(L->k_codes) && al(L->k_scales) && al(L->k_zeros) && al(L->v_codes) && al(L->v_scales) && al(L->v_zeros);
}

// number of residual CTAs per unit and tokens per CTA (multiple of 32)
void attn_mma_residual_plan(int res_len, int* n_res_splits, int* res_chunk) {
    int rs = (res_len + 32 * kWarps - 1) / (32 * kWarps);
    if (rs > 8) rs = 8;
    int chunk = rs ? (res_len + rs - 1) / rs : 0;
    chunk = (chunk + 31) / 32 * 32;
    *n_res_splits = chunk ? (res_len + chunk - 1) / chunk : 0;
    *res_chunk = chunk;
}

// the opt-in shared-memory size is a per-device attribute of the kernel
static int ensure_smem_attr(int* dev_out) {
    static std::atomic<bool> attr_set[64];
    int dev = 0;
    KIVI_CUDA_OK(cudaGetDevice(&dev));
    KIVI_REQUIRE(dev >= 0 && dev < 64, "device ordinal %d out of range", dev);
    if (!attr_set[dev].load(std::memory_order_acquire)) {
        for (auto* kernel : {attn_mma_kernel<false, false, false>, attn_mma_kernel<true, false, false>, attn_mma_kernel<false, true, false>,
                             attn_mma_kernel<true, true, false>, attn_mma_kernel<false, false, true>, attn_mma_kernel<true, false, true>})
            KIVI_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytesWide));
        attr_set[dev].store(true, std::memory_order_release);
    }
    if (dev_out) *dev_out = dev;
    return KIVI_OK;
}

// CTAs of the kernel that one SM holds at a time (registers and shared memory
// decide); asked from the runtime once per device.  0 = the query failed.
int attn_mma_ctas_per_sm() {
    static std::atomic<int> cached[64];
    int dev = 0;
    if (ensure_smem_attr(&dev) != KIVI_OK) return 0;
    int n = cached[dev].load(std::memory_order_acquire);
    if (n == 0) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, attn_mma_kernel<false, false, false>, kWarps * 32, kSmemBytesWide) != cudaSuccess || n <= 0)
            return 0;
        cached[dev].store(n, std::memory_order_release);
    }
    return n;
}

int run_attn_mma(const kivi_layer* L, int64_t quant_len, int res_start, int res_len,
                 const void* q, int q_dtype, int n_rep, float scale_log2, bool wide, int nq_splits, int gps,
                 int n_res_splits, int res_chunk, float* part_o, float* part_ml, const ClusterOut& direct, cudaStream_t st) {
    if (int rc = ensure_smem_attr(nullptr)) return rc;
    dim3 grid((unsigned)(nq_splits + n_res_splits) * (unsigned)L->num_units * (unsigned)((n_rep + 3) / 4));
    const bool fold = direct.out != nullptr;
    auto* const kernel = wide ? (fold ? attn_mma_kernel<true, true, false> : attn_mma_kernel<false, true, false>)
                       : n_rep == 1 ? (fold ? attn_mma_kernel<true, false, true> : attn_mma_kernel<false, false, true>)
                                    : (fold ? attn_mma_kernel<true, false, false> : attn_mma_kernel<false, false, false>);
    KIVI_CUDA_OK(launch_cluster(kernel, direct.out ? nq_splits + n_res_splits : 0, grid, kWarps * 32, wide ? kSmemBytesWide : kSmemBytes, st, true, *L, quant_len, res_start, res_len, q, q_dtype, scale_log2,
                        n_rep, gps, nq_splits, n_res_splits, res_chunk, part_o, part_ml, direct));
    return KIVI_OK;
}

// ---- self-test: how far below the largest product the tensor core keeps bits -------
// One m16n8k16 MMA per k: C = -1, products {1 * 1, 2^-a * 2^-b} with a + b = k.
// If the unit kept every bit the result would be exactly 2^-k; it aligns the
// addends on their exponent fields and truncates below a fixed distance from the
// largest, so from some k on the small product is lost.  (Why the kernel above
// contracts bytes, whose sums are exact.)
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__global__ void mma_alignment_probe_kernel(int* kept_out) {
    const int lane = threadIdx.x, gid = lane >> 2, tig = lane & 3;
    int kept = 0;
    for (int k = 8; k <= 34; ++k) {
        const int a_exp = k < 14 ? k : 14, b_exp = k - a_exp;          // both factors stay normal fp16 numbers
        // A[row][0] = 1, A[row][1] = 2^-a; B[0][col] = 1, B[1][col] = 2^-b; everything else 0
        const __half2 a01 = __halves2half2(__float2half(1.0f), __float2half(ldexpf(1.0f, -a_exp)));
        const __half2 b01 = __halves2half2(__float2half(1.0f), __float2half(ldexpf(1.0f, -b_exp)));
        uint32_t a[4] = {0u, 0u, 0u, 0u}, b0 = 0u;
        if (tig == 0) {                                                // k-slots 0 and 1 live in lanes with tig == 0
            a[0] = *reinterpret_cast<const uint32_t*>(&a01);
            a[1] = a[0];
            b0 = *reinterpret_cast<const uint32_t*>(&b01);
        }
        float c[4] = {-1.0f, -1.0f, -1.0f, -1.0f};
        mma_f16(c, a, b0, 0u);
        const bool ok = c[0] == ldexpf(1.0f, -k);
        if (__all_sync(0xffffffffu, ok)) kept = k;
    }
    (void)gid;
    if (lane == 0) *kept_out = kept;
}

int run_mma_alignment_probe(int* bits_out) {
    int* d = nullptr;
    KIVI_CUDA_OK(cudaMalloc(&d, sizeof(int)));
    mma_alignment_probe_kernel<<<1, 32>>>(d);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) e = cudaMemcpy(bits_out, d, sizeof(int), cudaMemcpyDeviceToHost);
    cudaFree(d);
    if (e != cudaSuccess) { set_error("tensor-core alignment probe failed: %s", cudaGetErrorString(e)); return KIVI_ERR_CUDA; }
    return KIVI_OK;
}

int attn_mma_fault_word(int* out) {
    KIVI_CUDA_OK(cudaMemcpyFromSymbol(out, g_fault_word, sizeof(int)));
    return KIVI_OK;
}

int attn_mma_fault_clear() {
    const int zero = 0;
    KIVI_CUDA_OK(cudaMemcpyToSymbol(g_fault_word, &zero, sizeof(int)));
    return KIVI_OK;
}

}  // namespace kivi
