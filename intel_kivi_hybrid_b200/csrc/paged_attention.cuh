// Arguments that the attention kernels over a paged cache share.
#pragma once

#include "paged_common.cuh"

namespace kivi {

struct PagedAttnArgs {
    kivi_paged_layer L;
    kivi_paged_batch b;
    kivi_rows q, k, v, out;
    int q_dtype, out_dtype, n_rep, vec;
    float scale_log2;
    int pieces, chunk;           // a block's tokens are cut into pieces of `chunk` (no block has more than `pieces`)
    float *part_o, *part_ml;     // [block][KV head][piece][row]: unnormalised output, (maximum, sum)
    int* rough;                  // [block][KV head][piece], or null: rows to be computed in fp32 after all
};

#ifdef __CUDACC__
__device__ __forceinline__ void settle_args(PagedAttnArgs& a) {
    settle_paged(a.L, a.b);
    a.q.data = settled(a.q.data); a.k.data = settled(a.k.data); a.v.data = settled(a.v.data);
    a.part_o = settled(a.part_o); a.part_ml = settled(a.part_ml); a.rough = settled(a.rough);
}
template <typename T> __device__ __forceinline__ float4 load4(const T* p, bool vec);
template <> __device__ __forceinline__ float4 load4<float>(const float* p, bool vec) {
    return vec ? *reinterpret_cast<const float4*>(p) : make_float4(p[0], p[1], p[2], p[3]);
}
template <> __device__ __forceinline__ float4 load4<__nv_bfloat16>(const __nv_bfloat16* p, bool vec) {
    if (!vec) return make_float4(__bfloat162float(p[0]), __bfloat162float(p[1]), __bfloat162float(p[2]), __bfloat162float(p[3]));
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
}
__device__ __forceinline__ float4 load4_as(const kivi_rows& r, int dtype, int64_t row, int head, int d, bool vec) {
    const int64_t at = row * r.row_stride + (int64_t)head * r.head_stride + d;
    return dtype == KIVI_BF16 ? load4(reinterpret_cast<const __nv_bfloat16*>(r.data) + at, vec) : load4(reinterpret_cast<const float*>(r.data) + at, vec);
}

// Four channels of token tt of group g of the pages.
__device__ __forceinline__ float4 packed_key4(const kivi_paged_layer& L, int64_t g, int tt, int d) {
    const int D = L.head_dim, Q = L.group_size / 4, sh = 2 * (tt & 3);
    const uint32_t w = *reinterpret_cast<const uint32_t*>(L.k_codes + g * (D * Q) + kblock_offset(d, tt >> 2, Q, D < 64 ? D : 64));
    const float4 s = *reinterpret_cast<const float4*>(L.k_scales + g * D + d), z = *reinterpret_cast<const float4*>(L.k_zeros + g * D + d);
    return make_float4(fmaf((float)((w >> sh) & 3u), s.x, z.x), fmaf((float)((w >> (sh + 8)) & 3u), s.y, z.y),
                       fmaf((float)((w >> (sh + 16)) & 3u), s.z, z.z), fmaf((float)((w >> (sh + 24)) & 3u), s.w, z.w));
}
__device__ __forceinline__ float4 packed_value4(const kivi_paged_layer& L, int64_t g, int tt, int d) {
    const int D = L.head_dim, G = L.group_size;
    const uint32_t c = L.v_codes[g * (D * (G / 4)) + vcode_offset(tt, d / 4, D, G)];
    const int64_t at = g * D + vmeta_index(tt, d / G, D, G);
    const float s = L.v_scales[at], z = L.v_zeros[at];
    return make_float4(fmaf((float)(c & 3u), s, z), fmaf((float)((c >> 2) & 3u), s, z), fmaf((float)((c >> 4) & 3u), s, z), fmaf((float)(c >> 6), s, z));
}
#endif

}  // namespace kivi
