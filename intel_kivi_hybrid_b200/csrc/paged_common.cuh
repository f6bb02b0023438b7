// What the kernels over a paged cache share: a sequence's place in a ragged batch, its
// pages and its window.
//
// A sequence of t tokens keeps the first quant_of(t) of them in pages (2 bits, whole
// groups of G tokens) and the others in its ring, token t in slot t % R.  quant_of is the
// flush policy of kivi_cache_plan as a function of the length alone: whole groups leave
// while the window holds R tokens or more, so what is left is R - G .. R - 1 tokens once
// anything has left, whichever way the tokens came in.  Lengths are therefore all that a
// sequence has of state, and they stay on the device.
#pragma once

#include "kivi_common.cuh"

namespace kivi {

constexpr int kPagedFault = 4;                     // bit of the device fault word: a batch's arrays point outside the cache

__host__ __device__ __forceinline__ int quant_of(int total, int G, int R) {
    return total >= R ? ((total - R) / G + 1) * G : 0;
}

#ifdef __CUDACC__

struct PagedSeq {
    int held, n;            // tokens before the step, new tokens
    int row0;               // its first row in the arrays of new tokens
    int slot;               // its ring
    const int32_t* pages;   // its row of the page table
};

// Sequence s of the batch; false (and held = n = 0, so that it is counted as an empty one where work
// is dealt out) for one whose numbers do not fit the arrays: no kernel follows them.  Every number
// that is used as an index below comes from here.
// (Layer: kivi_paged_layer or kivi_paged8_layer)
template <typename Layer>
__device__ __forceinline__ bool load_seq(const Layer& L, const kivi_paged_batch& b, int s, PagedSeq& q) {
    const int r0 = b.cu_new[s], r1 = b.cu_new[s + 1], held = b.seq_lens[s], slot = b.slots[s];
    q.pages = b.page_table + (int64_t)s * b.table_width;
    q.row0 = r0; q.held = 0; q.slot = slot; q.n = 0;
    if (r0 < 0 || r1 < r0 || r1 > b.total_new || r1 - r0 > b.max_new) return false;
    if (held < 0 || held > b.max_len - (r1 - r0) || slot < 0 || slot >= L.num_slots) return false;
    q.held = held;
    q.n = r1 - r0;
    return true;
}

// One block of a launch tells of the sequences that are left out.
template <typename Layer>
__device__ __forceinline__ void report_left_out(const Layer& L, const kivi_paged_batch& b, int* fault) {
    for (int s = threadIdx.x; s < b.num_seqs; s += blockDim.x) {
        PagedSeq q;
        if (!load_seq(L, b, s, q)) atomicOr(fault, kPagedFault);
    }
}

// page of group position t (t a token index below quant_of); a bad entry counts as page 0
// and is reported
template <typename Layer>
__device__ __forceinline__ int page_of(const Layer& L, const PagedSeq& q, int t, int* fault) {
    const int p = q.pages[t / L.page_tokens];
    if ((unsigned)p < (unsigned)L.num_pages) return p;
    atomicOr(fault, kPagedFault);
    return 0;
}

__device__ __forceinline__ int ring_slot(int t, int shift, int R) { return (int)(((unsigned)t + (unsigned)shift) % (unsigned)R); }

// The sequence that work item `item` belongs to and the item's number within it, where
// count(s) gives the items of sequence s.  Called by whole warps (every lane gets the
// answer); s = num_seqs when there are fewer items.
struct ItemPlace { int s, sub; };
template <typename F>
__device__ __forceinline__ ItemPlace find_item(int item, int num_seqs, const F& count) {
    const int lane = threadIdx.x & 31;
    int before = 0;
    for (int s0 = 0; s0 < num_seqs; s0 += 32) {
        const int c = s0 + lane < num_seqs ? count(s0 + lane) : 0;
        int sum = c;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += up;
        }
        const unsigned beyond = __ballot_sync(0xffffffffu, before + sum > item);
        if (beyond) {
            const int l = __ffs(beyond) - 1;
            const int first = before + __shfl_sync(0xffffffffu, sum - c, l);
            return {s0 + l, item - first};
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    return {num_seqs, 0};
}

__device__ __forceinline__ void settle_paged(kivi_paged_layer& L, kivi_paged_batch& b) {
    L.k_codes = settled(L.k_codes); L.k_scales = settled(L.k_scales); L.k_zeros = settled(L.k_zeros);
    L.v_codes = settled(L.v_codes); L.v_scales = settled(L.v_scales); L.v_zeros = settled(L.v_zeros);
    L.k_res = settled(L.k_res); L.v_res = settled(L.v_res);
    b.page_table = settled(b.page_table); b.slots = settled(b.slots);
    b.seq_lens = settled(b.seq_lens); b.cu_new = settled(b.cu_new);
}

#endif

// ---- host side -------------------------------------------------------------------
int validate_paged(const kivi_paged_layer* L);
int validate_batch(const kivi_paged_layer* L, const kivi_paged_batch* b);
// Rows that are written where rows are read: the same ones, or none of them (an element must not be
// written while another row's reader still wants it).
int validate_in_place(const kivi_rows* to, const char* to_name, const kivi_rows* from, const char* from_name, int rows, int heads, bool same_type);

}  // namespace kivi
