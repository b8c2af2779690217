// kq_attn.h — what the attention kernels (kq_attn.hip) and the step that
// stores new rows (kq_kv.hip) are given, and the device helpers they share.
#pragma once

#include "kq_device.h"
#include "kq_launch.h"

namespace kq {

// Where the rows of sequence s lie and how many keys of its own it has. What
// the arrays hold is clamped to the sizes the host gave, so no content of
// theirs leads out of a buffer.
struct SeqRows {
    int32_t first, last;   // packed rows [first, last)
    int32_t len;           // own keys
};
__device__ __forceinline__ SeqRows seq_rows(const AttnArgs &a, uint32_t s) {
    SeqRows r;
    if (a.q_start) {
        r.first = min(max(a.q_start[s], 0), (int32_t)a.n_rows);
        r.last = min(max(a.q_start[s + 1], r.first), (int32_t)a.n_rows);
    } else {
        r.first = (int32_t)s;
        r.last = r.first + 1;
    }
    r.len = min(max(a.kv_len[s], 0), (int32_t)a.max_kv);
    return r;
}
// The sequence that packed row `row` belongs to: the last s with q_start[s] <= row.
__device__ __forceinline__ uint32_t seq_of_row(const AttnArgs &a, int32_t row) {
    if (!a.q_start) return (uint32_t)row;
    uint32_t lo = 0, hi = a.n_seq - 1;
    while (lo < hi) {
        const uint32_t mid = (lo + hi + 1) / 2;
        if (a.q_start[mid] <= row) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
// Position of a packed row on its sequence's key axis (shared keys first).
__device__ __forceinline__ int32_t row_pos(const AttnArgs &a, const SeqRows &r, int32_t row) {
    return (int32_t)a.n_shared + r.len - (r.last - row);
}

}  // namespace kq
