// Device-side pieces of the operators over a packed run (several new tokens per sequence, see brasa_packed_run): whose a row is, and where
// a position lies in the pool. Everything read from device tables is held against the buffers' sizes before it becomes an address.
#pragma once
#include "attn_device.cuh"

namespace brasa_dev {

struct PackedView {
    const int32_t *table;   // [seqs][max_pages]
    const uint32_t *lens, *starts;
    uint32_t seqs, max_pages, num_pages, tokens, longest, hkv;
};

// The last sequence that begins at or before row t: the warp looks at 32 boundaries at a time. UINT32_MAX when none does.
__device__ __forceinline__ uint32_t packed_sequence(const uint32_t *starts, uint32_t seqs, uint32_t t, uint32_t lane) {
    uint32_t lo = 0, n = seqs;  // (starts[lo] <= t once a boundary was found)
    bool found = false;
    while (n > 1 || !found) {
        const uint32_t step = (n + 31) / 32, at = lane * step;
        const uint32_t c = __popc(__ballot_sync(0xffffffffu, at < n && starts[lo + at] <= t));
        if (c == 0) return UINT32_MAX;
        found = true;
        lo += (c - 1) * step;
        n = min(step, n - (c - 1) * step);
    }
    return lo;
}

// Row t of a run: its sequence and position; false for a row that is nobody's (behind the last sequence, past `longest`, starts that fall).
__device__ __forceinline__ bool packed_row(const PackedView &p, uint32_t t, uint32_t lane, uint32_t &seq, uint32_t &pos) {
    seq = packed_sequence(p.starts, p.seqs, t, lane);
    if (seq == UINT32_MAX || t >= p.starts[seq + 1]) return false;
    const uint32_t j = t - p.starts[seq];
    const uint64_t at = (uint64_t)p.lens[seq] + j;
    pos = (uint32_t)min(at, (uint64_t)UINT32_MAX);
    return j < p.longest;
}

// Page of a position, or -1 where there is none.
__device__ __forceinline__ int32_t packed_page(const PackedView &p, uint32_t seq, uint32_t pos) {
    const uint32_t i = pos / BRASA_KV_PAGE;
    if (i >= p.max_pages) return -1;
    const int32_t page = p.table[(size_t)seq * p.max_pages + i];
    return (uint32_t)page < p.num_pages ? page : -1;
}

}  // namespace brasa_dev
