// paged_kv.hpp -- a ragged batch of sequences over a key/value cache in
// pages, as its kernels see it.
//
// The cache is num_pages pages of page_size rows; row r of page p, key/value
// head hh, lies at p * page_stride + r * row_stride + hh * head_stride
// (elements).  Position j of sequence s is row j % page_size of page
// table[s, j / page_size].  Rows q_offsets[s] .. q_offsets[s + 1] - 1 of the
// new tokens belong to sequence s and are its last positions: row i of them is
// position kv_lens[s] - q_len + i.
//
// The table, offsets and lengths are device memory that the host does not
// read, so a captured graph can be replayed while they change.  What the host
// cannot check, the kernels do: offsets are clamped to the rows there are,
// lengths to what the table can hold, and a page outside the cache is neither
// read nor written.  Such lengths and pages, and tokens whose position the table
// does not hold, set a bit of *status.
#pragma once

#include "common.hpp"

namespace gfh {
namespace paged {

enum Status : int { kBadLength = 1, kBadPage = 2, kBadValue = 4 };

struct View {
    char *k, *v;
    int64_t num_pages;
    int64_t page_stride, row_stride, head_stride;  // elements
    const int32_t *table;
    int64_t table_stride;
    const int32_t *kv_lens, *q_offsets;
    int32_t *status;  // nullable
    int page_size, page_shift;  // shift: -1 unless page_size is a power of two
    int capacity;               // positions a row of the table can hold
    int num_seqs, tokens;
    int heads, group, hkv, d;   // group = heads / hkv query heads per key/value head
};

// (page and row of a position; the branch is uniform)
__device__ __forceinline__ int page_of(const View &p, int pos) {
    return p.page_shift >= 0 ? (int)((unsigned)pos >> p.page_shift) : (int)((unsigned)pos / (unsigned)p.page_size);
}

__device__ __forceinline__ void raise(const View &p, int bit) {
    if (p.status) atomicOr(p.status, bit);
}

// The number of leading i in [0, n) for which f(i) holds (f: true, then
// false), found by the whole wave: 64 candidates per step, so one round of
// loads up to n = 64, two up to 4096.  Whatever f is, the result is in [0, n].
template <typename F>
__device__ __forceinline__ int wave_leading(int n, int lane, F &&f) {
    int lo = 0, len = n;
    while (len > 0) {
        const int step = (len + 63) >> 6;
        const int i = lo + (lane + 1) * step - 1;  // the last of this lane's candidates
        const int c = __popcll(__ballot(i < lo + len && f(i)));
        len = min(step - 1, len - c * step);
        lo += c * step;
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

__device__ __forceinline__ int offset_at(const View &p, int s) {
    return min(max(p.q_offsets[s], 0), p.tokens);
}

__device__ __forceinline__ int length_at(const View &p, int s) {
    const int n = p.kv_lens[s];
    if (n < 0 || n > p.capacity) raise(p, kBadLength);
    return min(max(n, 0), p.capacity);
}

}  // namespace paged
}  // namespace gfh
