// What the kernels on paged caches share: whose row is whose, and where its position lies.
#pragma once
#include "common.h"

namespace tpamd {

// tpamd_pages as the kernels take it. Lengths, starts, counts and the table are read on the device and not trusted: they are held to the rows there
// are and the positions that the table has room for, and a page outside of the pool is no memory.
struct PagesView {
    char *k, *v;
    int64_t k_page, k_head, k_pos, v_page, v_head, v_pos;  // elements
    const int32_t *table, *lengths, *starts, *counts;
    int64_t table_row;
    int pages, shift;  // a page has 1 << shift positions
    int seqs, each;    // each: rows of a sequence where starts is NULL
    int rows, room;    // room: positions of a sequence that the table can name
};

struct SeqRows {
    int first, count, length;  // its new rows, and its positions with them
};
__device__ __forceinline__ SeqRows rows_of(const PagesView &p, int b) {
    SeqRows s;
    if (p.starts != nullptr) {
        const int from = p.starts[b], to = p.starts[b + 1];
        s.first = min(max(from, 0), p.rows);
        s.count = min(max(to, s.first), p.rows) - s.first;
    } else {
        s.first = b * p.each;
        s.count = p.counts != nullptr ? min(max(p.counts[b], 0), p.each) : p.each;
    }
    s.length = min(max(p.lengths[b], 0), p.room);
    return s;
}

// The page of a sequence's position (0 <= position < room), or -1.
__device__ __forceinline__ int page_of(const PagesView &p, int b, int position) {
    const int page = p.table[b * p.table_row + (position >> p.shift)];
    return static_cast<unsigned>(page) < static_cast<unsigned>(p.pages) ? page : -1;
}

// The sequence that a row belongs to, its place among the sequence's new rows in `place`; -1: none. All 64 lanes of a wavefront ask for one row. Of packed rows it is
// the last sequence that starts at or before the row: 64 starts are looked at at a time.
__device__ __forceinline__ int seq_of_row(const PagesView &p, int row, int &place) {
    if (p.starts == nullptr) {
        const int b = row / p.each;
        place = row - b * p.each;
        if (b >= p.seqs || (p.counts != nullptr && place >= p.counts[b])) return -1;
        return b;
    }
    const int lane = threadIdx.x & 63;
    int lo = 0, range = p.seqs;
    while (true) {
        const int step = (range + 63) / 64, at = lane * step;
        const bool before = at < range && p.starts[lo + at] <= row;
        const int n = __popcll(__ballot(before));
        if (n == 0) return -1;
        lo += (n - 1) * step;
        if (step == 1) break;
        range = min(step, range - (n - 1) * step);
    }
    place = row - p.starts[lo];
    return row < p.starts[lo + 1] ? lo : -1;
}

// Host side (paged.hip): checks a tpamd_pages for `rows` rows and fills in the view.
int take_pages(const char *who, const tpamd_pages *pages, int64_t rows, PagesView *out);

}  // namespace tpamd
