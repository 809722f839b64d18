// Operators on device memory around a paged K/V cache: rotary positions, rows written into pages, attention over pages,
// attention weights added up per cached position, and the cache cut back to a budget. Launch interface of the gfx950
// kernels (jfh_paged.hip) and the index arithmetic that they and the host share.
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>

#if defined(__HIPCC__)
#define JFH_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define JFH_HOST_DEVICE inline
#endif

namespace jfh::paged {

constexpr uint32_t kMaxHeadDim = 256;
constexpr uint32_t kMaxRotPairs = 128;
constexpr uint32_t kMaxPageSize = 65536;
constexpr uint32_t kComputeUnits = 256;  // of an MI355X
constexpr uint32_t kSlotStep = 65536;    // no kernel's loop over slots steps further, so that slots stay in 32 bits
constexpr uint32_t kMaxLength = 0x7FFFFFFF - kSlotStep;

// Value d of head h of row r lies at data[r * row_stride + h * head_stride + d] (strides in values).
struct Rows {
    void* data;
    int64_t row_stride, head_stride;
    uint32_t rows, heads, head_dim, type;
};

// Position i of page p of K/V head h: values at page_stride p + head_stride h + slot_stride i of k and v, its weight
// and position at (p n_head_kv + h) page_size + i.
struct Cache {
    void* k;
    void* v;
    float* weights;
    int32_t* positions;
    int64_t page_stride, head_stride, slot_stride;
    uint32_t n_pages, page_shift, n_head_kv, head_dim, type;
};

struct Batch {
    const int32_t* table;
    int32_t* lengths;
    const int32_t* row_starts;
    uint32_t n_seq, table_stride, max_rows, max_length;
};

// Rows [row0, row0 + rows) of the step are sequence s's; row row0 + r stands at slot first + r, of which those in
// [0, len) exist: the bounds leave out rows from max_rows and slots from max_length on, and move nothing. Whatever the
// device arrays hold, the rows lie inside the step's n_rows, [0, len) inside the table, and first + rows in 32 bits.
struct Span {
    int32_t row0, rows, len, first;
};

JFH_HOST_DEVICE int32_t clamped(int32_t v, int32_t lo, int32_t hi) { return v < lo ? lo : v > hi ? hi : v; }

JFH_HOST_DEVICE int32_t span_length(const Batch& b, uint32_t s) {
    return clamped(b.lengths[s], 0, static_cast<int32_t>(b.max_length));
}

JFH_HOST_DEVICE Span sequence_span(const Batch& b, uint32_t n_rows, uint32_t s) {
    const int32_t r0 = clamped(b.row_starts[s], 0, static_cast<int32_t>(n_rows)), end = b.row_starts[s + 1];
    const int32_t r1 = clamped(end, r0, static_cast<int32_t>(n_rows));
    const int32_t n = clamped(r1 - r0, 0, static_cast<int32_t>(b.max_rows));
    // row end - 1 stands at the last slot
    const int64_t first = static_cast<int64_t>(b.lengths[s] > 0 ? b.lengths[s] : 0) - end + r0;
    return Span{r0, n, span_length(b, s), static_cast<int32_t>(first < b.max_length ? first : b.max_length)};
}

// Slots that row row0 + r sees when it sees what is before it and itself.
JFH_HOST_DEVICE int32_t slots_seen(const Span& x, int32_t r) { return clamped(x.first + r + 1, 0, x.len); }

// Rows of a sequence before the first that sees a slot.
JFH_HOST_DEVICE int32_t rows_before(const Span& x, int32_t slot) {
    const int64_t n = static_cast<int64_t>(slot) - x.first;
    return n < 0 ? 0 : n < x.rows ? static_cast<int32_t>(n) : x.rows;
}

// The sequence of a row (row_starts ascending), or -1 for a row of none.
JFH_HOST_DEVICE int32_t sequence_of(const Batch& b, uint32_t n_rows, int32_t row, Span* span) {
    uint32_t lo = 0, hi = b.n_seq;  // the last s with row_starts[s] <= row
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (b.row_starts[mid] <= row) lo = mid;
        else hi = mid;
    }
    *span = sequence_span(b, n_rows, lo);
    return row >= span->row0 && row - span->row0 < span->rows ? static_cast<int32_t>(lo) : -1;
}

// The page that holds a slot, or -1 where the table names none of the cache's pages. 0 <= slot < table_stride pages.
JFH_HOST_DEVICE int32_t page_of(const Cache& c, const Batch& b, uint32_t s, int32_t slot) {
    const int32_t p = b.table[static_cast<size_t>(s) * b.table_stride + (static_cast<uint32_t>(slot) >> c.page_shift)];
    return static_cast<uint32_t>(p) < c.n_pages ? p : -1;
}

JFH_HOST_DEVICE int32_t slot_in_page(const Cache& c, int32_t slot) {
    return slot & ((1 << c.page_shift) - 1);
}

// Offset (values) of a slot of head 0 in k and v.
JFH_HOST_DEVICE int64_t slot_offset(const Cache& c, int32_t page, int32_t slot) {
    return page * c.page_stride + slot_in_page(c, slot) * c.slot_stride;
}

// Offset of a slot in weights and positions.
JFH_HOST_DEVICE int64_t slot_index(const Cache& c, int32_t page, uint32_t head, int32_t slot) {
    return ((static_cast<int64_t>(page) * c.n_head_kv + head) << c.page_shift) + slot_in_page(c, slot);
}

// A rotation: turns per position of each pair (angle / 2 pi) and the size of the rotated values.
struct Rotation {
    double turns[kMaxRotPairs];
    float size;
    uint32_t n_rot, interleaved;
};

struct Attend {
    Cache cache;
    Batch batch;
    Rows q, out;
    float* lse;       // [rows][heads] or null
    float* partial;   // [splits][rows * heads][head_dim], unnormalized
    float* marks;     // [splits][rows * heads][2]: running maximum (base 2) and sum
    float scale_log2; // scale * log2(e)
    uint32_t causal, splits;
};

struct Weigh {
    Cache cache;
    Batch batch;
    Rows q;
    const float* lse;
    float* partial;  // [splits][sequences * K/V heads][max_length]
    float scale_log2;
    uint32_t causal, splits;
};

struct Evict {
    Cache cache;
    Batch batch;
    int32_t budget, first, recent;
    int32_t width;   // most positions that move
    int32_t* lists;  // per (sequence, K/V head): their number (-1: nothing is cut), to [width], from [width]
};

// Parts that a step's keys are divided into, each a work-group of its own per K/V head and tile of query rows; more than
// one where the tiles do not fill the chip.
uint32_t attend_splits(const Cache& c, const Batch& b, uint32_t group);

// Parts that a step's queries are divided into when their weights are added up.
uint32_t weigh_splits(const Cache& c, const Batch& b, uint32_t group);

hipError_t launch_rotate(const Rotation& r, const Rows& x, const int32_t* positions, const Rows& y, hipStream_t stream);
hipError_t launch_append(const Rotation* r, const Cache& c, const Batch& b, const Rows& k, const Rows& v,
                         const int32_t* positions, hipStream_t stream);
hipError_t launch_attend(const Attend& a, hipStream_t stream);
hipError_t launch_weigh(const Weigh& a, hipStream_t stream);
hipError_t launch_evict(const Evict& a, hipStream_t stream);

}  // namespace jfh::paged
