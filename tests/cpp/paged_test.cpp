// The index arithmetic of the paged-cache operators on the host: whatever a table, lengths or row starts hold, spans
// lie inside the step's rows and the table, and no page outside the cache is named.
#include "jfh_paged.hpp"

#include <climits>
#include <cstdio>
#include <random>
#include <vector>

namespace paged = jfh::paged;

namespace {

int failures = 0;

void expect(bool ok, const char* what) {
    if (ok) return;
    std::printf("FAIL %s\n", what);
    ++failures;
}

paged::Cache cache_of(uint32_t pages, uint32_t shift) {
    paged::Cache c{};
    c.n_pages = pages;
    c.page_shift = shift;
    c.n_head_kv = 3;
    c.head_dim = 64;
    c.slot_stride = 64;
    c.head_stride = 64LL << shift;
    c.page_stride = 3 * c.head_stride;
    return c;
}

void pages() {
    const std::vector<int32_t> table = {0, 4, -1, 5, INT_MAX, INT_MIN, 2, 3};
    const paged::Cache c = cache_of(5, 4);
    paged::Batch b{};
    b.table = table.data();
    b.n_seq = 2;
    b.table_stride = 4;
    const int32_t want[2][4] = {{0, 4, -1, -1}, {-1, -1, 2, 3}};
    for (uint32_t s = 0; s < 2; ++s) {
        for (int32_t t = 0; t < 64; ++t) {
            expect(paged::page_of(c, b, s, t) == want[s][t / 16], "page of a slot");
            expect(paged::slot_in_page(c, t) == t % 16, "place in the page");
        }
    }
    // the last value of the last page lies inside the pool
    expect(paged::slot_offset(c, 4, 15) + 2 * c.head_stride + 63 == 5 * c.page_stride - 1, "last value");
    expect(paged::slot_index(c, 4, 2, 15) == 5 * 3 * 16 - 1, "last weight");
    // offsets beyond 32 bits
    paged::Cache big = cache_of(1U << 20, 7);
    expect(paged::slot_offset(big, (1 << 20) - 1, 127) == ((1LL << 20) - 1) * 3 * 64 * 128 + 127 * 64, "wide offset");
}

void spans() {
    std::mt19937 rng(7);
    const uint32_t total = 50;
    for (int round = 0; round < 20000; ++round) {
        std::vector<int32_t> starts(5), lengths(4);
        for (auto& x : starts) x = round % 3 == 0 ? static_cast<int32_t>(rng()) : static_cast<int32_t>(rng() % 70) - 10;
        for (auto& x : lengths) x = round % 2 == 0 ? static_cast<int32_t>(rng()) : static_cast<int32_t>(rng() % 200) - 20;
        paged::Batch b{};
        b.lengths = lengths.data();
        b.row_starts = starts.data();
        b.n_seq = 4;
        b.max_rows = 1 + rng() % 60;
        b.max_length = rng() % 128;
        for (uint32_t s = 0; s < 4; ++s) {
            const paged::Span x = paged::sequence_span(b, total, s);
            expect(x.row0 >= 0 && x.rows >= 0 && x.row0 + x.rows <= static_cast<int32_t>(total), "rows inside the step");
            expect(x.rows <= static_cast<int32_t>(b.max_rows), "rows within their bound");
            expect(x.len >= 0 && x.len <= static_cast<int32_t>(b.max_length), "slots within their bound");
        }
        for (int32_t row = 0; row < static_cast<int32_t>(total); ++row) {
            paged::Span x{};
            const int32_t s = paged::sequence_of(b, total, row, &x);
            expect(s >= -1 && s < 4, "sequence of a row");
            if (s >= 0) expect(row >= x.row0 && row < x.row0 + x.rows, "row inside its sequence");
        }
    }
}

void rows() {
    // sequences 0 and 3 without rows, rows 9.. of none
    const std::vector<int32_t> starts = {0, 0, 4, 9, 9}, lengths = {8, 4, 20, 1};
    paged::Batch b{};
    b.lengths = const_cast<int32_t*>(lengths.data());
    b.row_starts = starts.data();
    b.n_seq = 4;
    b.max_rows = 5;
    b.max_length = 20;
    for (int32_t row = 0; row < 12; ++row) {
        paged::Span x{};
        expect(paged::sequence_of(b, 12, row, &x) == (row < 4 ? 1 : row < 9 ? 2 : -1), "sequence of a row");
    }
}

}  // namespace

int main() {
    pages();
    spans();
    rows();
    if (failures == 0) std::printf("paged tests passed\n");
    return failures ? 1 : 0;
}
