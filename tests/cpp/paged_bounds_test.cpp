// Spans of a step on the host: with rows and lengths beyond a batch's bounds the others keep their slots, and whatever the
// arrays hold, no sum leaves 32 bits.
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

// Row i of a sequence's n stands at slot length - n + i, if it is below max_rows and the slot below max_length.
void kept_rows_keep_their_slots() {
    std::mt19937 rng(11);
    for (int round = 0; round < 20000; ++round) {
        std::vector<int32_t> starts(1, 0), lengths;
        for (int s = 0; s < 3; ++s) {
            starts.push_back(starts.back() + static_cast<int32_t>(rng() % 9));
            lengths.push_back(round % 9 == 0 ? INT_MAX - static_cast<int32_t>(rng() % 5) : static_cast<int32_t>(rng() % 40));
        }
        paged::Batch b{};
        b.lengths = lengths.data();
        b.row_starts = starts.data();
        b.n_seq = 3;
        b.max_rows = rng() % 10;
        b.max_length = round % 11 == 0 ? INT_MAX - 1024 : rng() % 40;
        const uint32_t total = static_cast<uint32_t>(starts.back());
        for (uint32_t s = 0; s < 3; ++s) {
            const paged::Span x = paged::sequence_span(b, total, s);
            const int64_t n = starts[s + 1] - starts[s], most = b.max_length;
            expect(x.row0 == starts[s] && x.rows == (n < b.max_rows ? n : b.max_rows), "rows up to their bound");
            expect(x.len == (lengths[s] < most ? lengths[s] : most), "slots up to their bound");
            for (int32_t r = 0; r < x.rows; ++r) {
                const int64_t slot = static_cast<int64_t>(lengths[s]) - n + r;
                expect(slot < most ? x.first + r == slot : x.first + r >= most, "slot of a row");
                const int64_t sees = slot + 1 < 0 ? 0 : slot + 1 < x.len ? slot + 1 : x.len;
                expect(paged::slots_seen(x, r) == sees, "slots that a row sees");
            }
            for (int32_t t = 0; t < x.len && t < 64; ++t) {
                int32_t before = 0;
                while (before < x.rows && paged::slots_seen(x, before) <= t) ++before;
                expect(paged::rows_before(x, t) == before, "rows before a slot");
            }
        }
    }
}

void sums_stay_in_32_bits() {
    const int32_t odd[] = {INT_MIN, INT_MIN + 1, -7, -1, 0, 1, 5, 50, INT_MAX - 1, INT_MAX};
    for (int32_t length : odd) {
        for (int32_t start : odd) {
            for (int32_t end : odd) {
                for (uint32_t total : {0U, 1U, 50U, 0x7FFFFFFFU}) {
                    for (uint32_t max_length : {0U, 9U, 0x7FFFFFFFU - 1024U}) {
                        std::vector<int32_t> starts = {start, end}, lengths = {length};
                        paged::Batch b{};
                        b.lengths = lengths.data();
                        b.row_starts = starts.data();
                        b.n_seq = 1;
                        b.max_rows = total;
                        b.max_length = max_length;
                        const paged::Span x = paged::sequence_span(b, total, 0);
                        const int64_t last = static_cast<int64_t>(x.first) + x.rows;
                        expect(x.rows >= 0 && x.row0 >= 0 && x.row0 + static_cast<int64_t>(x.rows) <= total, "rows inside the step");
                        expect(x.len >= 0 && x.len <= static_cast<int64_t>(max_length), "slots inside the table");
                        expect(x.rows == 0 || (last <= INT_MAX && x.first >= -INT_MAX), "first slot");
                        const int32_t before = paged::rows_before(x, x.len);
                        expect(before >= 0 && before <= x.rows, "rows before a slot");
                        if (x.rows > 0) expect(paged::slots_seen(x, x.rows - 1) <= x.len, "slots that a row sees");
                    }
                }
            }
        }
    }
}

}  // namespace

int main() {
    kept_rows_keep_their_slots();
    sums_stay_in_32_bits();
    if (failures == 0) std::printf("paged bounds tests passed\n");
    return failures ? 1 : 0;
}
