// C entry points of the paged-cache operators (include/jfh.h): argument checks, frequencies, launches.
#include "jfh_paged.hpp"

#include "jfh_status.hpp"

#include <algorithm>
#include <cmath>
#include <memory>

struct jfh_rope {
    jfh::paged::Rotation rotation;
};

namespace {

namespace paged = jfh::paged;

using jfh::capi::guarded;
using jfh::capi::require;

constexpr uint64_t kMaxIndex = 0x7FFFFFFF;

void check(hipError_t e, const char* what) {
    if (e == hipSuccess) return;
    (void) hipGetLastError();  // it is reported here: the next call's launch is not to find it
    if (e == hipErrorInvalidConfiguration) {
        throw jfh::Error(jfh::Status::InvalidArgument, std::string(what) + ": the step takes more threads than a launch holds");
    }
    throw jfh::Error(jfh::Status::DeviceError, std::string(what) + ": " + hipGetErrorString(e));
}

// The calling thread's device is `device` while this lives.
class OnDevice {
public:
    explicit OnDevice(int device) : device_(device) {
        check(hipGetDevice(&before_), "find the current device");
        if (before_ != device_) check(hipSetDevice(device_), "select the cache's device");
    }
    ~OnDevice() {
        if (before_ != device_) (void) hipSetDevice(before_);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;

private:
    int device_, before_ = 0;
};

bool aligned(const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

paged::Rows rows_of(const jfh_rows* x, const char* name) {
    const std::string n = name;
    require(x != nullptr, n + " rows are required");
    require(x->type >= JFH_VALUE_F32 && x->type <= JFH_VALUE_BF16, n + " rows have an unknown value type");
    require(x->n_rows <= kMaxIndex, n + " has more rows than a step can hold");
    require(x->n_head > 0 && x->n_head <= 65536 && x->head_dim > 0 && x->head_dim <= 65536,
            n + " rows have no heads, no values or too many");
    require(static_cast<uint64_t>(x->n_head) * x->head_dim <= 1U << 24, n + " rows hold too many values");
    require(x->row_stride >= 0 && x->head_stride >= 0, n + " rows have a negative stride");
    require(x->n_rows == 0 || (x->data != nullptr && aligned(x->data, x->type == JFH_VALUE_F32 ? 4 : 2)),
            n + " rows are missing or not aligned to their values");
    return paged::Rows{x->data, x->row_stride, x->head_stride, x->n_rows, x->n_head, x->head_dim, x->type};
}

// Rows that a call writes: each value has a place of its own, and the rows of the input are others or the same ones.
void written(const paged::Rows& x, const paged::Rows& out, const char* name) {
    const std::string n = name;
    // the larger stride passes over all that the smaller one reaches
    const bool by_rows = out.row_stride >= out.head_stride;
    const int64_t small = by_rows ? out.head_stride : out.row_stride, large = by_rows ? out.row_stride : out.head_stride;
    const int64_t inner = by_rows ? out.heads : out.rows, outer = by_rows ? out.rows : out.heads;
    const int64_t reach = static_cast<int64_t>(std::min<uint64_t>(static_cast<uint64_t>(small), 1ULL << 31)) * (inner - 1);
    require((inner <= 1 || small >= out.head_dim) && (outer <= 1 || large >= (inner <= 1 ? 0 : reach) + out.head_dim),
            n + "'s strides let its rows overlap");
    require(x.data != out.data || (x.type == out.type && x.row_stride == out.row_stride && x.head_stride == out.head_stride),
            "rows written in place must keep their type and strides");
}

paged::Cache cache_of(const jfh_paged_cache* c) {
    require(c != nullptr, "a cache is required");
    require(c->k && c->v && aligned(c->k, 16) && aligned(c->v, 16), "the cache's k and v must be 16-byte aligned");
    require(c->type == JFH_VALUE_F16 || c->type == JFH_VALUE_BF16, "a cache holds f16 or bf16 values");
    require(c->n_pages > 0 && c->n_pages <= kMaxIndex, "a cache needs pages");
    require(c->page_size > 0 && c->page_size <= paged::kMaxPageSize && (c->page_size & (c->page_size - 1)) == 0,
            "the page size must be a power of two up to 65536");
    require(c->n_head_kv > 0 && c->n_head_kv <= 65536, "a cache needs heads");
    require(c->head_dim >= 8 && c->head_dim <= paged::kMaxHeadDim && c->head_dim % 8 == 0,
            "the cache's head dim must be a multiple of 8 up to 256");
    require(c->page_stride % 8 == 0 && c->head_stride % 8 == 0 && c->slot_stride % 8 == 0 && c->page_stride >= 0 &&
                c->head_stride >= 0 && c->slot_stride >= 0,
            "the cache's strides must be multiples of 8 values");
    const int64_t dim = c->head_dim;
    require((c->page_size == 1 || c->slot_stride >= dim) && (c->n_head_kv == 1 || c->head_stride >= dim) &&
                (c->n_pages == 1 || c->page_stride >= dim),
            "the cache's strides let its rows overlap");
    require(aligned(c->weights, 4) && aligned(c->positions, 4), "the cache's weights and positions must be aligned");
    uint32_t shift = 0;
    while ((1U << shift) < c->page_size) ++shift;
    return paged::Cache{c->k, c->v, c->weights, c->positions, c->page_stride, c->head_stride, c->slot_stride,
                        c->n_pages, shift, c->n_head_kv, c->head_dim, c->type};
}

// A batch of a step of n_rows rows (no rows: of a call that looks at the sequences' slots alone).
paged::Batch batch_of(const jfh_paged_batch* b, const jfh_paged_cache& c, bool rows, uint32_t n_rows = 0) {
    require(b != nullptr, "a batch is required");
    require(b->n_seq <= 0xFFFFFF, "a batch holds at most 16777215 sequences");
    require(b->n_seq == 0 || (b->table && b->lengths && (b->row_starts || !rows)),
            "a batch needs its table, lengths and row starts");
    const uint64_t slots = static_cast<uint64_t>(b->table_stride) * c.page_size;
    require(b->max_length <= slots, "the batch's max_length exceeds its table");
    require(b->max_length <= paged::kMaxLength, "the batch's max_length exceeds 2^31 - 65537");
    require(b->max_rows <= kMaxIndex, "the batch's max_rows exceeds 2^31 - 1");
    return paged::Batch{b->table, b->lengths, b->row_starts, b->n_seq, b->table_stride,
                        std::min(b->max_rows, n_rows), b->max_length};
}

paged::Rotation rotation_of(const jfh_rope_params& p) {
    require(p.n_rot >= 2 && p.n_rot <= 2 * paged::kMaxRotPairs && p.n_rot % 2 == 0,
            "a rotation turns an even number of values, 2 to 256");
    require(p.layout <= JFH_ROPE_INTERLEAVED, "unknown rotation layout");
    require(p.scaling <= JFH_ROPE_YARN, "unknown rotation scaling");
    require(std::isfinite(p.base) && p.base > 1.0, "the rotation's base must be above 1");
    const bool scaled = p.scaling != JFH_ROPE_NONE;
    require(!scaled || (std::isfinite(p.factor) && p.factor >= 1.0), "the rotation's factor must be at least 1");
    require(p.scaling != JFH_ROPE_NTK || p.n_rot > 2, "this scaling needs more than one pair");
    const double n = p.n_rot, pi = std::acos(-1.0);
    double base = p.base, lo = 0.0, hi = 1.0;
    paged::Rotation r{};
    r.size = 1.0F;
    r.n_rot = p.n_rot;
    r.interleaved = p.layout == JFH_ROPE_INTERLEAVED ? 1U : 0U;
    if (p.scaling == JFH_ROPE_NTK) base *= std::pow(p.factor, n / (n - 2.0));
    if (p.scaling == JFH_ROPE_YARN) {
        require(p.original_context > 0 && std::isfinite(p.beta_fast) && std::isfinite(p.beta_slow) && p.beta_slow > 0.0 &&
                    p.beta_fast >= p.beta_slow,
                "this scaling needs the original context and beta_fast >= beta_slow > 0");
        require(std::isfinite(p.attention_factor) && p.attention_factor >= 0.0,
                "the attention factor must be 0 (by the factor) or above");
        // the pair that turns `turns` times over the original context
        const auto pair = [&](double turns) {
            return n * std::log(p.original_context / (turns * 2.0 * pi)) / (2.0 * std::log(p.base));
        };
        lo = std::max(std::floor(pair(p.beta_fast)), 0.0);
        hi = std::min(std::ceil(pair(p.beta_slow)), n - 1.0);
        r.size = static_cast<float>(p.attention_factor > 0.0 ? p.attention_factor : 0.1 * std::log(p.factor) + 1.0);
    }
    for (uint32_t i = 0; i < p.n_rot / 2; ++i) {
        double f = std::pow(base, -2.0 * i / n);
        if (p.scaling == JFH_ROPE_LINEAR) f /= p.factor;
        if (p.scaling == JFH_ROPE_YARN) {
            const double far = std::clamp((i - lo) / std::max(hi - lo, 1e-3), 0.0, 1.0);
            f = f * (1.0 - far) + f / p.factor * far;
        }
        r.turns[i] = f / (2.0 * pi);
    }
    return r;
}

// Rows that attention reads or writes: the cache's type and head dim, in steps of 16 bytes.
paged::Rows attended(const jfh_rows* x, const paged::Cache& c, const char* name) {
    const paged::Rows r = rows_of(x, name);
    const std::string n = name;
    require(r.type == c.type && r.head_dim == c.head_dim, n + " must have the cache's type and head dim");
    require(r.heads % c.n_head_kv == 0, n + "'s heads must be a multiple of the cache's");
    require(aligned(r.data, 16) && r.row_stride % 8 == 0 && r.head_stride % 8 == 0,
            n + " must be 16-byte aligned, with strides in multiples of 8 values");
    require(static_cast<uint64_t>(r.rows) * r.heads <= kMaxIndex / 2, n + " has more rows than a step can hold");
    return r;
}

float score_scale(float scale) {
    require(std::isfinite(scale) && scale > 0.0F, "the score scale must be above 0");
    const float base2 = static_cast<float>(static_cast<double>(scale) / std::log(2.0));
    require(std::isfinite(base2), "the score scale is too large");
    return base2;
}

struct AttendPlan {
    uint32_t splits;
    size_t partial, marks;  // bytes
};

AttendPlan attend_plan(const paged::Cache& c, const paged::Batch& b, const paged::Rows& q) {
    AttendPlan p{b.n_seq ? paged::attend_splits(c, b, q.heads / c.n_head_kv) : 1, 0, 0};
    if (p.splits > 1) {
        const size_t n = static_cast<size_t>(p.splits) * q.rows * q.heads;
        p.partial = n * c.head_dim * sizeof(float);
        p.marks = n * 2 * sizeof(float);
    }
    return p;
}

struct WeighPlan {
    uint32_t splits;
    size_t bytes;
};

WeighPlan weigh_plan(const paged::Cache& c, const paged::Batch& b, const paged::Rows& q) {
    WeighPlan p{b.n_seq ? paged::weigh_splits(c, b, q.heads / c.n_head_kv) : 1, 0};
    if (p.splits > 1) p.bytes = static_cast<size_t>(p.splits) * c.n_head_kv * b.n_seq * b.max_length * sizeof(float);
    return p;
}

// Most positions of a K/V head that move when sequences are cut, and the bytes of the lists that say which.
uint32_t evict_width(const paged::Batch& b, uint32_t budget) {
    return b.max_length > budget ? std::min(budget, b.max_length - budget) : 0;
}

size_t evict_bytes(const paged::Cache& c, const paged::Batch& b, uint32_t width) {
    return width ? static_cast<size_t>(b.n_seq) * c.n_head_kv * (1 + 2 * static_cast<size_t>(width)) * sizeof(int32_t) : 0;
}

void evicted(const paged::Cache& c, uint32_t budget) {
    require(c.weights && c.positions, "a cache that is cut needs weights and positions");
    require(budget > 0 && budget <= kMaxIndex, "a budget of at least one position is required");
}

}  // namespace

jfh_status jfh_rope_create(const jfh_rope_params* params, jfh_rope** out) {
    return guarded([&] {
        require(params && out, "rotation parameters and an output are required");
        *out = nullptr;
        *out = new jfh_rope{rotation_of(*params)};
    });
}

void jfh_rope_destroy(jfh_rope* rope) { delete rope; }

jfh_status jfh_rope_rotate(const jfh_rope* rope, const jfh_rows* x, const int32_t* positions, const jfh_rows* y,
                           int32_t device, void* stream) {
    return guarded([&] {
        require(rope != nullptr, "a rotation is required");
        const paged::Rows in = rows_of(x, "x"), out = rows_of(y, "y");
        require(in.rows == out.rows && in.heads == out.heads && in.head_dim == out.head_dim,
                "x and y must have the same rows, heads and head dim");
        require(rope->rotation.n_rot <= in.head_dim, "the rotation turns more values than a head has");
        if (in.rows == 0) return;
        written(in, out, "y");
        require(positions != nullptr && aligned(positions, 4), "positions are required");
        const OnDevice guard(device);
        check(paged::launch_rotate(rope->rotation, in, positions, out, static_cast<hipStream_t>(stream)), "rotate rows");
    });
}

jfh_status jfh_paged_append(const jfh_paged_cache* cache, const jfh_paged_batch* batch, const jfh_rows* k,
                            const jfh_rows* v, const jfh_rope* rope, const int32_t* positions, void* stream) {
    return guarded([&] {
        const paged::Cache c = cache_of(cache);
        const paged::Rows kr = rows_of(k, "k"), vr = rows_of(v, "v");
        const paged::Batch b = batch_of(batch, *cache, true, kr.rows);
        require(kr.rows == vr.rows, "k and v must have the same rows");
        require(kr.heads == c.n_head_kv && vr.heads == c.n_head_kv && kr.head_dim == c.head_dim && vr.head_dim == c.head_dim,
                "k and v must have the cache's heads and head dim");
        require(!rope || rope->rotation.n_rot <= c.head_dim, "the rotation turns more values than a head has");
        require((!rope && !c.positions) || positions, "positions are required with a rotation or cache positions");
        require(aligned(positions, 4), "positions must be aligned");
        if (kr.rows == 0 || b.n_seq == 0) return;
        const OnDevice guard(cache->device);
        check(paged::launch_append(rope ? &rope->rotation : nullptr, c, b, kr, vr, positions,
                                   static_cast<hipStream_t>(stream)),
              "append rows");
    });
}

jfh_status jfh_paged_attention_workspace(const jfh_paged_cache* cache, const jfh_paged_batch* batch, const jfh_rows* q,
                                         size_t* bytes) {
    return guarded([&] {
        require(bytes != nullptr, "an output for the workspace's size is required");
        const paged::Cache c = cache_of(cache);
        const paged::Rows x = attended(q, c, "q");
        const AttendPlan p = attend_plan(c, batch_of(batch, *cache, true, x.rows), x);
        *bytes = p.partial + p.marks;
    });
}

jfh_status jfh_paged_attention(const jfh_paged_cache* cache, const jfh_paged_batch* batch, const jfh_rows* q, float scale,
                               uint32_t causal, const jfh_rows* out, float* lse, void* workspace, size_t workspace_bytes,
                               void* stream) {
    return guarded([&] {
        paged::Attend a{};
        a.cache = cache_of(cache);
        a.q = attended(q, a.cache, "q");
        a.batch = batch_of(batch, *cache, true, a.q.rows);
        a.out = attended(out, a.cache, "out");
        require(a.q.rows == a.out.rows && a.q.heads == a.out.heads, "q and out must have the same rows and heads");
        if (a.q.rows > 0) written(a.q, a.out, "out");
        require(aligned(lse, 4), "lse must be aligned");
        a.lse = lse;
        a.scale_log2 = score_scale(scale);
        a.causal = causal ? 1U : 0U;
        if (a.q.rows == 0 || a.batch.n_seq == 0 || a.batch.max_rows == 0) return;
        const AttendPlan p = attend_plan(a.cache, a.batch, a.q);
        require(workspace_bytes >= p.partial + p.marks && (p.splits == 1 || workspace) && aligned(workspace, 16),
                "attention of this step needs " + std::to_string(p.partial + p.marks) +
                    " bytes of workspace, 16-byte aligned");
        a.splits = p.splits;
        a.partial = static_cast<float*>(workspace);
        a.marks = a.partial + p.partial / sizeof(float);
        const OnDevice guard(cache->device);
        check(paged::launch_attend(a, static_cast<hipStream_t>(stream)), "attention over pages");
    });
}

jfh_status jfh_paged_weigh_workspace(const jfh_paged_cache* cache, const jfh_paged_batch* batch, const jfh_rows* q,
                                     size_t* bytes) {
    return guarded([&] {
        require(bytes != nullptr, "an output for the workspace's size is required");
        const paged::Cache c = cache_of(cache);
        const paged::Rows x = attended(q, c, "q");
        *bytes = weigh_plan(c, batch_of(batch, *cache, true, x.rows), x).bytes;
    });
}

jfh_status jfh_paged_weigh(const jfh_paged_cache* cache, const jfh_paged_batch* batch, const jfh_rows* q, const float* lse,
                           float scale, uint32_t causal, void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&] {
        paged::Weigh a{};
        a.cache = cache_of(cache);
        require(a.cache.weights != nullptr, "the cache needs weights");
        a.q = attended(q, a.cache, "q");
        a.batch = batch_of(batch, *cache, true, a.q.rows);
        a.scale_log2 = score_scale(scale);
        a.causal = causal ? 1U : 0U;
        if (a.q.rows == 0 || a.batch.n_seq == 0 || a.batch.max_rows == 0 || a.batch.max_length == 0) return;
        require(lse != nullptr && aligned(lse, 4), "lse is required");
        a.lse = lse;
        const WeighPlan p = weigh_plan(a.cache, a.batch, a.q);
        require(workspace_bytes >= p.bytes && (p.splits == 1 || workspace) && aligned(workspace, 16),
                "weighing this step needs " + std::to_string(p.bytes) + " bytes of workspace, 16-byte aligned");
        a.splits = p.splits;
        a.partial = static_cast<float*>(workspace);
        const OnDevice guard(cache->device);
        check(paged::launch_weigh(a, static_cast<hipStream_t>(stream)), "weigh positions");
    });
}

jfh_status jfh_paged_evict_workspace(const jfh_paged_cache* cache, const jfh_paged_batch* batch, uint32_t budget,
                                     size_t* bytes) {
    return guarded([&] {
        require(bytes != nullptr, "an output for the workspace's size is required");
        const paged::Cache c = cache_of(cache);
        const paged::Batch b = batch_of(batch, *cache, false);
        evicted(c, budget);
        *bytes = evict_bytes(c, b, evict_width(b, budget));
    });
}

jfh_status jfh_paged_evict(const jfh_paged_cache* cache, const jfh_paged_batch* batch, uint32_t budget, uint32_t n_first,
                           uint32_t n_recent, void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&] {
        paged::Evict a{};
        a.cache = cache_of(cache);
        a.batch = batch_of(batch, *cache, false);
        evicted(a.cache, budget);
        require(n_first <= kMaxIndex && n_recent <= kMaxIndex, "more positions are protected than there can be");
        a.budget = static_cast<int32_t>(budget);
        a.first = static_cast<int32_t>(n_first);
        a.recent = static_cast<int32_t>(n_recent);
        a.width = static_cast<int32_t>(evict_width(a.batch, budget));
        if (a.width == 0 || a.batch.n_seq == 0) return;  // no sequence is longer
        const size_t need = evict_bytes(a.cache, a.batch, static_cast<uint32_t>(a.width));
        require(workspace && workspace_bytes >= need && aligned(workspace, 16),
                "cutting these sequences needs " + std::to_string(need) + " bytes of workspace, 16-byte aligned");
        a.lists = static_cast<int32_t*>(workspace);
        const OnDevice guard(cache->device);
        check(paged::launch_evict(a, static_cast<hipStream_t>(stream)), "cut sequences");
    });
}
