// The entry points of include/dci_hip.h that work on tokens: checks of the arguments, the caller's
// workspace laid out, launches.  No handle, no state; nothing here allocates, waits or throws.
#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <string>

#include "../../include/dci_hip.h"
#include "clip.h"
#include "scan.h"
#include "token_common.h"
#include "verify.h"

namespace dcih {
namespace {

constexpr int64_t kMaxCount = 0x7fffffff;      // ids, rows of a table

bool aligned(const void* p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

// What is wrong with an array of elements, null where nothing is.
const char* check_array(const void* p, int dtype) {
    if (!type_bytes(dtype)) return "unknown element type";
    if (!p) return "null array";
    return aligned(p, type_bytes(dtype)) ? nullptr : "array not aligned to its elements";
}

const char* check_ids(const void* p, int id_bytes) {
    if (id_bytes != 4 && id_bytes != 8) return "ids are of 4 or 8 bytes";
    if (!p) return "null ids";
    return aligned(p, id_bytes) ? nullptr : "ids not aligned to their size";
}

// Rows whose last byte has an address in 63 bits.
bool near_enough(int64_t n, int64_t stride) { return stride <= (INT64_MAX >> 4) / std::max<int64_t>(n, 1); }

bool all_aligned(std::initializer_list<const void*> arrays) {
    for (const void* p : arrays)
        if (!aligned(p, 4)) return false;
    return true;
}

int refuse(const char* who, const char* why) { return fail(DCIH_EINVAL, std::string(who) + ": " + why); }

const char* check_logits(const void* z, int dtype, int64_t n, int vocab, int64_t stride, float temperature) {
    if (const char* why = check_array(z, dtype)) return why;
    if (n < 0 || n > kMaxCount) return "bad number of rows";
    if (vocab <= 0 || vocab > DCIH_MAX_VOCAB) return "bad length of rows";
    if (stride < vocab || !near_enough(n, stride)) return "rows overlap or are too far apart";
    if (!(temperature > 1e-30f) || !(temperature < 1e30f)) return "temperature must be a positive number";
    return nullptr;
}

LogitArgs logit_args(const void* z, int dtype, int64_t n, int vocab, int64_t stride, float temperature, const void* ids, int id_bytes) {
    LogitArgs a{};
    a.z = z;
    a.n = n;
    a.stride = stride;
    a.vocab = vocab;
    a.inv_t = 1.f / temperature;
    a.half_t = 0.5f * temperature;
    const double c2 = 1.44269504088896340736 / (double)temperature;
    a.c2 = (float)c2;
    a.c2_rest = (float)(c2 - (double)a.c2);
    a.ids = ids;
    a.wide_ids = id_bytes == 8;
    a.splits = n ? logit_splits(n, vocab, dtype) : 1;
    return a;
}

// Workspace of a call on rows that are split: statistics and best entries of the splits, behind
// them the rows' statistics for a gradient formed by the same call.
int64_t part_bytes(const LogitArgs& a) { return a.splits > 1 ? a.n * a.splits * 16 : 0; }
int64_t part_top_bytes(const LogitArgs& a, int top) { return a.splits > 1 ? (a.n * a.splits * top * 8 + 15) / 16 * 16 : 0; }

const char* lay_out(LogitArgs& a, int top, bool stats, void* work, int64_t bytes) {
    const int64_t p = part_bytes(a), t = part_top_bytes(a, top), need = p + t + (stats ? a.n * 16 : 0);
    if (!need) return nullptr;
    if (!work || bytes < need) return "workspace too small";
    if (!aligned(work, 16)) return "workspace not aligned to 16 bytes";
    a.part = (float4*)work;
    a.part_top = (unsigned long long*)((char*)work + p);
    if (stats) a.stats = (float4*)((char*)work + p + t);
    return nullptr;
}

bool overlap(const void* a, int64_t bytes_a, const void* b, int64_t bytes_b) {
    return (uintptr_t)a < (uintptr_t)b + (uintptr_t)bytes_b && (uintptr_t)b < (uintptr_t)a + (uintptr_t)bytes_a;
}

// A gradient in the logits' place is of the same rows; anything between is refused.
const char* check_grad(const void* z, const void* grad, int dtype, int64_t n, int vocab, int64_t stride, int64_t grad_stride) {
    if (const char* why = check_array(grad, dtype)) return why;
    if (grad_stride < vocab || !near_enough(n, grad_stride)) return "rows of the gradient overlap or are too far apart";
    const int64_t b = type_bytes(dtype);
    if (n && !(z == grad && stride == grad_stride) &&
        overlap(z, ((n - 1) * stride + vocab) * b, grad, ((n - 1) * grad_stride + vocab) * b))
        return "the gradient overlaps the logits without being in their place";
    return nullptr;
}

const char* check_teacher(const void* teacher, int teacher_dtype, int slots, const void* ids, int id_bytes) {
    if (slots <= 0 || slots > kTeacherSlots) return "bad number of slots";
    if (const char* why = check_ids(ids, id_bytes)) return why;
    return check_array(teacher, teacher_dtype);
}

// Tokens of a scan: rows, length and dim that are in bounds, and addresses in 63 bits.
const char* check_scan_size(int64_t rows, int64_t length, int dim, int dtype, int64_t packed) {
    if (!type_bytes(dtype)) return "unknown element type";
    if (rows < 0 || rows > kMaxCount || length < 0 || length > kMaxCount || dim <= 0 || dim > DCIH_MAX_DIM || packed < 0 || packed > kMaxCount)
        return "bad size";
    if (packed && rows != 1) return "packed sequences are one row of tokens";
    if (!near_enough(rows * std::max<int64_t>(length, 1), dim)) return "too many tokens";
    return nullptr;
}

// Elements from the first of [rows][length][dim] to behind the last.
int64_t scan_extent(int64_t rows, int64_t length, int dim, int64_t row, int64_t step) { return (rows - 1) * row + (length - 1) * step + dim; }

const char* scan_args(ScanArgs& a, const void* x, int dtype, int64_t rows, int64_t length, int dim, int64_t x_row, int64_t x_step,
                      const void* gates, int64_t g_row, int64_t g_step, int flags, const float* state, const void* bounds, int id_bytes,
                      int64_t packed) {
    if (const char* why = check_scan_size(rows, length, dim, dtype, packed)) return why;
    if (flags & ~(DCIH_SCAN_DECAYS | DCIH_SCAN_SHARED)) return "unknown flags";
    if (packed && !bounds) return "packed sequences need offsets";
    if (bounds)
        if (const char* why = check_ids(bounds, id_bytes)) return why;
    if (!all_aligned({state})) return "states not aligned to their elements";
    a.shared = (flags & DCIH_SCAN_SHARED) != 0;
    if (rows && length) {
        if (const char* why = check_array(x, dtype)) return why;
        if (const char* why = check_array(gates, dtype)) return why;
        if (a.shared) g_row = g_step = 0;
        if (x_row < 0 || x_step < 0 || g_row < 0 || g_step < 0) return "distances are not negative";
        if (!near_enough(rows, std::max(x_row, g_row)) || !near_enough(length, std::max(x_step, g_step))) return "tokens are too far apart";
    }
    a.x = x;
    a.gates = gates;
    a.x_row = x_row;
    a.x_step = x_step;
    a.g_row = g_row;
    a.g_step = g_step;
    a.rows = rows;
    a.length = length;
    a.sequences = packed ? packed : rows;
    a.dim = dim;
    a.form = packed ? kPacked : kRows;
    a.decay = (flags & DCIH_SCAN_DECAYS) != 0;
    a.state = state;
    a.bounds = bounds;
    a.wide_bounds = id_bytes == 8;
    return nullptr;
}

const char* check_spans(const dcih_span* spans, int64_t n, bool written) {
    if (n < 0 || n > kMaxCount || (n && !spans)) return "bad number of spans";
    for (int64_t i = 0; i < n; i++) {
        const dcih_span& p = spans[i];
        if (p.count < 0 || p.count > INT64_MAX >> 8) return "bad length of a span";
        if (!p.count) continue;
        if (const char* why = check_array(p.data, p.dtype)) return why;
        if (!written) continue;
        if (const char* why = check_array(p.out, p.out_dtype)) return why;
        if (p.out_dtype != p.dtype && p.out_dtype != DCIH_F32) return "what is written is of the span's type or of 32 bits";
        if (!(p.out == p.data && p.out_dtype == p.dtype) && overlap(p.data, p.count * type_bytes(p.dtype), p.out, p.count * type_bytes(p.out_dtype)))
            return "what is written overlaps the span without being in its place";
    }
    return clip_fits(spans, n) ? nullptr : "too many elements";
}

const char* check_clip(const dcih_span* spans, int64_t n, bool written, double scale, const float* norm, const void* work, int64_t bytes) {
    if (const char* why = check_spans(spans, n, written)) return why;
    if (!std::isfinite(scale)) return "scale must be a finite number";
    if (!norm || !aligned(norm, 4)) return "no place for the norm";
    if (!work || bytes < clip_work_bytes(spans, n)) return "workspace too small";
    return aligned(work, 16) ? nullptr : "workspace not aligned to 16 bytes";
}

// What a call reads or writes; null where nothing was given.
struct Range {
    const void* p;
    int64_t bytes;
    bool meets(const Range& o) const { return p && o.p && bytes > 0 && o.bytes > 0 && overlap(p, bytes, o.p, o.bytes); }
};

// Whether something that is written lies over something that is read, or over something else that is written.  (Workgroups, and lanes that share a
// row's last piece, read what others have written by then.)
bool any_meets(std::initializer_list<Range> written, std::initializer_list<Range> read) {
    for (const Range* w = written.begin(); w != written.end(); w++) {
        for (const Range& r : read)
            if (w->meets(r)) return true;
        for (const Range* o = w + 1; o != written.end(); o++)
            if (w->meets(*o)) return true;
    }
    return false;
}

Range bounds_range(const ScanArgs& a) { return {a.bounds, (a.sequences + (a.form == kPacked)) * (a.wide_bounds ? 8 : 4)}; }

// States in their own place: where one thread does not have a channel from first to last, the new ones wait in the workspace.
int64_t last_bytes(int64_t sequences, int dim) { return (sequences * dim * 4 + 255) / 256 * 256; }

}  // namespace
}  // namespace dcih

using namespace dcih;

extern "C" {

int dcih_embed(const void* d_table, int dtype, int64_t num_rows, int dim, int64_t row_stride, const void* d_ids,
               int id_bytes, int64_t num_ids, float scale, void* d_out, void* stream) {
    const char* who = "dcih_embed";
    if (num_rows <= 0 || num_rows > kMaxCount || dim <= 0 || dim > DCIH_MAX_DIM || row_stride < dim || num_ids < 0 || num_ids > kMaxCount ||
        !near_enough(num_rows, row_stride))
        return refuse(who, "bad size");
    if (const char* why = check_array(d_table, dtype)) return refuse(who, why);
    if (!num_ids) return DCIH_OK;
    if (const char* why = check_ids(d_ids, id_bytes)) return refuse(who, why);
    if (const char* why = check_array(d_out, dtype)) return refuse(who, why);
    EmbedArgs a{};
    a.rows = d_table;
    a.num_rows = num_rows;
    a.stride = row_stride;
    a.dim = dim;
    a.ids = d_ids;
    a.wide_ids = id_bytes == 8;
    a.n = num_ids;
    a.scale = scale;
    a.out = d_out;
    return embed_rows(a, dtype, (hipStream_t)stream);
}

int64_t dcih_embed_grad_work(int64_t num_ids, int dim, int64_t num_rows) {
    if (num_ids < 0 || num_ids > kMaxCount || dim <= 0 || dim > DCIH_MAX_DIM || num_rows <= 0 || num_rows > kMaxCount) return refuse("dcih_embed_grad_work", "bad size");
    return (int64_t)embed_grad_bytes(num_ids, dim, num_rows);
}

int dcih_embed_grad(const void* d_grad, int dtype, int64_t num_ids, int dim, int64_t row_stride, const void* d_ids,
                    int id_bytes, int64_t num_rows, float scale, int accumulate, void* d_out, int out_dtype,
                    void* d_work, int64_t work_bytes, void* stream) {
    const char* who = "dcih_embed_grad";
    if (num_rows <= 0 || num_rows > kMaxCount || dim <= 0 || dim > DCIH_MAX_DIM || row_stride < dim || num_ids < 0 || num_ids > kMaxCount ||
        !near_enough(num_ids, row_stride))
        return refuse(who, "bad size");
    if (const char* why = check_array(d_out, out_dtype)) return refuse(who, why);
    if (out_dtype != dtype && out_dtype != DCIH_F32) return refuse(who, "sums are of the gradient's type or of 32 bits");
    if (num_ids) {
        if (const char* why = check_array(d_grad, dtype)) return refuse(who, why);
        if (const char* why = check_ids(d_ids, id_bytes)) return refuse(who, why);
    }
    if (!d_work || work_bytes < (int64_t)embed_grad_bytes(num_ids, dim, num_rows)) return refuse(who, "workspace too small");
    if (!aligned(d_work, 16)) return refuse(who, "workspace not aligned to 16 bytes");
    EmbedArgs a{};
    a.rows = d_grad;
    a.num_rows = num_rows;
    a.stride = row_stride;
    a.dim = dim;
    a.ids = d_ids;
    a.wide_ids = id_bytes == 8;
    a.n = num_ids;
    a.scale = scale;
    a.out = d_out;
    a.accumulate = accumulate != 0;
    a.work = d_work;
    return embed_grad(a, dtype, out_dtype, (hipStream_t)stream);
}

int64_t dcih_logits_work(int64_t num_rows, int vocab, int dtype, int top) {
    if (num_rows < 0 || num_rows > kMaxCount || vocab <= 0 || vocab > DCIH_MAX_VOCAB || !type_bytes(dtype) || top < 0 || top > kMaxTop)
        return refuse("dcih_logits_work", "bad argument");
    const LogitArgs a = logit_args(nullptr, dtype, num_rows, vocab, vocab, 1.f, nullptr, 4);
    return part_bytes(a) + part_top_bytes(a, top) + num_rows * 16;
}

int dcih_token_logprobs(const void* d_logits, int dtype, int64_t num_rows, int vocab, int64_t row_stride, const void* d_targets,
                        int id_bytes, float temperature, int top, float* d_logprobs, float* d_entropy, int32_t* d_top_ids,
                        float* d_top_logprobs, float* d_stats, void* d_work, int64_t work_bytes, void* stream) {
    const char* who = "dcih_token_logprobs";
    if (const char* why = check_logits(d_logits, dtype, num_rows, vocab, row_stride, temperature)) return refuse(who, why);
    if (top < 0 || top > kMaxTop || top > vocab) return refuse(who, "bad number of alternatives");
    if (!num_rows) return DCIH_OK;
    if (const char* why = check_ids(d_targets, id_bytes)) return refuse(who, why);
    if (!d_logprobs || !d_entropy || (top && (!d_top_ids || !d_top_logprobs))) return refuse(who, "null array");
    if (d_stats && !aligned(d_stats, 16)) return refuse(who, "statistics not aligned to 16 bytes");
    if (!all_aligned({d_logprobs, d_entropy, d_top_ids, d_top_logprobs})) return refuse(who, "results not aligned to their elements");
    LogitArgs a = logit_args(d_logits, dtype, num_rows, vocab, row_stride, temperature, d_targets, id_bytes);
    if (const char* why = lay_out(a, top, false, d_work, work_bytes)) return refuse(who, why);
    a.top = top;
    a.logprobs = d_logprobs;
    a.entropy = d_entropy;
    a.top_ids = d_top_ids;
    a.top_logprobs = d_top_logprobs;
    a.stats = (float4*)d_stats;
    return logit_stats(a, dtype, false, (hipStream_t)stream);
}

int dcih_token_logprobs_grad(const void* d_logits, int dtype, int64_t num_rows, int vocab, int64_t row_stride,
                             const void* d_targets, int id_bytes, float temperature, const float* d_stats,
                             const float* d_grad_logprobs, const float* d_grad_entropy, void* d_grad, int64_t grad_stride,
                             void* stream) {
    const char* who = "dcih_token_logprobs_grad";
    if (const char* why = check_logits(d_logits, dtype, num_rows, vocab, row_stride, temperature)) return refuse(who, why);
    if (!num_rows) return DCIH_OK;
    if (const char* why = check_ids(d_targets, id_bytes)) return refuse(who, why);
    if (!d_stats || !aligned(d_stats, 16)) return refuse(who, "statistics missing or not aligned to 16 bytes");
    if (const char* why = check_grad(d_logits, d_grad, dtype, num_rows, vocab, row_stride, grad_stride)) return refuse(who, why);
    LogitArgs a = logit_args(d_logits, dtype, num_rows, vocab, row_stride, temperature, d_targets, id_bytes);
    if (!all_aligned({d_grad_logprobs, d_grad_entropy})) return refuse(who, "factors not aligned to their elements");
    a.stats = (float4*)d_stats;
    a.grad_logprobs = d_grad_logprobs;
    a.grad_entropy = d_grad_entropy;
    a.grad = d_grad;
    a.grad_stride = grad_stride;
    return logit_grad(a, dtype, false, (hipStream_t)stream);
}

int dcih_distill(const void* d_logits, int dtype, int64_t num_rows, int vocab, int64_t row_stride, const void* d_ids,
                 int id_bytes, const void* d_teacher, int teacher_dtype, int slots, float temperature, float* d_losses,
                 float* d_stats, const float* d_weights, void* d_grad, int64_t grad_stride, void* d_work, int64_t work_bytes,
                 void* stream) {
    const char* who = "dcih_distill";
    if (const char* why = check_logits(d_logits, dtype, num_rows, vocab, row_stride, temperature)) return refuse(who, why);
    if (!num_rows) return DCIH_OK;
    if (const char* why = check_teacher(d_teacher, teacher_dtype, slots, d_ids, id_bytes)) return refuse(who, why);
    if (!d_losses) return refuse(who, "null array");
    if (!all_aligned({d_losses, d_weights})) return refuse(who, "losses or weights not aligned to their elements");
    if (d_stats && !aligned(d_stats, 16)) return refuse(who, "statistics not aligned to 16 bytes");
    if (d_grad)
        if (const char* why = check_grad(d_logits, d_grad, dtype, num_rows, vocab, row_stride, grad_stride)) return refuse(who, why);
    LogitArgs a = logit_args(d_logits, dtype, num_rows, vocab, row_stride, temperature, d_ids, id_bytes);
    if (const char* why = lay_out(a, 0, d_grad && !d_stats, d_work, work_bytes)) return refuse(who, why);
    if (d_stats) a.stats = (float4*)d_stats;
    a.teacher = d_teacher;
    a.teacher_dtype = teacher_dtype;
    a.slots = slots;
    a.losses = d_losses;
    a.weights = d_weights;
    a.grad = d_grad;
    a.grad_stride = grad_stride;
    if (d_grad && distill_by_rows(a, dtype)) {
        a.stats = (float4*)d_stats;
        return distill_rows(a, dtype, (hipStream_t)stream);
    }
    if (int rc = logit_stats(a, dtype, true, (hipStream_t)stream)) return rc;
    return d_grad ? logit_grad(a, dtype, true, (hipStream_t)stream) : DCIH_OK;
}

int dcih_distill_grad(const void* d_logits, int dtype, int64_t num_rows, int vocab, int64_t row_stride, const void* d_ids,
                      int id_bytes, const void* d_teacher, int teacher_dtype, int slots, float temperature,
                      const float* d_stats, const float* d_weights, void* d_grad, int64_t grad_stride, void* stream) {
    const char* who = "dcih_distill_grad";
    if (const char* why = check_logits(d_logits, dtype, num_rows, vocab, row_stride, temperature)) return refuse(who, why);
    if (!num_rows) return DCIH_OK;
    if (const char* why = check_teacher(d_teacher, teacher_dtype, slots, d_ids, id_bytes)) return refuse(who, why);
    if (!d_stats || !aligned(d_stats, 16)) return refuse(who, "statistics missing or not aligned to 16 bytes");
    if (const char* why = check_grad(d_logits, d_grad, dtype, num_rows, vocab, row_stride, grad_stride)) return refuse(who, why);
    LogitArgs a = logit_args(d_logits, dtype, num_rows, vocab, row_stride, temperature, d_ids, id_bytes);
    a.stats = (float4*)d_stats;
    a.teacher = d_teacher;
    a.teacher_dtype = teacher_dtype;
    if (!all_aligned({d_weights})) return refuse(who, "weights not aligned to their elements");
    a.slots = slots;
    a.weights = d_weights;
    a.grad = d_grad;
    a.grad_stride = grad_stride;
    return logit_grad(a, dtype, true, (hipStream_t)stream);
}

int64_t dcih_scan_states(int64_t rows, int64_t length, int dim, int dtype) {
    if (const char* why = check_scan_size(rows, length, dim, dtype, 0)) return refuse("dcih_scan_states", why);
    return scan_state_floats(rows, length, dim, dtype);
}

int64_t dcih_scan_work(int64_t rows, int64_t length, int dim, int dtype, int64_t packed_sequences) {
    if (const char* why = check_scan_size(rows, length, dim, dtype, packed_sequences)) return refuse("dcih_scan_work", why);
    return scan_work_bytes(rows, length, dim, dtype) + last_bytes(packed_sequences ? packed_sequences : rows, dim);
}

int dcih_scan(const void* d_x, int dtype, int64_t rows, int64_t length, int dim, int64_t x_row, int64_t x_step, const void* d_gates,
              int64_t g_row, int64_t g_step, int flags, const float* d_state, const void* d_bounds, int id_bytes,
              int64_t packed_sequences, void* d_h, float* d_last, float* d_states, void* d_work, int64_t work_bytes, void* stream) {
    const char* who = "dcih_scan";
    hipStream_t s = (hipStream_t)stream;
    ScanArgs a{};
    if (const char* why = scan_args(a, d_x, dtype, rows, length, dim, x_row, x_step, d_gates, g_row, g_step, flags, d_state, d_bounds, id_bytes, packed_sequences))
        return refuse(who, why);
    if (!all_aligned({d_last, d_states})) return refuse(who, "states not aligned to their elements");
    const int64_t states = a.sequences * dim;
    if (d_last && d_state && d_last != d_state && overlap(d_last, states * 4, d_state, states * 4))
        return refuse(who, "the last states overlap the first without being in their place");
    if (!rows || !length) return d_last && d_last != d_state && states ? scan_copy(d_state, d_last, states, s) : DCIH_OK;
    if (const char* why = check_array(d_h, dtype)) return refuse(who, why);
    const int64_t b = type_bytes(dtype), h_bytes = rows * length * dim * b;
    if (overlap(d_h, h_bytes, d_x, scan_extent(rows, length, dim, x_row, x_step) * b) ||
        overlap(d_h, h_bytes, d_gates, scan_extent(rows, length, dim, a.g_row, a.g_step) * b))
        return refuse(who, "h overlaps x or the gates");
    if (d_last && (overlap(d_last, states * 4, d_h, h_bytes) || overlap(d_last, states * 4, d_x, scan_extent(rows, length, dim, x_row, x_step) * b) ||
                   overlap(d_last, states * 4, d_gates, scan_extent(rows, length, dim, a.g_row, a.g_step) * b)))
        return refuse(who, "the last states overlap x, the gates or h");
    const Range first{d_state, states * 4}, bounds = bounds_range(a), kept{d_states, scan_state_floats(rows, length, dim, dtype) * 4};
    if (any_meets({{d_h, h_bytes}, kept}, {first, bounds, {d_x, scan_extent(rows, length, dim, x_row, x_step) * b}, {d_gates, scan_extent(rows, length, dim, a.g_row, a.g_step) * b}}) ||
        any_meets({{d_last, states * 4}}, {bounds, kept}))
        return refuse(who, "something that is written overlaps something else");
    const int64_t own = scan_work_bytes(rows, length, dim, dtype);
    if (work_bytes < own + last_bytes(a.sequences, dim) || !d_work) return refuse(who, "workspace too small");
    if (!aligned(d_work, 16)) return refuse(who, "workspace not aligned to 16 bytes");
    a.h = d_h;
    a.last = d_last;
    a.states = d_states;
    a.work = d_work;
    const bool waits = d_last && d_last == d_state && !scan_is_short(a, dtype);
    if (waits) a.last = (float*)((char*)d_work + own);
    if (int rc = scan(a, dtype, s)) return rc;
    return waits ? scan_copy(a.last, d_last, states, s) : DCIH_OK;
}

int dcih_scan_grad(const void* d_x, int dtype, int64_t rows, int64_t length, int dim, int64_t x_row, int64_t x_step, const void* d_gates,
                   int64_t g_row, int64_t g_step, int flags, const float* d_state, const void* d_bounds, int id_bytes,
                   int64_t packed_sequences, const float* d_states, const void* d_dh, const float* d_dlast, void* d_dx, void* d_dgates,
                   float* d_dstate, void* d_work, int64_t work_bytes, void* stream) {
    const char* who = "dcih_scan_grad";
    hipStream_t s = (hipStream_t)stream;
    ScanArgs a{};
    if (const char* why = scan_args(a, d_x, dtype, rows, length, dim, x_row, x_step, d_gates, g_row, g_step, flags, d_state, d_bounds, id_bytes, packed_sequences))
        return refuse(who, why);
    if (!all_aligned({d_states, d_dlast, d_dstate})) return refuse(who, "states not aligned to their elements");
    if (!aligned(d_dh, type_bytes(dtype)) || !aligned(d_dx, type_bytes(dtype)) || !aligned(d_dgates, type_bytes(dtype)))
        return refuse(who, "gradients not aligned to their elements");
    const int64_t b = type_bytes(dtype), states = a.sequences * dim, cells = rows * length * dim * b;
    if (any_meets({{d_dstate, states * 4}}, {{d_dlast, states * 4}, {d_state, states * 4}, bounds_range(a)}))
        return refuse(who, "the gradient by the first states overlaps what it is formed from");
    if (!rows || !length) {
        if (a.shared && d_dgates) return refuse(who, "no tokens to sum a shared gate's gradient over");
        return d_dstate && states ? scan_copy(d_dlast, d_dstate, states, s) : DCIH_OK;
    }
    if (!d_states) return refuse(who, "null array");
    if (any_meets({{d_dx, cells}, {d_dgates, a.shared ? dim * b : cells}, {d_dstate, states * 4}},
                  {{d_x, scan_extent(rows, length, dim, x_row, x_step) * b},
                   {d_gates, scan_extent(rows, length, dim, a.g_row, a.g_step) * b},
                   {d_dh, cells},
                   {d_dlast, states * 4},
                   {d_state, states * 4},
                   {d_states, scan_state_floats(rows, length, dim, dtype) * 4},
                   bounds_range(a)}))
        return refuse(who, "a gradient overlaps another one, or what it is formed from");
    if (work_bytes < scan_work_bytes(rows, length, dim, dtype) + last_bytes(a.sequences, dim) || !d_work) return refuse(who, "workspace too small");
    if (!aligned(d_work, 16)) return refuse(who, "workspace not aligned to 16 bytes");
    a.states = const_cast<float*>(d_states);
    a.dh = d_dh;
    a.dlast = d_dlast;
    a.dx = d_dx;
    a.dgates = d_dgates;
    a.dstate = d_dstate;
    a.work = d_work;
    return scan_grad(a, dtype, s);
}

int64_t dcih_clip_work(const dcih_span* spans, int64_t num_spans) {
    if (const char* why = check_spans(spans, num_spans, false)) return refuse("dcih_clip_work", why);
    return clip_work_bytes(spans, num_spans);
}

int dcih_grad_norm(const dcih_span* spans, int64_t num_spans, double scale, float* d_norm, void* d_work, int64_t work_bytes, void* stream) {
    if (const char* why = check_clip(spans, num_spans, false, scale, d_norm, d_work, work_bytes)) return refuse("dcih_grad_norm", why);
    return grad_norm(spans, num_spans, scale, d_norm, d_work, (hipStream_t)stream);
}

int dcih_clip(const dcih_span* spans, int64_t num_spans, double max_norm, double scale, float* d_norm, void* d_work, int64_t work_bytes,
              void* stream) {
    if (const char* why = check_clip(spans, num_spans, true, scale, d_norm, d_work, work_bytes)) return refuse("dcih_clip", why);
    if (!(max_norm >= 0.0)) return refuse("dcih_clip", "max_norm must not be negative");
    return clip_grads(spans, num_spans, max_norm, scale, d_norm, d_work, (hipStream_t)stream);
}

int64_t dcih_verify_work(int64_t num_sequences, int drafts, int vocab, int dtype) {
    if (num_sequences < 0 || drafts < 0 || drafts > kMaxDrafts || num_sequences > kMaxCount / (drafts + 1) || vocab <= 0 || vocab > DCIH_MAX_VOCAB ||
        !type_bytes(dtype))
        return refuse("dcih_verify_work", "bad argument");
    return verify_work_bytes(num_sequences * (drafts + 1), vocab, dtype);
}

int dcih_verify(const void* d_logits, int dtype, int64_t num_sequences, int drafts, int vocab, int64_t row_stride, const void* d_drafts,
                int id_bytes, const float* d_uniforms, const void* d_slot_ids, int slot_id_bytes, const void* d_teacher, int teacher_dtype,
                int slots, float temperature, int32_t* d_tokens, int32_t* d_accepted, float* d_logprobs, void* d_work, int64_t work_bytes,
                void* stream) {
    const char* who = "dcih_verify";
    if (drafts < 0 || drafts > kMaxDrafts) return refuse(who, "bad number of drafts");
    if (num_sequences < 0 || num_sequences > kMaxCount / (drafts + 1)) return refuse(who, "bad number of sequences");
    if (const char* why = check_logits(d_logits, dtype, num_sequences * (drafts + 1), vocab, row_stride, temperature)) return refuse(who, why);
    if (!num_sequences) return DCIH_OK;
    if (drafts)
        if (const char* why = check_ids(d_drafts, id_bytes)) return refuse(who, why);
    if (drafts && d_slot_ids)
        if (const char* why = check_teacher(d_teacher, teacher_dtype, slots, d_slot_ids, slot_id_bytes)) return refuse(who, why);
    if (!d_uniforms || !d_tokens || !d_accepted || !d_logprobs) return refuse(who, "null array");
    if (!all_aligned({d_uniforms, d_tokens, d_accepted, d_logprobs})) return refuse(who, "arrays not aligned to their elements");
    // (a sequence's random numbers are read before its log probabilities are written, by the same workgroup)
    const int64_t rows = num_sequences * (drafts + 1), slot_count = drafts && d_slot_ids ? num_sequences * drafts * slots : 0;
    if (any_meets({{d_tokens, rows * 4}, {d_accepted, num_sequences * 4}, {d_logprobs, rows * 4}},
                  {{d_logits, ((rows - 1) * row_stride + vocab) * type_bytes(dtype)},
                   {d_drafts, num_sequences * drafts * id_bytes},
                   {d_uniforms, (const void*)d_uniforms == d_logprobs ? 0 : rows * 4},
                   {d_slot_ids, slot_count * slot_id_bytes},
                   {d_teacher, slot_count * type_bytes(teacher_dtype)}}) ||
        any_meets({{d_tokens, rows * 4}, {d_accepted, num_sequences * 4}}, {{d_uniforms, rows * 4}}))
        return refuse(who, "something that is written overlaps something else");
    if (!d_work || work_bytes < verify_work_bytes(num_sequences * (drafts + 1), vocab, dtype)) return refuse(who, "workspace too small");
    if (!aligned(d_work, 16)) return refuse(who, "workspace not aligned to 16 bytes");
    VerifyArgs a{};
    a.z = d_logits;
    a.n = num_sequences;
    a.stride = row_stride;
    a.drafts = drafts;
    a.vocab = vocab;
    a.c2 = 1.44269504088896340736 / (double)temperature;
    a.ids = d_drafts;
    a.wide_ids = id_bytes == 8;
    a.uniforms = d_uniforms;
    a.slot_ids = drafts ? d_slot_ids : nullptr;
    a.wide_slots = slot_id_bytes == 8;
    a.teacher = d_teacher;
    a.teacher_dtype = teacher_dtype;
    a.slots = slots;
    a.tokens = d_tokens;
    a.accepted = d_accepted;
    a.logprobs = d_logprobs;
    a.work = d_work;
    return verify(a, dtype, (hipStream_t)stream);
}

}  // extern "C"
