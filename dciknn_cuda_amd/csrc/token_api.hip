// The entry points of include/dci_hip.h that work on tokens: checks of the arguments, the caller's
// workspace laid out, launches.  No handle, no state; nothing here allocates, waits or throws.
#include <algorithm>
#include <initializer_list>
#include <string>

#include "../../include/dci_hip.h"
#include "token_common.h"

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

}  // extern "C"
