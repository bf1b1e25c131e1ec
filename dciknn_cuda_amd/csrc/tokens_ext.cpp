// The token operators in the torch extension `_dci_cuda`: tensors checked, results and
// workspaces taken from torch's allocator on torch's current stream, gradients as autograd
// functions over the C-ABI's forward and backward entry points.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <stdexcept>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/dci_hip.h"

namespace py = pybind11;
using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

void check(int64_t rc) {
    if (rc < 0) throw std::runtime_error(std::string("libdci_hip: ") + dcih_last_error());
}

[[noreturn]] void bad_type(const std::string& what) { throw py::type_error(what); }
[[noreturn]] void bad_value(const std::string& what) { throw py::value_error(what); }

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

int type_code(const Tensor& t, const char* what) {
    if (!t.is_cuda()) bad_type(std::string(what) + " must be a cuda tensor");
    switch (t.scalar_type()) {
        case torch::kFloat32: return DCIH_F32;
        case torch::kFloat16: return DCIH_F16;
        case torch::kBFloat16: return DCIH_BF16;
        default: bad_type(std::string(what) + " must be float32, float16 or bfloat16");
    }
}

// Ids next to `where`: int32 or int64, any strides.
Tensor ids_of(const Tensor& ids, const Tensor& where, const char* what) {
    if (!ids.is_cuda()) bad_type(std::string(what) + " must be a cuda tensor");
    if (ids.scalar_type() != torch::kInt32 && ids.scalar_type() != torch::kInt64)
        bad_type(std::string(what) + " must be int32 or int64");
    if (ids.device() != where.device()) bad_value(std::string(what) + " must be on the other tensors' device");
    return ids.contiguous();
}

// Float32 factors of shape `shape`, any strides; broadcast ones are written out.
Tensor factors_of(const Tensor& t, c10::IntArrayRef shape, const Tensor& where, const char* what) {
    if (!t.is_cuda()) bad_type(std::string(what) + " must be a cuda tensor");
    if (t.scalar_type() != torch::kFloat32) bad_type(std::string(what) + " must be float32");
    if (t.device() != where.device()) bad_value(std::string(what) + " must be on the other tensors' device");
    if (t.sizes() != shape) bad_value(std::string(what) + " must have one value for each row");
    return t.contiguous();
}

// A tensor [..., len] as rows at one distance.
struct Rows {
    int64_t n = 1, len = 0, stride = 0;
    int dtype = 0;
};
Rows rows_of(const Tensor& t, const char* what) {
    Rows r;
    r.dtype = type_code(t, what);
    if (t.dim() < 1 || t.size(-1) < 1) bad_value(std::string(what) + " must have rows of one element or more");
    r.len = t.size(-1);
    if (r.len > DCIH_MAX_VOCAB) bad_value(std::string(what) + " has rows that are too long");
    if (r.len > 1 && t.stride(-1) != 1) bad_value(std::string(what) + ": the elements of a row must be next to one another");
    r.stride = r.len;
    for (int64_t d = t.dim() - 2; d >= 0; d--) {
        if (t.size(d) != 1 && t.numel()) {
            if (r.n == 1) r.stride = t.stride(d);
            else if (t.stride(d) != r.stride * r.n)
                bad_value(std::string(what) + ": the rows must be at one distance from each other; of a batch cut to fewer rows each take all rows, "
                                              "those cut off with ids of -1, or make it contiguous");
        }
        r.n *= t.size(d);
    }
    if (r.n == 0) r.stride = r.len;
    if (r.stride < r.len) bad_value(std::string(what) + ": rows must not overlap");
    if (r.n > 0x7fffffff) bad_value(std::string(what) + " has too many rows");
    return r;
}

float temperature_of(double t) {
    if (!(t > 1e-30) || !(t < 1e30)) bad_value("temperature must be a positive number");
    return (float)t;
}

c10::IntArrayRef leading(const Tensor& t) { return t.sizes().slice(0, t.dim() - 1); }

std::vector<int64_t> with_last(c10::IntArrayRef shape, int64_t last) {
    std::vector<int64_t> s(shape.begin(), shape.end());
    s.push_back(last);
    return s;
}

Tensor bytes(int64_t n, const Tensor& like) { return torch::empty({n}, like.options().dtype(torch::kUInt8).requires_grad(false)); }
Tensor floats(c10::IntArrayRef shape, const Tensor& like) {
    return torch::empty(shape, like.options().dtype(torch::kFloat32).requires_grad(false));
}
const float* data_or_null(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
int id_bytes(const Tensor& ids) { return ids.scalar_type() == torch::kInt64 ? 8 : 4; }

// A tangent of forward mode would be dropped in silence: its derivative is not formed.
void no_tangent(const Tensor& t) {
    if (t.defined() && t._fw_grad(0).defined()) throw std::runtime_error("the token operators have no derivatives in forward mode");
}

void once_only(const variable_list& grads) {
    for (const auto& g : grads) no_tangent(g);
    if (!torch::GradMode::is_enabled()) return;
    for (const auto& g : grads)
        if (g.defined() && g.requires_grad()) throw std::runtime_error("the token operators can be differentiated once only");
}

bool wants_grad(const Tensor& t) { return torch::GradMode::is_enabled() && t.requires_grad(); }

// ---- embedding lookup --------------------------------------------------------------------
Tensor embed_forward(const Tensor& table, const Tensor& ids_in, double scale) {
    const int dtype = type_code(table, "table");
    if (table.dim() != 2 || table.size(0) < 1 || table.size(1) < 1) bad_value("table must be [rows, dim]");
    if (table.size(1) > DCIH_MAX_DIM || table.size(0) > 0x7fffffff) bad_value("table is too large");
    const Rows r = rows_of(table, "table");
    const Tensor ids = ids_of(ids_in, table, "ids");
    if (ids.numel() > 0x7fffffff) bad_value("too many ids");
    c10::DeviceGuard guard(table.device());
    auto out = torch::empty(with_last(ids.sizes(), r.len), table.options().requires_grad(false));
    if (out.numel())
        check(dcih_embed(table.data_ptr(), dtype, r.n, (int)r.len, r.stride, ids.data_ptr(), id_bytes(ids), ids.numel(),
                         (float)scale, out.data_ptr(), stream_of(table)));
    return out;
}

Tensor embed_grad(const Tensor& grad, const Tensor& ids_in, int64_t num_rows, double scale, const c10::optional<Tensor>& into) {
    no_tangent(grad);
    if (wants_grad(grad)) bad_value("no gradient is formed by grad: detach it");
    const Rows r = rows_of(grad, "grad");
    const Tensor ids = ids_of(ids_in, grad, "ids");
    if (leading(grad) != ids.sizes()) bad_value("grad must have one row for each id");
    if (num_rows < 1 || num_rows > 0x7fffffff) bad_value("num_rows must be positive and below 2**31");
    if (r.len > DCIH_MAX_DIM) bad_value("grad has rows that are too long");
    Tensor out;
    if (into) {
        out = *into;
        no_tangent(out);
        const int code = type_code(out, "out");
        if (code != r.dtype && code != DCIH_F32) bad_type("out must be of grad's type or float32");
        if (out.device() != grad.device()) bad_value("out must be on the other tensors' device");
        if (out.sizes() != c10::IntArrayRef({num_rows, r.len}) || !out.is_contiguous()) bad_value("out must be [num_rows, dim] and contiguous");
        if (wants_grad(out)) bad_value("out must not require a gradient");
        if (out.is_alias_of(grad)) bad_value("out must not share grad's memory");
        out.unsafeGetTensorImpl()->bump_version();
    }
    c10::DeviceGuard guard(grad.device());
    if (!into) out = torch::empty({num_rows, r.len}, grad.options().requires_grad(false));
    const Tensor work = bytes(dcih_embed_grad_work(r.n, (int)r.len, num_rows), grad);
    check(dcih_embed_grad(grad.data_ptr(), r.dtype, r.n, (int)r.len, r.stride, ids.data_ptr(), id_bytes(ids), num_rows,
                          (float)scale, into ? 1 : 0, out.data_ptr(), out.scalar_type() == torch::kFloat32 ? DCIH_F32 : r.dtype,
                          work.data_ptr(), work.numel(), stream_of(grad)));
    return out;
}

struct Embed : torch::autograd::Function<Embed> {
    static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& ids, double scale) {
        ctx->save_for_backward({ids});
        ctx->saved_data["rows"] = table.size(0);
        ctx->saved_data["scale"] = scale;
        return embed_forward(table, ids, scale);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once_only(grads);
        const auto saved = ctx->get_saved_variables();
        return {embed_grad(grads[0].contiguous(), saved[0], ctx->saved_data["rows"].toInt(),
                           ctx->saved_data["scale"].toDouble(), c10::nullopt),
                Tensor(), Tensor()};
    }
};

Tensor embed(const Tensor& table, const Tensor& ids, double scale) {
    no_tangent(table);
    return wants_grad(table) ? Embed::apply(table, ids, scale) : embed_forward(table, ids, scale);
}

// ---- log probabilities -------------------------------------------------------------------
// (log probabilities, entropies, ids and log probabilities of alternatives, statistics)
std::vector<Tensor> logprobs_forward(const Tensor& logits, const Tensor& targets_in, int64_t top, double temperature, bool keep) {
    const Rows r = rows_of(logits, "logits");
    const Tensor targets = ids_of(targets_in, logits, "targets");
    if (leading(logits) != targets.sizes()) bad_value("targets must have one id for each row of logits");
    if (top < 0 || top > 64 || top > r.len) bad_value("top must be from 0 to 64 and at most the vocabulary");
    const float t = temperature_of(temperature);
    c10::DeviceGuard guard(logits.device());
    const Tensor lp = floats(targets.sizes(), logits), entropy = floats(targets.sizes(), logits);
    Tensor ids, lps, stats, work;
    if (top) {
        const auto shape = with_last(targets.sizes(), top);
        ids = torch::empty(shape, logits.options().dtype(torch::kInt32).requires_grad(false));
        lps = floats(shape, logits);
    }
    if (keep) stats = floats({r.n, 4}, logits);
    if (r.n) {
        const int64_t need = dcih_logits_work(r.n, (int)r.len, r.dtype, (int)top);
        check(need);
        work = bytes(need, logits);
        check(dcih_token_logprobs(logits.data_ptr(), r.dtype, r.n, (int)r.len, r.stride, targets.data_ptr(), id_bytes(targets), t,
                                  (int)top, lp.data_ptr<float>(), entropy.data_ptr<float>(),
                                  top ? ids.data_ptr<int32_t>() : nullptr, top ? lps.data_ptr<float>() : nullptr,
                                  keep ? stats.data_ptr<float>() : nullptr, work.data_ptr(), need, stream_of(logits)));
    }
    return {lp, entropy, ids, lps, stats};
}

struct Logprobs : torch::autograd::Function<Logprobs> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& targets, int64_t top, double temperature) {
        auto got = logprobs_forward(logits, targets, top, temperature, true);
        ctx->save_for_backward({logits, targets, got[4]});
        ctx->saved_data["temperature"] = temperature;
        ctx->set_materialize_grads(false);
        if (!top) return {got[0], got[1]};
        ctx->mark_non_differentiable({got[2], got[3]});
        return {got[0], got[1], got[2], got[3]};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once_only(grads);
        const auto saved = ctx->get_saved_variables();
        const Tensor& logits = saved[0];
        if (!grads[0].defined() && !grads[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        const Rows r = rows_of(logits, "logits");
        const Tensor targets = saved[1].contiguous();
        const Tensor g = grads[0].defined() ? grads[0].contiguous() : Tensor(), h = grads[1].defined() ? grads[1].contiguous() : Tensor();
        c10::DeviceGuard guard(logits.device());
        const Tensor out = torch::empty(logits.sizes(), logits.options().requires_grad(false).memory_format(torch::MemoryFormat::Contiguous));
        if (r.n)
            check(dcih_token_logprobs_grad(logits.data_ptr(), r.dtype, r.n, (int)r.len, r.stride, targets.data_ptr(), id_bytes(targets),
                                           (float)ctx->saved_data["temperature"].toDouble(), saved[2].data_ptr<float>(),
                                           data_or_null(g), data_or_null(h), out.data_ptr(), r.len, stream_of(logits)));
        return {out, Tensor(), Tensor(), Tensor()};
    }
};

py::tuple token_logprobs(const Tensor& logits, const Tensor& targets, int64_t top, double temperature) {
    no_tangent(logits);
    if (wants_grad(logits)) {
        const auto got = Logprobs::apply(logits, targets, top, temperature);
        return top ? py::make_tuple(got[0], got[1], got[2], got[3]) : py::make_tuple(got[0], got[1]);
    }
    const auto got = logprobs_forward(logits, targets, top, temperature, false);
    return top ? py::make_tuple(got[0], got[1], got[2], got[3]) : py::make_tuple(got[0], got[1]);
}

// ---- distillation ------------------------------------------------------------------------
struct Teacher {
    Tensor ids, logits;
    int dtype = 0, slots = 0;
};
Teacher teacher_of(const Tensor& ids, const Tensor& teacher, const Tensor& logits) {
    Teacher t;
    t.ids = ids_of(ids, logits, "ids");
    t.dtype = type_code(teacher, "teacher");
    if (teacher.device() != logits.device()) bad_value("teacher must be on the other tensors' device");
    if (teacher.sizes() != ids.sizes() || ids.dim() != logits.dim() || leading(ids) != leading(logits))
        bad_value("ids and teacher must be [..., slots] with the leading shape of logits");
    if (ids.size(-1) < 1 || ids.size(-1) > 1024) bad_value("a teacher has from 1 to 1024 slots");
    t.logits = teacher.contiguous();
    t.slots = (int)ids.size(-1);
    return t;
}

// (losses, statistics, gradient)
std::vector<Tensor> distill_forward(const Tensor& logits, const Tensor& ids, const Tensor& teacher, double temperature, bool keep,
                                    bool grad, const Tensor& weights, const Tensor& into) {
    for (const Tensor& x : {logits, teacher, weights, into}) no_tangent(x);
    const Rows r = rows_of(logits, "logits");
    const Teacher q = teacher_of(ids, teacher, logits);
    const float t = temperature_of(temperature);
    Rows o = r;
    o.stride = r.len;
    Tensor w, out = into;
    if (weights.defined()) w = factors_of(weights, leading(logits), logits, "weights");
    if (into.defined()) {
        if (into.sizes() != logits.sizes() || into.scalar_type() != logits.scalar_type() || into.device() != logits.device())
            bad_value("out must have the shape, type and device of logits");
        o = rows_of(into, "out");
        if (into.data_ptr() == logits.data_ptr() ? (o.stride != r.stride && r.n > 1) : into.is_alias_of(logits))
            bad_value("out must be logits itself or share no memory with it");
        into.unsafeGetTensorImpl()->bump_version();
    }
    c10::DeviceGuard guard(logits.device());
    const Tensor losses = floats(leading(logits), logits);
    Tensor stats, work;
    if (keep) stats = floats({r.n, 4}, logits);
    if (grad && !out.defined())
        out = torch::empty(logits.sizes(), logits.options().requires_grad(false).memory_format(torch::MemoryFormat::Contiguous));
    if (r.n) {
        const int64_t need = dcih_logits_work(r.n, (int)r.len, r.dtype, 0);
        check(need);
        work = bytes(need, logits);
        check(dcih_distill(logits.data_ptr(), r.dtype, r.n, (int)r.len, r.stride, q.ids.data_ptr(), id_bytes(q.ids), q.logits.data_ptr(),
                           q.dtype, q.slots, t, losses.data_ptr<float>(), keep ? stats.data_ptr<float>() : nullptr, data_or_null(w),
                           grad ? out.data_ptr() : nullptr, o.stride, work.data_ptr(), need, stream_of(logits)));
    }
    return {losses, stats, out};
}

struct Distill : torch::autograd::Function<Distill> {
    static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& ids, const Tensor& teacher, double temperature) {
        auto got = distill_forward(logits, ids, teacher, temperature, true, false, Tensor(), Tensor());
        ctx->save_for_backward({logits, ids, teacher, got[1]});
        ctx->saved_data["temperature"] = temperature;
        return got[0];
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once_only(grads);
        const auto saved = ctx->get_saved_variables();
        const Tensor& logits = saved[0];
        const Rows r = rows_of(logits, "logits");
        const Teacher q = teacher_of(saved[1], saved[2], logits);
        const Tensor w = grads[0].contiguous();
        c10::DeviceGuard guard(logits.device());
        const Tensor out = torch::empty(logits.sizes(), logits.options().requires_grad(false).memory_format(torch::MemoryFormat::Contiguous));
        if (r.n)
            check(dcih_distill_grad(logits.data_ptr(), r.dtype, r.n, (int)r.len, r.stride, q.ids.data_ptr(), id_bytes(q.ids),
                                    q.logits.data_ptr(), q.dtype, q.slots, (float)ctx->saved_data["temperature"].toDouble(),
                                    saved[3].data_ptr<float>(), w.data_ptr<float>(), out.data_ptr(), r.len, stream_of(logits)));
        return {out, Tensor(), Tensor(), Tensor()};
    }
};

Tensor distill_loss(const Tensor& logits, const Tensor& ids, const Tensor& teacher, double temperature) {
    if (wants_grad(teacher)) bad_value("no gradient is formed by the teacher's logits: detach them");
    if (wants_grad(logits)) return Distill::apply(logits, ids, teacher, temperature);
    return distill_forward(logits, ids, teacher, temperature, false, false, Tensor(), Tensor())[0];
}

std::tuple<Tensor, Tensor> distill_step(const Tensor& logits, const Tensor& ids, const Tensor& teacher, const c10::optional<Tensor>& weights,
                                        double temperature, const c10::optional<Tensor>& into) {
    // (logits that a model computed require a gradient, and theirs may take their place; a parameter's may not)
    if (into && wants_grad(*into) && (into->is_leaf() || !into->is_same(logits)))
        bad_value("out must not require a gradient, but for logits that are no leaf");
    torch::NoGradGuard no_grad;
    const auto got = distill_forward(logits, ids, teacher, temperature, false, true, weights ? *weights : Tensor(), into ? *into : Tensor());
    return {got[0], got[2]};
}

// ---- gated recurrence --------------------------------------------------------------------
// What a scan is over: x [rows, length, dim], or [tokens, dim] with sequences between offsets.
struct Scan {
    int dtype = 0, flags = 0, dim = 0;
    int64_t rows = 1, length = 0, sequences = 0, packed = 0;
    int64_t x_row = 0, x_step = 0, g_row = 0, g_step = 0;
    Tensor bounds;

    int bound_bytes() const { return bounds.defined() ? id_bytes(bounds) : 4; }
    const void* bound_data() const { return bounds.defined() ? bounds.data_ptr() : nullptr; }
};

// The states of all sequences, float32 and contiguous; undefined where none are given.
Tensor states_of(const c10::optional<Tensor>& t, const Scan& s, const Tensor& x, const char* what) {
    if (!t || !t->defined()) return Tensor();
    if (!t->is_cuda()) bad_type(std::string(what) + " must be a cuda tensor");
    if (t->scalar_type() != torch::kFloat32) bad_type(std::string(what) + " must be float32");
    if (t->device() != x.device()) bad_value(std::string(what) + " must be on the other tensors' device");
    if (t->sizes() != c10::IntArrayRef({s.sequences, s.dim})) bad_value(std::string(what) + " must be [sequences, dim]");
    return t->contiguous();
}

Scan scan_of(const Tensor& x, const Tensor& gates, bool decay, const Tensor& lengths, const Tensor& offsets) {
    Scan s;
    s.dtype = type_code(x, "x");
    if (type_code(gates, "gates") != s.dtype) bad_type("gates must be of x's type");
    if (gates.device() != x.device()) bad_value("gates must be on the other tensors' device");
    if (x.dim() != 2 && x.dim() != 3) bad_value("x must be [batch, length, dim] or [tokens, dim]");
    const bool batch = x.dim() == 3;
    if (x.size(-1) < 1 || x.size(-1) > DCIH_MAX_DIM) bad_value("x must have from 1 to 2**20 channels");
    s.dim = (int)x.size(-1);
    if (s.dim > 1 && (x.stride(-1) != 1 || gates.stride(-1) != 1)) bad_value("the channels of a token must be next to one another");
    const bool shared = gates.dim() == 1;
    if (shared ? gates.size(0) != s.dim : gates.sizes() != x.sizes()) bad_value("gates must be of x's shape, or one for each channel");
    s.flags = (decay ? DCIH_SCAN_DECAYS : 0) | (shared ? DCIH_SCAN_SHARED : 0);
    s.rows = batch ? x.size(0) : 1;
    s.length = x.size(-2);
    if (s.rows > 0x7fffffff || s.length > 0x7fffffff) bad_value("x has too many tokens");
    s.x_row = batch ? x.stride(0) : 0;
    s.x_step = x.stride(-2);
    if (!shared) {
        s.g_row = batch ? gates.stride(0) : 0;
        s.g_step = gates.stride(-2);
    }
    s.sequences = s.rows;
    if (lengths.defined()) {
        if (!batch) bad_value("lengths are for x of [batch, length, dim]; sequences of [tokens, dim] are between offsets");
        s.bounds = ids_of(lengths, x, "lengths");
        if (s.bounds.dim() != 1 || s.bounds.size(0) != s.rows) bad_value("lengths must be [batch]");
    }
    if (offsets.defined()) {
        if (batch) bad_value("offsets are for x of [tokens, dim]; a batch may have lengths");
        s.bounds = ids_of(offsets, x, "offsets");
        if (s.bounds.dim() != 1 || s.bounds.size(0) < 2) bad_value("offsets must be [sequences + 1]");
        if (s.bounds.size(0) - 1 > 0x7fffffff) bad_value("too many sequences");
        s.packed = s.sequences = s.bounds.size(0) - 1;
    }
    return s;
}

Tensor or_none(const c10::optional<Tensor>& t) { return t ? *t : Tensor(); }
c10::optional<Tensor> if_given(const Tensor& t) { return t.defined() ? c10::optional<Tensor>(t) : c10::nullopt; }

// (h, last states, states for the gradient)
variable_list scan_forward(const Scan& s, const Tensor& x, const Tensor& gates, const Tensor& state, const Tensor& into, bool keep) {
    c10::DeviceGuard guard(x.device());
    const Tensor h = torch::empty(x.sizes(), x.options().requires_grad(false).memory_format(torch::MemoryFormat::Contiguous));
    const Tensor last = into.defined() ? into : floats({s.sequences, s.dim}, x);
    Tensor states;
    if (keep) states = floats({dcih_scan_states(s.rows, s.length, s.dim, s.dtype)}, x);
    const int64_t need = dcih_scan_work(s.rows, s.length, s.dim, s.dtype, s.packed);
    check(need);
    const Tensor work = bytes(need, x);
    if (s.sequences)
        check(dcih_scan(x.data_ptr(), s.dtype, s.rows, s.length, s.dim, s.x_row, s.x_step, gates.data_ptr(), s.g_row, s.g_step, s.flags,
                        data_or_null(state), s.bound_data(), s.bound_bytes(), s.packed, h.data_ptr(), last.data_ptr<float>(),
                        keep ? states.data_ptr<float>() : nullptr, work.data_ptr(), need, stream_of(x)));
    return {h, last, states};
}

struct GatedScan : torch::autograd::Function<GatedScan> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& gates, const c10::optional<Tensor>& state_in, bool decay,
                                 const c10::optional<Tensor>& lengths_in, const c10::optional<Tensor>& offsets_in) {
        const Tensor state = or_none(state_in), lengths = or_none(lengths_in), offsets = or_none(offsets_in);
        const Scan s = scan_of(x, gates, decay, lengths, offsets);
        const auto got = scan_forward(s, x, gates, state, Tensor(), true);
        ctx->save_for_backward({x, gates, state, lengths, offsets, got[2]});
        ctx->saved_data["decay"] = decay;
        ctx->set_materialize_grads(false);
        return {got[0], got[1]};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once_only(grads);
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &gates = saved[1], &state = saved[2];
        const Scan s = scan_of(x, gates, ctx->saved_data["decay"].toBool(), saved[3], saved[4]);
        Tensor dx, dgates, dstate;
        if (grads[0].defined() || grads[1].defined()) {
            const Tensor dh = grads[0].defined() ? grads[0].contiguous() : Tensor(), dlast = grads[1].defined() ? grads[1].contiguous() : Tensor();
            c10::DeviceGuard guard(x.device());
            const auto plain = x.options().requires_grad(false).memory_format(torch::MemoryFormat::Contiguous);
            if (ctx->needs_input_grad(0)) dx = torch::empty(x.sizes(), plain);
            if (ctx->needs_input_grad(1)) dgates = s.rows && s.length ? torch::empty(gates.sizes(), plain) : torch::zeros(gates.sizes(), plain);
            if (state.defined() && ctx->needs_input_grad(2)) dstate = floats(state.sizes(), x);
            const int64_t need = dcih_scan_work(s.rows, s.length, s.dim, s.dtype, s.packed);
            check(need);
            const Tensor work = bytes(need, x);
            if (s.sequences)
                check(dcih_scan_grad(x.data_ptr(), s.dtype, s.rows, s.length, s.dim, s.x_row, s.x_step, gates.data_ptr(), s.g_row, s.g_step, s.flags,
                                     data_or_null(state), s.bound_data(), s.bound_bytes(), s.packed, saved[5].data_ptr<float>(),
                                     dh.defined() ? dh.data_ptr() : nullptr, data_or_null(dlast), dx.defined() && dx.numel() ? dx.data_ptr() : nullptr,
                                     dgates.defined() && s.rows && s.length ? dgates.data_ptr() : nullptr, dstate.defined() ? dstate.data_ptr<float>() : nullptr,
                                     work.data_ptr(), need, stream_of(x)));
        }
        return {dx, dgates, dstate, Tensor(), Tensor(), Tensor()};
    }
};

std::tuple<Tensor, Tensor> gated_scan(const Tensor& x, const Tensor& gates, const c10::optional<Tensor>& state_in, bool decay,
                                      const c10::optional<Tensor>& lengths_in, const c10::optional<Tensor>& offsets_in,
                                      const c10::optional<Tensor>& into) {
    const Tensor lengths = or_none(lengths_in), offsets = or_none(offsets_in);
    const Scan s = scan_of(x, gates, decay, lengths, offsets);
    const Tensor state = states_of(state_in, s, x, "state");
    for (const Tensor& t : {x, gates, state}) no_tangent(t);
    const bool wanted = wants_grad(x) || wants_grad(gates) || (state.defined() && wants_grad(state));
    if (!into) {
        if (!wanted) {
            const auto got = scan_forward(s, x, gates, state, Tensor(), false);
            return {got[0], got[1]};
        }
        const auto got = GatedScan::apply(x, gates, if_given(state), decay, lengths_in, offsets_in);
        return {got[0], got[1]};
    }
    if (wanted) bad_value("last is for calls without gradients");
    no_tangent(*into);
    if (into->is_cuda() && !into->is_contiguous()) bad_value("last must be contiguous");
    states_of(into, s, x, "last");
    if (wants_grad(*into)) bad_value("last must not require a gradient");
    if (into->is_alias_of(x) || into->is_alias_of(gates)) bad_value("last must not share the memory of x or gates");
    if (state.defined() && into->numel()) {
        const char *a = (const char*)state.data_ptr(), *b = (const char*)into->data_ptr();
        if (a != b && a < b + into->nbytes() && b < a + state.nbytes()) bad_value("last must be state, or share no memory with it");
    }
    into->unsafeGetTensorImpl()->bump_version();
    const auto got = scan_forward(s, x, gates, state, *into, false);
    return {got[0], *into};
}

// ---- norm of gradients, clipping ---------------------------------------------------------
// A list of tensors, looked at in place: a model has thousands of gradients.
struct Tensors {
    py::list list;
    size_t size() const { return list.size(); }
    bool empty() const { return list.empty(); }
    const Tensor& operator[](size_t i) const {
        PyObject* p = PyList_GET_ITEM(list.ptr(), (Py_ssize_t)i);
        if (!THPVariable_Check(p)) bad_type("a gradient must be a tensor");
        return THPVariable_Unpack(p);
    }
};

void no_gradient(const Tensor& t) {
    no_tangent(t);
    if (t.requires_grad() && torch::GradMode::is_enabled()) bad_value("no gradient is formed by or of the gradients: detach them");
}

std::vector<dcih_span> spans_of(const Tensors& grads, const Tensors* into) {
    if (into && into->size() != grads.size()) bad_value("out must have one tensor for each gradient");
    std::vector<dcih_span> spans;
    spans.reserve(grads.size());
    const size_t n = grads.size();
    c10::Device device(c10::kCPU);
    for (size_t i = 0; i < n; i++) {
        const Tensor &g = grads[i], &o = into ? (*into)[i] : g;
        dcih_span p{};
        p.dtype = type_code(g, "a gradient");
        if (!i) device = g.device();
        if (g.device() != device) bad_value("the gradients must be on one device");
        if (!g.is_non_overlapping_and_dense()) bad_value("a gradient's elements must be one behind the other in some order of its dimensions");
        no_gradient(g);
        p.out_dtype = into ? type_code(o, "out") : p.dtype;
        if (into) {
            if (p.out_dtype != p.dtype && p.out_dtype != DCIH_F32) bad_type("out must be of the gradient's type or float32");
            if (o.device() != device) bad_value("out must be on the gradients' device");
            bool alike = o.sizes() == g.sizes();
            for (int64_t d = 0; alike && d < g.dim(); d++) alike = g.size(d) == 1 || o.stride(d) == g.stride(d);
            if (!alike) bad_value("out must have the gradient's shape and strides");
            no_gradient(o);
        }
        p.data = g.data_ptr();
        p.out = into ? o.data_ptr() : const_cast<void*>(p.data);
        p.count = g.numel();
        if (p.count) spans.push_back(p);
    }
    return spans;
}

// No two of what is written may overlap, nor any of it another gradient.
void check_apart(const std::vector<dcih_span>& spans) {
    struct Range { uintptr_t from, to; bool written; };
    std::vector<Range> ranges;
    ranges.reserve(2 * spans.size());
    auto size = [](int dtype) { return dtype == DCIH_F32 ? 4 : 2; };
    for (const auto& p : spans) {
        ranges.push_back({(uintptr_t)p.out, (uintptr_t)p.out + p.count * size(p.out_dtype), true});
        if (p.data != p.out || p.dtype != p.out_dtype) ranges.push_back({(uintptr_t)p.data, (uintptr_t)p.data + p.count * size(p.dtype), false});
    }
    auto before = [](const Range& a, const Range& b) { return a.from < b.from; };
    if (!std::is_sorted(ranges.begin(), ranges.end(), before)) std::sort(ranges.begin(), ranges.end(), before);
    uintptr_t read = 0, written = 0;          // how far what lies before reaches
    for (const auto& r : ranges) {
        if (r.from < written || (r.written && r.from < read)) bad_value("a tensor that is written must not share memory with another one of the call");
        (r.written ? written : read) = std::max(r.written ? written : read, r.to);
    }
}

double scale_of(double scale) {
    if (!std::isfinite(scale)) bad_value("scale must be a finite number");
    return scale;
}

Tensor norm_of_none() { return torch::zeros({}, torch::kFloat32); }

Tensor grad_norm(const py::list& list, double scale) {
    const Tensors grads{list};
    scale_of(scale);
    if (grads.empty()) return norm_of_none();
    const auto spans = spans_of(grads, nullptr);
    c10::DeviceGuard guard(grads[0].device());
    const Tensor norm = floats({}, grads[0]);
    const int64_t need = dcih_clip_work(spans.data(), spans.size());
    check(need);
    const Tensor work = bytes(need, grads[0]);
    check(dcih_grad_norm(spans.data(), spans.size(), scale, norm.data_ptr<float>(), work.data_ptr(), need, stream_of(grads[0])));
    return norm;
}

Tensor clip_grads(const py::list& list, double max_norm, double scale, const c10::optional<py::list>& out) {
    const Tensors grads{list}, into{out ? *out : py::list()};
    scale_of(scale);
    if (!(max_norm >= 0.0)) bad_value("max_norm must not be negative");
    if (grads.empty() && into.empty()) return norm_of_none();
    const auto spans = spans_of(grads, out ? &into : nullptr);
    check_apart(spans);
    for (size_t i = 0; i < grads.size(); i++) (out ? into : grads)[i].unsafeGetTensorImpl()->bump_version();
    c10::DeviceGuard guard(grads[0].device());
    const Tensor norm = floats({}, grads[0]);
    const int64_t need = dcih_clip_work(spans.data(), spans.size());
    check(need);
    const Tensor work = bytes(need, grads[0]);
    check(dcih_clip(spans.data(), spans.size(), max_norm, scale, norm.data_ptr<float>(), work.data_ptr(), need, stream_of(grads[0])));
    return norm;
}

// ---- verification of drafts --------------------------------------------------------------
std::tuple<Tensor, Tensor, Tensor> verify_drafts(const Tensor& logits, const Tensor& drafts_in, const Tensor& uniforms, const c10::optional<Tensor>& ids_in,
                                                 const c10::optional<Tensor>& teacher_in, double temperature) {
    const Rows r = rows_of(logits, "logits");
    if (logits.dim() != 3 || logits.size(1) < 1) bad_value("logits must be [batch, drafts + 1, vocab]");
    const int64_t n = logits.size(0), k = logits.size(1) - 1;
    if (k > DCIH_MAX_DRAFTS) bad_value("a sequence has up to 256 drafts");
    const Tensor drafts = ids_of(drafts_in, logits, "drafts");
    if (drafts.sizes() != c10::IntArrayRef({n, k})) bad_value("drafts must be [batch, drafts], one fewer than rows of logits");
    const Tensor u = factors_of(uniforms, leading(logits), logits, "uniforms");
    if (ids_in.has_value() != teacher_in.has_value()) bad_value("ids and teacher are given together");
    const float t = temperature_of(temperature);
    Teacher q;
    if (ids_in) {
        const Tensor ids = ids_of(*ids_in, logits, "ids");
        q.dtype = type_code(*teacher_in, "teacher");
        if (teacher_in->device() != logits.device()) bad_value("teacher must be on the other tensors' device");
        if (ids.dim() != 3 || ids.size(0) != n || ids.size(1) != k || teacher_in->sizes() != ids.sizes()) bad_value("ids and teacher must be [batch, drafts, slots]");
        if (ids.size(2) < 1 || ids.size(2) > 1024) bad_value("a draft's distribution has from 1 to 1024 slots");
        q.ids = ids;
        q.logits = teacher_in->contiguous();
        q.slots = (int)ids.size(2);
    }
    for (const Tensor& x : {logits, uniforms, q.logits}) {
        no_tangent(x);
        if (x.defined() && wants_grad(x)) bad_value("no gradient is formed through tokens: detach the inputs");
    }
    c10::DeviceGuard guard(logits.device());
    const auto whole = logits.options().dtype(torch::kInt32).requires_grad(false);
    const Tensor tokens = torch::empty({n, k + 1}, whole), accepted = torch::empty({n}, whole), logprobs = floats({n, k + 1}, logits);
    if (n) {
        const int64_t need = dcih_verify_work(n, (int)k, (int)r.len, r.dtype);
        check(need);
        const Tensor work = bytes(need, logits);
        check(dcih_verify(logits.data_ptr(), r.dtype, n, (int)k, (int)r.len, r.stride, k ? drafts.data_ptr() : nullptr, id_bytes(drafts), u.data_ptr<float>(),
                          q.ids.defined() && k ? q.ids.data_ptr() : nullptr, q.ids.defined() ? id_bytes(q.ids) : 4,
                          q.logits.defined() && k ? q.logits.data_ptr() : nullptr, q.dtype, q.slots, t, tokens.data_ptr<int32_t>(),
                          accepted.data_ptr<int32_t>(), logprobs.data_ptr<float>(), work.data_ptr(), need, stream_of(logits)));
    }
    return {tokens, accepted, logprobs};
}

}  // namespace

void bind_tokens(py::module_& m) {
    m.def("_embed", &embed, "Rows of a table by ids, times a factor. (HIP)");
    m.def("_embed_grad", &embed_grad, "Gradient of _embed by the table. (HIP)");
    m.def("_token_logprobs", &token_logprobs, "Log probabilities, entropies, best alternatives. (HIP)");
    m.def("_distill_loss", &distill_loss, "Loss against a teacher's top logits. (HIP)");
    m.def("_gated_scan", &gated_scan, "Gated linear recurrence over the tokens of sequences. (HIP)");
    m.def("_grad_norm", &grad_norm, "Norm of a model's gradients. (HIP)");
    m.def("_clip_grads", &clip_grads, "Gradients clipped by their norm. (HIP)");
    m.def("_verify_drafts", &verify_drafts, "Drafted tokens against the model's probabilities. (HIP)");
    m.def("_distill_step", &distill_step, "Loss against a teacher's top logits and its gradient. (HIP)");
}
