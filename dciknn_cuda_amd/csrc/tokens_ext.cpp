// The token operators in the torch extension `_dci_cuda`: tensors checked, results and
// workspaces taken from torch's allocator on torch's current stream, gradients as autograd
// functions over the C-ABI's forward and backward entry points.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

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

}  // namespace

void bind_tokens(py::module_& m) {
    m.def("_embed", &embed, "Rows of a table by ids, times a factor. (HIP)");
    m.def("_embed_grad", &embed_grad, "Gradient of _embed by the table. (HIP)");
    m.def("_token_logprobs", &token_logprobs, "Log probabilities, entropies, best alternatives. (HIP)");
    m.def("_distill_loss", &distill_loss, "Loss against a teacher's top logits. (HIP)");
    m.def("_distill_step", &distill_step, "Loss against a teacher's top logits and its gradient. (HIP)");
}
