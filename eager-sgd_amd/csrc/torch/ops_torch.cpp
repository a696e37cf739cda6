// ops_torch.cpp — esgd._ops: the row operators (include/esgd_ops.h) on torch tensors.
//
// Checks the tensors, allocates the results and work memory (torch's allocator, the current
// stream) and makes the C calls.  All of a small call's cost is here and in the launch: in Python
// over ctypes the same steps took 7.6 us for a lookup of 16 tokens, here 4.5, of which the launch is 3.4.
// The C entry points come as addresses from esgd._lib, which has loaded libesgd.so, so that there is
// one library in the process whatever its path.  What a caller got wrong raises ValueError, a
// failed call EsgdError, as everywhere in the package.
#include <torch/extension.h>

#include <ATen/MemoryOverlap.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>

#include <cstdint>
#include <optional>
#include <string>
#include <tuple>
#include <unordered_map>

#include "esgd_ops.h"

namespace py = pybind11;
using at::Tensor;

namespace {

#define ESGD_OPS(X)                                                                                       \
    X(esgd_embedding) X(esgd_embedding_grad_work) X(esgd_embedding_grad) X(esgd_expert_sort_work)         \
    X(esgd_expert_sort) X(esgd_expert_dispatch) X(esgd_expert_dispatch_grad) X(esgd_expert_combine)       \
    X(esgd_expert_combine_grad) X(esgd_distill_work) X(esgd_distill_loss) X(esgd_distill_grad)            \
    X(esgd_distill_loss_grad)

struct Table {
#define X(name) decltype(&::name) name = nullptr;
    ESGD_OPS(X)
#undef X
} c;

void bind(const std::unordered_map<std::string, uint64_t> &address) {
#define X(name) c.name = reinterpret_cast<decltype(&::name)>(address.at(#name));
    ESGD_OPS(X)
#undef X
}

// ---- types, names and refusals ----
int type_of(at::ScalarType t) {   // 0: none of the operators'
    switch (t) {
    case at::kFloat: return ESGD_FLOAT;
    case at::kBFloat16: return ESGD_BF16;
    case at::kHalf: return ESGD_HALF;
    default: return 0;
    }
}
std::string name_of(at::ScalarType t) {   // as Python prints it
    switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kHalf: return "torch.float16";
    case at::kDouble: return "torch.float64";
    case at::kInt: return "torch.int32";
    case at::kLong: return "torch.int64";
    default: return c10::toString(t);
    }
}
std::string shape_of(at::IntArrayRef s) {
    std::string r = "(";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + (s.size() == 1 ? ",)" : ")");
}
#define REFUSE(cond, ...)                                                    \
    do {                                                                     \
        if (C10_UNLIKELY(cond)) throw py::value_error(c10::str(__VA_ARGS__)); \
    } while (0)

// Forward-mode derivatives stop here: a result without its tangent would tell of a derivative of zero.
// (In an autograd function's forward pass tangents are hidden until the mode is on again.)
void no_tangent(const char *who, const char *name, const Tensor &t) {
    const c10::AutoFwGradMode seen(true);
    REFUSE(t._fw_grad(0).defined(), who, ": ", name, " has a tangent; there is no forward-mode derivative");
}
void no_sign(const char *who, const char *name, const Tensor &t) {
    REFUSE(t.is_neg(), who, ": ", name, " is a view whose sign is still to be changed; resolve_neg() makes it a tensor");
}
int float_of(const char *who, const char *name, const Tensor &t, int64_t dims = -1) {
    const int code = type_of(t.scalar_type());
    REFUSE(!code, who, ": ", name, " is ", name_of(t.scalar_type()), "; float32, bfloat16 or float16 is needed");
    no_sign(who, name, t);
    no_tangent(who, name, t);
    REFUSE(dims >= 0 && t.dim() != dims, who, ": ", name, " has ", t.dim(), " dimensions, not ", dims);
    return code;
}
int bits_of(const char *who, const char *name, const Tensor &t) {
    const auto k = t.scalar_type();
    REFUSE(k != at::kInt && k != at::kLong, who, ": ", name, " is ", name_of(k), "; int32 or int64 is needed");
    return k == at::kLong ? 64 : 32;
}
// last of the checks: the tensors lie on one HIP device
void on_device(const char *who, const Tensor &first, std::initializer_list<const Tensor *> others) {
    REFUSE(!first.is_cuda(), who, ": tensors on ", first.device().str(),
           ", a HIP device is needed (there is no CPU path)");
    for (const Tensor *t : others)
        REFUSE(t->defined() && t->device() != first.device(), who, ": tensors on ", first.device().str(), " and ",
               t->device().str());
}

// `t` as (rows, width) with contiguous rows
Tensor rows_of(const Tensor &t, int64_t width) {
    Tensor r = t.dim() == 2 ? t : t.reshape({width ? t.numel() / width : 0, width});
    return r.stride(1) != 1 && width > 1 ? r.contiguous() : r;
}

// Whether `out`, contiguous, lies among the elements of `rows` (rows_of's): addresses are compared, row
// by row, since torch's own question (get_overlap_status) has no answer where rows stand apart.
bool touches(const Tensor &rows, const Tensor &out) {
    if (!rows.numel() || !out.numel()) return false;
    const auto at = [](const Tensor &t) { return reinterpret_cast<intptr_t>(t.const_data_ptr()); };
    const int64_t size = rows.element_size(), row = rows.size(1) * size, pitch = rows.stride(0) * size;
    const int64_t from = at(out) - at(rows), to = from + int64_t(out.nbytes());   // of out, from the first row
    // the first row that ends behind `from`
    const int64_t i = from < row || !pitch ? 0 : (from - row) / pitch + 1;
    return i < rows.size(0) && i * pitch < to && i * pitch + row > from;
}

void check(int rc, const char *what) {
    if (C10_UNLIKELY(rc)) py::module_::import("esgd._lib").attr("check")(rc, what);   // raises EsgdError
}
// the C call f(stream) on the tensor's device and its current stream
template <class F>
void call(const char *what, const Tensor &on, F &&f) {
    const auto index = on.device().index();
    const c10::DeviceGuard guard(on.device());
    hipStream_t s = c10::hip::getCurrentHIPStream(index).stream();
    int rc;
    {
        py::gil_scoped_release release;
        rc = f(s ? static_cast<void *>(s) : ESGD_STREAM_NULL);
    }
    check(rc, what);
}
Tensor work_of(const Tensor &on, size_t bytes) {
    return at::empty({int64_t(bytes)}, on.options().dtype(at::kByte));
}
// below autograd: nothing here is recorded, and torch's own calls skip that layer
using Below = at::AutoDispatchBelowADInplaceOrView;

// ---- embedding ----
Tensor embedding(const Tensor &weight, const Tensor &tokens, double scale, std::optional<at::ScalarType> dtype) {
    const char *who = "embedding";
    Below below;
    const int wtype = float_of(who, "weight", weight, 2), bits = bits_of(who, "tokens", tokens);
    const auto own = weight.scalar_type(), out_type = dtype.value_or(own);
    REFUSE(!type_of(out_type) || (out_type != own && own != at::kFloat), who, ": a ", name_of(own),
           " table gives rows of its own type", own == at::kFloat ? " or bfloat16 or float16" : "", ", not ",
           name_of(out_type));
    on_device(who, weight, {&tokens});
    const int64_t width = weight.size(1);
    const Tensor w = rows_of(weight, width), t = tokens.contiguous();
    c10::SmallVector<int64_t, 5> shape(tokens.sizes().begin(), tokens.sizes().end());
    shape.push_back(width);
    Tensor out = at::empty(shape, weight.options().dtype(out_type));
    call("esgd_embedding", w, [&](void *s) {
        return c.esgd_embedding(wtype, w.data_ptr(), w.stride(0), w.size(0), width, bits, t.data_ptr(), t.numel(),
                                float(scale), type_of(out_type), out.data_ptr(), width, s);
    });
    return out;
}

Tensor embedding_grad(const Tensor &grad, const Tensor &tokens, int64_t num_rows, double scale, int64_t skip,
                      std::optional<at::ScalarType> dtype, const std::optional<Tensor> &given, bool accumulate) {
    const char *who = "embedding_grad";
    Below below;
    const Tensor out = given.value_or(Tensor());
    const int gtype = float_of(who, "grad", grad), bits = bits_of(who, "tokens", tokens);
    REFUSE(grad.dim() < 1 || grad.sizes().slice(0, grad.dim() - 1) != tokens.sizes(), who, ": grad ",
           shape_of(grad.sizes()), " does not have a row for each of the tokens ", shape_of(tokens.sizes()));
    const int64_t width = grad.size(-1);
    REFUSE(num_rows < 0, who, ": num_rows ", num_rows, " is negative");
    REFUSE(accumulate && !out.defined(), who, ": accumulate needs out");
    if (out.defined()) {
        no_sign(who, "out", out);
        no_tangent(who, "out", out);
        REFUSE(out.requires_grad() && c10::GradMode::is_enabled(), who,
               ": out requires a gradient, and autograd does not see what is written to it (torch.no_grad() or detach())");
        REFUSE(out.dim() != 2 || out.size(0) != num_rows || out.size(1) != width || !out.is_contiguous(), who,
               ": out is not a contiguous (", num_rows, ", ", width, ") tensor");
        for (const Tensor *t : {&grad, &tokens}) {
            const auto o = at::get_overlap_status(out, *t);
            REFUSE(o == at::MemOverlapStatus::Full || o == at::MemOverlapStatus::Partial, who,
                   ": out shares memory with ", t == &grad ? "grad" : "tokens");
        }
        REFUSE(dtype && *dtype != out.scalar_type(), who, ": out is ", name_of(out.scalar_type()), ", dtype says ",
               name_of(dtype.value_or(at::kFloat)));
    }
    const auto own = grad.scalar_type(), table_type = out.defined() ? out.scalar_type() : dtype.value_or(own);
    REFUSE(!type_of(table_type) || (table_type != own && table_type != at::kFloat), who, ": ", name_of(own),
           " rows give a gradient of that type or float32, not ", name_of(table_type));
    size_t bytes = 0;
    check(c.esgd_embedding_grad_work(tokens.numel(), num_rows, width, &bytes), "esgd_embedding_grad_work");
    const Tensor g = rows_of(grad, width), t = tokens.contiguous();
    if (out.defined()) {
        REFUSE(touches(g, out), who, ": out shares memory with grad");
        REFUSE(touches(t.view({1, t.numel()}), out), who, ": out shares memory with tokens");
    }
    on_device(who, grad, {&tokens, &out});
    Tensor table = out.defined() ? out : at::empty({num_rows, width}, grad.options().dtype(table_type));
    const Tensor work = work_of(grad, bytes);
    call("esgd_embedding_grad", g, [&](void *s) {
        return c.esgd_embedding_grad(gtype, g.data_ptr(), g.stride(0), t.numel(), width, bits, t.data_ptr(), skip,
                                     float(scale), type_of(table_type), table.data_ptr(), num_rows, accumulate,
                                     work.data_ptr(), bytes, s);
    });
    if (out.defined() && !out.is_inference()) out.unsafeGetTensorImpl()->bump_version();   // for autograd, as any op in place
    return table;
}

// ---- tokens by expert ----
std::tuple<Tensor, Tensor> expert_sort(const Tensor &experts, int64_t num_experts) {
    const char *who = "expert_sort";
    Below below;
    const int bits = bits_of(who, "experts", experts);
    REFUSE((experts.dim() != 1 && experts.dim() != 2) || (experts.dim() == 2 && experts.size(1) < 1), who, ": experts ",
           shape_of(experts.sizes()), " is neither (tokens, choices) nor (tokens,)");
    const int64_t tokens = experts.size(0), choices = experts.dim() == 2 ? experts.size(1) : 1;
    size_t bytes = 0;
    check(c.esgd_expert_sort_work(tokens * choices, num_experts, &bytes), "esgd_expert_sort_work");
    on_device(who, experts, {});
    const Tensor e = experts.contiguous();
    const auto whole = experts.options().dtype(at::kInt);
    Tensor offsets = at::empty({num_experts + 1}, whole), slots = at::empty({tokens, choices}, whole);
    const Tensor work = work_of(experts, bytes);
    call("esgd_expert_sort", e, [&](void *s) {
        return c.esgd_expert_sort(bits, e.data_ptr(), tokens, choices, num_experts, offsets.data_ptr<int32_t>(),
                                  slots.data_ptr<int32_t>(), work.data_ptr(), bytes, s);
    });
    return {offsets, slots};
}

// a tensor with a row per token, or per pair
int row_type(const char *who, const char *name, const Tensor &t, const Tensor &slots, bool per_pair) {
    const int code = float_of(who, name, t, 2);
    const int64_t tokens = slots.size(0), choices = slots.size(1);
    REFUSE(t.size(0) != (per_pair ? tokens * choices : tokens), who, ": ", name, " has ", t.size(0), " rows for ",
           tokens, " tokens of ", choices, " choices");
    return code;
}
Tensor weights_of(const char *who, const Tensor &weights, const Tensor &slots) {
    float_of(who, "weights", weights);
    const int64_t tokens = slots.size(0), choices = slots.size(1);
    const bool fits = weights.dim() == 2 ? weights.size(0) == tokens && weights.size(1) == choices
                                         : weights.dim() == 1 && choices == 1 && weights.size(0) == tokens;
    REFUSE(!fits, who, ": weights ", shape_of(weights.sizes()), " for ", tokens, " tokens of ", choices, " choices");
    return weights.to(at::kFloat).contiguous();
}
void check_slots(const char *who, const Tensor &slots) {
    REFUSE(slots.dim() != 2 || slots.scalar_type() != at::kInt || !slots.is_contiguous() || slots.size(1) < 1, who,
           ": the order's slots are not what expert_sort gives");
}

Tensor expert_dispatch(const Tensor &x, const Tensor &slots) {
    const char *who = "expert_dispatch";
    Below below;
    check_slots(who, slots);
    const int code = row_type(who, "x", x, slots, false);
    on_device(who, x, {&slots});
    const int64_t tokens = slots.size(0), choices = slots.size(1), width = x.size(1);
    const Tensor r = rows_of(x, width);
    Tensor out = at::empty({tokens * choices, width}, x.options());
    call("esgd_expert_dispatch", r, [&](void *s) {
        return c.esgd_expert_dispatch(code, r.data_ptr(), r.stride(0), tokens, choices, width,
                                      slots.data_ptr<int32_t>(), out.data_ptr(), s);
    });
    return out;
}
Tensor expert_dispatch_grad(const Tensor &grad_rows, const Tensor &slots) {
    const char *who = "expert_dispatch_grad";
    Below below;
    check_slots(who, slots);
    const int code = row_type(who, "grad_rows", grad_rows, slots, true);
    on_device(who, grad_rows, {&slots});
    const int64_t tokens = slots.size(0), choices = slots.size(1), width = grad_rows.size(1);
    const Tensor r = rows_of(grad_rows, width);
    Tensor out = at::empty({tokens, width}, r.options());
    call("esgd_expert_dispatch_grad", r, [&](void *s) {
        return c.esgd_expert_dispatch_grad(code, r.data_ptr(), r.stride(0), tokens, choices, width,
                                           slots.data_ptr<int32_t>(), out.data_ptr(), s);
    });
    return out;
}
Tensor expert_combine(const Tensor &rows, const Tensor &weights, const Tensor &slots) {
    const char *who = "expert_combine";
    Below below;
    check_slots(who, slots);
    const Tensor w = weights_of(who, weights, slots);
    const int code = row_type(who, "rows", rows, slots, true);
    on_device(who, rows, {&w, &slots});
    const int64_t tokens = slots.size(0), choices = slots.size(1), width = rows.size(1);
    const Tensor r = rows_of(rows, width);
    Tensor out = at::empty({tokens, width}, r.options());
    call("esgd_expert_combine", r, [&](void *s) {
        return c.esgd_expert_combine(code, r.data_ptr(), r.stride(0), tokens, choices, width,
                                     slots.data_ptr<int32_t>(), w.data_ptr<float>(), out.data_ptr(), s);
    });
    return out;
}
std::tuple<Tensor, Tensor> expert_combine_grad(const Tensor &grad, const Tensor &rows, const Tensor &weights,
                                               const Tensor &slots) {
    const char *who = "expert_combine_grad";
    Below below;
    check_slots(who, slots);
    const Tensor w = weights_of(who, weights, slots);
    const int code = row_type(who, "grad", grad, slots, false);
    row_type(who, "rows", rows, slots, true);
    REFUSE(rows.scalar_type() != grad.scalar_type() || rows.size(1) != grad.size(1), who, ": rows of ", rows.size(1),
           " ", name_of(rows.scalar_type()), " and a gradient of ", grad.size(1), " ", name_of(grad.scalar_type()));
    on_device(who, grad, {&rows, &w, &slots});
    const int64_t tokens = slots.size(0), choices = slots.size(1), width = grad.size(1);
    const Tensor g = rows_of(grad, width), r = rows_of(rows, width);
    Tensor grad_rows = at::empty({tokens * choices, width}, r.options());
    Tensor grad_weights = at::empty({tokens, choices}, r.options().dtype(at::kFloat));
    call("esgd_expert_combine_grad", g, [&](void *s) {
        return c.esgd_expert_combine_grad(code, g.data_ptr(), g.stride(0), r.data_ptr(), r.stride(0), tokens, choices,
                                          width, slots.data_ptr<int32_t>(), w.data_ptr<float>(), grad_rows.data_ptr(),
                                          grad_weights.data_ptr<float>(), s);
    });
    return {grad_rows, grad_weights};
}

// ---- distillation ----
struct Distill {
    int type, top_type, bits;
    Tensor z, top, index, row_grad;   // row_grad in one dimension; undefined: none
    int64_t n, vocab, k;
    float temperature;
    at::IntArrayRef rows;   // the loss's shape, of the caller's logits
};
Distill distill_of(const char *who, const Tensor &logits, const Tensor &top_logits, const Tensor &top_index,
                   double temperature, const Tensor &row_grad) {
    Distill d;
    d.type = float_of(who, "logits", logits);
    d.top_type = float_of(who, "top_logits", top_logits);
    d.bits = bits_of(who, "top_index", top_index);
    const auto shape = logits.sizes(), top_shape = top_logits.sizes();
    REFUSE(shape.size() < 1 || shape.back() < 1, who, ": logits ", shape_of(shape), " have no vocabulary");
    d.rows = shape.slice(0, shape.size() - 1);
    REFUSE(top_shape.size() != shape.size() || top_shape.slice(0, shape.size() - 1) != d.rows ||
               top_index.sizes() != top_shape,
           who, ": logits ", shape_of(shape), ", top_logits ", shape_of(top_shape), " and top_index ",
           shape_of(top_index.sizes()), " do not go together");
    REFUSE(top_shape.back() > ESGD_DISTILL_TOP_MAX, who, ": ", top_shape.back(), " top logits a row, at most ",
           ESGD_DISTILL_TOP_MAX);
    REFUSE(!(temperature >= 1e-4 && temperature <= 1e4), who, ": temperature ", temperature, " outside [1e-4, 1e4]");
    if (row_grad.defined()) {
        float_of(who, "row_grad", row_grad);
        REFUSE(row_grad.scalar_type() != at::kFloat, who, ": row_grad is ", name_of(row_grad.scalar_type()),
               ", float32 is needed");
        REFUSE(row_grad.sizes() != d.rows, who, ": row_grad ", shape_of(row_grad.sizes()), " for rows ", shape_of(d.rows));
    }
    on_device(who, logits, {&top_logits, &top_index, &row_grad});
    d.vocab = shape.back();
    d.z = rows_of(logits, d.vocab);
    d.n = d.z.size(0);
    d.top = top_logits.contiguous();
    d.index = top_index.contiguous();
    d.k = top_shape.back();
    d.temperature = float(temperature);
    if (row_grad.defined()) d.row_grad = row_grad.dim() == 1 ? row_grad : row_grad.reshape({-1});   // an expanded scalar stays one value
    return d;
}

// (loss, stats)
std::tuple<Tensor, Tensor> distill_loss(const Tensor &logits, const Tensor &top_logits, const Tensor &top_index,
                                        double temperature) {
    Below below;
    const Distill d = distill_of("distill_loss", logits, top_logits, top_index, temperature, Tensor());
    const auto f32 = logits.options().dtype(at::kFloat);
    Tensor loss = at::empty(d.rows, f32), stats = at::empty({d.n, 4}, f32), work;
    size_t bytes = 0;
    check(c.esgd_distill_work(d.n, d.vocab, &bytes), "esgd_distill_work");
    if (bytes) work = work_of(logits, bytes);
    call("esgd_distill_loss", d.z, [&](void *s) {
        return c.esgd_distill_loss(d.type, d.z.data_ptr(), d.z.stride(0), d.n, d.vocab, d.top_type, d.top.data_ptr(),
                                   d.bits, d.index.data_ptr(), d.k, d.temperature, loss.data_ptr<float>(),
                                   stats.data_ptr<float>(), bytes ? work.data_ptr() : nullptr, bytes, s);
    });
    return {loss, stats};
}
Tensor distill_grad(const Tensor &logits, const Tensor &top_logits, const Tensor &top_index, double temperature,
                    const Tensor &stats, const Tensor &row_grad) {
    Below below;
    const Distill d = distill_of("distill_loss", logits, top_logits, top_index, temperature, row_grad);
    Tensor out = at::empty(logits.sizes(), logits.options());
    call("esgd_distill_grad", d.z, [&](void *s) {
        return c.esgd_distill_grad(d.type, d.z.data_ptr(), d.z.stride(0), d.n, d.vocab, d.top_type, d.top.data_ptr(),
                                   d.bits, d.index.data_ptr(), d.k, d.temperature, stats.data_ptr<float>(),
                                   d.row_grad.data_ptr<float>(), d.row_grad.stride(0), out.data_ptr(), s);
    });
    return out;
}
std::tuple<Tensor, Tensor> distill_loss_grad(const Tensor &logits, const Tensor &top_logits, const Tensor &top_index,
                                             const Tensor &row_grad, double temperature) {
    Below below;
    const Distill d = distill_of("distill_loss_grad", logits, top_logits, top_index, temperature, row_grad);
    size_t bytes = 0;
    check(c.esgd_distill_work(d.n, d.vocab, &bytes), "esgd_distill_work");
    Tensor loss = at::empty(d.rows, logits.options().dtype(at::kFloat));
    Tensor out = at::empty(logits.sizes(), logits.options());
    const size_t stats_bytes = size_t(d.n) * 16;   // of no use afterwards: with the work memory
    const Tensor work = work_of(logits, stats_bytes + bytes);
    char *w = static_cast<char *>(work.data_ptr());
    call("esgd_distill_loss_grad", d.z, [&](void *s) {
        return c.esgd_distill_loss_grad(d.type, d.z.data_ptr(), d.z.stride(0), d.n, d.vocab, d.top_type,
                                        d.top.data_ptr(), d.bits, d.index.data_ptr(), d.k, d.temperature,
                                        d.row_grad.data_ptr<float>(), d.row_grad.stride(0), loss.data_ptr<float>(),
                                        reinterpret_cast<float *>(w), out.data_ptr(), w + stats_bytes, bytes, s);
    });
    return {loss, out};
}

}  // namespace

PYBIND11_MODULE(_ops, m) {
    m.def("bind", &bind);
    m.def("embedding", &embedding);
    m.def("embedding_grad", &embedding_grad);
    m.def("expert_sort", &expert_sort);
    m.def("expert_dispatch", &expert_dispatch);
    m.def("expert_dispatch_grad", &expert_dispatch_grad);
    m.def("expert_combine", &expert_combine);
    m.def("expert_combine_grad", &expert_combine_grad);
    m.def("distill_loss", &distill_loss);
    m.def("distill_grad", &distill_grad);
    m.def("distill_loss_grad", &distill_loss_grad);
}
