// Host path of the operators of a training step: the norm behind a residual's addition, the read-out layer's loss, and the optimizer.
// Callers: rms_norm.py, cross_entropy.py, adamw.py.
#include <array>

#include "sa2_torch.hpp"

namespace {

void refuse_foreign(const char *what, std::initializer_list<const Tensor *> inputs) {
    for (const Tensor *t : inputs)
        if (t->defined() && foreign(*t)) raise(PyExc_RuntimeError, std::string(what) + " takes plain tensors (no batched, functionalised or forward-mode ones)");
}

// a backward that is itself recorded: its kernels have no derivative
void refuse_second(const char *what) {
    refuse_recorder(what);
    if (at::GradMode::is_enabled()) raise(PyExc_RuntimeError, std::string(what) + " has no second derivative: call its backward without create_graph");
}

// (..., dim) as rows of dim channels that lie `stride` elements apart, copied if they do not
Tensor as_matrix(const Tensor &t, int64_t dim) {
    if (t.dim() == 2 && (t.stride(1) == 1 || dim == 1)) return t;
    bool rows = t.dim() >= 1 && (t.stride(-1) == 1 || dim == 1);
    int64_t next = -1;                       // what the stride of the next dimension has to be (-1: any)
    for (int64_t x = t.dim() - 2; rows && x >= 0; --x) {
        if (t.size(x) == 1) continue;
        rows = next < 0 || t.stride(x) == next;
        next = t.stride(x) * t.size(x);
    }
    return rows ? t.view({-1, dim}) : t.contiguous().view({-1, dim});
}

int64_t row_stride(const Tensor &t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// ---- norm behind a residual's addition
using MaybeTensor = std::optional<Tensor>;

struct NormCall {
    Tensor x, residual, weight;              // matrices; residual and weight may be undefined
    sa2_norm_problem prob{};
    std::vector<int64_t> shape;
};

NormCall norm_call(const char *what, const Tensor &x, const MaybeTensor &residual, const MaybeTensor &weight, std::optional<double> eps) {
    refuse_recorder(what);
    for (const Tensor *t : {&x, residual ? &*residual : nullptr, weight ? &*weight : nullptr}) {
        if (!t) continue;
        refuse_foreign(what, {t});
        if (!t->is_cuda()) raise(PyExc_AssertionError, std::string(what) + " runs on the GPU only");
        if (element_of(*t) < 0) raise(PyExc_TypeError, std::string(what) + " takes bfloat16, float16 and float32 tensors");
        if (t->device() != x.device()) raise(PyExc_ValueError, std::string(what) + ": tensors on " + x.device().str() + " and " + t->device().str());
    }
    if (x.dim() < 1 || x.size(-1) < 1) raise(PyExc_ValueError, std::string(what) + ": rows without channels: " + shape_text(x));
    const int64_t dim = x.size(-1);
    if (residual && residual->sizes() != x.sizes()) raise(PyExc_ValueError, "residual " + shape_text(*residual) + " does not match " + shape_text(x));
    if (residual && residual->scalar_type() != x.scalar_type() && residual->scalar_type() != at::kFloat)
        raise(PyExc_TypeError, "the residual has the dtype of x, or float32");
    if (weight && (weight->dim() != 1 || weight->size(0) != dim)) raise(PyExc_ValueError, "weight " + shape_text(*weight) + " does not match " + std::to_string(dim) + " channels");
    const double e = eps ? *eps : (double)std::numeric_limits<float>::epsilon();
    if (!(e >= 0) || std::isinf(e)) raise(PyExc_ValueError, "eps must be finite and not negative");
    NormCall c;
    c.shape = x.sizes().vec();
    c.prob = {dim ? x.numel() / dim : 0, (int32_t)std::min<int64_t>(dim, INT32_MAX), element_of(x), element_of(residual ? *residual : x),
              weight ? element_of(*weight) : SA2_ELEMENT_F32, (float)e};
    const c10::DeviceGuard guard(x.device());
    if (c.prob.rows > 0) {
        c.x = as_matrix(x, dim);
        if (residual) c.residual = as_matrix(*residual, dim);
    }
    if (weight) c.weight = weight->contiguous();
    return c;
}

// whether the call of a module's norm is one that add_rms_norm does not refuse (functorch's tensors, tangents, subclasses and more rows than a launch takes go through torch)
bool norm_covers(const Tensor &x, const MaybeTensor &residual, const Tensor &weight) {
    for (const Tensor *t : {&x, residual ? &*residual : &x, &weight})
        if (foreign(*t) || t->layout() != at::kStrided || !t->is_cuda() || element_of(*t) < 0 || t->device() != x.device()) return false;
    if (x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > INT32_MAX || (residual && residual->sizes() != x.sizes()) || weight.dim() != 1 || weight.size(0) != x.size(-1)) return false;
    const int type = element_of(x), wide = element_of(residual ? *residual : x);
    const sa2_norm_problem prob{std::max<int64_t>(x.numel() / x.size(-1), 1), (int32_t)x.size(-1), type, wide, element_of(weight), 0};
    return sa2_add_rms_norm_bwd_workspace_bytes(&prob) >= 0;
}

const void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

struct AddNorm : public torch::autograd::Function<AddNorm> {
    // normed, and with a residual the sum; saved: the normalised rows, rstd and weight
    static variable_list run(const NormCall &c, const Tensor &x, const MaybeTensor &residual, variable_list *saved) {
        const c10::DeviceGuard guard(x.device());
        const Tensor normed = at::empty(c.shape, x.options());
        Tensor total, rstd;
        if (residual) total = at::empty(c.shape, residual->options());
        if (saved) rstd = at::empty({c.prob.rows}, x.options().dtype(at::kFloat));
        if (c.prob.rows > 0)
            check(sa2_add_rms_norm(&c.prob, c.x.data_ptr(), row_stride(c.x), ptr(c.residual), residual ? row_stride(c.residual) : 0, ptr(c.weight), normed.data_ptr(),
                                   residual ? total.data_ptr() : nullptr, saved ? static_cast<float *>(rstd.data_ptr()) : nullptr, stream_of(x)));
        if (saved) *saved = {residual ? total : x, rstd, c.weight};
        variable_list out{normed};
        if (residual) out.push_back(total);
        return out;
    }

    static variable_list forward(AutogradContext *ctx, const Tensor &x, const MaybeTensor &residual, const MaybeTensor &weight, std::optional<double> eps) {
        const NormCall c = norm_call("add_rms_norm", x, residual, weight, eps);
        variable_list saved;
        const variable_list out = run(c, x, residual, &saved);
        ctx->save_for_backward(saved);
        ctx->saved_data["types"] = c10::List<int64_t>({c.prob.x_type, c.prob.residual_type, c.prob.weight_type, (int64_t)residual.has_value()});
        ctx->saved_data["eps"] = (double)c.prob.eps;
        ctx->set_materialize_grads(false);
        return out;
    }

    static variable_list backward(AutogradContext *ctx, variable_list ups) {
        refuse_second("add_rms_norm");
        const variable_list s = ctx->get_saved_variables();
        const auto types = ctx->saved_data["types"].toIntVector();
        const bool has_residual = types[3] != 0;
        const Tensor &rows = s[0], &rstd = s[1], &weight = s[2];
        const Tensor up = ups[0], up_total = has_residual ? ups[1] : Tensor();
        for (const Tensor *t : {&up, &up_total})
            if (t->defined()) refuse_foreign("add_rms_norm", {t});
        const c10::DeviceGuard guard(rows.device());
        // (edges are counted over the tensors that were given)
        const bool want_x = ctx->needs_input_grad(0), want_r = has_residual && ctx->needs_input_grad(1), want_w = weight.defined() && ctx->needs_input_grad(has_residual ? 2 : 1);
        const auto x_type = types[0] == SA2_ELEMENT_F32 ? at::kFloat : types[0] == SA2_ELEMENT_F16 ? at::kHalf : at::kBFloat16;
        variable_list grads(4);
        if (!up.defined()) {                  // (the norm's output was not used)
            if (up_total.defined()) {
                if (want_x) grads[0] = up_total.to(x_type);
                if (want_r) grads[1] = up_total;
            }
            return grads;
        }
        const int64_t dim = rows.size(-1), count = dim ? rows.numel() / dim : 0;
        if (want_w) grads[2] = at::empty({dim}, weight.options());
        if (count == 0) {
            if (want_x) grads[0] = at::empty(rows.sizes(), rows.options().dtype(x_type));
            if (want_r) grads[1] = at::empty(rows.sizes(), rows.options());
            if (want_w) grads[2].zero_();
            return grads;
        }
        const sa2_norm_problem prob{count, (int32_t)dim, (int32_t)types[0], (int32_t)types[1], (int32_t)types[2], (float)ctx->saved_data["eps"].toDouble()};
        const bool same = prob.x_type == prob.residual_type;       // (one tensor is the gradient of both)
        if (want_x || (want_r && same)) grads[0] = at::empty(rows.sizes(), rows.options().dtype(x_type));
        if (want_r) grads[1] = same ? grads[0] : at::empty(rows.sizes(), rows.options());
        const Tensor t = as_matrix(rows, dim), g = as_matrix(up, dim), gt = up_total.defined() ? as_matrix(up_total, dim) : Tensor();
        Tensor ws;
        const int64_t bytes = want_w ? sa2_add_rms_norm_bwd_workspace_bytes(&prob) : 0;
        if (bytes > 0) ws = at::empty({bytes}, rows.options().dtype(at::kByte));
        check(sa2_add_rms_norm_bwd(&prob, t.data_ptr(), row_stride(t), ptr(weight), static_cast<float *>(rstd.data_ptr()), g.data_ptr(), row_stride(g), ptr(gt),
                                   gt.defined() ? row_stride(gt) : 0, const_cast<void *>(ptr(grads[0])), want_r && !same ? grads[1].data_ptr() : nullptr,
                                   const_cast<void *>(ptr(grads[2])), const_cast<void *>(ptr(ws)), bytes, stream_of(rows)));
        if (!want_x) grads[0] = Tensor();
        return grads;
    }
};

std::tuple<Tensor, Tensor> add_rms_norm(const Tensor &x, const MaybeTensor &residual, const MaybeTensor &weight, std::optional<double> eps) {
    variable_list out;
    if (in_autograd({&x, residual ? &*residual : &x, weight ? &*weight : &x})) {
        out = AddNorm::apply(x, residual, weight, eps);
    } else {
        out = AddNorm::run(norm_call("add_rms_norm", x, residual, weight, eps), x, residual, nullptr);
    }
    return {out[0], residual ? out[1] : x};
}

std::tuple<Tensor, Tensor, Tensor> add_rms_norm_8bit(const Tensor &x, const MaybeTensor &residual, const MaybeTensor &weight, std::optional<double> eps, int64_t group) {
    refuse_autograd("add_rms_norm_8bit", {&x, residual ? &*residual : &x, weight ? &*weight : &x});
    const NormCall c = norm_call("add_rms_norm_8bit", x, residual, weight, eps);
    if (group != 0 && group != 32 && group != 64 && group != 128) raise(PyExc_ValueError, "groups of " + std::to_string(group) + " channels: 32, 64, 128, or None for whole rows");
    const c10::DeviceGuard guard(x.device());
    auto shape = c.shape;
    const Tensor values = at::empty(shape, x.options().dtype(at::kFloat8_e4m3fn));
    shape.back() = group ? (c.prob.dim + group - 1) / group : 1;
    const Tensor scales = at::empty(shape, x.options().dtype(at::kFloat));
    Tensor total;
    if (residual) total = at::empty(c.shape, residual->options());
    if (c.prob.rows > 0)
        check(sa2_add_rms_norm_8bit(&c.prob, c.x.data_ptr(), row_stride(c.x), ptr(c.residual), residual ? row_stride(c.residual) : 0, ptr(c.weight), (int32_t)group, values.data_ptr(),
                                    static_cast<float *>(scales.data_ptr()), residual ? total.data_ptr() : nullptr, stream_of(x)));
    return {values, scales, residual ? total : x};
}

// ---- cross entropy of a read-out layer
struct LinearCE : public torch::autograd::Function<LinearCE> {
    // Rows of whole 16-byte pieces.  Others are copied, with channels of zeros behind them up to whole steps of the products (32 channels: their lines are read
    // once then, 219 rows of 852 channels over 15737 tokens 35 -> 27 us a pair of products); those of both operands in one launch.  Returns the channels with the zeros.
    static bool in_pieces(const Tensor &m) {
        return m.size(1) % 8 == 0 && reinterpret_cast<uintptr_t>(m.data_ptr()) % 16 == 0 &&
               (m.size(0) <= 1 || (m.stride(0) % 8 == 0 && m.stride(0) >= 0 && m.stride(0) <= SA2_LINEAR_CE_MOST_STRIDE));
    }
    static int64_t pieces(const Tensor &hidden, const Tensor &weight, int64_t dim, Tensor &h, Tensor &w) {
        h = as_matrix(hidden, dim);
        w = as_matrix(weight, dim);
        const int64_t padded = dim % 8 == 0 ? dim : (dim + 31) / 32 * 32;
        sa2_conversion items[2];
        std::array<Tensor, 2> from;
        int count = 0;
        for (Tensor *t : {&h, &w}) {
            if (in_pieces(*t)) continue;
            const Tensor &m = from[count] = *t;
            *t = at::empty({m.size(0), padded}, m.options());
            items[count++] = {{m.data_ptr(), 0, row_stride(m), 0}, {t->data_ptr(), 0, padded, 0}, element_of(m), element_of(m), (int32_t)dim, (int32_t)padded, 1, (int32_t)m.size(0), 1};
        }
        if (count) check(sa2_convert(items, count, stream_of(hidden)));
        return padded;
    }

    struct Call {
        Tensor hidden, weight, targets;
        sa2_linear_ce_problem prob{};
        int64_t dim = 0;
    };

    static Call checked(const Tensor &hidden, const Tensor &weight, const Tensor &targets, int64_t ignore_index, int64_t reduction) {
        refuse_recorder("linear_cross_entropy");
        for (const Tensor *t : {&hidden, &weight, &targets}) {
            refuse_foreign("linear_cross_entropy", {t});
            if (!t->is_cuda()) raise(PyExc_AssertionError, "linear_cross_entropy runs on the GPU only");
            if (t->device() != hidden.device()) raise(PyExc_ValueError, "linear_cross_entropy: tensors on " + hidden.device().str() + " and " + t->device().str());
        }
        if ((hidden.scalar_type() != at::kBFloat16 && hidden.scalar_type() != at::kHalf) || weight.scalar_type() != hidden.scalar_type())
            raise(PyExc_TypeError, "hidden and weight must share one dtype out of bfloat16 and float16");
        if (targets.scalar_type() != at::kLong && targets.scalar_type() != at::kInt) raise(PyExc_TypeError, "targets must be int64 or int32");
        if (weight.dim() != 2 || weight.size(0) < 1 || weight.size(1) < 1 || hidden.dim() < 1 || hidden.size(-1) != weight.size(1))
            raise(PyExc_ValueError, "hidden " + shape_text(hidden) + " does not match weight " + shape_text(weight));
        if (targets.sizes() != hidden.sizes().slice(0, hidden.dim() - 1)) raise(PyExc_ValueError, "targets " + shape_text(targets) + " do not match hidden " + shape_text(hidden));
        Call c;
        c.dim = hidden.size(-1);
        c.prob = {targets.numel(), (int32_t)std::min<int64_t>((c.dim + 7) / 8 * 8, INT32_MAX), (int32_t)std::min<int64_t>(weight.size(0), INT32_MAX), element_of(hidden),
                  (int32_t)reduction, (int32_t)std::min<int64_t>(c.dim, INT32_MAX), ignore_index};
        const c10::DeviceGuard guard(hidden.device());
        if (c.prob.rows > 0) {
            // (before anything is copied, or narrowed)
            if (sa2_linear_ce_workspace_bytes(&c.prob) < 0) check(SA2_ERR_BAD_SHAPE);
            c.prob.dim = (int32_t)pieces(hidden, weight, c.dim, c.hidden, c.weight);
            c.targets = targets.to(at::kLong).contiguous();
        }
        return c;
    }

    // the loss; saved: operands, targets, and what the backward needs of the rows
    static Tensor run(const Call &c, const Tensor &like, variable_list *saved) {
        const c10::DeviceGuard guard(like.device());
        const auto f32 = like.options().dtype(at::kFloat);
        if (c.prob.rows == 0) return c.prob.reduction == 0 ? at::empty(like.sizes(), f32) : at::full({}, c.prob.reduction == 1 ? std::nan("") : 0., f32);
        const Tensor loss = c.prob.reduction == 0 ? at::empty(like.sizes(), f32) : at::empty({}, f32);
        const int64_t blocks = (c.prob.rows + 31) / 32;
        // lse, then the count, then the mask
        const Tensor kept = at::empty({c.prob.rows + 1 + blocks}, f32);
        float *const lse = static_cast<float *>(kept.data_ptr());
        const int64_t bytes = sa2_linear_ce_workspace_bytes(&c.prob);
        Tensor ws;
        if (bytes > 0) ws = at::empty({bytes}, like.options().dtype(at::kByte));
        check(sa2_linear_ce(&c.prob, c.hidden.data_ptr(), row_stride(c.hidden), c.weight.data_ptr(), row_stride(c.weight), static_cast<const int64_t *>(c.targets.data_ptr()),
                            static_cast<float *>(loss.data_ptr()), lse, lse + c.prob.rows, reinterpret_cast<uint32_t *>(lse + c.prob.rows + 1), const_cast<void *>(ptr(ws)), std::max<int64_t>(bytes, 0),
                            stream_of(like)));
        if (saved) *saved = {c.hidden, c.weight, c.targets, kept};
        return loss;
    }

    static Tensor forward(AutogradContext *ctx, const Tensor &hidden, const Tensor &weight, const Tensor &targets, int64_t ignore_index, int64_t reduction) {
        const Call c = checked(hidden, weight, targets, ignore_index, reduction);
        variable_list saved;
        const Tensor loss = run(c, targets, &saved);
        ctx->save_for_backward(saved);
        ctx->saved_data["hidden"] = c10::List<int64_t>(hidden.sizes().vec());
        ctx->saved_data["weight"] = c10::List<int64_t>(weight.sizes().vec());
        ctx->saved_data["problem"] = c10::List<int64_t>({c.prob.rows, c.prob.dim, c.prob.vocab, c.prob.dtype, c.prob.reduction, c.prob.channels, c.prob.ignore_index});
        ctx->saved_data["type"] = (int64_t)hidden.scalar_type();
        return loss;
    }

    static variable_list backward(AutogradContext *ctx, variable_list ups) {
        refuse_second("linear_cross_entropy");
        refuse_foreign("linear_cross_entropy", {&ups[0]});
        const auto n = ctx->saved_data["problem"].toIntVector(), h_shape = ctx->saved_data["hidden"].toIntVector(), w_shape = ctx->saved_data["weight"].toIntVector();
        const sa2_linear_ce_problem prob{n[0], (int32_t)n[1], (int32_t)n[2], (int32_t)n[3], (int32_t)n[4], (int32_t)n[5], n[6]};
        const auto options = ups[0].options().dtype((at::ScalarType)ctx->saved_data["type"].toInt());
        const bool want_h = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
        const c10::DeviceGuard guard(ups[0].device());
        variable_list grads(5);
        if (prob.rows == 0) {
            if (want_h) grads[0] = at::empty(h_shape, options);
            if (want_w) grads[1] = at::zeros(w_shape, options);
            return grads;
        }
        const variable_list s = ctx->get_saved_variables();
        const Tensor &hidden = s[0], &weight = s[1], up = ups[0].contiguous();
        if (want_h) grads[0] = at::empty(h_shape, options);
        if (want_w) grads[1] = at::empty(w_shape, options);
        const int64_t bytes = sa2_linear_ce_bwd_workspace_bytes(&prob);
        const Tensor ws = at::empty({std::max<int64_t>(bytes, 0)}, options.dtype(at::kByte));
        const float *lse = static_cast<const float *>(s[3].data_ptr());
        check(sa2_linear_ce_bwd(&prob, hidden.data_ptr(), row_stride(hidden), weight.data_ptr(), row_stride(weight), static_cast<const int64_t *>(s[2].data_ptr()), lse, lse + prob.rows,
                                reinterpret_cast<const uint32_t *>(lse + prob.rows + 1), static_cast<const float *>(up.data_ptr()), const_cast<void *>(ptr(grads[0])),
                                const_cast<void *>(ptr(grads[1])), ws.data_ptr(), bytes, stream_of(up)));
        return grads;
    }
};

Tensor linear_cross_entropy(const Tensor &hidden, const Tensor &weight, const Tensor &targets, int64_t ignore_index, int64_t reduction) {
    if (in_autograd({&hidden, &weight})) return LinearCE::apply(hidden, weight, targets, ignore_index, reduction);
    return LinearCE::run(LinearCE::checked(hidden, weight, targets, ignore_index, reduction), targets, nullptr);
}

// whether the call of a model's loss is one that linear_cross_entropy does not refuse, the memory of its logits aside
bool loss_covers(const Tensor &hidden, const Tensor &weight, const Tensor &targets) {
    for (const Tensor *t : {&hidden, &weight, &targets})
        if (foreign(*t) || t->layout() != at::kStrided || !t->is_cuda() || t->device() != hidden.device()) return false;
    return weight.dim() == 2 && weight.size(0) >= 1 && weight.size(0) <= 1 << 24 && weight.size(1) >= 1 && weight.size(1) <= 65536 && targets.numel() <= 1 << 24 &&
           (targets.scalar_type() == at::kLong || targets.scalar_type() == at::kInt);
}

// ---- AdamW (lists of a hundred tensors and more: what is done per tensor is kept small)
const Tensor &tensor_of(PyObject *x, const char *name) {
    if (!THPVariable_Check(x)) raise(PyExc_TypeError, std::string(name) + " must be tensors");
    return THPVariable_Unpack(x);
}

bool laid_out_alike(const Tensor &a, const Tensor &b) {
    return a.sizes() == b.sizes() && ((a.is_contiguous() && b.is_contiguous()) || a.strides() == b.strides());
}

// a list or tuple by its items (borrowed; the sequence lives as long as this)
struct Items {
    py::object held;
    PyObject **at = nullptr;
    size_t count = 0;
    explicit Items(const py::handle &x, const char *name) {
        held = py::reinterpret_steal<py::object>(PySequence_Fast(x.ptr(), name));
        if (!held) throw py::error_already_set();
        at = PySequence_Fast_ITEMS(held.ptr());
        count = (size_t)PySequence_Fast_GET_SIZE(held.ptr());
    }
};

void adamw_step(const py::object &params_in, const py::object &grads_in, const py::object &averages_in, const py::object &squares_in, const py::object &masters_in,
                const py::object &step, const py::object &lr, double beta1, double beta2, double eps, double weight_decay, const MaybeTensor &grad_scale, int64_t seed, bool launch) {
    refuse_recorder("adamw_step");
    const Items params(params_in, "params must be a sequence of tensors"), grads(grads_in, "grads must be a sequence of tensors"),
        states[2] = {Items(averages_in, "exp_avgs must be a sequence"), Items(squares_in, "exp_avg_sqs must be a sequence")};
    std::optional<Items> masters;
    if (!masters_in.is_none()) masters.emplace(masters_in, "masters must be a sequence");
    const size_t count = params.count;
    if (grads.count != count || states[0].count != count || states[1].count != count || (masters && masters->count != count))
        raise(PyExc_ValueError, "as many gradients, states and masters as parameters are required");
    std::vector<sa2_adamw_tensor> items;
    std::vector<Tensor> alive;
    std::vector<c10::TensorImpl *> written;
    items.reserve(count);
    written.reserve(6 * count);
    static const c10::DispatchKeySet others({c10::DispatchKey::Batched, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Python,
                                             c10::DispatchKey::Functionalize});
    std::optional<at::Device> device;
    auto on_device = [&](const Tensor &t) {
        if (!t.is_cuda()) raise(PyExc_AssertionError, "adamw_step runs on the GPU only");
        if (!device) device = t.device();
        if (t.device() != *device) raise(PyExc_ValueError, "adamw_step: tensors on " + device->str() + " and " + t.device().str());
        if (t.key_set().has_any(others)) refuse_foreign("adamw_step", {&t});
    };
    for (size_t i = 0; i < count; ++i) {
        const Tensor &p = tensor_of(params.at[i], "parameters"), &given = tensor_of(grads.at[i], "gradients");
        on_device(p);
        on_device(given);
        if (element_of(p) < 0 || given.scalar_type() != p.scalar_type()) raise(PyExc_TypeError, "parameters are bfloat16, float16 or float32, and gradients of the same dtype");
        if (p.layout() != at::kStrided || given.layout() != at::kStrided || !p.is_non_overlapping_and_dense())
            raise(PyExc_ValueError, "parameters and gradients must be dense: " + shape_text(p));
        if (given.sizes() != p.sizes()) raise(PyExc_ValueError, "gradient " + shape_text(given) + " does not match its parameter's " + shape_text(p));
        sa2_adamw_tensor t{};
        t.param = p.data_ptr();
        if (!launch || laid_out_alike(p, given)) {
            t.grad = given.data_ptr();
        } else {
            const c10::DeviceGuard guard(p.device());
            const at::NoGradGuard no_grad;
            alive.push_back(at::empty_strided(p.sizes(), p.strides(), given.options()).copy_(given));
            t.grad = alive.back().data_ptr();
        }
        t.n = p.numel();
        t.type = element_of(p);
        written.push_back(p.unsafeGetTensorImpl());
        const bool eight = PyTuple_Check(states[0].at[i]);
        if (eight != (bool)PyTuple_Check(states[1].at[i])) raise(PyExc_TypeError, "both states of a parameter are tensors, or (values, scales) pairs");
        t.bits = eight ? 8 : 32;
        for (int which = 0; which < 2; ++which) {
            PyObject *const state = states[which].at[i];
            if (eight) {
                if (PyTuple_GET_SIZE(state) != 2) raise(PyExc_TypeError, "states in 8 bits are (values, scales) pairs");
                const Tensor &values = tensor_of(PyTuple_GET_ITEM(state, 0), "states"), &scales = tensor_of(PyTuple_GET_ITEM(state, 1), "scales");
                on_device(values);
                on_device(scales);
                if (values.scalar_type() != at::kFloat8_e4m3fn || scales.scalar_type() != at::kFloat) raise(PyExc_TypeError, "states in 8 bits are float8_e4m3fn values and float32 scales");
                if (values.numel() != t.n || !values.is_contiguous() || scales.numel() != (t.n + 255) / 256 || !scales.is_contiguous())
                    raise(PyExc_ValueError, "states " + shape_text(values) + " with scales " + shape_text(scales) + " do not match a parameter " + shape_text(p) + ": contiguous, one scale for 256 elements");
                (which ? t.exp_avg_sq : t.exp_avg) = values.data_ptr();
                (which ? t.exp_avg_sq_scales : t.exp_avg_scales) = static_cast<float *>(scales.data_ptr());
                written.push_back(values.unsafeGetTensorImpl());
                written.push_back(scales.unsafeGetTensorImpl());
            } else {
                const Tensor &values = tensor_of(state, "states");
                on_device(values);
                if (values.scalar_type() != at::kFloat) raise(PyExc_TypeError, "states are float32 tensors, or (values, scales) pairs in 8 bits");
                if (!laid_out_alike(p, values)) raise(PyExc_ValueError, "state " + shape_text(values) + " is not laid out as its parameter " + shape_text(p));
                (which ? t.exp_avg_sq : t.exp_avg) = values.data_ptr();
                written.push_back(values.unsafeGetTensorImpl());
            }
        }
        if (masters && masters->at[i] != Py_None) {
            const Tensor &m = tensor_of(masters->at[i], "masters");
            on_device(m);
            if (m.scalar_type() != at::kFloat) raise(PyExc_TypeError, "masters are float32");
            if (!laid_out_alike(p, m)) raise(PyExc_ValueError, "master " + shape_text(m) + " is not laid out as its parameter " + shape_text(p));
            t.master = static_cast<float *>(m.data_ptr());
            written.push_back(m.unsafeGetTensorImpl());
        }
        items.push_back(t);
    }
    sa2_adamw_step s{};
    s.beta1 = beta1;
    s.beta2 = beta2;
    s.eps = eps;
    s.weight_decay = weight_decay;
    s.seed = (uint32_t)seed;
    if (THPVariable_Check(step.ptr())) {
        const Tensor &t = THPVariable_Unpack(step.ptr());
        on_device(t);
        if (t.scalar_type() != at::kLong || t.numel() != 1) raise(PyExc_TypeError, "step is a number, or an int64 tensor of one");
        s.step_at = static_cast<const int64_t *>(t.data_ptr());
    } else {
        s.step = step.cast<int64_t>();
        if (s.step < 1) raise(PyExc_ValueError, "step counts from 1");
    }
    if (THPVariable_Check(lr.ptr())) {
        const Tensor &t = THPVariable_Unpack(lr.ptr());
        on_device(t);
        if (t.scalar_type() != at::kFloat || t.numel() != 1) raise(PyExc_TypeError, "lr is a number, or a float32 tensor of one");
        s.lr_at = static_cast<const float *>(t.data_ptr());
    } else {
        s.lr = lr.cast<double>();
    }
    if (grad_scale) {
        on_device(*grad_scale);
        if (grad_scale->scalar_type() != at::kFloat || grad_scale->numel() != 1) raise(PyExc_TypeError, "grad_scale is a float32 tensor of one number");
        s.grad_scale = static_cast<const float *>(grad_scale->data_ptr());
    }
    if (items.empty()) return;
    // (a tensor made in inference mode has no version to count)
    if (!c10::InferenceMode::is_enabled())
        for (c10::TensorImpl *t : written)
            if (t->is_inference()) raise(PyExc_RuntimeError, "adamw_step: a tensor made in inference mode is updated outside it");
    if (!launch) return check(sa2_adamw_check(items.data(), (int64_t)items.size(), &s));
    const c10::DeviceGuard guard(*device);
    check(sa2_adamw(items.data(), (int64_t)items.size(), &s, c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(device->index()).stream()));
    // (a graph that saved one of these sees that it has changed)
    for (c10::TensorImpl *t : written) t->bump_version();
}

}  // namespace

void bind_training(py::module_ &m) {
    m.def("add_rms_norm", &add_rms_norm);
    m.def("add_rms_norm_8bit", &add_rms_norm_8bit);
    m.def("norm_covers", &norm_covers);
    m.def("loss_covers", &loss_covers);
    m.def("linear_cross_entropy", &linear_cross_entropy);
    m.def("adamw_step", &adamw_step);
}
