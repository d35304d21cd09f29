// C entry points of the norm behind a residual's addition and of the optimizer (kernels: sa2_norm.hpp, sa2_adamw.hpp).
#include <algorithm>
#include <cmath>
#include <new>
#include <utility>
#include <vector>

#include "sa2.h"
#include "sa2_adamw.hpp"
#include "sa2_norm.hpp"
#include "sa2_status.hpp"

namespace {

using namespace sa2;

constexpr int64_t kMostGroups = 0xffffff;
constexpr int kMostDim = 16384;

int size_of(int type) { return type == SA2_ELEMENT_F32 ? 4 : 2; }

// f(integral_constant L, integral_constant E) for the lanes and pieces that hold a row of `dim` channels
template <typename F>
void with_shape(int dim, F &&f) {
    using std::integral_constant;
    auto go = [&](auto l, auto e) { f(l, e); };
    if (dim <= 32) go(integral_constant<int, 4>{}, integral_constant<int, 1>{});
    else if (dim <= 128) go(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    else if (dim <= 256) go(integral_constant<int, 32>{}, integral_constant<int, 1>{});
    else if (dim <= 512) go(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    else if (dim <= 1024) go(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    else if (dim <= 2048) go(integral_constant<int, 256>{}, integral_constant<int, 1>{});
    else if (dim <= 4096) go(integral_constant<int, 256>{}, integral_constant<int, 2>{});
    else if (dim <= 8192) go(integral_constant<int, 256>{}, integral_constant<int, 4>{});
    else go(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
}

template <typename F>
void with_types(int x, int r, F &&f) {
    using std::integral_constant;
    if (x == kBf16 && r == kBf16) f(integral_constant<int, kBf16>{}, integral_constant<int, kBf16>{});
    else if (x == kBf16) f(integral_constant<int, kBf16>{}, integral_constant<int, kF32>{});
    else if (x == kF16 && r == kF16) f(integral_constant<int, kF16>{}, integral_constant<int, kF16>{});
    else if (x == kF16) f(integral_constant<int, kF16>{}, integral_constant<int, kF32>{});
    else f(integral_constant<int, kF32>{}, integral_constant<int, kF32>{});
}

int rows_of(int dim) {
    int n = 1;
    with_shape(dim, [&](auto l, auto e) { n = NormShape<l.value, e.value>::ROWS; });
    return n;
}

int bwd_groups(int64_t rows, int dim) {
    // sixteen waves a CU (each workgroup leaves a row of partial gradients: with twice as many for the widest rows their sums take 15 us of 135 at 2048 x 16384)
    const int each = rows_of(dim);
    return (int)std::min<int64_t>((rows + each - 1) / each, dim > 8192 ? 256 : 1024);
}

bool element_aligned(const void *p, int type) { return (reinterpret_cast<uintptr_t>(p) & (size_of(type) - 1)) == 0; }

// a contiguous output that begins inside rows of an input, or these inside it.  (Rows that lie apart may have an output between them: of these the first counts.)
bool shared(const void *out, int64_t out_bytes, const void *in, int64_t rows, int64_t row_bytes, int64_t stride_bytes) {
    if (!out || !in) return false;
    const uintptr_t a = reinterpret_cast<uintptr_t>(out), b = reinterpret_cast<uintptr_t>(in);
    return a < b + (stride_bytes == row_bytes ? rows * row_bytes : row_bytes) && b < a + out_bytes;
}

int check_norm(const sa2_norm_problem *p) {
    if (!p) return fail_with(SA2_ERR_NULL_POINTER, "the problem is required");
    if (p->rows < 1 || p->dim < 1) return fail_with(SA2_ERR_BAD_SHAPE, "rows=%lld dim=%d", (long long)p->rows, p->dim);
    if (p->dim > kMostDim) return fail_with(SA2_ERR_UNSUPPORTED, "rows of %d channels, up to %d are covered", p->dim, kMostDim);
    for (const int t : {p->x_type, p->residual_type, p->weight_type})
        if (t < 0 || t > 2) return fail_with(SA2_ERR_UNSUPPORTED, "elements of type %d", t);
    if (p->residual_type != p->x_type && p->residual_type != SA2_ELEMENT_F32) return fail_with(SA2_ERR_UNSUPPORTED, "the residual has the type of x, or fp32");
    if (!(p->eps >= 0.f) || std::isinf(p->eps)) return fail_with(SA2_ERR_BAD_SHAPE, "eps=%g", (double)p->eps);
    if ((p->rows + rows_of(p->dim) - 1) / rows_of(p->dim) > kMostGroups / 4) return fail_with(SA2_ERR_BAD_SHAPE, "rows=%lld: too large for a 1-D grid", (long long)p->rows);
    return SA2_OK;
}

int forward(const sa2_norm_problem *p, const void *x, int64_t x_stride, const void *residual, int64_t residual_stride, const void *weight, int32_t group, bool eight,
            void *y, float *scales, void *total, float *rstd, void *hip_stream) {
    if (const int rc = check_norm(p)) return rc;
    if (!x || !y || (residual && !total) || (eight && !scales)) return fail_with(SA2_ERR_NULL_POINTER, "x, the outputs, and with a residual the sum are required");
    if (!element_aligned(x, p->x_type) || !element_aligned(residual, p->residual_type) || !element_aligned(weight, p->weight_type) || (!eight && !element_aligned(y, p->x_type)) ||
        !element_aligned(total, p->residual_type))
        return fail_with(SA2_ERR_ALIGNMENT, "tensors must be aligned to their elements");
    if (group != 0 && group != 32 && group != 64 && group != 128) return fail_with(SA2_ERR_UNSUPPORTED, "groups of %d channels: 32, 64, 128 or 0 for the row", group);
    const int64_t x_row = (int64_t)p->dim * size_of(p->x_type), r_row = (int64_t)p->dim * size_of(p->residual_type), y_row = eight ? p->dim : x_row;
    for (const auto &[out, row] : {std::pair<const void *, int64_t>(y, y_row), std::pair<const void *, int64_t>(total, r_row)})
        if (shared(out, p->rows * row, x, p->rows, x_row, x_stride * size_of(p->x_type)) || shared(out, p->rows * row, residual, p->rows, r_row, residual_stride * size_of(p->residual_type)))
            return fail_with(SA2_ERR_BAD_SHAPE, "outputs share memory with x or the residual");
    NormParams k{};
    k.x = static_cast<const char *>(x);
    k.r = static_cast<const char *>(residual);
    k.w = static_cast<const char *>(weight);
    k.y = static_cast<char *>(y);
    k.t = static_cast<char *>(total);
    k.rstd = rstd;
    k.rows = p->rows;
    k.x_row = x_stride * size_of(p->x_type);
    k.r_row = residual_stride * size_of(p->residual_type);
    k.dim = p->dim;
    k.w_type = p->weight_type;
    k.eps = p->eps;
    k.scales = scales;
    k.group_lanes = group && group < p->dim ? group / 8 : 0;
    k.groups = group ? (p->dim + group - 1) / group : 1;
    const hipStream_t s = static_cast<hipStream_t>(hip_stream);
    with_types(p->x_type, residual ? p->residual_type : p->x_type, [&](auto tx, auto tr) {
        with_shape(p->dim, [&](auto l, auto e) {
            using S = NormShape<l.value, e.value>;
            const dim3 grid((unsigned)((p->rows + S::ROWS - 1) / S::ROWS));
            if (eight) hipLaunchKernelGGL((norm_kernel<tx.value, tr.value, l.value, e.value, true>), grid, dim3(S::THREADS), 0, s, k);
            else hipLaunchKernelGGL((norm_kernel<tx.value, tr.value, l.value, e.value, false>), grid, dim3(S::THREADS), 0, s, k);
        });
    });
    return launched("norm");
}

// the call's checks; `all`: elements of each kind of launch (type, states in 8 bits)
int check_adamw(const sa2_adamw_tensor *tensors, int64_t count, const sa2_adamw_step *step, double (&all)[3][2]) {
    if (!step || (count > 0 && !tensors)) return fail_with(SA2_ERR_NULL_POINTER, "tensors and step are required");
    if (count < 0 || count > 0x7fffffff) return fail_with(SA2_ERR_BAD_SHAPE, "%lld tensors", (long long)count);
    if (!(step->beta1 >= 0 && step->beta1 < 1) || !(step->beta2 >= 0 && step->beta2 < 1) || !(step->eps >= 0) || !std::isfinite(step->eps) || !std::isfinite(step->lr) ||
        !(step->lr >= 0) || !(step->weight_decay >= 0) || !std::isfinite(step->weight_decay))
        return fail_with(SA2_ERR_BAD_SHAPE, "lr=%g betas=%g, %g eps=%g weight_decay=%g", step->lr, step->beta1, step->beta2, step->eps, step->weight_decay);
    if (!step->step_at && step->step < 1) return fail_with(SA2_ERR_BAD_SHAPE, "step=%lld, the first is 1", (long long)step->step);
    try {
        // what a step writes: no two of these may share memory (workgroups run in no order)
        std::vector<std::pair<uintptr_t, uintptr_t>> written;
        written.reserve(6 * count);
        for (int64_t i = 0; i < count; ++i) {
            const sa2_adamw_tensor &t = tensors[i];
            if (t.n < 1 || t.n > (int64_t)1 << 40 || t.type < 0 || t.type > 2) continue;      // (refused, or skipped, below)
            const int64_t state = t.bits == 8 ? t.n : 4 * t.n, scales = t.bits == 8 ? (t.n + 255) / 256 * 4 : 0;
            const auto add = [&](const void *at, int64_t bytes) {
                if (at && bytes) written.emplace_back(reinterpret_cast<uintptr_t>(at), reinterpret_cast<uintptr_t>(at) + bytes);
            };
            add(t.param, t.n * size_of(t.type));
            add(t.exp_avg, state);
            add(t.exp_avg_sq, state);
            add(t.exp_avg_scales, scales);
            add(t.exp_avg_sq_scales, scales);
            add(t.master, 4 * t.n);
        }
        std::sort(written.begin(), written.end(), [](const auto &a, const auto &b) { return a.first < b.first; });
        for (size_t i = 1; i < written.size(); ++i)
            if (written[i].first < written[i - 1].second) return fail_with(SA2_ERR_BAD_SHAPE, "parameters, masters or states share memory: each may be in the list once");
    } catch (const std::bad_alloc &) {
        return fail_with(SA2_ERR_BAD_SHAPE, "no memory for %lld tensors", (long long)count);
    }
    for (int64_t i = 0; i < count; ++i) {
        const sa2_adamw_tensor &t = tensors[i];
        if (t.n < 0) return fail_with(SA2_ERR_BAD_SHAPE, "tensor %lld of %lld elements", (long long)i, (long long)t.n);
        if (t.type < 0 || t.type > 2 || (t.bits != 32 && t.bits != 8)) return fail_with(SA2_ERR_UNSUPPORTED, "tensor %lld: type %d, states of %d bits", (long long)i, t.type, t.bits);
        if (t.n == 0) continue;
        if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq || (t.bits == 8 && (!t.exp_avg_scales || !t.exp_avg_sq_scales)))
            return fail_with(SA2_ERR_NULL_POINTER, "tensor %lld: parameter, gradient, states and, of 8-bit ones, scales are required", (long long)i);
        const int state = t.bits == 8 ? 0 : 3;
        if (!element_aligned(t.param, t.type) || !element_aligned(t.grad, t.type) || ((reinterpret_cast<uintptr_t>(t.exp_avg) | reinterpret_cast<uintptr_t>(t.exp_avg_sq)) & state) != 0 ||
            !element_aligned(t.master, 2) || !element_aligned(t.exp_avg_scales, 2) || !element_aligned(t.exp_avg_sq_scales, 2))
            return fail_with(SA2_ERR_ALIGNMENT, "tensor %lld: tensors must be aligned to their elements", (long long)i);
        if (t.n > (int64_t)1 << 40) return fail_with(SA2_ERR_BAD_SHAPE, "tensor %lld of %lld elements", (long long)i, (long long)t.n);
        all[t.type][t.bits == 8] += (double)t.n;
    }
    return SA2_OK;
}

}  // namespace

extern "C" {

int sa2_add_rms_norm(const sa2_norm_problem *p, const void *x, int64_t x_stride, const void *residual, int64_t residual_stride, const void *weight, void *normed,
                     void *total, float *rstd, void *hip_stream) {
    return forward(p, x, x_stride, residual, residual_stride, weight, 0, false, normed, nullptr, total, rstd, hip_stream);
}

int sa2_add_rms_norm_8bit(const sa2_norm_problem *p, const void *x, int64_t x_stride, const void *residual, int64_t residual_stride, const void *weight, int32_t group,
                          void *values, float *scales, void *total, void *hip_stream) {
    return forward(p, x, x_stride, residual, residual_stride, weight, group, true, values, scales, total, nullptr, hip_stream);
}

int64_t sa2_add_rms_norm_bwd_workspace_bytes(const sa2_norm_problem *p) {
    if (check_norm(p)) return -1;
    return (int64_t)bwd_groups(p->rows, p->dim) * p->dim * 4;
}

int sa2_add_rms_norm_bwd(const sa2_norm_problem *p, const void *total, int64_t total_stride, const void *weight, const float *rstd, const void *dnormed, int64_t dnormed_stride,
                         const void *dtotal, int64_t dtotal_stride, void *dx, void *dresidual, void *dweight, void *workspace, int64_t workspace_bytes, void *hip_stream) {
    if (const int rc = check_norm(p)) return rc;
    if (!total || !rstd || !dnormed) return fail_with(SA2_ERR_NULL_POINTER, "the sum, rstd and the output's gradient are required");
    if (!element_aligned(total, p->residual_type) || !element_aligned(weight, p->weight_type) || !element_aligned(dnormed, p->x_type) || !element_aligned(dtotal, p->residual_type) ||
        !element_aligned(dx, p->x_type) || !element_aligned(dresidual, p->residual_type) || !element_aligned(dweight, p->weight_type))
        return fail_with(SA2_ERR_ALIGNMENT, "tensors must be aligned to their elements");
    const int groups = bwd_groups(p->rows, p->dim);
    if (dweight && (!workspace || workspace_bytes < (int64_t)groups * p->dim * 4))
        return fail_with(SA2_ERR_BAD_SHAPE, "workspace of %lld bytes, %lld are needed", (long long)(workspace ? workspace_bytes : 0), (long long)groups * p->dim * 4);
    if (dweight && (reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return fail_with(SA2_ERR_ALIGNMENT, "the workspace must be 16-byte aligned");
    const int64_t x_row = (int64_t)p->dim * size_of(p->x_type), r_row = (int64_t)p->dim * size_of(p->residual_type);
    for (const auto &[out, row] : {std::pair<const void *, int64_t>(dx, x_row), std::pair<const void *, int64_t>(dresidual, r_row)})
        if (shared(out, p->rows * row, total, p->rows, r_row, total_stride * size_of(p->residual_type)) ||
            shared(out, p->rows * row, dnormed, p->rows, x_row, dnormed_stride * size_of(p->x_type)) || shared(out, p->rows * row, dtotal, p->rows, r_row, dtotal_stride * size_of(p->residual_type)))
            return fail_with(SA2_ERR_BAD_SHAPE, "gradients that are written share memory with what is read");
    NormParams k{};
    k.x = static_cast<const char *>(total);
    k.w = static_cast<const char *>(weight);
    k.rstd = const_cast<float *>(rstd);
    k.rows = p->rows;
    k.x_row = total_stride * size_of(p->residual_type);
    k.dim = p->dim;
    k.w_type = p->weight_type;
    k.dy = static_cast<const char *>(dnormed);
    k.dy_row = dnormed_stride * size_of(p->x_type);
    k.dt = static_cast<const char *>(dtotal);
    k.dt_row = dtotal_stride * size_of(p->residual_type);
    k.dx = static_cast<char *>(dx);
    k.dr = static_cast<char *>(dresidual);
    k.dw_parts = dweight ? static_cast<float *>(workspace) : nullptr;
    const hipStream_t s = static_cast<hipStream_t>(hip_stream);
    with_types(p->x_type, p->residual_type, [&](auto tx, auto tr) {
        with_shape(p->dim, [&](auto l, auto e) {
            using S = NormShape<l.value, e.value>;
            hipLaunchKernelGGL((norm_bwd_kernel<tx.value, tr.value, l.value, e.value>), dim3((unsigned)groups), dim3(S::THREADS), 0, s, k);
        });
    });
    if (const int rc = launched("norm backward")) return rc;
    if (!dweight) return SA2_OK;
    hipLaunchKernelGGL(norm_dw_kernel, dim3((unsigned)((p->dim + 31) / 32)), dim3(1024), 0, s, k.dw_parts, groups, p->dim, p->weight_type, static_cast<char *>(dweight));
    return launched("norm weight gradient");
}

int sa2_adamw_check(const sa2_adamw_tensor *tensors, int64_t count, const sa2_adamw_step *step) {
    double all[3][2] = {};
    return check_adamw(tensors, count, step, all);
}

int sa2_adamw(const sa2_adamw_tensor *tensors, int64_t count, const sa2_adamw_step *step, void *hip_stream) {
    double all[3][2] = {};
    if (const int rc = check_adamw(tensors, count, step, all)) return rc;
    AdamParams k{};
    k.seed = step->seed;
    k.step = (uint32_t)step->step;
    k.b1 = (float)step->beta1;
    k.c1 = (float)(1 - step->beta1);
    k.b2 = (float)step->beta2;
    k.c2 = (float)(1 - step->beta2);
    k.eps = (float)step->eps;
    k.step_at = step->step_at;
    k.lr_at = step->lr_at;
    k.grad_scale = step->grad_scale;
    k.beta1 = step->beta1;
    k.beta2 = step->beta2;
    k.lr = step->lr;
    k.decay = step->weight_decay;
    if (!step->step_at) {
        const double n = (double)step->step;
        k.keep = (float)(1 - step->lr * step->weight_decay);
        k.rate = (float)((step->lr_at ? 1. : step->lr) / (1 - std::pow(step->beta1, n)));
        k.inv_root = (float)(1 / std::sqrt(1 - std::pow(step->beta2, n)));
    }
    const hipStream_t s = static_cast<hipStream_t>(hip_stream);
    for (int type = 0; type < 3; ++type)
        for (int eight = 0; eight < 2; ++eight) {
            if (all[type][eight] == 0) continue;
            // workgroups enough for a launch of some of the tensors to fill the chip several times over, chunks of 2048 to 16384 elements
            int64_t chunk = 2048;
            while (chunk < 16384 && all[type][eight] > (double)chunk * 16384) chunk *= 2;
            while (all[type][eight] / (double)chunk > (double)kMostGroups / 2) chunk *= 2;
            k.chunk = (int)chunk;
            k.count = 0;
            int64_t chunks = 0;
            auto flush = [&]() -> int {
                if (k.count == 0) return SA2_OK;
                k.first[k.count] = (int32_t)chunks;
                const dim3 grid((unsigned)chunks);
                const auto go = [&](auto tp) {
                    if (eight) hipLaunchKernelGGL((adamw_kernel<tp.value, true>), grid, dim3(256), 0, s, k);
                    else hipLaunchKernelGGL((adamw_kernel<tp.value, false>), grid, dim3(256), 0, s, k);
                };
                if (type == kBf16) go(std::integral_constant<int, kBf16>{});
                else if (type == kF16) go(std::integral_constant<int, kF16>{});
                else go(std::integral_constant<int, kF32>{});
                k.count = 0;
                chunks = 0;
                return launched("AdamW");
            };
            for (int64_t i = 0; i < count; ++i) {
                const sa2_adamw_tensor &t = tensors[i];
                if (t.type != type || (t.bits == 8) != (eight == 1) || t.n == 0) continue;
                const int64_t more = (t.n + chunk - 1) / chunk;
                if (k.count == kAdamTensors || (k.count > 0 && chunks + more > kMostGroups))
                    if (const int rc = flush()) return rc;
                k.tensor[k.count] = {static_cast<char *>(t.param), static_cast<const char *>(t.grad), static_cast<char *>(t.exp_avg), static_cast<char *>(t.exp_avg_sq),
                                     t.exp_avg_scales, t.exp_avg_sq_scales, t.master, t.n};
                k.index[k.count] = (uint32_t)i;
                k.first[k.count++] = (int32_t)chunks;
                chunks += more;
            }
            if (const int rc = flush()) return rc;
        }
    return SA2_OK;
}

}  // extern "C"
