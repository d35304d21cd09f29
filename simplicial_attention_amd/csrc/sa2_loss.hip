// C entry points of the read-out layer's loss (kernels: sa2_linear_ce.hpp).
#include <algorithm>

#include "sa2.h"
#include "sa2_linear_ce.hpp"
#include "sa2_status.hpp"

namespace {

using namespace sa2;

constexpr int64_t kMostGroups = 0xffffff;
// elements between rows: 255 rows on is within 32 bits of bytes
constexpr int64_t kMostStride = SA2_LINEAR_CE_MOST_STRIDE;
constexpr int64_t kMostDzBytes = (int64_t)256 << 20;      // of a piece of dz, where 256 tokens take less

int64_t up_to(int64_t x, int64_t unit) { return (x + unit - 1) / unit * unit; }

// the tile (NB: 64 NB x 64 NB) and the shares of a product of l x r results over k
struct ProductPlan {
    int nb = 2;
    ProductShape shape{};
    int64_t groups() const { return (int64_t)shape.tiles_r * shape.tiles_l * shape.shares; }
};

// Of the tiles and shares whose workgroups fill the chip, those with the least estimated time.  A step of 256 x 256 takes a CU 0.83 us at the power that the
// matrix units draw (1.25 PFLOP/s over all), a workgroup of 256 x 256 9 us more (first loads, epilogue); two workgroups of 128 x 128 on a CU take 0.52 us a step and 4.5 us,
// one alone 0.30 us a step.  Shares write and read their fp32 results (4 TB/s, and a launch).  Measured: gradient of 4096 rows of 1024 channels over 50021 tokens 386 us in
// 256 x 256 with four shares, 467 in 128 x 128 with two; of 1237 rows of 328 channels over 10007 tokens 38 and 24 us.
ProductPlan plan_of(int64_t l, int64_t r, int64_t k, bool shared, bool masked) {
    ProductPlan best;
    double least = 0;
    const int64_t steps = (k + 31) / 32;
    for (const int nb : {2, 4})
        for (int64_t shares = 1; shares <= (shared ? 64 : 1) && (shares == 1 || steps / shares >= 4); shares += shares < 8 ? 1 : shares / 4) {
            const int64_t t = 64 * nb, tiles_l = (l + t - 1) / t, tiles_r = (r + t - 1) / t;
            int64_t per = (steps + shares - 1) / shares;
            if (masked) per = std::min<int64_t>(per, kProductMostSteps);
            const int64_t real = (steps + per - 1) / per, groups = tiles_l * tiles_r * real, slots = nb == 4 ? 256 : 512;
            const double step = nb == 4 ? 0.83 : groups <= 256 ? 0.30 : 0.52, fixed = nb == 4 ? 9 : 4.5, rounds = (double)groups / (double)slots;
            double us = (rounds <= 1 ? 1. : rounds + 0.3) * ((double)per * step + fixed);
            if (real > 1) us += 3 + (double)real * (double)l * (double)r * 8 / 4e6;
            if (best.shape.shares == 0 || us < least) {
                least = us;
                best.nb = nb;
                best.shape = {(int)k, (int)tiles_r, (int)tiles_l, (int)real, (int)per};
            }
        }
    return best;
}

struct CePlan {
    ProductPlan logits, dz, dh, dw;
    int64_t piece = 0, pieces = 0;
    int64_t dz_row = 0, dz_bytes = 0, h_bytes = 0, w_bytes = 0;
    int64_t parts_bytes = 0;
};

int check_problem(const sa2_linear_ce_problem *p) {
    if (!p) return fail_with(SA2_ERR_NULL_POINTER, "the problem is required");
    if (p->rows < 1 || p->rows > 1 << 24 || p->vocab < 1 || p->vocab > 1 << 24 || p->dim < 8 || p->dim > 65536 || p->dim % 8 != 0)
        return fail_with(SA2_ERR_BAD_SHAPE, "rows=%lld vocab=%d (1 to 2^24) dim=%d (multiples of 8 up to 65536)", (long long)p->rows, p->vocab, p->dim);
    if (p->dtype != SA2_ELEMENT_BF16 && p->dtype != SA2_ELEMENT_F16) return fail_with(SA2_ERR_UNSUPPORTED, "hidden rows and weights of type %d: bf16 and fp16 are covered", p->dtype);
    if (p->reduction < 0 || p->reduction > 2) return fail_with(SA2_ERR_BAD_SHAPE, "reduction=%d", p->reduction);
    return SA2_OK;
}

CePlan plan(const sa2_linear_ce_problem &p) {
    CePlan c;
    c.logits = plan_of(p.rows, p.vocab, p.dim, false, false);
    c.parts_bytes = up_to((int64_t)c.logits.shape.tiles_r * 2 * p.rows * 8, 256);
    const int64_t most = std::max<int64_t>(256, kMostDzBytes / (2 * p.rows) / 256 * 256);
    c.pieces = (p.vocab + most - 1) / most;
    c.piece = up_to((p.vocab + c.pieces - 1) / c.pieces, 256);
    c.pieces = (p.vocab + c.piece - 1) / c.piece;
    c.dz = plan_of(p.rows, c.piece, p.dim, false, false);
    c.dh = plan_of(p.rows, p.dim, c.piece, true, false);
    c.dw = plan_of(c.piece, p.dim, p.rows, true, true);
    // (rows of a power of two of bytes would all begin in the same channel of the L2)
    c.dz_row = c.piece * 2 + 256;
    c.dz_bytes = up_to(p.rows * c.dz_row, 256);
    c.h_bytes = c.pieces > 1 || c.dh.shape.shares > 1 ? up_to((int64_t)c.dh.shape.shares * p.rows * p.dim * 4, 256) : 0;
    c.w_bytes = c.dw.shape.shares > 1 ? up_to((int64_t)c.dw.shape.shares * c.piece * p.dim * 4, 256) : 0;
    return c;
}

bool too_large(const CePlan &c) {
    return c.logits.groups() > kMostGroups || c.dz.groups() > kMostGroups || c.dh.groups() > kMostGroups || c.dw.groups() > kMostGroups;
}

int check_rows(const sa2_linear_ce_problem &p, const void *hidden, int64_t hidden_stride, const void *weight, int64_t weight_stride) {
    if (!hidden || !weight) return fail_with(SA2_ERR_NULL_POINTER, "hidden rows and weights are required");
    if (((reinterpret_cast<uintptr_t>(hidden) | reinterpret_cast<uintptr_t>(weight)) & 15) != 0 || hidden_stride % 8 != 0 || weight_stride % 8 != 0)
        return fail_with(SA2_ERR_ALIGNMENT, "rows must be 16-byte aligned");
    if (hidden_stride < 0 || weight_stride < 0 || hidden_stride > kMostStride || weight_stride > kMostStride)
        return fail_with(SA2_ERR_UNSUPPORTED, "rows %lld and %lld elements apart, up to %d are covered", (long long)hidden_stride, (long long)weight_stride, (int)kMostStride);
    return SA2_OK;
}

int check_workspace(const void *workspace, int64_t given, int64_t needed) {
    if (!workspace || given < needed) return fail_with(SA2_ERR_BAD_SHAPE, "workspace of %lld bytes, %lld are needed", (long long)(workspace ? given : 0), (long long)needed);
    if ((reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return fail_with(SA2_ERR_ALIGNMENT, "the workspace must be 16-byte aligned");
    return SA2_OK;
}

int64_t blocks_of(const sa2_linear_ce_problem &p) { return (p.rows + 31) / 32; }
int64_t forward_bytes(const sa2_linear_ce_problem &p, const CePlan &c) { return c.parts_bytes + up_to(p.rows * 4, 256) + up_to(blocks_of(p) * 8, 256) + 256; }
int64_t backward_bytes(const CePlan &c) { return 256 + c.dz_bytes + c.h_bytes + c.w_bytes; }

// f(integral_constant type, integral_constant NB)
template <typename F>
void with_kernel(int type, int nb, F &&f) {
    using std::integral_constant;
    auto go = [&](auto t) { nb == 4 ? f(t, integral_constant<int, 4>{}) : f(t, integral_constant<int, 2>{}); };
    if (type == SA2_ELEMENT_F16) go(integral_constant<int, kF16>{});
    else go(integral_constant<int, kBf16>{});
}

CeParams params_of(const sa2_linear_ce_problem &p, const int64_t *targets) {
    CeParams k{};
    k.rows = (int)p.rows;
    k.vocab = p.vocab;
    k.dim = p.dim;
    k.reduction = p.reduction;
    k.targets = targets;
    k.ignore = p.ignore_index;
    return k;
}

}  // namespace

extern "C" {

int64_t sa2_linear_ce_workspace_bytes(const sa2_linear_ce_problem *p) {
    if (check_problem(p)) return -1;
    const CePlan c = plan(*p);
    return too_large(c) ? -1 : forward_bytes(*p, c);
}

int64_t sa2_linear_ce_bwd_workspace_bytes(const sa2_linear_ce_problem *p) {
    if (check_problem(p)) return -1;
    const CePlan c = plan(*p);
    return too_large(c) ? -1 : backward_bytes(c);
}

int sa2_linear_ce(const sa2_linear_ce_problem *p, const void *hidden, int64_t hidden_stride, const void *weight, int64_t weight_stride, const int64_t *targets, float *loss,
                  float *lse, float *count, uint32_t *mask, void *workspace, int64_t workspace_bytes, void *hip_stream) {
    if (const int rc = check_problem(p)) return rc;
    if (!targets || !loss || !lse || !count || !mask) return fail_with(SA2_ERR_NULL_POINTER, "targets, loss, lse, count and mask are required");
    if (const int rc = check_rows(*p, hidden, hidden_stride, weight, weight_stride)) return rc;
    const CePlan c = plan(*p);
    if (too_large(c)) return fail_with(SA2_ERR_BAD_SHAPE, "rows=%lld vocab=%d dim=%d: too large for a 1-D grid", (long long)p->rows, p->vocab, p->dim);
    if (const int rc = check_workspace(workspace, workspace_bytes, forward_bytes(*p, c))) return rc;
    CeParams k = params_of(*p, targets);
    k.shape = c.logits.shape;
    k.w = {static_cast<const char *>(weight), weight_stride * 2, p->vocab};
    k.h = {static_cast<const char *>(hidden), hidden_stride * 2, (int)p->rows};
    char *ws = static_cast<char *>(workspace);
    k.parts = reinterpret_cast<float2 *>(ws);
    k.at_target = reinterpret_cast<float *>(ws + c.parts_bytes);
    k.sums = reinterpret_cast<float *>(ws + c.parts_bytes + up_to(p->rows * 4, 256));
    k.ticket = reinterpret_cast<uint32_t *>(ws + forward_bytes(*p, c) - 256);
    k.n_parts = 2 * c.logits.shape.tiles_r;
    k.loss = loss;
    k.lse = lse;
    k.count = count;
    k.mask = mask;
    const hipStream_t s = static_cast<hipStream_t>(hip_stream);
    with_kernel(p->dtype, c.logits.nb, [&](auto t, auto nb) { hipLaunchKernelGGL((ce_logits_kernel<t.value, nb.value>), dim3((unsigned)c.logits.groups()), dim3(256), 0, s, k); });
    if (const int rc = launched("logits")) return rc;
    // few parts: a thread a row
    if (k.n_parts <= 16) hipLaunchKernelGGL((ce_merge_kernel<256, 1>), dim3((unsigned)((p->rows + 255) / 256)), dim3(256), 0, s, k);
    else hipLaunchKernelGGL((ce_merge_kernel<32, 32>), dim3((unsigned)blocks_of(*p)), dim3(1024), 0, s, k);
    return launched("cross entropy");
}

int sa2_linear_ce_bwd(const sa2_linear_ce_problem *p, const void *hidden, int64_t hidden_stride, const void *weight, int64_t weight_stride, const int64_t *targets,
                      const float *lse, const float *count, const uint32_t *mask, const float *dloss, void *dhidden, void *dweight, void *workspace, int64_t workspace_bytes,
                      void *hip_stream) {
    if (const int rc = check_problem(p)) return rc;
    if (!targets || !lse || !count || !mask || !dloss) return fail_with(SA2_ERR_NULL_POINTER, "targets, lse, count, mask and the loss's gradient are required");
    if (const int rc = check_rows(*p, hidden, hidden_stride, weight, weight_stride)) return rc;
    if (((reinterpret_cast<uintptr_t>(dhidden) | reinterpret_cast<uintptr_t>(dweight)) & 15) != 0) return fail_with(SA2_ERR_ALIGNMENT, "gradients must be 16-byte aligned");
    const CePlan c = plan(*p);
    if (too_large(c)) return fail_with(SA2_ERR_BAD_SHAPE, "rows=%lld vocab=%d dim=%d: too large for a 1-D grid", (long long)p->rows, p->vocab, p->dim);
    if (const int rc = check_workspace(workspace, workspace_bytes, backward_bytes(c))) return rc;
    if (!dhidden && !dweight) return SA2_OK;
    CeParams k = params_of(*p, targets);
    char *ws = static_cast<char *>(workspace);
    k.lse = const_cast<float *>(lse);
    k.count = const_cast<float *>(count);
    k.mask = const_cast<uint32_t *>(mask);
    k.up = dloss;
    k.most = reinterpret_cast<float *>(ws);
    k.dz = ws + 256;
    k.dz_row = c.dz_row;
    float *const h_parts = reinterpret_cast<float *>(ws + 256 + c.dz_bytes), *const w_parts = reinterpret_cast<float *>(ws + 256 + c.dz_bytes + c.h_bytes);
    const hipStream_t s = static_cast<hipStream_t>(hip_stream);
    if (p->reduction == kCeNone) hipLaunchKernelGGL(ce_most_kernel, dim3(1), dim3(1024), 0, s, dloss, mask, (int)p->rows, reinterpret_cast<float *>(ws));
    const ProductOperand h{static_cast<const char *>(hidden), hidden_stride * 2, (int)p->rows};
    for (int64_t i = 0; i < c.pieces; ++i) {
        const int64_t first = i * c.piece, tokens = std::min<int64_t>(c.piece, p->vocab - first);
        k.first = (int)first;
        const ProductOperand w{static_cast<const char *>(weight) + first * weight_stride * 2, weight_stride * 2, (int)tokens};
        // (the last piece may be shorter)
        ProductPlan dz = c.dz, dw = c.dw;
        dz.shape.tiles_r = (int)((tokens + 64 * dz.nb - 1) / (64 * dz.nb));
        dw.shape.tiles_l = (int)((tokens + 64 * dw.nb - 1) / (64 * dw.nb));
        k.shape = dz.shape;
        k.w = w;
        k.h = h;
        with_kernel(p->dtype, dz.nb, [&](auto t, auto nb) { hipLaunchKernelGGL((ce_dz_kernel<t.value, nb.value>), dim3((unsigned)dz.groups()), dim3(256), 0, s, k); });
        if (dhidden) {
            k.shape = c.dh.shape;
            k.shape.k = (int)tokens;
            k.w = {w.ptr, w.row, p->dim};
            k.h = {k.dz, k.dz_row, (int)p->rows};
            const bool done = i + 1 == c.pieces;
            const CeOutput o{c.h_bytes == 0 ? static_cast<char *>(dhidden) : nullptr, h_parts, (int)p->rows, i > 0, 1};
            with_kernel(p->dtype, c.dh.nb, [&](auto t, auto nb) { 
                const dim3 grid((unsigned)c.dh.groups());
                if (o.out) hipLaunchKernelGGL((ce_dh_kernel<t.value, nb.value, true>), grid, dim3(256), 0, s, k, o);
                else hipLaunchKernelGGL((ce_dh_kernel<t.value, nb.value, false>), grid, dim3(256), 0, s, k, o);
            });
            if (done && c.h_bytes > 0) {
                const dim3 grid((unsigned)((p->rows * p->dim / 4 + 255) / 256));
                with_kernel(p->dtype, 2, [&](auto t, auto) { hipLaunchKernelGGL(ce_combine_kernel<t.value>, grid, dim3(256), 0, s, k, o, static_cast<char *>(dhidden)); });
            }
        }
        if (dweight) {
            k.shape = dw.shape;
            k.w = {h.ptr, h.row, p->dim};
            k.h = {k.dz, k.dz_row, (int)up_to(tokens, 8)};          // (tiles of dz end with zeros)
            char *const out = static_cast<char *>(dweight) + first * p->dim * 2;
            const CeOutput o{c.dw.shape.shares == 1 ? out : nullptr, w_parts, (int)tokens, 0, 0};
            with_kernel(p->dtype, c.dw.nb, [&](auto t, auto nb) { 
                const dim3 grid((unsigned)dw.groups());
                if (o.out) hipLaunchKernelGGL((ce_dw_kernel<t.value, nb.value, true>), grid, dim3(256), 0, s, k, o);
                else hipLaunchKernelGGL((ce_dw_kernel<t.value, nb.value, false>), grid, dim3(256), 0, s, k, o);
            });
            if (c.dw.shape.shares > 1) {
                const dim3 grid((unsigned)((tokens * p->dim / 4 + 255) / 256));
                with_kernel(p->dtype, 2, [&](auto t, auto) { hipLaunchKernelGGL(ce_combine_kernel<t.value>, grid, dim3(256), 0, s, k, o, out); });
            }
        }
        if (const int rc = launched("cross entropy backward")) return rc;
    }
    return SA2_OK;
}

}  // extern "C"
