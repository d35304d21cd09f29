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

// the tile (64 nl x 64 nr) and the shares of a product of l x r results over k
struct ProductPlan {
    int nl = 0, nr = 0;
    double us = 0;
    ProductShape shape{};
    int64_t groups() const { return (int64_t)shape.tiles_r * shape.tiles_l * shape.shares; }
};

// What a workgroup takes, in us: a step with few others on the chip, with one on each CU, with as many as fit (the matrix units' power is shared); and the
// first loads and the epilogue.  Measured: logits of 8192 x 32000 over 512 channels 301 us in 128 x 256 (256 x 256: 325, 128 x 128: 373), of 300 x 40000 over 4096 144
// (197, 168); weight's gradient of 25024 x 1024 over 4096 rows 193 us in 256 x 256 (222, 235).
struct ProductCost {
    int nl, nr, per_cu;
    double few, each, most, fixed;
};
// (operands of rows of k; where one is read transposed out of LDS 128 x 256 is slower)
constexpr ProductCost kRowCosts[3] = {{2, 2, 2, 0.28, 0.31, 0.60, 4.2}, {2, 4, 2, 0.45, 0.51, 0.95, 4.5}, {4, 4, 1, 0.65, 0.83, 0.83, 7}};
constexpr ProductCost kTransposedCosts[3] = {{2, 2, 2, 0.28, 0.31, 0.58, 4.2}, {2, 4, 2, 0.55, 0.65, 1.15, 5}, {4, 4, 1, 0.65, 0.83, 0.83, 7}};

double product_us(const ProductCost &c, int64_t groups, int64_t steps) {
    const int64_t slots = 256 * c.per_cu, rest = groups % slots;
    // (where some CUs have two, their time counts)
    const double step = rest <= 256 ? c.few + (c.each - c.few) * (double)rest / 256 : c.most * (0.85 + 0.15 * (double)(rest - 256) / 256);
    return (double)(groups / slots) * ((double)steps * c.most + c.fixed) + (rest ? (double)steps * step + c.fixed : 0);
}

// Of the tiles and shares that there are, those with the least estimated time.  Shares write and read their fp32 results (4 TB/s, and a launch).
// `gradient`: not of the logits, of which a launch more makes what they are wanted for.
ProductPlan plan_of(int64_t l, int64_t r, int64_t k, bool gradient, bool masked, int64_t most_shares = 64) {
    ProductPlan best;
    double least = 0;
    const int64_t steps = (k + 31) / 32;
    for (const ProductCost &c : gradient ? kTransposedCosts : kRowCosts)
        for (int64_t shares = 1; shares <= most_shares && (shares == 1 || steps / shares >= 4); shares += shares < 8 ? 1 : shares / 4) {
            const int64_t tiles_l = (l + 64 * c.nl - 1) / (64 * c.nl), tiles_r = (r + 64 * c.nr - 1) / (64 * c.nr);
            int64_t per = (steps + shares - 1) / shares;
            if (masked) per = std::min<int64_t>(per, kProductMostSteps);
            const int64_t real = (steps + per - 1) / per, groups = tiles_l * tiles_r * real;
            double us = product_us(c, groups, per);
            if (real > 1) us += (gradient ? 3 : 5) + (double)real * (double)l * (double)r * 8 / 4e6;
            if (best.nl == 0 || us < least) {
                least = us;
                best = {c.nl, c.nr, us, {(int)k, (int)tiles_r, (int)tiles_l, (int)real, (int)per}};
            }
        }
    return best;
}

struct CePlan {
    ProductPlan logits, dz, dh, dw;
    int64_t piece = 0, pieces = 0;
    int64_t dz_row = 0, dz_bytes = 0, rows_bytes = 0, h_bytes = 0, w_bytes = 0, z_bytes = 0;
    int64_t parts = 0, parts_bytes = 0, logits_bytes = 0;           // parts: of a row's maximum and sum
};

int check_problem(const sa2_linear_ce_problem *p) {
    if (!p) return fail_with(SA2_ERR_NULL_POINTER, "the problem is required");
    if (p->rows < 1 || p->rows > 1 << 24 || p->vocab < 1 || p->vocab > 1 << 24 || p->dim < 8 || p->dim > 65536 || p->dim % 8 != 0)
        return fail_with(SA2_ERR_BAD_SHAPE, "rows=%lld vocab=%d (1 to 2^24) dim=%d (multiples of 8 up to 65536)", (long long)p->rows, p->vocab, p->dim);
    if (p->dtype != SA2_ELEMENT_BF16 && p->dtype != SA2_ELEMENT_F16) return fail_with(SA2_ERR_UNSUPPORTED, "hidden rows and weights of type %d: bf16 and fp16 are covered", p->dtype);
    if (p->channels < 0 || p->channels > p->dim) return fail_with(SA2_ERR_BAD_SHAPE, "%d channels of %d", p->channels, p->dim);
    if (p->reduction < 0 || p->reduction > 2) return fail_with(SA2_ERR_BAD_SHAPE, "reduction=%d", p->reduction);
    return SA2_OK;
}

// the shares of the logits of `tokens` tokens
int64_t shares_bytes(const ProductPlan &p, int64_t rows, int64_t tokens) { return p.shape.shares > 1 ? up_to(p.shape.shares * rows * up_to(tokens, 8) * 4, 256) : 0; }

CePlan plan(const sa2_linear_ce_problem &p) {
    CePlan c;
    const bool two = p.dtype == SA2_ELEMENT_F16 && p.reduction == kCeNone;              // dz with and without the rows' weights
    const int64_t most = std::max<int64_t>(256, kMostDzBytes / (two ? 4 : 2) / p.rows / 256 * 256);
    c.pieces = (p.vocab + most - 1) / most;
    c.piece = up_to((p.vocab + c.pieces - 1) / c.pieces, 256);
    c.pieces = (p.vocab + c.piece - 1) / c.piece;
    c.dh = plan_of(p.rows, p.dim, c.piece, true, false);
    c.dw = plan_of(c.piece, p.dim, p.rows, true, true);
    c.logits = plan_of(p.rows, p.vocab, p.dim, false, false, 1);
    c.dz = plan_of(p.rows, c.piece, p.dim, false, false, 1);
    // Few tiles of logits over many channels leave most of the chip without work: shares of them take two launches more, which cost a training call of less than 70 us
    // of kernels 5 us of the host's time (6 rows of 832 channels over 2900 tokens: 69 us, 75 in shares; 172 of 3816 over 745: 98 and 74, 5 of 3992 over 1148: 86 and 77,
    // 106 of 1992 over 8439: 96 and 80).
    if (p.rows * p.vocab <= 1 << 24 && c.logits.us + c.dz.us + c.dh.us + c.dw.us > 70) {
        c.logits = plan_of(p.rows, p.vocab, p.dim, false, false);
        c.dz = plan_of(p.rows, c.piece, p.dim, false, false);
    }
    c.parts = c.logits.shape.shares > 1 ? (p.vocab + kCeColumns - 1) / kCeColumns : 2 * c.logits.shape.tiles_r;
    c.parts_bytes = up_to(c.parts * p.rows * 8, 256);
    c.logits_bytes = shares_bytes(c.logits, p.rows, p.vocab);
    c.z_bytes = shares_bytes(c.dz, p.rows, c.piece);
    // (rows of a power of two of bytes would all begin in the same channel of the L2)
    c.dz_row = c.piece * 2 + 256;
    c.dz_bytes = up_to(p.rows * c.dz_row, 256);
    c.rows_bytes = two ? c.dz_bytes : 0;
    c.h_bytes = c.pieces > 1 || c.dh.shape.shares > 1 ? up_to((int64_t)c.dh.shape.shares * p.rows * p.dim * 4, 256) : 0;
    c.w_bytes = c.dw.shape.shares > 1 ? up_to((int64_t)c.dw.shape.shares * c.piece * p.dim * 4, 256) : 0;
    return c;
}

int check_size(const sa2_linear_ce_problem &p, const CePlan &c) {
    if (c.logits.groups() <= kMostGroups && c.dz.groups() <= kMostGroups && c.dh.groups() + 7 + c.dw.groups() <= kMostGroups) return SA2_OK;
    return fail_with(SA2_ERR_BAD_SHAPE, "rows=%lld vocab=%d dim=%d: too large for a 1-D grid", (long long)p.rows, p.vocab, p.dim);
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
int64_t forward_bytes(const sa2_linear_ce_problem &p, const CePlan &c) { return c.logits_bytes + c.parts_bytes + up_to(p.rows * 4, 256) + up_to(blocks_of(p) * 8, 256) + 256; }
int64_t backward_bytes(const CePlan &c) { return 256 + c.dz_bytes + c.rows_bytes + c.h_bytes + c.w_bytes + c.z_bytes; }

// f(integral_constant type, integral_constants nl and nr)
template <typename F>
void with_kernel(int type, const ProductPlan &plan, F &&f) {
    using std::integral_constant;
    using Two = integral_constant<int, 2>;
    using Four = integral_constant<int, 4>;
    auto go = [&](auto t) { plan.nl == 4 ? f(t, Four{}, Four{}) : plan.nr == 4 ? f(t, Two{}, Four{}) : f(t, Two{}, Two{}); };
    if (type == SA2_ELEMENT_F16) go(integral_constant<int, kF16>{});
    else go(integral_constant<int, kBf16>{});
}

// the logits of `tokens` tokens in shares, and what is made of their sums
template <bool DZ>
void shared_logits(int type, const ProductPlan &plan, CeParams k, float *shares, int64_t tokens, hipStream_t s) {
    k.dim = (int)up_to(tokens, 8);
    const CeOutput o{nullptr, shares, k.rows, 0, 0, 0};
    const int chunks = (k.dim + kCeColumns - 1) / kCeColumns;
    with_kernel(type, plan, [&](auto t, auto nl, auto nr) {
        hipLaunchKernelGGL((ce_shares_kernel<t.value, nl.value, nr.value>), dim3((unsigned)plan.groups()), dim3(256), 0, s, k, o);
        hipLaunchKernelGGL((ce_shared_logits_kernel<t.value, DZ>), dim3((unsigned)(((int64_t)k.rows * chunks + 3) / 4)), dim3(256), 0, s, k, o, chunks);
    });
}

// (2^33 results and more: a launch has at most 2^32 threads in one dimension)
dim3 combine_grid(int64_t results, int outputs) {
    const int64_t groups = (results + 1023) / 1024, x = std::min<int64_t>(groups, kMostGroups / 2);
    return dim3((unsigned)x, (unsigned)outputs, (unsigned)((groups + x - 1) / x));
}

CeParams params_of(const sa2_linear_ce_problem &p, const int64_t *targets) {
    CeParams k{};
    k.rows = (int)p.rows;
    k.vocab = p.vocab;
    k.dim = p.dim;
    k.channels = p.channels ? p.channels : p.dim;
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
    return check_size(*p, c) ? -1 : forward_bytes(*p, c);
}

int64_t sa2_linear_ce_bwd_workspace_bytes(const sa2_linear_ce_problem *p) {
    if (check_problem(p)) return -1;
    const CePlan c = plan(*p);
    return check_size(*p, c) ? -1 : backward_bytes(c);
}

int sa2_linear_ce(const sa2_linear_ce_problem *p, const void *hidden, int64_t hidden_stride, const void *weight, int64_t weight_stride, const int64_t *targets, float *loss,
                  float *lse, float *count, uint32_t *mask, void *workspace, int64_t workspace_bytes, void *hip_stream) {
    if (const int rc = check_problem(p)) return rc;
    if (!targets || !loss || !lse || !count || !mask) return fail_with(SA2_ERR_NULL_POINTER, "targets, loss, lse, count and mask are required");
    if (const int rc = check_rows(*p, hidden, hidden_stride, weight, weight_stride)) return rc;
    const CePlan c = plan(*p);
    if (const int rc = check_size(*p, c)) return rc;
    if (const int rc = check_workspace(workspace, workspace_bytes, forward_bytes(*p, c))) return rc;
    CeParams k = params_of(*p, targets);
    k.shape = c.logits.shape;
    k.w = {static_cast<const char *>(weight), weight_stride * 2, p->vocab};
    k.h = {static_cast<const char *>(hidden), hidden_stride * 2, (int)p->rows};
    float *const shares = static_cast<float *>(workspace);
    char *ws = static_cast<char *>(workspace) + c.logits_bytes;
    k.parts = reinterpret_cast<float2 *>(ws);
    k.at_target = reinterpret_cast<float *>(ws + c.parts_bytes);
    k.sums = reinterpret_cast<float *>(ws + c.parts_bytes + up_to(p->rows * 4, 256));
    k.ticket = reinterpret_cast<uint32_t *>(static_cast<char *>(workspace) + forward_bytes(*p, c) - 256);
    k.n_parts = (int)c.parts;
    k.loss = loss;
    k.lse = lse;
    k.count = count;
    k.mask = mask;
    const hipStream_t s = static_cast<hipStream_t>(hip_stream);
    if (c.logits.shape.shares > 1) shared_logits<false>(p->dtype, c.logits, k, shares, p->vocab, s);
    else with_kernel(p->dtype, c.logits, [&](auto t, auto nl, auto nr) { hipLaunchKernelGGL((ce_logits_kernel<t.value, nl.value, nr.value>), dim3((unsigned)c.logits.groups()), dim3(256), 0, s, k); });
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
    // (rows of other channels than whole pieces are written at any alignment of their elements)
    const int unit = p->channels % 8 == 0 ? 15 : 1;
    if (((reinterpret_cast<uintptr_t>(dhidden) | reinterpret_cast<uintptr_t>(dweight)) & unit) != 0) return fail_with(SA2_ERR_ALIGNMENT, "gradients must be 16-byte aligned, or to their elements");
    const CePlan c = plan(*p);
    if (const int rc = check_size(*p, c)) return rc;
    if (const int rc = check_workspace(workspace, workspace_bytes, backward_bytes(c))) return rc;
    if (!dhidden && !dweight) return SA2_OK;
    CeParams k = params_of(*p, targets);
    char *ws = static_cast<char *>(workspace);
    k.lse = const_cast<float *>(lse);
    k.count = const_cast<float *>(count);
    k.mask = const_cast<uint32_t *>(mask);
    k.up = dloss;
    k.most = reinterpret_cast<float *>(ws);
    k.dz = dweight || c.rows_bytes == 0 ? ws + 256 : nullptr;
    k.dz_rows = dhidden && c.rows_bytes > 0 ? ws + 256 + c.dz_bytes : nullptr;
    k.dz_row = c.dz_row;
    float *const h_parts = reinterpret_cast<float *>(ws + 256 + c.dz_bytes + c.rows_bytes), *const w_parts = h_parts + c.h_bytes / 4, *const z_parts = w_parts + c.w_bytes / 4;
    const hipStream_t s = static_cast<hipStream_t>(hip_stream);
    if (p->reduction == kCeNone) hipLaunchKernelGGL(ce_most_kernel, dim3(1), dim3(1024), 0, s, dloss, mask, (int)p->rows, reinterpret_cast<float *>(ws));
    const ProductOperand h{static_cast<const char *>(hidden), hidden_stride * 2, (int)p->rows};
    for (int64_t i = 0; i < c.pieces; ++i) {
        const int64_t first = i * c.piece, tokens = std::min<int64_t>(c.piece, p->vocab - first);
        k.first = (int)first;
        const ProductOperand w{static_cast<const char *>(weight) + first * weight_stride * 2, weight_stride * 2, (int)tokens};
        // (the last piece may be shorter)
        ProductPlan dz = c.dz, dw = c.dw;
        dz.shape.tiles_r = (int)((tokens + 64 * dz.nr - 1) / (64 * dz.nr));
        dw.shape.tiles_l = (int)((tokens + 64 * dw.nl - 1) / (64 * dw.nl));
        k.shape = dz.shape;
        k.w = w;
        k.h = h;
        if (dz.shape.shares > 1) shared_logits<true>(p->dtype, dz, k, z_parts, tokens, s);
        else with_kernel(p->dtype, dz, [&](auto t, auto nl, auto nr) {
            const auto go = [&](auto two) { hipLaunchKernelGGL((ce_dz_kernel<t.value, nl.value, nr.value, two.value>), dim3((unsigned)dz.groups()), dim3(256), 0, s, k); };
            if constexpr (t.value == kF16) k.dz_rows ? go(std::true_type{}) : go(std::false_type{});
            else go(std::false_type{});
        });
        CeParams kh = k, kw = k;
        CeOutput oh{}, ow{};
        CeSum sums[2];
        int count = 0;
        const auto combine = [&](const CeSum &a, const CeSum &b, int outputs) {
            const dim3 grid = combine_grid((int64_t)std::max(a.o.rows, b.o.rows) * p->dim, outputs);
            with_kernel(p->dtype, dz, [&](auto t, auto, auto) { hipLaunchKernelGGL(ce_combine_kernel<t.value>, grid, dim3(256), 0, s, k, a, b); });
        };
        if (dhidden) {
            kh.shape = c.dh.shape;
            kh.shape.k = (int)tokens;
            kh.w = {w.ptr, w.row, p->dim};
            kh.h = {k.dz_rows ? k.dz_rows : k.dz, k.dz_row, (int)p->rows};
            oh = {c.h_bytes == 0 ? static_cast<char *>(dhidden) : nullptr, h_parts, (int)p->rows, i > 0, 1, k.dz_rows != nullptr};
            if (c.h_bytes > 0 && i + 1 == c.pieces) sums[count++] = {oh, static_cast<char *>(dhidden), c.dh.shape.shares, p->dim};
        }
        if (dweight) {
            kw.shape = dw.shape;
            kw.w = {h.ptr, h.row, p->dim};
            kw.h = {k.dz, k.dz_row, (int)up_to(tokens, 8)};          // (tiles of dz end with zeros)
            char *const out = static_cast<char *>(dweight) + first * k.channels * 2;
            ow = {c.dw.shape.shares == 1 ? out : nullptr, w_parts, (int)tokens, 0, 0, 0};
            if (!ow.out) sums[count++] = {ow, out, dw.shape.shares, p->dim};
        }
        if (dhidden && dweight && c.dh.nr == 2 && dw.nr == 2) {
            const dim3 grid((unsigned)(up_to(c.dh.groups(), 8) + dw.groups()));
            with_kernel(p->dtype, dz, [&](auto t, auto, auto) {
                const auto go = [&](auto h_direct, auto w_direct) {
                    hipLaunchKernelGGL((ce_gradients_kernel<t.value, h_direct.value, w_direct.value>), grid, dim3(256), 0, s, kh, oh, kw, ow, (int)c.dh.groups());
                };
                if (oh.out) ow.out ? go(std::true_type{}, std::true_type{}) : go(std::true_type{}, std::false_type{});
                else ow.out ? go(std::false_type{}, std::true_type{}) : go(std::false_type{}, std::false_type{});
            });
            if (count > 0) combine(sums[0], sums[count - 1], count);
        } else {
            // (shares are added up while the caches hold them: 300 rows of 4096 channels over 40000 tokens 9.1 us, behind both products 13.3)
            if (dhidden) {
                with_kernel(p->dtype, c.dh, [&](auto t, auto nl, auto nr) {
                    const dim3 grid((unsigned)c.dh.groups());
                    if (oh.out) hipLaunchKernelGGL((ce_dh_kernel<t.value, nl.value, nr.value, true>), grid, dim3(256), 0, s, kh, oh);
                    else hipLaunchKernelGGL((ce_dh_kernel<t.value, nl.value, nr.value, false>), grid, dim3(256), 0, s, kh, oh);
                });
                if (count > 0 && sums[0].out == dhidden) combine(sums[0], sums[0], 1);
            }
            if (dweight) {
                with_kernel(p->dtype, dw, [&](auto t, auto nl, auto nr) {
                    const dim3 grid((unsigned)dw.groups());
                    if (ow.out) hipLaunchKernelGGL((ce_dw_kernel<t.value, nl.value, nr.value, true>), grid, dim3(256), 0, s, kw, ow);
                    else hipLaunchKernelGGL((ce_dw_kernel<t.value, nl.value, nr.value, false>), grid, dim3(256), 0, s, kw, ow);
                });
                if (!ow.out) combine(sums[count - 1], sums[count - 1], 1);
            }
        }
        if (const int rc = launched("cross entropy backward")) return rc;
    }
    return SA2_OK;
}

}  // extern "C"
