// Context-free entry points of the learned inputs: layer norm and gated unit (include/gpbo.h).  Argument checks, then launches.
#include <algorithm>
#include <cmath>

#include "k_gated_plan.hpp"
#include "k_norm.hpp"

using namespace gpbo_static;

namespace {

constexpr int64_t MOST = INT32_MAX;

bool is_float_type(int32_t t) { return t == GPBO_TYPE_F32 || t == GPBO_TYPE_BF16 || t == GPBO_TYPE_F16; }
bool matrix_ok(int64_t rows, int64_t cols, int64_t stride) {
    return rows >= 0 && rows <= MOST && cols >= 1 && cols <= MOST && (stride >= cols || rows <= 1);
}
bool unit_ok(int64_t rows, int64_t cols, int64_t hidden) {
    return matrix_ok(rows, cols, cols) && matrix_ok(rows, hidden, hidden) && cols <= MOST_ACROSS && hidden <= MOST_ACROSS;
}
bool work_ok(const void* p, int64_t bytes, int64_t need) {
    return need >= 0 && (need == 0 || (p && bytes >= need && (reinterpret_cast<uintptr_t>(p) & 255) == 0));
}
int result(hipError_t e) { return e == hipSuccess ? GPBO_OK : GPBO_ERR_HIP; }

template <typename F>
auto by_type(int32_t dtype, F&& f) {
    switch (dtype) {
        case GPBO_TYPE_F32: return f(float{});
        case GPBO_TYPE_BF16: return f(bf16{});
        default: return f(f16{});
    }
}

GatedArgs unit_of(const void* x, int64_t x_stride, int64_t rows, int64_t cols, const void* wg, const void* wu, int64_t w_stride, int64_t hidden) {
    GatedArgs g{};
    g.a[0] = {x, x_stride, 1}, g.b[0] = {wg, w_stride, 1}, g.b[1] = {wu, w_stride, 1};
    g.m = rows, g.n = hidden, g.k = cols;
    return g;
}

}  // namespace

extern "C" {

int gpbo_layernorm(int32_t device, void* stream, int32_t dtype, const void* x, int64_t x_stride, int64_t rows, int64_t cols,
                   const void* w, const void* b, double eps, void* y, int64_t y_stride, float* mean_out, float* rstd_out) {
    if (!is_float_type(dtype) || !matrix_ok(rows, cols, x_stride) || !matrix_ok(rows, cols, y_stride)) return GPBO_ERR_BAD_ARG;
    if (!(eps >= 0.0) || !std::isfinite(eps) || device < 0 || device >= MAX_DEVICES) return GPBO_ERR_BAD_ARG;
    if (rows == 0) return GPBO_OK;
    if (!x || !y) return GPBO_ERR_BAD_ARG;
    DeviceGuard guard(device);
    if (!guard.ok) return GPBO_ERR_HIP;
    NormArgs a{};
    a.x = x, a.w = w, a.b = b, a.y = y, a.rows = rows, a.cols = cols, a.xs = x_stride, a.ys = y_stride, a.eps = (float)eps;
    a.mean = mean_out, a.rstd = rstd_out;
    return result(by_type(dtype, [&](auto t) { return norm_forward<decltype(t)>((hipStream_t)stream, a); }));
}

int64_t gpbo_layernorm_backward_workspace(int32_t dtype, int64_t rows, int64_t cols) {
    if (!is_float_type(dtype) || !matrix_ok(rows, cols, cols)) return -1;
    if (rows == 0) return 0;
    return norm_plan(rows, cols, (int)(16 / type_bytes(dtype)), true).groups * 2 * cols * 4;
}

int gpbo_layernorm_backward(int32_t device, void* stream, int32_t dtype, const void* dy, int64_t dy_stride, const void* x,
                            int64_t x_stride, int64_t rows, int64_t cols, const void* w, const float* mean, const float* rstd,
                            void* dx, int64_t dx_stride, void* dw, void* db, void* workspace, int64_t workspace_bytes) {
    if (!is_float_type(dtype) || !matrix_ok(rows, cols, x_stride) || !matrix_ok(rows, cols, dy_stride) ||
        !matrix_ok(rows, cols, dx_stride) || device < 0 || device >= MAX_DEVICES)
        return GPBO_ERR_BAD_ARG;
    if (rows > 0 && (!dy || !x || !mean || !rstd || !dx)) return GPBO_ERR_BAD_ARG;
    const bool cols_wanted = dw || db;
    if (cols_wanted && !work_ok(workspace, workspace_bytes, gpbo_layernorm_backward_workspace(dtype, rows, cols))) return GPBO_ERR_BAD_ARG;
    DeviceGuard guard(device);
    if (!guard.ok) return GPBO_ERR_HIP;
    NormArgs a{};
    a.x = x, a.w = w, a.dy = dy, a.dx = dx, a.rows = rows, a.cols = cols, a.xs = x_stride, a.dys = dy_stride, a.dxs = dx_stride;
    a.mean = const_cast<float*>(mean), a.rstd = const_cast<float*>(rstd), a.part = cols_wanted ? (float*)workspace : nullptr;
    return result(by_type(dtype, [&](auto t) { return norm_backward<decltype(t)>((hipStream_t)stream, a, dw, db); }));
}

int64_t gpbo_gated_workspace(int32_t dtype, int64_t rows, int64_t cols, int64_t hidden) {
    if (!is_float_type(dtype) || !unit_ok(rows, cols, hidden)) return -1;
    return by_type(dtype, [&](auto t) { return forward_plan<decltype(t)>(rows, cols, hidden).bytes(); });
}

int64_t gpbo_gated_workspace_for(int32_t dtype, const void* x, int64_t x_stride, int64_t rows, int64_t cols, const void* wg, const void* wu,
                                 int64_t w_stride, int64_t hidden) {
    if (!is_float_type(dtype) || !unit_ok(rows, cols, hidden) || !matrix_ok(rows, cols, x_stride) || !matrix_ok(hidden, cols, w_stride)) return -1;
    const GatedArgs g = unit_of(x, x_stride, rows, cols, wg, wu, w_stride, hidden);
    return by_type(dtype, [&](auto t) { return forward_bytes<decltype(t)>(g); });
}

int gpbo_gated(int32_t device, void* stream, int32_t dtype, int32_t act, const void* x, int64_t x_stride, int64_t rows,
               int64_t cols, const void* wg, const void* wu, int64_t w_stride, int64_t hidden, void* h, int64_t h_stride,
               float* keep_g, float* keep_u, void* workspace, int64_t workspace_bytes) {
    if (!is_float_type(dtype) || (act != GPBO_ACT_SILU && act != GPBO_ACT_GELU) || !matrix_ok(rows, cols, x_stride) ||
        !matrix_ok(hidden, cols, w_stride) || !matrix_ok(rows, hidden, h_stride) || device < 0 || device >= MAX_DEVICES)
        return GPBO_ERR_BAD_ARG;
    if (!!keep_g != !!keep_u || !unit_ok(rows, cols, hidden)) return GPBO_ERR_BAD_ARG;
    if (rows == 0) return GPBO_OK;
    if (!x || !wg || !wu || !h ||
        !work_ok(workspace, workspace_bytes, gpbo_gated_workspace_for(dtype, x, x_stride, rows, cols, wg, wu, w_stride, hidden)))
        return GPBO_ERR_BAD_ARG;
    DeviceGuard guard(device);
    if (!guard.ok) return GPBO_ERR_HIP;
    GatedArgs g = unit_of(x, x_stride, rows, cols, wg, wu, w_stride, hidden);
    g.out[0] = h, g.os = h_stride, g.keep_g = keep_g, g.keep_u = keep_u, g.act = act, g.splits = 1;
    return result(by_type(dtype, [&](auto t) { return gated_forward<decltype(t)>((hipStream_t)stream, g, (char*)workspace); }));
}

int64_t gpbo_gated_backward_workspace(int32_t dtype, int64_t rows, int64_t cols, int64_t hidden) {
    if (!is_float_type(dtype) || !unit_ok(rows, cols, hidden)) return -1;
    return by_type(dtype, [&](auto t) { return backward_plan<decltype(t)>(rows, cols, hidden).bytes(); });
}

int gpbo_gated_backward(int32_t device, void* stream, int32_t dtype, int32_t act, const void* dh, int64_t dh_stride, const void* x,
                        int64_t x_stride, int64_t rows, int64_t cols, const void* wg, const void* wu, int64_t w_stride,
                        int64_t hidden, const float* keep_g, const float* keep_u, void* dx, int64_t dx_stride, void* dwg, void* dwu,
                        int64_t dw_stride, void* workspace, int64_t workspace_bytes) {
    if (!is_float_type(dtype) || (act != GPBO_ACT_SILU && act != GPBO_ACT_GELU) || !matrix_ok(rows, cols, x_stride) ||
        !matrix_ok(hidden, cols, w_stride) || !matrix_ok(rows, hidden, dh_stride) || device < 0 || device >= MAX_DEVICES)
        return GPBO_ERR_BAD_ARG;
    if (!!dwg != !!dwu || (dx && !matrix_ok(rows, cols, dx_stride)) || (dwg && !matrix_ok(hidden, cols, dw_stride))) return GPBO_ERR_BAD_ARG;
    if (!unit_ok(rows, cols, hidden)) return GPBO_ERR_BAD_ARG;
    if (rows > 0 && (!dh || !x || !wg || !wu || !keep_g || !keep_u)) return GPBO_ERR_BAD_ARG;
    if (!work_ok(workspace, workspace_bytes, gpbo_gated_backward_workspace(dtype, rows, cols, hidden))) return GPBO_ERR_BAD_ARG;
    DeviceGuard guard(device);
    if (!guard.ok) return GPBO_ERR_HIP;
    return result(by_type(dtype, [&](auto t) {
        return gated_backward<decltype(t)>((hipStream_t)stream, dh, dh_stride, x, x_stride, wg, wu, w_stride, keep_g, keep_u, rows, cols,
                                           hidden, act, dx, dx_stride, dwg, dwu, dw_stride, (char*)workspace);
    }));
}

}  // extern "C"
