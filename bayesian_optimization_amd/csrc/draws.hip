// Context-free entry point of the draws from scores (include/gpbo.h).  Argument checks, then launches.
#include <algorithm>
#include <cmath>

#include "k_draw.hpp"

using namespace gpbo_static;

namespace {
constexpr int64_t MOST_COLS = (int64_t)1 << 28, MOST_ROWS = INT32_MAX;
}

extern "C" {

int64_t gpbo_draw_static_workspace(int32_t dtype, int64_t rows, int64_t cols, int64_t draws) {
    if (type_bytes(dtype) == 0 || rows < 0 || rows > MOST_ROWS || cols < 1 || cols > MOST_COLS || draws < 0 || draws > MOST_ROWS) return -1;
    if (draw_long(rows, cols) && rows > MOST_LONG_ROWS) return -1;
    switch (dtype) {
        case GPBO_TYPE_F64: return draw_work_bytes<double>(rows, cols);
        case GPBO_TYPE_F32: return draw_work_bytes<float>(rows, cols);
        case GPBO_TYPE_BF16: return draw_work_bytes<bf16>(rows, cols);
        default: return draw_work_bytes<f16>(rows, cols);
    }
}

int gpbo_draw_static(int32_t device, void* stream, int32_t dtype, const void* scores, int64_t score_stride, int64_t rows,
                     int64_t cols, const double* u, int64_t draws, double temperature, int64_t top_k, double top_p, double min_p,
                     const double* params, int64_t* index_out, double* logp_out, void* workspace, int64_t workspace_bytes) {
    const int64_t need = gpbo_draw_static_workspace(dtype, rows, cols, draws);
    if (need < 0 || (rows > 1 && score_stride < cols) || device < 0 || device >= MAX_DEVICES) return GPBO_ERR_BAD_ARG;
    if (!params && (!(temperature >= 0.0) || !std::isfinite(temperature) || top_k < 0 || !(top_p >= 0.0 && top_p <= 1.0) ||
                    !(min_p >= 0.0 && min_p <= 1.0)))
        return GPBO_ERR_BAD_ARG;
    if (rows == 0 || draws == 0) return GPBO_OK;
    if (!scores || !u || !index_out) return GPBO_ERR_BAD_ARG;
    if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255))) return GPBO_ERR_BAD_ARG;
    DeviceGuard guard(device);
    if (!guard.ok) return GPBO_ERR_HIP;
    DrawArgs a{};
    a.scores = scores, a.rows = rows, a.cols = cols, a.stride = score_stride, a.u = u, a.draws = draws;
    a.temperature = temperature, a.top_k = top_k, a.top_p = top_p, a.min_p = min_p, a.params = params;
    a.index = index_out, a.logp = logp_out;
    const hipStream_t st = (hipStream_t)stream;
    hipError_t e;
    switch (dtype) {
        case GPBO_TYPE_F64: e = draw_rows<double>(st, a, (char*)workspace); break;
        case GPBO_TYPE_F32: e = draw_rows<float>(st, a, (char*)workspace); break;
        case GPBO_TYPE_BF16: e = draw_rows<bf16>(st, a, (char*)workspace); break;
        default: e = draw_rows<f16>(st, a, (char*)workspace); break;
    }
    return e == hipSuccess ? GPBO_OK : GPBO_ERR_HIP;
}

}  // extern "C"
