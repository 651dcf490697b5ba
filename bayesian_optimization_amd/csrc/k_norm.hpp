// Layer norm of the rows of a matrix, forward and backward.
//   mu = mean(x), rstd = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) rstd, y = xh w + b
//   g = dy w;  dx = rstd (g - mean(g) - xh mean(g xh));  dw = sum over rows of dy xh;  db = sum over rows of dy
// Bound by memory: forward reads x and writes y, backward reads x and dy and writes dx, a dozen operations an element.  So
// a row is read once and stays in registers: the centred second moment is taken from there (two sums, no cancellation, all
// in 32 bits), TPR threads share a row in 16-byte packs, and a workgroup walks over rows with weight and bias (and, going
// back, the column sums of dw and db) in registers too.  The column sums of every row group go to the workspace and are
// added by a second launch in a fixed order: no atomics, the same bits every time.
// (Backward at 16384 elements a row spills 7 registers in float32 and float16.)
// Measured: 1 M x 621 bf16 forward 516 us, 5.0 TB/s; 16384 x 4096 bf16 forward + backward 152 us, 4.4 TB/s with x read in both.
#pragma once

#include "static_ops.hpp"

namespace gpbo_static {

// Sum over the TPR threads of a row (TPR <= 64: part of a wave; above: the whole workgroup through LDS, two slots so that one
// barrier a sum is enough as long as consecutive sums alternate the slot).
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* lds) {
    if constexpr (TPR <= 64) {
#pragma unroll
        for (int o = TPR / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
        return v;
    } else {
        v = wave_sum(v);
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) lds[wave] = v;
        __syncthreads();
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) s += lds[i];
        return s;
    }
}

// Two of them with one barrier.
template <int TPR>
__device__ __forceinline__ void row_sum2(float& v, float& u, float* lds_v, float* lds_u) {
    if constexpr (TPR <= 64) {
        v = row_sum<TPR>(v, nullptr), u = row_sum<TPR>(u, nullptr);
    } else {
        v = wave_sum(v), u = wave_sum(u);
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) lds_v[wave] = v, lds_u[wave] = u;
        __syncthreads();
        v = u = 0.0f;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) v += lds_v[i], u += lds_u[i];
    }
}

// Pack c of a row of `cols` elements.  The last pack of a row whose length is no multiple of N is moved back so that it ends
// with the row: it is loaded and stored whole, its first `dup` elements are the pack before's (left out of sums, stored twice
// with the same value).  Rows shorter than one pack go element by element.
template <typename T>
struct Span {
    static constexpr int V = Pack<T>::N;
    int64_t e;
    int dup, len;                              // elements dup .. len are this pack's own; len 0: behind the row's end
    __device__ __forceinline__ Span(int64_t c, int64_t cols) {
        const int64_t s = c * V;
        e = s, dup = 0, len = s < cols ? V : 0;
        if (s < cols && s + V > cols) {
            if (cols >= V) e = cols - V, dup = (int)(s - e);
            else len = (int)cols;
        }
    }
    __device__ __forceinline__ bool own(int i) const { return i >= dup && i < len; }
    __device__ __forceinline__ Pack<T> load(const T* row) const {
        if (len == V) return load_pack(row + e);
        Pack<T> r;
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[i] = i < len ? row[e + i] : from_float<T>(0.0f);
        return r;
    }
    __device__ __forceinline__ void store(T* row, const Pack<T>& p) const {
        if (len == V) {
            store_pack(row + e, p);
            return;
        }
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < len) row[e + i] = p.v[i];
    }
};

struct NormArgs {
    const void *x, *w, *b, *dy;
    void *y, *dx;
    int64_t rows, cols, xs, ys, dys, dxs;      // row strides in elements
    float eps;
    float *mean, *rstd;
    float* part;                               // [groups][2][cols] column sums of dy xh and dy
    int row_blocks;                            // backward: > 0 if further workgroups take the column sums (few rows)
    void *dw, *db;                             // then
};

// Rows of more than TPR * (NCH - 1) and up to TPR * NCH packs: only a thread's last pack can be broken or missing, so only there
// does an element need to be asked whether it counts.  Held as 32-bit numbers from the load on: per element one conversion, two
// additions and two products, then the output -- on a row of a few hundred elements the vector instructions bind as much as memory.
template <typename T, int TPR, int NCH>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void k_norm_fwd(NormArgs a) {
    constexpr int V = Pack<T>::N, BLOCK = TPR > 256 ? TPR : 256, RPB = BLOCK / TPR;
    __shared__ float lds[2][16];
    const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
    const T *w = (const T*)a.w, *b = (const T*)a.b;
    const int cols = (int)a.cols;
    const Span<T> tail(lane + (NCH - 1) * TPR, cols);
    auto at = [&](int k) { return (int64_t)(lane + k * TPR) * V; };
    Pack<T> pw[NCH], pb[NCH];
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
        if (w) pw[k] = k < NCH - 1 ? load_pack(w + at(k)) : tail.load(w);
        if (b) pb[k] = k < NCH - 1 ? load_pack(b + at(k)) : tail.load(b);
    }
    const float n = (float)cols;
    // the trip count is the same for all threads of a workgroup: row sums of wide rows hold barriers
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB) {
        const int64_t r = r0 + group;
        const bool on = r < a.rows;
        const T* x = (const T*)a.x + (on ? r : 0) * a.xs;
        float v[NCH][V];
        float s = 0.0f;
        Pack<T> px[NCH];
#pragma unroll
        for (int k = 0; k < NCH; ++k) px[k] = k < NCH - 1 ? load_pack(x + at(k)) : tail.load(x);
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[k][i] = to_float(px[k].v[i]);
                s += k < NCH - 1 || tail.own(i) ? v[k][i] : 0.0f;
            }
        const float mu = row_sum<TPR>(s, lds[0]) / n;
        float q = 0.0f;
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[k][i] -= mu;
                const float d = k < NCH - 1 || tail.own(i) ? v[k][i] : 0.0f;
                q = fmaf(d, d, q);
            }
        const float rstd = 1.0f / sqrtf(row_sum<TPR>(q, lds[1]) / n + a.eps);
        if (!on) continue;                     // only where TPR <= 64: no barrier is skipped
        T* y = (T*)a.y + r * a.ys;
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            Pack<T> py;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xh = v[k][i] * rstd;
                py.v[i] = from_float<T>(fmaf(xh, w ? to_float(pw[k].v[i]) : 1.0f, b ? to_float(pb[k].v[i]) : 0.0f));
            }
            if (k < NCH - 1) store_pack(y + at(k), py);
            else tail.store(y, py);
        }
        if (lane == 0) {
            if (a.mean) a.mean[r] = mu;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

// Any length: one workgroup a row, three passes over it (the later ones from the caches).
template <typename T>
__global__ __launch_bounds__(1024) void k_norm_fwd_long(NormArgs a) {
    constexpr int V = Pack<T>::N;
    __shared__ float lds[2][16];
    const int64_t chunks = (a.cols + V - 1) / V;
    const float n = (float)a.cols;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = (const T*)a.x + r * a.xs;
        float s = 0.0f;
        for (int64_t c = threadIdx.x; c < chunks; c += 1024) {
            const Span<T> sp(c, a.cols);
            const Pack<T> p = sp.load(x);
            float t = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) t += sp.own(i) ? to_float(p.v[i]) : 0.0f;
            s += t;
        }
        const float mu = row_sum<1024>(s, lds[0]) / n;
        float q = 0.0f;
        for (int64_t c = threadIdx.x; c < chunks; c += 1024) {
            const Span<T> sp(c, a.cols);
            const Pack<T> p = sp.load(x);
            float t = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = to_float(p.v[i]) - mu;
                t += sp.own(i) ? d * d : 0.0f;
            }
            q += t;
        }
        const float rstd = 1.0f / sqrtf(row_sum<1024>(q, lds[1]) / n + a.eps);
        T* y = (T*)a.y + r * a.ys;
        for (int64_t c = threadIdx.x; c < chunks; c += 1024) {
            const Span<T> sp(c, a.cols);
            const Pack<T> p = sp.load(x);
            Pack<T> pw, pb, py;
            if (a.w) pw = sp.load((const T*)a.w);
            if (a.b) pb = sp.load((const T*)a.b);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xh = (to_float(p.v[i]) - mu) * rstd;
                py.v[i] = from_float<T>((a.w ? xh * to_float(pw.v[i]) : xh) + (a.b ? to_float(pb.v[i]) : 0.0f));
            }
            sp.store(y, py);
        }
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[r] = mu;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

// dw and db of 64 columns over all rows, with mean and rstd from the forward pass: what a few rows' column sums need is in the
// caches, and reading it twice is sooner done than a second launch for the sums of sums.
template <typename T, int BLOCK>
__device__ __forceinline__ void norm_columns(const NormArgs& a, int64_t which) {
    __shared__ float sums[2][BLOCK / 64][64];
    const int cl = threadIdx.x & 63, group = threadIdx.x >> 6;
    const int64_t c = which * 64 + cl;
    float w = 0.0f, b = 0.0f;
    if (c < a.cols) {
#pragma unroll 8
        for (int64_t r = group; r < a.rows; r += BLOCK / 64) {
            const float d = to_float(((const T*)a.dy)[r * a.dys + c]);
            w = fmaf(d, (to_float(((const T*)a.x)[r * a.xs + c]) - a.mean[r]) * a.rstd[r], w);
            b += d;
        }
    }
    sums[0][group][cl] = w, sums[1][group][cl] = b;
    __syncthreads();
    if (group > 0 || c >= a.cols) return;
    w = b = 0.0f;
#pragma unroll
    for (int i = 0; i < BLOCK / 64; ++i) w += sums[0][i][cl], b += sums[1][i][cl];
    if (a.dw) ((T*)a.dw)[c] = from_float<T>(w);
    if (a.db) ((T*)a.db)[c] = from_float<T>(b);
}

template <typename T, int TPR, int NCH>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void k_norm_bwd(NormArgs a) {
    constexpr int V = Pack<T>::N, BLOCK = TPR > 256 ? TPR : 256, RPB = BLOCK / TPR;
    const int blocks = a.row_blocks ? a.row_blocks : gridDim.x;
    if ((int)blockIdx.x >= blocks) {
        norm_columns<T, BLOCK>(a, blockIdx.x - blocks);
        return;
    }
    __shared__ float lds[4][16];
    const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
    const T* w = (const T*)a.w;
    const int cols = (int)a.cols;
    const Span<T> tail(lane + (NCH - 1) * TPR, cols);
    auto at = [&](int k) { return (int64_t)(lane + k * TPR) * V; };
    Pack<T> pw[NCH];
    float aw[NCH][V], ab[NCH][V];
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
        if (w) pw[k] = k < NCH - 1 ? load_pack(w + at(k)) : tail.load(w);
#pragma unroll
        for (int i = 0; i < V; ++i) aw[k][i] = ab[k][i] = 0.0f;
    }
    const float n = (float)cols;
    int par = 0;
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)blocks * RPB) {
        const int64_t r = r0 + group;
        const bool on = r < a.rows;
        const int64_t rr = on ? r : 0;
        const T *x = (const T*)a.x + rr * a.xs, *dy = (const T*)a.dy + rr * a.dys;
        Pack<T> px[NCH], pd[NCH];
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            px[k] = k < NCH - 1 ? load_pack(x + at(k)) : tail.load(x);
            pd[k] = k < NCH - 1 ? load_pack(dy + at(k)) : tail.load(dy);
        }
        const float mu = a.mean[rr], rstd = a.rstd[rr];
        float s1 = 0.0f, s2 = 0.0f;
        float xh[NCH][V];
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                xh[k][i] = (to_float(px[k].v[i]) - mu) * rstd;
                const float d = RPB == 1 || on ? to_float(pd[k].v[i]) : 0.0f;      // rows behind the last add nothing
                const float g = w ? d * to_float(pw[k].v[i]) : d;
                const bool own = k < NCH - 1 || tail.own(i);
                s1 += own ? g : 0.0f;
                s2 = fmaf(own ? g : 0.0f, xh[k][i], s2);
                aw[k][i] = fmaf(d, xh[k][i], aw[k][i]);
                ab[k][i] += d;
            }
        row_sum2<TPR>(s1, s2, lds[par], lds[par + 1]);
        par ^= 2;
        const float m1 = s1 / n, m2 = s2 / n;
        if (!on) continue;
        T* dx = (T*)a.dx + r * a.dxs;
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
            Pack<T> po;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = to_float(pd[k].v[i]), g = w ? d * to_float(pw[k].v[i]) : d;
                po.v[i] = from_float<T>(rstd * (g - m1 - xh[k][i] * m2));
            }
            if (k < NCH - 1) store_pack(dx + at(k), po);
            else tail.store(dx, po);
        }
    }
    if (!a.part) return;
    // one pair of column sums a workgroup: row groups of a wave by exchange, waves through LDS, in a fixed order
    if constexpr (TPR < 64) {
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int o = 32; o >= TPR; o >>= 1) {
                    aw[k][i] += __shfl_xor(aw[k][i], o);
                    ab[k][i] += __shfl_xor(ab[k][i], o);
                }
    }
    if constexpr (TPR <= 64) {
        __shared__ float sums[4][2 * NCH * V][64];
        const int wave = threadIdx.x >> 6, wl = threadIdx.x & 63;
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) sums[wave][k * V + i][wl] = aw[k][i], sums[wave][(NCH + k) * V + i][wl] = ab[k][i];
        __syncthreads();
        if (wave > 0 || wl >= TPR) return;
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                aw[k][i] = (sums[0][k * V + i][wl] + sums[1][k * V + i][wl]) + (sums[2][k * V + i][wl] + sums[3][k * V + i][wl]);
                ab[k][i] = (sums[0][(NCH + k) * V + i][wl] + sums[1][(NCH + k) * V + i][wl]) +
                           (sums[2][(NCH + k) * V + i][wl] + sums[3][(NCH + k) * V + i][wl]);
            }
    }
    float* part = a.part + (int64_t)blockIdx.x * 2 * a.cols;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
        const Span<T> sp(lane + k * TPR, cols);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (sp.own(i)) {
                part[sp.e + i] = aw[k][i];
                part[cols + sp.e + i] = ab[k][i];
            }
    }
}

// Any length: the row sums by one workgroup a row, dx in a second pass; dw and db by k_norm_bwd_long_cols.
template <typename T>
__global__ __launch_bounds__(1024) void k_norm_bwd_long(NormArgs a) {
    constexpr int V = Pack<T>::N;
    __shared__ float lds[4][16];
    const int64_t chunks = (a.cols + V - 1) / V;
    const float n = (float)a.cols;
    int par = 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = (const T*)a.x + r * a.xs;
        const T* dy = (const T*)a.dy + r * a.dys;
        const float mu = a.mean[r], rstd = a.rstd[r];
        float s1 = 0.0f, s2 = 0.0f;
        for (int64_t c = threadIdx.x; c < chunks; c += 1024) {
            const Span<T> sp(c, a.cols);
            const Pack<T> px = sp.load(x), pd = sp.load(dy);
            Pack<T> pw;
            if (a.w) pw = sp.load((const T*)a.w);
            float t1 = 0.0f, t2 = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (!sp.own(i)) continue;
                const float g = a.w ? to_float(pd.v[i]) * to_float(pw.v[i]) : to_float(pd.v[i]);
                t1 += g;
                t2 += g * ((to_float(px.v[i]) - mu) * rstd);
            }
            s1 += t1;
            s2 += t2;
        }
        row_sum2<1024>(s1, s2, lds[par], lds[par + 1]);
        par ^= 2;
        const float m1 = s1 / n, m2 = s2 / n;
        T* dx = (T*)a.dx + r * a.dxs;
        for (int64_t c = threadIdx.x; c < chunks; c += 1024) {
            const Span<T> sp(c, a.cols);
            const Pack<T> px = sp.load(x), pd = sp.load(dy);
            Pack<T> pw, po;
            if (a.w) pw = sp.load((const T*)a.w);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float g = a.w ? to_float(pd.v[i]) * to_float(pw.v[i]) : to_float(pd.v[i]);
                po.v[i] = from_float<T>(rstd * (g - m1 - (to_float(px.v[i]) - mu) * rstd * m2));
            }
            sp.store(dx, po);
        }
    }
}

// Column sums of rows too long for registers: a workgroup takes 256 packs' columns and every gridDim.y-th row.
template <typename T>
__global__ __launch_bounds__(256) void k_norm_bwd_long_cols(NormArgs a) {
    constexpr int V = Pack<T>::N;
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c * V >= a.cols) return;
    const Span<T> sp(c, a.cols);
    float aw[V], ab[V];
#pragma unroll
    for (int i = 0; i < V; ++i) aw[i] = ab[i] = 0.0f;
    for (int64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
        const Pack<T> px = sp.load((const T*)a.x + r * a.xs), pd = sp.load((const T*)a.dy + r * a.dys);
        const float mu = a.mean[r], rstd = a.rstd[r];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float d = to_float(pd.v[i]);
            aw[i] += d * ((to_float(px.v[i]) - mu) * rstd);
            ab[i] += d;
        }
    }
    float* part = a.part + (int64_t)blockIdx.y * 2 * a.cols;
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (sp.own(i)) {
            part[sp.e + i] = aw[i];
            part[a.cols + sp.e + i] = ab[i];
        }
}

// dw (blockIdx.y = 0) and db (1) of the columns from `first` on: the groups' partial sums, 16 interleaved running sums a column joined in a
// fixed order.
template <typename T>
__global__ __launch_bounds__(1024) void k_norm_cols(const float* __restrict__ part, int groups, int64_t cols, int64_t first, T* __restrict__ dw,
                                                    T* __restrict__ db) {
    __shared__ float lds[16][64];
    T* out = blockIdx.y ? db : dw;
    if (!out) return;
    const int cl = threadIdx.x & 63, s = threadIdx.x >> 6;
    const int64_t c = first + (int64_t)blockIdx.x * 64 + cl;
    float v = 0.0f;
    if (c < cols) {
        const float* p = part + (int64_t)blockIdx.y * cols + c;
#pragma unroll 8
        for (int g = s; g < groups; g += 16) v += p[(int64_t)g * 2 * cols];
    }
    lds[s][cl] = v;
    __syncthreads();
    if (s == 0 && c < cols) {
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t += lds[i][cl];
        out[c] = from_float<T>(t);
    }
}

// How a row length is laid out: threads a row and packs a thread (0 packs: the any-length kernels).
struct NormPlan {
    int tpr, nch;
    int64_t grid, groups;
    bool few;
};

// Threads a row, by the packs it has: as few as leave a thread at most 5 packs (forward) or 3 (backward, which holds two column
// sums an element as well), so that several short rows share a wave and few of its lanes idle (621 elements of 16 bits, 78 packs:
// 16 threads of 5 packs waste 2 of 80, a wave of 2 packs 50 of 128: 942 -> 525 us on a million rows, 5.0 TB/s); from there a workgroup of
// 256 or 1024, sums through LDS (2048 float32 rows of 12000: 61 -> 33 us against reading them again, with the backward pass 179 -> 96);
// beyond 16384 elements the row does not fit into registers and is read again.
inline NormPlan norm_plan(int64_t rows, int64_t cols, int vec, bool backward) {
    const int64_t packs = ceil_div(cols, vec);
    NormPlan p{};
    const int most_packs = backward ? 3 : 5;
    if (packs <= 8) p.tpr = 8;
    else if (packs <= 16 * most_packs) p.tpr = 16;
    else if (packs <= 128) p.tpr = backward ? 64 : 32;
    else if (packs <= 512) p.tpr = 256;
    else p.tpr = 1024;
    p.nch = packs * vec > 16384 ? 0 : (int)ceil_div(packs, p.tpr);
    const int64_t block = p.tpr > 256 ? p.tpr : 256, rpb = block / p.tpr;
    // forward: as many workgroups as the card holds; backward: fewer, since each leaves column sums behind
    const int64_t most = backward ? (p.tpr == 1024 ? 256 : 1024) : (p.tpr == 1024 ? 512 : 2048);
    p.grid = std::max<int64_t>(1, std::min<int64_t>(ceil_div(rows, rpb), most));
    // few rows: the columns' workgroups read all of them again, 64 columns each (up to 512 rows of at most 1 MB together)
    p.few = backward && p.nch > 0 && rows <= 512 && rows * cols * 16 / vec <= (int64_t)1 << 20;
    p.groups = p.few ? 0 : backward && p.nch == 0 ? std::max<int64_t>(1, std::min<int64_t>(rows, 64)) : p.grid;
    return p;
}

// The kernels that norm_plan names.
template <typename T>
void launch_norm(hipStream_t st, const NormArgs& a, const NormPlan& p, bool backward) {
    const dim3 grid((unsigned)(p.grid + (a.row_blocks ? ceil_div(a.cols, 64) : 0))), block(p.tpr > 256 ? p.tpr : 256);
    auto fwd = [&](auto k) { hipLaunchKernelGGL(k, grid, block, 0, st, a); };
    switch (p.tpr * 8 + p.nch) {
        case 8 * 8 + 1: return backward ? fwd(k_norm_bwd<T, 8, 1>) : fwd(k_norm_fwd<T, 8, 1>);
        case 16 * 8 + 1: return backward ? fwd(k_norm_bwd<T, 16, 1>) : fwd(k_norm_fwd<T, 16, 1>);
        case 16 * 8 + 2: return backward ? fwd(k_norm_bwd<T, 16, 2>) : fwd(k_norm_fwd<T, 16, 2>);
        case 16 * 8 + 3: return backward ? fwd(k_norm_bwd<T, 16, 3>) : fwd(k_norm_fwd<T, 16, 3>);
        case 16 * 8 + 4: return fwd(k_norm_fwd<T, 16, 4>);
        case 16 * 8 + 5: return fwd(k_norm_fwd<T, 16, 5>);
        case 32 * 8 + 3: return fwd(k_norm_fwd<T, 32, 3>);
        case 32 * 8 + 4: return fwd(k_norm_fwd<T, 32, 4>);
        case 64 * 8 + 1: return fwd(k_norm_bwd<T, 64, 1>);
        case 64 * 8 + 2: return fwd(k_norm_bwd<T, 64, 2>);
        case 256 * 8 + 1: return backward ? fwd(k_norm_bwd<T, 256, 1>) : fwd(k_norm_fwd<T, 256, 1>);
        case 256 * 8 + 2: return backward ? fwd(k_norm_bwd<T, 256, 2>) : fwd(k_norm_fwd<T, 256, 2>);
        case 1024 * 8 + 1: return backward ? fwd(k_norm_bwd<T, 1024, 1>) : fwd(k_norm_fwd<T, 1024, 1>);
        case 1024 * 8 + 2: return backward ? fwd(k_norm_bwd<T, 1024, 2>) : fwd(k_norm_fwd<T, 1024, 2>);
        case 1024 * 8 + 3:
        case 1024 * 8 + 4:                     // packs of four 32-bit numbers: 16384 elements are four a thread
            if constexpr (sizeof(T) == 4) {
                if (p.nch == 3) return backward ? fwd(k_norm_bwd<T, 1024, 3>) : fwd(k_norm_fwd<T, 1024, 3>);
                return backward ? fwd(k_norm_bwd<T, 1024, 4>) : fwd(k_norm_fwd<T, 1024, 4>);
            }
            return;                            // (no such plan in 16 bits)
        default: return backward ? fwd(k_norm_bwd_long<T>) : fwd(k_norm_fwd_long<T>);      // p.nch == 0
    }
}

template <typename T>
hipError_t norm_forward(hipStream_t st, const NormArgs& a) {
    if (a.rows == 0) return hipSuccess;
    launch_norm<T>(st, a, norm_plan(a.rows, a.cols, Pack<T>::N, false), false);
    return hipGetLastError();
}

template <typename T>
hipError_t norm_backward(hipStream_t st, NormArgs a, void* dw, void* db) {
    const NormPlan p = norm_plan(a.rows, a.cols, Pack<T>::N, true);
    if (a.rows > 0) {
        if (p.few) {
            a.part = nullptr;
            if (dw || db) a.row_blocks = (int)p.grid, a.dw = dw, a.db = db;
            launch_norm<T>(st, a, p, true);
            return hipGetLastError();
        }
        launch_norm<T>(st, a, p, true);
        if (p.nch == 0 && a.part)
            hipLaunchKernelGGL(k_norm_bwd_long_cols<T>, dim3((unsigned)ceil_div(ceil_div(a.cols, Pack<T>::N), 256), (unsigned)p.groups), dim3(256), 0,
                               st, a);
    }
    constexpr int64_t MOST = (int64_t)1 << 27;      // columns of a launch, which takes fewer than 2^32 threads, 16 a column
    for (int64_t c = 0; (dw || db) && c < a.cols; c += MOST)
        hipLaunchKernelGGL(k_norm_cols<T>, dim3((unsigned)ceil_div(std::min(MOST, a.cols - c), 64), 2), dim3(1024), 0, st, (const float*)a.part,
                           a.rows > 0 ? (int)p.groups : 0, a.cols, c, (T*)dw, (T*)db);
    return hipGetLastError();
}

}  // namespace gpbo_static
