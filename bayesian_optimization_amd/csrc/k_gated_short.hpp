// Backward pass of the gated unit with many rows, up to 64 columns of x (16 bits: 16) and more hidden units than that (a wide map of a few
// raw inputs).  Nearly all of the traffic is dh and the kept g and u; the tiles for large operands write dg and du four times over and
// multiply mostly padding.  Here dg and du are worked out on the way into the matrix instructions and never stored: once for dx, once for
// the weights' gradients, so the three arrays are read twice and nothing else moves; the products are those of 32 bits for every type (145829 x 30 -> 3235: backward 10.7 -> 3.7 ms, of 2.4 that two
// passes over them take; 1 M x 4 -> 128: 2.7 -> 1.1 ms).
#pragma once

#include "k_gated_narrow.hpp"

namespace gpbo_static {

constexpr int64_t SHORT_COLS = 64;

template <typename T>
struct ShortBack {
    const T *dh, *x, *w[2];
    const float *kg, *ku;
    int64_t dhs, xs, ws, m, k, h;
    int act;
    T* out[2];                    // dx, or dwg and dwu
    int64_t os;
    int splits;
    float* part;                  // [z][split][h][k]
};

// Four neighbouring numbers as they lie in memory (those from `len` on zero): converted where they are used, so that nothing waits for
// the load before.
template <typename T>
struct Four {
    T v[4];
    __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(v, p, sizeof(v)); }
    __device__ __forceinline__ void load(const T* p, int64_t len) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = i < len ? p[i] : from_float<T>(0.0f);
    }
};
template <typename T>
__device__ __forceinline__ void store4(T* p, const f32x4& v, int64_t len) {
    T o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = from_float<T>(v[i]);
    if (len >= 4) __builtin_memcpy(p, o, sizeof(o));
    else
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < len) p[i] = o[i];
}

// dg and du of four neighbours.
template <typename T>
__device__ __forceinline__ void slopes4(const Four<T>& dh, const f32x4& g, const f32x4& u, int act, f32x4& dg, f32x4& du) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a, da;
        activation<T>(g[i], act, a, da);
        const float d = to_float(dh.v[i]);
        dg[i] = d * u[i] * da, du[i] = d * a;
    }
}

// dx = dg wg + du wu: a workgroup has 16 RF rows and all columns, in CF fragments of 16; its waves take slabs of 16 hidden units in turn and
// join their sums through LDS in a fixed order.
template <typename T, int CF>
__global__ __launch_bounds__(256, 2) void k_gated_short_dx(ShortBack<T> g) {
    constexpr int RF = CF <= 3 ? 2 : 1;          // (what two slabs leave of the registers)
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, q = lane >> 4;
    const int64_t row0 = (int64_t)blockIdx.x * (16 * RF);
    struct Slab {
        Four<T> dh[RF];
        f32x4 g[RF], u[RF];
        T w[2][4][CF];
    };
    const T* pd[RF];
    const float *pg[RF], *pu[RF];                // rows behind the last repeat it: not stored
#pragma unroll
    for (int i = 0; i < RF; ++i) {
        const int64_t r = min(row0 + i * 16 + r16, g.m - 1);
        pd[i] = g.dh + r * g.dhs + q * 4, pg[i] = g.kg + r * g.h + q * 4, pu[i] = g.ku + r * g.h + q * 4;
    }
    int col[CF];
#pragma unroll
    for (int j = 0; j < CF; ++j) col[j] = min(j * 16 + r16, (int)g.k - 1);
    f32x4 acc[RF][CF] = {};
    auto load = [&](Slab& s, int64_t t) {
#pragma unroll
        for (int i = 0; i < RF; ++i) {
            s.dh[i].load(pd[i] + t * 16);
            __builtin_memcpy(&s.g[i], pg[i] + t * 16, 16);
            __builtin_memcpy(&s.u[i], pu[i] + t * 16, 16);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t at = (t * 16 + q * 4 + e) * g.ws;
#pragma unroll
            for (int j = 0; j < CF; ++j) s.w[0][e][j] = g.w[0][at + col[j]], s.w[1][e][j] = g.w[1][at + col[j]];
        }
    };
    auto multiply = [&](const Slab& s) {
#pragma unroll
        for (int i = 0; i < RF; ++i) {
            f32x4 d[2];
            slopes4(s.dh[i], s.g[i], s.u[i], g.act, d[0], d[1]);
#pragma unroll
            for (int z = 0; z < 2; ++z)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int j = 0; j < CF; ++j) acc[i][j] = mma4(to_float(s.w[z][e][j]), d[z][e], acc[i][j]);
        }
    };
    const int64_t whole = g.h / 16;
    walk_slabs<Slab>(wave, whole, 4, load, multiply);
    if (g.h % 16 && whole % 4 == wave) {         // the broken last one
        Slab s;
        const int64_t len = g.h - whole * 16 - q * 4;
#pragma unroll
        for (int i = 0; i < RF; ++i) {
            s.dh[i].load(pd[i] + whole * 16, len);
            s.g[i] = load4(pg[i] + whole * 16, len), s.u[i] = load4(pu[i] + whole * 16, len);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < CF; ++j) {
                const int64_t at = (whole * 16 + q * 4 + e) * g.ws + col[j];
                s.w[0][e][j] = e < len ? g.w[0][at] : from_float<T>(0.0f), s.w[1][e][j] = e < len ? g.w[1][at] : from_float<T>(0.0f);
            }
        multiply(s);
    }
    __shared__ f32x4 sums[2][RF * CF][64];
#pragma unroll
    for (int step = 2; step > 0; step >>= 1) {
        if (wave >= step && wave < 2 * step)
#pragma unroll
            for (int i = 0; i < RF; ++i)
#pragma unroll
                for (int j = 0; j < CF; ++j) sums[wave - step][i * CF + j][lane] = acc[i][j];
        __syncthreads();
        if (wave < step)
#pragma unroll
            for (int i = 0; i < RF; ++i)
#pragma unroll
                for (int j = 0; j < CF; ++j) acc[i][j] += sums[wave][i * CF + j][lane];
        __syncthreads();
    }
    if (wave > 0) return;
#pragma unroll
    for (int i = 0; i < RF; ++i) {
        const int64_t row = row0 + i * 16 + r16;
        if (row >= g.m) continue;
#pragma unroll
        for (int j = 0; j < CF; ++j) {
            const int64_t c = j * 16 + q * 4;
            store4(g.out[0] + row * g.os + c, acc[i][j], g.k - c);
        }
    }
}

// dwg = dg^T x, dwu = du^T x: a workgroup has 64 hidden units (the last ones end with the row and may repeat some) and a piece of the rows, whose
// slabs of 4 E rows its waves take in turn.  A lane has four neighbouring hidden units of a row, one for each of four fragments.  (With more than
// 48 columns 28 registers are spilled.)
template <typename T, int CF>
__global__ __launch_bounds__(256, 2) void k_gated_short_dw(ShortBack<T> g) {
    constexpr int E = CF <= 2 ? 4 : 2;           // what two slabs and the sums leave of the registers
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, q = lane >> 4;
    const int64_t h0 = min((int64_t)blockIdx.x * 64, g.h - 64);
    const int64_t slabs = (g.m + 4 * E - 1) / (4 * E), per = (slabs + g.splits - 1) / g.splits;
    const int64_t sb = min((int64_t)blockIdx.y * per, slabs), se = min(sb + per, slabs);
    struct Slab {
        Four<T> dh[E];
        f32x4 g[E], u[E];
        T x[E][CF];
    };
    int col[CF];
#pragma unroll
    for (int j = 0; j < CF; ++j) col[j] = min(j * 16 + r16, (int)g.k - 1);
    f32x4 acc[2][4][CF] = {};
    auto load = [&](Slab& s, int64_t t) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int64_t r = min(t * 4 * E + e * 4 + q, g.m - 1), at = r * g.h + h0 + r16 * 4;
            s.dh[e].load(g.dh + r * g.dhs + h0 + r16 * 4);
            __builtin_memcpy(&s.g[e], g.kg + at, 16);
            __builtin_memcpy(&s.u[e], g.ku + at, 16);
#pragma unroll
            for (int j = 0; j < CF; ++j) s.x[e][j] = g.x[r * g.xs + col[j]];
        }
    };
    auto multiply = [&](const Slab& s) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            f32x4 d[2];
            slopes4(s.dh[e], s.g[e], s.u[e], g.act, d[0], d[1]);
#pragma unroll
            for (int z = 0; z < 2; ++z)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < CF; ++j) acc[z][i][j] = mma4(to_float(s.x[e][j]), d[z][i], acc[z][i][j]);
        }
    };
    const int64_t whole = max(sb, min(se, g.m / (4 * E)));
    walk_slabs<Slab>(sb + wave, whole, 4, load, multiply);
    if (whole < se && (int)((whole - sb) & 3) == wave) {      // the broken last one: rows behind the last as zeros
        Slab s;
        load(s, whole);
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (whole * 4 * E + e * 4 + q >= g.m) {
                s.dh[e].load(g.dh, 0);
                s.g[e] = s.u[e] = f32x4{};
#pragma unroll
                for (int j = 0; j < CF; ++j) s.x[e][j] = from_float<T>(0.0f);
            }
        multiply(s);
    }
    __shared__ f32x4 sums[2][8 * CF][64];
#pragma unroll
    for (int step = 2; step > 0; step >>= 1) {
        if (wave >= step && wave < 2 * step)
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < CF; ++j) sums[wave - step][i * CF + j][lane] = acc[i >> 2][i & 3][j];
        __syncthreads();
        if (wave < step)
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < CF; ++j) acc[i >> 2][i & 3][j] += sums[wave][i * CF + j][lane];
        __syncthreads();
    }
    if (wave > 0) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t row = h0 + r16 * 4 + (i & 3), z = i >> 2;
        float* const part = g.part + ((z * g.splits + blockIdx.y) * g.h + row) * g.k;
        T* const out = (z ? g.out[1] : g.out[0]) + row * g.os;
#pragma unroll
        for (int j = 0; j < CF; ++j) {
            const int64_t c = j * 16 + q * 4;
            if (g.splits > 1) store4(part + c, acc[i >> 2][i & 3][j], g.k - c);
            else store4(out + c, acc[i >> 2][i & 3][j], g.k - c);
        }
    }
}

}  // namespace gpbo_static
