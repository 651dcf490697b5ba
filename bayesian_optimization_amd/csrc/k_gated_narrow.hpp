// The gated unit in 32 bits with many rows and up to 64 hidden units (a map of a large pool of rows to a few learned features).  The 128 x
// 128 tiles of large operands would be empty for the most part there, and x, which is nearly all of the traffic, would be read
// several times and packed first.  A 16x16x4 instruction holds the matrix unit for 32 cycles and takes one number a lane: fragments
// straight from memory, 16 bytes a lane, keep it busy without LDS and at any alignment, and either index of an operand may be
// the contiguous one, so nothing is transposed.  The two projections stand side by side as one product of 2 h columns (h in
// eights): x is read once forward, and once and dx written once back.  Bound by memory up to some 16 hidden units, beyond by the matrix
// instructions and the loads that feed them (1 M x 621 -> 24: forward 0.99 ms, 2.5 TB/s of x; backward 1.90; 114765 x 483 -> 64: 0.20
// and 0.40 ms, 70 TFLOP/s).
#pragma once

#include "k_gated.hpp"

namespace gpbo_static {

constexpr int64_t NARROW_HIDDEN = 64, NARROW_STRIDE = 1 << 22;      // (64 rows of 16 MB: lanes' offsets stay below 2^31 bytes)

__device__ __forceinline__ f32x4 mma4(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// `bytes` from an address that all lanes share: one register a lane.
template <typename V>
__device__ __forceinline__ void load_at(V& v, const float* base, uint32_t bytes) {
    __builtin_memcpy(&v, (const char*)base + bytes, sizeof(V));
}
// Four neighbouring numbers, those from `len` on zero.
__device__ __forceinline__ f32x4 load4(const float* p, int64_t len) {
    f32x4 v = {};
    if (len >= 4) __builtin_memcpy(&v, p, 16);
    else
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < len) v[i] = p[i];
    return v;
}

// Loads of the next slab in front of the products of this one, two sets of registers in turn.  Behind the last slab it is loaded again:
// loads under a condition would make the wait in front of the products one for all of them.
template <typename Slab, typename L, typename M>
__device__ __forceinline__ void walk_slabs(int64_t first, int64_t last, int64_t by, L&& load, M&& multiply) {
    const int64_t count = (last - first + by - 1) / by;
    if (count <= 0) return;
    Slab f0, f1;
    load(f0, first);
    int64_t s = 0;
    for (; s + 1 < count; s += 2) {
        load(f1, first + (s + 1) * by);
        __builtin_amdgcn_sched_barrier(0);
        multiply(f0);
        load(f0, first + min(s + 2, count - 1) * by);
        __builtin_amdgcn_sched_barrier(0);
        multiply(f1);
    }
    if (s < count) multiply(f0);
}

// Forward: a wave has 32 rows of x and all hidden units, in F fragments of 16 weight rows: the first half wg's, the others wu's, or, for
// odd F, eight rows of each in turn (row r is hidden unit 8 f + r / 2, of wu for odd r).  Either way a lane ends up with g and u
// of the same hidden units.
template <int F>
__global__ __launch_bounds__(256, 2) void k_gated_narrow(GatedArgs g) {
    constexpr bool ODD = F % 2;
    constexpr int RF = 2, H = ODD ? F : F / 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, q = lane >> 4;
    const int64_t row0 = ((int64_t)blockIdx.x * 4 + wave) * (16 * RF);
    if (row0 >= g.m) return;
    struct Slab {
        f32x4 a[RF], b[F];
    };
    const float *const xb = (const float*)g.a[0].p + row0 * g.a[0].sr, *const w0 = (const float*)g.b[0].p, *const w1 = (const float*)g.b[1].p;
    const float* const mine = r16 & 1 ? w1 : w0;
    uint32_t oa[RF], ob[H];                      // rows behind the last and hidden units behind the last repeat it: not stored
#pragma unroll
    for (int i = 0; i < RF; ++i) oa[i] = (uint32_t)((min((int64_t)i * 16 + r16, g.m - 1 - row0) * g.a[0].sr + q * 4) * 4);
#pragma unroll
    for (int f = 0; f < H; ++f) ob[f] = (uint32_t)((min((int64_t)(ODD ? f * 8 + r16 / 2 : f * 16 + r16), g.n - 1) * g.b[0].sr + q * 4) * 4);
    auto weights = [&](int f, int64_t k) { return (const char*)((ODD ? mine : f < H ? w0 : w1) + k) + ob[f % H]; };
    f32x4 acc[RF][F] = {};
    auto load = [&](Slab& s, int64_t k) {
#pragma unroll
        for (int i = 0; i < RF; ++i) load_at(s.a[i], xb + k * 16, oa[i]);
#pragma unroll
        for (int f = 0; f < F; ++f) __builtin_memcpy(&s.b[f], weights(f, k * 16), 16);
    };
    auto multiply = [&](const Slab& s) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int i = 0; i < RF; ++i)
#pragma unroll
                for (int f = 0; f < F; ++f) acc[i][f] = mma4(s.b[f][e], s.a[i][e], acc[i][f]);
    };
    walk_slabs<Slab>(0, g.k / 16, 1, load, multiply);
    if (g.k % 16) {
        const int64_t k = g.k / 16 * 16, len = g.k - k - q * 4;
        Slab s;
#pragma unroll
        for (int i = 0; i < RF; ++i) s.a[i] = load4((const float*)((const char*)(xb + k) + oa[i]), len);
#pragma unroll
        for (int f = 0; f < F; ++f) s.b[f] = load4((const float*)weights(f, k), len);
        multiply(s);
    }
    constexpr int N = ODD ? 2 : 4;               // neighbouring outputs a lane has
#pragma unroll
    for (int i = 0; i < RF; ++i) {
        const int64_t row = row0 + i * 16 + r16;
        if (row >= g.m) continue;
#pragma unroll
        for (int f = 0; f < H; ++f) {
            const int64_t col = f * 4 * N + q * N, len = g.n - col;
            float gv[N], uv[N], hv[N];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                gv[e] = ODD ? acc[i][f][2 * e] : acc[i][f][e], uv[e] = ODD ? acc[i][f][2 * e + 1] : acc[i][f + F - H][e];
                hv[e] = activate<float>(gv[e], g.act) * uv[e];
            }
            float *p = (float*)g.out[0] + row * g.os + col, *kg = g.keep_g + row * g.n + col, *ku = g.keep_u + row * g.n + col;
            if (len >= N) {
                __builtin_memcpy(p, hv, sizeof(hv));
                if (g.keep_g) __builtin_memcpy(kg, gv, sizeof(gv)), __builtin_memcpy(ku, uv, sizeof(uv));
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (e < len) {
                        p[e] = hv[e];
                        if (g.keep_g) kg[e] = gv[e], ku[e] = uv[e];
                    }
            }
        }
    }
}

// Backward: row r of d holds dg of row r, zeros up to hp, du, zeros up to 2 hp = 16 F.
struct NarrowBack {
    const float* d;
    int64_t hp, m, k, h;
    const float *w[2], *x;
    int64_t ws, xs;
    float* out[2];                // dx, or dwg and dwu
    int64_t os;
    int splits;
    float* part;                  // [z][split][h][k]
};

// d itself.
__global__ __launch_bounds__(256) void k_gated_narrow_slopes(const float* __restrict__ dh, int64_t dhs, const float* __restrict__ kg,
                                                             const float* __restrict__ ku, int64_t m, int64_t h, int act, float* __restrict__ d, int64_t hp) {
    const int64_t packs = hp / 4;
    for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < m * packs; id += (int64_t)gridDim.x * 256) {
        const int64_t row = id / packs, c = id % packs * 4, len = h - c;
        const f32x4 dv = load4(dh + row * dhs + c, len), gv = load4(kg + row * h + c, len), uv = load4(ku + row * h + c, len);
        f32x4 og, ou;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float a, da;
            activation<float>(gv[i], act, a, da);
            og[i] = i < len ? dv[i] * uv[i] * da : 0.0f;
            ou[i] = i < len ? dv[i] * a : 0.0f;
        }
        __builtin_memcpy(d + row * 2 * hp + c, &og, 16);
        __builtin_memcpy(d + row * 2 * hp + hp + c, &ou, 16);
    }
}

// dx = d [wg; wu]: a wave keeps 16 RF rows of d in registers and walks over the columns, 64 at a time (the last 64 end with the row and
// may repeat some).  Number e of a lane's four of d meets weight row 4 (lane / 16) + e of a slab of 16, of which the lane has four
// neighbouring columns, one for each of four fragments.  Lane 4 a + b has columns 16 b + 4 a: output r of the four lanes of a row
// is then 16 neighbouring columns, stored by one instruction (with columns in the order of the lanes 194 us instead of 100 for
// 114765 x 483 with 4 hidden units).
template <int RF, int F>
__global__ __launch_bounds__(256, 2) void k_gated_narrow_dx(NarrowBack g) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, q = lane >> 4;
    const int64_t row0 = ((int64_t)blockIdx.x * 4 + wave) * (16 * RF), tiles = (g.k + 63) / 64;
    if (row0 >= g.m) return;
    struct Slab {
        f32x4 b[4];
    };
    f32x4 a[F][RF];
#pragma unroll
    for (int i = 0; i < RF; ++i) {
        const float* p = g.d + min(row0 + i * 16 + r16, g.m - 1) * (16 * F) + q * 4;
#pragma unroll
        for (int s = 0; s < F; ++s) __builtin_memcpy(&a[s][i], p + s * 16, 16);
    }
    const int mine = (lane & 3) * 16 + (r16 >> 2) * 4;
    constexpr bool ODD = F % 2;                  // the middle slab then holds eight rows of each weight matrix
    // first weight row of a slab's rows of this lane, and how many of its four exist
    auto up = [&](int s) { return (ODD ? s * 16 + q * 4 >= (int)g.hp : s >= F / 2) ? 1 : 0; };
    auto first = [&](int s) { return s * 16 + q * 4 - up(s) * (int)g.hp; };
    auto walk = [&](auto is_short) {
        constexpr bool SHORT = is_short.value;
        auto load = [&](Slab& f, int s, int64_t c) {
            const float* w = (up(s) ? g.w[1] : g.w[0]) + c;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t at = (uint32_t)((min(first(s) + e, (int)g.h - 1) * (int)g.ws + mine) * 4);
                if constexpr (SHORT) f.b[e] = load4((const float*)((const char*)w + at), g.k - mine);
                else load_at(f.b[e], w, at);
            }
        };
        auto column = [&](int64_t t) { return SHORT ? (int64_t)0 : min(t * 64, g.k - 64); };
        Slab now, next;
        load(now, 0, column(blockIdx.y));          // (gridDim.y <= tiles)
        for (int64_t t = blockIdx.y; t < tiles; t += gridDim.y) {
            const int64_t c = column(t), after = column(t + gridDim.y < tiles ? t + gridDim.y : t);
            f32x4 acc[RF][4] = {};
#pragma unroll
            for (int s = 0; s < F; ++s) {
                load(next, (s + 1) % F, s + 1 < F ? c : after);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // rows behind the last repeat it; d is zero there, but zero times an infinite weight is not
                    if (first(s) + e >= (int)g.h) now.b[e] = f32x4{};
#pragma unroll
                    for (int i = 0; i < RF; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[i][j] = mma4(now.b[e][j], a[s][i][e], acc[i][j]);
                }
                now = next;
            }
#pragma unroll
            for (int i = 0; i < RF; ++i) {
                const int64_t row = row0 + i * 16 + r16;
                if (row >= g.m) continue;
                float* p = g.out[0] + row * g.os + c;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int64_t at = r * 16 + q * 4;
                    const f32x4 v = {acc[i][0][r], acc[i][1][r], acc[i][2][r], acc[i][3][r]};
                    if (!SHORT || at + 4 <= g.k) __builtin_memcpy(p + at, &v, 16);
                    else
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (at + j < g.k) p[at + j] = v[j];
                }
            }
        }
    };
    if (g.k < 64) walk(std::true_type{});
    else walk(std::false_type{});
}

// [dwg; dwu] = d^T x: a workgroup has all 16 F rows x 64 columns of a piece of the contraction, whose slabs of 4 E rows of x its waves take
// in turn and join through LDS in a fixed order.  A lane has F neighbouring numbers of a row of d and four of a row of x.
template <int F>
__global__ __launch_bounds__(256, 2) void k_gated_narrow_dw(NarrowBack g) {
    constexpr int E = F <= 4 ? 4 : 2;            // what two slabs and the sums of 16 F x 64 leave of the registers
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, q = lane >> 4;
    const int64_t col0 = g.k < 64 ? 0 : min((int64_t)blockIdx.x * 64, g.k - 64);
    const int64_t slabs = (g.m + 4 * E - 1) / (4 * E), per = (slabs + g.splits - 1) / g.splits;
    const int64_t sb = min((int64_t)blockIdx.y * per, slabs), se = min(sb + per, slabs);
    struct Mine {
        float v[F];
    };
    struct Slab {
        Mine a[E];
        f32x4 b[E];
    };
    const int mine = (lane & 3) * 16 + (r16 >> 2) * 4;
    uint32_t oa[E], ob[E];
#pragma unroll
    for (int e = 0; e < E; ++e) oa[e] = (uint32_t)(((q + e * 4) * 16 * F + r16 * F) * 4), ob[e] = (uint32_t)(((q + e * 4) * g.xs + mine) * 4);
    f32x4 acc[F][4] = {};
    auto load = [&](Slab& f, int64_t s) {
        const float *d = g.d + s * 64 * E * F, *x = g.x + s * 4 * E * g.xs + col0;
#pragma unroll
        for (int e = 0; e < E; ++e) load_at(f.a[e], d, oa[e]), load_at(f.b[e], x, ob[e]);
    };
    auto load_some = [&](Slab& f, int64_t s) {
        const float *d = g.d + s * 64 * E * F, *x = g.x + s * 4 * E * g.xs + col0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const bool in = s * 4 * E + q + e * 4 < g.m;
            f.a[e] = Mine{};
            if (in) load_at(f.a[e], d, oa[e]);
            f.b[e] = load4((const float*)((const char*)x + ob[e]), in ? g.k - col0 - mine : 0);
        }
    };
    auto multiply = [&](const Slab& f) {
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = mma4(f.b[e][j], f.a[e].v[i], acc[i][j]);
    };
    const int64_t whole = g.k < 64 ? sb : max(sb, min(se, g.m / (4 * E)));      // slabs from here on are asked number by number
    walk_slabs<Slab>(sb + wave, whole, 4, load, multiply);
    for (int64_t s = whole + (wave - (int)((whole - sb) & 3) & 3); s < se; s += 4) {
        Slab f;
        load_some(f, s);
        multiply(f);
    }
    __shared__ f32x4 sums[2][F * 4][64];
#pragma unroll
    for (int step = 2; step > 0; step >>= 1) {
        if (wave >= step && wave < 2 * step)
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) sums[wave - step][i * 4 + j][lane] = acc[i][j];
        __syncthreads();
        if (wave < step)
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] += sums[wave][i * 4 + j][lane];
        __syncthreads();
    }
    if (wave > 0) return;
#pragma unroll
    for (int i = 0; i < F; ++i) {
        const int64_t both = r16 * F + i, z = both >= g.hp, row = both - (z ? g.hp : 0);
        if (row >= g.h) continue;
        float* p = g.splits > 1 ? g.part + ((z * g.splits + blockIdx.y) * g.h + row) * g.k : (z ? g.out[1] : g.out[0]) + row * g.os;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int64_t c = col0 + r * 16 + q * 4;
            const f32x4 v = {acc[i][0][r], acc[i][1][r], acc[i][2][r], acc[i][3][r]};
            if (c + 4 <= g.k) __builtin_memcpy(p + c, &v, 16);
            else
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c + j < g.k) p[c + j] = v[j];
        }
    }
}

}  // namespace gpbo_static
