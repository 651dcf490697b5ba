// Which kernels a call of the gated unit takes, and its workspace.
#pragma once

#include "k_gated_short.hpp"
#include "k_gated_fast.hpp"

namespace gpbo_static {

inline bool aligned16(const void* p, int64_t stride, int64_t bytes) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride * bytes % 16 == 0 && stride * bytes < (1 << 23);
}

// A launch takes fewer than 2^32 threads: at 256 for 64 x 64 outputs, 2^23 such tiles at a time.  MOST_ACROSS columns of outputs (also the
// most that the entry points take) leave 128 rows of them.
constexpr int64_t MOST_ACROSS = 1 << 28;
template <typename T, typename L>
void by_rows(const GatedArgs& g, L&& launch) {
    const int64_t most = ((int64_t)1 << 23) / ceil_div(g.n, TB) * TB;
    for (int64_t r = 0; r < g.m; r += most) {
        GatedArgs p = g;
        p.m = std::min(most, g.m - r);
        for (Operand* o : {&p.a[0], &p.a[1], &p.rest[0], &p.rest[1]})
            if (o->p) o->p = (const T*)o->p + r * o->sr;
        p.out[0] = (T*)g.out[0] + r * g.os;
        if (g.keep_g) p.keep_g = g.keep_g + r * g.n, p.keep_u = g.keep_u + r * g.n;
        launch(p);
    }
}

// Few hidden units in 32 bits: a wave has 32 rows, so it takes 16384 of them to give every second SIMD one, and x has to outweigh the
// rest (20000 x 483 -> 24: forward 20 us, 25 with the small form; with the backward pass 74 and 141; 1 M x 621 -> 24: 0.99 and 2.9 ms,
// 3.5 and 10.2 with the tiles for large operands).
template <typename T>
bool narrow(int64_t m, int64_t k, int64_t h) {
    return sizeof(T) == 4 && h <= NARROW_HIDDEN && m >= 16384 && m * k >= (int64_t)1 << 20;
}
// 16 F rows of weights, of both matrices together: hidden units in eights (from 32 on in sixteens, which saves two sets of kernels).
inline int narrow_fragments(int64_t h) { return (int)(h <= 32 ? ceil_div(h, 8) : 2 * ceil_div(h, 16)); }
template <typename L>
void by_fragments(int f, L&& launch) {
    switch (f) {
        case 1: return launch(std::integral_constant<int, 1>{});
        case 2: return launch(std::integral_constant<int, 2>{});
        case 3: return launch(std::integral_constant<int, 3>{});
        case 4: return launch(std::integral_constant<int, 4>{});
        case 6: return launch(std::integral_constant<int, 6>{});
        default: return launch(std::integral_constant<int, 8>{});
    }
}

// Tiles of 256 x 256, one a CU at a time, or of 128 x 128, two a CU: by the rounds that the card takes over them.  A round of the large ones is
// as much work as two of the small ones, which take an eighth longer over it (float32, 25000 x 640 -> 382, 294 tiles or 1176: 311 us with the
// large ones, 201 with the small; 50000 x 640 -> 146: 311 and 200; 16384 x 2048 -> 8192, 16 full rounds: 1.27 and 1.44 ms in bf16).
inline int better_tile(int64_t t256, int64_t t128) {
    return t256 >= 256 && 32 * ceil_div(t256, 256) <= 18 * ceil_div(t128, 512) ? 256 : 128;
}

struct ForwardPlan {
    bool narrow = false, fast = false, stream = false;
    int tile = 128;
    int64_t kp = 0, rows = 0, x_bytes = 0, w_bytes = 0;      // rows: of x packed at a time
    int64_t bytes() const { return fast ? x_bytes + 2 * w_bytes : 0; }
};
// The loads straight into LDS need whole steps and 16-byte rows.  What has neither is packed into the workspace first, which pays from
// some 2 GFLOP on (8192 x 2048 -> 4096 bf16 on rows that start anywhere: 653 us with the any-shape kernel, 295 packed, 265 where they do not need it);
// below, and for few tiles, the any-shape kernel starts sooner.
template <typename T>
ForwardPlan forward_plan(int64_t m, int64_t k, int64_t h) {
    constexpr int KS = STEP_BYTES / sizeof(T);
    ForwardPlan p;
    p.narrow = narrow<T>(m, k, h);
    if (p.narrow) return p;
    p.kp = round_up(k, KS);
    p.fast = m * h >= 128 * 64 * 64 && 4 * m * h * k >= (int64_t)1 << 31 && k * (int64_t)sizeof(T) < (1 << 23);
    // at least two tiles of rows for every workgroup of the streaming form
    p.stream = sizeof(T) == 2 && p.kp <= STREAM_MOST && m * h >= (int64_t)1 << 21 && ceil_div(m, STREAM_ROWS) * ceil_div(h, 256) >= 512;
    p.fast = p.fast || p.stream;
    if (k >= 8 * KS) p.tile = better_tile(ceil_div(m, 256) * ceil_div(h, 128), ceil_div(m, 128) * ceil_div(h, 64));
    // (8 GB of rows at most: a thousand of the longest, and a few columns are padded to many times their size)
    p.rows = std::max<int64_t>(1, std::min(m, ((int64_t)1 << 33) / (p.kp * (int64_t)sizeof(T))));
    p.x_bytes = round_up(p.rows * p.kp * (int64_t)sizeof(T), 256);
    p.w_bytes = round_up(h * p.kp * (int64_t)sizeof(T), 256);
    return p;
}

template <typename T, int MODE>
void launch_fast(hipStream_t st, const GatedArgs& g, int tile) {
    const int zs = MODE == GATED_PAIR ? 2 : 1;
    if (tile == 256)
        hipLaunchKernelGGL((k_gated_fast<T, MODE, 256, 256, 2, 4>),
                           dim3((unsigned)(ceil_div(g.m, 256) * ceil_div(g.n, MODE == GATED_FWD ? 128 : 256)), (unsigned)g.splits, zs), dim3(512), 0, st, g);
    else
        hipLaunchKernelGGL((k_gated_fast<T, MODE, 128, 128, 2, 2>),
                           dim3((unsigned)(ceil_div(g.m, 128) * ceil_div(g.n, MODE == GATED_FWD ? 64 : 128)), (unsigned)g.splits, zs), dim3(256), 0, st, g);
}

template <typename T>
void launch_stream(hipStream_t st, const GatedArgs& g) {
    if constexpr (sizeof(T) == 2) {
        int wn = 1;
        while (wn < 8 && wn * 32 < g.n) wn *= 2;
        const int groups = (int)ceil_div(g.n, wn * 32);
        int64_t walkers = std::max<int64_t>(1, std::min<int64_t>(256 / std::min(groups, 256), ceil_div(g.m, STREAM_ROWS)));
        if (walkers > 8) walkers -= walkers % 8;
        auto launch = [&](auto silu, auto gelu) {
            hipLaunchKernelGGL(g.act == GPBO_ACT_SILU ? silu : gelu, dim3((unsigned)(groups * walkers)), dim3(512), 0, st, g, wn, groups);
        };
        if (g.k <= 64) launch(k_gated_stream<T, 2, GPBO_ACT_SILU>, k_gated_stream<T, 2, GPBO_ACT_GELU>);
        else if (g.k <= 128) launch(k_gated_stream<T, 4, GPBO_ACT_SILU>, k_gated_stream<T, 4, GPBO_ACT_GELU>);
        else if (g.k <= 192) launch(k_gated_stream<T, 6, GPBO_ACT_SILU>, k_gated_stream<T, 6, GPBO_ACT_GELU>);
        else launch(k_gated_stream<T, 8, GPBO_ACT_SILU>, k_gated_stream<T, 8, GPBO_ACT_GELU>);
    }
}

inline void launch_narrow(hipStream_t st, const GatedArgs& g) {
    by_rows<float>(g, [&](const GatedArgs& part) {
        by_fragments(narrow_fragments(g.n), [&](auto f) {
            hipLaunchKernelGGL(k_gated_narrow<f.value>, dim3((unsigned)ceil_div(part.m, 128)), dim3(256), 0, st, part);
        });
    });
}

// Whether the loads straight into LDS can take the operands as they are.
template <typename T>
bool direct(const GatedArgs& g) {
    return g.k * (int64_t)sizeof(T) % STEP_BYTES == 0 && aligned16(g.a[0].p, g.a[0].sr, sizeof(T)) && aligned16(g.b[0].p, g.b[0].sr, sizeof(T)) &&
           aligned16(g.b[1].p, g.b[1].sr, sizeof(T));
}
template <typename T>
int64_t forward_bytes(const GatedArgs& g) {
    return direct<T>(g) ? 0 : forward_plan<T>(g.m, g.k, g.n).bytes();
}

template <typename T>
hipError_t gated_forward(hipStream_t st, GatedArgs g, char* work) {
    const ForwardPlan p = forward_plan<T>(g.m, g.k, g.n);
    if (p.narrow && std::max(g.a[0].sr, g.b[0].sr) < NARROW_STRIDE) {
        launch_narrow(st, g);
    } else if (p.fast) {
        auto launch = [&](const GatedArgs& part) { p.stream ? launch_stream<T>(st, part) : launch_fast<T, GATED_FWD>(st, part, p.tile); };
        if (direct<T>(g)) {
            by_rows<T>(g, launch);
        } else {
            for (int64_t r = 0; r < g.m; r += p.rows) {      // (weights with the first rows)
                GatedArgs part = g;
                part.m = std::min(p.rows, g.m - r);
                PackArgs a{};
                a.count = r == 0 ? 3 : 1;
                a.job[0] = {(const T*)g.a[0].p + r * g.a[0].sr, g.a[0].sr, part.m, g.k, work, p.kp, ceil_div(part.m, 64) * ceil_div(p.kp, 64)};
                a.job[1] = {g.b[0].p, g.b[0].sr, g.n, g.k, work + p.x_bytes, p.kp, ceil_div(g.n, 64) * ceil_div(p.kp, 64)};
                a.job[2] = {g.b[1].p, g.b[1].sr, g.n, g.k, work + p.x_bytes + p.w_bytes, p.kp, a.job[1].blocks};
                hipLaunchKernelGGL((k_gated_pack<T, false>), dim3((unsigned)(a.job[0].blocks + (r == 0 ? 2 * a.job[1].blocks : 0))), dim3(256), 0, st, a);
                part.a[0] = {work, p.kp, 1}, part.b[0] = {a.job[1].dst, p.kp, 1}, part.b[1] = {a.job[2].dst, p.kp, 1}, part.k = p.kp;
                part.out[0] = (T*)g.out[0] + r * g.os;
                if (g.keep_g) part.keep_g = g.keep_g + r * g.n, part.keep_u = g.keep_u + r * g.n;
                by_rows<T>(part, launch);
            }
        }
    } else if (g.m <= 16) {
        const int64_t fours = ceil_div(g.n, 4), x = std::min<int64_t>(fours, 1 << 22);
        const dim3 grid((unsigned)x, (unsigned)ceil_div(g.m, 8), (unsigned)ceil_div(fours, x));
        if (g.m == 1) hipLaunchKernelGGL((k_gated_few<T, 1>), grid, dim3(256), 0, st, g);
        else if (g.m == 2) hipLaunchKernelGGL((k_gated_few<T, 2>), grid, dim3(256), 0, st, g);
        else if (g.m <= 4) hipLaunchKernelGGL((k_gated_few<T, 4>), grid, dim3(256), 0, st, g);
        else hipLaunchKernelGGL((k_gated_few<T, 8>), grid, dim3(256), 0, st, g);
    } else {
        const AnyPlan any = any_plan<T>(g.m, g.n, g.k, 1, false);
        by_rows<T>(g, [&](const GatedArgs& part) { launch_any<T, GATED_FWD, true, true, 1>(st, part, any); });
    }
    return hipGetLastError();
}

// Backward.  Large: dg and du are written both ways round, x and the weights transposed, so that every product contracts along
// rows; these copies are a few per cent of the products' time.
struct BackwardPlan {
    bool fast = false, one = false, narrow = false, few_cols = false;      // one: k_gated_small_back
    bool parts = false;                                                    // dg and du in two parts
    int tile_x = 128, tile_w = 128, splits_x = 1, splits_w = 1;
    AnyPlan any_x, any_w;
    int64_t hp = 0, mp = 0;
    int64_t range_bytes = 0, d_bytes = 0, rest_bytes = 0, dt_bytes = 0, xt_bytes = 0, wt_bytes = 0, part_bytes = 0;
    int splits_narrow = 1;
    int64_t narrow_d_bytes = 0, narrow_bytes = 0;
    int64_t bytes() const { return std::max(narrow_bytes, range_bytes + 2 * d_bytes + 2 * rest_bytes + 2 * dt_bytes + xt_bytes + 2 * wt_bytes + part_bytes); }
};
template <typename T>
BackwardPlan backward_plan(int64_t m, int64_t k, int64_t h) {
    constexpr int KS = STEP_BYTES / sizeof(T);
    constexpr int64_t B = sizeof(T);
    BackwardPlan p;
    p.narrow = narrow<T>(m, k, h);
    if (p.narrow) {                            // (with the any-shape kernels as a way out for rows of weights that lie too far apart)
        const int f = narrow_fragments(h);
        // workgroups that the card holds at once, by the registers of their sums
        p.splits_narrow = (int)std::max<int64_t>(1, std::min<int64_t>((f == 1 ? 1024 : f <= 3 ? 768 : 512) / ceil_div(k, 64), m / 512));
        p.narrow_d_bytes = round_up(m * 16 * f * 4, 256);
        p.narrow_bytes = p.narrow_d_bytes + (p.splits_narrow > 1 ? 2 * p.splits_narrow * h * k * 4 : 0);
    }
    // few columns: worth it from four million hidden outputs on (50000 x 16 -> 256: 290 us with the forward pass, 163 here; 8000 x 16 -> 256: 50 and 55);
    // in 16 bits, where the other way has faster products, up to 16 of them and from eight million on (1 M x 4 -> 128: 1055 and 898; 50000 x
    // 64 -> 256: 120 and 167)
    p.few_cols = k <= (B == 4 ? SHORT_COLS : 16) && h > NARROW_HIDDEN && m >= 4096 && m * h >= (B == 4 ? (int64_t)1 << 22 : (int64_t)1 << 23);
    if (p.few_cols) {
        p.splits_w = (int)std::max<int64_t>(1, std::min<int64_t>(512 / ceil_div(h, 64), m / 512));
        p.part_bytes = p.splits_w > 1 ? 2 * p.splits_w * h * k * 4 : 0;
        return p;
    }
    // Below these the copies cost more than they save: 4 GFLOP in 32 bits (2000 x 520 -> 200, 1.7: 83 us with the forward pass, 125 with them), in 16
    // bits 1.9 (1000 x 520 -> 1000, 4.2: 98 without, 66 with; 1000 x 520 -> 400, 1.7: 44 and 57) or, over many rows, 1 (2000 x 520 -> 200: 59
    // and 53); or two million elements over many rows.
    const int64_t enough = B == 4 ? (int64_t)1 << 32 : m >= 2000 ? (int64_t)1 << 30 : (int64_t)7 << 28;
    // In two parts where a gradient has few elements (with the forward pass 20000 x 5 -> 77 bf16 57 us without, 64 with; 1000 x 520 ->
    // 400, where it would take away less than the gradients' own roundings, 44 and 61).  The any-shape kernels do that, whatever the size: the
    // whole-step kernels with a second part are slower still (backward 8192 x 1 -> 256 28 us, 88 with them, 35 with one part; 1 M x 60 -> 64
    // 992, 1215 and 564).
    const bool few_elements = SLOPE_PARTS<T> == 2 && std::min(m, h) * k < 4096;
    p.fast = !p.narrow && !few_elements && m >= 128 && (8 * m * h * k >= enough || (m >= 4096 && std::max(h, k) >= 128 && m * std::max(h, k) >= (int64_t)1 << 21)) && m * B < (1 << 23) && h * B < (1 << 23);
    if (p.fast) {
        p.hp = round_up(h, 64), p.mp = round_up(m, 64);
        auto choose = [&](int64_t rows, int64_t cols, int64_t zs, int64_t steps, int& tile, int& splits) {
            const int64_t t256 = zs * ceil_div(rows, 256) * ceil_div(cols, 256), t128 = zs * ceil_div(rows, 128) * ceil_div(cols, 128);
            tile = better_tile(t256, t128);
            splits = tile == 256 || t128 >= 256 ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>(512 / t128, steps / 8));
        };
        choose(m, k, 1, p.hp / KS, p.tile_x, p.splits_x);
        choose(h, k, 2, p.mp / KS, p.tile_w, p.splits_w);
        p.d_bytes = round_up(m * p.hp * B, 256), p.dt_bytes = round_up(h * p.mp * B, 256);
        p.xt_bytes = round_up(k * p.mp * B, 256), p.wt_bytes = round_up(k * p.hp * B, 256);
    } else {
        // one launch while all tiles together work out dg and du no more than a million times, and a tile's waves have few slabs: with the
        // forward pass 22 us against 30 with three launches (95 x 621 -> 128, 400 x 30 -> 24), even at 512 rows or 256 hidden units
        // (27 to 29 and 30), worse from there on (1000 x 30 -> 24: 44, 20 x 30 -> 1000: 60)
        p.one = m > 0 && 4 * m * h * ceil_div(k, SB) <= (int64_t)1 << 20 && std::max(m, 2 * h) <= 512;
        if (p.one) return p;
        p.d_bytes = round_up(m * h * B, 256), p.parts = few_elements, p.rest_bytes = p.parts ? p.d_bytes : 0;
        p.any_x = any_plan<T>(m, k, h, 1, true), p.any_w = any_plan<T>(h, k, m, 2, true);
        p.splits_x = p.any_x.splits, p.splits_w = p.any_w.splits;
    }
    p.range_bytes = RANGED<T> && m > 0 ? RANGE_BYTES : 0;
    p.part_bytes = std::max<int64_t>(p.splits_x > 1 ? p.splits_x * m * k * 4 : 0, p.splits_w > 1 ? 2 * p.splits_w * h * k * 4 : 0);
    return p;
}

template <typename T>
hipError_t gated_backward(hipStream_t st, const void* dh, int64_t dhs, const void* x, int64_t xs, const void* wg, const void* wu, int64_t ws,
                          const float* kg, const float* ku, int64_t m, int64_t k, int64_t h, int act, void* dx, int64_t dxs, void* dwg,
                          void* dwu, int64_t dws, char* work) {
    constexpr int64_t B = sizeof(T);
    const BackwardPlan p = backward_plan<T>(m, k, h);
    if (p.narrow && std::max(xs, ws) < NARROW_STRIDE) {
        const int fragments = narrow_fragments(h);
        NarrowBack g{};
        g.d = (const float*)work, g.hp = 8 * fragments, g.m = m, g.k = k, g.h = h, g.x = (const float*)x, g.xs = xs, g.ws = ws;
        g.w[0] = (const float*)wg, g.w[1] = (const float*)wu;
        hipLaunchKernelGGL(k_gated_narrow_slopes, dim3((unsigned)std::min<int64_t>(ceil_div(m * g.hp / 4, 256), 8192)), dim3(256), 0, st,
                           (const float*)dh, dhs, kg, ku, m, h, act, (float*)work, g.hp);
        if (dx) {
            constexpr int64_t MOST = (int64_t)1 << 29;      // rows of a launch, at 4 threads a row or fewer
            by_fragments(fragments, [&](auto f) {
                // (a wave of 16 rows, where d takes more registers, has three of its kind on a SIMD as well)
                constexpr int RF = f.value <= 4 ? 2 : 1;
                for (int64_t r = 0; r < m; r += MOST) {
                    NarrowBack part = g;
                    part.m = std::min(MOST, m - r), part.d = g.d + r * 16 * f.value, part.out[0] = (float*)dx + r * dxs, part.os = dxs;
                    const int64_t walkers = ceil_div(part.m, 64 * RF), beside = std::max<int64_t>(1, std::min<int64_t>(ceil_div(k, 64), 1024 / walkers));
                    hipLaunchKernelGGL((k_gated_narrow_dx<RF, f.value>), dim3((unsigned)walkers, (unsigned)beside), dim3(256), 0, st, part);
                }
            });
        }
        if (dwg) {
            g.out[0] = (float*)dwg, g.out[1] = (float*)dwu, g.os = dws, g.splits = p.splits_narrow, g.part = (float*)(work + p.narrow_d_bytes);
            by_fragments(fragments, [&](auto f) {
                hipLaunchKernelGGL(k_gated_narrow_dw<f.value>, dim3((unsigned)ceil_div(k, 64), (unsigned)g.splits), dim3(256), 0, st, g);
            });
            GatedArgs j{};
            j.m = h, j.n = k, j.out[0] = dwg, j.out[1] = dwu, j.os = dws, j.splits = g.splits, j.part = g.part;
            if (j.splits > 1) hipLaunchKernelGGL(k_gated_join<T>, dim3((unsigned)ceil_div(h * k, 256), 2), dim3(256), 0, st, j);
        }
        return hipGetLastError();
    }
    if (p.one) {
        const int64_t nt = ceil_div(k, SB), tiles = (dx ? ceil_div(m, SB) * nt : 0) + (dwg ? 2 * ceil_div(h, SB) * nt : 0);
        if (tiles > 0)
            hipLaunchKernelGGL(k_gated_small_back<T>, dim3((unsigned)tiles), dim3(64 * SMALL_WAVES), 0, st, SlopeOperand{dh, kg, ku, dhs, h, act},
                               Operand{x, 1, xs}, Operand{wg, 1, ws}, Operand{wu, 1, ws}, m, k, h, dx, dxs, dwg, dwu, dws);
        return hipGetLastError();
    }
    if (p.few_cols) {
        ShortBack<T> g{};
        g.dh = (const T*)dh, g.kg = kg, g.ku = ku, g.x = (const T*)x, g.w[0] = (const T*)wg, g.w[1] = (const T*)wu;
        g.dhs = dhs, g.xs = xs, g.ws = ws, g.m = m, g.k = k, g.h = h, g.act = act;
        auto by_columns = [&](auto&& launch) {
            if (k <= 16) launch(std::integral_constant<int, 1>{});
            if constexpr (B == 4) {
                if (k > 16 && k <= 32) launch(std::integral_constant<int, 2>{});
                if (k > 32 && k <= 48) launch(std::integral_constant<int, 3>{});
                if (k > 48) launch(std::integral_constant<int, 4>{});
            }
        };
        if (dx) {
            g.out[0] = (T*)dx, g.os = dxs;
            by_columns([&](auto c) { hipLaunchKernelGGL((k_gated_short_dx<T, c.value>), dim3((unsigned)ceil_div(m, c.value <= 3 ? 32 : 16)), dim3(256), 0, st, g); });
        }
        if (dwg) {
            g.out[0] = (T*)dwg, g.out[1] = (T*)dwu, g.os = dws, g.splits = p.splits_w, g.part = (float*)work;
            by_columns([&](auto c) {
                hipLaunchKernelGGL((k_gated_short_dw<T, c.value>), dim3((unsigned)ceil_div(h, 64), (unsigned)g.splits), dim3(256), 0, st, g);
            });
            GatedArgs j{};
            j.m = h, j.n = k, j.out[0] = dwg, j.out[1] = dwu, j.os = dws, j.splits = g.splits, j.part = g.part;
            if (j.splits > 1) hipLaunchKernelGGL(k_gated_join<T>, dim3((unsigned)ceil_div(h * k, 256), 2), dim3(256), 0, st, j);
        }
        return hipGetLastError();
    }
    float* const range = p.range_bytes ? (float*)work : nullptr;
    if (range)
        hipLaunchKernelGGL(k_gated_range<T>, dim3((unsigned)std::min<int64_t>(ceil_div(m * ceil_div(h, 4), RANGE_THREADS), RANGE_PIECES)), dim3(RANGE_THREADS),
                           0, st, (const T*)dh, dhs, kg, ku, m, h, act, range);
    char* at = work + p.range_bytes;
    auto take = [&](int64_t bytes) { char* r = at; at += bytes; return r; };
    T *dg = (T*)take(p.d_bytes), *du = (T*)take(p.d_bytes), *dg_rest = (T*)take(p.rest_bytes), *du_rest = (T*)take(p.rest_bytes), *dgt = (T*)take(p.dt_bytes), *dut = (T*)take(p.dt_bytes), *xt = (T*)take(p.xt_bytes),
      *wgt = (T*)take(p.wt_bytes), *wut = (T*)take(p.wt_bytes);
    float* part = (float*)take(p.part_bytes);
    auto by_parts = [&](auto&& launch) {
        if (p.parts) launch(std::integral_constant<int, SLOPE_PARTS<T>>{});
        else launch(std::integral_constant<int, 1>{});
    };
    if (p.fast) {
        hipLaunchKernelGGL(k_gated_slopes_both<T>, dim3((unsigned)(p.mp / 64 * (p.hp / 64))), dim3(256), 0, st, (const T*)dh, dhs, kg, ku, m, h, act,
                           range, dg, du, p.hp, dgt, dut, p.mp);
        PackArgs a{};
        if (dwg) a.job[a.count++] = {x, xs, m, k, xt, p.mp, p.mp / 64 * ceil_div(k, 64)};
        if (dx) {
            a.job[a.count++] = {wg, ws, h, k, wgt, p.hp, p.hp / 64 * ceil_div(k, 64)};
            a.job[a.count++] = {wu, ws, h, k, wut, p.hp, p.hp / 64 * ceil_div(k, 64)};
        }
        int64_t blocks = 0;
        for (int i = 0; i < a.count; ++i) blocks += a.job[i].blocks;
        if (blocks) hipLaunchKernelGGL((k_gated_pack<T, true>), dim3((unsigned)blocks), dim3(256), 0, st, a);
    } else if (m > 0) {
        const int64_t packs = m * ceil_div(h, Pack<T>::N);
        by_parts([&](auto parts) {
            hipLaunchKernelGGL((k_gated_slopes<T, parts.value == 2>), dim3((unsigned)std::min<int64_t>(ceil_div(packs, 256), 8192)), dim3(256), 0, st,
                               (const T*)dh, dhs, kg, ku, m, h, act, range, dg, du, dg_rest, du_rest);
        });
    }
    if (dx && m > 0) {
        GatedArgs g{};
        g.m = m, g.n = k, g.out[0] = dx, g.os = dxs, g.splits = p.splits_x, g.part = part, g.range = range;
        if (p.fast) {
            g.a[0] = {dg, p.hp, 1}, g.a[1] = {du, p.hp, 1}, g.b[0] = {wgt, p.hp, 1}, g.b[1] = {wut, p.hp, 1}, g.k = p.hp;
            launch_fast<T, GATED_SUM>(st, g, p.tile_x);
        } else {
            g.a[0] = {dg, h, 1}, g.a[1] = {du, h, 1}, g.b[0] = {wg, 1, ws}, g.b[1] = {wu, 1, ws}, g.k = h;
            g.rest[0] = {dg_rest, h, 1}, g.rest[1] = {du_rest, h, 1};
            by_parts([&](auto parts) {
                by_rows<T>(g, [&](const GatedArgs& part) { launch_any<T, GATED_SUM, true, false, parts.value>(st, part, p.any_x); });
            });
        }
        if (g.splits > 1) hipLaunchKernelGGL(k_gated_join<T>, dim3((unsigned)ceil_div(m * k, 256), 1), dim3(256), 0, st, g);
    }
    if (dwg) {
        GatedArgs g{};
        g.m = h, g.n = k, g.out[0] = dwg, g.out[1] = dwu, g.os = dws, g.splits = p.splits_w, g.part = part, g.range = range;
        if (p.fast) {
            g.a[0] = {dgt, p.mp, 1}, g.a[1] = {dut, p.mp, 1}, g.b[0] = g.b[1] = {xt, p.mp, 1}, g.k = p.mp;
            launch_fast<T, GATED_PAIR>(st, g, p.tile_w);
        } else {
            g.a[0] = {dg, 1, h}, g.a[1] = {du, 1, h}, g.b[0] = g.b[1] = {x, 1, xs}, g.k = m;
            g.rest[0] = {dg_rest, 1, h}, g.rest[1] = {du_rest, 1, h};
            by_parts([&](auto parts) { launch_any<T, GATED_PAIR, false, false, parts.value>(st, g, p.any_w); });
        }
        if (g.splits > 1) hipLaunchKernelGGL(k_gated_join<T>, dim3((unsigned)ceil_div(h * k, 256), 2), dim3(256), 0, st, g);
    }
    return hipGetLastError();
}

}  // namespace gpbo_static
