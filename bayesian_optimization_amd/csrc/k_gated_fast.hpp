// The gated unit's products on large operands: both operands contiguous along the contraction, in 128-byte steps, straight from
// memory into LDS.
#pragma once

#include "k_gated.hpp"

namespace gpbo_static {

// Tile of BM x BN outputs by WM x WN waves; a step is 128 bytes of contraction of BM + BN rows.  The step after the current one
// is on its way into the other LDS buffer (16 bytes a lane, no registers) while the current one is multiplied: one barrier a
// step.  Row r of a step lies at 128 r, its 16-byte chunk c at slot c ^ swap(r): a fragment read touches 16 rows, and without the
// exchange all of them would start in the same bank; the loads do the exchange by the address each lane fetches from, since
// their destination is fixed (wave base + 16 lane).  Fragments of the second operand come in pairs over 32 output columns, dealt
// out by fours, so that a lane ends up with 8 neighbouring outputs of a row (16384 x 2048 -> 8192 in 16 bits: the forward pass
// 1.40 -> 1.29 ms, each backward product 0.91 -> 0.88 ms, 1.24 PFLOP/s).
template <typename T, int MODE, int BM, int BN, int WM, int WN>
struct FastTile {
    static constexpr int THREADS = 64 * WM * WN, KS = STEP_BYTES / sizeof(T);
    static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;              // 16 x 16 fragments of a wave
    static constexpr int LA = BM * 8 / THREADS, LB = BN * 8 / THREADS;      // 16-byte loads of a thread and step
    static constexpr int COLS = MODE == GATED_FWD ? BN / 2 : BN;            // output columns of a tile
};

// The slots of 8 rows that one access touches are all different for rows 8 n .. 8 n + 7 as well as for rows 16 n + {0..3, 8..11} and
// 16 n + {4..7, 12..15}.
__device__ __forceinline__ constexpr int swap_of(int r) { return (r ^ ((r >> 1) & 4)) & 7; }

typedef __attribute__((address_space(3))) void* LdsPtr;

// A tile's operand as a buffer: 16 bytes from byte `lane_offset + step_offset` behind p into LDS at `lds` + 16 lane.  Every offset is
// in range by construction (rows behind the last repeat it), so the descriptor's bound is left open.
__device__ __forceinline__ void load_lds(__amdgpu_buffer_rsrc_t r, uint4* lds, uint32_t lane_offset, uint32_t step_offset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LdsPtr)lds, 16, lane_offset, step_offset, 0, 0);
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, 0xffffffffu, 0x00020000);
}

// Workgroups of one XCD (consecutive ids go round the eight of them) take neighbouring tiles, GROUP tile rows at a time, so that
// what one XCD works on shares rows of both operands in its L2.
__device__ __forceinline__ void tile_of(uint32_t id, uint32_t tm, uint32_t tn, uint32_t& im, uint32_t& in) {
    constexpr uint32_t XCDS = 8, GROUP = 8;
    const uint32_t tiles = tm * tn, per = tiles / XCDS, rest = tiles % XCDS, x = id % XCDS;
    const uint32_t t = x * per + min(x, rest) + id / XCDS;
    const uint32_t band = t / (GROUP * tn), rows = min(GROUP, tm - band * GROUP), in_band = t - band * GROUP * tn;
    im = __builtin_amdgcn_readfirstlane(band * GROUP + in_band % rows);      // the same in all lanes: divisions leave it in vector registers
    in = __builtin_amdgcn_readfirstlane(in_band / rows);
}

template <typename T, int MODE, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, BM == 256 ? 1 : 2) void k_gated_fast(GatedArgs g) {
    using F = FastTile<T, MODE, BM, BN, WM, WN>;
    constexpr int FM = F::FM, FN = F::FN, KS = F::KS;
    __shared__ uint4 buf0[(BM + BN) * 8], buf1[(BM + BN) * 8];
    uint32_t im, in;
    tile_of(blockIdx.x, (uint32_t)((g.m + BM - 1) / BM), (uint32_t)((g.n + F::COLS - 1) / F::COLS), im, in);
    const int64_t row0 = (int64_t)im * BM, col0 = (int64_t)in * F::COLS;
    const int z = MODE == GATED_PAIR ? blockIdx.z : 0, split = blockIdx.y;
    const uint32_t all_steps = (uint32_t)(g.k / KS), per = (all_steps + g.splits - 1) / (uint32_t)g.splits;
    const uint32_t s0 = __builtin_amdgcn_readfirstlane(min(split * per, all_steps));
    const int steps1 = (int)__builtin_amdgcn_readfirstlane(min(s0 + per, all_steps) - s0), steps = MODE == GATED_SUM ? 2 * steps1 : steps1;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;

    // what this thread loads of a step: byte offsets from the tile's first row
    uint32_t oa[F::LA], ob[F::LB];
    const int64_t sa = g.a[0].sr * (int64_t)sizeof(T), sb = g.b[0].sr * (int64_t)sizeof(T);
#pragma unroll
    for (int i = 0; i < F::LA; ++i) {
        const int r = (i * F::THREADS + tid) >> 3, c = (tid & 7) ^ swap_of(r);
        oa[i] = (uint32_t)(min((int64_t)r, g.m - 1 - row0) * sa + c * 16);
    }
#pragma unroll
    for (int i = 0; i < F::LB; ++i) {
        const int r = (i * F::THREADS + tid) >> 3, c = (tid & 7) ^ swap_of(r);
        const int q = MODE == GATED_FWD ? r % F::COLS : r;
        ob[i] = (uint32_t)(min((int64_t)q, g.n - 1 - col0) * sb + c * 16);
    }
    const int64_t at_a = row0 * sa + (int64_t)s0 * STEP_BYTES, at_b = col0 * sb + (int64_t)s0 * STEP_BYTES;
    const auto ra0 = buffer_of((const char*)(MODE == GATED_PAIR && z ? g.a[1].p : g.a[0].p) + at_a);
    const auto ra1 = buffer_of((const char*)g.a[1].p + at_a);
    const auto rb0 = buffer_of((const char*)g.b[0].p + at_b), rb1 = buffer_of((const char*)g.b[1].p + at_b);
    auto fetch = [&](uint4* buf, int s) {
        const bool second = MODE == GATED_SUM && s >= steps1;
        const uint32_t k = (uint32_t)(s - (second ? steps1 : 0)) * STEP_BYTES;
#pragma unroll
        for (int i = 0; i < F::LA; ++i) load_lds(second ? ra1 : ra0, buf + i * F::THREADS + wave * 64, oa[i], k);
#pragma unroll
        for (int i = 0; i < F::LB; ++i) {
            const bool up = MODE == GATED_FWD ? i * F::THREADS / 8 >= F::COLS : second;
            load_lds(up ? rb1 : rb0, buf + BM * 8 + i * F::THREADS + wave * 64, ob[i], k);
        }
    };

    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    auto multiply = [&](const uint4* buf) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            uint4 fa[FM], fb[FN];
            const int m = lane & 15, c = kk * 4 + (lane >> 4), deal = (m >> 2) * 8 + (m & 3);
            const uint4* pa = buf + (wm * FM * 16 + m) * 8 + (c ^ swap_of(m));
            const uint4* pb = buf + (BM + (MODE == GATED_FWD ? wn * (FN / 2 * 16) : wn * FN * 16) + deal) * 8;
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                // pairs of fragments: 32 columns each; going forward the second half of them is the other weight matrix
                const int at = MODE == GATED_FWD ? (j >= FN / 2) * F::COLS + (j % (FN / 2)) / 2 * 32 : j / 2 * 32;
                fb[j] = pb[(at + (j & 1) * 4) * 8 + (c ^ swap_of(deal + (j & 1) * 4))];
            }
#pragma unroll
            for (int i = 0; i < FM; ++i) fa[i] = pa[i * 16 * 8];
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = mma<T>(fb[j], fa[i], acc[i][j]);
        }
    };
    if (steps > 0) {
        fetch(buf0, 0);
        __syncthreads();
        int s = 0;
        for (; s + 1 < steps; s += 2) {
            fetch(buf1, s + 1);
            __builtin_amdgcn_sched_barrier(0);       // the loads stay in front of the products that hide them
            multiply(buf0);
            __syncthreads();
            fetch(buf0, min(s + 2, steps - 1));      // behind the last step: loaded again, not used
            __builtin_amdgcn_sched_barrier(0);
            multiply(buf1);
            __syncthreads();
        }
        if (s < steps) multiply(buf0);
    }

    // lane: row lane % 16 of a fragment, eight neighbouring columns of a pair of them
    static_assert(FN % 4 == 0, "fragments come in pairs, of both weight matrices");
    float down = 1.0f;
    if constexpr (MODE != GATED_FWD) down = range_down<T>(g.splits > 1 ? nullptr : g.range);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int64_t row = row0 + wm * FM * 16 + i * 16 + (lane & 15);
        if (row >= g.m) continue;
#pragma unroll
        for (int j = 0; j < (MODE == GATED_FWD ? FN / 2 : FN); j += 2) {
            const int64_t col = col0 + (MODE == GATED_FWD ? wn * (FN / 2 * 16) : wn * FN * 16) + j * 16 + (lane >> 4) * 8;
            if (col >= g.n) continue;
            const int len = (int)min((int64_t)8, g.n - col);
            constexpr int UP = MODE == GATED_FWD ? FN / 2 : 0;
            float v[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                if constexpr (MODE == GATED_FWD) v[r] = activate<T>(acc[i][j + (r >> 2)][r & 3], g.act) * acc[i][j + (r >> 2) + UP][r & 3];
                else v[r] = acc[i][j + (r >> 2)][r & 3] * down;
            }
            if (MODE != GATED_FWD && g.splits > 1) {
                float* p = g.part + (((int64_t)z * g.splits + split) * g.m + row) * g.n + col;
                if (len == 8) __builtin_memcpy(p, v, 32);
                else
#pragma unroll
                    for (int r = 0; r < 8; ++r)
                        if (r < len) p[r] = v[r];
                continue;
            }
            T o[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) o[r] = from_float<T>(v[r]);
            T* p = (T*)(z ? g.out[1] : g.out[0]) + row * g.os + col;
            if (len == 8) __builtin_memcpy(p, o, sizeof(o));
            else
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (r < len) p[r] = o[r];
            if (MODE == GATED_FWD && g.keep_g) {
                // (stores past the caches were no faster: an instruction leaves out every other 16 bytes, which only the L2 joins)
                float *kg = g.keep_g + row * g.n + col, *ku = g.keep_u + row * g.n + col;
                if (len == 8) {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        __builtin_memcpy(kg + q * 4, &acc[i][j + q], 16);
                        __builtin_memcpy(ku + q * 4, &acc[i][j + q + UP], 16);
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < 8; ++r)
                        if (r < len) kg[r] = acc[i][j + (r >> 2)][r & 3], ku[r] = acc[i][j + (r >> 2) + UP][r & 3];
                }
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Operands laid out for it.  Rows padded with zeros to whole steps.
struct PackJob {
    const void* src;
    int64_t stride, rows, cols;   // source
    void* dst;
    int64_t pitch;                // elements of a destination row
    int64_t blocks;               // tiles of 64 x 64
};
struct PackArgs {
    PackJob job[3];
    int count;
};

// dst[r][c] = src[r][c] (TRANSPOSE: dst[c][r] = src[r][c]), zero up to the pitch.  16 bytes a load and store (the pitch is a whole
// number of them); a transposed tile goes through LDS.
template <typename T, bool TRANSPOSE>
__global__ __launch_bounds__(256) void k_gated_pack(PackArgs a) {
    constexpr int V = Pack<T>::N, ACROSS = 64 / V, DOWN = 256 / ACROSS;
    int64_t id = blockIdx.x;
    int which = 0;
    while (which + 1 < a.count && id >= a.job[which].blocks) id -= a.job[which++].blocks;
    const PackJob& jb = a.job[which];
    __shared__ T tile[64][64 + 4 / sizeof(T)];
    const T* src = (const T*)jb.src;
    T* dst = (T*)jb.dst;
    const int tx = threadIdx.x % ACROSS, ty = threadIdx.x / ACROSS;
    // the grid covers the padded destination: destination columns are source columns, or (transposed) source rows
    const int64_t tiles_c = ((TRANSPOSE ? jb.cols : jb.pitch) + 63) / 64;
    const int64_t r0 = id / tiles_c * 64, c0 = id % tiles_c * 64;
#pragma unroll
    for (int i = 0; i < 64 / DOWN; ++i) {
        const int64_t r = r0 + ty + i * DOWN, c = c0 + tx * V;
        Pack<T> p;
        if (r < jb.rows && c + V <= jb.cols) p = load_pack(src + r * jb.stride + c);
        else
#pragma unroll
            for (int j = 0; j < V; ++j) p.v[j] = r < jb.rows && c + j < jb.cols ? src[r * jb.stride + c + j] : from_float<T>(0.0f);
        if constexpr (TRANSPOSE) {
#pragma unroll
            for (int j = 0; j < V; ++j) tile[ty + i * DOWN][tx * V + j] = p.v[j];
        } else if (r < jb.rows && c < jb.pitch) {
            store_pack(dst + r * jb.pitch + c, p);
        }
    }
    if constexpr (TRANSPOSE) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 64 / DOWN; ++i) {
            const int64_t c = c0 + ty + i * DOWN, r = r0 + tx * V;      // the pitch is a multiple of 64: r < pitch
            Pack<T> p;
#pragma unroll
            for (int j = 0; j < V; ++j) p.v[j] = tile[tx * V + j][ty + i * DOWN];
            if (c < jb.cols) store_pack(dst + c * jb.pitch + r, p);
        }
    }
}

// dg and du, row by row (pitch hp) and transposed (pitch mp), zero in the padding of both.  Bound by memory (16384 x 8192 of 16 bits:
// 0.53 ms for 2.4 GB).
template <typename T>
__global__ __launch_bounds__(256) void k_gated_slopes_both(const T* __restrict__ dh, int64_t dhs, const float* __restrict__ kg,
                                                           const float* __restrict__ ku, int64_t m, int64_t n, int act, const float* range,
                                                           T* __restrict__ dg, T* __restrict__ du, int64_t hp, T* __restrict__ dgt, T* __restrict__ dut, int64_t mp) {
    __shared__ T tg[64][66], tu[64][66];
    const float up = range_up<T>(range);
    const int64_t tiles_c = hp / 64, r0 = blockIdx.x / tiles_c * 64, c0 = blockIdx.x % tiles_c * 64;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;      // four columns a thread, 16 rows a pass
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t r = r0 + ty + i * 16, c = c0 + tx * 4;
        const int len = r < m ? (int)max((int64_t)0, min((int64_t)4, n - c)) : 0;
        float gv[4] = {0.0f, 0.0f, 0.0f, 0.0f}, uv[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        T dv[4], og[4], ou[4];
        if (len == 4) {
            __builtin_memcpy(gv, kg + r * n + c, 16);
            __builtin_memcpy(uv, ku + r * n + c, 16);
            __builtin_memcpy(dv, dh + r * dhs + c, sizeof(dv));
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                dv[k] = k < len ? dh[r * dhs + c + k] : from_float<T>(0.0f);
                if (k < len) gv[k] = kg[r * n + c + k], uv[k] = ku[r * n + c + k];
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float a, da;
            activation<T>(gv[k], act, a, da);
            og[k] = from_float<T>(k < len ? to_float(dv[k]) * uv[k] * da * up : 0.0f);
            ou[k] = from_float<T>(k < len ? to_float(dv[k]) * a * up : 0.0f);
            tg[ty + i * 16][tx * 4 + k] = og[k];
            tu[ty + i * 16][tx * 4 + k] = ou[k];
        }
        if (r < m) {
            __builtin_memcpy(dg + r * hp + c, og, sizeof(og));
            __builtin_memcpy(du + r * hp + c, ou, sizeof(ou));
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t c = c0 + ty + i * 16, r = r0 + tx * 4;
        if (c >= n) continue;
        T og[4], ou[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) og[k] = tg[tx * 4 + k][ty + i * 16], ou[k] = tu[tx * 4 + k][ty + i * 16];
        __builtin_memcpy(dgt + c * mp + r, og, sizeof(og));
        __builtin_memcpy(dut + c * mp + r, ou, sizeof(ou));
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Many rows, a short contraction (up to 256 elements of 16 bits): the tiles above would spend their time starting and ending.  Here
// a wave keeps its 32 hidden units' weights for the whole contraction in registers (128 of them at 256 elements) and the
// workgroup walks over tiles of 128 rows of x, the next one on its way into LDS while this one is multiplied; a row fragment is
// read once for four matrix instructions.  wn of the 8 waves stand side by side over hidden units, the others share the rows.
// Bound by matrix instructions (busy 58 % of the time) and the activation's vector instructions (48 cycles an output and wave), which
// two waves a SIMD overlap: 1 M x 256 -> 512 f16 in 0.525 ms, 1.05 PFLOP/s, of 1.45 of a large library product; with the tiles
// above 0.99 ms.  The weight rows are dealt to the fragments so that a lane ends up with 8 neighbouring outputs: 16-byte stores.
constexpr int STREAM_ROWS = 128, STREAM_MOST = 256;
template <typename T, int SL, int ACT>
__global__ __launch_bounds__(512) void k_gated_stream(GatedArgs g, int wn, int groups) {
    constexpr int CHUNKS = SL * 4, LOADS = STREAM_ROWS * CHUNKS / 512;
    __shared__ uint4 buf0[STREAM_ROWS * CHUNKS], buf1[STREAM_ROWS * CHUNKS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // workgroups on the same rows land on the same XCD (ids go round the eight of them) and share x in its L2
    const int stride = gridDim.x / groups, spread = stride % 8 == 0 ? 8 : 1;
    const int group = blockIdx.x / spread % groups, first = blockIdx.x / (spread * groups) * spread + blockIdx.x % spread;
    const int64_t base = (int64_t)group * wn * 32 + (wave % wn) * 32;
    const int64_t tiles = (g.m + STREAM_ROWS - 1) / STREAM_ROWS;
    uint4 fb[2][2][SL];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t h = min(base + ((lane & 15) >> 2) * 8 + j * 4 + (lane & 3), g.n - 1);
#pragma unroll
        for (int s = 0; s < SL; ++s) {
            const int64_t at = s * 64 + (lane >> 4) * 16;
            fb[j][0][s] = *(const uint4*)((const char*)g.b[0].p + h * g.b[0].sr * (int64_t)sizeof(T) + at);
            fb[j][1][s] = *(const uint4*)((const char*)g.b[1].p + h * g.b[1].sr * (int64_t)sizeof(T) + at);
        }
    }
    const int64_t sa = g.a[0].sr * (int64_t)sizeof(T);
    auto fetch = [&](uint4* buf, int64_t t) {
        const int64_t row0 = t * STREAM_ROWS, last = g.m - 1 - row0;
        const auto ra = buffer_of((const char*)g.a[0].p + row0 * sa);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int id = i * 512 + tid, r = id / CHUNKS, c = (id % CHUNKS) ^ (r & 7);
            load_lds(ra, buf + i * 512 + wave * 64, (uint32_t)(min((int64_t)r, last) * sa + c * 16), 0);
        }
    };
    const int64_t col = base + (lane >> 4) * 8;
    const int len = (int)max((int64_t)0, min((int64_t)8, g.n - col));
    T* const out = (T*)g.out[0] + (lane & 15) * g.os + col;
    float *const kg = g.keep_g ? g.keep_g + (lane & 15) * g.n + col : nullptr, *const ku = g.keep_g ? g.keep_u + (lane & 15) * g.n + col : nullptr;
    const bool whole_cols = base + 32 <= g.n;
    auto work_as = [&](const uint4* buf, int64_t t, auto whole) {
        auto load = [&](uint4 (&fa)[SL], int f) {
            const uint4* pa = buf + (f * 16 + (lane & 15)) * CHUNKS;
            const uint4 *even = pa + ((lane >> 4) ^ (lane & 7)), *odd = pa + ((4 + (lane >> 4)) ^ (lane & 7));
#pragma unroll
            for (int s = 0; s < SL; ++s) fa[s] = (s & 1 ? odd : even)[s / 2 * 8];
        };
        auto one = [&](const uint4 (&fa)[SL], int f) {
            f32x4 acc[2][2];
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[j][0] = acc[j][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < SL; ++s)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    acc[j][0] = mma<T>(fb[j][0][s], fa[s], acc[j][0]);
                    acc[j][1] = mma<T>(fb[j][1][s], fa[s], acc[j][1]);
                }
            const int64_t row = t * STREAM_ROWS + f * 16;                      // the fragment's first
            T o[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) o[r] = from_float<T>(activate<T>(acc[r >> 2][0][r & 3], ACT) * acc[r >> 2][1][r & 3]);
            T* p = out + row * g.os;
            if constexpr (whole.value) {
                __builtin_memcpy(p, o, sizeof(o));
                if (kg) {
                    __builtin_memcpy(kg + row * g.n, &acc[0][0], 16);
                    __builtin_memcpy(kg + row * g.n + 4, &acc[1][0], 16);
                    __builtin_memcpy(ku + row * g.n, &acc[0][1], 16);
                    __builtin_memcpy(ku + row * g.n + 4, &acc[1][1], 16);
                }
            } else if (row + (lane & 15) < g.m) {
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (r < len) {
                        p[r] = o[r];
                        if (kg) kg[row * g.n + r] = acc[r >> 2][0][r & 3], ku[row * g.n + r] = acc[r >> 2][1][r & 3];
                    }
            }
        };
        // the next fragment of rows is on its way from LDS while this one is multiplied
        const int by = 8 / wn, last = STREAM_ROWS / 16 - by + wave / wn;
        uint4 f0[SL], f1[SL];
        int f = wave / wn;
        load(f0, f);
        for (; f < last; f += 2 * by) {
            load(f1, f + by);
            __builtin_amdgcn_sched_barrier(0);
            one(f0, f);
            load(f0, min(f + 2 * by, last));
            __builtin_amdgcn_sched_barrier(0);
            one(f1, f + by);
        }
        if (f == last) one(f0, f);
    };
    auto work = [&](const uint4* buf, int64_t t) {
        if (whole_cols && (t + 1) * STREAM_ROWS <= g.m) work_as(buf, t, std::true_type{});      // no lane has anything to leave out
        else work_as(buf, t, std::false_type{});
    };
    if (first >= tiles) return;
    fetch(buf0, first);
    __syncthreads();
    for (int64_t t = first;; t += 2 * stride) {
        const bool more = t + stride < tiles;
        if (more) fetch(buf1, t + stride);
        __builtin_amdgcn_sched_barrier(0);
        work(buf0, t);
        __syncthreads();
        if (!more) break;
        const bool again = t + 2 * stride < tiles;
        if (again) fetch(buf0, t + 2 * stride);
        __builtin_amdgcn_sched_barrier(0);
        work(buf1, t + stride);
        __syncthreads();
        if (!again) break;
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// A few rows (one candidate at a time): bound by reading the weights once.  A wave takes one hidden unit: both its weight rows in
// 16-byte packs, R rows of x against them, sums over the lanes at the end (1 x 2048 -> 8192 bf16: 12 us, 5.6 TB/s; the small form 82).
template <typename T, int R>
__global__ __launch_bounds__(256) void k_gated_few(GatedArgs g) {
    constexpr int V = Pack<T>::N;
    const int lane = threadIdx.x & 63;
    const int64_t h = ((int64_t)blockIdx.z * gridDim.x + blockIdx.x) * 4 + (threadIdx.x >> 6), row0 = (int64_t)blockIdx.y * R;
    if (h >= g.n) return;
    const T *wg = (const T*)g.b[0].p + h * g.b[0].sr, *wu = (const T*)g.b[1].p + h * g.b[1].sr;
    const T* x[R];
    float sg[R], su[R];
#pragma unroll
    for (int r = 0; r < R; ++r) x[r] = (const T*)g.a[0].p + min(row0 + r, g.m - 1) * g.a[0].sr, sg[r] = su[r] = 0.0f;
    const int64_t whole = g.k / V * V;
#pragma unroll 4
    for (int64_t k = lane * V; k < whole; k += 64 * V) {
        const Pack<T> pg = load_pack(wg + k), pu = load_pack(wu + k);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const Pack<T> px = load_pack(x[r] + k);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                sg[r] = fmaf(to_float(px.v[i]), to_float(pg.v[i]), sg[r]);
                su[r] = fmaf(to_float(px.v[i]), to_float(pu.v[i]), su[r]);
            }
        }
    }
    if (whole + lane < g.k) {
        const float vg = to_float(wg[whole + lane]), vu = to_float(wu[whole + lane]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float v = to_float(x[r][whole + lane]);
            sg[r] = fmaf(v, vg, sg[r]);
            su[r] = fmaf(v, vu, su[r]);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float a = wave_sum(sg[r]), b = wave_sum(su[r]);
        if (lane == 0 && row0 + r < g.m) {
            ((T*)g.out[0])[(row0 + r) * g.os + h] = from_float<T>(activate<T>(a, g.act) * b);
            if (g.keep_g) g.keep_g[(row0 + r) * g.n + h] = a, g.keep_u[(row0 + r) * g.n + h] = b;
        }
    }
}

}  // namespace gpbo_static
