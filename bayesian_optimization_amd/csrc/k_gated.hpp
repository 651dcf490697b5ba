// Gated unit: h = act(x Wg^T) * (x Wu^T), forward and backward.
//   g = x Wg^T, u = x Wu^T;  silu: act(g) = g / (1 + exp(-g)),  gelu: act(g) = g Phi(g)
//   dg = dh u act'(g), du = dh act(g);  dx = dg Wg + du Wu;  dWg = dg^T x, dWu = du^T x
// Four products' worth of matrix work forward (two projections), eight back.  Both projections of a tile are formed by the
// same workgroup from one staged tile of x, so the activation and the product are an epilogue on the accumulators and g, u
// never go to memory unless the caller keeps them for the backward pass.  Sums are held in 32 bits, and so are the kept g and
// u: rounded to 16 bits they would put two more roundings of the same size under every gradient.  h is rounded once.  dg and du are
// operands of the matrix instructions, so of the type of x, rounded once each (in float16 scaled into its range): in 16 bits, over a gradient's
// many elements, the error is then 1.4 times that of the gradient's own rounding.  Over few elements, where terms may cancel in all of
// them, it can be several times (3 with 10 in float16), so that there (under 4096 elements) the products take a sum of two numbers of 16
// bits: the rounded one and what the rounding left.  The kernels for small problems and for few columns take them in 32 bits.
#pragma once

#include <type_traits>

#include "static_ops.hpp"

namespace gpbo_static {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;

// One 16-byte fragment a lane: row lane % 16 of the operand, elements (lane / 16) * N .. + N of a slab of 4 N along the
// contraction (N = 8 in 16 bits: one 16x16x32 instruction; N = 4 in 32 bits: four 16x16x4 instructions, which take element i
// of every lane -- the contraction index is permuted, in both operands alike).
// D: row (lane / 16) * 4 + r comes from the first operand, column lane % 16 from the second.
template <typename T>
__device__ __forceinline__ f32x4 mma(const uint4& a, const uint4& b, f32x4 c);
template <>
__device__ __forceinline__ f32x4 mma<bf16>(const uint4& a, const uint4& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mma<f16>(const uint4& a, const uint4& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mma<float>(const uint4& a, const uint4& b, f32x4 c) {
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
}

// act(g) and act'(g), with the hardware's exponential and reciprocal (one unit in the last place each).  silu through the logistic
// function, whose exponential saturates to 0 or infinity with the right limit; gelu through q = Phi(-|g|) = 1/2 erfc(|g| / sqrt 2) = exp(-g^2 / 2)
// t R(t), t = 1 / (1 + c |g|), which keeps the far negative tail that 1 + erf loses: R has six terms for results of 16 bits (relative error
// 4.9e-5, a tenth of half a step of float16, and 1.7e-7 in q) and ten for 32 bits (2e-8; scripts/gelu_tail_fit.py has the fit).  With all
// roundings a result of 32 bits is within 3 units of 2^-24 (1 + |g|) min(|g|, 1); relative to itself it is off by the rounding of the
// exponent as well, g^2 units of 2^-24, which is less than what the roundings of g, a sum, do to it.  The activation of every output is as much
// vector work as a short contraction is matrix work (1 M x 256 -> 512 in 16 bits, with tiles: 1.27 -> 0.83 ms against expf and erfcf).
template <typename T>
__device__ __forceinline__ void activation(float g, int act, float& a, float& da) {
    if (act == GPBO_ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896341f * g));
        a = g * s;
        da = s + a * (1.0f - s);
        return;
    }
    constexpr bool WIDE = sizeof(T) == 4;
    const float e = __builtin_amdgcn_exp2f(-0.72134752044448170f * g * g);      // exp(-g^2 / 2)
    const float t = __builtin_amdgcn_rcpf(1.0f + ((WIDE ? 0.3354f : 0.6014f) * 0.70710678118654752f) * fabsf(g));
    constexpr int TERMS = WIDE ? 10 : 6;
    constexpr float R[2][10] = {{0.338197976f, 0.357509732f, 0.166214883f, 0.482815653f, -0.461610645f, 0.116872713f},
                                {0.18920809f, 0.189721197f, 0.173563048f, 0.186824769f, 0.016709242f, 0.365303278f, -0.393553346f, 0.497524679f, -0.279960424f, 0.0546594486f}};
    float r = R[WIDE][TERMS - 1];
#pragma unroll
    for (int i = TERMS - 2; i >= 0; --i) r = fmaf(r, t, R[WIDE][i]);
    const float q = 0.5f * e * t * r;
    const float cdf = g < 0.0f ? q : 1.0f - q;
    a = g * cdf;
    da = cdf + 0.39894228040143268f * g * e;
}
template <typename T>
__device__ __forceinline__ float activate(float g, int act) {
    float a, da;
    activation<T>(g, act, a, da);
    return a;
}

// A product's operand: element (row, k) at p + row * sr + k * sk, one of the two strides 1.
struct Operand {
    const void* p;
    int64_t sr, sk;
};

constexpr int GATED_FWD = 0;      // a[0] b[0] and a[0] b[1] side by side, epilogue act(.) * (.)
constexpr int GATED_SUM = 1;      // a[0] b[0] + a[1] b[1]
constexpr int GATED_PAIR = 2;     // a[z] b[0] to out[z], z = 0, 1

struct GatedArgs {
    Operand a[2], b[2], rest[2];  // rest: what the rounding of a[0], a[1] left (where that is an operand of two parts)
    int64_t m, n, k;              // out is (m, n), k the contraction (of each part)
    void* out[2];
    int64_t os;                   // row stride of out
    float *keep_g, *keep_u;       // (m, n) contiguous, or null
    int act, splits;
    float* part;                  // splits > 1: [z][split][m][n] sums in 32 bits
    const float* range;           // float16: the range of a, or null
};

// Float16 holds 40 powers of two, of which dg and du, products of three numbers, leave any one part: below 6e-8 they would be nothing and beyond
// 65504 infinite where the gradients themselves are neither.  So in float16 they are multiplied by the power of two that puts the largest
// of both next to the upper end, and the products by its inverse: exact, and what is lost at the lower end is 2^-39 of the largest.
// k_gated_range leaves the largest in 256 pieces, which every wave that needs the factor puts together.
template <typename T>
constexpr bool RANGED = std::is_same_v<T, f16>;
constexpr int RANGE_PIECES = 256;
constexpr int64_t RANGE_BYTES = RANGE_PIECES * 4;
// The exponent of the factor; all lanes of the wave take part.
__device__ __forceinline__ int range_exponent(const float* range) {
    if (!range) return 0;
    f32x4 v;
    __builtin_memcpy(&v, range + (threadIdx.x & 63) * 4, 16);
    float most = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
    if (!(most > 0.0f)) return 0;
    return min(100, 14 + 127 - (int)(__float_as_uint(most) >> 23));      // the largest comes to 2^14 .. 2^15
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
template <typename T>
__device__ __forceinline__ float range_up(const float* range) {
    if constexpr (RANGED<T>) return power_of_two(range_exponent(range));
    return 1.0f;
}
template <typename T>
__device__ __forceinline__ float range_down(const float* range) {
    if constexpr (RANGED<T>) return power_of_two(-range_exponent(range));
    return 1.0f;
}

// Numbers of type T that make up one element of dg and du where they are not rounded to one.
template <typename T>
constexpr int SLOPE_PARTS = sizeof(T) == 2 ? 2 : 1;
template <int N>
struct Parts {
    uint4 v[N];
};
// The sums of a product's parts; what the roundings left is left out where it met an infinity (zero times it is no number, and the rounded
// part alone says what becomes of it).
template <int N>
struct Sums {
    f32x4 v[N] = {};
    __device__ __forceinline__ f32x4 all() const {
        if constexpr (N == 1) return v[0];
        f32x4 r = v[0];
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] += fabsf(v[N - 1][i]) < INFINITY ? v[N - 1][i] : 0.0f;
        return r;
    }
};
// What the rounding of d to hi left; nothing if hi is beyond the type's range.
template <typename T>
__device__ __forceinline__ T rounding_rest(float d, T hi) {
    const float h = to_float(hi);
    return from_float<T>(fabsf(h) < INFINITY ? d - h : 0.0f);
}

// ---------------------------------------------------------------------------------------------------------------------
// Tile kernel for every shape, stride and alignment: 64 x 64 outputs, 4 waves of 32 x 32, 128 bytes of contraction a step,
// staged through registers (guarded at every edge) into LDS.  Slot (row, chunk) of a staged tile lives at chunk ^ (row & 7):
// the 16 rows that one fragment read touches then fall into different banks.
constexpr int TB = 64, STEP_BYTES = 128;

template <typename T, bool KC>
struct TileLoad {
    static constexpr int V = 16 / sizeof(T), KS = STEP_BYTES / sizeof(T);
    static constexpr int PACKS = TB * KS / V / 256;
    Pack<T> r[PACKS];
    __device__ __forceinline__ void load(const Operand& o, int64_t row0, int64_t rows, int64_t k0, int64_t k1) {
        const T* p = (const T*)o.p;
#pragma unroll
        for (int i = 0; i < PACKS; ++i) {
            const int id = threadIdx.x + i * 256;
            if constexpr (KC) {
                const int64_t row = row0 + id / 8, k = k0 + (id % 8) * V;
                if (row < rows && k + V <= k1) r[i] = load_pack(p + row * o.sr + k);
                else
#pragma unroll
                    for (int j = 0; j < V; ++j) r[i].v[j] = (row < rows && k + j < k1) ? p[row * o.sr + k + j] : from_float<T>(0.0f);
            } else {
                const int64_t row = row0 + (id % (TB / V)) * V, k = k0 + id / (TB / V);
                if (k < k1 && row + V <= rows) r[i] = load_pack(p + k * o.sk + row);
                else
#pragma unroll
                    for (int j = 0; j < V; ++j) r[i].v[j] = (k < k1 && row + j < rows) ? p[k * o.sk + row + j] : from_float<T>(0.0f);
            }
        }
    }
    __device__ __forceinline__ void store(uint4* lds) const {
#pragma unroll
        for (int i = 0; i < PACKS; ++i) {
            const int id = threadIdx.x + i * 256;
            if constexpr (KC) {
                const int row = id / 8, c = id % 8;
                lds[row * 8 + (c ^ (row & 7))] = __builtin_bit_cast(uint4, r[i]);
            } else {
                const int row = (id % (TB / V)) * V, k = id / (TB / V);
                T* l = reinterpret_cast<T*>(lds);
#pragma unroll
                for (int j = 0; j < V; ++j) l[((row + j) * 8 + ((k / V) ^ ((row + j) & 7))) * V + k % V] = r[i].v[j];
            }
        }
    }
};

template <typename T, int MODE, bool AKC, bool BKC, int NA>
__global__ __launch_bounds__(256) void k_gated_tile(GatedArgs g) {
    constexpr int KS = STEP_BYTES / sizeof(T), NB = MODE == GATED_FWD ? 2 : 1;
    __shared__ uint4 la[NA][TB * 8], lb[NB][TB * 8];
    const int64_t nt = (g.n + TB - 1) / TB;
    const int64_t row0 = (int64_t)(blockIdx.x / nt) * TB, col0 = (int64_t)(blockIdx.x % nt) * TB;
    const int z = MODE == GATED_PAIR ? blockIdx.z : 0, split = blockIdx.y;
    const int64_t per = ((g.k + g.splits - 1) / g.splits + KS - 1) / KS * KS;
    const int64_t kb = min(split * per, g.k), ke = min(kb + per, g.k);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wr = (wave >> 1) * 32, wc = (wave & 1) * 32;
    Sums<NA> acc[NB][2][2];
    const int64_t steps1 = (ke - kb + KS - 1) / KS, steps = MODE == GATED_SUM ? 2 * steps1 : steps1;
    TileLoad<T, AKC> ta[NA];
    TileLoad<T, BKC> tb[NB];
    auto fetch = [&](int64_t s) {
        const int part = MODE == GATED_SUM && s >= steps1;
        const int64_t k0 = kb + (s - (part ? steps1 : 0)) * KS;
        ta[0].load(g.a[MODE == GATED_PAIR ? z : part], row0, g.m, k0, ke);
        if constexpr (NA == 2) ta[1].load(g.rest[MODE == GATED_PAIR ? z : part], row0, g.m, k0, ke);
        tb[0].load(g.b[part], col0, g.n, k0, ke);
        if constexpr (NB == 2) tb[1].load(g.b[1], col0, g.n, k0, ke);
    };
    if (steps > 0) fetch(0);
    for (int64_t s = 0; s < steps; ++s) {
#pragma unroll
        for (int a = 0; a < NA; ++a) ta[a].store(la[a]);
#pragma unroll
        for (int b = 0; b < NB; ++b) tb[b].store(lb[b]);
        __syncthreads();
        if (s + 1 < steps) fetch(s + 1);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            uint4 fa[NA][2], fb[NB][2];
            const int c = kk * 4 + (lane >> 4);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = wr + i * 16 + (lane & 15);
#pragma unroll
                for (int a = 0; a < NA; ++a) fa[a][i] = la[a][r * 8 + (c ^ (r & 7))];
                const int q = wc + i * 16 + (lane & 15);
#pragma unroll
                for (int b = 0; b < NB; ++b) fb[b][i] = lb[b][q * 8 + (c ^ (q & 7))];
            }
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int a = 0; a < NA; ++a) acc[b][i][j].v[a] = mma<T>(fb[b][j], fa[a][i], acc[b][i][j].v[a]);
        }
        __syncthreads();
    }
    float down = 1.0f;
    if constexpr (MODE != GATED_FWD) down = range_down<T>(g.range);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int64_t row = row0 + wr + i * 16 + (lane & 15), col = col0 + wc + j * 16 + (lane >> 4) * 4;
            if (row >= g.m) continue;
            const f32x4 first = acc[0][i][j].all(), second = acc[NB - 1][i][j].all();
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (col + r >= g.n) continue;
                if constexpr (MODE == GATED_FWD) {
                    const float gv = first[r], uv = second[r];
                    ((T*)g.out[0])[row * g.os + col + r] = from_float<T>(activate<T>(gv, g.act) * uv);
                    if (g.keep_g) {
                        g.keep_g[row * g.n + col + r] = gv;
                        g.keep_u[row * g.n + col + r] = uv;
                    }
                } else {
                    const float v = first[r];
                    if (g.splits > 1) g.part[(((int64_t)z * g.splits + split) * g.m + row) * g.n + col + r] = v;
                    else ((T*)g.out[z])[row * g.os + col + r] = from_float<T>(v * down);
                }
            }
        }
}

// ---------------------------------------------------------------------------------------------------------------------
// Small products: what counts is how soon the last load is back, so FR x FR fragments of outputs a workgroup, its 8 waves take turns
// along the contraction with fragments loaded straight into registers, and their sums are joined in LDS in a fixed order.  No
// staging, no barrier until then (95 x 621 -> 128 in 32 bits: 40 us with the 64 x 64 tile, which has 4 workgroups of 20 steps there;
// 12 with 2 x 2 fragments, where 12 CUs are short of matrix instructions; 7 with one).
constexpr int SB = 32, SMALL_WAVES = 8;

template <typename T, bool KC, bool WHOLE>
__device__ __forceinline__ uint4 small_fragment(const Operand& o, int64_t row, int64_t k, int64_t k1) {
    constexpr int V = 16 / sizeof(T);
    const T* p = (const T*)o.p;
    Pack<T> r;
    if constexpr (KC && WHOLE) {
        r = load_pack(p + row * o.sr + k);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) r.v[j] = WHOLE || k + j < k1 ? p[KC ? row * o.sr + k + j : (k + j) * o.sk + row] : from_float<T>(0.0f);
    }
    return __builtin_bit_cast(uint4, r);
}

// What the backward products of a small problem need of dg (which = 0) and du (1), computed where it is used, in 32 bits: element (row, k)
// of the operand is element (row, k) of dh, g, u if KC, else (k, row).
struct SlopeOperand {
    const void* dh;
    const float *kg, *ku;
    int64_t dhs, n;               // row strides of dh; of kg and ku
    int act;
};
template <typename T>
struct Slopes {
    float v[Pack<T>::N];
};
template <typename T, bool KC, bool WHOLE>
__device__ __forceinline__ Slopes<T> slope_fragment(const SlopeOperand& o, int which, int64_t row, int64_t k, int64_t k1) {
    Slopes<T> r;
#pragma unroll
    for (int j = 0; j < Pack<T>::N; ++j) {
        const int64_t i = KC ? row : k + j, c = KC ? k + j : row;
        r.v[j] = 0.0f;
        if (WHOLE || k + j < k1) {
            float a, da;
            activation<T>(o.kg[i * o.n + c], o.act, a, da);
            const float d = to_float(((const T*)o.dh)[i * o.dhs + c]);
            r.v[j] = which ? d * a : d * o.ku[i * o.n + c] * da;
        }
    }
    return r;
}

// A fragment of the second operand against one of the first, in parts of the same type or in 32 bits (instructions of 32 bits then, which take
// element j of every lane: a sixteenth of the speed, over a contraction of a few hundred).
template <typename T, int NA>
__device__ __forceinline__ void product(const uint4& b, const Parts<NA>& a, Sums<NA>& c) {
#pragma unroll
    for (int p = 0; p < NA; ++p) c.v[p] = mma<T>(b, a.v[p], c.v[p]);
}
template <typename T>
__device__ __forceinline__ void product(const uint4& b, const Slopes<T>& a, Sums<1>& c) {
    const Pack<T> v = __builtin_bit_cast(Pack<T>, b);
#pragma unroll
    for (int j = 0; j < Pack<T>::N; ++j) c.v[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(to_float(v.v[j]), a.v[j], c.v[0], 0, 0, 0);
}

// The body: NB products side by side (one first operand, in fragments of type A, NB second ones), slabs of contraction [kb, ke) dealt to the waves; fa(i, k, whole)
// and fb(b, i, k, whole) give fragments i < FR.
template <typename T, typename A, int NA, int NB, int FR, typename FA, typename FB>
__device__ __forceinline__ void small_sums(Sums<NA> (&acc)[NB][FR][FR], int64_t kb, int64_t ke, FA&& fa, FB&& fb) {
    constexpr int SLAB = 64 / sizeof(T), V = 16 / sizeof(T);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t slabs = (ke - kb) / SLAB;
    auto slab = [&](int64_t k0, auto whole) {
        const int64_t k = k0 + (lane >> 4) * V;
        A a[FR];
        uint4 b[NB][FR];
#pragma unroll
        for (int i = 0; i < FR; ++i) {
            a[i] = fa(i, k, whole);
#pragma unroll
            for (int q = 0; q < NB; ++q) b[q][i] = fb(q, i, k, whole);
        }
#pragma unroll
        for (int q = 0; q < NB; ++q)
#pragma unroll
            for (int i = 0; i < FR; ++i)
#pragma unroll
                for (int j = 0; j < FR; ++j) product<T>(b[q][j], a[i], acc[q][i][j]);
    };
#pragma unroll 4
    for (int64_t s = wave; s < slabs; s += SMALL_WAVES) slab(kb + s * SLAB, std::true_type{});
    if (kb + slabs * SLAB < ke && slabs % SMALL_WAVES == wave) slab(kb + slabs * SLAB, std::false_type{});      // the broken last one
}
// The waves' sums, in wave order: fragment `wave` of the FR * FR in v of the first waves.
template <int NA, int NB, int FR>
__device__ __forceinline__ void small_join(const Sums<NA> (&acc)[NB][FR][FR], f32x4 (&v)[NB], f32x4 (*sums)[NB * FR * FR][64]) {
    constexpr int F = FR * FR;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < FR; ++i)
#pragma unroll
            for (int j = 0; j < FR; ++j) sums[wave][b * F + i * FR + j][lane] = acc[b][i][j].all();
    __syncthreads();
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        v[b] = sums[0][b * F + wave % F][lane];
#pragma unroll
        for (int w = 1; w < SMALL_WAVES; ++w) v[b] += sums[w][b * F + wave % F][lane];
    }
}

template <typename T, int MODE, bool AKC, bool BKC, int FR, int NA>
__global__ __launch_bounds__(64 * SMALL_WAVES) void k_gated_small(GatedArgs g) {
    constexpr int SLAB = 64 / sizeof(T), NB = MODE == GATED_FWD ? 2 : 1, SB = 16 * FR;
    __shared__ f32x4 sums[SMALL_WAVES][NB * FR * FR][64];
    const int64_t nt = (g.n + SB - 1) / SB;
    const int64_t row0 = (int64_t)(blockIdx.x / nt) * SB, col0 = (int64_t)(blockIdx.x % nt) * SB;
    const int z = MODE == GATED_PAIR ? blockIdx.z : 0, split = blockIdx.y;
    const int64_t per = ((g.k + g.splits - 1) / g.splits + SLAB - 1) / SLAB * SLAB;
    const int64_t kb = min(split * per, g.k), ke = min(kb + per, g.k);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Sums<NA> acc[NB][FR][FR];
    int64_t ra[FR], rb[FR];                      // rows behind the last repeat it: their outputs are not stored
#pragma unroll
    for (int i = 0; i < FR; ++i) ra[i] = min(row0 + i * 16 + (lane & 15), g.m - 1), rb[i] = min(col0 + i * 16 + (lane & 15), g.n - 1);
#pragma unroll
    for (int part = 0; part < (MODE == GATED_SUM ? 2 : 1); ++part) {
        const Operand oa = MODE == GATED_PAIR && z ? g.a[1] : g.a[part], ob = g.b[part], ob2 = g.b[1];
        const Operand rest = MODE == GATED_PAIR && z ? g.rest[1] : g.rest[part];
        small_sums<T, Parts<NA>>(acc, kb, ke, [&](int i, int64_t k, auto whole) {
                              Parts<NA> r;
                              r.v[0] = small_fragment<T, AKC, whole.value>(oa, ra[i], k, ke);
                              if constexpr (NA == 2) r.v[1] = small_fragment<T, AKC, whole.value>(rest, ra[i], k, ke);
                              return r;
                          },
                          [&](int b, int i, int64_t k, auto whole) { return small_fragment<T, BKC, whole.value>(b ? ob2 : ob, rb[i], k, ke); });
    }
    f32x4 v[NB];
    small_join(acc, v, sums);
    if (wave >= FR * FR) return;
    float down = 1.0f;
    if constexpr (MODE != GATED_FWD) down = range_down<T>(g.range);
    const int64_t row = row0 + wave / FR * 16 + (lane & 15), col = col0 + wave % FR * 16 + (lane >> 4) * 4;
    if (row >= g.m) return;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (col + r >= g.n) continue;
        if constexpr (MODE == GATED_FWD) {
            ((T*)g.out[0])[row * g.os + col + r] = from_float<T>(activate<T>(v[0][r], g.act) * v[NB - 1][r]);
            if (g.keep_g) g.keep_g[row * g.n + col + r] = v[0][r], g.keep_u[row * g.n + col + r] = v[NB - 1][r];
        } else if (g.splits > 1) {
            g.part[(((int64_t)z * g.splits + split) * g.m + row) * g.n + col + r] = v[0][r];
        } else {
            ((T*)(z ? g.out[1] : g.out[0]))[row * g.os + col + r] = from_float<T>(v[0][r] * down);
        }
    }
}

// The whole backward pass of a small problem in one launch: the tiles of dx, then those of dwg and of dwu, each with its part of dg
// and du computed on the way into the matrix instructions (every tile column again, which is why it has to be small; 95 x 621 -> 128 in
// 32 bits: 14 us, bound by the chain of loads and erfc; forward + backward 25 us, 31 with three launches).  dg and du stay in 32 bits, and
// so do the products: as two numbers of 16 bits they took as long, and in float16 a launch more for their range.
template <typename T>
__global__ __launch_bounds__(64 * SMALL_WAVES) void k_gated_small_back(SlopeOperand s, Operand x, Operand wg, Operand wu, int64_t m, int64_t k, int64_t h,
                                                                       void* dx, int64_t dxs, void* dwg, void* dwu, int64_t dws) {
    __shared__ f32x4 sums[SMALL_WAVES][4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t nt = (k + SB - 1) / SB, tiles_x = dx ? (m + SB - 1) / SB * nt : 0, tiles_w = (h + SB - 1) / SB * nt;
    int64_t id = blockIdx.x;
    Sums<1> acc[1][2][2];
    f32x4 v[1];
    const int64_t col0 = id < tiles_x ? id % nt * SB : (id - tiles_x) % nt * SB;
    int64_t rb[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) rb[i] = min(col0 + i * 16 + (lane & 15), k - 1);
    void* out;
    int64_t row0, rows, os;
    if (id < tiles_x) {                        // dx = dg wg + du wu, contraction over the hidden units
        row0 = id / nt * SB, rows = m, os = dxs, out = dx;
        int64_t ra[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) ra[i] = min(row0 + i * 16 + (lane & 15), m - 1);
#pragma unroll
        for (int which = 0; which < 2; ++which)
            small_sums<T, Slopes<T>>(acc, 0, h, [&](int i, int64_t q, auto whole) { return slope_fragment<T, true, whole.value>(s, which, ra[i], q, h); },
                             [&](int, int i, int64_t q, auto whole) { return small_fragment<T, false, whole.value>(which ? wu : wg, rb[i], q, h); });
    } else {                                   // dw = d^T x, contraction over the rows
        id -= tiles_x;
        const int which = id >= tiles_w;
        if (which) id -= tiles_w;
        row0 = id / nt * SB, rows = h, os = dws, out = which ? dwu : dwg;
        int64_t ra[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) ra[i] = min(row0 + i * 16 + (lane & 15), h - 1);
        small_sums<T, Slopes<T>>(acc, 0, m, [&](int i, int64_t q, auto whole) { return slope_fragment<T, false, whole.value>(s, which, ra[i], q, m); },
                         [&](int, int i, int64_t q, auto whole) { return small_fragment<T, false, whole.value>(x, rb[i], q, m); });
    }
    small_join(acc, v, sums);
    if (wave >= 4) return;
    const int64_t row = row0 + (wave >> 1) * 16 + (lane & 15), col = col0 + (wave & 1) * 16 + (lane >> 4) * 4;
    if (row >= rows) return;
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (col + r < k) ((T*)out)[row * os + col + r] = from_float<T>(v[0][r]);
}

// The split sums of one output, added in split order.
template <typename T>
__global__ __launch_bounds__(256) void k_gated_join(GatedArgs g) {
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x, z = blockIdx.y;
    const float down = range_down<T>(g.range);
    if (e >= g.m * g.n) return;
    const float* p = g.part + z * g.splits * g.m * g.n + e;
    float v = 0.0f;
#pragma unroll 8
    for (int s = 0; s < g.splits; ++s) v += p[(int64_t)s * g.m * g.n];
    ((T*)g.out[z])[e / g.n * g.os + e % g.n] = from_float<T>(v * down);
}

// The largest finite |dg| and |du|, in pieces.  One more pass over dh and the kept products (16384 x 8192: 0.3 ms).
constexpr int RANGE_THREADS = 1024;
template <typename T>
__global__ __launch_bounds__(RANGE_THREADS) void k_gated_range(const T* __restrict__ dh, int64_t dhs, const float* __restrict__ kg, const float* __restrict__ ku,
                                                     int64_t m, int64_t n, int act, float* __restrict__ range) {
    constexpr int V = 4;
    const int64_t packs = (n + V - 1) / V;
    float most = 0.0f;
    auto look = [&](float d, float gv, float uv) {
        float a, da;
        activation<T>(gv, act, a, da);
        const float g = fabsf(d * uv * da), u = fabsf(d * a);
        most = fmaxf(most, g < INFINITY ? g : 0.0f);
        most = fmaxf(most, u < INFINITY ? u : 0.0f);
    };
    for (int64_t id = (int64_t)blockIdx.x * RANGE_THREADS + threadIdx.x; id < m * packs; id += (int64_t)gridDim.x * RANGE_THREADS) {
        const int64_t row = id / packs, c = (id % packs) * V, e = row * n + c;
        const T* d = dh + row * dhs + c;
        if (c + V <= n) {
            T pd[V];
            float gv[V], uv[V];
            __builtin_memcpy(pd, d, sizeof(pd));
            __builtin_memcpy(gv, kg + e, sizeof(gv));
            __builtin_memcpy(uv, ku + e, sizeof(uv));
#pragma unroll
            for (int i = 0; i < V; ++i) look(to_float(pd[i]), gv[i], uv[i]);
        } else {
            for (int i = 0; c + i < n; ++i) look(to_float(d[i]), kg[e + i], ku[e + i]);
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
    __shared__ float waves[RANGE_THREADS / 64];
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = most;
    __syncthreads();
    // a piece a workgroup; the first one clears those that no workgroup has
    if (threadIdx.x == 0) {
#pragma unroll
        for (int i = 0; i < RANGE_THREADS / 64; ++i) most = fmaxf(most, waves[i]);
        range[blockIdx.x] = most;
    }
    if (blockIdx.x == 0 && threadIdx.x >= gridDim.x && threadIdx.x < RANGE_PIECES) range[threadIdx.x] = 0.0f;
}

// dg = dh u act'(g), du = dh act(g), and what their roundings left.
template <typename T, bool REST>
__global__ __launch_bounds__(256) void k_gated_slopes(const T* __restrict__ dh, int64_t dhs, const float* __restrict__ kg,
                                                      const float* __restrict__ ku, int64_t m, int64_t n, int act, const float* range,
                                                      T* __restrict__ dg, T* __restrict__ du, T* __restrict__ dg_rest, T* __restrict__ du_rest) {
    constexpr int V = Pack<T>::N;
    const int64_t packs = (n + V - 1) / V;
    const float up = range_up<T>(range);
    for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < m * packs; id += (int64_t)gridDim.x * 256) {
        const int64_t row = id / packs, c = (id % packs) * V;
        const int64_t e = row * n + c;
        const T* d = dh + row * dhs + c;
        const int len = (int)min((int64_t)V, n - c);
        Pack<T> pd, og, ou, rg, ru;
        float gv[V], uv[V];
        if (len == V) {
            pd = load_pack(d);
            __builtin_memcpy(gv, kg + e, sizeof(gv));
            __builtin_memcpy(uv, ku + e, sizeof(uv));
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                pd.v[i] = i < len ? d[i] : from_float<T>(0.0f);
                gv[i] = i < len ? kg[e + i] : 0.0f;
                uv[i] = i < len ? ku[e + i] : 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float a, da;
            activation<T>(gv[i], act, a, da);
            const float sg = to_float(pd.v[i]) * uv[i] * da * up, su = to_float(pd.v[i]) * a * up;
            og.v[i] = from_float<T>(sg), ou.v[i] = from_float<T>(su);
            if constexpr (REST) rg.v[i] = rounding_rest(sg, og.v[i]), ru.v[i] = rounding_rest(su, ou.v[i]);
        }
        if (len == V) {
            store_pack(dg + e, og);
            store_pack(du + e, ou);
            if constexpr (REST) store_pack(dg_rest + e, rg), store_pack(du_rest + e, ru);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (i >= len) continue;
                dg[e + i] = og.v[i], du[e + i] = ou.v[i];
                if constexpr (REST) dg_rest[e + i] = rg.v[i], du_rest[e + i] = ru.v[i];
            }
        }
    }
}

// A product that the whole-step kernels do not take: the small form up to two workgroups of 512 threads a CU (twice over), the 64 x 64
// tiles above; either with the contraction in pieces where the outputs alone leave CUs empty, of at least 4 steps.
struct AnyPlan {
    bool small = true;
    int fragments = 2, splits = 1;      // of the small form, in each direction
};
template <typename T>
AnyPlan any_plan(int64_t m, int64_t n, int64_t k, int zs, bool can_split) {
    AnyPlan p;
    const int64_t t32 = zs * ceil_div(m, SB) * ceil_div(n, SB), t64 = zs * ceil_div(m, TB) * ceil_div(n, TB);
    p.small = t32 <= 1024;
    if (t32 < 128 && !can_split) p.fragments = 1;      // (a product that can be split fills the card that way)
    const int64_t tiles = p.small ? t32 : t64, step = p.small ? SMALL_WAVES * 64 / (int64_t)sizeof(T) : STEP_BYTES / (int64_t)sizeof(T);
    if (can_split && tiles > 0 && tiles < 256) p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(512, tiles), k / (4 * step)));
    return p;
}
template <typename T, int MODE, bool AKC, bool BKC, int NA>
void launch_any(hipStream_t st, const GatedArgs& g, const AnyPlan& p) {
    const int64_t b = p.small ? 16 * p.fragments : TB;
    const dim3 grid((unsigned)(ceil_div(g.m, b) * ceil_div(g.n, b)), (unsigned)g.splits, MODE == GATED_PAIR ? 2 : 1);
    if (p.small && MODE == GATED_FWD && p.fragments == 1)
        hipLaunchKernelGGL((k_gated_small<T, GATED_FWD, true, true, 1, 1>), grid, dim3(64 * SMALL_WAVES), 0, st, g);
    else if (p.small) hipLaunchKernelGGL((k_gated_small<T, MODE, AKC, BKC, 2, NA>), grid, dim3(64 * SMALL_WAVES), 0, st, g);
    else hipLaunchKernelGGL((k_gated_tile<T, MODE, AKC, BKC, NA>), grid, dim3(256), 0, st, g);
}

}  // namespace gpbo_static
