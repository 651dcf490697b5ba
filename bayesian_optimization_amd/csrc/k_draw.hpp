// Draws from rows of scores: temperature, top-k, min-p, top-p, then one index per given uniform number.
//   valid scores: neither NaN nor -inf;  t_i = (s_i - max) / T (0 where s_i = max),  w_i = exp(t_i)
//   rank: falling score, rising index on ties.  Kept: the first top_k; of those w_i >= min_p; of those position p as long as
//   the mass in front of it is < top_p times their mass (the first always).
//   pick(u): the lowest kept i, in index order, with C_i > u Z;  C the running sum of kept w, Z their mass;  logp = t_i - log Z.
// No sort of the row: the kept set is { score > cut } plus the first few, by index, of those equal to the cut, and the cut is
// found digit by digit.  A score's bits are mapped to an unsigned key of the same order; a histogram over 11 bits of it, counts
// for top-k, masses for top-p, names the digit that holds the cut, until at most LIST keys are left to be ranked against each
// other.  Counts are integers, and the masses of a histogram are integers too (two words of 35 bits behind the point each), so
// that the order in which atomics arrive changes nothing; all other sums are in 64 bits in a fixed order.
#pragma once

#include <hip/hip_runtime.h>

#include "static_ops.hpp"

namespace gpbo_static {

constexpr int DRAW_THREADS = 1024, LIST = 1024, TILES = 1024;
constexpr int DIGIT = 11, BINS = 1 << DIGIT;

template <typename T>
struct Score {
    using Key = uint32_t;
    static constexpr int BITS = 32;
    // order-preserving; 0 for NaN and -inf (never drawn); -0 and +0 alike
    static __device__ __forceinline__ Key key(T v) {
        const float f = to_float(v) + 0.0f;
        if (!(f > -INFINITY)) return 0;
        const uint32_t b = __float_as_uint(f);
        return (b >> 31) ? ~b : (b | 0x80000000u);
    }
    static __device__ __forceinline__ double value(Key k) {
        return (double)__uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k);
    }
};
template <>
struct Score<double> {
    using Key = uint64_t;
    static constexpr int BITS = 64;
    static __device__ __forceinline__ Key key(double v) {
        const double f = v + 0.0;
        if (!(f > -INFINITY)) return 0;
        const uint64_t b = (uint64_t)__double_as_longlong(f);
        return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
    }
    static __device__ __forceinline__ double value(Key k) {
        return __longlong_as_double((long long)((k >> 63) ? (k & 0x7fffffffffffffffull) : ~k));
    }
};

struct DrawArgs {
    const void* scores;
    int64_t rows, cols, stride;
    const double* u;
    int64_t draws;
    double temperature, top_p, min_p;
    int64_t top_k;
    const double* params;         // per row {temperature, top_k, top_p, min_p}, or null
    int64_t* index;
    double* logp;                 // or null
};

// One row's settings; values outside their range mean the nearest end of it (a row's settings come from device memory and
// cannot be refused).
struct DrawRow {
    double temperature, top_p, min_p;
    int64_t top_k;                // 0: all
    bool greedy;
    __device__ __forceinline__ DrawRow(const DrawArgs& a, int64_t row) {
        double k;
        if (a.params) {
            const double* p = a.params + row * 4;
            temperature = p[0], k = p[1], top_p = p[2], min_p = p[3];
        } else {
            temperature = a.temperature, k = (double)a.top_k, top_p = a.top_p, min_p = a.min_p;
        }
        top_k = (k >= 1.0 && k < (double)a.cols) ? (int64_t)k : 0;
        if (!(top_p < 1.0)) top_p = 1.0;
        if (!(min_p > 0.0)) min_p = 0.0;
        if (min_p > 1.0) min_p = 1.0;
        greedy = !(temperature > 0.0) || top_k == 1 || top_p <= 0.0;
    }
};

template <typename T>
__device__ __forceinline__ double draw_t(typename Score<T>::Key k, typename Score<T>::Key top, double temperature) {
    return k == top ? 0.0 : (Score<T>::value(k) - Score<T>::value(top)) / temperature;
}

// A weight in [0, 1] as two integers: 35 bits behind the point, and the next 35.  2^28 of them add up without overflow.
__device__ __forceinline__ void to_fixed(double w, unsigned long long& hi, unsigned long long& lo) {
    const double s = w * 34359738368.0;
    const double h = floor(s);
    hi = (unsigned long long)h;
    lo = (unsigned long long)((s - h) * 34359738368.0);
}
__device__ __forceinline__ double from_fixed(unsigned long long hi, unsigned long long lo) {
    return (double)hi * (1.0 / 34359738368.0) + (double)lo * (1.0 / 34359738368.0 / 34359738368.0);
}

// Inclusive sums over the workgroup's threads, in thread order; the total comes back too.  Two barriers; red: 32 doubles.
template <typename V>
__device__ __forceinline__ V block_scan(V v, V* red, V& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const V x = __shfl_up(v, o);
        if (lane >= o) v += x;
    }
    __syncthreads();                           // earlier reads of red are done
    if (lane == 63) red[wave] = v;
    __syncthreads();
    V before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < DRAW_THREADS / 64; ++i) {
        if (i == wave) before = all;
        all += red[i];
    }
    total = all;
    return before + v;
}

template <typename T>
struct DrawLds {
    using Key = typename Score<T>::Key;
    union {
        struct {
            unsigned int count[BINS];
            unsigned long long hi[BINS], lo[BINS];
        } h;
        struct {
            Key key[LIST], key2[LIST];
            uint32_t idx[LIST], idx2[LIST];
            double c[LIST];
            uint32_t pick[LIST];
        } l;
        struct {
            double c[TILES];                   // kept mass up to and including a tile
            uint32_t ties[TILES];              // scores equal to the cut in front of a tile
        } t;
    };
    double red[32];
    unsigned long long red_u[32];
    Key best_key[16];
    uint32_t best_idx[16];
    Key cut;
    uint32_t cut_ties, n_list, pick_bin;
    unsigned int bin_count;
    double above, target;
    long long rank_left;
};

// Everything behind the list: n <= LIST (key, index) pairs in l.key, l.idx that hold every score that can be kept.
template <typename T>
__device__ void draw_from_list(DrawLds<T>& s, const DrawArgs& a, const DrawRow& p, int64_t row, int n, typename Score<T>::Key top) {
    using Key = typename Score<T>::Key;
    const int tid = threadIdx.x;
    __syncthreads();
    const Key k = tid < n ? s.l.key[tid] : 0;
    const uint32_t ix = tid < n ? s.l.idx[tid] : 0;
    if (tid < n) {
        int rank = 0;
        for (int j = 0; j < n; ++j) {
            const Key kj = s.l.key[j];
            rank += (kj > k) || (kj == k && s.l.idx[j] < ix);
        }
        s.l.key2[rank] = k;
        s.l.idx2[rank] = ix;
    }
    __syncthreads();
    // by rank from here on: thread = position
    const Key kr = tid < n ? s.l.key2[tid] : 0;
    const double w = kr ? exp(draw_t<T>(kr, top, p.temperature)) : 0.0;
    bool keep = kr != 0 && (p.top_k == 0 || tid < p.top_k) && w >= p.min_p;
    double total;
    double run = block_scan(keep ? w : 0.0, s.red, total);
    if (p.top_p < 1.0) {
        keep = keep && (tid == 0 || run - w < p.top_p * total);
        __syncthreads();
    }
    // the kept ones are the first `kept` positions; now in index order
    unsigned long long kept;
    block_scan<unsigned long long>(keep ? 1ull : 0ull, s.red_u, kept);
    const uint32_t my = s.l.idx2[tid < n ? tid : 0];
    int place = 0;
    if (keep)
        for (int j = 0; j < (int)kept; ++j) place += s.l.idx2[j] < my;
    __syncthreads();
    if (keep) {
        s.l.c[place] = w;
        s.l.pick[place] = my;
        s.l.key[place] = kr;
    }
    __syncthreads();
    const double wi = tid < (int)kept ? s.l.c[tid] : 0.0;
    const double ci = block_scan(wi, s.red, total);
    __syncthreads();
    if (tid < (int)kept) s.l.c[tid] = ci;
    __syncthreads();
    for (int64_t q = tid; q < a.draws; q += DRAW_THREADS) {
        const double goal = fmax(a.u[row * a.draws + q], 0.0) * total;
        int lo = 0, hi = (int)kept - 1;        // the first c > goal; the last kept one if rounding leaves none
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (s.l.c[mid] > goal) hi = mid;
            else lo = mid + 1;
        }
        // a weight of zero is never drawn: step back over those at the end
        while (lo > 0 && s.l.c[lo] == s.l.c[lo - 1]) --lo;
        a.index[row * a.draws + q] = s.l.pick[lo];
        if (a.logp) a.logp[row * a.draws + q] = draw_t<T>(s.l.key[lo], top, p.temperature) - log(total);
    }
}

// One workgroup a row.
template <typename T>
__global__ __launch_bounds__(DRAW_THREADS) void k_draw_row(DrawArgs a) {
    using S = Score<T>;
    using Key = typename S::Key;
    __shared__ DrawLds<T> s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x;
    const T* x = (const T*)a.scores + row * a.stride;
    const uint32_t n = (uint32_t)a.cols;
    const DrawRow p(a, row);

    // the best score and the lowest index that has it
    Key bk = 0;
    uint32_t bi = 0;
    for (uint32_t i = tid; i < n; i += DRAW_THREADS) {
        const Key k = S::key(x[i]);
        if (k > bk) bk = k, bi = i;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const Key k = __shfl_xor(bk, o);
        const uint32_t i = __shfl_xor(bi, o);
        if (k > bk || (k == bk && i < bi)) bk = k, bi = i;
    }
    if (lane == 0) s.best_key[wave] = bk, s.best_idx[wave] = bi;
    __syncthreads();
    bk = 0, bi = 0;
    for (int i = 0; i < DRAW_THREADS / 64; ++i) {
        const Key k = s.best_key[i];
        if (k > bk || (k == bk && s.best_idx[i] < bi)) bk = k, bi = s.best_idx[i];
    }
    const Key top = bk;
    if (top == 0 || p.greedy) {                // nothing can be drawn: index -1; or there is no choice
        for (int64_t q = tid; q < a.draws; q += DRAW_THREADS) {
            a.index[row * a.draws + q] = top ? (int64_t)bi : -1;
            if (a.logp) a.logp[row * a.draws + q] = top ? 0.0 : -INFINITY;
        }
        return;
    }
    if (n <= LIST) {
        if (tid < (int)n) s.l.key[tid] = S::key(x[tid]), s.l.idx[tid] = tid;
        draw_from_list<T>(s, a, p, row, (int)n, top);
        return;
    }

    // kept = { key > cut } + the first cut_ties of those equal to it (by index), with w >= min_p
    Key cut = 0;
    uint32_t cut_ties = 0;
    // mode 0: the cut of top-k, by counts; mode 1: of top-p, by masses, among what mode 0 left
    for (int mode = 0; mode < 2; ++mode) {
        if (mode == 0 ? p.top_k == 0 : !(p.top_p < 1.0)) continue;
        const Key floor_key = cut;             // mode 1: keys at the cut of top-k are one group below all others
        const uint32_t floor_ties = cut_ties;
        double floor_mass = 0.0;
        if (mode == 1 && floor_ties) {
            const double w = exp(draw_t<T>(floor_key, top, p.temperature));
            if (w >= p.min_p) floor_mass = w * floor_ties;
        }
        Key prefix = 0;
        int left = S::BITS;                    // bits below the prefix
        double above = 0.0, goal = 0.0;
        long long rank = p.top_k;
        bool done = false, spare = false;
        while (!done) {
            const int digit = min(DIGIT, left), shift = left - digit;
            for (int b = tid; b < BINS; b += DRAW_THREADS) s.h.count[b] = 0, s.h.hi[b] = 0, s.h.lo[b] = 0;
            __syncthreads();
            for (uint32_t i = tid; i < n; i += DRAW_THREADS) {
                const Key k = S::key(x[i]);
                if (k == 0 || (left < S::BITS && (k >> (left & (S::BITS - 1))) != prefix)) continue;
                const int b = (int)((k >> shift) & ((1u << digit) - 1));
                if (mode == 0) {
                    atomicAdd(&s.h.count[b], 1u);
                } else {
                    if (k <= floor_key) continue;
                    const double w = exp(draw_t<T>(k, top, p.temperature));
                    if (!(w >= p.min_p)) continue;
                    unsigned long long hi, lo;
                    to_fixed(w, hi, lo);
                    atomicAdd(&s.h.count[b], 1u);
                    atomicAdd(&s.h.hi[b], hi);
                    if (lo) atomicAdd(&s.h.lo[b], lo);
                }
            }
            __syncthreads();
            // thread t owns bins from the top: BINS - 1 - 2t and the next lower one
            const int b1 = BINS - 1 - 2 * tid, b0 = b1 - 1;
            if (mode == 0) {
                const unsigned long long c1 = s.h.count[b1], c0 = s.h.count[b0];
                unsigned long long all;
                const unsigned long long run = block_scan(c1 + c0, s.red_u, all) - c1 - c0;
                if (left == S::BITS && all <= (unsigned long long)rank) {      // fewer valid scores than top_k: no cut
                    spare = true;
                } else {
                    const long long r1 = (long long)run, r0 = (long long)(run + c1);
                    if (c1 && r1 < rank && r1 + (long long)c1 >= rank) s.pick_bin = b1, s.rank_left = rank - r1, s.bin_count = (unsigned)c1;
                    if (c0 && r0 < rank && r0 + (long long)c0 >= rank) s.pick_bin = b0, s.rank_left = rank - r0, s.bin_count = (unsigned)c0;
                }
            } else {
                const double m1 = from_fixed(s.h.hi[b1], s.h.lo[b1]), m0 = from_fixed(s.h.hi[b0], s.h.lo[b0]);
                double all;
                const double incl = block_scan(m1 + m0, s.red, all);
                if (left == S::BITS) goal = p.top_p * (all + floor_mass);
                // the digit in which the running mass first reaches the goal; the lowest one in use if rounding leaves none
                if (tid == 0) s.pick_bin = 0xffffffffu, s.cut_ties = 0xffffffffu;
                __syncthreads();
                spare = left == S::BITS && !(above + all >= goal);            // everything above the group is kept
                if (s.h.count[b1] && above + (incl - m1 - m0) + m1 >= goal) atomicMin(&s.pick_bin, (unsigned)(BINS - 1 - b1));
                if (s.h.count[b0] && above + incl >= goal) atomicMin(&s.pick_bin, (unsigned)(BINS - 1 - b0));
                __syncthreads();
                unsigned bin = s.pick_bin != 0xffffffffu ? BINS - 1 - s.pick_bin : 0xffffffffu;
                if (bin == 0xffffffffu && !spare) {
                    if (s.h.count[b0]) atomicMin(&s.cut_ties, (unsigned)b0);
                    else if (s.h.count[b1]) atomicMin(&s.cut_ties, (unsigned)b1);
                    __syncthreads();
                    bin = s.cut_ties;
                }
                if (bin == (unsigned)b1) s.above = above + (incl - m1 - m0), s.bin_count = s.h.count[b1], s.rank_left = b1;
                if (bin == (unsigned)b0) s.above = above + (incl - m0), s.bin_count = s.h.count[b0], s.rank_left = b0;
            }
            __syncthreads();
            if (spare) break;
            unsigned bin;
            if (mode == 0) {
                bin = s.pick_bin;
                rank = s.rank_left;
            } else {
                bin = (unsigned)s.rank_left;
                above = s.above;
            }
            const unsigned in_bin = s.bin_count;
            prefix = (prefix << digit) | (Key)bin;
            left = shift;
            __syncthreads();
            if (left == 0) {                   // one key: all of them ties
                cut = prefix;
                if (mode == 0) {
                    cut_ties = (uint32_t)rank;
                } else {
                    const double w = exp(draw_t<T>(cut, top, p.temperature));
                    double r = ceil((goal - above) / w);
                    if (!(r >= 1.0)) r = 1.0;
                    cut_ties = (uint32_t)fmin(r, (double)in_bin);
                }
                done = true;
            } else if (in_bin <= LIST) {       // few enough to rank them against each other
                if (tid == 0) s.n_list = 0;
                __syncthreads();
                for (uint32_t i = tid; i < n; i += DRAW_THREADS) {
                    const Key k = S::key(x[i]);
                    if (k == 0 || (k >> left) != prefix) continue;
                    if (mode == 1 && (k <= floor_key || !(exp(draw_t<T>(k, top, p.temperature)) >= p.min_p))) continue;
                    const uint32_t at = atomicAdd(&s.n_list, 1u);
                    s.l.key[at] = k, s.l.idx[at] = i;
                }
                __syncthreads();
                const int m = (int)s.n_list;
                const Key k = tid < m ? s.l.key[tid] : 0;
                const uint32_t ix = tid < m ? s.l.idx[tid] : 0;
                if (tid < m) {
                    int r = 0;
                    for (int j = 0; j < m; ++j) {
                        const Key kj = s.l.key[j];
                        r += (kj > k) || (kj == k && s.l.idx[j] < ix);
                    }
                    s.l.key2[r] = k;
                }
                __syncthreads();
                const Key kr = tid < m ? s.l.key2[tid] : 0;
                bool in = false;
                if (mode == 0) {
                    in = tid < rank;
                } else {
                    const double w = kr ? exp(draw_t<T>(kr, top, p.temperature)) : 0.0;
                    double all;
                    const double incl = block_scan(w, s.red, all);
                    in = kr != 0 && (tid == 0 || above + (incl - w) < goal);
                }
                unsigned long long taken;
                block_scan<unsigned long long>(in ? 1ull : 0ull, s.red_u, taken);
                cut = s.l.key2[(int)taken - 1];
                unsigned long long same;
                block_scan<unsigned long long>(in && kr == cut ? 1ull : 0ull, s.red_u, same);
                cut_ties = (uint32_t)same;
                done = true;
                __syncthreads();
            }
        }
        if (spare && mode == 1) {              // all above the group, and of the group as many as the mass still asks for
            cut = floor_key;
            cut_ties = floor_ties;
            if (floor_ties) {
                const double w = exp(draw_t<T>(floor_key, top, p.temperature));
                double strict;
                // mass above the group, again from the histogram: the total of its first level
                const int b1 = BINS - 1 - 2 * tid, b0 = b1 - 1;
                block_scan(from_fixed(s.h.hi[b1], s.h.lo[b1]) + from_fixed(s.h.hi[b0], s.h.lo[b0]), s.red, strict);
                double r = w > 0.0 ? ceil((goal - strict) / w) : 0.0;
                if (!(r >= 0.0)) r = 0.0;
                cut_ties = (uint32_t)fmin(r, (double)floor_ties);
            }
            __syncthreads();
        }
    }

    // kept mass of TILES pieces of the row, in index order: ties with the cut are counted first (they are kept by index)
    const uint32_t piece = (uint32_t)round_up(ceil_div(n, TILES), 64);
    __syncthreads();
    for (uint32_t t = wave; t < TILES; t += DRAW_THREADS / 64) {
        uint32_t c = 0;
        if (cut_ties)
            for (uint32_t i = 0; i < piece; i += 64) {
                const uint64_t e = (uint64_t)t * piece + i + lane;
                c += __popcll(__ballot(e < n && S::key(x[e < n ? e : 0]) == cut));
            }
        if (lane == 0) s.t.ties[t] = c;
    }
    __syncthreads();
    {
        const unsigned long long v = s.t.ties[tid];
        unsigned long long all;
        const unsigned long long incl = block_scan(v, s.red_u, all);
        __syncthreads();
        s.t.ties[tid] = (uint32_t)(incl - v);
        __syncthreads();
    }
    auto weight = [&](uint64_t e, uint32_t& ties) -> double {     // of element e of this wave's 64; ties: of the cut so far
        const Key k = e < n ? S::key(x[e]) : 0;
        const bool tie = k == cut && cut_ties;
        const unsigned long long votes = __ballot(tie);
        const uint32_t mine = ties + __popcll(votes & ((1ull << lane) - 1));
        ties += __popcll(votes);
        if (k == 0 || (k <= cut && !(tie && mine < cut_ties))) return 0.0;
        const double w = exp(draw_t<T>(k, top, p.temperature));
        return w >= p.min_p ? w : 0.0;
    };
    for (uint32_t t = wave; t < TILES; t += DRAW_THREADS / 64) {
        uint32_t ties = s.t.ties[t];
        double m = 0.0;
        for (uint32_t i = 0; i < piece; i += 64) m += weight((uint64_t)t * piece + i + lane, ties);
        m = wave_sum(m);
        if (lane == 0) s.t.c[t] = m;
    }
    __syncthreads();
    double total;
    {
        const double incl = block_scan(s.t.c[tid], s.red, total);
        __syncthreads();
        s.t.c[tid] = incl;
        __syncthreads();
    }
    for (int64_t q = wave; q < a.draws; q += DRAW_THREADS / 64) {
        const double goal = fmax(a.u[row * a.draws + q], 0.0) * total;
        int lo = 0, hi = TILES - 1;            // the first tile whose sum passes the goal, the last with any mass if none does
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (s.t.c[mid] > goal) hi = mid;
            else lo = mid + 1;
        }
        while (lo > 0 && s.t.c[lo] == s.t.c[lo - 1]) --lo;
        uint32_t ties = s.t.ties[lo];
        double run = lo ? s.t.c[lo - 1] : 0.0;
        int64_t pick = -1;
        for (uint32_t i = 0; i < piece; i += 64) {
            const uint64_t e = (uint64_t)lo * piece + i + lane;
            const double w = weight(e, ties);
            double c = w;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const double v = __shfl_up(c, o);
                if (lane >= o) c += v;
            }
            const unsigned long long any = __ballot(w > 0.0), hit = __ballot(w > 0.0 && run + c > goal);
            const uint64_t at = (uint64_t)lo * piece + i;
            if (hit) {
                pick = (int64_t)(at + __ffsll((unsigned long long)hit) - 1);
                break;
            }
            if (any) pick = (int64_t)(at + 63 - __clzll((long long)any));
            run += __shfl(c, 63);
        }
        if (lane == 0) {
            a.index[row * a.draws + q] = pick;
            if (a.logp) a.logp[row * a.draws + q] = draw_t<T>(S::key(x[pick]), top, p.temperature) - log(total);
        }
    }
}

template <typename T>
hipError_t draw_rows(hipStream_t st, const DrawArgs& a) {
    hipLaunchKernelGGL(k_draw_row<T>, dim3((unsigned)a.rows), dim3(DRAW_THREADS), 0, st, a);
    return hipGetLastError();
}

}  // namespace gpbo_static
