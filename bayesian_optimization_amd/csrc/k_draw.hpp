// Draws from rows of scores: temperature, top-k, min-p, top-p, then one index per given uniform number.
//   valid scores: neither NaN nor -inf;  t_i = (s_i - max) / T (0 where s_i = max),  w_i = exp(t_i)
//   rank: falling score, rising index on ties.  Kept: the first top_k; of those w_i >= min_p; of those position p as long as
//   the mass in front of it is < top_p times their mass (the first always).
//   pick(u): the lowest kept i, in index order, with C_i > u Z;  C the running sum of kept w, Z their mass;  logp = t_i - log Z.
// No sort of the row: the kept set is { score > cut } plus the first few, by index, of those equal to the cut.  The cut is found by
// histograms of 2048 bins over the range of scores that can hold it, counts for top-k, masses for top-p: the first two linear in
// the score, which spreads what lies near the best over many bins, further ones of the range of keys that is left (a score's
// bits, mapped to an unsigned key of the same order), until at most LIST keys remain to be sorted.  Where a list holds all that
// can be kept, the rest of the work is done on it alone; that is tried first where a bound is at hand: the k-th best of the
// maxima of disjoint parts of the row is a lower bound of the k-th best score, and min_p is one of all that is kept.
// Counts are integers, and so are the masses of a histogram (two words of 35 bits each), so that the order in which atomics
// arrive changes nothing; all other sums are in 64 bits in a fixed order.
// Bound by memory: a pass over the row per step, two to five of them, and by the exponential of the scores of a top-p step.
// Short rows: one workgroup a row does everything (k_draw_row).  Long rows: the same steps with many workgroups a row, one
// launch a step, the state of a row in the workspace; the last workgroup to arrive at a step takes its decision.
// Measured: 256 rows of 65537 scores of 16 bits with top_k and top_p 35 us (a pass over them 7 at the rate of a copy; what is left is
// one workgroup's chain of small steps, whose kernel spills 17 to 28 of its 128 registers), 16.8 M float64 scores with min_p and top_p 88
// to 94 us where 1024 of them or fewer pass min_p, else 108, 97 to 123 with scores that no cache holds (two passes of 30, launches with
// nothing to do 2 to 4 each, the cut and the picks 20 or 35 in one workgroup).
#pragma once

#include <hip/hip_runtime.h>

#include "static_ops.hpp"

namespace gpbo_static {

constexpr int DRAW_THREADS = 1024, LIST = 1024, LONG_LIST = 16384, TILES = 1024;
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
    static __device__ __forceinline__ Key key_of(double v) {      // of the nearest 32-bit number
        const float f = (float)v + 0.0f;
        const uint32_t b = __float_as_uint(f);
        return !(f > -INFINITY) ? 0 : (b >> 31) ? ~b : (b | 0x80000000u);
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
    static __device__ __forceinline__ Key key_of(double v) { return key(v); }
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

// Inclusive sums over the workgroup's threads, in thread order; the total comes back too.  Two barriers; red: a place a wave.
// Every sum is that of the aligned half blocks in front of it, joined from the right, so that the picks can rely on two things in
// floating point as well: the sums never fall, and one where nothing is added has its predecessor's bits (a scan in which every lane adds up
// a window that ends with it has neither: of 5000 scores whose last 2000 have no weight, a third of the rows then ended in a step there).
template <int THREADS = DRAW_THREADS, typename V>
__device__ __forceinline__ V block_scan(V v, V* red, V& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const V x = __shfl(v, (lane & -2 * o) | (o - 1));      // the sum of the half block in front
        if (lane & o) v += x;
    }
    __syncthreads();                           // earlier reads of red are done
    if (lane == 63) red[wave] = v;
    __syncthreads();
    V before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) {
        if (i == wave) before = all;
        all += red[i];
    }
    total = all;
    return before + v;
}

// How many threads, from the first on, `in` holds for without a gap.  Two barriers; red: a place a wave.
template <int THREADS = DRAW_THREADS>
__device__ __forceinline__ int block_leading(bool in, unsigned long long* red) {
    const unsigned long long out = __ballot(!in);
    __syncthreads();                           // earlier reads of red are done
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = out ? threadIdx.x + __ffsll(out) - 1 : THREADS;
    __syncthreads();
    unsigned long long first = THREADS;
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) first = min(first, red[i]);
    return (int)first;
}

// Mass in front of which a draw lies: u times the whole, u out of range counting as the nearest end.  It is below the whole, whatever that
// is ((1 - 2^-53) Z rounds to less than Z), and the running sums end at the whole without falling: there is a first sum above it, that
// sum is above its predecessor, and so its place has a weight.
__device__ __forceinline__ double draw_goal(double u, double total) { return fmin(fmax(u, 0.0), 1.0 - 0x1p-53) * total; }

// Where the search for the cut stands.  Lives in LDS (one workgroup a row) or in the workspace (many).
enum { PHASE_TOPK = 0, PHASE_TOPP = 1, PHASE_PICK = 2, PHASE_DONE = 3 };
template <typename T>
struct DrawState {
    using Key = typename Score<T>::Key;
    Key top, bot;                 // best and lowest valid key
    Key klo, khi;                 // the cut lies among keys klo .. khi
    Key cut, floor_key;           // PHASE_TOPP: the cut of top-k, whose ties are one group below all other keys
    double above, goal;           // PHASE_TOPP: mass above khi; mass to reach
    double floor_mass;
    long long rank;               // PHASE_TOPK: how many of klo .. khi are kept
    long long count_above;        // keys above khi that may be kept
    int phase, first;             // first: no histogram of this phase has been taken yet
    int linear_left;              // linear steps still to try
    int gather;                   // this step collects a list: 1 of klo .. khi, 2 of all that can be kept, 3 the same, on trial
    uint32_t cut_ties, floor_ties;
    unsigned int n_list, ticket;
    unsigned int listed;          // long rows: > 0 if the row's list in memory holds that many scores, all that can be kept
};

// What of a score counts in the present step; w is its weight (PHASE_TOPP).
template <typename T>
struct DrawStep {
    using S = Score<T>;
    using Key = typename S::Key;
    Key top, klo, khi, floor_key;
    double base, scale, min_p, temperature;
    int phase, gather, shift;
    bool linear;
    __device__ __forceinline__ DrawStep(const DrawState<T>& st, const DrawRow& p)
        : top(st.top), klo(st.klo), khi(st.khi), floor_key(st.floor_key), base(S::value(st.khi)), min_p(p.min_p), temperature(p.temperature),
          phase(st.phase), gather(st.gather) {
        const Key width = khi - klo;
        const int bits = width == 0 ? 0 : S::BITS == 64 ? 64 - __clzll((long long)width) : 32 - __clz((int)width);
        shift = bits > DIGIT ? bits - DIGIT : 0;
        const double span = base - S::value(klo);
        scale = (double)(BINS - 1) / span;
        linear = st.linear_left > 0 && shift > 0 && span < INFINITY && scale > 0.0 && scale < INFINITY;
    }
    __device__ __forceinline__ bool counts(Key k, double& w) const {
        if (k < klo || k == 0) return false;
        if (gather == 3) return true;
        if (k > khi && gather != 2) return false;
        if (phase == PHASE_TOPP) {
            if (k <= floor_key) return false;
            w = exp(draw_t<T>(k, top, temperature));
            return w >= min_p;
        }
        return true;
    }
    // bins from the top down; never falling as the key falls
    __device__ __forceinline__ int bin(Key k) const {
        if (!linear) return (int)((khi - k) >> shift);
        const double v = (base - S::value(k)) * scale;
        return v >= (double)(BINS - 1) ? BINS - 1 : (int)v;
    }
    // the keys of a bin: for the linear step the first and last key that `bin` puts there, by bisection
    __device__ void ends(int b, Key& lo, Key& hi) const {
        if (!linear) {
            const Key span = ((Key)1 << shift) - 1;
            hi = khi - ((Key)b << shift);
            lo = hi - klo > span ? hi - span : klo;
            return;
        }
        auto last_at_most = [&](int q) -> Key {       // lowest key with bin(key) <= q
            Key l = klo, h = khi;                     // bin(khi) = 0
            const Key guess = S::key_of(base - (q + 1) / scale);
            if (guess > klo && guess < khi) {         // the bisection starts around it, in growing steps
                for (Key step = 4;; step <<= 4) {
                    const Key a = guess - klo > step ? guess - step : klo, z = khi - guess > step ? guess + step : khi;
                    if ((a == klo || bin(a) > q) && bin(z) <= q) {
                        l = a, h = z;
                        break;
                    }
                    if (a == klo && z == khi) break;
                    if (step >> (S::BITS - 5)) break;
                }
            }
            while (l < h) {
                const Key mid = l + ((h - l) >> 1);
                if (bin(mid) <= q) h = mid;
                else l = mid + 1;
            }
            return h;
        };
        lo = last_at_most(b);
        hi = b == 0 ? khi : last_at_most(b - 1) - 1;
    }
};

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
    DrawState<T> st;
    double red[32];
    unsigned long long red_u[32];
    Key red_k[2][16];
    uint32_t red_i[16];
    unsigned int bin, any_bin, last;
};

// Every score of elements [begin, end) of a row, 16 bytes a load, the workgroup's threads side by side: f(key, index).  SCORES
// of them are under way before the first is looked at: with fewer, what f does with it stands between a load and the next.
template <typename T, int SCORES = 8, typename F>
__device__ __forceinline__ void each_score(const T* x, uint32_t begin, uint32_t end, F&& f) {
    constexpr uint32_t V = Pack<T>::N;
    const uint32_t packs = (end - begin) / V;
    constexpr uint32_t U = V >= SCORES ? 1 : SCORES / V;
    uint32_t c = threadIdx.x;
    for (; c + (U - 1) * DRAW_THREADS < packs; c += U * DRAW_THREADS) {
        Pack<T> p[U];
#pragma unroll
        for (uint32_t j = 0; j < U; ++j) p[j] = load_pack(x + begin + (c + j * DRAW_THREADS) * V);
#pragma unroll
        for (uint32_t j = 0; j < U; ++j)
#pragma unroll
            for (uint32_t i = 0; i < V; ++i) f(Score<T>::key(p[j].v[i]), begin + (c + j * DRAW_THREADS) * V + i);
    }
    for (; U > 1 && c < packs; c += DRAW_THREADS) {
        const Pack<T> p = load_pack(x + begin + c * V);
#pragma unroll
        for (uint32_t i = 0; i < V; ++i) f(Score<T>::key(p.v[i]), begin + c * V + i);
    }
    for (uint32_t i = begin + packs * V + threadIdx.x; i < end; i += DRAW_THREADS) f(Score<T>::key(x[i]), i);
}

// What a step looks at: a share of a row, or (listed > 0) a long list that other workgroups left in memory, read past this one's
// caches, that holds all scores that can be kept.
template <typename T>
struct DrawFrom {
    using Key = typename Score<T>::Key;
    const T* x;
    uint32_t begin, end;
    const Key* key = nullptr;
    const uint32_t* idx = nullptr;
    uint32_t listed = 0;
    template <int SCORES = 8, typename F>
    __device__ __forceinline__ void each(F&& f) const {
        if (listed) {
            for (uint32_t i = threadIdx.x; i < listed; i += DRAW_THREADS)
                f((Key)__hip_atomic_load(key + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT),
                  (uint32_t)__hip_atomic_load(idx + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
        } else {
            each_score<T, SCORES>(x, begin, end, f);
        }
    }
};

// Best key with its lowest index, and lowest valid key, of [begin, end); own: the best key this thread saw.
template <typename T>
__device__ void draw_extremes(DrawLds<T>& s, const T* x, uint32_t begin, uint32_t end, typename Score<T>::Key& top, typename Score<T>::Key& bot, uint32_t& idx,
                              typename Score<T>::Key& own) {
    using Key = typename Score<T>::Key;
    Key bk = 0, lk = ~(Key)0;
    uint32_t bi = 0;
    each_score<T, 32>(x, begin, end, [&](Key k, uint32_t i) {
        if (k > bk) bk = k, bi = i;            // a thread meets its indices in rising order
        if (k != 0 && k < lk) lk = k;
    });
    own = bk;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const Key k = __shfl_xor(bk, o), l = __shfl_xor(lk, o);
        const uint32_t i = __shfl_xor(bi, o);
        if (k > bk || (k == bk && i < bi)) bk = k, bi = i;
        if (l < lk) lk = l;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane == 0) s.red_k[0][wave] = bk, s.red_k[1][wave] = lk, s.red_i[wave] = bi;
    __syncthreads();
    top = 0, bot = ~(Key)0, idx = 0;
    for (int i = 0; i < DRAW_THREADS / 64; ++i) {
        const Key k = s.red_k[0][i];
        if (k > top || (k == top && s.red_i[i] < idx)) top = k, idx = s.red_i[i];
        if (s.red_k[1][i] < bot) bot = s.red_k[1][i];
    }
    __syncthreads();
}

// Nothing to choose: no valid score (index -1), or the best one.
template <typename T>
__device__ void draw_same(const DrawArgs& a, int64_t row, int64_t index, double logp) {
    for (int64_t q = threadIdx.x; q < a.draws; q += blockDim.x) {
        a.index[row * a.draws + q] = index;
        if (a.logp) a.logp[row * a.draws + q] = logp;
    }
}

// Thread 0: the first step of a phase, or the next phase that has any.  bound: a key that at least top_k valid keys reach, or 0; a list
// from there on is tried for a top_k of up to `most`.
template <typename T>
__device__ void draw_begin(DrawState<T>& st, const DrawRow& p, int phase, typename Score<T>::Key bound = 0, int most = LIST / 2) {
    using S = Score<T>;
    using Key = typename S::Key;
    if (phase == PHASE_TOPK && p.top_k == 0) phase = PHASE_TOPP;
    if (phase == PHASE_TOPP && !(p.top_p < 1.0) && p.min_p == 0.0) phase = PHASE_PICK;
    st.phase = phase;
    if (phase >= PHASE_PICK) return;
    st.klo = st.bot, st.khi = st.top;
    st.above = st.goal = st.floor_mass = 0.0;
    st.count_above = 0;
    st.rank = p.top_k;
    st.first = 1, st.linear_left = 2, st.gather = 0, st.n_list = 0;
    st.floor_key = 0, st.floor_ties = 0;
    if (phase == PHASE_TOPK) {
        if (bound) {
            st.klo = bound;
            if (p.top_k <= most) st.gather = 3;
        }
        return;
    }
    st.floor_key = st.cut, st.floor_ties = st.cut_ties;
    if (st.floor_ties) {
        const double w = exp(draw_t<T>(st.floor_key, st.top, p.temperature));
        if (w >= p.min_p) st.floor_mass = w * st.floor_ties;
    }
    // below e^-48.6 a weight is nothing in a histogram's fixed point, below min_p it is not kept: with room for all roundings
    double reach = 48.6;
    if (p.min_p > 0.0) {
        reach = fmin(reach, -log(p.min_p) + 1e-9);
        st.gather = 3;
    }
    const double smax = S::value(st.top);
    const Key low = S::key_of(smax - reach * p.temperature * (1.0 + 1e-12) - fabs(smax) * 1e-14);
    if (smax < INFINITY && low > st.klo) st.klo = low > 4 ? low - 4 : low;
}

// A step's histogram over `from` into LDS.  The last bin of the linear step, where all that lies far from the best falls, is
// summed in registers: thousands of atomics on one address would take their turns.
template <typename T>
__device__ void draw_histogram(DrawLds<T>& s, const DrawStep<T>& d, const DrawFrom<T>& from) {
    using Key = typename Score<T>::Key;
    for (int b = threadIdx.x; b < BINS; b += DRAW_THREADS) s.h.count[b] = 0, s.h.hi[b] = 0, s.h.lo[b] = 0;
    __syncthreads();
    unsigned int rest = 0;
    unsigned long long rest_hi = 0, rest_lo = 0;
    from.each([&](Key k, uint32_t) {
        double w = 0.0;
        if (!d.counts(k, w)) return;
        const int b = d.bin(k);
        unsigned long long hi = 0, lo = 0;
        if (d.phase == PHASE_TOPP) to_fixed(w, hi, lo);
        if (d.linear && b == BINS - 1) {
            rest += 1, rest_hi += hi, rest_lo += lo;
        } else {
            atomicAdd(&s.h.count[b], 1u);
            if (hi) atomicAdd(&s.h.hi[b], hi);
            if (lo) atomicAdd(&s.h.lo[b], lo);
        }
    });
    if (d.linear) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            rest += __shfl_xor(rest, o);
            rest_hi += __shfl_xor(rest_hi, o);
            rest_lo += __shfl_xor(rest_lo, o);
        }
        if ((threadIdx.x & 63) == 0 && rest) {
            atomicAdd(&s.h.count[BINS - 1], rest);
            atomicAdd(&s.h.hi[BINS - 1], rest_hi);
            atomicAdd(&s.h.lo[BINS - 1], rest_lo);
        }
    }
    __syncthreads();
}

// The whole histogram of a step is in LDS: find the bin that holds the cut and move the state there.
template <typename T>
__device__ void draw_decide(DrawLds<T>& s, const DrawRow& p) {
    using S = Score<T>;
    using Key = typename S::Key;
    const int tid = threadIdx.x, b0 = 2 * tid, b1 = b0 + 1;      // bins from the top down
    DrawState<T>& st = s.st;
    const DrawStep<T> d(st, p);
    const bool first = st.first;
    if (tid == 0) s.bin = 0xffffffffu, s.any_bin = 0;
    const unsigned long long c0 = s.h.count[b0], c1 = s.h.count[b1];
    unsigned long long all_c;
    const unsigned long long run_c = block_scan(c0 + c1, s.red_u, all_c);      // up to and with this thread's bins
    bool spare = false;
    double m0 = 0.0, m1 = 0.0, run_m = 0.0, all_m = 0.0, goal = st.goal;
    const double above = st.above;
    const long long rank = st.rank;
    if (st.phase == PHASE_TOPK) {
        spare = first && all_c < (unsigned long long)rank;                     // fewer valid scores than top_k: no cut
        const long long before = (long long)(run_c - c0 - c1);
        if (c0 && before < rank && before + (long long)c0 >= rank) s.bin = b0;
        if (c1 && before + (long long)c0 < rank && before + (long long)(c0 + c1) >= rank) s.bin = b1;
    } else {
        m0 = from_fixed(s.h.hi[b0], s.h.lo[b0]), m1 = from_fixed(s.h.hi[b1], s.h.lo[b1]);
        run_m = block_scan(m0 + m1, s.red, all_m);
        if (first) goal = p.top_p * (all_m + st.floor_mass);
        spare = first && !(all_m >= goal);                                     // all above the group of the top-k cut is kept
        // the first bin with which the running mass reaches the goal; the last one in use if rounding leaves none
        // (one lane a wave asks: a thousand atomics on one address took 8 us)
        const bool reach0 = c0 && above + (run_m - m1) >= goal, reach1 = c1 && above + run_m >= goal;
        const unsigned long long reach = __ballot(reach0 || reach1), any = __ballot(c0 || c1);
        const int lane = tid & 63;
        if (reach && lane == __ffsll(reach) - 1) atomicMin(&s.bin, (unsigned)(reach0 ? b0 : b1));
        if (any && lane == 63 - __clzll((long long)any)) atomicMax(&s.any_bin, (unsigned)(c1 ? b1 : b0));
    }
    __syncthreads();
    const unsigned bin = s.bin != 0xffffffffu ? s.bin : s.any_bin;
    if (spare) {
        if (tid == 0) {
            if (st.phase == PHASE_TOPK) {
                st.cut = 0, st.cut_ties = 0;
                draw_begin(st, p, PHASE_TOPP);
            } else {                           // of the group, as many as the mass still asks for
                st.cut = st.floor_key;
                st.cut_ties = 0;
                if (st.floor_ties) {
                    const double w = exp(draw_t<T>(st.floor_key, st.top, p.temperature));
                    const double r = w > 0.0 ? ceil((goal - all_m) / w) : 0.0;
                    st.cut_ties = (uint32_t)fmin(fmax(r, 0.0), (double)st.floor_ties);
                }
                st.phase = PHASE_PICK;
            }
        }
    } else if (bin == (unsigned)b0 || bin == (unsigned)b1) {
        const bool low = bin == (unsigned)b1;
        const unsigned long long cnt = low ? c1 : c0, before_c = run_c - (low ? c1 : c0 + c1);
        Key lo, hi;
        d.ends((int)bin, lo, hi);
        st.klo = lo, st.khi = hi;
        st.first = 0, st.linear_left -= 1;
        st.count_above += (long long)before_c;
        if (st.phase == PHASE_TOPK) {
            st.rank = rank - (long long)before_c;
        } else {
            st.goal = goal;
            st.above = above + (low ? run_m - m1 : run_m - m1 - m0);
        }
        if (st.klo == st.khi) {                // one key: all of them ties
            st.cut = st.klo;
            if (st.phase == PHASE_TOPK) {
                st.cut_ties = (uint32_t)st.rank;
                draw_begin(st, p, PHASE_TOPP);
            } else {
                const double w = exp(draw_t<T>(st.cut, st.top, p.temperature));
                const double r = ceil((st.goal - st.above) / w);
                st.cut_ties = (uint32_t)fmin(r >= 1.0 ? r : 1.0, (double)cnt);
                st.phase = PHASE_PICK;
            }
        } else if (st.count_above + (long long)cnt <= LIST) {
            st.gather = 2;
        } else if (cnt <= LIST) {
            st.gather = 1;
        }
        st.n_list = 0;
    }
    __syncthreads();
}

// The value of lane `lane ^ X`, by vector instructions: an exchange through LDS hardware (__shfl_xor) takes several times as long.
template <int X>
__device__ __forceinline__ uint32_t xor_lane(uint32_t v) {
    if constexpr (X == 1) return __builtin_amdgcn_update_dpp(0, v, 0xb1, 0xf, 0xf, true);                     // quad_perm 1 0 3 2
    if constexpr (X == 2) return __builtin_amdgcn_update_dpp(0, v, 0x4e, 0xf, 0xf, true);                     // quad_perm 2 3 0 1
    if constexpr (X == 4) {                                                                                   // i ^ 7, then i ^ 3
        const uint32_t m = __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true);                          // row_half_mirror
        return __builtin_amdgcn_update_dpp(0, m, 0x1b, 0xf, 0xf, true);                                       // quad_perm 3 2 1 0
    }
    if constexpr (X == 8) return __builtin_amdgcn_update_dpp(0, v, 0x128, 0xf, 0xf, true);                    // row_ror 8
    if constexpr (X == 16) {                   // both results from v: rows 0 0 2 2 and 1 1 3 3
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return threadIdx.x & 16 ? r[0] : r[1];
    }
    if constexpr (X == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return threadIdx.x & 32 ? r[0] : r[1];
    }
}
template <int X>
__device__ __forceinline__ uint64_t xor_lane(uint64_t v) {
    return (uint64_t)xor_lane<X>((uint32_t)(v >> 32)) << 32 | xor_lane<X>((uint32_t)v);
}

// Bitonic sort of one pair a thread over the first `size` threads (a power of two, at least 64): by rank, or by index.  Partners
// in one wave exchange by vector instructions, others through LDS (buf_k, buf_i): 1024 pairs take 55 exchanges, 10 of them with
// barriers (a draw from 400 scores: 11.5 us, 14.3 with __shfl_xor; every pair counting the ones in front of it took 27 alone).
template <typename Key, bool BY_INDEX>
__device__ __forceinline__ void block_sort(Key& k, uint32_t& i, int size, Key* buf_k, uint32_t* buf_i) {
    const int tid = threadIdx.x;
    for (int run = 2; run <= size; run <<= 1) {
        const bool up = (tid & run) == 0 || run == size;
        auto exchange = [&](int step, Key ok, uint32_t oi) {
            const bool mine_first = BY_INDEX ? i < oi : (k > ok || (k == ok && i < oi));
            if (mine_first != (((tid & step) == 0) == up)) k = ok, i = oi;      // equal pairs are the fillers: either way the same
        };
        for (int step = run >> 1; step >= 64; step >>= 1) {
            __syncthreads();
            if (tid < size) buf_k[tid] = k, buf_i[tid] = i;
            __syncthreads();
            exchange(step, buf_k[tid ^ step], buf_i[tid ^ step]);
        }
        if (run >= 64) exchange(32, xor_lane<32>(k), xor_lane<32>(i));
        if (run >= 32) exchange(16, xor_lane<16>(k), xor_lane<16>(i));
        if (run >= 16) exchange(8, xor_lane<8>(k), xor_lane<8>(i));
        if (run >= 8) exchange(4, xor_lane<4>(k), xor_lane<4>(i));
        if (run >= 4) exchange(2, xor_lane<2>(k), xor_lane<2>(i));
        exchange(1, xor_lane<1>(k), xor_lane<1>(i));
    }
}

// LIST keys or fewer in l.key, l.idx: sort them by rank into l.key2, l.idx2 (behind them keys of 0).
template <typename T>
__device__ void draw_rank(DrawLds<T>& s, int n) {
    using Key = typename Score<T>::Key;
    const int tid = threadIdx.x;
    int size = 64;
    while (size < n) size <<= 1;
    __syncthreads();
    Key k = tid < n ? s.l.key[tid] : 0;
    uint32_t ix = tid < n ? s.l.idx[tid] : 0xffffffffu;
    block_sort<Key, false>(k, ix, size, s.l.key2, s.l.idx2);
    __syncthreads();
    if (tid < size) s.l.key2[tid] = k, s.l.idx2[tid] = ix;
    __syncthreads();
}

// The list holds the keys klo .. khi of a step: the cut is one of them.
template <typename T>
__device__ void draw_cut_from_list(DrawLds<T>& s, const DrawRow& p, int n) {
    using Key = typename Score<T>::Key;
    const int tid = threadIdx.x;
    DrawState<T>& st = s.st;
    draw_rank(s, n);
    const Key k = tid < n ? s.l.key2[tid] : 0;
    bool in;
    if (st.phase == PHASE_TOPK) {
        in = tid < st.rank;
    } else {
        const double w = k ? exp(draw_t<T>(k, st.top, p.temperature)) : 0.0;
        double all;
        const double incl = block_scan(w, s.red, all);
        in = k != 0 && (tid == 0 || st.above + (incl - w) < st.goal);
    }
    const int taken = block_leading(in, s.red_u);
    const Key cut = s.l.key2[taken ? taken - 1 : 0];
    unsigned long long same;
    block_scan(tid < taken && k == cut ? 1ull : 0ull, s.red_u, same);
    __syncthreads();
    if (tid == 0) {
        st.cut = cut, st.cut_ties = (uint32_t)same;
        if (st.phase == PHASE_TOPK) draw_begin(st, p, PHASE_TOPP);
        else st.phase = PHASE_PICK;
    }
    __syncthreads();
}

// Everything behind the list: n <= LIST pairs that hold every score that can be kept.  goal < 0: top_p of the mass that top-k and
// min-p leave; else the mass to reach.
template <typename T>
__device__ void draw_from_list(DrawLds<T>& s, const DrawArgs& a, const DrawRow& p, int64_t row, int n, typename Score<T>::Key top, double goal) {
    using Key = typename Score<T>::Key;
    const int tid = threadIdx.x;
    draw_rank(s, n);
    // by rank from here on: thread = position
    const Key kr = tid < n ? s.l.key2[tid] : 0;
    const double w = kr ? exp(draw_t<T>(kr, top, p.temperature)) : 0.0;
    bool keep = kr != 0 && (p.top_k == 0 || tid < p.top_k) && w >= p.min_p;
    double total;
    const double run = block_scan(keep ? w : 0.0, s.red, total);
    if (p.top_p < 1.0) {
        if (goal < 0.0) goal = p.top_p * total;
        keep = keep && (tid == 0 || run - w < goal);
    }
    // the kept ones are the first `kept` positions, also should an exponential not fall where its argument does; now in index order
    const int kept = block_leading(keep, s.red_u);
    Key ki = tid < kept ? kr : 0;
    uint32_t ii = tid < kept ? s.l.idx2[tid] : 0xffffffffu;
    int few = 64;                              // they stand in front: no more than they need to be sorted
    while (few < kept) few <<= 1;
    block_sort<Key, true>(ki, ii, few, s.l.key, s.l.idx);
    const double wi = tid < kept ? exp(draw_t<T>(ki, top, p.temperature)) : 0.0;
    const double ci = block_scan(wi, s.red, total);      // its barriers stand between the sort's last reads of l.key and this
    if (tid < kept) s.l.key[tid] = ki, s.l.pick[tid] = ii;
    if (tid < kept) s.l.c[tid] = ci;
    __syncthreads();
    for (int64_t q = tid; q < a.draws; q += DRAW_THREADS) {
        const double at = draw_goal(a.u[row * a.draws + q], total);
        int lo = 0, hi = kept - 1;        // the first c > at
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (s.l.c[mid] > at) hi = mid;
            else lo = mid + 1;
        }
        a.index[row * a.draws + q] = s.l.pick[lo];
        if (a.logp) a.logp[row * a.draws + q] = draw_t<T>(s.l.key[lo], top, p.temperature) - log(total);
    }
}

// One workgroup: the scores of `from` that count go to the list; behind LIST of them nothing is written and the counter
// stops growing soon.
template <typename T>
__device__ void draw_gather(DrawLds<T>& s, const DrawStep<T>& d, const DrawFrom<T>& from) {
    using Key = typename Score<T>::Key;
    auto take = [&](Key k, uint32_t i) {
        if (__hip_atomic_load(&s.st.n_list, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) > LIST) return;
        const uint32_t at = atomicAdd(&s.st.n_list, 1u);
        if (at < LIST) s.l.key[at] = k, s.l.idx[at] = i;
    };
    if (d.gather == 3) {                       // all from klo up: nothing to work out, more loads at a time
        const Key bound = d.klo ? d.klo : 1;
        from.template each<32>([&](Key k, uint32_t i) {
            if (k >= bound) take(k, i);
        });
    } else {
        from.each([&](Key k, uint32_t i) {
            double w;
            if (d.counts(k, w)) take(k, i);
        });
    }
    __syncthreads();
}

// A list of a step is in l: the picks (true), or the next step.
template <typename T>
__device__ bool draw_use_list(DrawLds<T>& s, const DrawArgs& a, const DrawRow& p, int64_t row) {
    const int gather = s.st.gather, m = min((int)s.st.n_list, LIST);
    const bool over = s.st.n_list > LIST;
    if (gather == 1) {
        draw_cut_from_list(s, p, m);
    } else if (gather == 3 && over) {          // the trial failed: on with histograms
        __syncthreads();
        if (threadIdx.x == 0) {
            s.st.gather = 0;
            s.st.n_list = 0;
            if (s.st.phase == PHASE_TOPP && !(p.top_p < 1.0)) s.st.phase = PHASE_PICK;
        }
        __syncthreads();
    } else {
        draw_from_list<T>(s, a, p, row, m, s.st.top, gather == 2 && s.st.phase == PHASE_TOPP ? s.st.goal : -1.0);
        return true;
    }
    return false;
}

// One workgroup takes all steps that are left; true if that included the picks.
template <typename T>
__device__ bool draw_search(DrawLds<T>& s, const DrawArgs& a, const DrawRow& p, const DrawFrom<T>& from, int64_t row) {
    while (s.st.phase < PHASE_PICK) {
        const DrawStep<T> d(s.st, p);
        if (s.st.gather) {
            draw_gather(s, d, from);
            if (draw_use_list(s, a, p, row)) return true;
        } else {
            draw_histogram(s, d, from);
            draw_decide(s, p);
        }
    }
    return false;
}

// Rows of up to LIST scores, a workgroup each, as many threads as scores or the next power of two, thread = index: one sort by rank
// gives the best and the last kept pair; whether a thread's own score is kept is then a comparison, and the running sum in index
// order needs no second sort (400 scores with 512 threads 8.9 us, with 1024 11.5; 10000 rows of 60 15 us, 164).
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void k_draw_short(DrawArgs a) {
    using Key = typename Score<T>::Key;
    __shared__ Key key_s[THREADS], top_s, cut_s;
    __shared__ uint32_t idx_s[THREADS], top_i, cut_i;
    __shared__ double c_s[THREADS], red[16];
    __shared__ unsigned long long red_u[16];
    const int tid = threadIdx.x, n = (int)a.cols;
    const int64_t row = blockIdx.x;
    const T* x = (const T*)a.scores + row * a.stride;
    const DrawRow p(a, row);
    const Key mine = tid < n ? Score<T>::key(x[tid]) : 0;
    Key k = mine;
    uint32_t i = tid;
    block_sort<Key, false>(k, i, THREADS, key_s, idx_s);
    if (tid == 0) top_s = k, top_i = i;
    __syncthreads();
    const Key top = top_s;
    if (top == 0 || p.greedy) {
        draw_same<T>(a, row, top ? (int64_t)top_i : -1, top ? 0.0 : -INFINITY);
        return;
    }
    const double w = k ? exp(draw_t<T>(k, top, p.temperature)) : 0.0;
    bool in = k != 0 && (p.top_k == 0 || tid < p.top_k) && w >= p.min_p;
    double total;
    if (p.top_p < 1.0) {
        const double run = block_scan<THREADS>(in ? w : 0.0, red, total);
        in = in && (tid == 0 || run - w < p.top_p * total);
    }
    // the kept ones are the first in rank, the best among them
    if (tid == block_leading<THREADS>(in, red_u) - 1) cut_s = k, cut_i = i;
    __syncthreads();
    const Key cut = cut_s;
    const bool keep = mine != 0 && (mine > cut || (mine == cut && (uint32_t)tid <= cut_i));
    const double c = block_scan<THREADS>(keep ? exp(draw_t<T>(mine, top, p.temperature)) : 0.0, red, total);
    c_s[tid] = c;
    key_s[tid] = mine;
    __syncthreads();
    for (int64_t q = tid; q < a.draws; q += THREADS) {
        const double at = draw_goal(a.u[row * a.draws + q], total);
        int lo = 0, hi = n - 1;                // the first c > at
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (c_s[mid] > at) hi = mid;
            else lo = mid + 1;
        }
        a.index[row * a.draws + q] = lo;
        if (a.logp) a.logp[row * a.draws + q] = draw_t<T>(key_s[lo], top, p.temperature) - log(total);
    }
}

// The weights of a row once the cut is known.
template <typename T>
struct DrawKept {
    using S = Score<T>;
    using Key = typename S::Key;
    Key top, cut;
    double temperature, min_p, tie_w;
    __device__ __forceinline__ DrawKept(const DrawState<T>& st, const DrawRow& p) : top(st.top), cut(st.cut), temperature(p.temperature), min_p(p.min_p) {
        const double w = cut ? exp(draw_t<T>(cut, top, temperature)) : 0.0;
        tie_w = w >= min_p ? w : 0.0;
    }
    __device__ __forceinline__ double strict(Key k) const {      // weight of a key above the cut
        if (k <= cut) return 0.0;              // (an invalid score's key is 0)
        const double w = exp(draw_t<T>(k, top, temperature));
        return w >= min_p ? w : 0.0;
    }
};

// One wave: mass above the cut, and ties with the cut, of elements [begin, end).
template <typename T>
__device__ void draw_tile_mass(const DrawKept<T>& kw, const T* x, uint32_t begin, uint32_t end, double& mass, uint32_t& ties) {
    using Key = typename Score<T>::Key;
    constexpr uint32_t V = Pack<T>::N;
    const uint32_t lane = threadIdx.x & 63;
    double m = 0.0;
    uint32_t c = 0;
    auto one = [&](T v) {
        const Key k = Score<T>::key(v);
        m += kw.strict(k);
        c += k == kw.cut && k != 0;
    };
    for (uint32_t i = begin + lane * V; i < end; i += 64 * V) {
        if (i + V <= end) {
            const Pack<T> p = load_pack(x + i);
#pragma unroll
            for (uint32_t j = 0; j < V; ++j) one(p.v[j]);
        } else {
            for (uint32_t j = i; j < end; ++j) one(x[j]);
        }
    }
    mass = wave_sum(m);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o);
    ties = c;
}

// One wave: the same for the neighbouring tiles of `tile` < 64 V elements (a power of two, at least 64) that 64 packs cover, from
// `begin` on: the lanes of a tile add up among themselves, and each of them has its tile's sums.
template <typename T>
__device__ void draw_tiles_mass(const DrawKept<T>& kw, const T* x, uint32_t begin, uint32_t end, uint32_t tile, double& mass, uint32_t& ties) {
    using Key = typename Score<T>::Key;
    constexpr uint32_t V = Pack<T>::N;
    double m = 0.0;
    uint32_t c = 0;
    auto one = [&](T v) {
        const Key k = Score<T>::key(v);
        m += kw.strict(k);
        c += k == kw.cut && k != 0;
    };
    const uint32_t i = begin + (threadIdx.x & 63) * V;
    if (i + V <= end) {
        const Pack<T> p = load_pack(x + i);
#pragma unroll
        for (uint32_t j = 0; j < V; ++j) one(p.v[j]);
    } else {
        for (uint32_t j = i; j < end; ++j) one(x[j]);
    }
    for (uint32_t o = tile / V / 2; o > 0; o >>= 1) {
        m += __shfl_xor(m, o);
        c += __shfl_xor(c, o);
    }
    mass = m, ties = c;
}

// One wave: the pick inside [begin, end), of at most 64 * 64 elements, for mass `goal` with `run` in front of it and `ties` of the
// cut's ties already met (of which cut_ties are kept).  A lane sums a run of neighbours, the lane that holds the goal is found
// by a scan over the lanes, and then its run is spread over the lanes.  Only lanes with a weight are asked: these sums and those over the
// tiles differ in their last bits, and where none passes the goal for that it is the last one.  The pick lies in the tile whatever the sums are.
template <typename T>
__device__ int64_t draw_in_tile(const DrawKept<T>& kw, const T* x, uint32_t begin, uint32_t end, double run, uint32_t ties, uint32_t cut_ties, double goal) {
    using Key = typename Score<T>::Key;
    constexpr uint32_t V = Pack<T>::N;
    const uint32_t lane = threadIdx.x & 63;
    uint32_t each = (end - begin + 63) / 64;
    for (int stage = 0; stage < 2; ++stage) {
        const uint32_t b = min(end, begin + lane * each), e = min(end, b + each);
        double m = 0.0;
        uint32_t c = 0;
        auto one = [&](T v) {
            const Key k = Score<T>::key(v);
            m += kw.strict(k);
            c += k == kw.cut && k != 0;
        };
        uint32_t i = b;
        for (; i + V <= e; i += V) {
            const Pack<T> p = load_pack(x + i);
#pragma unroll
            for (uint32_t j = 0; j < V; ++j) one(p.v[j]);
        }
        for (; i < e; ++i) one(x[i]);
        uint32_t before = c;                   // ties in front of this lane
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t v = __shfl_up(before, o);
            if (lane >= (uint32_t)o) before += v;
        }
        before += ties - c;
        const uint32_t kept = before >= cut_ties ? 0 : min(c, cut_ties - before);
        m += kept * kw.tie_w;
        double incl = m;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double v = __shfl_up(incl, o);
            if (lane >= (uint32_t)o) incl += v;
        }
        const unsigned long long any = __ballot(m > 0.0), hit = __ballot(m > 0.0 && run + incl > goal);
        const int at = hit ? __ffsll(hit) - 1 : 63 - __clzll((long long)(any | 1));
        run += __shfl(incl - m, at);
        ties = __shfl(before, at);
        begin = min(end - 1, begin + at * each);
        end = min(end, begin + each);
        if (each == 1) break;
        each = 1;
    }
    return begin;
}

constexpr uint32_t TILE = 4096;

// One workgroup a row (up to TILES tiles long).
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
    Key top, bot, own;
    uint32_t idx;
    draw_extremes(s, x, 0, n, top, bot, idx, own);
    if (top == 0 || p.greedy) {
        draw_same<T>(a, row, top ? (int64_t)idx : -1, top ? 0.0 : -INFINITY);
        return;
    }
    // A lower bound of the top_k-th score: the top_k-th of the maxima of groups of threads, sorted.  A quarter more groups than
    // top_k keep the list behind the bound short (some n log n of them, at most), and few of them are sooner sorted: 64 without leaving
    // a wave (256 x 65537 scores of 16 bits, top_k 50: 40 us with all 1024, 38.5 with 64).
    Key bound = 0;
    if (p.top_k > 0 && p.top_k <= DRAW_THREADS) {
        const int groups = p.top_k * 5 <= 64 * 4 ? 64 : p.top_k * 5 <= 256 * 4 ? 256 : DRAW_THREADS, each = DRAW_THREADS / groups;
        for (int o = each / 2; o > 0; o >>= 1) {
            const Key k = __shfl_xor(own, o);
            if (k > own) own = k;
        }
        if (tid % each == 0) s.l.key[tid / each] = own;
        __syncthreads();
        own = tid < groups ? s.l.key[tid] : 0;
        uint32_t none = tid;
        block_sort<Key, false>(own, none, groups, s.l.key2, s.l.idx2);
        if (tid == (int)p.top_k - 1) s.red_k[0][0] = own;
        __syncthreads();
        bound = s.red_k[0][0];
    }
    if (tid == 0) {
        s.st.top = top, s.st.bot = bot, s.st.cut = 0, s.st.cut_ties = 0;
        draw_begin(s.st, p, PHASE_TOPK, bound);
    }
    __syncthreads();
    if (draw_search(s, a, p, DrawFrom<T>{x, 0, n}, row)) return;

    // kept mass of the row's tiles, in index order
    const DrawKept<T> kw(s.st, p);
    constexpr uint32_t V = Pack<T>::N;
    uint32_t tile = 64;                        // as short as TILES of them allow: a pick looks through one
    while ((uint64_t)tile * TILES < n) tile <<= 1;
    const uint32_t tiles = (n + tile - 1) / tile;
    s.t.c[tid] = 0.0, s.t.ties[tid] = 0;
    __syncthreads();
    if (tile < 64 * V) {
        const uint32_t lanes = tile / V, at_once = 64 / lanes;
        for (uint32_t t = wave * at_once; t < tiles; t += DRAW_THREADS / 64 * at_once) {
            double m;
            uint32_t c;
            draw_tiles_mass(kw, x, t * tile, n, tile, m, c);
            if (lane % lanes == 0 && t + lane / lanes < tiles) s.t.c[t + lane / lanes] = m, s.t.ties[t + lane / lanes] = c;
        }
    } else {
        for (uint32_t t = wave; t < tiles; t += DRAW_THREADS / 64) {
            double m;
            uint32_t c;
            draw_tile_mass(kw, x, t * tile, min(n, (t + 1) * tile), m, c);
            if (lane == 0) s.t.c[t] = m, s.t.ties[t] = c;
        }
    }
    __syncthreads();
    const uint32_t mine = s.t.ties[tid];
    unsigned long long all_ties;
    const uint32_t before = (uint32_t)(block_scan((unsigned long long)mine, s.red_u, all_ties) - mine);
    const uint32_t cut_ties = s.st.cut_ties;
    const uint32_t kept = before >= cut_ties ? 0 : min(mine, cut_ties - before);
    double total;
    const double incl = block_scan(s.t.c[tid] + kept * kw.tie_w, s.red, total);
    s.t.c[tid] = incl, s.t.ties[tid] = before;
    __syncthreads();
    for (int64_t q = wave; q < a.draws; q += DRAW_THREADS / 64) {
        const double goal = draw_goal(a.u[row * a.draws + q], total);
        int lo = 0, hi = (int)tiles - 1;       // the first tile whose sum passes the goal
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (s.t.c[mid] > goal) hi = mid;
            else lo = mid + 1;
        }
        const int64_t pick = draw_in_tile(kw, x, lo * tile, min(n, (lo + 1) * tile), lo ? s.t.c[lo - 1] : 0.0, s.t.ties[lo], cut_ties, goal);
        if (lane == 0) {
            a.index[row * a.draws + q] = pick;
            if (a.logp) a.logp[row * a.draws + q] = draw_t<T>(S::key(x[pick]), top, p.temperature) - log(total);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Long rows: up to SHARES workgroups a row and step (one a CU: a step with nothing to do costs less, 16.8 M scores take 116 us and 124
// with two).  Workspace of a row: its state, one histogram, the list, the extremes of every workgroup's share, and mass and ties
// of every tile.
constexpr int SHARES = 256;
template <typename T>
struct DrawWork {
    using Key = typename Score<T>::Key;
    DrawState<T> st;
    unsigned int count[BINS];
    unsigned long long hi[BINS], lo[BINS];
    Key key[LONG_LIST];
    uint32_t idx[LONG_LIST];
    Key top[SHARES], bot[SHARES], quarter[4 * SHARES];
    uint32_t top_idx[SHARES];
    double total;
};
template <typename T>
__host__ __device__ constexpr int64_t draw_row_bytes(int64_t cols) {
    return round_up((int64_t)sizeof(DrawWork<T>), 256) + round_up(ceil_div(cols, TILE) * 8, 256) + round_up(ceil_div(cols, TILE) * 4, 256);
}
template <typename T>
struct DrawRowWork {
    DrawWork<T>* w;
    double* c;
    uint32_t* ties;
    __device__ __forceinline__ DrawRowWork(char* work, int64_t row, int64_t cols) {
        char* at = work + row * draw_row_bytes<T>(cols);
        w = (DrawWork<T>*)at;
        c = (double*)(at + round_up((int64_t)sizeof(DrawWork<T>), 256));
        ties = (uint32_t*)((char*)c + round_up(ceil_div(cols, TILE) * 8, 256));
    }
};

// The share of workgroup b of `blocks` of a row of n elements: whole packs.
__device__ __forceinline__ void draw_share(uint32_t n, uint32_t b, uint32_t blocks, uint32_t& begin, uint32_t& end) {
    const uint32_t each = (uint32_t)round_up(ceil_div(n, blocks), 16);
    begin = min(n, b * each);
    end = min(n, begin + each);
}

// True in the workgroup that arrives last of the `blocks` of its row; what the others wrote before is then visible to it.  One
// thread fences for its workgroup, behind the barrier that orders the other threads' writes before it: a fence writes the L2
// back, and one of every wave cost 8 times the step itself.  The counter is back at zero for the next step.
__device__ __forceinline__ bool draw_last(unsigned int& last, unsigned int* ticket, uint32_t blocks) {
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        const unsigned int t = atomicAdd(ticket, 1u);
        last = t == blocks - 1;
        if (last) {
            __threadfence();
            *ticket = 0;
        }
    }
    __syncthreads();
    return last;
}

// Extremes of every share, a clean histogram and counters.
template <typename T>
__global__ __launch_bounds__(DRAW_THREADS) void k_draw_start(DrawArgs a, char* work) {
    using Key = typename Score<T>::Key;
    __shared__ DrawLds<T> s;
    const int64_t row = blockIdx.y;
    const DrawRowWork<T> rw(work, row, a.cols);
    const T* x = (const T*)a.scores + row * a.stride;
    uint32_t begin, end;
    draw_share((uint32_t)a.cols, blockIdx.x, gridDim.x, begin, end);
    Key top, bot, own;
    uint32_t idx;
    draw_extremes(s, x, begin, end, top, bot, idx, own);
    if (threadIdx.x == 0) rw.w->top[blockIdx.x] = top, rw.w->bot[blockIdx.x] = bot, rw.w->top_idx[blockIdx.x] = idx;
    if (threadIdx.x < 4) {                     // (the waves' best keys are still there)
        Key k = 0;
        for (int i = 0; i < DRAW_THREADS / 256; ++i) k = max(k, s.red_k[0][threadIdx.x * (DRAW_THREADS / 256) + i]);
        rw.w->quarter[blockIdx.x * 4 + threadIdx.x] = k;
    }
    if (blockIdx.x == 0) {
        for (int b = threadIdx.x; b < BINS; b += DRAW_THREADS) rw.w->count[b] = 0, rw.w->hi[b] = 0, rw.w->lo[b] = 0;
        if (threadIdx.x == 0) rw.w->st.ticket = 0;
    }
}

// Joins the extremes; the first step, or the result where there is nothing to choose.  One workgroup a row.
template <typename T>
__global__ __launch_bounds__(DRAW_THREADS) void k_draw_begin(DrawArgs a, char* work, int shares) {
    using Key = typename Score<T>::Key;
    __shared__ Key rk[2][16], sort_k[LIST], bound_s;
    __shared__ uint32_t ri[16], sort_i[LIST];
    const int64_t row = blockIdx.x;
    const DrawRowWork<T> rw(work, row, a.cols);
    const DrawRow p(a, row);
    const int tid = threadIdx.x;
    Key bk = tid < shares ? rw.w->top[tid] : 0, lk = tid < shares ? rw.w->bot[tid] : ~(Key)0;
    uint32_t bi = tid < shares ? rw.w->top_idx[tid] : 0;
    Key bound = 0;
    if (p.top_k > 0 && p.top_k <= 4 * shares) {      // the maxima of shares, or quarters of them, sorted: top_k of them reach the top_k-th
        const bool fine = p.top_k > shares;
        Key own = fine ? (tid < 4 * shares ? rw.w->quarter[tid] : 0) : bk;
        uint32_t none = tid;
        block_sort<Key, false>(own, none, fine ? DRAW_THREADS : SHARES, sort_k, sort_i);
        if (tid == (int)p.top_k - 1) bound_s = own;
        __syncthreads();
        bound = bound_s;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const Key k = __shfl_xor(bk, o), l = __shfl_xor(lk, o);
        const uint32_t i = __shfl_xor(bi, o);
        if (k > bk || (k == bk && i < bi)) bk = k, bi = i;
        if (l < lk) lk = l;
    }
    if ((tid & 63) == 0) rk[0][tid >> 6] = bk, rk[1][tid >> 6] = lk, ri[tid >> 6] = bi;
    __syncthreads();
    for (int i = 0; i < DRAW_THREADS / 64; ++i) {
        if (rk[0][i] > bk || (rk[0][i] == bk && ri[i] < bi)) bk = rk[0][i], bi = ri[i];
        if (rk[1][i] < lk) lk = rk[1][i];
    }
    if (bk == 0 || p.greedy) draw_same<T>(a, row, bk ? (int64_t)bi : -1, bk ? 0.0 : -INFINITY);
    if (tid == 0) {
        DrawState<T>& st = rw.w->st;
        st.top = bk, st.bot = lk, st.cut = 0, st.cut_ties = 0, st.n_list = 0, st.listed = 0;
        if (bk == 0 || p.greedy) st.phase = PHASE_DONE;
        else draw_begin(st, p, PHASE_TOPK, bound, DRAW_THREADS);
    }
}

// A step over all shares; the last workgroup to arrive decides.  A list on trial may hold up to LONG_LIST scores: the steps that then
// remain need no others, and are left to k_draw_rest.
template <typename T>
__global__ __launch_bounds__(DRAW_THREADS) void k_draw_step(DrawArgs a, char* work) {
    using Key = typename Score<T>::Key;
    __shared__ DrawLds<T> s;
    const int64_t row = blockIdx.y;
    const DrawRowWork<T> rw(work, row, a.cols);
    if (rw.w->st.phase >= PHASE_PICK || rw.w->st.listed) return;
    const int tid = threadIdx.x;
    const T* x = (const T*)a.scores + row * a.stride;
    const DrawRow p(a, row);
    const DrawStep<T> d(rw.w->st, p);
    const bool gather = rw.w->st.gather;
    uint32_t begin, end;
    draw_share((uint32_t)a.cols, blockIdx.x, gridDim.x, begin, end);
    if (gather) {                              // a list of the share's own, then one place in the row's
        if (tid == 0) s.st.n_list = 0;
        __syncthreads();
        draw_gather(s, d, DrawFrom<T>{x, begin, end});
        if (tid == 0 && s.st.n_list) s.bin = atomicAdd(&rw.w->st.n_list, s.st.n_list > LIST ? LONG_LIST + 1 : s.st.n_list);
        __syncthreads();
        const uint32_t mine = s.st.n_list, at = mine ? s.bin + tid : LONG_LIST;
        if (mine <= LIST && tid < (int)mine && at < LONG_LIST) rw.w->key[at] = s.l.key[tid], rw.w->idx[at] = s.l.idx[tid];
    } else {
        draw_histogram(s, d, DrawFrom<T>{x, begin, end});
        for (int b = tid; b < BINS; b += DRAW_THREADS)
            if (s.h.count[b]) {
                atomicAdd(&rw.w->count[b], s.h.count[b]);
                if (s.h.hi[b]) atomicAdd(&rw.w->hi[b], s.h.hi[b]);
                if (s.h.lo[b]) atomicAdd(&rw.w->lo[b], s.h.lo[b]);
            }
    }
    if (!draw_last(s.last, &rw.w->st.ticket, gridDim.x)) return;
    // what other workgroups left is read past this one's caches
    auto fresh32 = [](unsigned int* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    if (tid == 0) {
        s.st = rw.w->st;
        s.st.n_list = fresh32(&rw.w->st.n_list);
        s.st.ticket = 0;
    }
    __syncthreads();
    if (!gather) {
        for (int b = tid; b < BINS; b += DRAW_THREADS) {
            s.h.count[b] = fresh32(&rw.w->count[b]);
            s.h.hi[b] = __hip_atomic_load(&rw.w->hi[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            s.h.lo[b] = __hip_atomic_load(&rw.w->lo[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            rw.w->count[b] = 0, rw.w->hi[b] = 0, rw.w->lo[b] = 0;
        }
        __syncthreads();
        draw_decide(s, p);
    } else {
        if (s.st.n_list <= LIST && tid < (int)s.st.n_list) {
            s.l.key[tid] = __hip_atomic_load(&rw.w->key[tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            s.l.idx[tid] = fresh32(&rw.w->idx[tid]);
        }
        const unsigned int n = s.st.n_list;
        const bool trial = s.st.gather == 3;
        __syncthreads();
        const bool done = draw_use_list(s, a, p, row);
        __syncthreads();
        if (tid == 0) {
            if (done) s.st.phase = PHASE_DONE;
            else if (trial && n <= LONG_LIST) s.st.listed = n;
            s.st.n_list = 0;
        }
    }
    __syncthreads();
    if (tid == 0) rw.w->st = s.st;
}

// What the launched steps left over, one workgroup a row: the steps over a long list (16.8 M scores of which 1800 pass min_p: two passes
// over the row less, 138 -> 124 us), or, if scores are spread so badly that there are any, further ones over the row.
template <typename T>
__global__ __launch_bounds__(DRAW_THREADS) void k_draw_rest(DrawArgs a, char* work) {
    __shared__ DrawLds<T> s;
    const int64_t row = blockIdx.x;
    const DrawRowWork<T> rw(work, row, a.cols);
    if (rw.w->st.phase >= PHASE_PICK) return;
    const DrawRow p(a, row);
    if (threadIdx.x == 0) s.st = rw.w->st;
    __syncthreads();
    const bool done = draw_search(s, a, p, DrawFrom<T>{(const T*)a.scores + row * a.stride, 0, (uint32_t)a.cols, rw.w->key, rw.w->idx, s.st.listed}, row);
    __syncthreads();
    if (threadIdx.x == 0) {
        if (done) s.st.phase = PHASE_DONE;
        rw.w->st = s.st;
    }
}

// Mass above the cut and ties of every tile, a wave each; the last workgroup to arrive turns them into running sums, 1024 tiles at a
// time.
template <typename T>
__global__ __launch_bounds__(DRAW_THREADS) void k_draw_mass(DrawArgs a, char* work) {
    __shared__ double red[32];
    __shared__ unsigned long long red_u[32];
    __shared__ unsigned int last;
    const int64_t row = blockIdx.y;
    const DrawRowWork<T> rw(work, row, a.cols);
    if (rw.w->st.phase != PHASE_PICK) return;
    const DrawRow p(a, row);
    const DrawKept<T> kw(rw.w->st, p);
    const T* x = (const T*)a.scores + row * a.stride;
    const uint32_t n = (uint32_t)a.cols, tiles = (n + TILE - 1) / TILE;
    for (uint32_t t = blockIdx.x * (DRAW_THREADS / 64) + (threadIdx.x >> 6); t < tiles; t += gridDim.x * (DRAW_THREADS / 64)) {
        double m;
        uint32_t c;
        draw_tile_mass(kw, x, t * TILE, min(n, (t + 1) * TILE), m, c);
        if ((threadIdx.x & 63) == 0) rw.c[t] = m, rw.ties[t] = c;
    }
    if (!draw_last(last, &rw.w->st.ticket, gridDim.x)) return;
    const uint32_t cut_ties = rw.w->st.cut_ties;
    double carry = 0.0;
    unsigned long long carry_t = 0;
    for (uint32_t t0 = 0; t0 < tiles; t0 += DRAW_THREADS) {
        const uint32_t t = t0 + threadIdx.x;
        const uint32_t mine = t < tiles ? __hip_atomic_load(rw.ties + t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
        const double mass = t < tiles ? __hip_atomic_load(rw.c + t, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
        unsigned long long all_t;
        const unsigned long long before = carry_t + block_scan((unsigned long long)mine, red_u, all_t) - mine;
        const uint32_t kept = before >= cut_ties ? 0 : (uint32_t)min((unsigned long long)mine, cut_ties - before);
        double all;
        const double incl = block_scan(mass + kept * kw.tie_w, red, all);
        if (t < tiles) rw.c[t] = carry + incl, rw.ties[t] = (uint32_t)before;
        carry += all;
        carry_t += all_t;
    }
    if (threadIdx.x == 0) rw.w->total = carry;
}

// A wave a draw.
template <typename T>
__global__ __launch_bounds__(256) void k_draw_pick(DrawArgs a, char* work) {
    const int64_t row = blockIdx.y;
    const DrawRowWork<T> rw(work, row, a.cols);
    if (rw.w->st.phase != PHASE_PICK) return;
    const DrawRow p(a, row);
    const DrawKept<T> kw(rw.w->st, p);
    const T* x = (const T*)a.scores + row * a.stride;
    const uint32_t n = (uint32_t)a.cols, tiles = (n + TILE - 1) / TILE;
    const double total = rw.w->total;
    for (int64_t q = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); q < a.draws; q += (int64_t)gridDim.x * 4) {
        const double goal = draw_goal(a.u[row * a.draws + q], total);
        int lo = 0, hi = (int)tiles - 1;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (rw.c[mid] > goal) hi = mid;
            else lo = mid + 1;
        }
        const int64_t pick = draw_in_tile(kw, x, (uint32_t)lo * TILE, min(n, (uint32_t)(lo + 1) * TILE), lo ? rw.c[lo - 1] : 0.0, rw.ties[lo],
                                          rw.w->st.cut_ties, goal);
        if ((threadIdx.x & 63) == 0) {
            a.index[row * a.draws + q] = pick;
            if (a.logp) a.logp[row * a.draws + q] = draw_t<T>(Score<T>::key(x[pick]), kw.top, p.temperature) - log(total);
        }
    }
}

// One workgroup a row while the rows fill the card or a row is short; else many workgroups a row.
constexpr int64_t MOST_LONG_ROWS = 65535;      // a grid's second dimension (more of them would not fit into the card's memory)
inline bool draw_long(int64_t rows, int64_t cols) { return cols > (int64_t)TILE * TILES || (cols > 32768 && rows * 4 < 256 * 2); }

template <typename T>
int64_t draw_work_bytes(int64_t rows, int64_t cols) {
    return draw_long(rows, cols) ? rows * draw_row_bytes<T>(cols) : 0;
}

template <typename T>
hipError_t draw_rows(hipStream_t st, const DrawArgs& a, char* work) {
    // one workgroup a row; a launch takes fewer than 2^32 threads, so that many rows go in pieces
    auto launch = [&](auto k, int threads) {
        const int64_t most = ((int64_t)1 << 31) / threads;
        for (int64_t r = 0; r < a.rows; r += most) {
            DrawArgs p = a;
            p.rows = std::min(most, a.rows - r);
            p.scores = (const T*)a.scores + r * a.stride, p.u = a.u + r * a.draws, p.index = a.index + r * a.draws;
            if (a.params) p.params = a.params + r * 4;
            if (a.logp) p.logp = a.logp + r * a.draws;
            hipLaunchKernelGGL(k, dim3((unsigned)p.rows), dim3(threads), 0, st, p);
        }
    };
    if (a.cols <= LIST) {
        if (a.cols <= 64) launch(k_draw_short<T, 64>, 64);
        else if (a.cols <= 128) launch(k_draw_short<T, 128>, 128);
        else if (a.cols <= 256) launch(k_draw_short<T, 256>, 256);
        else if (a.cols <= 512) launch(k_draw_short<T, 512>, 512);
        else launch(k_draw_short<T, 1024>, 1024);
        return hipGetLastError();
    }
    if (!draw_long(a.rows, a.cols)) {
        launch(k_draw_row<T>, DRAW_THREADS);
        return hipGetLastError();
    }
    // a workgroup of 1024 threads a CU over all rows, shares of at least 16 K
    const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>(ceil_div(SHARES, a.rows), ceil_div(a.cols, 16384)));
    const dim3 wide((unsigned)blocks, (unsigned)a.rows), one((unsigned)a.rows);
    hipLaunchKernelGGL(k_draw_start<T>, wide, dim3(DRAW_THREADS), 0, st, a, work);
    hipLaunchKernelGGL(k_draw_begin<T>, one, dim3(DRAW_THREADS), 0, st, a, work, (int)blocks);
    // a phase rarely takes more than a list on trial, two linear steps, one on the keys and one more list; what is decided
    // earlier leaves the rest of the launches with nothing to do, what is not is left to one workgroup a row
    const bool by_row = a.params != nullptr;
    const int phases = (by_row || (a.top_k > 0 && a.top_k < a.cols)) + (by_row || a.top_p < 1.0 || a.min_p > 0.0);
    const int steps = phases == 0 ? 0 : a.top_p < 1.0 || phases == 2 || by_row ? 1 + 4 * phases : 4;
    for (int i = 0; i < steps; ++i) hipLaunchKernelGGL(k_draw_step<T>, wide, dim3(DRAW_THREADS), 0, st, a, work);
    if (phases) hipLaunchKernelGGL(k_draw_rest<T>, one, dim3(DRAW_THREADS), 0, st, a, work);
    const int64_t tiles = ceil_div(a.cols, TILE);
    hipLaunchKernelGGL(k_draw_mass<T>, dim3((unsigned)std::min<int64_t>(ceil_div(tiles, DRAW_THREADS / 64), blocks), (unsigned)a.rows), dim3(DRAW_THREADS), 0,
                       st, a, work);
    hipLaunchKernelGGL(k_draw_pick<T>, dim3((unsigned)std::min<int64_t>(ceil_div(a.draws, 4), 4096), (unsigned)a.rows), dim3(256), 0, st, a, work);
    return hipGetLastError();
}

}  // namespace gpbo_static
