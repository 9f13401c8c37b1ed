// gate.hip -- a learned gate over the cells: which k cells a row goes to and with what weights, the gradient of the weights, and the
// rows of every cell in one stable order.  (mnr_route is the geometric router: distances to centroids instead of scores.)
//
//   s_e = softmax_e(x) or sigmoid(x_e) over the open cells (mask set, logit > -inf);   v_e = s_e + bias_e (x_e where there is no bias)
//   groups of n / n_groups cells: the k_groups groups with the largest sum of their group_top best (s + bias) stay open
//   chosen: the k largest v of what is open, largest first, the lowest index of equals;  w_j = scale s_j [ / sum_chosen s ]
//   gradient (cells fixed), g = scale dw:    softmax, renormalised: dx_j = p_j (g_j - sum p g) over the chosen, p = w / scale
//       softmax: dx_e = s_e (g_e [e chosen] - sum_chosen s g);   sigmoid: dx_j = s_j (1 - s_j) g_j, renormalised p_j (1 - s_j) (g_j - sum p g)
//
// Bound by HBM for few cells (a row is read once), by the instructions of the arg-max rounds for many.  A lane holds neighbouring cells in
// registers, up to 32 where the logits decide and in the gradient (a thread is a row of up to 32 cells, 256 cells are 8 lanes), up to 16
// where scores do (256 cells are 16 lanes): a round is a local maximum, a DPP maximum over the lanes and a ballot that names the lowest
// lane that has it.  (With 4 cells a lane and 8 lanes a row every instruction served 8 rows instead of 64: 25 cells took 20 us; 8 cells
// and 32 lanes: 256 cells 122 us.)  25 cells, 196608 rows: 16 us forward, 16.5 us backward.
// Where no score enters a comparison the values are the logits themselves (exact).  Otherwise the scores are formed in fp32 and every
// decision is checked: a row where two values that a decision kept apart are closer than fp32's error is decided again in 64 bits, so the
// choice is the one of the definition (all rows in 64 bits: 65536 rows of 256 bf16 cells in 8 groups took 266 us; checked, 86 to 93).
// Such rows go one after the other through their wave, and equal scores are among them although the lowest index already decides there:
// the same 65536 rows take 243 us with a bias of zeros (16-bit logits tie in about a third of them) and 395 us where all logits are equal too,
// 196608 rows of 8 fp32 cells 9.4, 9.6 and 115 us, of 25 bf16 cells 20.6, 26.6 and 121 us.
// Weights are formed from the logits of the chosen (log-sigmoids for sigmoid), so renormalising never divides by an underflowed sum.
#include <type_traits>

#include "row_sort.h"

namespace mnr {

template <int STEP> __device__ __forceinline__ double other_of(double x) {
    const uint64_t b = (uint64_t)__double_as_longlong(x);
    return __longlong_as_double((long long)(((uint64_t)lane_other<STEP>((uint32_t)(b >> 32)) << 32) | lane_other<STEP>((uint32_t)b)));
}
template <int STEP> __device__ __forceinline__ int other_of(int x) { return (int)lane_other<STEP>((uint32_t)x); }
template <int STEP> __device__ __forceinline__ void halves_of(int x, int &a, int &b) {
    uint32_t p, q;
    lane_halves<STEP>((uint32_t)x, p, q);
    a = (int)p; b = (int)q;
}
template <int STEP> __device__ __forceinline__ void halves_of(double x, double &a, double &b) {
    const uint64_t v = (uint64_t)__double_as_longlong(x);
    uint32_t pl, ql, ph, qh;
    lane_halves<STEP>((uint32_t)v, pl, ql);
    lane_halves<STEP>((uint32_t)(v >> 32), ph, qh);
    a = __longlong_as_double((long long)(((uint64_t)ph << 32) | pl));
    b = __longlong_as_double((long long)(((uint64_t)qh << 32) | ql));
}
// fp32 values are compared as whole numbers of the same order (one instruction for a maximum of three, and no care for NaNs; -0 counts as
// 0).  none<V>() is what -inf becomes.
__device__ __forceinline__ int key_of(float x) {
    const int b = __float_as_int(x + 0.f);
    return b ^ (b >> 31 & 0x7fffffff);
}
__device__ __forceinline__ float value_of(int k) { return __int_as_float(k ^ (k >> 31 & 0x7fffffff)); }
__device__ __forceinline__ double value_of(double v) { return v; }
__device__ __forceinline__ int max_of(int a, int b) { return max(a, b); }
__device__ __forceinline__ int min_of(int a, int b) { return min(a, b); }
__device__ __forceinline__ double max_of(double a, double b) { return b > a ? b : a; }
__device__ __forceinline__ double min_of(double a, double b) { return b < a ? b : a; }
template <class V> __device__ __forceinline__ V none_of();
template <> __device__ __forceinline__ int none_of<int>() { return (int)0x807fffff; }
template <> __device__ __forceinline__ double none_of<double>() { return -__builtin_huge_val(); }

template <int LANES> __device__ __forceinline__ double lane_sum64(double x) {
    auto add = [&](auto step) {
        constexpr int S = step;
        if constexpr (S >= 16) {
            double a, b;
            halves_of<S>(x, a, b);
            x = a + b;
        } else {
            x += other_of<S>(x);
        }
    };
    if constexpr (LANES >= 2) add(std::integral_constant<int, 1>{});
    if constexpr (LANES >= 4) add(std::integral_constant<int, 2>{});
    if constexpr (LANES >= 8) add(std::integral_constant<int, 4>{});
    if constexpr (LANES >= 16) add(std::integral_constant<int, 8>{});
    if constexpr (LANES >= 32) add(std::integral_constant<int, 16>{});
    if constexpr (LANES >= 64) add(std::integral_constant<int, 32>{});
    return x;
}

struct GateArgs {
    const void *logits;  int64_t ldl;
    const float *bias;                   // [n] or NULL
    const uint8_t *mask;  int64_t ldm;   // NULL: all open; ldm 0: one row for all
    int64_t rows;
    int n, k, sigmoid, n_groups, k_groups, group_top, renormalise;
    float scale;
};

constexpr int GATE_MAX_K = 32;
constexpr float GATE_NONE = -__builtin_huge_valf();

__device__ __forceinline__ float log_sigmoid(float x) { return fminf(x, 0.f) - log1pf(expf(-fabsf(x))); }

// this lane's cells e0 .. of a row: the logits of the open ones, GATE_NONE elsewhere
template <class T, int EPL>
__device__ __forceinline__ void gate_load(float (&x)[EPL], const GateArgs &a, const T *row, int64_t r, int e0, bool live) {
    constexpr int N = EPL < Vec<T>::N ? EPL : Vec<T>::N;
    typedef T part __attribute__((ext_vector_type(N)));
    typedef part part_at __attribute__((aligned(sizeof(T))));
    typedef uint8_t bytes __attribute__((ext_vector_type(N)));
    typedef bytes bytes_at __attribute__((aligned(1)));
    const int left = live ? a.n - e0 : 0;
    const uint8_t *open = a.mask + r * a.ldm + e0;
#pragma unroll
    for (int j = 0; j < EPL; j += N) {
        if (left >= j + N) {
            const part v = *reinterpret_cast<const part_at *>(row + e0 + j);
#pragma unroll
            for (int i = 0; i < N; ++i) x[j + i] = (float)v[i];
            if (a.mask) {
                const bytes m = *reinterpret_cast<const bytes_at *>(open + j);
#pragma unroll
                for (int i = 0; i < N; ++i) x[j + i] = m[i] ? x[j + i] : GATE_NONE;
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                x[j + i] = GATE_NONE;
                if (j + i < left && !(a.mask && !open[j + i])) x[j + i] = (float)row[e0 + j + i];
            }
        }
    }
}

// the ballot of this lane's group, its lowest lane in bit 0
template <int LPR> __device__ __forceinline__ uint64_t group_ballot(bool b) {
    if constexpr (LPR == 1) return b;
    const uint64_t m = __ballot(b);
    if constexpr (LPR == 64) return m;
    return (m >> ((threadIdx.x & 63) / LPR * LPR)) & ((1ull << LPR) - 1);
}
template <int STEP, class V> __device__ __forceinline__ V max_step(V x) {
    if constexpr (STEP >= 16) {
        V a, b;
        halves_of<STEP>(x, a, b);
        return max_of(a, b);
    } else {
        return max_of(x, other_of<STEP>(x));
    }
}
template <int LPR, class V> __device__ __forceinline__ V group_max(V x) {
    if constexpr (LPR >= 2) x = max_step<1>(x);
    if constexpr (LPR >= 4) x = max_step<2>(x);
    if constexpr (LPR >= 8) x = max_step<4>(x);
    if constexpr (LPR >= 16) x = max_step<8>(x);
    if constexpr (LPR >= 32) x = max_step<16>(x);
    if constexpr (LPR >= 64) x = max_step<32>(x);
    return x;
}

// Takes the largest of the group's values out of v: its value, and on the lane that had it `mine` = its number there, else -1
template <int LPR, int EPL, class V> __device__ __forceinline__ V take_best(V (&v)[EPL], int &mine) {
    const V none = none_of<V>();
    V high = v[0];
#pragma unroll
    for (int j = 1; j < EPL; ++j) high = max_of(high, v[j]);
    const V best = group_max<LPR>(high);
    bool own = best > none;
    if constexpr (LPR > 1) {
        const uint64_t who = group_ballot<LPR>(high == best);
        own = own && (int)(threadIdx.x % LPR) == __ffsll((unsigned long long)who) - 1;
    }
    mine = -1;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
        const bool hit = own && v[j] == best;
        v[j] = hit ? none : v[j];
        mine = hit ? j : mine;
        own = own && !hit;
    }
    return best;
}

// The two largest of two pairs of (largest, second)
template <class V> __device__ __forceinline__ void merge_two(V &a1, V &a2, V b1, V b2) {
    const V low = min_of(a1, b1);
    a1 = max_of(a1, b1);
    a2 = max_of(low, max_of(a2, b2));
}
template <class V> __device__ __forceinline__ void merge_one(V &a1, V &a2, V b) {
    const V low = min_of(a1, b);
    a1 = max_of(a1, b);
    a2 = max_of(a2, low);
}
template <int STEP, class V> __device__ __forceinline__ void merge_two_step(V &a1, V &a2) {
    if constexpr (STEP >= 16) {
        V p1, q1, p2, q2;
        halves_of<STEP>(a1, p1, q1);
        halves_of<STEP>(a2, p2, q2);
        a1 = p1; a2 = p2;
        merge_two(a1, a2, q1, q2);
    } else {
        merge_two(a1, a2, other_of<STEP>(a1), other_of<STEP>(a2));
    }
}
template <int LANES, class V> __device__ __forceinline__ void merge_two_lanes(V &a1, V &a2) {
    if constexpr (LANES >= 2) merge_two_step<1>(a1, a2);
    if constexpr (LANES >= 4) merge_two_step<2>(a1, a2);
    if constexpr (LANES >= 8) merge_two_step<4>(a1, a2);
    if constexpr (LANES >= 16) merge_two_step<8>(a1, a2);
    if constexpr (LANES >= 32) merge_two_step<16>(a1, a2);
    if constexpr (LANES >= 64) merge_two_step<32>(a1, a2);
}
__device__ __forceinline__ int group_total(int a1, int a2, int top) {
    return top > 1 && a2 > none_of<int>() ? key_of(value_of(a1) + value_of(a2)) : a1;      // (a1 none: none)
}
__device__ __forceinline__ double group_total(double a1, double a2, int top) { return top > 1 && a2 > none_of<double>() ? a1 + a2 : a1; }
// whether two values that a decision kept apart are closer than `margin`
__device__ __forceinline__ bool too_near(int a, int b, float margin) { return b > none_of<int>() && value_of(a) - value_of(b) <= margin; }
__device__ __forceinline__ bool too_near(double, double, float) { return false; }

// Closes the cells of the groups that are not among the best k_groups.  `near` becomes true where the choice hangs on a difference of at
// most `margin`.  LANES: a group is the cells of a power of two of whole lanes (one pass for all groups); else any size, group by group.
template <int LPR, int EPL, bool LANES, class V>
__device__ __forceinline__ void gate_groups(V (&v)[EPL], const GateArgs &a, float margin, bool &near) {
    const V none = none_of<V>();
    const int t = threadIdx.x % LPR, per_group = a.n / a.n_groups;
    V last = none;
    if constexpr (LANES) {
        const int lanes = per_group / EPL;
        V a1 = v[0], a2 = none;
#pragma unroll
        for (int j = 1; j < EPL; ++j) merge_one(a1, a2, v[j]);
        if constexpr (LPR >= 4) { if (lanes >= 2) merge_two_step<1>(a1, a2); }
        if constexpr (LPR >= 8) { if (lanes >= 4) merge_two_step<2>(a1, a2); }
        if constexpr (LPR >= 16) { if (lanes >= 8) merge_two_step<4>(a1, a2); }
        if constexpr (LPR >= 32) { if (lanes >= 16) merge_two_step<8>(a1, a2); }
        if constexpr (LPR >= 64) { if (lanes >= 32) merge_two_step<16>(a1, a2); }
        V total[1] = {(t & (lanes - 1)) == 0 ? group_total(a1, a2, a.group_top) : none};         // its first lane holds it
        bool keep = false;
        for (int q = 0; q <= a.k_groups && q < a.n_groups; ++q) {
            int mine;
            const V best = take_best<LPR, 1>(total, mine);
            if (q == a.k_groups) near = near || too_near(last, best, margin);
            else {
                last = best;
                const uint64_t who = group_ballot<LPR>(mine >= 0);
                keep = keep || (who && ((__ffsll((unsigned long long)who) - 1) ^ t) < lanes);
            }
        }
#pragma unroll
        for (int j = 0; j < EPL; ++j) v[j] = keep ? v[j] : none;
    } else {
        V total[EPL];                                  // of groups t EPL + j
#pragma unroll
        for (int j = 0; j < EPL; ++j) total[j] = none;
        for (int g = 0; g < a.n_groups; ++g) {
            V a1 = none, a2 = none;
            // this lane's cells of group g: from `from` up to `from + per_group`
            const int from = g * per_group - t * EPL;
#pragma unroll
            for (int j = 0; j < EPL; ++j) merge_one(a1, a2, (unsigned)(j - from) < (unsigned)per_group ? v[j] : none);
            merge_two_lanes<LPR>(a1, a2);
#pragma unroll
            for (int j = 0; j < EPL; ++j)
                if (t * EPL + j == g) total[j] = group_total(a1, a2, a.group_top);
        }
        uint32_t keep = 0;
        for (int q = 0; q <= a.k_groups && q < a.n_groups; ++q) {
            int mine;
            const V best = take_best<LPR, EPL>(total, mine);
            if (q == a.k_groups) near = near || too_near(last, best, margin);
            else {
                last = best;
                int g = mine;                          // which group that was, for all lanes
                if constexpr (LPR > 1) {
                    const uint64_t who = group_ballot<LPR>(mine >= 0);
                    const int lane = who ? __ffsll((unsigned long long)who) - 1 : 0, its = __shfl(mine, (int)(threadIdx.x & 63) - t + lane);
                    g = its < 0 ? -1 : lane * EPL + its;
                }
                const int from = g < 0 ? EPL : g * per_group - t * EPL;
#pragma unroll
                for (int j = 0; j < EPL; ++j)
                    if ((unsigned)(j - from) < (unsigned)per_group) keep |= 1u << j;
            }
        }
#pragma unroll
        for (int j = 0; j < EPL; ++j) v[j] = (keep >> j) & 1 ? v[j] : none;
    }
}

// Writes the chosen cells to `chosen` [k] (LDS, -1 where there are no more).  `near` as above, over the order of the chosen and the last
// one's lead over the rest.
template <int LPR, int EPL, class V>
__device__ __forceinline__ void gate_choose(V (&v)[EPL], int k, bool check, float margin, bool &near, int *chosen) {
    const int t = threadIdx.x % LPR;
    V last = none_of<V>();
    for (int s = 0; s < k + (check ? 1 : 0); ++s) {
        int mine;
        const V best = take_best<LPR, EPL>(v, mine);
        if (check) {                                   // (uniform)
            near = near || (s > 0 && too_near(last, best, margin));
            last = best;
        }
        if (s < k) {
            if (mine >= 0) chosen[s] = t * EPL + mine;
            else if (t == 0 && !(best > none_of<V>())) chosen[s] = -1;
        }
    }
}

// the choice of row r in 64 bits, by all lanes of the wave, EPL cells each
template <class T, int EPL> __device__ __forceinline__ void gate_exact(const GateArgs &a, int64_t r, int *chosen) {
    const int e0 = (int)(threadIdx.x & 63) * EPL;
    float x[EPL], at = GATE_NONE;
    gate_load<T, EPL>(x, a, reinterpret_cast<const T *>(a.logits) + r * a.ldl, r, e0, true);
#pragma unroll
    for (int j = 0; j < EPL; ++j) at = fmaxf(at, x[j]);
    at = lane_max<64>(at);
    double v[EPL], total = 0.;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
        v[j] = a.sigmoid ? 1. / (1. + exp(-(double)x[j])) : exp((double)x[j] - (double)at);
        total += v[j];
    }
    total = a.sigmoid ? 1. : lane_sum64<64>(total);
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
        v[j] = v[j] / total;
        if (a.bias) v[j] += e0 + j < a.n ? (double)a.bias[e0 + j] : 0.;
        v[j] = x[j] > GATE_NONE ? v[j] : (double)GATE_NONE;
    }
    bool done = false;
    if (a.n_groups > 1) gate_groups<64, EPL, false>(v, a, -1.f, done);
    if (!a.bias)
#pragma unroll
        for (int j = 0; j < EPL; ++j) v[j] = v[j] > (double)GATE_NONE ? (double)x[j] : (double)GATE_NONE;
    gate_choose<64, EPL>(v, a.k, false, -1.f, done, chosen);
}

// LPR lanes share a row, lane t holds cells t EPL ... and slots t, t + LPR, ...
template <class T, int LPR, int EPL, bool SCORED, bool LANES>
__global__ __launch_bounds__(256, SCORED ? 2 : 3) void k_gate_fwd(float *__restrict__ weights, int32_t *__restrict__ cells, GateArgs a) {
    constexpr int RPB = 256 / LPR, MAX_K = LPR * EPL < GATE_MAX_K ? LPR * EPL : GATE_MAX_K;
    __shared__ int chosen[RPB][MAX_K + 1];             // (+1: a column's entries fall into different banks)
    const int t = threadIdx.x % LPR, e0 = t * EPL;
    int *const mine = chosen[threadIdx.x / LPR];
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB) {
        const int64_t r = r0 + threadIdx.x / LPR;
        const bool live = r < a.rows;
        const T *row = reinterpret_cast<const T *>(a.logits) + r * a.ldl;
        float x[EPL], high = GATE_NONE;
        gate_load<T, EPL>(x, a, row, r, e0, live);
        bool bad = false;                              // a NaN, or +inf under softmax
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
            bad = bad || !(a.sigmoid ? x[j] <= __builtin_huge_valf() : x[j] < __builtin_huge_valf());
            high = fmaxf(high, x[j]);
        }
        if (!a.sigmoid) high = lane_max<LPR>(high);
        const float at = high > GATE_NONE ? high : 0.f;      // (softmax: what the exponents are relative to)
        float all = 1.f;                                     // the softmax's sum, where it is needed
        if (!a.sigmoid && (SCORED || !a.renormalise)) {
            all = 0.f;
#pragma unroll
            for (int j = 0; j < EPL; ++j) all += expf(x[j] - at);
            all = lane_sum<LPR>(all);
        }
        wave_sync();                                         // the last row's list has been read
        if constexpr (!SCORED) {
            int v[EPL];
#pragma unroll
            for (int j = 0; j < EPL; ++j) v[j] = key_of(x[j]);
            bool exact = false;
            if (a.n_groups > 1) gate_groups<LPR, EPL, LANES>(v, a, -1.f, exact);
            bad = group_ballot<LPR>(bad) != 0;
            gate_choose<LPR, EPL>(v, a.k, false, -1.f, exact, mine);
        } else {
            bool near = false;
            const float each = all > 0.f ? 1.f / all : 0.f;
            float w[EPL], span = 0.f;
#pragma unroll
            for (int j = 0; j < EPL; ++j) w[j] = a.sigmoid ? __builtin_amdgcn_rcpf(1.f + __expf(-x[j])) : __expf(x[j] - at) * each;
            if (a.bias)
#pragma unroll
                for (int j = 0; j < EPL; j += 4) {
                    float b[4];
                    load_part<float>(b, a.bias + e0 + j, a.n - e0 - j);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        w[j + i] += b[i];
                        if (fabsf(b[i]) < __builtin_huge_valf()) span = fmaxf(span, fabsf(b[i]));
                    }
                }
            // In units of 2^-24: a row's scores are off by 4 (sigmoid) or by 43 of their own sum, which is at most 1 (softmax: 32 + 6
            // additions, exp, the reciprocal), a sum with the bias by 1 + |bias| more; four values take part where two groups' two best
            // are compared.  Decisions that hang on less than this are left to 64 bits.
            const float margin = 6e-8f * (64.f + 8.f * lane_max<LPR>(span));
            int v[EPL];
#pragma unroll
            for (int j = 0; j < EPL; ++j) {
                const bool open = x[j] > GATE_NONE;
                bad = bad || (open && w[j] != w[j]);
                v[j] = open ? key_of(w[j]) : none_of<int>();
            }
            if (a.n_groups > 1) gate_groups<LPR, EPL, LANES>(v, a, margin, near);
            // without a bias the choice inside the groups goes by the logits (scores that saturate still differ there), read again: kept,
            // they would cost every row 32 registers
            if (!a.bias) {
                float y[EPL];
                gate_load<T, EPL>(y, a, row, r, e0, live);
#pragma unroll
                for (int j = 0; j < EPL; ++j) v[j] = v[j] > none_of<int>() ? key_of(y[j]) : none_of<int>();
            }
            bad = group_ballot<LPR>(bad) != 0;
            gate_choose<LPR, EPL>(v, a.k, a.bias != nullptr, margin, near, mine);
            // rows whose choice hangs on fp32's error, one after the other, each by the whole wave
            for (uint64_t doubt = __ballot(near && live && !bad && t == 0); doubt; doubt &= doubt - 1) {
                const int own = ((int)(threadIdx.x & ~63) + __ffsll((unsigned long long)doubt) - 1) / LPR;
                gate_exact<T, (LPR * EPL + 63) / 64>(a, r0 + own, chosen[own]);
            }
        }
        wave_sync();
        // weights from the logits of the chosen: the largest of them, then the sum, then the weights (a lane's slots are few)
        const int slots = live && !bad ? a.k : 0;
        float base = GATE_NONE, total = 0.f;
        auto log_score = [&](int c) {
            const float l = (float)row[c];
            return a.sigmoid ? log_sigmoid(l) : l;
        };
        if (a.renormalise) {
            for (int s = t; s < slots; s += LPR)
                if (mine[s] >= 0) base = fmaxf(base, log_score(mine[s]));
            base = lane_max<LPR>(base);
            if (!(base > GATE_NONE)) base = 0.f;
            for (int s = t; s < slots; s += LPR)
                if (mine[s] >= 0) total += expf(log_score(mine[s]) - base);
            total = lane_sum<LPR>(total);
        } else {
            base = a.sigmoid ? 0.f : at;
            total = all;
        }
        if (!(total > 0.f)) total = 1.f;
        if (!live) continue;
        for (int s = t; s < a.k; s += LPR) {
            const int c = bad ? -1 : mine[s];
            cells[r * a.k + s] = c;
            weights[r * a.k + s] = bad ? __builtin_nanf("") : c >= 0 ? expf(log_score(c) - base) / total * a.scale : 0.f;
        }
    }
}

template <class T, int LPR, int EPL>
__global__ __launch_bounds__(256) void k_gate_bwd(T *__restrict__ dx, int64_t ldd, const float *__restrict__ dw, int64_t lddw,
                                                  const int32_t *__restrict__ cells, GateArgs a) {
    constexpr int RPB = 256 / LPR;
    __shared__ float out[RPB][LPR * EPL + 1];             // d of the chosen cells, 0 elsewhere; a group's own lanes alone use its row
    const int t = threadIdx.x % LPR, e0 = t * EPL;
    float *const mine = out[threadIdx.x / LPR];
    const bool all = !a.sigmoid && !a.renormalise;        // the softmax over all open cells: all logits are read
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB) {
        const int64_t r = r0 + threadIdx.x / LPR;
        const bool live = r < a.rows;
        const T *row = reinterpret_cast<const T *>(a.logits) + r * a.ldl;
        const int slots = live ? a.k : 0;
        auto cell_of = [&](int s) {
            const int c = cells[r * a.k + s];
            return c < a.n ? c : -1;
        };
        auto log_score = [&](float l) { return a.sigmoid ? log_sigmoid(l) : l; };
        wave_sync();                                      // the last row has been read
#pragma unroll
        for (int j = 0; j < EPL; ++j) mine[e0 + j] = 0.f;
        // what the scores are relative to, their sum, and sum p g
        float base = GATE_NONE, total = 0.f, mean = 0.f, some = -1.f, xa[EPL];
        if (all) {
            gate_load<T, EPL>(xa, a, row, r, e0, live);
#pragma unroll
            for (int j = 0; j < EPL; ++j) base = fmaxf(base, xa[j]);
        }
        for (int s = t; s < slots; s += LPR) {
            const int c = cell_of(s);
            some = fmaxf(some, (float)c);
            if (c >= 0 && !all) base = fmaxf(base, log_score((float)row[c]));
        }
        some = lane_max<LPR>(some);
        base = lane_max<LPR>(base);
        if (!(base > GATE_NONE) || (a.sigmoid && !a.renormalise)) base = 0.f;
        if (all) {
#pragma unroll
            for (int j = 0; j < EPL; ++j) {
                xa[j] = expf(xa[j] - base);
                total += xa[j];
            }
        }
        for (int s = t; s < slots; s += LPR) {
            const int c = cell_of(s);
            if (c < 0) continue;
            const float p = expf(log_score((float)row[c]) - base);
            if (!all) total += p;
            mean += p * (dw[r * lddw + s] * a.scale);
        }
        total = lane_sum<LPR>(total);
        mean = lane_sum<LPR>(mean);
        if (a.sigmoid && !a.renormalise) { total = 1.f; mean = 0.f; }
        if (!(total > 0.f)) total = 1.f;
        mean /= total;
        wave_sync();                                      // the zeros are there
        for (int s = t; s < slots; s += LPR) {
            const int c = cell_of(s);
            if (c < 0) continue;
            const float l = (float)row[c], g = dw[r * lddw + s] * a.scale;
            float d = expf(log_score(l) - base) / total * (all ? g : g - mean);
            if (a.sigmoid) d *= 1.f / (1.f + expf(l));    // 1 - s
            mine[c] = d;
        }
        wave_sync();
        if (!live) continue;
        constexpr int N = EPL < Vec<T>::N ? EPL : Vec<T>::N;
        typedef T part __attribute__((ext_vector_type(N)));
        typedef part part_at __attribute__((aligned(sizeof(T))));
        T *to = dx + r * ldd + e0;
        const float share = mean / total;
#pragma unroll
        for (int j = 0; j < EPL; j += N) {
            part v;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float d = mine[e0 + j + i];
                if (all) d -= xa[j + i] * share;
                v[i] = (T)(some >= 0.f ? d : 0.f);        // (a row without cells has no gradient)
            }
            if (e0 + j + N <= a.n) *reinterpret_cast<part_at *>(to + j) = v;
            else
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (e0 + j + i < a.n) to[j + i] = v[i];
        }
    }
}

__global__ void k_gate_no_offsets(int32_t *__restrict__ offsets, int n) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c < n) offsets[c] = 0;
}

// lanes and cells per lane for n cells: the fewest lanes at up to MOST (32, or 16 where scores are compared: with 32 those kernels take
// 220 registers, two waves a SIMD) values each
template <int MOST, class F> static int gate_shape(int n, F &&f) {
    static_assert(MOST == 16 || MOST == 32, "64 lanes of 16 cells or 32 lanes of 32 hold the most there are");
    using std::integral_constant;
    if (n <= 8) return f(integral_constant<int, 1>{}, integral_constant<int, 8>{});
    if (n <= 16) return f(integral_constant<int, 1>{}, integral_constant<int, 16>{});
    if (n <= MOST) return f(integral_constant<int, 1>{}, integral_constant<int, MOST>{});
    if (n <= 2 * MOST) return f(integral_constant<int, 2>{}, integral_constant<int, MOST>{});
    if (n <= 4 * MOST) return f(integral_constant<int, 4>{}, integral_constant<int, MOST>{});
    if (n <= 8 * MOST) return f(integral_constant<int, 8>{}, integral_constant<int, MOST>{});
    if (n <= 16 * MOST) return f(integral_constant<int, 16>{}, integral_constant<int, MOST>{});
    if constexpr (MOST == 32) return f(integral_constant<int, 32>{}, integral_constant<int, MOST>{});       // (1024 cells, the most there are)
    else {
        if (n <= 32 * MOST) return f(integral_constant<int, 32>{}, integral_constant<int, MOST>{});
        return f(integral_constant<int, 64>{}, integral_constant<int, MOST>{});
    }
}

static unsigned gate_blocks(int64_t rows, int rpb) {
    const int64_t n = (rows + rpb - 1) / rpb;
    return (unsigned)(n < 8192 ? n : 8192);
}

template <class T, bool SCORED> static int gate_forward_as(float *weights, int32_t *cells, const GateArgs &a, hipStream_t st) {
    return gate_shape<SCORED ? 16 : 32>(a.n, [&](auto lpr, auto epl) {
        constexpr int L = lpr, E = epl;
        const int per_group = a.n / a.n_groups, lanes = per_group / E;
        const bool whole = L > 1 && a.n_groups > 1 && per_group % E == 0 && (lanes & (lanes - 1)) == 0 && lanes < L;     // groups of whole lanes
        const dim3 grid(gate_blocks(a.rows, 256 / L));
        if (whole) hipLaunchKernelGGL((k_gate_fwd<T, L, E, SCORED, (L > 1)>), grid, dim3(256), 0, st, weights, cells, a);
        else hipLaunchKernelGGL((k_gate_fwd<T, L, E, SCORED, false>), grid, dim3(256), 0, st, weights, cells, a);
        return check_launch("k_gate_fwd");
    });
}
template <class T> static int gate_forward(float *weights, int32_t *cells, const GateArgs &a, hipStream_t st) {
    const bool scored = a.bias || (a.n_groups > 1 && a.group_top > 1);
    return scored ? gate_forward_as<T, true>(weights, cells, a, st) : gate_forward_as<T, false>(weights, cells, a, st);
}
template <class T>
static int gate_backward(void *dx, int64_t ldd, const float *dw, int64_t lddw, const int32_t *cells, const GateArgs &a, hipStream_t st) {
    return gate_shape<32>(a.n, [&](auto lpr, auto epl) {
        constexpr int L = lpr, E = epl;
        hipLaunchKernelGGL((k_gate_bwd<T, L, E>), dim3(gate_blocks(a.rows, 256 / L)), dim3(256), 0, st, (T *)dx, ldd, dw, lddw, cells, a);
        return check_launch("k_gate_bwd");
    });
}

}  // namespace mnr

using namespace mnr;

static int gate_check(const char *who, const void *logits, int64_t ldl, const uint8_t *mask, int64_t ldm, int64_t rows, int n_cells, int k, int score,
                      int type) {
    MNR_REQUIRE(type_ok(type), "unknown element type passed to %s", who);
    MNR_REQUIRE(rows >= 0 && rows < (1ll << 31) && n_cells >= 1 && n_cells <= 1024, "%s needs 0 <= rows < 2^31 and 1 to 1024 cells", who);
    MNR_REQUIRE(k >= 1 && k <= n_cells && k <= GATE_MAX_K, "%s chooses 1 to 32 cells, at most as many as there are", who);
    MNR_REQUIRE(score == 0 || score == 1, "the score of %s is 0 (softmax) or 1 (sigmoid)", who);
    MNR_REQUIRE(rows == 0 || logits, "null pointer passed to %s", who);
    MNR_REQUIRE(rows <= 1 || ldl >= n_cells, "row pitch smaller than a row passed to %s", who);
    MNR_REQUIRE(!mask || rows <= 1 || ldm == 0 || ldm >= n_cells, "mask pitch smaller than a row passed to %s", who);
    return MNR_OK;
}

extern "C" int mnr_gate_forward(float *weights_dev, int32_t *cells_dev, const void *logits_dev, int64_t ldl, const float *bias_dev,
                                const uint8_t *mask_dev, int64_t ldm, int64_t rows, int n_cells, int k, int score, int n_groups, int k_groups,
                                int group_top, int renormalise, float scale, int type, void *stream) {
    const int rc = gate_check("mnr_gate_forward", logits_dev, ldl, mask_dev, ldm, rows, n_cells, k, score, type);
    if (rc != MNR_OK) return rc;
    MNR_REQUIRE(n_groups >= 1 && n_cells % n_groups == 0, "mnr_gate_forward: the groups divide the cells evenly");
    MNR_REQUIRE(k_groups >= 1 && k_groups <= n_groups && (int64_t)k <= (int64_t)k_groups * (n_cells / n_groups),
                "mnr_gate_forward: 1 <= k_groups <= n_groups, and the open groups hold k cells");
    MNR_REQUIRE(group_top == 1 || group_top == 2, "mnr_gate_forward: a group counts by its best cell or its best two");
    if (rows == 0) return MNR_OK;
    MNR_REQUIRE(weights_dev && cells_dev, "null pointer passed to mnr_gate_forward");
    const GateArgs a{logits_dev, ldl, bias_dev, mask_dev, ldm, rows, n_cells, k, score, n_groups, k_groups, group_top, renormalise, scale};
    hipStream_t st = as_stream(stream);
    if (type == MNR_F32) return gate_forward<float>(weights_dev, cells_dev, a, st);
    if (type == MNR_F16) return gate_forward<f16_t>(weights_dev, cells_dev, a, st);
    return gate_forward<bf16_t>(weights_dev, cells_dev, a, st);
}

extern "C" int mnr_gate_backward(void *dlogits_dev, int64_t ldd, const float *dweights_dev, int64_t lddw, const void *logits_dev, int64_t ldl,
                                 const int32_t *cells_dev, const uint8_t *mask_dev, int64_t ldm, int64_t rows, int n_cells, int k, int score,
                                 int renormalise, float scale, int type, void *stream) {
    const int rc = gate_check("mnr_gate_backward", logits_dev, ldl, mask_dev, ldm, rows, n_cells, k, score, type);
    if (rc != MNR_OK) return rc;
    if (rows == 0) return MNR_OK;
    MNR_REQUIRE(dlogits_dev && dweights_dev && cells_dev, "null pointer passed to mnr_gate_backward");
    MNR_REQUIRE(rows == 1 || (ldd >= n_cells && lddw >= k), "row pitch smaller than a row passed to mnr_gate_backward");
    const GateArgs a{logits_dev, ldl, nullptr, mask_dev, ldm, rows, n_cells, k, score, 1, 1, 1, renormalise, scale};
    hipStream_t st = as_stream(stream);
    if (type == MNR_F32) return gate_backward<float>(dlogits_dev, ldd, dweights_dev, lddw, cells_dev, a, st);
    if (type == MNR_F16) return gate_backward<f16_t>(dlogits_dev, ldd, dweights_dev, lddw, cells_dev, a, st);
    return gate_backward<bf16_t>(dlogits_dev, ldd, dweights_dev, lddw, cells_dev, a, st);
}

extern "C" size_t mnr_gate_dispatch_workspace_bytes(int64_t slots, int n_cells) {
    return slots < 0 || slots >= (1ll << 31) || n_cells < 1 ? 0 : (size_t)slots * 4 + sort_rows_bytes(slots, n_cells) + 16;
}

extern "C" int mnr_gate_dispatch(int32_t *order_dev, int32_t *offsets_dev, const int32_t *cells_dev, int64_t slots, int n_cells, void *workspace_dev,
                                 size_t workspace_bytes, void *stream) {
    MNR_REQUIRE(slots >= 0 && slots < (1ll << 31) && n_cells >= 1 && n_cells < (1 << 24), "mnr_gate_dispatch needs 0 <= slots < 2^31 and 1 to 2^24 - 1 cells");
    MNR_REQUIRE(offsets_dev && (slots == 0 || (order_dev && cells_dev)), "null pointer passed to mnr_gate_dispatch");
    MNR_REQUIRE(slots == 0 || (workspace_dev && workspace_bytes >= mnr_gate_dispatch_workspace_bytes(slots, n_cells)),
                "mnr_gate_dispatch needs %zu bytes of workspace", mnr_gate_dispatch_workspace_bytes(slots, n_cells));
    hipStream_t st = as_stream(stream);
    if (slots == 0) {
        hipLaunchKernelGGL(k_gate_no_offsets, dim3((n_cells + 256) / 256), dim3(256), 0, st, offsets_dev, n_cells + 1);
        return check_launch("k_gate_no_offsets");
    }
    int32_t *keys = reinterpret_cast<int32_t *>(workspace_dev);
    return sort_rows(KeySource{cells_dev, MNR_I32, 1, n_cells}, slots, order_dev, keys, keys + slots, SortExtras{nullptr, 0, 0, offsets_dev}, st);
}
