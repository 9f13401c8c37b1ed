// gate.hip -- a learned gate over the cells: which k cells a row goes to and with what weights, the gradient of the weights, and the
// rows of every cell in one stable order.  (mnr_route is the geometric router: distances to centroids instead of scores.)
//
//   s_e = softmax_e(x) or sigmoid(x_e) over the open cells (mask set, logit > -inf);   v_e = s_e + bias_e (x_e where there is no bias)
//   groups of n / n_groups cells: the k_groups groups with the largest sum of their group_top best (s + bias) stay open
//   chosen: the k largest v of what is open, largest first, the lowest index of equals;  w_j = scale s_j [ / sum_chosen s ]
//   gradient (cells fixed), g = scale dw:    softmax, renormalised: dx_j = p_j (g_j - sum p g) over the chosen, p = w / scale
//       softmax: dx_e = s_e (g_e [e chosen] - sum_chosen s g);   sigmoid: dx_j = s_j (1 - s_j) g_j, renormalised p_j (1 - s_j) (g_j - sum p g)
//
// Bound by HBM for few cells (a row is read once), by the rounds of arg-max for many.  8 to 64 lanes share a row and keep its
// selection values in registers; a round is a local scan and a DPP reduction.  Where no score enters a comparison the values are the
// logits themselves (exact); otherwise they are in 64 bits, so that the choice is the one of the definition.
// Weights are formed from the logits of the chosen (log-sigmoids for sigmoid), so renormalising never divides by an underflowed sum.
#include "row_sort.h"

namespace mnr {

template <class V> struct Best { V v; int e; };

template <int STEP> __device__ __forceinline__ float other_of(float x) { return __uint_as_float(lane_other<STEP>(__float_as_uint(x))); }
template <int STEP> __device__ __forceinline__ double other_of(double x) {
    const uint64_t b = (uint64_t)__double_as_longlong(x);
    return __longlong_as_double((long long)(((uint64_t)lane_other<STEP>((uint32_t)(b >> 32)) << 32) | lane_other<STEP>((uint32_t)b)));
}
template <int STEP> __device__ __forceinline__ int other_of(int x) { return (int)lane_other<STEP>((uint32_t)x); }
template <int STEP> __device__ __forceinline__ void halves_of(float x, float &a, float &b) {
    uint32_t p, q;
    lane_halves<STEP>(__float_as_uint(x), p, q);
    a = __uint_as_float(p); b = __uint_as_float(q);
}
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
template <class V> __device__ __forceinline__ void better(Best<V> &a, V v, int e) {
    if (v > a.v || (v == a.v && e < a.e)) { a.v = v; a.e = e; }
}
template <int STEP, class V> __device__ __forceinline__ void best_step(Best<V> &a) {
    if constexpr (STEP >= 16) {
        V va, vb;
        int ea, eb;
        halves_of<STEP>(a.v, va, vb);
        halves_of<STEP>(a.e, ea, eb);
        a.v = va; a.e = ea;
        better(a, vb, eb);
    } else {
        better(a, other_of<STEP>(a.v), other_of<STEP>(a.e));
    }
}
// the largest value of a group of LANES lanes and its lowest index, on every lane
template <int LANES, class V> __device__ __forceinline__ void lane_best(Best<V> &a) {
    if constexpr (LANES >= 2) best_step<1>(a);
    if constexpr (LANES >= 4) best_step<2>(a);
    if constexpr (LANES >= 8) best_step<4>(a);
    if constexpr (LANES >= 16) best_step<8>(a);
    if constexpr (LANES >= 32) best_step<16>(a);
    if constexpr (LANES >= 64) best_step<32>(a);
}
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

// LPR lanes share a row; lane t holds cells t, t + LPR, ... (EPL of them) and slots t, t + LPR, ... (KPL of them)
template <class T, int LPR, int EPL, class V>
__global__ __launch_bounds__(256) void k_gate_fwd(float *__restrict__ weights, int32_t *__restrict__ cells, GateArgs a) {
    constexpr int RPB = 256 / LPR, KPL = (GATE_MAX_K + LPR - 1) / LPR < EPL ? (GATE_MAX_K + LPR - 1) / LPR : EPL;
    constexpr bool WIDE = sizeof(V) == 8;
    const V none = (V)GATE_NONE;
    const int t = threadIdx.x % LPR;
    const int per_group = a.n / a.n_groups;
    int group[EPL];
    if (a.n_groups > 1)
#pragma unroll
        for (int j = 0; j < EPL; ++j) group[j] = (j * LPR + t) / per_group;
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB) {
        const int64_t r = r0 + threadIdx.x / LPR;
        const bool live = r < a.rows;
        const T *row = reinterpret_cast<const T *>(a.logits) + r * a.ldl;
        float x[EPL], high = GATE_NONE, bad = 0.f;
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
            const int e = j * LPR + t;
            bool open = live && e < a.n;
            if (open && a.mask) open = a.mask[r * a.ldm + e] != 0;
            x[j] = open ? (float)row[e] : GATE_NONE;
            if (!(x[j] < __builtin_huge_valf()) && !(a.sigmoid && x[j] == x[j])) bad = 1.f;       // a NaN, or +inf under softmax
            high = fmaxf(high, x[j]);
        }
        high = lane_max<LPR>(high);
        const float at = high > GATE_NONE ? high : 0.f;
        V v[EPL];                                     // what is compared
        if constexpr (WIDE) {
            double total = 0.;
#pragma unroll
            for (int j = 0; j < EPL; ++j) {
                v[j] = a.sigmoid ? 1. / (1. + exp(-(double)x[j])) : exp((double)x[j] - (double)at);
                total += v[j];
            }
            total = a.sigmoid ? 1. : lane_sum64<LPR>(total);
#pragma unroll
            for (int j = 0; j < EPL; ++j) {
                v[j] = x[j] > GATE_NONE ? v[j] / total : none;
                if (a.bias && x[j] > GATE_NONE) {
                    v[j] += (double)a.bias[j * LPR + t];
                    if (v[j] != v[j]) bad = 1.f;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < EPL; ++j) v[j] = x[j];
        }
        bad = lane_max<LPR>(bad);
        if (a.n_groups > 1) {
            V total[EPL];                             // of groups t, t + LPR, ...
#pragma unroll
            for (int j = 0; j < EPL; ++j) total[j] = none;
            for (int g = 0; g < a.n_groups; ++g) {
                Best<V> b{none, 1 << 30};
#pragma unroll
                for (int j = 0; j < EPL; ++j)
                    if (group[j] == g) better(b, v[j], j * LPR + t);
                lane_best<LPR>(b);
                V sum = b.v;
                if (a.group_top > 1 && b.v > none) {
                    Best<V> c{none, 1 << 30};
#pragma unroll
                    for (int j = 0; j < EPL; ++j)
                        if (group[j] == g && j * LPR + t != b.e) better(c, v[j], j * LPR + t);
                    lane_best<LPR>(c);
                    if (c.v > none) sum += c.v;
                }
#pragma unroll
                for (int j = 0; j < EPL; ++j)
                    if (j * LPR + t == g) total[j] = sum;
            }
            uint32_t keep = 0;
            for (int q = 0; q < a.k_groups; ++q) {
                Best<V> b{none, 1 << 30};
#pragma unroll
                for (int j = 0; j < EPL; ++j) better(b, total[j], j * LPR + t);
                lane_best<LPR>(b);
#pragma unroll
                for (int j = 0; j < EPL; ++j) {
                    if (b.v > none && group[j] == b.e) keep |= 1u << j;
                    if (j * LPR + t == b.e) total[j] = none;
                }
            }
            // without a bias the choice inside the groups goes by the logits (scores that saturate still differ there)
#pragma unroll
            for (int j = 0; j < EPL; ++j) {
                if (WIDE && !a.bias) v[j] = x[j];
                if (!((keep >> j) & 1)) v[j] = none;
            }
        }
        int cell[KPL];
#pragma unroll
        for (int q = 0; q < KPL; ++q) cell[q] = -1;
        for (int s = 0; s < a.k; ++s) {
            Best<V> b{none, 1 << 30};
#pragma unroll
            for (int j = 0; j < EPL; ++j) better(b, v[j], j * LPR + t);
            lane_best<LPR>(b);
#pragma unroll
            for (int j = 0; j < EPL; ++j)
                if (j * LPR + t == b.e) v[j] = none;
#pragma unroll
            for (int q = 0; q < KPL; ++q)
                if (q * LPR + t == s && b.v > none) cell[q] = b.e;
        }
        // weights from the logits of the chosen
        float w[KPL], total = 0.f, base = GATE_NONE;
#pragma unroll
        for (int q = 0; q < KPL; ++q) {
            if (bad > 0.f) cell[q] = -1;
            w[q] = cell[q] >= 0 ? (float)row[cell[q]] : GATE_NONE;
            if (a.sigmoid && cell[q] >= 0) w[q] = log_sigmoid(w[q]);
            base = fmaxf(base, w[q]);
        }
        if (a.renormalise) base = lane_max<LPR>(base);
        else base = a.sigmoid ? 0.f : at;
        if (!(base > GATE_NONE)) base = 0.f;
#pragma unroll
        for (int q = 0; q < KPL; ++q) {
            w[q] = cell[q] >= 0 ? expf(w[q] - base) : 0.f;
            total += w[q];
        }
        if (!a.renormalise) {
            total = 0.f;
#pragma unroll
            for (int j = 0; j < EPL; ++j) total += x[j] > GATE_NONE ? expf(x[j] - at) : 0.f;
        }
        total = lane_sum<LPR>(total);
        if (!a.renormalise && a.sigmoid) total = 1.f;
        if (!(total > 0.f)) total = 1.f;
        if (!live) continue;
#pragma unroll
        for (int q = 0; q < KPL; ++q) {
            const int s = q * LPR + t;
            if (s < a.k) {
                cells[r * a.k + s] = cell[q];
                weights[r * a.k + s] = bad > 0.f ? __builtin_nanf("") : w[q] / total * a.scale;
            }
        }
    }
}

template <class T, int LPR, int EPL>
__global__ __launch_bounds__(256) void k_gate_bwd(T *__restrict__ dx, int64_t ldd, const float *__restrict__ dw, int64_t lddw,
                                                  const int32_t *__restrict__ cells, GateArgs a) {
    constexpr int RPB = 256 / LPR, KPL = (GATE_MAX_K + LPR - 1) / LPR < EPL ? (GATE_MAX_K + LPR - 1) / LPR : EPL;
    __shared__ float out[RPB][LPR * EPL];             // g of the chosen cells, 0 elsewhere
    const int t = threadIdx.x % LPR, own = threadIdx.x / LPR;
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows; r0 += (int64_t)gridDim.x * RPB) {
        const int64_t r = r0 + own;
        const bool live = r < a.rows;
        const T *row = reinterpret_cast<const T *>(a.logits) + r * a.ldl;
        int cell[KPL];
        float x[KPL], g[KPL], base = GATE_NONE;
#pragma unroll
        for (int q = 0; q < KPL; ++q) {
            const int s = q * LPR + t;
            cell[q] = live && s < a.k ? cells[r * a.k + s] : -1;
            if (cell[q] >= a.n) cell[q] = -1;
            x[q] = cell[q] >= 0 ? (float)row[cell[q]] : GATE_NONE;
            g[q] = cell[q] >= 0 ? dw[r * lddw + s] * a.scale : 0.f;
        }
        const bool all = !a.sigmoid && !a.renormalise;    // the softmax over all open cells: their logits are read again
        float xa[EPL], total = 0.f;
        if (all) {
#pragma unroll
            for (int j = 0; j < EPL; ++j) {
                const int e = j * LPR + t;
                bool open = live && e < a.n;
                if (open && a.mask) open = a.mask[r * a.ldm + e] != 0;
                xa[j] = open ? (float)row[e] : GATE_NONE;
                base = fmaxf(base, xa[j]);
            }
        }
        float some = -1.f;                                // a row without cells has no gradient
#pragma unroll
        for (int q = 0; q < KPL; ++q) some = fmaxf(some, (float)cell[q]);
        some = lane_max<LPR>(some);
        float l[KPL];                                     // log of the score, up to a constant of the row
#pragma unroll
        for (int q = 0; q < KPL; ++q) {
            l[q] = a.sigmoid && cell[q] >= 0 ? log_sigmoid(x[q]) : x[q];
            if (!all) base = fmaxf(base, l[q]);
        }
        base = lane_max<LPR>(base);
        if (!(base > GATE_NONE) || (a.sigmoid && !a.renormalise)) base = 0.f;
        if (all) {
#pragma unroll
            for (int j = 0; j < EPL; ++j) {
                xa[j] = xa[j] > GATE_NONE ? expf(xa[j] - base) : 0.f;
                total += xa[j];
            }
        }
        float p[KPL];
#pragma unroll
        for (int q = 0; q < KPL; ++q) {
            p[q] = cell[q] >= 0 ? expf(l[q] - base) : 0.f;
            if (!all) total += p[q];
        }
        total = lane_sum<LPR>(total);
        if (a.sigmoid && !a.renormalise) total = 1.f;
        if (!(total > 0.f)) total = 1.f;
        float mean = 0.f;
#pragma unroll
        for (int q = 0; q < KPL; ++q) {
            p[q] /= total;
            mean += p[q] * g[q];
        }
        mean = lane_sum<LPR>(mean);
        if (a.sigmoid && !a.renormalise) mean = 0.f;
#pragma unroll
        for (int j = 0; j < EPL; ++j) out[own][j * LPR + t] = 0.f;
        __syncthreads();
#pragma unroll
        for (int q = 0; q < KPL; ++q) {
            if (cell[q] < 0) continue;
            float d = p[q] * (all ? g[q] : g[q] - mean);
            if (a.sigmoid) d *= 1.f / (1.f + expf(x[q]));     // 1 - s
            out[own][cell[q]] = d;
        }
        __syncthreads();
        if (live)
#pragma unroll
            for (int j = 0; j < EPL; ++j) {
                const int e = j * LPR + t;
                float d = out[own][e];
                if (all) d -= xa[j] / total * mean;
                if (e < a.n) dx[r * ldd + e] = (T)(some >= 0.f ? d : 0.f);
            }
        __syncthreads();
    }
}

__global__ void k_gate_no_offsets(int32_t *__restrict__ offsets, int n) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c < n) offsets[c] = 0;
}

// lanes and cells per lane for n cells: the fewest lanes at up to 8 (above 512 cells 16) values each
template <class F> static int gate_shape(int n, F &&f) {
    using std::integral_constant;
    if (n <= 8) return f(integral_constant<int, 8>{}, integral_constant<int, 1>{});
    if (n <= 16) return f(integral_constant<int, 8>{}, integral_constant<int, 2>{});
    if (n <= 32) return f(integral_constant<int, 8>{}, integral_constant<int, 4>{});
    if (n <= 64) return f(integral_constant<int, 16>{}, integral_constant<int, 4>{});
    if (n <= 128) return f(integral_constant<int, 16>{}, integral_constant<int, 8>{});
    if (n <= 256) return f(integral_constant<int, 32>{}, integral_constant<int, 8>{});
    if (n <= 512) return f(integral_constant<int, 64>{}, integral_constant<int, 8>{});
    return f(integral_constant<int, 64>{}, integral_constant<int, 16>{});
}

static unsigned gate_blocks(int64_t rows, int rpb) {
    const int64_t n = (rows + rpb - 1) / rpb;
    return (unsigned)(n < 8192 ? n : 8192);
}

template <class T> static int gate_forward(float *weights, int32_t *cells, const GateArgs &a, hipStream_t st) {
    const bool wide = a.bias || (a.n_groups > 1 && a.group_top > 1);
    return gate_shape(a.n, [&](auto lpr, auto epl) {
        constexpr int L = lpr, E = epl;
        if (wide) hipLaunchKernelGGL((k_gate_fwd<T, L, E, double>), dim3(gate_blocks(a.rows, 256 / L)), dim3(256), 0, st, weights, cells, a);
        else hipLaunchKernelGGL((k_gate_fwd<T, L, E, float>), dim3(gate_blocks(a.rows, 256 / L)), dim3(256), 0, st, weights, cells, a);
        return check_launch("k_gate_fwd");
    });
}
template <class T>
static int gate_backward(void *dx, int64_t ldd, const float *dw, int64_t lddw, const int32_t *cells, const GateArgs &a, hipStream_t st) {
    return gate_shape(a.n, [&](auto lpr, auto epl) {
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
