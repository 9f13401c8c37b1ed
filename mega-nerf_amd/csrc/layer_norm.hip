// layer_norm.hip -- layer norm over the last dimension and its adjoint.
//
//   y[r][c] = (x[r][c] - mean_r) rstd_r w[c] + b[c],   mean_r = sum_c x / C,  rstd_r = 1 / sqrt(sum_c (x - mean_r)^2 / C + eps)
//   with g = dy w,  h = (x - mean) rstd:   dx = rstd (g - mean_c(g) - h mean_c(g h)),   dw = sum_r dy h,   db = sum_r dy
//
// Bound by HBM: the forward reads x and writes y, the backward reads x and dy and writes dx.  So a row stays in registers from its
// one load on: the variance is the second pass over registers (centred: no cancellation of E x^2 - mean^2), and the backward keeps
// the column sums of dw / db of all its rows in registers too, writes them once per workgroup and joins the workgroups' sums in a
// second launch in a fixed order (no atomics: the same bits every time).  Statistics and sums are fp32; outputs round once.  The next
// row is on its way while a row is summed (backward of 20011 x 319 bf16: 38.8 -> 17.6 us).  196608 x 512 fp32: forward 145 us (5.5 TB/s),
// backward 238 + 5 us (5.1 TB/s), where a plain copy reaches 4.9.
#include "common.h"
#include "op_device.h"

namespace mnr {

// sum over the TPR threads that share a row: lanes of one wave, or a whole workgroup of 256 through LDS
template <int TPR> __device__ __forceinline__ float row_sum(float s, float *lds) {
    if constexpr (TPR <= 64) return lane_sum<TPR>(s);
    s = lane_sum<64>(s);
    const int wave = threadIdx.x >> 6;
    __syncthreads();                                   // the previous sum has been read
    if ((threadIdx.x & 63) == 0) lds[wave] = s;
    __syncthreads();
    float t = lds[0];
#pragma unroll
    for (int w = 1; w < TPR / 64; ++w) t += lds[w];
    return t;
}

// the chunk of w and b at column c, of which n columns exist (1 and 0 where there is none)
template <int V>
__device__ __forceinline__ void ln_affine(float (&wv)[V], float (&bv)[V], const void *w, const void *b, int wtype, int64_t c, int n) {
#pragma unroll
    for (int i = 0; i < V; ++i) { wv[i] = 1.f; bv[i] = 0.f; }
    if (w) load_any_part<V>(wv, w, c, n, wtype);
    if (b) load_any_part<V>(bv, b, c, n, wtype);
}

// TPR threads share a row, each holds NCH chunks of 16 bytes: chunk j of thread t covers columns (j TPR + t) V ...
template <class T, int TPR, int NCH>
__global__ __launch_bounds__(256) void k_ln_fwd(T *__restrict__ y, int64_t ldy, float *__restrict__ mean_out, float *__restrict__ rstd_out,
                                                const T *__restrict__ x, int64_t ldx, const void *__restrict__ w, const void *__restrict__ b,
                                                int wtype, int64_t rows, int C, float eps) {
    constexpr int V = Vec<T>::N, RPB = 256 / TPR;
    __shared__ float lds[4];
    const int t = threadIdx.x % TPR;
    const float inv = 1.f / (float)C;
    constexpr bool HOLD = NCH * V <= 16;               // w and b stay in registers over all rows where they are few
    float wv[HOLD ? NCH : 1][V], bv[HOLD ? NCH : 1][V];
    if (HOLD)
#pragma unroll
        for (int j = 0; j < (HOLD ? NCH : 1); ++j) ln_affine<V>(wv[j], bv[j], w, b, wtype, (j * TPR + t) * V, C - (j * TPR + t) * V);
    // (a group whose row is past the end runs along without loading or storing: lane and workgroup exchanges stay whole)
    typename Vec<T>::raw ahead[NCH];                   // the next row's 16 bytes, on their way while this row is summed
    auto fetch = [&](int64_t r) {
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            const int c = (j * TPR + t) * V;
            ahead[j] = load_raw<T>(x + r * ldx + c, r < rows ? C - c : 0);
        }
    };
    const int64_t step = (int64_t)gridDim.x * RPB;
    fetch((int64_t)blockIdx.x * RPB + threadIdx.x / TPR);
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < rows; r0 += step) {
        const int64_t r = r0 + threadIdx.x / TPR;
        const bool live = r < rows;
        float v[NCH][V];
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[j][i] = (float)ahead[j][i];
                s += v[j][i];
            }
        fetch(r + step);
        // the mean of what is left after the first mean corrects its rounding: a row far from zero keeps its precision
        const float mean = row_sum<TPR>(s, lds) * inv;
        float q = 0.f, d = 0.f;
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            const int n = C - (j * TPR + t) * V;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[j][i] = i < n ? v[j][i] - mean : 0.f;
                d += v[j][i];
                q += v[j][i] * v[j][i];
            }
        }
        d = row_sum<TPR>(d, lds) * inv;
        q = row_sum<TPR>(q, lds) * inv - d * d;
        const float rstd = 1.f / sqrtf(fmaxf(q, 0.f) + eps);
        if (!live) continue;
        if (t == 0) {
            if (mean_out) mean_out[r] = mean + d;
            if (rstd_out) rstd_out[r] = rstd;
        }
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            const int c = (j * TPR + t) * V, n = C - c;
            if (!HOLD) ln_affine<V>(wv[0], bv[0], w, b, wtype, c, n);
#pragma unroll
            for (int i = 0; i < V; ++i) v[j][i] = (v[j][i] - d) * rstd * wv[HOLD ? j : 0][i] + bv[HOLD ? j : 0][i];
            store_part<T>(y + r * ldy + c, v[j], n);
        }
    }
}

// The adjoint: dx of every row, and this workgroup's sums of dy h and dy over its rows -> part[blockIdx.x][2][C]
template <class T, int TPR, int NCH>
__global__ __launch_bounds__(256) void k_ln_bwd(T *__restrict__ dx, int64_t lddx, float *__restrict__ part, const T *__restrict__ dy,
                                                int64_t lddy, const T *__restrict__ x, int64_t ldx, const void *__restrict__ w, int wtype,
                                                const float *__restrict__ mean_in, const float *__restrict__ rstd_in, int64_t rows, int C) {
    constexpr int V = Vec<T>::N, RPB = 256 / TPR;
    __shared__ float lds[4];
    extern __shared__ float cols[];                    // [RPB][TPR * NCH * V]: the groups' column sums meet here
    const int t = threadIdx.x % TPR;
    const float inv = 1.f / (float)C;
    constexpr bool HOLD = NCH * V <= 16;
    float wv[HOLD ? NCH : 1][V], none[V];
    if (HOLD)
#pragma unroll
        for (int j = 0; j < (HOLD ? NCH : 1); ++j) ln_affine<V>(wv[j], none, w, nullptr, wtype, (j * TPR + t) * V, C - (j * TPR + t) * V);
    float sw[NCH][V], sb[NCH][V];
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) sw[j][i] = sb[j][i] = 0.f;
    typename Vec<T>::raw xa[NCH], ga[NCH];             // the next row's, on their way while this row is summed
    float mean_a, rstd_a;
    auto fetch = [&](int64_t r) {
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            const int c = (j * TPR + t) * V, n = r < rows ? C - c : 0;
            xa[j] = load_raw<T>(x + r * ldx + c, n);
            ga[j] = load_raw<T>(dy + r * lddy + c, n);
        }
        mean_a = r < rows ? mean_in[r] : 0.f;
        rstd_a = r < rows ? rstd_in[r] : 0.f;
    };
    const int64_t step = (int64_t)gridDim.x * RPB;
    fetch((int64_t)blockIdx.x * RPB + threadIdx.x / TPR);
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < rows; r0 += step) {
        const int64_t r = r0 + threadIdx.x / TPR;
        const bool live = r < rows;
        float h[NCH][V], g[NCH][V];
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) { h[j][i] = (float)xa[j][i]; g[j][i] = (float)ga[j][i]; }
        const float mean = mean_a, rstd = rstd_a;
        fetch(r + step);
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            const int c = (j * TPR + t) * V, n = live ? C - c : 0;
            if (!HOLD) ln_affine<V>(wv[0], none, w, nullptr, wtype, c, n);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                h[j][i] = i < n ? (h[j][i] - mean) * rstd : 0.f;
                sw[j][i] += g[j][i] * h[j][i];
                sb[j][i] += g[j][i];
                g[j][i] *= wv[HOLD ? j : 0][i];
                s1 += g[j][i];
                s2 += g[j][i] * h[j][i];
            }
        }
        s1 = row_sum<TPR>(s1, lds) * inv;
        s2 = row_sum<TPR>(s2, lds) * inv;
        if (!live || !dx) continue;
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            const int c = (j * TPR + t) * V;
#pragma unroll
            for (int i = 0; i < V; ++i) g[j][i] = rstd * (g[j][i] - s1 - h[j][i] * s2);
            store_part<T>(dx + r * lddx + c, g[j], C - c);
        }
    }
    if (!part) return;
    constexpr int W = TPR * NCH * V;
    for (int which = 0; which < 2; ++which) {
        float *out = part + ((int64_t)blockIdx.x * 2 + which) * C;
        if constexpr (RPB == 1) {
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const int c = (j * TPR + t) * V + i;
                    if (c < C) out[c] = which ? sb[j][i] : sw[j][i];
                }
        } else {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i) cols[(threadIdx.x / TPR) * W + (j * TPR + t) * V + i] = which ? sb[j][i] : sw[j][i];
            __syncthreads();
            for (int c = threadIdx.x; c < C; c += 256) {
                float s = 0.f;
#pragma unroll 4
                for (int k = 0; k < RPB; ++k) s += cols[k * W + c];
                out[c] = s;
            }
        }
    }
}

// dw / db = sum of the workgroups' partial sums, in one fixed order: 16 columns x 64 phases per workgroup
__global__ __launch_bounds__(1024) void k_ln_join(void *__restrict__ dw, void *__restrict__ db, int wtype, const float *__restrict__ part,
                                                  int n_part, int C) {
    __shared__ float lds[64][17];
    const int i = threadIdx.x & 15, c = blockIdx.x * 16 + i, ph = threadIdx.x >> 4, which = blockIdx.y;
    void *out = which ? db : dw;
    if (!out) return;
    float s = 0.f;
    if (c < C)
#pragma unroll 4
        for (int p = ph; p < n_part; p += 64) s += part[((int64_t)p * 2 + which) * C + c];
    lds[ph][i] = s;
    __syncthreads();
    if (ph < 8) {
        s = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) s += lds[ph * 8 + k][i];
        lds[ph * 8][i] = s;                            // (read by this thread alone before)
    }
    __syncthreads();
    if (ph == 0 && c < C) {
        s = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) s += lds[k * 8][i];
        store_any(out, c, s, wtype);
    }
}

// ---- rows wider than the registers of a workgroup ---------------------------------------------------------------------------------
// The forward reads a row three times, the gradient x and dy twice for dx and once more for the column sums.  The L2s do not hold the rows
// of all workgroups in between: per row the forward fetches 3.0 times, and k_ln_dx_wide 1.9 to 2.0 times, what one reading of it fetches
// (FETCH_SIZE against that of k_ln_cols_wide, which reads once).  12000 x 8192 fp32: forward 228 us (3.4 TB/s of one read and one write;
// 4096 columns, held in registers, reach 5.3), dx 288, column sums 153; 6000 x 16384 bf16: 136, 207 and 122 us.
template <class T>
__global__ __launch_bounds__(256) void k_ln_fwd_wide(T *__restrict__ y, int64_t ldy, float *__restrict__ mean_out, float *__restrict__ rstd_out,
                                                     const T *__restrict__ x, int64_t ldx, const void *__restrict__ w,
                                                     const void *__restrict__ b, int wtype, int64_t rows, int64_t C, float eps) {
    constexpr int V = Vec<T>::N;
    __shared__ float lds[4];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T *xr = x + r * ldx;
        float v[V], s = 0.f, q = 0.f;
        auto part = [&](int64_t c) { return (int)(C - c < V ? C - c : V); };
        for (int64_t c = (int64_t)threadIdx.x * V; c < C; c += 256 * V) {
            load_part<T>(v, xr + c, part(c));
#pragma unroll
            for (int i = 0; i < V; ++i) s += v[i];
        }
        const float mean = row_sum<256>(s, lds) / (float)C;
        float d = 0.f;                                 // the mean's correction, kept apart from it to the end: their sum rounds to fp32
        for (int64_t c = (int64_t)threadIdx.x * V; c < C; c += 256 * V) {
            const int n = part(c);
            load_part<T>(v, xr + c, n);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float e = i < n ? v[i] - mean : 0.f;
                d += e;
                q += e * e;
            }
        }
        d = row_sum<256>(d, lds) / (float)C;
        const float rstd = 1.f / sqrtf(fmaxf(row_sum<256>(q, lds) / (float)C - d * d, 0.f) + eps);
        if (threadIdx.x == 0) {
            if (mean_out) mean_out[r] = mean + d;
            if (rstd_out) rstd_out[r] = rstd;
        }
        for (int64_t c = (int64_t)threadIdx.x * V; c < C; c += 256 * V) {
            const int n = part(c);
            load_part<T>(v, xr + c, n);
            float wv[V], bv[V];
            ln_affine<V>(wv, bv, w, b, wtype, c, n);
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = (v[i] - mean - d) * rstd * wv[i] + bv[i];
            store_part<T>(y + r * ldy + c, v, n);
        }
    }
}

template <class T>
__global__ __launch_bounds__(256) void k_ln_dx_wide(T *__restrict__ dx, int64_t lddx, const T *__restrict__ dy, int64_t lddy,
                                                    const T *__restrict__ x, int64_t ldx, const void *__restrict__ w, int wtype,
                                                    const float *__restrict__ mean_in, const float *__restrict__ rstd_in, int64_t rows,
                                                    int64_t C) {
    constexpr int V = Vec<T>::N;
    __shared__ float lds[4];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const float mean = mean_in[r], rstd = rstd_in[r];
        float h[V], g[V], s1 = 0.f, s2 = 0.f;
        auto fetch = [&](int64_t c, int n) {
            load_part<T>(h, x + r * ldx + c, n);
            load_part<T>(g, dy + r * lddy + c, n);
            float wv[V], none[V];
            ln_affine<V>(wv, none, w, nullptr, wtype, c, n);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                h[i] = i < n ? (h[i] - mean) * rstd : 0.f;
                g[i] *= wv[i];
            }
        };
        for (int64_t c = (int64_t)threadIdx.x * V; c < C; c += 256 * V) {
            fetch(c, (int)(C - c < V ? C - c : V));
#pragma unroll
            for (int i = 0; i < V; ++i) { s1 += g[i]; s2 += g[i] * h[i]; }
        }
        s1 = row_sum<256>(s1, lds) / (float)C;
        s2 = row_sum<256>(s2, lds) / (float)C;
        for (int64_t c = (int64_t)threadIdx.x * V; c < C; c += 256 * V) {
            const int n = (int)(C - c < V ? C - c : V);
            fetch(c, n);
#pragma unroll
            for (int i = 0; i < V; ++i) g[i] = rstd * (g[i] - s1 - h[i] * s2);
            store_part<T>(dx + r * lddx + c, g, n);
        }
    }
}

// column sums of a strip of rows: 64 columns x 4 row phases per workgroup -> part[blockIdx.y][2][C]
template <class T>
__global__ __launch_bounds__(256) void k_ln_cols_wide(float *__restrict__ part, const T *__restrict__ dy, int64_t lddy, const T *__restrict__ x,
                                                      int64_t ldx, const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
                                                      int64_t rows, int64_t C) {
    __shared__ float lds[2][4][64];
    const int lane = threadIdx.x & 63, ph = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    const int64_t per = (rows + gridDim.y - 1) / gridDim.y, r0 = (int64_t)blockIdx.y * per, r1 = r0 + per < rows ? r0 + per : rows;
    float sw = 0.f, sb = 0.f;
    if (c < C)
        for (int64_t r = r0 + ph; r < r1; r += 4) {
            const float g = (float)dy[r * lddy + c];
            sw += g * (((float)x[r * ldx + c] - mean_in[r]) * rstd_in[r]);
            sb += g;
        }
    lds[0][ph][lane] = sw;
    lds[1][ph][lane] = sb;
    __syncthreads();
    if (ph < 2 && c < C) part[((int64_t)blockIdx.y * 2 + ph) * C + c] = (lds[ph][0][lane] + lds[ph][1][lane]) + (lds[ph][2][lane] + lds[ph][3][lane]);
}

// ---- launches --------------------------------------------------------------------------------------------------------------------

// Threads per row and chunks per thread for C columns: the fewest threads that hold the row, so that narrow rows share a wave.
struct LnShape { int tpr, nch; };
template <class T> static LnShape ln_shape(int64_t C) {
    const int64_t ch = (C + Vec<T>::N - 1) / Vec<T>::N;
    if (ch <= 8) return {8, 1};
    if (ch <= 16) return {16, 1};
    if (ch <= 32) return {32, 1};
    if (ch <= 64) return {64, 1};
    if (ch <= 128) return {64, 2};
    if (ch <= 256) return {64, 4};
    if (ch <= 512) return {256, 2};
    if (ch <= 1024) return {256, 4};
    return {0, 0};                                     // wide form
}

template <class F> static int ln_dispatch(LnShape s, F &&f) {
    using std::integral_constant;
    if (s.tpr == 8) return f(integral_constant<int, 8>{}, integral_constant<int, 1>{});
    if (s.tpr == 16) return f(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    if (s.tpr == 32) return f(integral_constant<int, 32>{}, integral_constant<int, 1>{});
    if (s.tpr == 64 && s.nch == 1) return f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    if (s.tpr == 64 && s.nch == 2) return f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    if (s.tpr == 64) return f(integral_constant<int, 64>{}, integral_constant<int, 4>{});
    if (s.nch == 2) return f(integral_constant<int, 256>{}, integral_constant<int, 2>{});
    return f(integral_constant<int, 256>{}, integral_constant<int, 4>{});
}

// workgroups of the backward pass: each row group gets 4 rows or more to spread its 2 C partial sums over, at most 4 workgroups a CU.
// Both launches together with 2 / 4 / 8 / 16 / 32 rows a group: 500 x 4096 fp32 19 / 16 / 20 / 30 / 50 us, 2000 x 2048 fp32 22 / 19 / 20 /
// 26 / 42, 20011 x 319 bf16 21 / 21 / 24 / 35 / 58, 1000 x 64 fp32 5.7 / 6.4 / 8.1 / 12 / 19: few rows want their groups short.  Wide
// 16-bit rows in the thousands do not: 4000 x 8192 bf16 115 / 114 / 81 / 64 / 91, where the partial sums, written and read again, move twice the bytes of dx.
static int64_t ln_bwd_blocks(int64_t rows, int tpr) {
    const int64_t per = (256 / (tpr ? tpr : 256)) * 4, n = (rows + per - 1) / per;
    return n < 1 ? 1 : (n > 1024 ? 1024 : n);
}
static int64_t ln_strips(int64_t rows) { return rows < 64 ? 1 : (rows < 64 * 64 ? rows / 64 : 64); }

template <class T>
static int ln_forward(void *y, int64_t ldy, float *mean, float *rstd, const void *x, int64_t ldx, const void *w, const void *b, int wtype,
                      int64_t rows, int64_t C, float eps, hipStream_t st) {
    const LnShape s = ln_shape<T>(C);
    if (!s.tpr) {
        const int64_t n = rows < 2048 ? rows : 2048;
        hipLaunchKernelGGL((k_ln_fwd_wide<T>), dim3((unsigned)n), dim3(256), 0, st, (T *)y, ldy, mean, rstd, (const T *)x, ldx, w, b, wtype, rows, C, eps);
        return check_launch("k_ln_fwd_wide");
    }
    return ln_dispatch(s, [&](auto tpr, auto nch) {
        const int64_t n = (rows + 256 / tpr - 1) / (256 / tpr);
        hipLaunchKernelGGL((k_ln_fwd<T, tpr, nch>), dim3((unsigned)(n < 2048 ? n : 2048)), dim3(256), 0, st, (T *)y, ldy, mean, rstd, (const T *)x, ldx,
                           w, b, wtype, rows, (int)C, eps);
        return check_launch("k_ln_fwd");
    });
}

template <class T>
static int ln_backward(void *dx, int64_t lddx, void *dw, void *db, const void *dy, int64_t lddy, const void *x, int64_t ldx, const void *w,
                       int wtype, const float *mean, const float *rstd, int64_t rows, int64_t C, float *part, hipStream_t st) {
    const LnShape s = ln_shape<T>(C);
    const bool sums = dw || db;
    int64_t n_part;
    int rc = MNR_OK;
    if (!s.tpr) {
        n_part = ln_strips(rows);
        if (dx && rows > 0) {
            const int64_t n = rows < 2048 ? rows : 2048;
            hipLaunchKernelGGL((k_ln_dx_wide<T>), dim3((unsigned)n), dim3(256), 0, st, (T *)dx, lddx, (const T *)dy, lddy, (const T *)x, ldx, w, wtype,
                               mean, rstd, rows, C);
            rc = check_launch("k_ln_dx_wide");
        }
        if (rc == MNR_OK && sums) {
            hipLaunchKernelGGL((k_ln_cols_wide<T>), dim3((unsigned)((C + 63) / 64), (unsigned)n_part), dim3(256), 0, st, part, (const T *)dy, lddy,
                               (const T *)x, ldx, mean, rstd, rows, C);
            rc = check_launch("k_ln_cols_wide");
        }
    } else {
        n_part = ln_bwd_blocks(rows, s.tpr);
        rc = ln_dispatch(s, [&](auto tpr, auto nch) {
            const size_t lds = tpr < 256 ? (size_t)256 * nch * Vec<T>::N * sizeof(float) : 0;
            hipLaunchKernelGGL((k_ln_bwd<T, tpr, nch>), dim3((unsigned)n_part), dim3(256), lds, st, (T *)dx, lddx, sums ? part : nullptr, (const T *)dy,
                               lddy, (const T *)x, ldx, w, wtype, mean, rstd, rows, (int)C);
            return check_launch("k_ln_bwd");
        });
    }
    if (rc != MNR_OK || !sums) return rc;
    hipLaunchKernelGGL(k_ln_join, dim3((unsigned)((C + 15) / 16), 2), dim3(1024), 0, st, dw, db, wtype, part, (int)n_part, (int)C);
    return check_launch("k_ln_join");
}

static bool ln_sizes_ok(int64_t rows, int64_t C) { return rows >= 0 && C >= 1 && C <= (1 << 24); }

}  // namespace mnr

using namespace mnr;

extern "C" int mnr_layer_norm_forward(void *y_dev, int64_t ldy, float *mean_dev, float *rstd_dev, const void *x_dev, int64_t ldx,
                                      const void *w_dev, const void *b_dev, int64_t rows, int64_t cols, float eps, int type, int w_type,
                                      void *stream) {
    MNR_REQUIRE(type_ok(type) && type_ok(w_type), "unknown element type passed to mnr_layer_norm_forward");
    MNR_REQUIRE(ln_sizes_ok(rows, cols), "mnr_layer_norm_forward needs rows >= 0 and 1 <= cols <= 2^24");
    if (rows == 0) return MNR_OK;
    MNR_REQUIRE(x_dev && y_dev, "null pointer passed to mnr_layer_norm_forward");
    MNR_REQUIRE(rows == 1 || (ldx >= cols && ldy >= cols), "row pitch smaller than a row passed to mnr_layer_norm_forward");
    hipStream_t st = as_stream(stream);
    if (type == MNR_F32) return ln_forward<float>(y_dev, ldy, mean_dev, rstd_dev, x_dev, ldx, w_dev, b_dev, w_type, rows, cols, eps, st);
    if (type == MNR_F16) return ln_forward<f16_t>(y_dev, ldy, mean_dev, rstd_dev, x_dev, ldx, w_dev, b_dev, w_type, rows, cols, eps, st);
    return ln_forward<bf16_t>(y_dev, ldy, mean_dev, rstd_dev, x_dev, ldx, w_dev, b_dev, w_type, rows, cols, eps, st);
}

extern "C" size_t mnr_layer_norm_backward_workspace_bytes(int64_t rows, int64_t cols, int type) {
    if (!type_ok(type) || !ln_sizes_ok(rows, cols)) return 0;
    const LnShape s = type == MNR_F32 ? ln_shape<float>(cols) : ln_shape<f16_t>(cols);
    const int64_t n = s.tpr ? ln_bwd_blocks(rows, s.tpr) : ln_strips(rows);
    return (size_t)n * 2 * (size_t)cols * sizeof(float);
}

extern "C" int mnr_layer_norm_backward(void *dx_dev, int64_t lddx, void *dw_dev, void *db_dev, const void *dy_dev, int64_t lddy,
                                       const void *x_dev, int64_t ldx, const void *w_dev, const float *mean_dev, const float *rstd_dev,
                                       int64_t rows, int64_t cols, int type, int w_type, void *workspace_dev, size_t workspace_bytes,
                                       void *stream) {
    MNR_REQUIRE(type_ok(type) && type_ok(w_type), "unknown element type passed to mnr_layer_norm_backward");
    MNR_REQUIRE(ln_sizes_ok(rows, cols), "mnr_layer_norm_backward needs rows >= 0 and 1 <= cols <= 2^24");
    MNR_REQUIRE(rows == 0 || (dy_dev && x_dev && mean_dev && rstd_dev), "null pointer passed to mnr_layer_norm_backward");
    MNR_REQUIRE(rows <= 1 || (ldx >= cols && lddy >= cols && (!dx_dev || lddx >= cols)),
                "row pitch smaller than a row passed to mnr_layer_norm_backward");
    if (dw_dev || db_dev)
        MNR_REQUIRE(workspace_dev && workspace_bytes >= mnr_layer_norm_backward_workspace_bytes(rows, cols, type),
                    "mnr_layer_norm_backward needs %zu bytes of workspace", mnr_layer_norm_backward_workspace_bytes(rows, cols, type));
    if (rows == 0 && !dw_dev && !db_dev) return MNR_OK;
    hipStream_t st = as_stream(stream);
    float *part = reinterpret_cast<float *>(workspace_dev);
    if (type == MNR_F32) return ln_backward<float>(dx_dev, lddx, dw_dev, db_dev, dy_dev, lddy, x_dev, ldx, w_dev, w_type, mean_dev, rstd_dev, rows, cols, part, st);
    if (type == MNR_F16) return ln_backward<f16_t>(dx_dev, lddx, dw_dev, db_dev, dy_dev, lddy, x_dev, ldx, w_dev, w_type, mean_dev, rstd_dev, rows, cols, part, st);
    return ln_backward<bf16_t>(dx_dev, lddx, dw_dev, db_dev, dy_dev, lddy, x_dev, ldx, w_dev, w_type, mean_dev, rstd_dev, rows, cols, part, st);
}
