// int8_product.hip -- rows quantised to 8 bits with a scale each, and the product of two such matrices.
//
//   q[r][c] = round(127 x[r][c] / m_r), scale_r = m_r / 127, m_r = max_c |x[r][c]|      (to the nearest, ties to even)
//   y[m][n] = act( sa[m] sb[n] sum_k a[m][k] b[n][k] + bias[n] )                        (the sum exact in int32)
//
// The quantiser is bound by HBM: a row stays in registers between its maximum and its rounding.
#include <type_traits>

#include "common.h"
#include "op_device.h"

namespace mnr {

// 127 x / m to the nearest: fp32 is within 2e-5 of the quotient (two roundings of 2^-24 at 127), so only a value that near to a half
// is decided in 64 bits, where 127 x is exact and the quotient is at least 2^-33 from a half it does not equal.
__device__ __forceinline__ int quantised(float x, float inv, float m) {
    const float t = x * inv, q = rintf(t);
    if (fabsf(t - q) <= 0.4999f) return (int)q;
    return (int)rint((double)x * 127.0 / (double)m);
}

// four or eight values as bytes
template <int V> __device__ __forceinline__ void store_bytes(int8_t *p, const int (&q)[V]) {
#pragma unroll
    for (int i = 0; i < V; i += 4)
        *reinterpret_cast<uint32_t *>(p + i) = (q[i] & 255) | (q[i + 1] & 255) << 8 | (q[i + 2] & 255) << 16 | (uint32_t)(q[i + 3] & 255) << 24;
}

// TPR lanes of a wave share a row and hold NCH chunks of 16 bytes each (NCH 0: any width, the row is read twice)
template <class T, int TPR, int NCH>
__global__ __launch_bounds__(256) void k_quantize(int8_t *__restrict__ out, int64_t pitch, float *__restrict__ scale, const T *__restrict__ x,
                                                  int64_t ldx, int64_t rows, int64_t cols) {
    constexpr int V = Vec<T>::N, RPB = 256 / TPR;
    const int t = threadIdx.x % TPR;
    for (int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; r < rows; r += (int64_t)gridDim.x * RPB) {
        const T *row = x + r * ldx;
        float v[NCH ? NCH : 1][V], m = 0.f, z = 0.f;
        auto part = [&](int64_t c) { return (int)(cols - c < V ? cols - c : V); };
        auto look = [&](float (&w)[V], int64_t c) {
            load_part<T>(w, row + c, part(c));
#pragma unroll
            for (int i = 0; i < V; ++i) {
                m = fmaxf(m, fabsf(w[i]));
                z += w[i] * 0.f;                       // NaN if any value is an inf or NaN
            }
        };
        if constexpr (NCH > 0) {
#pragma unroll
            for (int j = 0; j < NCH; ++j) look(v[j], (int64_t)(j * TPR + t) * V);
        } else {
            for (int64_t c = (int64_t)t * V; c < cols; c += TPR * V) look(v[0], c);
        }
        m = lane_max<TPR>(m);
        z = lane_sum<TPR>(z);
        const bool dead = !(z == 0.f) || m == 0.f;
        const float inv = 127.f / m;
        if (t == 0) scale[r] = z == 0.f ? m / 127.f : __builtin_nanf("");
        auto put = [&](const float (&w)[V], int64_t c) {
            if (c >= pitch) return;                    // (pitch is a multiple of 16, so a chunk is all inside or all behind it)
            int q[V];
#pragma unroll
            for (int i = 0; i < V; ++i) q[i] = dead ? 0 : quantised(w[i], inv, m);
            store_bytes<V>(out + r * pitch + c, q);
        };
        if constexpr (NCH > 0) {
#pragma unroll
            for (int j = 0; j < NCH; ++j) put(v[j], (int64_t)(j * TPR + t) * V);
        } else {
            for (int64_t c = (int64_t)t * V; c < pitch; c += TPR * V) {
                load_part<T>(v[0], row + c, part(c));
                put(v[0], c);
            }
        }
    }
}

typedef int int4v __attribute__((ext_vector_type(4)));
typedef int int16v __attribute__((ext_vector_type(16)));

struct ProductArgs {
    void *y;  int64_t ldy;
    const int8_t *a;  int64_t lda;  const float *sa;
    const int8_t *b;  int64_t ldb;  const float *sb;
    const float *bias;
    int64_t m, n, k;
    int relu;
};

template <class T> __device__ __forceinline__ void put_product(const ProductArgs &p, int64_t m, int64_t n, int acc, float sa, float sb, float bias) {
    float y = (float)acc * sa * sb + bias;
    if (p.relu) y = y < 0.f ? 0.f : y;
    reinterpret_cast<T *>(p.y)[m * p.ldy + n] = (T)y;
}

// 128 x 128 tile, 64 bytes of K per step through LDS, four waves of 64 x 64 (2 x 2 v_mfma_i32_32x32x32_i8)
constexpr int PT = 128, PK = 64, PLD = PK + 16;        // (+16: the 32 rows of a fragment read fall into different banks)
template <class T> __global__ __launch_bounds__(256) void k_product(ProductArgs p) {
    __shared__ int8_t As[PT * PLD] __attribute__((aligned(16)));
    __shared__ int8_t Bs[PT * PLD] __attribute__((aligned(16)));
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wr = wave >> 1, wc = wave & 1, i32 = lane & 31, half = lane >> 5;
    const int64_t m0 = (int64_t)blockIdx.y * PT, n0 = (int64_t)blockIdx.x * PT;
    int16v acc[2][2] = {};
    for (int64_t k0 = 0; k0 < p.k; k0 += PK) {
        int4v ra[2], rb[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int e = threadIdx.x + i * 256, row = e >> 2;
            const int64_t kq = k0 + (e & 3) * 16;
            ra[i] = rb[i] = int4v{0, 0, 0, 0};
            if (kq < p.k && m0 + row < p.m) ra[i] = *reinterpret_cast<const int4v *>(p.a + (m0 + row) * p.lda + kq);
            if (kq < p.k && n0 + row < p.n) rb[i] = *reinterpret_cast<const int4v *>(p.b + (n0 + row) * p.ldb + kq);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int e = threadIdx.x + i * 256, at = (e >> 2) * PLD + (e & 3) * 16;
            *reinterpret_cast<int4v *>(As + at) = ra[i];
            *reinterpret_cast<int4v *>(Bs + at) = rb[i];
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < PK; kk += 32) {
            int4v af[2], bf[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                af[i] = *reinterpret_cast<const int4v *>(As + (wr * 64 + i * 32 + i32) * PLD + kk + half * 16);
                bf[i] = *reinterpret_cast<const int4v *>(Bs + (wc * 64 + i * 32 + i32) * PLD + kk + half * 16);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(af[i], bf[j], acc[i][j], 0, 0, 0);
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t n = n0 + wc * 64 + j * 32 + i32;
        if (n >= p.n) continue;
        const float sb = p.sb[n], bias = p.bias ? p.bias[n] : 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int64_t m = m0 + wr * 64 + i * 32 + (r & 3) + 8 * (r >> 2) + 4 * half;
                if (m < p.m) put_product<T>(p, m, n, acc[i][j][r], p.sa[m], sb, bias);
            }
    }
}

template <class T> static int product(const ProductArgs &p, hipStream_t st) {
    hipLaunchKernelGGL((k_product<T>), dim3((unsigned)((p.n + PT - 1) / PT), (unsigned)((p.m + PT - 1) / PT)), dim3(256), 0, st, p);
    return check_launch("k_product");
}

template <class T>
static int quantize(int8_t *out, int64_t pitch, float *scale, const void *x, int64_t ldx, int64_t rows, int64_t cols, hipStream_t st) {
    auto go = [&](auto tpr, auto nch) {
        constexpr int L = tpr, C = nch;
        const int64_t n = (rows + 256 / L - 1) / (256 / L);
        hipLaunchKernelGGL((k_quantize<T, L, C>), dim3((unsigned)(n < 16384 ? n : 16384)), dim3(256), 0, st, out, pitch, scale, (const T *)x, ldx, rows, cols);
        return check_launch("k_quantize");
    };
    using std::integral_constant;
    const int64_t ch = (pitch + Vec<T>::N - 1) / Vec<T>::N;
    if (ch <= 16) return go(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    if (ch <= 64) return go(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    if (ch <= 128) return go(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    if (ch <= 256) return go(integral_constant<int, 64>{}, integral_constant<int, 4>{});
    if (ch <= 512) return go(integral_constant<int, 64>{}, integral_constant<int, 8>{});
    return go(integral_constant<int, 64>{}, integral_constant<int, 0>{});
}

}  // namespace mnr

using namespace mnr;

extern "C" int mnr_quantize_rows(int8_t *values_dev, int64_t pitch, float *scale_dev, const void *x_dev, int64_t ldx, int64_t rows, int64_t cols,
                                 int type, void *stream) {
    MNR_REQUIRE(type_ok(type), "unknown element type passed to mnr_quantize_rows");
    MNR_REQUIRE(rows >= 0 && rows < (1ll << 31) && cols >= 1 && cols <= (1 << 24), "mnr_quantize_rows needs 0 <= rows < 2^31 and 1 <= cols <= 2^24");
    MNR_REQUIRE(pitch >= cols && pitch % 16 == 0, "the pitch of mnr_quantize_rows is a multiple of 16 and holds a row");
    if (rows == 0) return MNR_OK;
    MNR_REQUIRE(values_dev && scale_dev && x_dev, "null pointer passed to mnr_quantize_rows");
    MNR_REQUIRE((reinterpret_cast<uintptr_t>(values_dev) & 15) == 0, "the values of mnr_quantize_rows start at a multiple of 16 bytes");
    MNR_REQUIRE(rows == 1 || ldx >= cols, "row pitch smaller than a row passed to mnr_quantize_rows");
    hipStream_t st = as_stream(stream);
    if (type == MNR_F32) return quantize<float>(values_dev, pitch, scale_dev, x_dev, ldx, rows, cols, st);
    if (type == MNR_F16) return quantize<f16_t>(values_dev, pitch, scale_dev, x_dev, ldx, rows, cols, st);
    return quantize<bf16_t>(values_dev, pitch, scale_dev, x_dev, ldx, rows, cols, st);
}

extern "C" size_t mnr_int8_product_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    (void)m; (void)n; (void)k;
    return 0;
}

extern "C" int mnr_int8_product(void *y_dev, int64_t ldy, const int8_t *a_dev, int64_t lda, const float *a_scale_dev, const int8_t *b_dev, int64_t ldb,
                                const float *b_scale_dev, const float *bias_dev, int64_t m, int64_t n, int64_t k, int act, int type,
                                void *workspace_dev, size_t workspace_bytes, void *stream) {
    MNR_REQUIRE(type_ok(type), "unknown element type passed to mnr_int8_product");
    MNR_REQUIRE(act == 0 || act == 1, "the activation of mnr_int8_product is 0 (none) or 1 (ReLU)");
    MNR_REQUIRE(m >= 0 && n >= 0 && m < (1ll << 31) && n < (1ll << 31), "mnr_int8_product needs 0 <= m, n < 2^31");
    MNR_REQUIRE(k >= 1 && k <= 131071, "mnr_int8_product needs 1 <= k <= 131071: longer sums may leave int32");
    if (m == 0 || n == 0) return MNR_OK;
    MNR_REQUIRE(y_dev && a_dev && a_scale_dev && b_dev && b_scale_dev, "null pointer passed to mnr_int8_product");
    const int64_t k16 = (k + 15) / 16 * 16;
    MNR_REQUIRE(((reinterpret_cast<uintptr_t>(a_dev) | reinterpret_cast<uintptr_t>(b_dev)) & 15) == 0 && lda % 16 == 0 && ldb % 16 == 0,
                "a and b of mnr_int8_product start at multiples of 16 bytes, with pitches that are multiples of 16");
    MNR_REQUIRE((m == 1 || lda >= k16) && (n == 1 || ldb >= k16) && (m == 1 || ldy >= n), "row pitch smaller than a row passed to mnr_int8_product");
    MNR_REQUIRE(workspace_bytes >= mnr_int8_product_workspace_bytes(m, n, k), "mnr_int8_product needs %zu bytes of workspace",
                mnr_int8_product_workspace_bytes(m, n, k));
    (void)workspace_dev;
    const ProductArgs p{y_dev, ldy, a_dev, lda, a_scale_dev, b_dev, ldb, b_scale_dev, bias_dev, m, n, k, act};
    hipStream_t st = as_stream(stream);
    if (type == MNR_F32) return product<float>(p, st);
    if (type == MNR_F16) return product<f16_t>(p, st);
    return product<bf16_t>(p, st);
}
