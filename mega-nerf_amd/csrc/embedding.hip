// embedding.hip -- table lookup with a scale, and the table's gradient by sorted indices.
//
//   out[r] = scale table[idx[r]]             grad[v] = scale sum_{r : idx[r] = v} dy[r]
//
// Bound by HBM.  The lookup reads 16 bytes per lane wherever the row starts.  The gradient sorts the rows by index (row_sort.hip,
// stable) and walks the sorted order in tiles: a lane group keeps its columns' fp32 sum of the run it is in, and writes it once when
// the index changes.  A run that crosses tiles leaves one fp32 sum per tile, joined by k_emb_join in tile order.  No atomics: sums
// are in row order, the same bits every time, and a popular index costs what an unpopular one does.
#include "row_sort.h"

namespace mnr {

template <class T, int LPR>
__global__ __launch_bounds__(256) void k_emb_fwd(T *__restrict__ out, int64_t ldo, const T *__restrict__ table, int64_t ldt, int width, KeySource src,
                                                 float scale, int64_t rows) {
    constexpr int V = Vec<T>::N, GROUPS = 256 / LPR, R = 4;
    const int lane = threadIdx.x % LPR;
    const int64_t r0 = (int64_t)blockIdx.x * (GROUPS * R) + threadIdx.x / LPR;
    int64_t k[R];
#pragma unroll
    for (int j = 0; j < R; ++j) k[j] = r0 + j * GROUPS < rows ? src(r0 + j * GROUPS) : 0;
    for (int c = lane * V; c < width; c += LPR * V) {
        float v[R][V];
#pragma unroll
        for (int j = 0; j < R; ++j) load_part<T>(v[j], table + k[j] * ldt + c, r0 + j * GROUPS < rows ? width - c : 0);
#pragma unroll
        for (int j = 0; j < R; ++j) {
            if (r0 + j * GROUPS >= rows) continue;
#pragma unroll
            for (int i = 0; i < V; ++i) v[j][i] *= scale;
            store_part<T>(out + (r0 + j * GROUPS) * ldo + c, v[j], width - c);
        }
    }
}

constexpr int EMB_TILE = 32, EMB_STEP = 8;             // sorted rows of a tile; rows in flight

__global__ __launch_bounds__(256) void k_emb_zero(uint32_t *__restrict__ p, int64_t words, int tail_halves) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) p[i] = 0;
    if (tail_halves && blockIdx.x == 0 && threadIdx.x == 0) reinterpret_cast<uint16_t *>(p + words)[0] = 0;
}

template <class T>
__device__ __forceinline__ void emb_write(void *grad, int64_t at, float (&v)[Vec<T>::N], int n, float scale, int grad_f32) {
    constexpr int V = Vec<T>::N;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] *= scale;
    if (grad_f32) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) reinterpret_cast<float *>(grad)[at + i] = v[i];
    } else {
        store_part<T>(reinterpret_cast<T *>(grad) + at, v, n);
    }
}

// `head[t]`: the sum of tile t's first run where that run began in an earlier tile; `tail[t]`: of its last run where that run began in
// t and goes on behind it
template <class T, int LPR>
__global__ __launch_bounds__(256) void k_emb_sum(void *__restrict__ grad, int grad_f32, float *__restrict__ head, float *__restrict__ tail,
                                                 const T *__restrict__ dy, int64_t ldy, const int32_t *__restrict__ keys,
                                                 const int32_t *__restrict__ order, int64_t n, int width, int64_t padding, float scale) {
    constexpr int V = Vec<T>::N, GROUPS = 256 / LPR;
    const int64_t tile = (int64_t)blockIdx.x * GROUPS + threadIdx.x / LPR, p0 = tile * EMB_TILE;
    const int c = ((int)blockIdx.y * LPR + (int)(threadIdx.x % LPR)) * V, m = width - c;
    if (p0 >= n || m <= 0) return;
    const int64_t p1 = p0 + EMB_TILE < n ? p0 + EMB_TILE : n;
    int cur = keys[p0];
    bool first = p0 > 0 && keys[p0 - 1] == cur;        // the run began before this tile
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    for (int64_t p = p0; p < p1; p += EMB_STEP) {
        float v[EMB_STEP][V];
        int k[EMB_STEP];
#pragma unroll
        for (int u = 0; u < EMB_STEP; ++u) {
            const bool in = p + u < p1;
            k[u] = in ? keys[p + u] : cur;
            load_part<T>(v[u], dy + (in ? (int64_t)order[p + u] : 0) * ldy + c, in ? m : 0);
        }
#pragma unroll
        for (int u = 0; u < EMB_STEP; ++u) {
            if (p + u >= p1) break;
            if (k[u] != cur) {
                if (first) store_part<float>(head + tile * width + c, reinterpret_cast<float (&)[4]>(acc[0]), m);
                if constexpr (V == 8) { if (first) store_part<float>(head + tile * width + c + 4, reinterpret_cast<float (&)[4]>(acc[4]), m - 4); }
                if (!first && cur != padding) emb_write<T>(grad, (int64_t)cur * width + c, acc, m, scale, grad_f32);
                first = false;
                cur = k[u];
#pragma unroll
                for (int i = 0; i < V; ++i) acc[i] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += v[u][i];
        }
    }
    const bool goes_on = p1 < n && keys[p1] == cur;
    if (first || goes_on) {
        float *dst = (first ? head : tail) + tile * width + c;
#pragma unroll
        for (int i = 0; i < V; i += 4) store_part<float>(dst + i, reinterpret_cast<float (&)[4]>(acc[i]), m - i);
    } else if (cur != padding) {
        emb_write<T>(grad, (int64_t)cur * width + c, acc, m, scale, grad_f32);
    }
}

// The tile in which a run begins that goes on behind it owns the run: tail[t] + head[t + 1] + ... + head[the tile of its end]
template <class T, int LPR>
__global__ __launch_bounds__(256) void k_emb_join(void *__restrict__ grad, int grad_f32, const float *__restrict__ head,
                                                  const float *__restrict__ tail, const int32_t *__restrict__ keys, int64_t n, int width,
                                                  int64_t padding, float scale) {
    constexpr int V = Vec<T>::N, PH = 256 / LPR;
    __shared__ float lds[PH > 1 ? PH : 1][LPR * V];
    const int lane = threadIdx.x % LPR, ph = threadIdx.x / LPR;
    const int c = ((int)blockIdx.y * LPR + lane) * V, m = width - c;
    for (int64_t t = blockIdx.x; (t + 1) * EMB_TILE < n; t += gridDim.x) {
        const int64_t p0 = t * EMB_TILE, p1 = p0 + EMB_TILE;
        const int k = keys[p1 - 1];
        if (keys[p1] != k || k == padding || (p0 > 0 && keys[p0] == k && keys[p0 - 1] == k)) continue;      // (the whole workgroup alike)
        int64_t lo = p1, hi = n;                       // first place behind the run
        while (lo < hi) {
            const int64_t mid = (lo + hi) >> 1;
            if (keys[mid] == k) lo = mid + 1; else hi = mid;
        }
        const int64_t last = (lo - 1) / EMB_TILE;
        float acc[V], v[4];
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            load_part<float>(v, tail + t * width + c + i, ph == 0 ? m - i : 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i + j] = v[j];
        }
        for (int64_t u = t + 1 + ph; u <= last; u += PH)
#pragma unroll
            for (int i = 0; i < V; i += 4) {
                load_part<float>(v, head + u * width + c + i, m - i);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i + j] += v[j];
            }
        __syncthreads();                               // the last run's sums have been read
#pragma unroll
        for (int i = 0; i < V; ++i) lds[ph][lane * V + i] = acc[i];
        __syncthreads();
        if (ph == 0) {
            for (int q = 1; q < PH; ++q)
#pragma unroll
                for (int i = 0; i < V; ++i) acc[i] += lds[q][lane * V + i];
            if (m > 0) emb_write<T>(grad, (int64_t)k * width + c, acc, m, scale, grad_f32);
        }
    }
}

template <class F> static int emb_lanes(int64_t width, int v, F &&f) {
    using std::integral_constant;
    const int64_t ch = (width + v - 1) / v;
    if (ch <= 8) return f(integral_constant<int, 8>{});
    if (ch <= 16) return f(integral_constant<int, 16>{});
    if (ch <= 32) return f(integral_constant<int, 32>{});
    return f(integral_constant<int, 64>{});
}

template <class T>
static int emb_forward(void *out, int64_t ldo, const void *table, int64_t ldt, int width, const KeySource &src, float scale, int64_t rows,
                       hipStream_t st) {
    return emb_lanes(width, Vec<T>::N, [&](auto lpr) {
        const int64_t per = 256 / lpr * 4;
        hipLaunchKernelGGL((k_emb_fwd<T, lpr>), dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, st, (T *)out, ldo, (const T *)table, ldt, width,
                           src, scale, rows);
        return check_launch("k_emb_fwd");
    });
}

static int64_t emb_tiles(int64_t n) { return (n + EMB_TILE - 1) / EMB_TILE; }

template <class T>
static int emb_backward(void *grad, int grad_f32, const void *dy, int64_t ldy, int width, const KeySource &src, int64_t rows, int64_t padding,
                        float scale, char *ws, hipStream_t st) {
    const int64_t words = src.n_keys * width * (grad_f32 ? 4 : (int64_t)sizeof(T)) / 4;
    const int64_t zb = (words + 1023) / 1024;
    hipLaunchKernelGGL(k_emb_zero, dim3((unsigned)(zb < 1 ? 1 : (zb > 4096 ? 4096 : zb))), dim3(256), 0, st, (uint32_t *)grad, words,
                       !grad_f32 && sizeof(T) == 2 && (src.n_keys * width) % 2 ? 1 : 0);
    int rc = check_launch("k_emb_zero");
    if (rc != MNR_OK || rows == 0) return rc;
    const int64_t tiles = emb_tiles(rows);
    int32_t *order = reinterpret_cast<int32_t *>(ws), *keys = order + rows;
    float *head = reinterpret_cast<float *>(keys + rows), *tail = head + tiles * width;
    rc = sort_rows(src, rows, order, keys, tail + tiles * width, st);
    if (rc != MNR_OK) return rc;
    return emb_lanes(width, Vec<T>::N, [&](auto lpr) {
        constexpr int L = lpr;
        const unsigned gy = (unsigned)((width + L * Vec<T>::N - 1) / (L * Vec<T>::N));
        const int64_t per = 256 / L;
        hipLaunchKernelGGL((k_emb_sum<T, L>), dim3((unsigned)((tiles + per - 1) / per), gy), dim3(256), 0, st, grad, grad_f32, head, tail, (const T *)dy,
                           ldy, keys, order, rows, width, padding, scale);
        if (tiles > 1)
            hipLaunchKernelGGL((k_emb_join<T, L>), dim3((unsigned)(tiles - 1 < 65536 ? tiles - 1 : 65536), gy), dim3(256), 0, st, grad, grad_f32, head, tail, keys, rows, width,
                               padding, scale);
        return check_launch("k_emb_sum / k_emb_join");
    });
}

}  // namespace mnr

using namespace mnr;

static bool emb_sizes_ok(int64_t rows, int64_t count, int64_t width) {
    return rows >= 0 && rows < (1ll << 31) && count >= 1 && count < (1ll << 31) && width >= 1 && width <= (1 << 20);
}

extern "C" int mnr_embedding_forward(void *out_dev, int64_t ldo, const void *table_dev, int64_t ldt, int64_t count, int64_t width,
                                     const void *idx_dev, int idx_type, float scale, int64_t rows, int type, void *stream) {
    MNR_REQUIRE(type_ok(type), "unknown element type passed to mnr_embedding_forward");
    MNR_REQUIRE(key_type_ok(idx_type), "indices of mnr_embedding_forward are int32, int64 or fp32");
    MNR_REQUIRE(emb_sizes_ok(rows, count, width), "mnr_embedding_forward needs 0 <= rows < 2^31, 1 <= count < 2^31, 1 <= width <= 2^20");
    if (rows == 0) return MNR_OK;
    MNR_REQUIRE(out_dev && table_dev && idx_dev, "null pointer passed to mnr_embedding_forward");
    MNR_REQUIRE((rows == 1 || ldo >= width) && (count == 1 || ldt >= width), "row pitch smaller than a row passed to mnr_embedding_forward");
    const KeySource src{idx_dev, idx_type, 0, count};
    hipStream_t st = as_stream(stream);
    if (type == MNR_F32) return emb_forward<float>(out_dev, ldo, table_dev, ldt, (int)width, src, scale, rows, st);
    if (type == MNR_F16) return emb_forward<f16_t>(out_dev, ldo, table_dev, ldt, (int)width, src, scale, rows, st);
    return emb_forward<bf16_t>(out_dev, ldo, table_dev, ldt, (int)width, src, scale, rows, st);
}

extern "C" size_t mnr_embedding_backward_workspace_bytes(int64_t rows, int64_t count, int64_t width) {
    if (!emb_sizes_ok(rows, count, width)) return 0;
    return (size_t)rows * 8 + (size_t)emb_tiles(rows) * width * 8 + sort_rows_bytes(rows, count) + 16;
}

extern "C" int mnr_embedding_backward(void *grad_dev, int grad_type, const void *dy_dev, int64_t ldy, const void *idx_dev, int idx_type,
                                      int64_t rows, int64_t count, int64_t width, int64_t padding_idx, float scale, int type,
                                      void *workspace_dev, size_t workspace_bytes, void *stream) {
    MNR_REQUIRE(type_ok(type) && (grad_type == type || grad_type == MNR_F32), "mnr_embedding_backward: the gradient is fp32 or of dy's type");
    MNR_REQUIRE(key_type_ok(idx_type), "indices of mnr_embedding_backward are int32, int64 or fp32");
    MNR_REQUIRE(emb_sizes_ok(rows, count, width), "mnr_embedding_backward needs 0 <= rows < 2^31, 1 <= count < 2^31, 1 <= width <= 2^20");
    MNR_REQUIRE(padding_idx >= -1 && padding_idx < count, "padding_idx of mnr_embedding_backward is a table row, or -1 for none");
    MNR_REQUIRE(grad_dev && (rows == 0 || (dy_dev && idx_dev)), "null pointer passed to mnr_embedding_backward");
    MNR_REQUIRE((reinterpret_cast<uintptr_t>(grad_dev) & 3) == 0, "the gradient of mnr_embedding_backward starts at a multiple of 4 bytes");
    MNR_REQUIRE(rows <= 1 || ldy >= width, "row pitch smaller than a row passed to mnr_embedding_backward");
    MNR_REQUIRE(rows == 0 || (workspace_dev && workspace_bytes >= mnr_embedding_backward_workspace_bytes(rows, count, width)),
                "mnr_embedding_backward needs %zu bytes of workspace", mnr_embedding_backward_workspace_bytes(rows, count, width));
    const KeySource src{idx_dev, idx_type, 0, count};
    hipStream_t st = as_stream(stream);
    char *ws = reinterpret_cast<char *>(workspace_dev);
    const int f32 = grad_type == MNR_F32;
    if (type == MNR_F32) return emb_backward<float>(grad_dev, f32, dy_dev, ldy, (int)width, src, rows, padding_idx, scale, ws, st);
    if (type == MNR_F16) return emb_backward<f16_t>(grad_dev, f32, dy_dev, ldy, (int)width, src, rows, padding_idx, scale, ws, st);
    return emb_backward<bf16_t>(grad_dev, f32, dy_dev, ldy, (int)width, src, rows, padding_idx, scale, ws, st);
}
