// embedding.hip -- table lookup with a scale, and the table's gradient by sorted indices.
//
//   out[r] = scale table[idx[r]]             grad[v] = scale sum_{r : idx[r] = v} dy[r]
//
// The lookup is bound by HBM: 16 bytes per lane wherever the row starts.  The gradient sorts the rows by index (row_sort.hip, stable; the
// sort's first launch clears the gradient) and walks the sorted order in tiles of 16 rows: a lane group keeps its columns' fp32 sum of
// the run it is in, and writes it once when the index changes.  A run that crosses tiles leaves one fp32 sum per tile, joined by
// k_emb_join.  No atomics: inside a tile rows are added in row order, tiles in interleaved phases that width, type and the run's length
// fix, so the same inputs give the same bits.  What bounds the gradient is the sort and the joins, not its bytes: 196608 rows of 48 fp32
// columns in runs of 192 take 11.5 us for the lookup, 22 to sort, 8 for the sums and 15 for the joins; 65521 rows of 512 bf16 columns,
// skewed so that long runs hold most of them, 19, 35, 17 and 24 us.
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

constexpr int EMB_TILE = 16;                           // sorted rows of a tile: all of them in flight at once (64 registers)

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

template <class T>
__device__ __forceinline__ void store_sum(float *p, const float (&v)[Vec<T>::N], int n) {
#pragma unroll
    for (int i = 0; i < Vec<T>::N; i += 4) store_part<float>(p + i, reinterpret_cast<const float (&)[4]>(v[i]), n - i);
}

// `head[t]`: the sum of tile t's first run where that run began in an earlier tile; `tail[t]`: of its last run where that run began in
// t and goes on behind it
template <class T, int LPR>
__global__ __launch_bounds__(256) void k_emb_sum(void *__restrict__ grad, int grad_f32, float *__restrict__ head, float *__restrict__ tail,
                                                 const T *__restrict__ dy, int64_t ldy, const int32_t *__restrict__ keys,
                                                 const int32_t *__restrict__ order, int64_t n, int width, int64_t padding, float scale) {
    constexpr int V = Vec<T>::N, GROUPS = 256 / LPR, EACH = (EMB_TILE + LPR - 1) / LPR;
    const int64_t tile = (int64_t)blockIdx.x * GROUPS + threadIdx.x / LPR, p0 = tile * EMB_TILE;
    const int t = threadIdx.x % LPR, base = (threadIdx.x & 63) - t;
    const int c = ((int)blockIdx.y * LPR + t) * V, m = width - c;
    const int live = p0 >= n ? 0 : (n - p0 < EMB_TILE ? (int)(n - p0) : EMB_TILE);
    // the group's lanes fetch the tile's keys and rows, one or two each, and hand them round
    int kk[EACH], oo[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int u = e * LPR + t;
        kk[e] = u < live ? keys[p0 + u] : -1;
        oo[e] = u < live ? order[p0 + u] : 0;
    }
    const int before = live && p0 > 0 ? keys[p0 - 1] : -1, behind = live == EMB_TILE && p0 + EMB_TILE < n ? keys[p0 + EMB_TILE] : -1;
    typename Vec<T>::raw v[EMB_TILE];
#pragma unroll
    for (int u = 0; u < EMB_TILE; ++u) {
        const int64_t row = __shfl(oo[u / LPR], base + u % LPR);
        v[u] = load_raw<T>(dy + row * ldy + c, u < live ? m : 0);
    }
    int cur = __shfl(kk[0], base);
    bool first = live && before == cur;                // the run began before this tile
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll
    for (int u = 0; u < EMB_TILE; ++u) {
        const int k = __shfl(kk[u / LPR], base + u % LPR);
        if (u < live && k != cur) {
            if (first) store_sum<T>(head + tile * width + c, acc, m);
            else if (cur != padding && m > 0) emb_write<T>(grad, (int64_t)cur * width + c, acc, m, scale, grad_f32);
            first = false;
            cur = k;
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] += (float)v[u][i];
    }
    if (!live || m <= 0) return;
    if (first || behind == cur) store_sum<T>((first ? head : tail) + tile * width + c, acc, m);
    else if (cur != padding) emb_write<T>(grad, (int64_t)cur * width + c, acc, m, scale, grad_f32);
}

// The tile in which a run begins that goes on behind it owns the run: tail[t] + head[t + 1] + ... + head[the tile of its end].  Runs of up
// to EMB_SHORT more tiles: a wave per tile.  Longer ones: workgroups of their own (blockIdx.y > 0) that look over 64 tiles at once and
// add a run up with 8 lanes across and 32 phases, the columns spread over blockIdx.y: a run over a sixth of 65521 rows (676 tiles of 512
// columns) took 77 us with one workgroup of 4 phases.
constexpr int EMB_SHORT = 16, EMB_LOOK = 64;

// head[u0], head[u0 + step] ... up to head[last], added to acc
template <class T>
__device__ __forceinline__ void emb_add_heads(float (&acc)[Vec<T>::N], const float *head, int64_t u0, int64_t step, int64_t last, int width, int c, int m) {
#pragma unroll 4
    for (int64_t u = u0; u <= last; u += step)
#pragma unroll
        for (int i = 0; i < Vec<T>::N; i += 4) {
            float v[4];
            load_part<float>(v, head + u * width + c + i, m - i);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i + j] += v[j];
        }
}

// the key of the run that tile t owns, -1 if it owns none; `further`: whether the run goes on behind tile t + EMB_SHORT
__device__ __forceinline__ int emb_owned(const int32_t *keys, int64_t t, int64_t n, int64_t padding, bool &further) {
    const int64_t p0 = t * EMB_TILE, p1 = p0 + EMB_TILE, far = p1 + EMB_SHORT * EMB_TILE;
    further = false;
    if (p1 >= n) return -1;
    const int k = keys[p1 - 1], next = keys[p1], first = keys[p0], before = p0 > 0 ? keys[p0 - 1] : -1, there = far < n ? keys[far] : -1;
    if (next != k || k == padding || (first == k && before == k)) return -1;
    further = there == k;
    return k;
}

template <class T, int LPR>
__global__ __launch_bounds__(256) void k_emb_join(void *__restrict__ grad, int grad_f32, const float *__restrict__ head,
                                                  const float *__restrict__ tail, const int32_t *__restrict__ keys, int64_t n, int width,
                                                  int64_t padding, float scale, int short_y) {
    constexpr int V = Vec<T>::N;
    __shared__ float lds[256 * V];
    __shared__ int keys_of[EMB_LOOK];
    const int64_t tiles = (n + EMB_TILE - 1) / EMB_TILE;
    if ((int)blockIdx.y < short_y) {
        constexpr int WPH = 64 / LPR;
        const int lane = threadIdx.x % LPR, ph = (threadIdx.x & 63) / LPR;
        const int c = ((int)blockIdx.y * LPR + lane) * V, m = width - c;
        float *mine = lds + (threadIdx.x >> 6) * 64 * V;                     // [WPH][LPR * V] of this wave
        for (int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); t < tiles - 1; t += (int64_t)gridDim.x * 4) {
            bool further;
            const int k = emb_owned(keys, t, n, padding, further);
            if (k < 0 || further) continue;                                  // (the whole wave alike)
            // lane i: does the run leave tile t + 1 + i?  The first that it leaves is its last
            const int64_t mark = (t + 2 + (threadIdx.x & 63)) * EMB_TILE;
            const int more = __ffsll((unsigned long long)__ballot(mark >= n || keys[mark < n ? mark : n - 1] != k));
            float acc[V];
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = 0.f;
            if (ph == 0) emb_add_heads<T>(acc, tail, t, 1, t, width, c, m);
            emb_add_heads<T>(acc, head, t + 1 + ph, WPH, t + more, width, c, m);
            if constexpr (WPH > 1) {
                wave_sync();
#pragma unroll
                for (int i = 0; i < V; ++i) mine[ph * LPR * V + lane * V + i] = acc[i];
                wave_sync();
                if (ph == 0)
                    for (int q = 1; q < WPH; ++q)
#pragma unroll
                        for (int i = 0; i < V; ++i) acc[i] += mine[q * LPR * V + lane * V + i];
            }
            if (ph == 0 && m > 0) emb_write<T>(grad, (int64_t)k * width + c, acc, m, scale, grad_f32);
        }
        return;
    }
    constexpr int PH = 32;
    const int lane = threadIdx.x % 8, ph = threadIdx.x / 8;
    const int c = (((int)blockIdx.y - short_y) * 8 + lane) * V, m = width - c;
    for (int64_t b0 = (int64_t)blockIdx.x * EMB_LOOK; b0 < tiles - 1; b0 += (int64_t)gridDim.x * EMB_LOOK) {
        __syncthreads();
        bool further = false;
        int own = -1;
        if (threadIdx.x < EMB_LOOK) own = emb_owned(keys, b0 + threadIdx.x, n, padding, further);
        if (threadIdx.x < EMB_LOOK) keys_of[threadIdx.x] = further ? own : -1;
        if (!__syncthreads_or(further)) continue;
        for (int o = 0; o < EMB_LOOK; ++o) {
            const int k = keys_of[o];
            if (k < 0) continue;                                             // (the whole workgroup alike)
            const int64_t t = b0 + o;
            // first place behind the run, in [lo, hi]: 256 probes at a time (each place before it holds k, none behind it)
            int64_t lo = (t + 1 + EMB_SHORT) * EMB_TILE + 1, hi = n;
            while (lo < hi) {
                const int64_t each = (hi - lo + 255) / 256, at = lo + each * threadIdx.x;
                const int64_t in = __syncthreads_count(at < hi && keys[at < hi ? at : lo] == k);         // probes inside the run
                if (in == 0) { hi = lo; break; }
                const int64_t upto = lo + each * in;
                lo += each * (in - 1) + 1;
                hi = upto < hi ? upto : hi;
            }
            const int64_t last = (hi - 1) / EMB_TILE;
            float acc[V];
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = 0.f;
            if (ph == 0) emb_add_heads<T>(acc, tail, t, 1, t, width, c, m);
            emb_add_heads<T>(acc, head, t + 1 + ph, PH, last, width, c, m);
            __syncthreads();                                                 // the last run's sums have been read
#pragma unroll
            for (int i = 0; i < V; ++i) lds[ph * 8 * V + lane * V + i] = acc[i];
            __syncthreads();
            if (ph == 0 && m > 0) {
                for (int q = 1; q < PH; ++q)
#pragma unroll
                    for (int i = 0; i < V; ++i) acc[i] += lds[q * 8 * V + lane * V + i];
                emb_write<T>(grad, (int64_t)k * width + c, acc, m, scale, grad_f32);
            }
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
    const int64_t halves = src.n_keys * width * (grad_f32 ? 2 : (int64_t)sizeof(T) / 2);
    const SortExtras clear{(uint32_t *)grad, halves / 2, (int)(halves % 2), nullptr};
    if (rows == 0) return clear_words(clear, st);
    const int64_t tiles = emb_tiles(rows);
    int32_t *order = reinterpret_cast<int32_t *>(ws), *keys = order + rows;
    float *head = reinterpret_cast<float *>(keys + rows), *tail = head + tiles * width;
    const int rc = sort_rows(src, rows, order, keys, tail + tiles * width, clear, st);
    if (rc != MNR_OK) return rc;
    return emb_lanes(width, Vec<T>::N, [&](auto lpr) {
        constexpr int L = lpr;
        const unsigned gy = (unsigned)((width + L * Vec<T>::N - 1) / (L * Vec<T>::N));
        const int64_t per = 256 / L, joins = (tiles - 1 + 3) / 4;
        hipLaunchKernelGGL((k_emb_sum<T, L>), dim3((unsigned)((tiles + per - 1) / per), gy), dim3(256), 0, st, grad, grad_f32, head, tail, (const T *)dy,
                           ldy, keys, order, rows, width, padding, scale);
        const unsigned gl = tiles > EMB_SHORT ? (unsigned)((width + 8 * Vec<T>::N - 1) / (8 * Vec<T>::N)) : 0;
        if (tiles > 1)
            hipLaunchKernelGGL((k_emb_join<T, L>), dim3((unsigned)(joins < 1024 ? joins : 1024), gy + gl), dim3(256), 0, st, grad, grad_f32, head, tail, keys,
                               rows, width, padding, scale, (int)gy);
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
