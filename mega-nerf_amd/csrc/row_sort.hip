// row_sort.hip -- stable sort of rows by a small integer key: counting passes over digits of at most 8 bits, lowest first.
//
// A pass puts row i at  base[digit] + (rows of earlier workgroups with that digit) + (earlier rows of this workgroup with it):
// k_sort_count counts digits per workgroup, k_sort_scan turns the counts into positions, k_sort_place ranks and writes.  Inside a
// wave a lane's rank is the number of lower lanes with its digit, from one ballot per bit.  Counts are whole numbers, so the order
// does not depend on which workgroup ran first; keys of b bits take ceil(b / 8) passes of equal width.  Up to 4096 rows one workgroup
// does all passes in LDS (one launch).  Traffic is 8 bytes a row and pass each way; at the sizes here (200 K rows) the passes cost
// their launches, not their bytes.
#include "row_sort.h"

namespace mnr {

constexpr int SORT_BLOCK = 256, SORT_ITEMS = 16, SORT_TILE = SORT_BLOCK * SORT_ITEMS, SORT_SMALL = 4096;

// lanes of this wave with the same digit as this lane (only lanes with `live` take part)
__device__ __forceinline__ uint64_t same_digit(int digit, int bits, bool live) {
    uint64_t m = __ballot(live);
    for (int b = 0; b < bits; ++b) {
        const uint64_t s = __ballot((digit >> b) & 1);
        m &= (digit >> b) & 1 ? s : ~s;
    }
    return m;
}

// this lane's place: counter[digit] before the wave's rows + its rank among them; counter[digit] moves on by the wave's rows
__device__ __forceinline__ int take_place(int *counter, int digit, int bits, bool live) {
    const uint64_t m = same_digit(digit, bits, live);
    const int lane = threadIdx.x & 63, first = m ? __ffsll((unsigned long long)m) - 1 : lane;
    int at = 0;
    if (live && lane == first) at = atomicAdd(counter + digit, __popcll(m));
    at = __shfl(at, first);
    return at + __popcll(m & ((1ull << lane) - 1));
}

__global__ __launch_bounds__(512) void k_sort_small(KeySource src, int n, int bits_per, int passes, int32_t *__restrict__ order,
                                                    int32_t *__restrict__ keys_out) {
    __shared__ int key[2][SORT_SMALL];
    __shared__ uint16_t pos[2][SORT_SMALL];
    __shared__ int count[8][256];
    __shared__ int wave_total[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int per = ((n + 7) / 8 + 63) / 64 * 64;                    // rows of a wave, whole steps
    const int i0 = wave * per, i1 = min(n, i0 + per);
    for (int i = threadIdx.x; i < n; i += 512) { key[0][i] = src(i); pos[0][i] = (uint16_t)i; }
    const int digits = 1 << bits_per, mask = digits - 1;
    for (int p = 0; p < passes; ++p) {
        const int shift = p * bits_per, in = p & 1, out = in ^ 1;
        for (int d = threadIdx.x; d < 8 * 256; d += 512) (&count[0][0])[d] = 0;
        __syncthreads();
        for (int i = i0 + lane; i < i1; i += 64) atomicAdd(&count[wave][(key[in][i] >> shift) & mask], 1);
        __syncthreads();
        // thread d: rows of digit d, then the running sum over digits (4 waves of 64 digits)
        const int d = threadIdx.x;
        int total = 0, sum = 0;
        if (d < 256) {
            for (int w = 0; w < 8; ++w) total += count[w][d];
            sum = total;
            for (int o = 1; o < 64; o <<= 1) {
                const int u = __shfl_up(sum, o);
                if (lane >= o) sum += u;
            }
            if (lane == 63) wave_total[wave] = sum;
        }
        __syncthreads();
        if (d < 256) {
            int at = sum - total;
            for (int w = 0; w < wave; ++w) at += wave_total[w];
            for (int w = 0; w < 8; ++w) {
                const int c = count[w][d];
                count[w][d] = at;
                at += c;
            }
        }
        __syncthreads();
        for (int i = i0; i < i0 + per; i += 64) {
            const bool live = i + lane < i1;
            const int k = live ? key[in][i + lane] : 0;
            const int at = take_place(count[wave], (k >> shift) & mask, bits_per, live);
            if (live) { key[out][at] = k; pos[out][at] = pos[in][i + lane]; }
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < n; i += 512) {
        order[i] = pos[passes & 1][i];
        keys_out[i] = key[passes & 1][i];
    }
}

// hist[digit][workgroup]
__global__ __launch_bounds__(SORT_BLOCK) void k_sort_count(KeySource src, const int32_t *__restrict__ keys, int64_t n, int shift, int digits,
                                                           int32_t *__restrict__ hist) {
    __shared__ int count[256];
    count[threadIdx.x] = 0;
    __syncthreads();
    const int64_t b0 = (int64_t)blockIdx.x * SORT_TILE;
#pragma unroll 4
    for (int j = 0; j < SORT_ITEMS; ++j) {
        const int64_t i = b0 + j * SORT_BLOCK + threadIdx.x;
        if (i < n) atomicAdd(&count[((keys ? keys[i] : src(i)) >> shift) & (digits - 1)], 1);
    }
    __syncthreads();
    if ((int)threadIdx.x < digits) hist[(int64_t)threadIdx.x * gridDim.x + blockIdx.x] = count[threadIdx.x];
}

// one workgroup per digit: its counts -> rows of that digit in earlier workgroups; total[digit]
__global__ __launch_bounds__(256) void k_sort_scan(int32_t *__restrict__ hist, int blocks, int32_t *__restrict__ total) {
    __shared__ int part[4];
    int32_t *row = hist + (int64_t)blockIdx.x * blocks;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int run = 0;
    for (int b0 = 0; b0 < blocks; b0 += 256) {
        const int b = b0 + threadIdx.x, v = b < blocks ? row[b] : 0;
        int sum = v;
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(sum, o);
            if (lane >= o) sum += u;
        }
        __syncthreads();
        if (lane == 63) part[wave] = sum;
        __syncthreads();
        int before = run;
        for (int w = 0; w < wave; ++w) before += part[w];
        if (b < blocks) row[b] = before + sum - v;
        run += part[0] + part[1] + part[2] + part[3];
    }
    if (threadIdx.x == 0) total[blockIdx.x] = run;
}

__global__ __launch_bounds__(SORT_BLOCK) void k_sort_place(KeySource src, const int32_t *__restrict__ keys, const int32_t *__restrict__ rows,
                                                           int64_t n, int shift, int bits, const int32_t *__restrict__ hist,
                                                           const int32_t *__restrict__ total, int32_t *__restrict__ keys_out,
                                                           int32_t *__restrict__ rows_out) {
    __shared__ int count[4][256];
    __shared__ int part[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, digits = 1 << bits, mask = digits - 1;
    for (int d = threadIdx.x; d < 4 * 256; d += SORT_BLOCK) (&count[0][0])[d] = 0;
    __syncthreads();
    const int64_t i0 = (int64_t)blockIdx.x * SORT_TILE + wave * (SORT_TILE / 4) + lane;
    int k[SORT_ITEMS];
#pragma unroll
    for (int j = 0; j < SORT_ITEMS; ++j) {
        const int64_t i = i0 + j * 64;
        k[j] = i < n ? (keys ? keys[i] : src(i)) : 0;
        if (i < n) atomicAdd(&count[wave][(k[j] >> shift) & mask], 1);
    }
    const int d = threadIdx.x, t = d < digits ? total[d] : 0;
    int sum = t;
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(sum, o);
        if (lane >= o) sum += u;
    }
    if (lane == 63) part[wave] = sum;
    __syncthreads();
    if (d < digits) {
        int at = sum - t + hist[(int64_t)d * gridDim.x + blockIdx.x];
        for (int w = 0; w < wave; ++w) at += part[w];
        for (int w = 0; w < 4; ++w) {
            const int c = count[w][d];
            count[w][d] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SORT_ITEMS; ++j) {
        const int64_t i = i0 + j * 64;
        const bool live = i < n;
        const int at = take_place(count[wave], (k[j] >> shift) & mask, bits, live);
        if (live) {
            keys_out[at] = k[j];
            rows_out[at] = rows ? rows[i] : (int32_t)i;
        }
    }
}

static int key_bits(int64_t n_keys) {                  // keys 0 .. n_keys
    int b = 1;
    while (((int64_t)1 << b) <= n_keys) ++b;
    return b;
}
static int64_t sort_blocks(int64_t n) { return (n + SORT_TILE - 1) / SORT_TILE; }

size_t sort_rows_bytes(int64_t n, int64_t n_keys) {
    (void)n_keys;
    if (n <= SORT_SMALL) return 0;
    return (size_t)(4 * n + 256 * sort_blocks(n) + 256) * sizeof(int32_t);
}

int sort_rows(const KeySource &src, int64_t n, int32_t *order, int32_t *keys_out, void *ws, hipStream_t st) {
    const int bits = key_bits(src.n_keys), passes = (bits + 7) / 8, per = (bits + passes - 1) / passes;
    if (n <= SORT_SMALL) {
        hipLaunchKernelGGL(k_sort_small, dim3(1), dim3(512), 0, st, src, (int)n, per, passes, order, keys_out);
        return check_launch("k_sort_small");
    }
    const int blocks = (int)sort_blocks(n);
    int32_t *buf = reinterpret_cast<int32_t *>(ws), *hist = buf + 4 * n, *total = hist + (int64_t)256 * blocks;
    const int32_t *ki = nullptr, *ri = nullptr;
    for (int p = 0; p < passes; ++p) {
        const bool last = p == passes - 1;
        int32_t *ko = last ? keys_out : buf + (p & 1) * 2 * n, *ro = last ? order : ko + n;
        hipLaunchKernelGGL(k_sort_count, dim3(blocks), dim3(SORT_BLOCK), 0, st, src, ki, n, p * per, 1 << per, hist);
        hipLaunchKernelGGL(k_sort_scan, dim3(1 << per), dim3(256), 0, st, hist, blocks, total);
        hipLaunchKernelGGL(k_sort_place, dim3(blocks), dim3(SORT_BLOCK), 0, st, src, ki, ri, n, p * per, per, hist, total, ko, ro);
        ki = ko;
        ri = ro;
    }
    return check_launch("k_sort_place");
}

}  // namespace mnr
