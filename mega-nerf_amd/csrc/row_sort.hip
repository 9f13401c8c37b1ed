// row_sort.hip -- stable sort of rows by a small integer key: counting passes over digits of at most 11 bits, lowest first.
//
// A pass puts row i at  base[digit] + (rows of earlier workgroups with that digit) + (earlier rows of this workgroup with it):
// k_sort_count counts digits per workgroup, k_sort_scan turns the counts into positions, k_sort_place ranks and writes.  Inside a
// wave a lane's rank is the number of lower lanes with its digit, from one ballot per bit.  Counts are whole numbers, so the order
// does not depend on which workgroup ran first.  Keys of b bits take ceil(b / 11) passes of equal width: 2048 counters a wave are 32 KB of
// LDS, and 2000 images sort in one pass (3 launches: 22 us for 196608 rows, two passes of 8 bits took 52).  Up to 4096 rows one workgroup
// does all passes in LDS (one launch).  At the sizes here the passes cost their launches and the ranking, not their bytes.
#include "row_sort.h"

namespace mnr {

constexpr int SORT_SMALL = 4096, SORT_MAX_BITS = 11, SORT_MAX_DIGITS = 1 << SORT_MAX_BITS;

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

// sum of v over this and lower lanes
__device__ __forceinline__ int scan_wave(int v) {
    const int lane = threadIdx.x & 63;
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(v, o);
        if (lane >= o) v += u;
    }
    return v;
}

__device__ __forceinline__ void clear_part(const SortExtras &x, int64_t worker, int64_t workers) {
    for (int64_t i = worker; i < x.words; i += workers) x.zero[i] = 0;
    if (x.half && worker == 0) reinterpret_cast<uint16_t *>(x.zero + x.words)[0] = 0;
}

// first place in the sorted keys that is not below c
__device__ __forceinline__ int64_t first_not_below(const int32_t *keys, int64_t n, int64_t c) {
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (keys[mid] < c) lo = mid + 1; else hi = mid;
    }
    return lo;
}

// workgroup 0 sorts; the others clear
__global__ __launch_bounds__(512) void k_sort_small(KeySource src, int n, int bits_per, int passes, int32_t *__restrict__ order,
                                                    int32_t *__restrict__ keys_out, SortExtras x) {
    if (blockIdx.x > 0) {
        clear_part(x, (int64_t)(blockIdx.x - 1) * 512 + threadIdx.x, (int64_t)(gridDim.x - 1) * 512);
        return;
    }
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
            sum = scan_wave(total);
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
    const int last = passes & 1;
    for (int i = threadIdx.x; i < n; i += 512) {
        order[i] = pos[last][i];
        keys_out[i] = key[last][i];
    }
    if (x.offsets)
        for (int64_t c = threadIdx.x; c <= src.n_keys; c += 512) x.offsets[c] = (int32_t)first_not_below(key[last], n, c);
}

// hist[workgroup][digit] for the first `blocks` workgroups; the others clear
__global__ __launch_bounds__(256) void k_sort_count(KeySource src, const int32_t *__restrict__ keys, int64_t n, int per_block, int blocks, int shift,
                                                    int digits, int32_t *__restrict__ hist, SortExtras x) {
    if ((int)blockIdx.x >= blocks) {
        clear_part(x, (int64_t)(blockIdx.x - blocks) * 256 + threadIdx.x, (int64_t)(gridDim.x - blocks) * 256);
        return;
    }
    __shared__ int count[SORT_MAX_DIGITS];
    for (int d = threadIdx.x; d < digits; d += 256) count[d] = 0;
    __syncthreads();
    const int64_t b0 = (int64_t)blockIdx.x * per_block, b1 = b0 + per_block < n ? b0 + per_block : n;
#pragma unroll 4
    for (int64_t i = b0 + threadIdx.x; i < b1; i += 256) atomicAdd(&count[((keys ? keys[i] : src(i)) >> shift) & (digits - 1)], 1);
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += 256) hist[(int64_t)blockIdx.x * digits + d] = count[d];
}

// 64 digits x 16 segments of workgroups per workgroup: counts -> rows of that digit in earlier workgroups; total[digit]
__global__ __launch_bounds__(1024) void k_sort_scan(int32_t *__restrict__ hist, int blocks, int digits, int32_t *__restrict__ total) {
    __shared__ int part[16][64];
    const int lane = threadIdx.x & 63, seg = threadIdx.x >> 6, d = blockIdx.x * 64 + lane;
    const int per = (blocks + 15) / 16, b0 = seg * per, b1 = min(blocks, b0 + per);
    int sum = 0;
    if (d < digits) {
#pragma unroll 4
        for (int b = b0; b < b1; ++b) sum += hist[(int64_t)b * digits + d];
    }
    part[seg][lane] = sum;
    __syncthreads();
    if (d >= digits) return;
    int at = 0;
    for (int s = 0; s < seg; ++s) at += part[s][lane];
    if (seg == 15) total[d] = at + sum;
#pragma unroll 4
    for (int b = b0; b < b1; ++b) {
        const int c = hist[(int64_t)b * digits + d];
        hist[(int64_t)b * digits + d] = at;
        at += c;
    }
}

__global__ __launch_bounds__(256) void k_sort_place(KeySource src, const int32_t *__restrict__ keys, const int32_t *__restrict__ rows, int64_t n,
                                                    int per_block, int shift, int bits, const int32_t *__restrict__ hist,
                                                    const int32_t *__restrict__ total, int32_t *__restrict__ keys_out,
                                                    int32_t *__restrict__ rows_out, int32_t *__restrict__ offsets) {
    extern __shared__ int count[];                     // [4][digits], 4 wave totals
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, digits = 1 << bits, mask = digits - 1;
    int *part = count + 4 * digits;
    for (int d = threadIdx.x; d < 4 * digits; d += 256) count[d] = 0;
    __syncthreads();
    int *mine = count + wave * digits;
    const int64_t i0 = (int64_t)blockIdx.x * per_block + wave * (per_block / 4), end = i0 + per_block / 4 < n ? i0 + per_block / 4 : n;
#pragma unroll 4
    for (int64_t i = i0 + lane; i < end; i += 64) atomicAdd(mine + (((keys ? keys[i] : src(i)) >> shift) & mask), 1);
    // the digits' bases: a thread sums up its digits / 256 (at least one) neighbours, the workgroup scans the sums
    const int per = digits >= 256 ? digits / 256 : 1, d0 = threadIdx.x * per;
    int t[SORT_MAX_DIGITS / 256], sum = 0;
#pragma unroll
    for (int j = 0; j < SORT_MAX_DIGITS / 256; ++j) {
        t[j] = j < per && d0 + j < digits ? total[d0 + j] : 0;
        sum += t[j];
    }
    const int upto = scan_wave(sum);
    if (lane == 63) part[wave] = upto;
    __syncthreads();
    int base = upto - sum;
    for (int w = 0; w < wave; ++w) base += part[w];
#pragma unroll
    for (int j = 0; j < SORT_MAX_DIGITS / 256; ++j) {
        const int d = d0 + j;
        if (j < per && d < digits) {
            if (offsets && blockIdx.x == 0 && d <= src.n_keys) offsets[d] = base;
            int at = base + hist[(int64_t)blockIdx.x * digits + d];
            for (int w = 0; w < 4; ++w) {
                const int c = count[w * digits + d];
                count[w * digits + d] = at;
                at += c;
            }
            base += t[j];
        }
    }
    __syncthreads();
    for (int64_t i = i0; i < i0 + per_block / 4; i += 64) {
        const bool live = i + lane < end;
        const int k = live ? (keys ? keys[i + lane] : src(i + lane)) : 0;
        const int at = take_place(mine, (k >> shift) & mask, bits, live);
        if (live) {
            keys_out[at] = k;
            rows_out[at] = rows ? rows[i + lane] : (int32_t)(i + lane);
        }
    }
}

__global__ __launch_bounds__(256) void k_sort_offsets(int32_t *__restrict__ offsets, const int32_t *__restrict__ keys, int64_t n, int64_t n_keys) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c <= n_keys) offsets[c] = (int32_t)first_not_below(keys, n, c);
}

__global__ __launch_bounds__(256) void k_clear(SortExtras x) { clear_part(x, (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256); }

static int key_bits(int64_t n_keys) {                  // keys 0 .. n_keys
    int b = 1;
    while (((int64_t)1 << b) <= n_keys) ++b;
    return b;
}
// rows of a workgroup: 1024, doubled from 2^20 rows on, so that there are at most 1024 sets of counters.  (65521 rows are 64 workgroups and
// 196608 rows 192, on 256 CUs; smaller shares were not measured.)
static int sort_per_block(int64_t n) {
    int64_t per = 1024;
    while ((n + per - 1) / per > 1024) per *= 2;
    return (int)per;
}
static int64_t sort_blocks(int64_t n) { return (n + sort_per_block(n) - 1) / sort_per_block(n); }
static unsigned clear_blocks(const SortExtras &x) {
    if (!x.words && !x.half) return 0;
    const int64_t n = (x.words + 2047) / 2048;
    return (unsigned)(n < 1 ? 1 : (n > 2048 ? 2048 : n));
}

size_t sort_rows_bytes(int64_t n, int64_t n_keys) {
    if (n <= SORT_SMALL) return 0;
    const int bits = key_bits(n_keys), passes = (bits + SORT_MAX_BITS - 1) / SORT_MAX_BITS, per = (bits + passes - 1) / passes;
    return (size_t)((passes > 1 ? 4 * n : 0) + (sort_blocks(n) + 1) * ((int64_t)1 << per)) * sizeof(int32_t);
}

int clear_words(const SortExtras &x, hipStream_t st) {
    if (!clear_blocks(x)) return MNR_OK;
    hipLaunchKernelGGL(k_clear, dim3(clear_blocks(x)), dim3(256), 0, st, x);
    return check_launch("k_clear");
}

int sort_rows(const KeySource &src, int64_t n, int32_t *order, int32_t *keys_out, void *ws, const SortExtras &x, hipStream_t st) {
    const int bits = key_bits(src.n_keys);
    if (n <= SORT_SMALL) {
        const int passes = (bits + 7) / 8, per = (bits + passes - 1) / passes;
        hipLaunchKernelGGL(k_sort_small, dim3(1 + clear_blocks(x)), dim3(512), 0, st, src, (int)n, per, passes, order, keys_out, x);
        return check_launch("k_sort_small");
    }
    const int passes = (bits + SORT_MAX_BITS - 1) / SORT_MAX_BITS, per = (bits + passes - 1) / passes, digits = 1 << per;
    const int blocks = (int)sort_blocks(n), rows = sort_per_block(n);
    int32_t *buf = reinterpret_cast<int32_t *>(ws), *hist = buf + (passes > 1 ? 4 * n : 0), *total = hist + (int64_t)digits * blocks;
    const int32_t *ki = nullptr, *ri = nullptr;
    SortExtras none = {};
    for (int p = 0; p < passes; ++p) {
        const bool last = p == passes - 1;
        int32_t *ko = last ? keys_out : buf + (p & 1) * 2 * n, *ro = last ? order : ko + n;
        hipLaunchKernelGGL(k_sort_count, dim3(blocks + (p ? 0 : clear_blocks(x))), dim3(256), 0, st, src, ki, n, rows, blocks, p * per, digits, hist,
                           p ? none : x);
        hipLaunchKernelGGL(k_sort_scan, dim3((digits + 63) / 64), dim3(1024), 0, st, hist, blocks, digits, total);
        hipLaunchKernelGGL(k_sort_place, dim3(blocks), dim3(256), (size_t)(4 * digits + 4) * sizeof(int), st, src, ki, ri, n, rows, p * per, per, hist,
                           total, ko, ro, passes == 1 ? x.offsets : nullptr);
        ki = ko;
        ri = ro;
    }
    if (x.offsets && passes > 1)
        hipLaunchKernelGGL(k_sort_offsets, dim3((unsigned)((src.n_keys + 256) / 256)), dim3(256), 0, st, x.offsets, keys_out, n, src.n_keys);
    return check_launch("k_sort_place");
}

}  // namespace mnr
