// int8_product.hip -- rows quantised to 8 bits with a scale each, and the product of two such matrices.
//
//   q[r][c] = round(127 x[r][c] / m_r), scale_r = m_r / 127, m_r = max_c |x[r][c]|      (to the nearest, ties to even)
//   y[m][n] = act( sa[m] sb[n] sum_k a[m][k] b[n][k] + bias[n] )                        (the sum exact in int32)
//
// The quantiser is bound by HBM: a row stays in registers between its maximum and its rounding (65536 x 2048 bf16: 78 to 91 us, 4.4 to
// 5.1 TB/s).  The product of 65536 x 2048 x 2048 takes 295 to 350 us as the chip's clock allows (1.6 to 1.9 POP/s; 8192 cubed 2.0, and
// 2.6 on zeros: it is power that bounds it), 9 us for 9973 x 319 x 256.
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

typedef __attribute__((address_space(3))) void lds_void_t;
typedef __attribute__((address_space(1))) const void global_cvoid_t;

// ---- the tiled product ------------------------------------------------------------------------------------------------------------
// WR x WC waves, each with RB x CB blocks of 32 x 32 of the output.  K goes by in steps of 64 bytes through a ring of four LDS stages:
// while step k multiplies, both operands' 64 bytes of every row of step k + 3 are fetched straight into LDS (16 bytes a lane, no
// registers), a few fetches at a time between the matrix instructions: all at once they fill the fetch queue, and the waves wait to
// issue instead of multiplying.  A stage is read as ds_read_b128 fragments of v_mfma_i32_32x32x32_i8, one set ahead of its use.  The
// stages are separate LDS objects, so that the compiler's waits tell the fetches into one from the reads of another.  The four 16-byte
// pieces of a row lie at piece ^ (row >> 2 & 3): sixteen neighbouring rows of a fragment read then cover all 64 banks.
// Rows past the end fetch the last row again (their results are not stored); pieces behind column k fetch the last piece again, and the
// left operand's are zeroed in LDS before the last step is read, so whatever the right operand has there counts nothing.  A tile takes a
// multiple of four steps; those behind k only keep the ring going.
constexpr int TK = 64;

template <int WR, int WC, int RB, int CB> struct Tile {
    static constexpr int WAVES = WR * WC, THREADS = 64 * WAVES, BM = WR * RB * 32, BN = WC * CB * 32;
    static constexpr int A16 = BM * TK / 16, B16 = BN * TK / 16;             // 16-byte pieces of a stage
    static constexpr int FA = BM / (16 * WAVES), FB = BN / (16 * WAVES);     // fetches of a wave for a stage
};

// s_waitcnt vmcnt(n), the other counters left alone
template <int n> __device__ __forceinline__ void wait_fetches() { __builtin_amdgcn_s_waitcnt(0x0f70 | (n & 15) | (n >> 4) << 14); }

template <class T, int WR, int WC, int RB, int CB>
__global__ __launch_bounds__(64 * WR * WC) void k_product(ProductArgs p, int n_tiles, int total) {
    using S = Tile<WR, WC, RB, CB>;
    __shared__ int4v ring0[S::A16 + S::B16], ring1[S::A16 + S::B16], ring2[S::A16 + S::B16], ring3[S::A16 + S::B16];
    __shared__ float scales[S::BM + 2 * S::BN] __attribute__((aligned(16)));             // a's, b's, bias of the tile
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave / WC, wc = wave % WC, i32 = lane & 31, half = lane >> 5;
    const int k16 = (int)((p.k + 15) / 16 * 16), tail = k16 % TK / 16;       // pieces of the last step, 0: all four
    const int steps = (k16 + TK - 1) / TK, steps4 = (steps + 3) & ~3;
    auto stage = [&](auto j) -> int4v * {
        constexpr int J = decltype(j)::value;
        return J == 0 ? ring0 : J == 1 ? ring1 : J == 2 ? ring2 : ring3;
    };

    const int frow = wave * 16 + (lane >> 2);          // this lane's row among the 16 WAVES rows that one fetch of all waves covers
    const int fpiece = ((lane & 3) ^ (lane >> 4)) * 16;
    // where a tile's rows start: a base per operand, and this lane's rows as 32-bit offsets
    struct Cursor { const int8_t *a, *b; unsigned ra[S::FA], rb[S::FB]; };
    auto at_tile = [&](int tile) {
        const int64_t m0 = (int64_t)(tile / n_tiles) * S::BM, n0 = (int64_t)(tile % n_tiles) * S::BN;
        const int am = (int)(p.m - 1 - m0 < S::BM ? p.m - 1 - m0 : S::BM), bn = (int)(p.n - 1 - n0 < S::BN ? p.n - 1 - n0 : S::BN);
        Cursor f;
        f.a = p.a + m0 * p.lda;
        f.b = p.b + n0 * p.ldb;
#pragma unroll
        for (int i = 0; i < S::FA; ++i) {
            const int r = i * 16 * S::WAVES + frow;
            f.ra[i] = (unsigned)((r < am ? r : am) * (int)p.lda);
        }
#pragma unroll
        for (int i = 0; i < S::FB; ++i) {
            const int r = i * 16 * S::WAVES + frow;
            f.rb[i] = (unsigned)((r < bn ? r : bn) * (int)p.ldb);
        }
        return f;
    };
    auto fetch_a = [&](auto j, const Cursor &f, int step) {
        const int at = step * TK + fpiece, kb = at < k16 ? at : k16 - 16;
#pragma unroll
        for (int i = 0; i < S::FA; ++i)
            __builtin_amdgcn_global_load_lds((global_cvoid_t *)(f.a + (f.ra[i] + kb)), (lds_void_t *)(stage(j) + i * 64 * S::WAVES + wave * 64), 16, 0, 0);
    };
    auto fetch_b = [&](auto j, const Cursor &f, int step) {
        const int at = step * TK + fpiece, kb = at < k16 ? at : k16 - 16;
#pragma unroll
        for (int i = 0; i < S::FB; ++i)
            __builtin_amdgcn_global_load_lds((global_cvoid_t *)(f.b + (f.rb[i] + kb)), (lds_void_t *)(stage(j) + S::A16 + i * 64 * S::WAVES + wave * 64), 16, 0, 0);
    };
    int16v acc[CB][RB];
    // everyone's part of the next stage is in LDS, and nobody reads the stage before it any more.  (__syncthreads would also wait for
    // the fetches of later stages and for the last tile's stores.)
    auto meet = [&]() {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // step k from stage j; the fetches of step `fk` of `f` into the stage before it.  (Every step fetches, under no condition, the last
    // tile's last steps something that nobody reads: so the counts of the waits are the same on every path, for the compiler's own
    // waits too.)
    auto multiply = [&](auto j, int k, const Cursor &f, int fk) {
        constexpr int J = decltype(j)::value;
        const std::integral_constant<int, (J + 3) & 3> free;
        int4v af[2][RB], bf[2][CB];
        auto products = [&](int q) {
#pragma unroll
            for (int c = 0; c < CB; ++c)
#pragma unroll
                for (int r = 0; r < RB; ++r) acc[c][r] = __builtin_amdgcn_mfma_i32_32x32x32_i8(bf[q][c], af[q][r], acc[c][r], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        };
        if (k + 1 == steps && tail) {
            for (int e = threadIdx.x; e < S::BM * 4; e += S::THREADS)
                if ((e & 3) >= tail) stage(j)[(e & ~3) + ((e & 3) ^ (e >> 4 & 3))] = int4v{0, 0, 0, 0};
            meet();
        }
        fetch_a(free, f, fk);
        if (k < steps) {
            // (indexes that the compiler cannot take apart: behind a longer chain of pointers it loses track of which stage a read is from)
            const int ra = (wr * RB * 32 + i32) * 4, rb = S::A16 + (wc * CB * 32 + i32) * 4;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                int at = (2 * q + half) ^ (i32 >> 2 & 3), pa = ra + at, pb = rb + at;
                asm("" : "+v"(pa), "+v"(pb));
#pragma unroll
                for (int r = 0; r < RB; ++r) af[q][r] = stage(j)[pa + r * 128];
#pragma unroll
                for (int c = 0; c < CB; ++c) bf[q][c] = stage(j)[pb + c * 128];
            }
            products(0);
        }
        fetch_b(free, f, fk);
        asm("" : "+s"(k));                             // (or the two ifs become one, and the fetch between them is on two paths)
        if (k < steps) products(1);
    };
    const std::integral_constant<int, 0> s0;
    const std::integral_constant<int, 1> s1;
    const std::integral_constant<int, 2> s2;
    const std::integral_constant<int, 3> s3;
    // consecutive tiles (which share the rows of a) on one XCD
    int tile = blockIdx.x;
    if ((gridDim.x & 7) == 0) tile = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    if (tile >= total) return;
    Cursor f = at_tile(tile);
    fetch_a(s0, f, 0); fetch_b(s0, f, 0);
    fetch_a(s1, f, 1); fetch_b(s1, f, 1);
    fetch_a(s2, f, 2); fetch_b(s2, f, 2);
    constexpr int PER_STAGE = S::FA + S::FB;
    wait_fetches<0>();
    for (; tile < total; tile += gridDim.x) {
        const Cursor next = at_tile(tile + (int)gridDim.x < total ? tile + (int)gridDim.x : tile);
#pragma unroll
        for (int c = 0; c < CB; ++c)
#pragma unroll
            for (int r = 0; r < RB; ++r) {
                acc[c][r] = int16v(0);
                asm volatile("" : "+v"(acc[c][r]));    // (else the first step gets a copy of the loop of its own)
            }
        // four steps; the last three fetches of a tile are the next tile's first three.  A tile's first three stages were waited for
        // before the last tile's stores were issued: no wait for those here.
        auto four = [&](auto first, int k) {
            constexpr bool WAIT = !decltype(first)::value;
            const bool end = k + 4 == steps4;
            const int fk = end ? 0 : k + 4;
            if (WAIT) wait_fetches<2 * PER_STAGE>();
            meet();
            multiply(s0, k, f, k + 3);
            f.a = end ? next.a : f.a;                  // (selects, not a branch)
            f.b = end ? next.b : f.b;
#pragma unroll
            for (int i = 0; i < S::FA; ++i) f.ra[i] = end ? next.ra[i] : f.ra[i];
#pragma unroll
            for (int i = 0; i < S::FB; ++i) f.rb[i] = end ? next.rb[i] : f.rb[i];
            if (WAIT) wait_fetches<2 * PER_STAGE>();
            meet();
            multiply(s1, k + 1, f, fk);
            if (WAIT) wait_fetches<2 * PER_STAGE>();
            meet();
            multiply(s2, k + 2, f, fk + 1);
            wait_fetches<2 * PER_STAGE>();
            meet();
            multiply(s3, k + 3, f, fk + 2);
        };
        four(std::true_type{}, 0);
#pragma clang loop unroll(disable)
        for (int k = 4; k < steps4; k += 4) four(std::false_type{}, k);
        // Epilogue.  A lane has one row (the operands are swapped) and registers 4 g .. 4 g + 3 columns 8 g + 4 half ..: stored as they lie
        // that would be 8 or 16 bytes to each of 32 rows.  So 32 rows x 128 bytes at a time go through this wave's 4 KB of stage 3 (which
        // nobody reads now) and out as whole 128-byte rows (65536 x 2048 x 2048 in bf16: 541 -> 381 us), past the caches (371 -> 350).  The tile's scales and bias come by way of LDS, and before the first store:
        // loads and stores are counted in one queue, and a load behind a store would wait for it.
        const int64_t m0 = (int64_t)(tile / n_tiles) * S::BM, n0 = (int64_t)(tile % n_tiles) * S::BN;
        constexpr int VALUES = S::BM + 2 * S::BN, TURNS = (VALUES + S::THREADS - 1) / S::THREADS;
        float held[TURNS];
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
            const int e = i * S::THREADS + (int)threadIdx.x;
            held[i] = 0.f;
            if (e < S::BM) held[i] = p.sa[m0 + e < p.m ? m0 + e : p.m - 1];
            else if (e < S::BM + S::BN) held[i] = p.sb[n0 + e - S::BM < p.n ? n0 + e - S::BM : p.n - 1];
            else if (e < VALUES && p.bias) held[i] = p.bias[n0 + e - S::BM - S::BN < p.n ? n0 + e - S::BM - S::BN : p.n - 1];
        }
        wait_fetches<0>();                             // (these loads, and with them the next tile's first three stages)
#pragma unroll
        for (int i = 0; i < TURNS; ++i)
            if (i * S::THREADS + (int)threadIdx.x < VALUES) scales[i * S::THREADS + threadIdx.x] = held[i];
        meet();                                        // (and nobody reads stage 3 any more)
        const float low = p.relu ? 0.f : -__builtin_huge_valf();
        constexpr int PER = 128 / (32 * (int)sizeof(T));         // column blocks in 128 bytes: 1 (fp32) or 2
        constexpr int V = Vec<T>::N;
        static_assert(CB % PER == 0 && S::A16 + S::B16 >= S::WAVES * 256, "a wave's 4 KB of stage 3");
        char *mine = reinterpret_cast<char *>(ring3 + wave * 256);
#pragma unroll
        for (int r = 0; r < RB; ++r) {
            const float sa = scales[wr * RB * 32 + r * 32 + i32];
#pragma unroll
            for (int c0 = 0; c0 < CB; c0 += PER) {
#pragma unroll
                for (int c = c0; c < c0 + PER; ++c)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        typedef T quad __attribute__((ext_vector_type(4)));
                        const int n = (wc * CB + c) * 32 + 8 * g + 4 * half;
                        const float4 sb = *reinterpret_cast<const float4 *>(scales + S::BM + n), bias = *reinterpret_cast<const float4 *>(scales + S::BM + S::BN + n);
                        const float s4[4] = {sb.x, sb.y, sb.z, sb.w}, b4[4] = {bias.x, bias.y, bias.z, bias.w};
                        quad y;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float v = (float)acc[c][r][4 * g + i] * sa * s4[i] + b4[i];
                            y[i] = (T)(v < low ? low : v);
                        }
                        const int byte = ((c - c0) * 32 + 8 * g + 4 * half) * (int)sizeof(T);
                        *reinterpret_cast<quad *>(mine + i32 * 128 + (((byte >> 4) ^ (i32 >> 1 & 7)) << 4) + (byte & 15)) = y;
                    }
                wave_sync();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = i * 8 + (lane >> 3), piece = lane & 7;
                    const typename Vec<T>::raw y = *reinterpret_cast<const typename Vec<T>::raw *>(mine + row * 128 + ((piece ^ (row >> 1 & 7)) << 4));
                    const int64_t m = m0 + (wr * RB + r) * 32 + row, n = n0 + (wc * CB + c0) * 32 + piece * V;
                    T *dst = reinterpret_cast<T *>(p.y) + m * p.ldy + n;
                    if (m < p.m && n + V <= p.n) __builtin_nontemporal_store(y, reinterpret_cast<typename Vec<T>::type *>(dst));
                    else if (m < p.m)
#pragma unroll
                        for (int j = 0; j < V - 1; ++j)
                            if (n + j < p.n) dst[j] = y[j];
                }
                wave_sync();
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
}

template <class T, int WR, int WC, int RB, int CB> static int tiled(const ProductArgs &p, int cus_per, hipStream_t st) {
    using S = Tile<WR, WC, RB, CB>;
    const int64_t nt = (p.n + S::BN - 1) / S::BN, total = nt * ((p.m + S::BM - 1) / S::BM);
    if (total >= (1ll << 30)) return set_err(MNR_E_INVALID, "the output of mnr_int8_product is too large (%lld tiles)", (long long)total);
    const int64_t most = 256ll * cus_per;
    hipLaunchKernelGGL((k_product<T, WR, WC, RB, CB>), dim3((unsigned)(total < most ? total : most)), dim3(S::THREADS), 0, st, p, (int)nt, (int)total);
    return check_launch("k_product");
}

// ---- few tiles: K split over the waves ---------------------------------------------------------------------------------------------
// A workgroup of four waves makes 16 columns x 16 MT rows; wave w takes the 64-byte steps w, w + 4, ... of K straight from memory as
// fragments of v_mfma_i32_16x16x64_i8 (a lane: 16 bytes of one row), four steps in flight, and the waves' int32 sums meet in LDS.  What
// bounds it is the weight's bytes and the way to them: one row through 2048 x 2048 takes 4 MB and no reuse, 14.6 us by 16 tiles of 128 x
// 128 and 4.1 us by 128 of these workgroups; 512 x 512 x 4096 takes 14 us, where 16 tiles take 64 steps one after the other.
template <class T, int MT>
__global__ __launch_bounds__(256) void k_product_thin(ProductArgs p) {
    __shared__ int4v part[3][MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, quarter = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * 16 * MT;
    const int k16 = (int)((p.k + 15) / 16 * 16), steps = (k16 + 63) / 64;
    const int64_t nr = n0 + i16 < p.n ? n0 + i16 : p.n - 1;
    const int8_t *b = p.b + nr * p.ldb, *a[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) a[i] = p.a + (m0 + i * 16 + i16 < p.m ? m0 + i * 16 + i16 : p.m - 1) * p.lda;
    int4v acc[MT] = {};
    constexpr int AHEAD = 4;
    for (int s0 = wave; s0 < steps; s0 += 4 * AHEAD) {
        int4v bf[AHEAD], af[AHEAD][MT];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int at = (s0 + 4 * u) * 64 + quarter * 16;
            const bool in = at < k16;                  // behind k: the first piece again, times zero
            bf[u] = *reinterpret_cast<const int4v *>(b + (in ? at : 0));
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                af[u][i] = *reinterpret_cast<const int4v *>(a[i] + (in ? at : 0));
                af[u][i] = in ? af[u][i] : int4v{0, 0, 0, 0};
            }
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[u], af[u][i], acc[i], 0, 0, 0);
    }
    if (wave)
#pragma unroll
        for (int i = 0; i < MT; ++i) part[wave - 1][i][lane] = acc[i];
    __syncthreads();
    if (wave) return;
    // lane -> row m0 + 16 i + i16, registers -> columns n0 + 4 quarter ...
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
        for (int w = 0; w < 3; ++w) acc[i] += part[w][i][lane];
        const int64_t m = m0 + i * 16 + i16;
        if (m >= p.m) continue;
        const float sa = p.sa[m];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t n = n0 + quarter * 4 + j;
            if (n >= p.n) continue;
            float y = (float)acc[i][j] * sa * p.sb[n] + (p.bias ? p.bias[n] : 0.f);
            if (p.relu && y < 0.f) y = 0.f;
            reinterpret_cast<T *>(p.y)[m * p.ldy + n] = (T)y;
        }
    }
}

template <class T, int MT> static int thin(const ProductArgs &p, hipStream_t st) {
    hipLaunchKernelGGL((k_product_thin<T, MT>), dim3((unsigned)((p.n + 15) / 16), (unsigned)((p.m + 16 * MT - 1) / (16 * MT))), dim3(256), 0, st, p);
    return check_launch("k_product_thin");
}

template <class T> static int product(const ProductArgs &p, hipStream_t st) {
    // 256 x 256 tiles where they fill most of the chip, 128 x 128 tiles (two workgroups a CU) where those fill a fair part of it, and K
    // split over waves below that
    const int64_t big = ((p.m + 255) / 256) * ((p.n + 255) / 256), mid = ((p.m + 127) / 128) * ((p.n + 127) / 128);
    if (big >= 192) return tiled<T, 2, 4, 4, 2>(p, 1, st);
    if (mid >= 96) return tiled<T, 2, 2, 2, 2>(p, 2, st);
    if (p.m <= 16) return thin<T, 1>(p, st);
    if (p.m <= 32) return thin<T, 2>(p, st);
    return thin<T, 4>(p, st);
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

static int product_check(const char *who, const void *y, int64_t ldy, const int8_t *b, int64_t ldb, const float *sb, int64_t m, int64_t n, int64_t k,
                         int act, int type) {
    MNR_REQUIRE(type_ok(type), "unknown element type passed to %s", who);
    MNR_REQUIRE(act == 0 || act == 1, "the activation of %s is 0 (none) or 1 (ReLU)", who);
    MNR_REQUIRE(m >= 0 && n >= 0 && m < (1ll << 31) && n < (1ll << 31), "%s needs 0 <= m, n < 2^31", who);
    MNR_REQUIRE(k >= 1 && k <= 131071, "%s needs 1 <= k <= 131071: longer sums may leave int32", who);
    if (m == 0 || n == 0) return MNR_OK;
    const int64_t k16 = (k + 15) / 16 * 16;
    MNR_REQUIRE(y && b && sb, "null pointer passed to %s", who);
    MNR_REQUIRE((reinterpret_cast<uintptr_t>(b) & 15) == 0 && ldb % 16 == 0 && ldb < (1 << 22),
                "the operands of %s start at multiples of 16 bytes, with pitches that are multiples of 16 below 2^22", who);
    MNR_REQUIRE((n == 1 || ldb >= k16) && (m == 1 || ldy >= n), "row pitch smaller than a row passed to %s", who);
    return MNR_OK;
}

static int run_product(const ProductArgs &p, int type, hipStream_t st) {
    if (type == MNR_F32) return product<float>(p, st);
    if (type == MNR_F16) return product<f16_t>(p, st);
    return product<bf16_t>(p, st);
}

extern "C" int mnr_int8_product(void *y_dev, int64_t ldy, const int8_t *a_dev, int64_t lda, const float *a_scale_dev, const int8_t *b_dev, int64_t ldb,
                                const float *b_scale_dev, const float *bias_dev, int64_t m, int64_t n, int64_t k, int act, int type, void *stream) {
    const int rc = product_check("mnr_int8_product", y_dev, ldy, b_dev, ldb, b_scale_dev, m, n, k, act, type);
    if (rc != MNR_OK || m == 0 || n == 0) return rc;
    MNR_REQUIRE(a_dev && a_scale_dev, "null pointer passed to mnr_int8_product");
    MNR_REQUIRE((reinterpret_cast<uintptr_t>(a_dev) & 15) == 0 && lda % 16 == 0 && lda < (1 << 22),
                "the operands of mnr_int8_product start at multiples of 16 bytes, with pitches that are multiples of 16 below 2^22");
    MNR_REQUIRE(m == 1 || lda >= (k + 15) / 16 * 16, "row pitch smaller than a row passed to mnr_int8_product");
    return run_product(ProductArgs{y_dev, ldy, a_dev, lda, a_scale_dev, b_dev, ldb, b_scale_dev, bias_dev, m, n, k, act}, type, as_stream(stream));
}

static int64_t linear_pitch(int64_t k) { return (k + 127) / 128 * 128; }

extern "C" size_t mnr_int8_linear_workspace_bytes(int64_t m, int64_t k) {
    return m < 0 || k < 1 ? 0 : (size_t)m * (size_t)linear_pitch(k) + (size_t)m * sizeof(float);
}

extern "C" int mnr_int8_linear(void *y_dev, int64_t ldy, const void *x_dev, int64_t ldx, int x_type, const int8_t *b_dev, int64_t ldb,
                               const float *b_scale_dev, const float *bias_dev, int64_t m, int64_t n, int64_t k, int act, int type,
                               void *workspace_dev, size_t workspace_bytes, void *stream) {
    int rc = product_check("mnr_int8_linear", y_dev, ldy, b_dev, ldb, b_scale_dev, m, n, k, act, type);
    if (rc != MNR_OK || m == 0 || n == 0) return rc;
    MNR_REQUIRE(workspace_dev && (reinterpret_cast<uintptr_t>(workspace_dev) & 15) == 0 && workspace_bytes >= mnr_int8_linear_workspace_bytes(m, k),
                "mnr_int8_linear needs %zu bytes of workspace at a multiple of 16", mnr_int8_linear_workspace_bytes(m, k));
    const int64_t pitch = linear_pitch(k);
    int8_t *q = reinterpret_cast<int8_t *>(workspace_dev);
    float *scale = reinterpret_cast<float *>(q + m * pitch);
    rc = mnr_quantize_rows(q, pitch, scale, x_dev, ldx, m, k, x_type, stream);
    if (rc != MNR_OK) return rc;
    return run_product(ProductArgs{y_dev, ldy, q, pitch, scale, b_dev, ldb, b_scale_dev, bias_dev, m, n, k, act}, type, as_stream(stream));
}
