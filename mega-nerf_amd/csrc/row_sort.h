// row_sort.h -- stable order of rows by a small integer key (table index, cell number): what the embedding's gradient and the
// gate's dispatch share.
#pragma once
#include "common.h"
#include "op_device.h"

namespace mnr {

// Indices as the callers hold them: int32, int64, or fp32 (the image index column of a ray).  What lies outside [0, n_keys) is
// clamped, as mnr_gather_rows does (a NaN counts as 0), or with `drop` becomes n_keys, which sorts behind all others.
struct KeySource {
    const void *idx;
    int type;                  // MNR_I32, MNR_I64, MNR_F32
    int drop;
    int64_t n_keys;
    __device__ __forceinline__ int operator()(int64_t i) const {
        int64_t k;
        if (type == MNR_I32) k = reinterpret_cast<const int32_t *>(idx)[i];
        else if (type == MNR_I64) k = reinterpret_cast<const int64_t *>(idx)[i];
        else {
            const float f = reinterpret_cast<const float *>(idx)[i];
            k = f >= (float)n_keys ? n_keys : (f > -1.f ? (int64_t)f : (f <= -1.f ? -1 : 0));
        }
        if (k < 0 || k >= n_keys) k = drop ? n_keys : (k < 0 ? 0 : n_keys - 1);
        return (int)k;
    }
};
inline bool key_type_ok(int t) { return t == MNR_I32 || t == MNR_I64 || t == MNR_F32; }

// bytes of scratch for n keys of [0, n_keys] (whole numbers below 2^31)
size_t sort_rows_bytes(int64_t n, int64_t n_keys);
// What else the sort's launches do.  zero: memory that its first launch clears with the workgroups it has to spare (`words` words and
// then `half` 16-bit words); offsets (NULL: not wanted): [n_keys + 1], first place of every key, rows with key n_keys left out.
struct SortExtras {
    uint32_t *zero;  int64_t words;  int half;
    int32_t *offsets;
};
// order[p] = row of the p-th smallest (key, row), keys_out[p] = its key; n >= 1
int sort_rows(const KeySource &src, int64_t n, int32_t *order, int32_t *keys_out, void *ws, const SortExtras &x, hipStream_t st);
// x.zero alone (no rows to sort)
int clear_words(const SortExtras &x, hipStream_t st);

}  // namespace mnr
