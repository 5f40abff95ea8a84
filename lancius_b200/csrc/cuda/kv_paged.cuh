// The paged 4-bit key/value cache: what its kernels and launchers share.
// Format and batch description: lcu_kv_pages / lcu_kv_batch in lancius_cuda.h.
#pragma once
#include "lcu_internal.h"
#include <cuda_fp16.h>

struct KvPagesDev {
    uint8_t *k_codes, *v_codes, *k_scales, *v_scales;
    float k_unit, v_unit;
    int n_pages, page_shift, heads;
};
struct KvBatchDev {
    const int32_t *table, *seq_len, *start;   // start == NULL: one token per sequence
    int width, n_seqs, n_tokens, max_len, max_new;
};

// Checks both descriptions and fills the device forms (max_len, max_new resolved).
lancius_error lcu_kv_describe(const lcu_kv_pages* pages, const lcu_kv_batch* batch, KvPagesDev* p, KvBatchDev* b);

// First row and number of new tokens of sequence s, clipped to the token arrays, and the rows that the clipping left out
// behind them: row first + i has position seq_len[s] - count - behind + i. False: some rows are not in the arrays.
__device__ __forceinline__ bool kv_new_tokens(const KvBatchDev& b, int s, int& first, int& count, int& behind) {
    first = b.start ? b.start[s] : s;
    const int last = b.start ? b.start[s + 1] : s + 1, end = min(last, b.n_tokens), from = max(first, 0);
    const bool whole = first == from && last == end;
    first = from;
    count = end > first ? end - first : 0;
    behind = last - end;
    return whole;
}

// Index of a cache row in units of rows ([page][head][slot]), or -1 when the position or its
// page lies outside the table or the cache.
__device__ __forceinline__ long long kv_row(const KvPagesDev& p, const KvBatchDev& b, int s, int pos, int head) {
    const int at = pos >> p.page_shift;
    if (at >= b.width || pos >= b.max_len) return -1;
    const int page = b.table[(size_t)s * b.width + at];
    if (page < 0 || page >= p.n_pages) return -1;
    return ((((long long)page * p.heads + head) << p.page_shift) + (pos & ((1 << p.page_shift) - 1)));
}

// two e4m3 bytes (low, high) -> half2; exact, NaN stays NaN
__device__ __forceinline__ uint32_t kv_scales_to_half(uint32_t two) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
    return h;
}
// one e4m3 byte -> float
__device__ __forceinline__ float kv_scale(uint32_t byte) {
    const uint32_t h = kv_scales_to_half(byte);
    return __low2float(*reinterpret_cast<const __half2*>(&h));
}
