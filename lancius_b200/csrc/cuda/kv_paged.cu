// Appending to and reading from the paged 4-bit key/value cache.
//
// Append, per new token at position p: q and k rows are rotated, (x0, x1) -> (x0 cos a - x1 sin a,
// x0 sin a + x1 cos a) with a = p * base^(-2c/D); k and v rows are then held as codes -7 .. 7 with
// one e4m3 scale per 16 channels: scale = e4m3(max|x| / 7), code = round(x / scale).
// Angles, their sines and the rotation are in FP64 and rounded to FP32 once: an FP32 angle of
// position 100000 is off by 0.004 rad, and a rounding border crossed by one ulp changes a stored
// value by a whole step. One CTA computes the D/2 sines of its token once for all heads.
// Both divisions are IEEE (__fdiv_rn): max|x| / 7 then rounds to the right side of every e4m3
// border and x / scale to the right side of every half, since 7 * border and scale * half are FP32
// numbers, and a number next to them differs by more than half a step of the quotient.
//
// Bound: HBM, q + k + v read and q written in FP32, 0.56 bytes a cached element. Four adjacent
// threads hold one 16-channel group as float4s, so loads are 512 contiguous bytes a warp, a
// group's maximum takes two shuffles and its codes are written as 64-byte runs.
#include "kv_paged.cuh"
#include <math.h>

namespace {

constexpr int THREADS = 256;

__device__ int g_kv_fault = 0;

// sequence of token t, or -1 for a row that belongs to none (every thread of the block gets it)
__device__ int find_sequence(const KvBatchDev& b, int t) {
    if (!b.start) return t < b.n_seqs ? t : -1;
    int before = 0;   // sequences that start at or before t; the last of them holds it (earlier ones are empty or end)
    for (int i0 = 0; i0 < b.n_seqs; i0 += THREADS) {
        const int i = i0 + threadIdx.x;
        before += __syncthreads_count(i < b.n_seqs && b.start[i] <= t);
    }
    return before > 0 && t < b.start[before] ? before - 1 : -1;
}

__device__ __forceinline__ float4 load4(const float* p, bool vec) {
    return vec ? __ldcs(reinterpret_cast<const float4*>(p)) : make_float4(p[0], p[1], p[2], p[3]);
}

// x[4] of one thread, the group's other 12 in its neighbours: 4 codes (16 bits) and the scale byte
__device__ __forceinline__ uint32_t quantise(float4 x, float unit, uint32_t& scale_byte) {
    if (unit != 1.f) {
        x.x = __fdiv_rn(x.x, unit); x.y = __fdiv_rn(x.y, unit);
        x.z = __fdiv_rn(x.z, unit); x.w = __fdiv_rn(x.w, unit);
    }
    // the bits of |x| order like the numbers, with infinity and NaN above all of them
    uint32_t m = max(max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu),
                     max(__float_as_uint(x.z) & 0x7fffffffu, __float_as_uint(x.w) & 0x7fffffffu));
    const uint32_t quad = 0xfu << (threadIdx.x & 28);
    m = max(m, __shfl_xor_sync(quad, m, 1));
    m = max(m, __shfl_xor_sync(quad, m, 2));
    if (m >= 0x7f800000u) { scale_byte = 0x7f; return 0x8888; }
    uint16_t s2;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(s2) : "f"(0.f), "f"(__fdiv_rn(__uint_as_float(m), 7.f)));
    scale_byte = s2 & 0xff;
    if (!scale_byte) return 0x8888;   // the whole group is below half of the smallest scale
    const float s = kv_scale(scale_byte);
    auto code = [s](float y) { return (uint32_t)(min(7, max(-7, __float2int_rn(__fdiv_rn(y, s)))) + 8); };
    return code(x.x) | code(x.y) << 4 | code(x.z) << 8 | code(x.w) << 12;
}

// grid.x = token, grid.y = parts of its (Hq + 2 Hkv) D / 4 float4s
template <int D>
__global__ void __launch_bounds__(THREADS) k_kv_append(KvPagesDev p, KvBatchDev b, float* q_out, const float* q,
                                                       size_t q_ld, int hq, const float* __restrict__ k, size_t k_ld,
                                                       const float* __restrict__ v, size_t v_ld, double log2_base, int rotate,
                                                       int q_vec, int k_vec, int v_vec) {
    __shared__ double2 turn[D / 2];   // (cos, sin)
    const int t = blockIdx.x;
    const int s = find_sequence(b, t);
    if (s < 0) return;
    const int pos = b.seq_len[s] - ((b.start ? b.start[s + 1] : s + 1) - t);
    if (pos < 0) return;
    if (rotate && threadIdx.x < D / 2) {
        double sn, cs;
        sincos((double)pos * exp2(-(double)(2 * threadIdx.x) / D * log2_base), &sn, &cs);
        turn[threadIdx.x] = make_double2(cs, sn);
    }
    __syncthreads();
    constexpr int C = D / 4;   // float4s of a row
    const int rows = hq + 2 * p.heads;
    for (int c = blockIdx.y * THREADS + threadIdx.x; c < rows * C; c += gridDim.y * THREADS) {
        const int row = c / C, e = c % C;
        const bool is_q = row < hq, is_v = row >= hq + p.heads;
        const int head = is_q ? row : is_v ? row - hq - p.heads : row - hq;
        const float* src = is_q ? q + (size_t)t * q_ld : is_v ? v + (size_t)t * v_ld : k + (size_t)t * k_ld;
        float4 x = load4(src + (size_t)head * D + 4 * e, is_q ? q_vec : is_v ? v_vec : k_vec);
        if (rotate && !is_v) {
            const double2 a = turn[2 * e], z = turn[2 * e + 1];
            const double x0 = x.x, x1 = x.y, x2 = x.z, x3 = x.w;
            x.x = (float)(x0 * a.x - x1 * a.y); x.y = (float)(x0 * a.y + x1 * a.x);
            x.z = (float)(x2 * z.x - x3 * z.y); x.w = (float)(x2 * z.y + x3 * z.x);
        }
        if (is_q) {
            float* dst = q_out + (size_t)t * hq * D + (size_t)head * D + 4 * e;
            if (q_vec) *reinterpret_cast<float4*>(dst) = x;
            else { dst[0] = x.x; dst[1] = x.y; dst[2] = x.z; dst[3] = x.w; }
            continue;
        }
        uint32_t sb;
        const uint32_t codes = quantise(x, is_v ? p.v_unit : p.k_unit, sb);
        const long long at = kv_row(p, b, s, pos, head);
        if (at < 0) { g_kv_fault = 1; continue; }
        *reinterpret_cast<uint16_t*>((is_v ? p.v_codes : p.k_codes) + at * (D / 2) + 2 * e) = (uint16_t)codes;
        if ((e & 3) == 0) (is_v ? p.v_scales : p.k_scales)[at * (D / 16) + (e >> 2)] = (uint8_t)sb;
    }
}

template <int D>
__global__ void __launch_bounds__(THREADS) k_kv_read(float* __restrict__ k_out, float* __restrict__ v_out, KvPagesDev p,
                                                     KvBatchDev b) {
    const int t = blockIdx.x;
    const int s = find_sequence(b, t);
    if (s < 0) return;
    const int pos = b.seq_len[s] - ((b.start ? b.start[s + 1] : s + 1) - t);
    if (pos < 0) return;
    constexpr int C = D / 4;
    for (int c = blockIdx.y * THREADS + threadIdx.x; c < 2 * p.heads * C; c += gridDim.y * THREADS) {
        const int row = c / C, e = c % C;
        const bool is_v = row >= p.heads;
        const int head = is_v ? row - p.heads : row;
        const long long at = kv_row(p, b, s, pos, head);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (at < 0) {
            g_kv_fault = 1;
        } else {
            const uint32_t c = *reinterpret_cast<const uint16_t*>((is_v ? p.v_codes : p.k_codes) + at * (D / 2) + 2 * e);
            const float sc = kv_scale((is_v ? p.v_scales : p.k_scales)[at * (D / 16) + (e >> 2)]);
            auto value = [&](int i) { return (float)((int)(c >> (4 * i) & 15) - 8) * sc * (is_v ? p.v_unit : p.k_unit); };
            x = make_float4(value(0), value(1), value(2), value(3));
        }
        *reinterpret_cast<float4*>((is_v ? v_out : k_out) + ((size_t)t * p.heads + head) * D + 4 * e) = x;
    }
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
lancius_error bad(lancius_error e) { lancius_set_error(e); return e; }

// CTAs per token: enough for about two CTAs per SM when tokens are few, at most one pass each
unsigned parts(int tokens, int float4s) {
    const int most = (float4s + THREADS - 1) / THREADS, want = (2 * LCU_SMS + tokens - 1) / tokens;
    return (unsigned)(want < most ? want : most);
}

}  // namespace

lancius_error lcu_kv_describe(const lcu_kv_pages* pages, const lcu_kv_batch* batch, KvPagesDev* p, KvBatchDev* b) {
    if (!pages || !batch) return bad(LANCIUS_ERROR_NULL_PTR);
    if (!pages->k_codes || !pages->v_codes || !pages->k_scales || !pages->v_scales) return bad(LANCIUS_ERROR_NULL_PTR);
    if (!aligned16(pages->k_codes) || !aligned16(pages->v_codes) || !aligned16(pages->k_scales) || !aligned16(pages->v_scales))
        return bad(LANCIUS_ERROR_UNSUPPORTED_DTYPE);
    if (pages->head_dim != 64 && pages->head_dim != 128 && pages->head_dim != 256) return bad(LANCIUS_ERROR_UNSUPPORTED_OP);
    const size_t ps = pages->page_size;
    if (!ps || ps > 4096 || (ps & (ps - 1)) || !pages->n_heads || pages->n_heads > 65535 || pages->n_pages > (size_t)INT32_MAX)
        return bad(LANCIUS_ERROR_SHAPE_MISMATCH);
    if (!(pages->k_unit > 0.f) || !(pages->v_unit > 0.f) || isinf(pages->k_unit) || isinf(pages->v_unit))
        return bad(LANCIUS_ERROR_SHAPE_MISMATCH);
    if (batch->n_seqs && (!batch->seq_len || (batch->table_width && !batch->page_table))) return bad(LANCIUS_ERROR_NULL_PTR);
    if (batch->n_seqs > 65535 || batch->n_tokens > (size_t)INT32_MAX / 2 || batch->table_width > (size_t)INT32_MAX / ps)
        return bad(LANCIUS_ERROR_SHAPE_MISMATCH);
    if (!batch->token_start && batch->n_tokens < batch->n_seqs) return bad(LANCIUS_ERROR_SHAPE_MISMATCH);
    if (pages->n_pages > 0xfffffffeull / ps / pages->n_heads) return bad(LANCIUS_ERROR_SHAPE_MISMATCH);   // 32-bit row numbers
    const size_t whole = batch->table_width * ps;
    p->k_codes = pages->k_codes; p->v_codes = pages->v_codes;
    p->k_scales = pages->k_scales; p->v_scales = pages->v_scales;
    p->k_unit = pages->k_unit; p->v_unit = pages->v_unit;
    p->n_pages = (int)pages->n_pages; p->heads = (int)pages->n_heads;
    p->page_shift = 0;
    while (((size_t)1 << p->page_shift) < ps) p->page_shift++;
    b->table = batch->page_table; b->seq_len = batch->seq_len; b->start = batch->token_start;
    b->width = (int)batch->table_width; b->n_seqs = (int)batch->n_seqs; b->n_tokens = (int)batch->n_tokens;
    b->max_len = (int)(batch->max_seq_len && batch->max_seq_len < whole ? batch->max_seq_len : whole);
    const size_t most = batch->token_start ? batch->n_tokens : 1;
    b->max_new = (int)(batch->max_new && batch->max_new < most ? batch->max_new : most);
    return LANCIUS_ERROR_OK;
}

extern "C" {

int* lcu_kv_fault_addr(void) {
    void* p = nullptr;
    return cudaGetSymbolAddress(&p, g_kv_fault) == cudaSuccess ? static_cast<int*>(p) : nullptr;
}

lancius_error lcu_kv_append_paged(const lcu_kv_pages* pages, const lcu_kv_batch* batch, float* q_out, const float* q,
                                  size_t q_ld, size_t n_q_heads, const float* k, size_t k_ld, const float* v, size_t v_ld,
                                  double rope_base, void* stream) {
    KvPagesDev p;
    KvBatchDev b;
    lancius_error e = lcu_kv_describe(pages, batch, &p, &b);
    if (e != LANCIUS_ERROR_OK) return e;
    if (!b.n_seqs || !b.n_tokens) return LANCIUS_ERROR_OK;
    if (!k || !v || (n_q_heads && (!q || !q_out))) return bad(LANCIUS_ERROR_NULL_PTR);
    const size_t D = pages->head_dim, kv = pages->n_heads * D;
    if (n_q_heads > 65535 || (n_q_heads && q_ld < n_q_heads * D) || k_ld < kv || v_ld < kv || isnan(rope_base) || isinf(rope_base))
        return bad(LANCIUS_ERROR_SHAPE_MISMATCH);
    if (n_q_heads && q == q_out && q_ld != n_q_heads * D) return bad(LANCIUS_ERROR_SHAPE_MISMATCH);
    const int rotate = rope_base > 0;
    const double lb = rotate ? log2(rope_base) : 0.0;
    const int qv = aligned16(q) && aligned16(q_out) && q_ld % 4 == 0, kvec = aligned16(k) && k_ld % 4 == 0,
              vvec = aligned16(v) && v_ld % 4 == 0;
    const int hq = (int)n_q_heads;
    const dim3 grid((unsigned)b.n_tokens, parts(b.n_tokens, (hq + 2 * p.heads) * (int)D / 4));
    cudaStream_t st = lcu_as_stream(stream);
    if (D == 64) k_kv_append<64><<<grid, THREADS, 0, st>>>(p, b, q_out, q, q_ld, hq, k, k_ld, v, v_ld, lb, rotate, qv, kvec, vvec);
    else if (D == 128) k_kv_append<128><<<grid, THREADS, 0, st>>>(p, b, q_out, q, q_ld, hq, k, k_ld, v, v_ld, lb, rotate, qv, kvec, vvec);
    else k_kv_append<256><<<grid, THREADS, 0, st>>>(p, b, q_out, q, q_ld, hq, k, k_ld, v, v_ld, lb, rotate, qv, kvec, vvec);
    lcu_note_launch();
    return lcu_launch_status();
}

lancius_error lcu_kv_read_paged(float* k_out, float* v_out, const lcu_kv_pages* pages, const lcu_kv_batch* batch,
                                void* stream) {
    KvPagesDev p;
    KvBatchDev b;
    lancius_error e = lcu_kv_describe(pages, batch, &p, &b);
    if (e != LANCIUS_ERROR_OK) return e;
    if (!b.n_seqs || !b.n_tokens) return LANCIUS_ERROR_OK;
    if (!k_out || !v_out) return bad(LANCIUS_ERROR_NULL_PTR);
    if (!aligned16(k_out) || !aligned16(v_out)) return bad(LANCIUS_ERROR_UNSUPPORTED_DTYPE);
    const size_t D = pages->head_dim;
    const dim3 grid((unsigned)b.n_tokens, parts(b.n_tokens, 2 * p.heads * (int)D / 4));
    cudaStream_t st = lcu_as_stream(stream);
    if (D == 64) k_kv_read<64><<<grid, THREADS, 0, st>>>(k_out, v_out, p, b);
    else if (D == 128) k_kv_read<128><<<grid, THREADS, 0, st>>>(k_out, v_out, p, b);
    else k_kv_read<256><<<grid, THREADS, 0, st>>>(k_out, v_out, p, b);
    lcu_note_launch();
    return lcu_launch_status();
}

}  // extern "C"
