// Appending to and reading from the paged 4-bit key/value cache.
//
// Append, per new token at position p: q and k rows are rotated, (x0, x1) -> (x0 cos a - x1 sin a,
// x0 sin a + x1 cos a) with a = p * base^(-2c/D); k and v rows are then held as codes -7 .. 7 with
// one e4m3 scale per 16 channels: scale = e4m3(max|x| / 7), code = round(x / scale).
// Angles, their sines and the rotation are in FP64 and rounded to FP32 once: an FP32 angle of
// position 100000 is off by 0.004 rad, and a rounding border crossed by one ulp changes a stored
// value by a whole step. A warp computes the D/2 sines of its token once for all heads. With a unit other than 1, x stands
// for x / unit rounded to FP32, which is infinite where it does not fit.
// Roundings are those of exact quotients, although the fast path multiplies with reciprocals: where the product is so
// near a border that it could lie on the wrong side (a relative 2^-22 for max|x| / 7, 2^-18 of a step for x / scale),
// the group takes IEEE divisions, and those do not err: 7 * border and scale * half are FP32 numbers, and a number next
// to one differs by more than half a step of the quotient.
//
// Bound: HBM, q + k + v read and q written in FP32, 0.56 bytes a cached element. One warp works on one token (or on a
// part of its rows, when tokens are few): a lane keeps 8 channels and their four sines and walks down the rows of q, k
// and v, so that two neighbours hold a 16-channel group and a warp reads 1024 contiguous bytes. Four channels a lane
// took 142 instructions per 128 elements, and the kernel was bound by their issue. 8863 tokens of 16 + 32 heads of 64,
// appended and read back (238 MB): 55.0 us, 4.3 TB/s. The append alone takes 37 us against a floor of 24, the
// reading back 18 against 13. Neither fills HBM nor the issue slots (52 and 46 %): with the 28 and 38 warps an SM that fit, they
// wait for their loads in 5.2 of 13.4 and 9.9 of 20.2 clocks per instruction. One token of 32 + 16 heads of 128, both calls: 5.1 us.
#include "kv_paged.cuh"
#include <math.h>

namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;

__device__ int g_kv_fault = 0;
std::atomic<bool> g_used{false};   // a kernel of this file has been launched: before that the word needs no reading

// Where one warp works: token, sequence, position, and the cache row of (token, head 0) or -1.
struct Place {
    int token, part, pos;
    long long row;      // of head 0
    bool any;
};

__device__ __forceinline__ Place find_place(const KvPagesDev& p, const KvBatchDev& b, int part_shift) {
    Place at;
    const unsigned id = blockIdx.x * WARPS + threadIdx.x / 32;
    const int lane = threadIdx.x & 31;
    at.token = (int)(id >> part_shift);
    at.part = (int)(id & ((1u << part_shift) - 1));
    at.any = at.token < b.n_tokens;
    int s = -1, end = 0;
    if (!b.start) {
        s = at.any && at.token < b.n_seqs ? at.token : -1;
        end = s + 1;
    } else {   // the last sequence that starts at or before the token holds it, unless it has ended
        int before = 0, from = 0, to = 0;
        if (id == 0) { from = b.start[0]; to = b.start[b.n_seqs]; }
#pragma unroll 4
        for (int i0 = 0; i0 < b.n_seqs; i0 += 32) {
            const int i = i0 + lane;
            before += __popc(__ballot_sync(0xffffffffu, i < b.n_seqs && b.start[i] <= at.token));
        }
        if (from < 0 || to > b.n_tokens) g_kv_fault = 1;   // rows outside the arrays
        end = b.start[before];
        if (before > 0 && at.any && at.token < end) s = before - 1;
    }
    at.any = s >= 0;
    at.pos = at.any ? b.seq_len[s] - (end - at.token) : -1;
    at.any = at.any && at.pos >= 0;
    at.row = at.any ? kv_row(p, b, s, at.pos, 0) : -1;
    return at;
}
// 8 floats by the widest access that their alignment allows (wide: 2: 32 bytes, 1: 16, 0: 4)
__device__ __forceinline__ void load8(float (&x)[8], const float* p, int wide) {
    if (wide == 2) {
        asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7])
                     : "l"(p));
    } else if (wide == 1) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = p[i];
    }
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8], int wide) {
    if (wide == 2) {
        asm volatile("st.global.v8.f32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]),
                     "f"(x[5]), "f"(x[6]), "f"(x[7]), "l"(p) : "memory");
    } else if (wide == 1) {
        *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = x[i];
    }
}
__device__ __forceinline__ float max_abs(float a, float b) {   // up to its sign; NaN if either is
    float r;
    asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// x[8] of one lane, the group's other 8 in its neighbour: 8 codes and the scale byte
__device__ __forceinline__ uint32_t quantise(float (&x)[8], float unit, uint32_t& scale_byte) {
    if (unit != 1.f) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = __fdiv_rn(x[i], unit);
    }
    float m = max_abs(max_abs(max_abs(x[0], x[1]), max_abs(x[2], x[3])), max_abs(max_abs(x[4], x[5]), max_abs(x[6], x[7])));
    m = fabsf(max_abs(m, __shfl_xor_sync(3u << (threadIdx.x & 30), m, 1)));
    if (!(m < INFINITY)) { scale_byte = 0x7f; return 0x88888888u; }
    // the scale of m (1 -+ 2^-22) / 7: where they differ, of the quotient itself
    uint16_t s2;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(s2) : "f"(m * (0.14285714924335480f * (1 + 0x1p-22f))), "f"(m * (0.14285714924335480f * (1 - 0x1p-22f))));
    if ((s2 & 0xff) != s2 >> 8) asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(s2) : "f"(0.f), "f"(__fdiv_rn(m, 7.f)));
    scale_byte = s2 & 0xff;
    if (!scale_byte) return 0x88888888u;   // the whole group is below half of the smallest scale
    const float s = kv_scale(scale_byte);
    float inv;
    asm("rcp.approx.f32 %0, %1;" : "=f"(inv) : "f"(s));
    constexpr float MAGIC = 12582912.f;   // 1.5 * 2^23: y + MAGIC - MAGIC is y rounded
    float r[8], off = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float y = x[i] * inv;
        r[i] = (y + MAGIC) - MAGIC;
        off = fmaxf(off, fabsf(y - r[i]));
    }
    // scales of at least 2^-6 have all their bits, so |x / scale| < 7.5
    if (!(off < 0.5f - 0x1p-18f && scale_byte >= 8 && scale_byte < 0x7e)) {
#pragma unroll
        for (int i = 0; i < 8; i++) r[i] = fminf(fmaxf(rintf(__fdiv_rn(x[i], s)), -7.f), 7.f);
    }
    // four codes are the digits of a number below 2^16; 2^23 + it has them in its low bits
    auto four = [&](int i) {
        return __float_as_uint(fmaf(fmaf(fmaf(r[i + 3], 16.f, r[i + 2]), 16.f, r[i + 1]), 16.f, r[i]) + (8388608.f + 0x8888));
    };
    return __byte_perm(four(0), four(4), 0x5410);
}

// 2^part_shift warps per token, each takes every so manieth set of rows
template <int D>
__global__ void __launch_bounds__(THREADS, 4) k_kv_append(KvPagesDev p, KvBatchDev b, int part_shift, float* q_out, const float* q,
                                                       size_t q_ld, int hq, const float* __restrict__ k, size_t k_ld,
                                                       const float* __restrict__ v, size_t v_ld, double log2_base, int rotate,
                                                       int wide) {
    __shared__ double2 turn[WARPS][4][D / 8];         // (cos, sin) of pair 4e + i at [i][e]
    constexpr int C = D / 8, ROWS = 32 / C, U = 2;    // lanes of a row, rows a warp takes at once, rows in flight
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, e = lane % C;
    const unsigned id = blockIdx.x * WARPS + warp;
    const size_t t = id >> part_shift;                // the token, if there is one
    const int step = ROWS << part_shift, rows = hq + 2 * p.heads;   // of q, then k, then v
    int row = (int)(id & ((1u << part_shift) - 1)) * ROWS + lane / C;
    const float* qs = q + t * q_ld + 8 * e;
    const float* ks = k + t * k_ld + 8 * e - (size_t)hq * D;
    const float* vs = v + t * v_ld + 8 * e - (size_t)(hq + p.heads) * D;
    auto fetch = [&](float (&x)[8], int r) {
        if (r < rows) load8(x, (r < hq ? qs : r < hq + p.heads ? ks : vs) + (size_t)r * D, wide);
    };
    float x[U][8];
    if (t < (size_t)b.n_tokens) {                     // while the token's place is looked up
#pragma unroll
        for (int u = 0; u < U; u++) fetch(x[u], row + u * step);
    }
    const Place at = find_place(p, b, part_shift);
    if (!at.any) return;
    if (at.row < 0 && lane == 0) g_kv_fault = 1;
    if (rotate) {
#pragma unroll
        for (int i = lane; i < D / 2; i += 32) {
            double sn, cs;
            sincos((double)at.pos * exp2(-(double)(2 * i) / D * log2_base), &sn, &cs);
            turn[warp][i % 4][i / 4] = make_double2(cs, sn);
        }
        __syncwarp();
    }
    float* qd = q_out + t * hq * D + 8 * e;
    auto handle = [&](float (&y)[8], int r) {
        const bool is_v = r >= hq + p.heads;
        if (rotate && !is_v) {   // not when there is nothing to do: infinities stay
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const double2 a = turn[warp][i][e];
                const double y0 = y[2 * i], y1 = y[2 * i + 1];
                y[2 * i] = (float)(y0 * a.x - y1 * a.y);
                y[2 * i + 1] = (float)(y0 * a.y + y1 * a.x);
            }
        }
        if (r < hq) {            // may be q's own place: a lane has read it, and only it does
            store8(qd + (size_t)r * D, y, wide);
        } else if (at.row >= 0) {
            uint32_t sb;
            const uint32_t c = quantise(y, is_v ? p.v_unit : p.k_unit, sb);
            const size_t to = (size_t)at.row + ((size_t)(r - hq - (is_v ? p.heads : 0)) << p.page_shift);
            *reinterpret_cast<uint32_t*>((is_v ? p.v_codes : p.k_codes) + to * (D / 2) + 4 * e) = c;
            if ((e & 1) == 0) (is_v ? p.v_scales : p.k_scales)[to * (D / 16) + (e >> 1)] = (uint8_t)sb;
        }
    };
    while (row < rows) {
#pragma unroll
        for (int u = 0; u < U; u++)
            if (row < rows) {
                handle(x[u], row);
                fetch(x[u], row + U * step);
                row += step;
            }
    }
}

template <int D>
__global__ void __launch_bounds__(THREADS) k_kv_read(float* __restrict__ k_out, float* __restrict__ v_out, KvPagesDev p,
                                                     KvBatchDev b, int part_shift, int wide) {
    constexpr int C = D / 8, ROWS = 32 / C, U = 4;
    const int lane = threadIdx.x % 32, e = lane % C;
    const Place at = find_place(p, b, part_shift);
    if (!at.any) return;
    if (at.row < 0 && lane == 0) g_kv_fault = 1;
    const int step = ROWS << part_shift;
    int row = at.part * ROWS + lane / C;   // of k, then v
    auto get = [&](float* out, const uint8_t* codes, const uint8_t* scales, float unit) {
        out += (size_t)at.token * p.heads * D + 8 * e;
        if (at.row >= 0) {
            codes += at.row * (D / 2) + 4 * e;
            scales += at.row * (D / 16) + (e >> 1);
        }
        while (row < p.heads) {
            uint32_t c[U], sb[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const size_t r = (size_t)(row + u * step) << p.page_shift;
                const bool there = row + u * step < p.heads && at.row >= 0;
                c[u] = there ? __ldcs(reinterpret_cast<const uint32_t*>(codes + r * (D / 2))) : 0;
                sb[u] = there ? scales[r * (D / 16)] : 0;   // scale 0 reads as zeros
            }
#pragma unroll
            for (int u = 0; u < U; u++)
                if (row < p.heads) {
                    const float sc = kv_scale(sb[u]);
                    float x[8];
                    // n or'ed into the mantissa of 2^23 is 2^23 + n; (n - 8) * scale is exact, the unit rounds
#pragma unroll
                    for (int i = 0; i < 8; i++) x[i] = (__uint_as_float(0x4b000000u | (c[u] >> (4 * i) & 15)) - 8388616.f) * sc * unit;
                    store8(out + (size_t)row * D, x, wide);
                    row += step;
                }
        }
        row -= p.heads;
    };
    get(k_out, p.k_codes, p.k_scales, p.k_unit);
    get(v_out, p.v_codes, p.v_scales, p.v_unit);
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
lancius_error bad(lancius_error e) { lancius_set_error(e); return e; }

// Warps per token, as a power of two: the number with the least rounds of 32 warps per SM times the steps of a warp over its
// rows, where the start of a warp with its sines counts as 2 steps. Above 8 warps per SM at least 2 steps, whose loads are in
// flight together. (5380 tokens of 32 + 16 heads of 128: one warp 57.6 us, as they are just over one round, 46.6
// with four; 2000 tokens 35.3 and 28.4; 128 tokens 4.5 with 2 steps a warp, 5.2 with one.)
int part_shift(int tokens, int rows, int rows_at_once) {
    int best = 0;
    size_t least = SIZE_MAX;
    for (int shift = 0; shift == 0 || (rows_at_once << (shift - 1)) < rows; shift++) {
        const size_t warps = (size_t)tokens << shift, at_once = (size_t)rows_at_once << shift;
        const size_t rounds = (warps + 32 * LCU_SMS - 1) / (32 * LCU_SMS), steps = (rows + at_once - 1) / at_once;
        if (shift && steps < 2 && warps > 8 * LCU_SMS) break;
        if (rounds * (steps + 2) < least) { least = rounds * (steps + 2); best = shift; }
    }
    return best;
}
unsigned part_blocks(int tokens, int shift) { return (unsigned)((((size_t)tokens << shift) + WARPS - 1) / WARPS); }
// widest access to rows `ld` floats apart (load8, store8)
int width(const void* p, size_t ld) {
    return (uintptr_t)p % 32 == 0 && ld % 8 == 0 ? 2 : (uintptr_t)p % 16 == 0 && ld % 4 == 0 ? 1 : 0;
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
    if (!g_used.load(std::memory_order_relaxed)) return nullptr;
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
    int wide = n_q_heads ? min(width(q, q_ld), width(q_out, 0)) : 2;
    wide = min(wide, min(width(k, k_ld), width(v, v_ld)));
    const int hq = (int)n_q_heads;
    const int shift = part_shift(b.n_tokens, hq + 2 * p.heads, 256 / (int)D);
    const unsigned grid = part_blocks(b.n_tokens, shift);
    cudaStream_t st = lcu_as_stream(stream);
    auto kernel = D == 64 ? k_kv_append<64> : D == 128 ? k_kv_append<128> : k_kv_append<256>;
    g_used.store(true, std::memory_order_relaxed);
    kernel<<<grid, THREADS, 0, st>>>(p, b, shift, q_out, q, q_ld, hq, k, k_ld, v, v_ld, lb, rotate, wide);
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
    const size_t D = pages->head_dim;
    const int shift = part_shift(b.n_tokens, 2 * p.heads, 256 / (int)D);
    const int wide = min(width(k_out, 0), width(v_out, 0));
    auto kernel = D == 64 ? k_kv_read<64> : D == 128 ? k_kv_read<128> : k_kv_read<256>;
    g_used.store(true, std::memory_order_relaxed);
    kernel<<<part_blocks(b.n_tokens, shift), THREADS, 0, lcu_as_stream(stream)>>>(k_out, v_out, p, b, shift, wide);
    lcu_note_launch();
    return lcu_launch_status();
}

}  // extern "C"
