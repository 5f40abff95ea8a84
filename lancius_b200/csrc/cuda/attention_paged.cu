// Attention of a step's tokens over the paged 4-bit cache (lcu_attention_paged).
//
// out[t][h] = sum_j p_j V_j, p = softmax(q . K_j / sqrt(D)), j = 0 .. position of row t, as one pass with a
// running maximum and sum. One CTA per (row, query head); a warp takes every fourth key, its lanes D / 32
// channels each.
#include "kv_paged.cuh"
#include <math.h>

namespace {

constexpr int WARPS = 4, THREADS = 32 * WARPS;

__device__ int g_attn_paged_fault = 0;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <int D>
__device__ __forceinline__ void row_values(const uint8_t* codes, const uint8_t* scales, long long at, int lane, float (&x)[D / 32]) {
#pragma unroll
    for (int i = 0; i < D / 32; i += 2) {
        const int ch = lane * (D / 32) + i;
        const uint32_t c = codes[at * (D / 2) + ch / 2];
        const float sc = kv_scale(scales[at * (D / 16) + ch / 16]);
        x[i] = (float)((int)(c & 15) - 8) * sc;
        x[i + 1] = (float)((int)(c >> 4) - 8) * sc;
    }
}

template <int D>
__global__ void __launch_bounds__(THREADS) k_attn_paged(float* __restrict__ out, const float* __restrict__ q, size_t q_ld,
                                                        int hq, KvPagesDev p, KvBatchDev b, float scale_log2) {
    constexpr int R = D / 32;
    __shared__ float sm_m[WARPS], sm_l[WARPS], sm_o[WARPS][D];
    const int s = blockIdx.z, h = blockIdx.y, i = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int first, count;
    kv_new_tokens(b, s, first, count);
    if (count > b.max_new && i == 0) g_attn_paged_fault = 1;
    if (i >= count) return;
    const int t = first + i, len = b.seq_len[s];
    int limit = len - (count - i) + 1;   // keys that this row sees
    if (limit > b.max_len) { limit = b.max_len; g_attn_paged_fault = 1; }
    const int head = h / (hq / p.heads);
    float qr[R], o[R], x[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        qr[r] = q[(size_t)t * q_ld + (size_t)h * D + lane * R + r] * scale_log2 * p.k_unit;
        o[r] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int j = warp; j < limit; j += WARPS) {
        const long long at = kv_row(p, b, s, j, head);
        if (at < 0) g_attn_paged_fault = 1;
        float acc = 0.f;
        if (at >= 0) {
            row_values<D>(p.k_codes, p.k_scales, at, lane, x);
#pragma unroll
            for (int r = 0; r < R; r++) acc = fmaf(qr[r], x[r], acc);
        }
        acc = warp_sum(acc);
        const float mx = fmaxf(m, acc), corr = m == -INFINITY ? 0.f : ex2(m - mx), pj = ex2(acc - mx);
#pragma unroll
        for (int r = 0; r < R; r++) x[r] = 0.f;
        if (at >= 0) row_values<D>(p.v_codes, p.v_scales, at, lane, x);
        bool nan = false;
#pragma unroll
        for (int r = 0; r < R; r++) {
            nan = nan || x[r] != x[r];
            o[r] = fmaf(pj, x[r], o[r] * corr);
        }
        l = l * corr + pj;
        if (__any_sync(0xffffffffu, nan)) l = NAN;
        m = mx;
    }
    if (lane == 0) { sm_m[warp] = m; sm_l[warp] = l; }
#pragma unroll
    for (int r = 0; r < R; r++) sm_o[warp][lane * R + r] = o[r];
    __syncthreads();
    float M = -INFINITY, L = 0.f;
    for (int w = 0; w < WARPS; w++) M = fmaxf(M, sm_m[w]);
    for (int w = 0; w < WARPS; w++) L += sm_m[w] == -INFINITY && sm_l[w] == 0.f ? 0.f : ex2(sm_m[w] - M) * sm_l[w];
    for (int d = threadIdx.x; d < D; d += THREADS) {
        float acc = 0.f;
        for (int w = 0; w < WARPS; w++) acc += sm_m[w] == -INFINITY && sm_l[w] == 0.f ? 0.f : ex2(sm_m[w] - M) * sm_o[w][d];
        out[(size_t)t * hq * D + (size_t)h * D + d] = limit > 0 ? acc / L * p.v_unit : 0.f;
    }
}

lancius_error bad(lancius_error e) { lancius_set_error(e); return e; }

}  // namespace

extern "C" {

int* lcu_attn_paged_fault_addr(void) {
    void* p = nullptr;
    return cudaGetSymbolAddress(&p, g_attn_paged_fault) == cudaSuccess ? static_cast<int*>(p) : nullptr;
}

size_t lcu_attention_paged_workspace(const lcu_kv_pages* pages, const lcu_kv_batch* batch, size_t n_q_heads) {
    (void)pages; (void)batch; (void)n_q_heads;
    return 0;
}

lancius_error lcu_attention_paged(float* out, const float* q, size_t q_ld, size_t n_q_heads, const lcu_kv_pages* pages,
                                  const lcu_kv_batch* batch, void* workspace, size_t workspace_bytes, void* stream) {
    KvPagesDev p;
    KvBatchDev b;
    lancius_error e = lcu_kv_describe(pages, batch, &p, &b);
    if (e != LANCIUS_ERROR_OK) return e;
    if (!b.n_seqs || !b.n_tokens || !n_q_heads) return LANCIUS_ERROR_OK;
    if (!out || !q) return bad(LANCIUS_ERROR_NULL_PTR);
    const size_t D = pages->head_dim;
    if (n_q_heads > 65535 || n_q_heads % pages->n_heads || q_ld < n_q_heads * D) return bad(LANCIUS_ERROR_SHAPE_MISMATCH);
    const float scale_log2 = (float)(1.4426950408889634 / sqrt((double)D));
    const dim3 grid((unsigned)b.max_new, (unsigned)n_q_heads, (unsigned)b.n_seqs);
    cudaStream_t st = lcu_as_stream(stream);
    const int hq = (int)n_q_heads;
    if (D == 64) k_attn_paged<64><<<grid, THREADS, 0, st>>>(out, q, q_ld, hq, p, b, scale_log2);
    else if (D == 128) k_attn_paged<128><<<grid, THREADS, 0, st>>>(out, q, q_ld, hq, p, b, scale_log2);
    else k_attn_paged<256><<<grid, THREADS, 0, st>>>(out, q, q_ld, hq, p, b, scale_log2);
    (void)workspace; (void)workspace_bytes;
    lcu_note_launch();
    return lcu_launch_status();
}

}  // extern "C"
