// Attention of a step's tokens over the paged 4-bit cache (lcu_attention_paged).
//
// out[t][h] = sum_j p_j V_j, p = softmax(q . K_j / sqrt(D)), j = 0 .. position of row t, in one pass over the
// cache with a running maximum and sum per row.
//
// Bound: the floor is HBM. A key/value pair of one head is D + D / 8 bytes and is read once for all rows of its key
// head ((new token, query head) pairs, up to 24 per CTA); at the measured copy rate an SM receives about 46 codes a
// clock, so turning codes into operands is the work that has to fit beside the loads. What bounds the kernel is the
// issue of that work: 770 instructions a warp and tile of 32 keys of 128 with up to 4 rows, 805 with 8, in which the
// tensor pipe is busy for 20 and 38 %. Four warps a quarter of an SM issue them at nine tenths of the rate within the
// loop, at 60 to 62 % over the kernel, as a CTA spends a quarter of its time on lengths, first loads and its merge. MMAs
// do not overlap with the half-rate LOP3 and HFMA2 (18.3 clocks for a group with its MMA, 9.5 without).
//   131072 keys of one sequence, 8 key heads of 128, 4 rows each: 40.8 us, 3.7 TB/s (0.57 of the measured copy rate)
//   32 sequences of up to 8192 keys, 8 key heads of 128, one row each: 66.5 us, 3.55 TB/s (0.54)
//   64 sequences of up to 8000 keys, 8 key heads of 128, 8 rows each: 137 us, 3.3 TB/s (0.50); the loads alone 83 us
//   24 sequences of up to 3001 keys, 4 key heads of 64, 20 rows each: 19.5 us
//   16 sequences of up to 5000 keys, one key head of 256, 8 rows: 12.4 us
// Prompts run through the same kernel, 24 rows (16 of heads of 256) at a time, each of which reads the keys that they see and
// turns them into operands again: 8192 new tokens of 8192, 32 heads on 8 of 128, take 4.6 ms, 121 TFLOP/s. The
// shapes of 16 rows spill 140 (heads of 128) and 212 bytes (256) a thread.
//
// Products run as mma.sync m16n8k16 (f16 in, FP32 out). Measured 0.5 of them per clock and SM; two serve 256 codes
// and 8 rows, so 64 codes a clock, above the HBM rate. tcgen05 would need the operands written to shared or tensor
// memory as f16 first, four times the bytes of the codes. The operands are exact: a dequantised value
// (n - 8) * scale has 8 significant bits, so K and V fit f16 as they are; q (scaled to [1, 2) by a power of two) and p are
// split into two f16 halves, 22 bits, one MMA each. The codes are operand A (16 keys or 16 channels), q and p operand B (8
// rows): of the two assignments the one whose accumulator for O is half as large, which decides how many warps
// fit (with q and p as A, halves stacked in its 16 rows, it took 160 registers and 63.4 us for the first of these, and
// 60.0 with the codes as A at the same stage). Up to 4 rows put both halves into one operand: 47.7.
//
// Dequantising, a known way for 4-bit weights (Kim et al., "Who Says Elephants Can't Run", 2022): a code or'ed into the
// mantissa of an f16 constant, then one HFMA2 with the group's factor and offset gives (n - 8) scale / 16 without
// rounding (scale_of). Eight codes take 5 integer and 4 HFMA2 instructions. (4-bit
// floating point needs cvt, measured 25 codes a clock and SM, or more shifts.)
//   S^T = K Q^T: A = K wants channel pairs of one key: a thread holds D / 4 contiguous channels of a key, any order of
//     channels will do if q's fragment has the same.
//   O^T += V^T P^T: A = V^T wants key pairs of one channel: the words of two keys are first interleaved by 16-bit
//     halves (2 PRMT per 16 codes). P^T comes from S^T's accumulators by movmatrix.
//
// Work: CTA = (chunk of keys, key head, sequence, block of rows), 4 warps that each take every fourth tile of 32
// keys through a ring of cp.async stages of their own (no block barrier in the loop) and are merged at the end.
// Shared-memory rows are swizzled in 16-byte pieces so that both fragment reads are free of bank conflicts.
// Chunks of a sequence are joined by k_attn_paged_join or, where they are few, by their cluster. Rows past a tile's last
// visible key are filled with zeros by cp.async, so stale bytes never reach an MMA.
#include "kv_paged.cuh"
#include <cooperative_groups.h>
#include <math.h>
#include <type_traits>

namespace cg = cooperative_groups;

namespace {

constexpr int WARPS = 4, THREADS = 32 * WARPS, TILE = 32;
// Keys of a CTA, at most, where all run at once and in rounds. An MMA truncates its sum, and a warp of the CTA adds a
// fourth of them up in one accumulator.
constexpr int MAX_CHUNK = 2048, ROUND = 1280;
constexpr int MAX_CLUSTER = 8;
constexpr float P_BIAS = 7.f;     // p = 2^(s - m + 7): more of the small weights stay above f16's smallest step
constexpr uint32_t NONE = 0xffffffffu;
constexpr float RAISE = 8.f;      // the running maximum moves only when exceeded by 2^8: p <= 2^15 fits f16
// From here on a score may lie 1/4 and more from its FP32 number, and a maximum held in FP32 that far from the score it
// came from: scores are rounded before the maximum is taken off, so that the largest is 0 and not some 2^n.
constexpr float FAR = 4194304.f;

__device__ int g_attn_paged_fault = 0;
std::atomic<bool> g_used{false};   // a kernel of this file has been launched: before that the word needs no reading

template <int D, int ROWS>   // ROWS of q per CTA: 4 or a multiple of 8
struct Shape {
    static constexpr int ROW = D / 2, SROW = D / 16;            // code and scale bytes of a cached row
    static constexpr int STAGES = D == 256 ? 2 : D == 128 ? (ROWS >= 16 ? 3 : 2) : 4;
    static constexpr int CODES = TILE * ROW, SCALES = TILE * SROW;
    static constexpr int STAGE = 2 * (CODES + SCALES);
    static constexpr int NT = (ROWS + 7) / 8;                   // 8-column operands
    static constexpr bool PACK = ROWS == 4;                     // hi and lo halves share one
    static constexpr int STEPS = D / 16;
    static constexpr int Q_BYTES = STEPS * (PACK ? 256 : 512) * NT;
    static constexpr int RING = WARPS * STAGES * STAGE;
    static constexpr int O_LD = D + 4;
    static constexpr int MERGE = WARPS * ROWS * O_LD * 4;       // reuses the ring
    static constexpr int SMEM = Q_BYTES + (RING > MERGE ? RING : MERGE);
    static constexpr int RESIDENT = D == 256 ? 2 : D == 128 ? (ROWS <= 8 ? 4 : ROWS == 16 ? 3 : 2)
                                             : ROWS <= 8 ? 5 : ROWS == 16 ? 4 : 3;   // CTAs per SM
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <int N>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src));
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N));
}
template <int N>   // zeros when !valid
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool valid) {
    const int n = valid ? N : 0;
    if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n));
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(n), "n"(N));
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ __half2 as_half2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

// Scales of two groups or keys (the halves of `two`) as the factors and offsets of its codes: codes in bits 0-3 of a 16-bit
// half, or'ed with 0x6400, are the f16 number 1024 + n, those in bits 4-7 are 16 (64 + n). All are exact: s has 4
// significant bits, 129 * 15 < 2^11. Values come out as (n - 8) s / 16, so that 64.5 s stays below f16's largest.
struct Scale { __half2 m0, b0, m4, b4; };
__device__ __forceinline__ Scale scale_of(uint32_t two) {
    const __half2 s = as_half2(two);
    return Scale{__hmul2(s, __float2half2_rn(0.0625f)), __hmul2(s, __float2half2_rn(-64.5f)),
                 __hmul2(s, __float2half2_rn(0.00390625f)), __hmul2(s, __float2half2_rn(-4.5f))};
}
__device__ __forceinline__ Scale half_of(const Scale& s, int high) {
    return high ? Scale{__high2half2(s.m0), __high2half2(s.b0), __high2half2(s.m4), __high2half2(s.b4)}
                : Scale{__low2half2(s.m0), __low2half2(s.b0), __low2half2(s.m4), __low2half2(s.b4)};
}
// The masks are held in registers that the compiler cannot see through: (w & mask) | bias with two immediates would
// take two LOP3, and these are the instructions that the kernel executes most.
struct Masks { uint32_t m0, m4; };
__device__ __forceinline__ uint32_t code_bits(uint32_t w, uint32_t mask) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, 0x64006400, 0xea;" : "=r"(r) : "r"(w), "r"(mask));
    return r;
}
// the 4 codes of both 16-bit halves of w -> 4 half2
__device__ __forceinline__ void dequantise(uint32_t w, const Scale& s, const Masks& k, uint32_t (&h)[4]) {
    const uint32_t v = w >> 8;
    h[0] = as_u32(__hfma2(as_half2(code_bits(w, k.m0)), s.m0, s.b0));
    h[1] = as_u32(__hfma2(as_half2(code_bits(w, k.m4)), s.m4, s.b4));
    h[2] = as_u32(__hfma2(as_half2(code_bits(v, k.m0)), s.m0, s.b0));
    h[3] = as_u32(__hfma2(as_half2(code_bits(v, k.m4)), s.m4, s.b4));
}

// byte offset of 16-byte piece c of cached row r in a stage (128-byte lines, pieces permuted per line)
template <int D>
__device__ __forceinline__ int piece(int r, int c) {
    if (D == 64) { const int line = r >> 2; return line * 128 + ((((r & 3) * 2 + c) ^ ((line & 1) << 1)) << 4); }
    if (D == 128) { const int line = r >> 1; return line * 128 + ((((r & 1) * 4 + c) ^ ((line & 3) << 1)) << 4); }
    return r * 128 + ((c ^ ((((r >> 1) & 3) << 1) | (r & 1))) << 4);
}

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {   // of an 8 x 8 f16 matrix held by the warp
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
// split of p0, p1 into f16 halves
__device__ __forceinline__ void split(float p0, float p1, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(p0, p1);
    const float2 f = __half22float2(h);
    hi = as_u32(h);
    lo = as_u32(__floats2half2_rn(p0 - f.x, p1 - f.y));
}

// A row's factor for its sums, in which V comes as value / 16; 0 for a row without a key. The unit is multiplied on after
// it: 16 units may be more than FP32 holds, and a small one over L less than it holds in full.
__device__ __forceinline__ float weighed(float L) { return L == 0.f ? 0.f : 16.f / L; }
__device__ __forceinline__ void store4(float* to, float4 sum, float L, float unit) {
    const float inv = weighed(L);
    to[0] = sum.x * inv * unit; to[1] = sum.y * inv * unit; to[2] = sum.z * inv * unit; to[3] = sum.w * inv * unit;
}

// 16 log2(e) / sqrt(D) * k_unit = factor * 2^exponent, as its product with a row's power of two may leave FP32's range
struct Scores {
    float factor;   // 0.5 .. 1
    int exponent;
};

struct Split {
    int chunk, splits;
    bool cluster;   // k_attn_paged's CLUSTER
};

__device__ __forceinline__ int chunks_of(int keys, int chunk) { return keys / chunk + (keys % chunk != 0); }

// CLUSTER: the splits of a block of rows are a cluster, whose CTAs join their sums without another kernel
template <int D, int ROWS, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, Shape<D, ROWS>::RESIDENT)
k_attn_paged(float* __restrict__ out, const float* __restrict__ q, size_t q_ld, bool q_wide, int hq, KvPagesDev p, KvBatchDev b,
             Scores scores, Split sp, float* __restrict__ part_o, float2* __restrict__ part_ml) {
    using S = Shape<D, ROWS>;
    constexpr int COLS = ROWS, NT = S::NT, R = 2 * NT;
    constexpr bool PACK = S::PACK;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float col_scale[COLS];
    __shared__ float sm_m[WARPS][COLS], sm_l[WARPS][COLS];
    __shared__ float2 cl_ml[COLS];
    asm volatile("griddepcontrol.launch_dependents;");

    const uint32_t zero = (uint32_t)p.heads >> 31;
    const Masks masks{0x000f000fu + zero, 0x00f000f0u + zero};
    const int group = hq / p.heads, blocks = gridDim.x / sp.splits;
    const int split_id = CLUSTER ? blockIdx.x % sp.splits : blockIdx.x / blocks;
    const int block = CLUSTER ? blockIdx.x / sp.splits : blockIdx.x % blocks, head = blockIdx.y, s = blockIdx.z;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    int first, count, behind;
    const bool whole = kv_new_tokens(b, s, first, count, behind);
    const int len = b.seq_len[s];
    const int used = count < b.max_new ? count : b.max_new;       // rows that are computed
    const int keys = min(max(len, 0), b.max_len);
    if (split_id == 0 && block == 0 && tid == 0 && (len > b.max_len || count > b.max_new || !whole)) g_attn_paged_fault = 1;
    const int cols = min(COLS, used * group - block * COLS);     // rows of this block
    const int parts = max(1, chunks_of(keys, sp.chunk));          // of this sequence
    if (cols <= 0 || split_id >= parts) {
        if (CLUSTER && cols > 0 && parts > 1) {   // the others' barriers
            cg::this_cluster().sync();
            cg::this_cluster().sync();
        }
        return;
    }

    // this thread's R rows of q: 2t, 2t + 1 (and 8 more); packed: 2 (t % 2) and the next, held by t and t ^ 2
    auto row_at = [&](int r) { return PACK ? 2 * (t & 1) + r : 2 * t + (r & 1) + (r >> 1) * 8; };
    // keys that row c of the block sees: those up to its token's position
    const int seen = len - count - behind + 1;
    auto limit_of = [&](int c) {
        const int i = (block * COLS + c) / group;
        return c < cols ? min(seen + i, b.max_len) : 0;
    };
    int limit[R], least = 0x7fffffff;
#pragma unroll
    for (int r = 0; r < R; r++) limit[r] = limit_of(row_at(r));
    least = limit_of(0);                                          // positions rise with the row
    const int begin = split_id * sp.chunk, end = begin + min(sp.chunk, limit_of(cols - 1) - begin);

    // q: a lane takes 8 channels, on their way while the first tiles are asked for
    constexpr int LANES = D / 8, QC = (COLS * LANES + THREADS - 1) / THREADS;   // lanes of a row, rows of a lane
    const int q_owner = lane % LANES & 3, q_octet = lane % LANES >> 2;
    auto q_col = [&](int k) { return (warp + k * WARPS) * (32 / LANES) + lane / LANES; };
    float qx[QC][8];
#pragma unroll
    for (int k = 0; k < QC; k++) {
        const int c = q_col(k), ci = block * COLS + c;
        const float* from = q + (size_t)(first + ci / group) * q_ld + (size_t)(head * group + ci % group) * D + q_owner * (D / 4) +
                            q_octet * 8;
#pragma unroll
        for (int i = 0; i < 8; i++) qx[k][i] = 0.f;
        if (c < cols && q_wide) {
            const float4 u = *reinterpret_cast<const float4*>(from), v = *reinterpret_cast<const float4*>(from + 4);
            qx[k][0] = u.x; qx[k][1] = u.y; qx[k][2] = u.z; qx[k][3] = u.w;
            qx[k][4] = v.x; qx[k][5] = v.y; qx[k][6] = v.z; qx[k][7] = v.w;
        } else if (c < cols) {
#pragma unroll
            for (int i = 0; i < 8; i++) qx[k][i] = from[i];
        }
    }

    // loads: tile i of this warp holds keys begin + 32 (warp + 4 i) ...
    const int tiles_all = end > begin ? (end - begin + TILE - 1) / TILE : 0;
    const int tiles = tiles_all > warp ? (tiles_all - warp + WARPS - 1) / WARPS : 0;
    uint8_t* ring = smem + S::Q_BYTES + warp * S::STAGES * S::STAGE;
    const int32_t* table = b.table + (size_t)s * b.width;
    const int slot_mask = (1 << p.page_shift) - 1;
    const uint32_t heads = p.heads;
    auto row_of = [&](int i) {   // cache row of this lane's key of tile i, NONE: no key, or no such page
        const uint32_t key = (uint32_t)begin + TILE * (warp + WARPS * i) + lane;
        if (i >= tiles || key >= (uint32_t)end) return NONE;
        const int page = table[key >> p.page_shift];
        if (page >= 0 && page < p.n_pages) return (((uint32_t)page * heads + head) << p.page_shift) + (key & slot_mask);
        g_attn_paged_fault = 1;
        return NONE;
    };
    // a row's pieces are copied by neighbouring lanes, PER rows an instruction
    constexpr int C = S::ROW / 16, PER = 32 / C;
    const uint8_t* k_from = p.k_codes + 16 * (lane % C);
    const uint8_t* v_from = p.v_codes + 16 * (lane % C);
    const uint32_t ring_at = smem_u32(ring), piece_at = piece<D>(lane / C, lane % C), scale_at = 2 * S::CODES + lane * S::SROW;
    auto issue = [&](bool any, uint32_t row, uint32_t stage) {
        if (any) {
            const uint32_t at = ring_at + stage;
            if (__all_sync(0xffffffffu, row != NONE)) {
#pragma unroll
                for (int it = 0; it < C; it++) {
                    const size_t from = (size_t)__shfl_sync(0xffffffffu, row, it * PER + lane / C) * S::ROW;
                    const uint32_t to = at + (D == 256 && (it & 1) ? piece_at ^ 64 : piece_at) + it * PER * S::ROW;
                    copy_async<16>(to, k_from + from);
                    copy_async<16>(to + S::CODES, v_from + from);
                }
                copy_async<S::SROW>(at + scale_at, p.k_scales + (size_t)row * S::SROW);
                copy_async<S::SROW>(at + scale_at + S::SCALES, p.v_scales + (size_t)row * S::SROW);
            } else {   // the last tile, or a bad page: zeros for the rows that are not there
#pragma unroll
                for (int it = 0; it < C; it++) {
                    const uint32_t r = __shfl_sync(0xffffffffu, row, it * PER + lane / C);
                    const size_t from = r != NONE ? (size_t)r * S::ROW : 0;
                    const uint32_t to = at + (D == 256 && (it & 1) ? piece_at ^ 64 : piece_at) + it * PER * S::ROW;
                    copy_async<16>(to, k_from + from, r != NONE);
                    copy_async<16>(to + S::CODES, v_from + from, r != NONE);
                }
                const size_t from = row != NONE ? (size_t)row * S::SROW : 0;
                copy_async<S::SROW>(at + scale_at, p.k_scales + from, row != NONE);
                copy_async<S::SROW>(at + scale_at + S::SCALES, p.v_scales + from, row != NONE);
            }
        }
        asm volatile("cp.async.commit_group;");
    };
    uint32_t ahead[S::STAGES];
#pragma unroll
    for (int i = 0; i < S::STAGES; i++) ahead[i] = row_of(i);
#pragma unroll
    for (int i = 0; i < S::STAGES - 1; i++) issue(i < tiles, ahead[i], i * S::STAGE);
    uint32_t row_ahead = ahead[S::STAGES - 1];

    // q as B fragments in shared memory: [8 rows][step][lane][hi 0, hi 1, lo 0, lo 1]; packed: [step][lane][2], columns 0-3
    // hi, 4-7 lo. Of 8 channels 0, 4, 1, 5 are one step's and 2, 6, 3, 7 the next one's.
#pragma unroll
    for (int k = 0; k < QC; k++) {
        const int c = q_col(k);
        const float(&x)[8] = qx[k];
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) amax = fmaxf(amax, fabsf(x[i]));
#pragma unroll
        for (int i = LANES / 2; i > 0; i >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, i));
        int e = (int)(__float_as_uint(amax) >> 23) - 127;          // 2^e <= amax < 2^(e + 1)
        if (amax == 0.f || e > 127) e = 0;
        e = min(max(e, -126), 126);
        const float down = __uint_as_float((uint32_t)(127 - e) << 23);
        if (c >= COLS) continue;
        // K comes as value / 16. Sums of products lie below 2^18 and are multiples of 2^-37: with a scale of 2^100 the
        // largest takes all the weight, as with any larger scale, and stays finite; with 2^-126 all weigh the same. The scale
        // is never 0, which would make NaN of a masked score.
        if (lane % LANES == 0)
            col_scale[c] = scores.factor * __uint_as_float((uint32_t)(127 + min(max(e + scores.exponent, -125), 100)) << 23);
#pragma unroll
        for (int u = 0; u < 2; u++) {
            uint4 f;
            split(x[2 * u] * down, x[2 * u + 4] * down, f.x, f.z);
            split(x[2 * u + 1] * down, x[2 * u + 5] * down, f.y, f.w);
            const int step = 2 * q_octet + u;
            if (PACK) {
                uint2* to = reinterpret_cast<uint2*>(smem) + step * 32 + c * 4 + q_owner;
                to[0] = make_uint2(f.x, f.y);
                to[16] = make_uint2(f.z, f.w);
            } else {
                reinterpret_cast<uint4*>(smem)[((c >> 3) * S::STEPS + step) * 32 + (c & 7) * 4 + q_owner] = f;
            }
        }
    }
    __syncthreads();

    float o[NT][D / 16][4], m[R], l[R], cs[R];   // o: channels g D/8 + 2j, + 2j + 1 of rows 2t, 2t + 1
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int j = 0; j < D / 16; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) o[nt][j][r] = 0.f;
#pragma unroll
    for (int r = 0; r < R; r++) { m[r] = -INFINITY; l[r] = 0.f; cs[r] = col_scale[row_at(r)]; }
    const uint4* q_frag = reinterpret_cast<const uint4*>(smem) + lane;
    const uint2* q_pack = reinterpret_cast<const uint2*>(smem) + lane;

    // this thread's pieces of a stage: K rows n * 8 + g (channels t D/4 ...), V rows 16 kb + 2t + {0, 1, 8, 9} (channels
    // g D/8 ...); rows 8 apart have the same permutation
    const int k_at = D == 64 ? piece<D>(g, t >> 1) + (t & 1) * 8 : piece<D>(g, t * (D / 128));
    const int k_at2 = D == 256 ? piece<D>(g, 2 * t + 1) : 0;
    const int v_piece = D == 64 ? g >> 2 : D == 128 ? g >> 1 : g, v_in = D == 64 ? (g & 3) * 4 : D == 128 ? (g & 1) * 8 : 0;
    const int v_at[2] = {S::CODES + piece<D>(2 * t, v_piece) + v_in, S::CODES + piece<D>(2 * t + 1, v_piece) + v_in};
    const int ks_at = 2 * S::CODES + g * S::SROW + t * (D / 64);
    constexpr int VG = D == 256 ? 2 : 1;   // groups of a thread's channels of V
    const int vs_at = 2 * S::CODES + S::SCALES + 2 * t * S::SROW + (D == 64 ? g >> 1 : g * VG);
    int stage = 0, stage_in = (S::STAGES - 1) * S::STAGE;
    bool far = false;   // some running maximum of the warp is at least FAR

    for (int i = 0; i < tiles; i++) {
        asm volatile("cp.async.wait_group %0;" ::"n"(S::STAGES - 2));
        __syncwarp();   // the tile is there for all lanes, and the stage before it is free
        issue(i + S::STAGES - 1 < tiles, row_ahead, stage_in);
        row_ahead = row_of(i + S::STAGES);
        const uint8_t* st = ring + stage;
        stage = stage == (S::STAGES - 1) * S::STAGE ? 0 : stage + S::STAGE;
        stage_in = stage_in == (S::STAGES - 1) * S::STAGE ? 0 : stage_in + S::STAGE;
        const int key0 = begin + TILE * (warp + WARPS * i);

        // ---- S^T = K Q^T, 32 keys for each of q's fragments
        uint32_t kw[4][D / 32];
        // [.][16 keys]: (key g, rows 2t, 2t + 1), (key g + 8, the same). An MMA truncates its sum, so the products with q's lo
        // halves, and the second half of 256 channels, add up apart: as many truncations of a large sum less.
        constexpr int HALVES = D == 256 ? 2 : 1;
        float a[NT][2][4], a_hi[HALVES][NT][2][4], a_lo[NT][2][4];
#pragma unroll
        for (int n = 0; n < 4; n++) {
            const uint8_t* at = st + k_at + n * 8 * S::ROW;
            if constexpr (D == 64) {
                const uint2 v = *reinterpret_cast<const uint2*>(at);
                kw[n][0] = v.x; kw[n][1] = v.y;
            } else {
                const uint4 v = *reinterpret_cast<const uint4*>(at);
                kw[n][0] = v.x; kw[n][1] = v.y; kw[n][2] = v.z; kw[n][3] = v.w;
                if constexpr (D == 256) {
                    const uint4 u = *reinterpret_cast<const uint4*>(st + k_at2 + n * 8 * S::ROW);
                    kw[n][4] = u.x; kw[n][5] = u.y; kw[n][6] = u.z; kw[n][7] = u.w;
                }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int x = 0; x < 8; x++) {
                a_lo[nt][x >> 2][x & 3] = 0.f;
#pragma unroll
                for (int h = 0; h < HALVES; h++) a_hi[h][nt][x >> 2][x & 3] = 0.f;
            }
        Scale pair[4][D == 256 ? 2 : 1];           // factors of two groups
#pragma unroll
        for (int n = 0; n < 4; n++) {
            const uint8_t* at = st + ks_at + n * 8 * S::SROW;
            if constexpr (D == 64) pair[n][0] = scale_of(kv_scales_to_half(*at));
            else if constexpr (D == 128) pair[n][0] = scale_of(kv_scales_to_half(*reinterpret_cast<const uint16_t*>(at)));
            else {
                const uint32_t v = *reinterpret_cast<const uint32_t*>(at);
                pair[n][0] = scale_of(kv_scales_to_half(v & 0xffff));
                pair[n][1] = scale_of(kv_scales_to_half(v >> 16));
            }
        }
#pragma unroll
        for (int gr = 0; gr < D / 64; gr++) {      // groups of this thread's channels, two words each
            Scale sc[4];
#pragma unroll
            for (int n = 0; n < 4; n++) sc[n] = half_of(pair[n][gr / 2], gr & 1);
#pragma unroll
            for (int wi = 2 * gr; wi < 2 * gr + 2; wi++) {
                uint4 f[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        if constexpr (PACK) {
                            const uint2 v = q_pack[(2 * wi + u) * 32];
                            f[nt][u] = make_uint4(v.x, v.y, 0, 0);
                        } else f[nt][u] = q_frag[(nt * S::STEPS + 2 * wi + u) * 32];
                    }
#pragma unroll
                for (int kb = 0; kb < 2; kb++) {
                    uint32_t h[4], h8[4];
                    dequantise(kw[2 * kb][wi], sc[2 * kb], masks, h);
                    dequantise(kw[2 * kb + 1][wi], sc[2 * kb + 1], masks, h8);
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const uint32_t ka[4] = {h[2 * u], h8[2 * u], h[2 * u + 1], h8[2 * u + 1]};
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            mma(a_hi[wi * HALVES / (D / 32)][nt][kb], ka, f[nt][u].x, f[nt][u].y);
                            if (!PACK) mma(a_lo[nt][kb], ka, f[nt][u].z, f[nt][u].w);
                        }
                    }
                }
            }
        }

        // ---- V's scales: pairs (key 2t, 2t + 1) and (2t + 8, 2t + 9) of each 16-key half
        uint32_t vs[2][2][VG];
        uint32_t nan = 0;
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int y = 0; y < 2; y++)
#pragma unroll
                for (int x = 0; x < VG; x++) {
                    const uint8_t* sc = st + vs_at + (16 * kb + 8 * y) * S::SROW + x;
                    vs[kb][y][x] = (uint32_t)sc[0] + (uint32_t)sc[S::SROW] * 256u;
                    nan |= vs[kb][y][x] + 0x0101u;
                }
        // A NaN in a value must not meet the zero weights of rows that do not see it: its scale becomes 0 and the
        // weights of the rows that see it become NaN.
        uint32_t poison = 0;   // keys of the tile
        if (__any_sync(0xffffffffu, nan & 0x8080u)) {
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int y = 0; y < 2; y++)
#pragma unroll
                    for (int x = 0; x < VG; x++)
#pragma unroll
                        for (int z = 0; z < 2; z++)
                            if ((vs[kb][y][x] >> (8 * z) & 0x7f) == 0x7f) {
                                vs[kb][y][x] &= ~(0xffu << (8 * z));
                                poison |= 1u << (16 * kb + 8 * y + 2 * t + z);
                            }
            poison = __reduce_or_sync(0xffffffffu, poison);
        }

#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int x = 0; x < 8; x++)
                a[nt][x >> 2][x & 3] = a_hi[0][nt][x >> 2][x & 3] + (HALVES == 2 ? a_hi[HALVES - 1][nt][x >> 2][x & 3] : 0.f) +
                                       (PACK ? 0.f : a_lo[nt][x >> 2][x & 3]);
        if (PACK) {   // hi + lo columns: t < 2 adds up and weighs the first 16 keys, its partner t ^ 2 the others
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const float other = __shfl_xor_sync(0xffffffffu, t < 2 ? a[0][1][x] : a[0][0][x], 2);
                a[0][0][x] = (t < 2 ? a[0][0][x] : a[0][1][x]) + other;
            }
        }

        // ---- weights. Value x of a row: key key1 + 16 (x >> 1) + 8 (x & 1)
        constexpr int X = PACK ? 2 : 4;
        const int key1 = key0 + g + (PACK && t >= 2 ? 16 : 0);
        float sv[R][X], top[R];
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int x = 0; x < X; x++) sv[r][x] = a[r >> 1][x >> 1][2 * (x & 1) + (r & 1)];   // times cs[r]: log2 units
        if (key0 > least - TILE) {
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int x = 0; x < X; x++)
                    if (key1 + 8 * x >= limit[r]) sv[r][x] = -INFINITY;
        }
        bool raise = false;
#pragma unroll
        for (int r = 0; r < R; r++) {
            top[r] = fmaxf(sv[r][0], sv[r][1]);
            if (X == 4) top[r] = fmaxf(top[r], fmaxf(sv[r][X - 2], sv[r][X - 1]));
            top[r] *= cs[r];
            raise = raise || top[r] > m[r] + RAISE;
        }
        if (__any_sync(0xffffffffu, raise)) {   // some key exceeds its row's maximum by enough
            float f[R];
            far = false;
#pragma unroll
            for (int r = 0; r < R; r++) {
#pragma unroll
                for (int x = PACK ? 2 : 4; x < 32; x = x == 2 ? 4 : 2 * x) top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], x));
                const float mx = fmaxf(m[r], top[r]);
                f[r] = m[r] == -INFINITY ? 0.f : ex2(m[r] - mx);   // nothing was summed before the first key
                m[r] = mx;
                l[r] *= f[r];
                far = far || (fabsf(mx) >= FAR && mx > -INFINITY);
            }
            far = __any_sync(0xffffffffu, far);
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < D / 16; j++)
#pragma unroll
                    for (int x = 0; x < 4; x++) o[nt][j][x] *= f[2 * nt + (x & 1)];
        }
        uint32_t hi[NT][4], lo[NT][4];   // P^T fragments of keys 8 x ...
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float pw[2][X];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int r = 2 * nt + u;
                const float base = m[r] == -INFINITY ? 0.f : m[r] - P_BIAS;
#pragma unroll
                for (int x = 0; x < X; x++) pw[u][x] = ex2(fmaf(sv[r][x], cs[r], -base));
            }
            if (poison || far) {
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int x = 0; x < X; x++) {
                        const int r = 2 * nt + u;
                        const float top = m[r] == -INFINITY ? 0.f : m[r];
                        if (far) pw[u][x] = ex2(__fsub_rn(__fmul_rn(sv[r][x], cs[r]), top) + P_BIAS);
                        if ((poison >> (key1 - key0 + 8 * x) & 1) && key1 + 8 * x < limit[r]) pw[u][x] = NAN;
                    }
            }
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int x = 0; x < X; x++) l[2 * nt + u] += pw[u][x];
            if (PACK) {   // t < 2 gets the hi halves of all 32 keys, t >= 2 the lo halves
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    uint32_t h, k;
                    split(pw[0][x], pw[1][x], h, k);
                    const uint32_t other = __shfl_xor_sync(0xffffffffu, t < 2 ? k : h, 2);
                    hi[nt][x] = transpose8(t < 2 ? h : other);
                    hi[nt][2 + x] = transpose8(t < 2 ? other : k);
                }
            } else {
#pragma unroll
                for (int x = 0; x < X; x++) {
                    split(pw[0][x], pw[1][x], hi[nt][x], lo[nt][x]);
                    hi[nt][x] = transpose8(hi[nt][x]);
                    lo[nt][x] = transpose8(lo[nt][x]);
                }
            }
        }

        // ---- O^T += V^T P^T, 16 keys at a time
#pragma unroll
        for (int kb = 0; kb < 2; kb++) {
            uint32_t w[4][D / 64];   // keys 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
            for (int y = 0; y < 4; y++) {
                const uint8_t* at = st + v_at[y & 1] + (16 * kb + (y >> 1) * 8) * S::ROW;
                if constexpr (D == 64) {
                    w[y][0] = *reinterpret_cast<const uint32_t*>(at);
                } else if constexpr (D == 128) {
                    const uint2 v = *reinterpret_cast<const uint2*>(at);
                    w[y][0] = v.x; w[y][1] = v.y;
                } else {
                    const uint4 v = *reinterpret_cast<const uint4*>(at);
                    w[y][0] = v.x; w[y][1] = v.y; w[y][2] = v.z; w[y][3] = v.w;
                }
            }
#pragma unroll
            for (int wi = 0; wi < D / 64; wi++) {
                const Scale sa = scale_of(kv_scales_to_half(vs[kb][0][wi / 2 % VG]));
                const Scale sb = scale_of(kv_scales_to_half(vs[kb][1][wi / 2 % VG]));
#pragma unroll
                for (int half = 0; half < 2; half++) {   // channels 0-3, 4-7 of the words
                    const uint32_t sel = half ? 0x7632 : 0x5410;
                    uint32_t h0[4], h1[4];
                    dequantise(__byte_perm(w[0][wi], w[1][wi], sel), sa, masks, h0);
                    dequantise(__byte_perm(w[2][wi], w[3][wi], sel), sb, masks, h1);
#pragma unroll
                    for (int j = 0; j < 2; j++) {   // channels 2j, 2j + 1 of the four
                        const uint32_t va[4] = {h0[2 * j], h0[2 * j + 1], h1[2 * j], h1[2 * j + 1]};
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            mma(o[nt][4 * wi + 2 * half + j], va, hi[nt][2 * kb], hi[nt][2 * kb + 1]);
                            if (!PACK) mma(o[nt][4 * wi + 2 * half + j], va, lo[nt][2 * kb], lo[nt][2 * kb + 1]);
                        }
                    }
                }
            }
        }
    }
    asm volatile("cp.async.wait_all;");

    // ---- merge the warps
#pragma unroll
    for (int r = 0; r < R; r++) {
#pragma unroll
        for (int x = PACK ? 2 : 4; x < 32; x = x == 2 ? 4 : 2 * x) l[r] += __shfl_xor_sync(0xffffffffu, l[r], x);
        const int c = row_at(r);
        if (g == 0) { sm_m[warp][c] = m[r]; sm_l[warp][c] = l[r]; }
    }
    if (PACK) {
#pragma unroll
        for (int x = 0; x < D / 4; x++) o[0][x >> 2][x & 3] += __shfl_xor_sync(0xffffffffu, o[0][x >> 2][x & 3], 2);
    }
    __syncthreads();   // every ring is idle
    float* so = reinterpret_cast<float*>(smem + S::Q_BYTES);
#pragma unroll
    for (int r = 0; r < R; r++) {
        float* at = so + (warp * COLS + row_at(r)) * S::O_LD + g * (D / 8);
#pragma unroll
        for (int j = 0; j < D / 16; j += 2)
            if (!PACK || t < 2)
                *reinterpret_cast<float4*>(at + 2 * j) = make_float4(o[r >> 1][j][r & 1], o[r >> 1][j][2 + (r & 1)],
                                                                     o[r >> 1][j + 1][r & 1], o[r >> 1][j + 1][2 + (r & 1)]);
    }
    __syncthreads();
    for (int x = tid; x < cols * (D / 4); x += THREADS) {
        const int c = x / (D / 4), d = x % (D / 4) * 4, ci = block * COLS + c;
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; w++) M = fmaxf(M, sm_m[w][c]);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            // a warp without a key has l = 0, or NaN where every score it saw was NaN
            const float f = sm_m[w][c] == -INFINITY ? 1.f : ex2(sm_m[w][c] - M);
            L += f * sm_l[w][c];
            const float4 v = *reinterpret_cast<const float4*>(so + (w * COLS + c) * S::O_LD + d);
            acc.x += f * v.x; acc.y += f * v.y; acc.z += f * v.z; acc.w += f * v.w;
        }
        const size_t row = (size_t)(first + ci / group) * hq + head * group + ci % group;
        if (CLUSTER && parts > 1) {
            reinterpret_cast<float4*>(smem)[x] = acc;   // q's fragments are done with
            if (d == 0) cl_ml[c] = make_float2(M, L);
        } else if (parts == 1) {
            store4(out + row * D + d, acc, L, p.v_unit);
        } else {
            const size_t at = row * sp.splits + split_id;
            *reinterpret_cast<float4*>(part_o + at * D + d) = acc;
            if (d == 0) part_ml[at] = make_float2(M, L);
        }
    }
    if (!CLUSTER || parts == 1) return;
    // out row = sum over the chunks of 2^(m - M) o / sum of 2^(m - M) l, the row's channels shared out over the cluster
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    for (int x = split_id * THREADS + tid; x < cols * (D / 4); x += parts * THREADS) {
        const int c = x / (D / 4), ci = block * COLS + c;
        float2 ml[MAX_CLUSTER];
        float4 v[MAX_CLUSTER];
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int r = 0; r < MAX_CLUSTER; r++)
            if (r < parts) {
                ml[r] = *cl.map_shared_rank(&cl_ml[c], r);
                v[r] = *cl.map_shared_rank(reinterpret_cast<float4*>(smem) + x, r);
                M = fmaxf(M, ml[r].x);
            }
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int r = 0; r < MAX_CLUSTER; r++)
            if (r < parts) {
                const float f = ml[r].x == -INFINITY ? 1.f : ex2(ml[r].x - M);   // a chunk without a visible key holds zeros (or NaN)
                L += f * ml[r].y;
                acc.x += f * v[r].x; acc.y += f * v[r].y; acc.z += f * v[r].z; acc.w += f * v[r].w;
            }
        store4(out + ((size_t)(first + ci / group) * hq + head * group + ci % group) * D + x % (D / 4) * 4, acc, L, p.v_unit);
    }
    cl.sync();   // nobody leaves while its sums are read
}

// out row = sum over its chunks of 2^(m - M) o / sum of 2^(m - M) l; one CTA of JOIN warps per row, chunk c is warp
// c % JOIN's. A warp asks for 8 chunks before it knows their weights.
template <int D, int JOIN>
__global__ void __launch_bounds__(32 * JOIN) k_attn_paged_join(float* __restrict__ out, int hq, KvBatchDev b, float v_unit, Split sp,
                                                               const float* __restrict__ part_o, const float2* __restrict__ part_ml) {
    constexpr int N = D / 32, BATCH = 8;
    using Piece = std::conditional_t<N == 2, float2, float4>;
    constexpr int PIECES = N * 4 / (int)sizeof(Piece), W = sizeof(Piece) / 4;
    __shared__ float sm_l[JOIN];
    __shared__ __align__(16) float sm_o[JOIN][D];
    const int s = blockIdx.z, i = blockIdx.y, h = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int first, count, behind;
    kv_new_tokens(b, s, first, count, behind);
    const int keys = min(max(b.seq_len[s], 0), b.max_len), parts = chunks_of(keys, sp.chunk);
    asm volatile("griddepcontrol.wait;" ::: "memory");   // also before an early return: the next kernel waits for this one only
    if (i >= count || parts <= 1) return;
    const size_t row = (size_t)(first + i) * hq + h;
    const float2* ml = part_ml + row * sp.splits;
    const float* po = part_o + row * sp.splits * D + lane * W;
    Piece v[BATCH][PIECES];
    auto fetch = [&](int c0) {
#pragma unroll
        for (int x = 0; x < BATCH; x++)
            if (c0 + x * JOIN < parts)
#pragma unroll
                for (int y = 0; y < PIECES; y++) v[x][y] = *reinterpret_cast<const Piece*>(po + (size_t)(c0 + x * JOIN) * D + 32 * W * y);
    };
    fetch(warp);
    float M = -INFINITY;   // every warp finds the maximum by itself
    for (int c = lane; c < parts; c += 32) M = fmaxf(M, ml[c].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    float l = 0.f, o[N];
#pragma unroll
    for (int n = 0; n < N; n++) o[n] = 0.f;
    for (int c0 = warp; c0 < parts; c0 += BATCH * JOIN) {
        if (c0 > warp) fetch(c0);
        const int c = c0 + lane * JOIN;
        float f = 0.f;
        if (lane < BATCH && c < parts) {
            const float2 w = ml[c];
            f = w.x == -INFINITY ? 1.f : ex2(w.x - M);   // a chunk without a visible key holds zeros (or NaN)
            l += f * w.y;
        }
#pragma unroll
        for (int x = 0; x < BATCH; x++) {
            const float fx = __shfl_sync(0xffffffffu, f, x);
            if (c0 + x * JOIN < parts)
#pragma unroll
                for (int n = 0; n < N; n++) o[n] = fmaf(fx, reinterpret_cast<const float*>(&v[x][n / W])[n % W], o[n]);
        }
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
    if (lane == 0) sm_l[warp] = l;
#pragma unroll
    for (int n = 0; n < N; n++) sm_o[warp][lane * W + n / W * 32 * W + n % W] = o[n];
    __syncthreads();
    float L = 0.f;
#pragma unroll
    for (int w = 0; w < JOIN; w++) L += sm_l[w];
    const float inv = weighed(L);
    for (int d = threadIdx.x; d < D; d += 32 * JOIN) {
        float acc = 0.f;
#pragma unroll
        for (int w = 0; w < JOIN; w++) acc += sm_o[w][d];
        out[row * D + d] = acc * inv * v_unit;
    }
}

lancius_error bad(lancius_error e) { lancius_set_error(e); return e; }

// Rows of q per CTA. Up to 4 fit one operand with both halves of q (half the MMAs); more rows share the cost of turning
// the codes into operands, as far as the accumulators allow. Rows over that are spread evenly.
int block_rows(int D, int rows) {
    if (rows <= 4) return 4;
    const int most = D == 256 ? 16 : 24, n = (rows + most - 1) / most;
    return ((rows + n - 1) / n + 7) / 8 * 8;
}
size_t row_blocks(int D, int rows) { const int n = block_rows(D, rows); return ((size_t)rows + n - 1) / n; }

template <int N>
using Int = std::integral_constant<int, N>;

// f(Int<D>, Int<rows of q per CTA>)
template <typename F>
auto with_shape(int D, int rows, F f) {
    const int n = block_rows(D, rows);
    auto of = [&](auto d) {
        constexpr int C = decltype(d)::value;
        if (n == 4) return f(d, Int<4>());
        if (n == 8) return f(d, Int<8>());
        if constexpr (C <= 128) if (n == 24) return f(d, Int<24>());
        return f(d, Int<16>());
    };
    return D == 64 ? of(Int<64>()) : D == 128 ? of(Int<128>()) : of(Int<256>());
}

// Keys per CTA. Few keys: every CTA that fits on the GPU gets one chunk (131072 keys of one sequence, 8 heads of 128, when
// first measured: 47.5 us in one round of CTAs, 54.9 in two, 66.7 in three). Many keys: rounds of at most ROUND, as short
// ones cost more starts and joins and long ones an idle end (64 sequences of up to 8000 keys, 8 heads with 8 rows: 146.8 us
// with 512 keys, 137.4 with 1024, 135.6 with 1280, 135.8 with 1536; 32 of up to 8192, 8 heads with one: 71.0, 69.3, 69.2,
// 70.6). Sequences of a batch are taken as three quarters of the longest. A multiple of one tile per warp.
// Up to 8 chunks of up to 8 rows, where all CTAs run at once, join as a cluster (777 keys: 5.0 us in one launch, 5.4 in two).
Split plan(const KvPagesDev& p, const KvBatchDev& b, int D, int group) {
    const int rows = group * b.max_new;
    const size_t slots = LCU_SMS * with_shape(D, rows, [](auto d, auto n) { return (size_t)Shape<d, n>::RESIDENT; });
    const size_t ctas = (size_t)b.n_seqs * p.heads * row_blocks(D, rows), len = b.max_len > 0 ? b.max_len : 1;
    const size_t keys = len * ctas / 4 * (b.n_seqs > 1 ? 3 : 4);
    size_t chunk = (keys + slots - 1) / slots;
    const size_t most = D == 256 ? ROUND : MAX_CHUNK;
    if (chunk > most) chunk /= (chunk + ROUND - 1) / ROUND;
    constexpr size_t STEP = TILE * WARPS;
    chunk = (chunk + STEP - 1) / STEP * STEP;
    if (chunk < STEP) chunk = STEP;
    if (chunk > most) chunk = most;
    const size_t splits = (len + chunk - 1) / chunk;
    return Split{(int)chunk, (int)splits, rows <= 8 && splits > 1 && splits <= MAX_CLUSTER && splits * ctas <= slots};
}
size_t part_rows(const KvBatchDev& b, size_t hq, Split sp) { return (size_t)b.n_tokens * hq * sp.splits; }

lancius_error check_call(const lcu_kv_pages* pages, const lcu_kv_batch* batch, size_t n_q_heads, KvPagesDev* p, KvBatchDev* b) {
    lancius_error e = lcu_kv_describe(pages, batch, p, b);
    if (e != LANCIUS_ERROR_OK) return e;
    if (n_q_heads > 65535 || n_q_heads % pages->n_heads || b->max_new > 65535 ||
        n_q_heads / pages->n_heads * b->max_new > (size_t)INT32_MAX / 2)
        return bad(LANCIUS_ERROR_SHAPE_MISMATCH);
    const Split sp = plan(*p, *b, (int)pages->head_dim, (int)(n_q_heads / pages->n_heads));
    if ((size_t)sp.splits * row_blocks((int)pages->head_dim, (int)(n_q_heads / pages->n_heads) * b->max_new) > (size_t)INT32_MAX ||
        part_rows(*b, n_q_heads, sp) > (size_t)1 << 40)
        return bad(LANCIUS_ERROR_SHAPE_MISMATCH);
    return LANCIUS_ERROR_OK;
}

template <int D, int ROWS, bool CLUSTER>
lancius_error launch(float* out, const float* q, size_t q_ld, int hq, const KvPagesDev& p, const KvBatchDev& b, Split sp,
                     float* part_o, float2* part_ml, cudaStream_t st) {
    using S = Shape<D, ROWS>;
    static std::atomic<unsigned long long> allowed{0};   // devices on which the kernel may use its shared memory
    auto kernel = k_attn_paged<D, ROWS, CLUSTER>;
    cudaError_t ce = lcu_allow_smem(allowed, kernel, S::SMEM);
    if (ce != cudaSuccess) return lcu_check_cuda(ce);
    const dim3 grid((unsigned)(sp.splits * row_blocks(D, hq / p.heads * b.max_new)), (unsigned)p.heads, (unsigned)b.n_seqs);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    cfg.gridDim = grid;
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = CLUSTER;
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = sp.splits;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    Scores scores;
    scores.factor = (float)frexp(16 * 1.4426950408889634 / sqrt((double)D) * p.k_unit, &scores.exponent);
    ce = cudaLaunchKernelEx(&cfg, kernel, out, q, q_ld, q_ld % 4 == 0 && (uintptr_t)q % 16 == 0, hq, p, b,
                            scores, sp, part_o, part_ml);
    if (ce != cudaSuccess) {
        cudaGetLastError();
        return lcu_check_cuda(ce);
    }
    lcu_note_launch();
    if (sp.splits == 1 || CLUSTER) return lcu_launch_status();
    ce = cudaGetLastError();
    if (ce != cudaSuccess) return lcu_check_cuda(ce);
    cfg = {};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // starts while the chunks finish
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)hq, (unsigned)b.max_new, (unsigned)b.n_seqs);
    const bool many = sp.splits > 16;
    cfg.blockDim = dim3(many ? 512 : 128);
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    ce = cudaLaunchKernelEx(&cfg, many ? k_attn_paged_join<D, 16> : k_attn_paged_join<D, 4>, out, hq, b, p.v_unit, sp, (const float*)part_o, (const float2*)part_ml);
    if (ce != cudaSuccess) {
        cudaGetLastError();
        return lcu_check_cuda(ce);
    }
    lcu_note_launch();
    return lcu_launch_status();
}

}  // namespace

extern "C" {

int* lcu_attn_paged_fault_addr(void) {
    void* p = nullptr;
    if (!g_used.load(std::memory_order_relaxed)) return nullptr;
    return cudaGetSymbolAddress(&p, g_attn_paged_fault) == cudaSuccess ? static_cast<int*>(p) : nullptr;
}

size_t lcu_attention_paged_workspace(const lcu_kv_pages* pages, const lcu_kv_batch* batch, size_t n_q_heads) {
    KvPagesDev p;
    KvBatchDev b;
    if (check_call(pages, batch, n_q_heads, &p, &b) != LANCIUS_ERROR_OK || !b.n_seqs || !b.n_tokens || !n_q_heads) return 0;
    const Split sp = plan(p, b, (int)pages->head_dim, (int)(n_q_heads / pages->n_heads));
    return sp.splits == 1 || sp.cluster ? 0 : part_rows(b, n_q_heads, sp) * (pages->head_dim + 2) * sizeof(float);
}

lancius_error lcu_attention_paged(float* out, const float* q, size_t q_ld, size_t n_q_heads, const lcu_kv_pages* pages,
                                  const lcu_kv_batch* batch, void* workspace, size_t workspace_bytes, void* stream) {
    KvPagesDev p;
    KvBatchDev b;
    lancius_error e = check_call(pages, batch, n_q_heads, &p, &b);
    if (e != LANCIUS_ERROR_OK) return e;
    if (!b.n_seqs || !b.n_tokens || !n_q_heads) return LANCIUS_ERROR_OK;
    if (!out || !q) return bad(LANCIUS_ERROR_NULL_PTR);
    const size_t D = pages->head_dim;
    if (q_ld < n_q_heads * D) return bad(LANCIUS_ERROR_SHAPE_MISMATCH);
    const int hq = (int)n_q_heads;
    const Split sp = plan(p, b, (int)D, hq / p.heads);
    float* part_o = nullptr;
    float2* part_ml = nullptr;
    if (sp.splits > 1 && !sp.cluster) {
        const size_t rows = part_rows(b, n_q_heads, sp);
        if (!workspace) return bad(LANCIUS_ERROR_NULL_PTR);
        if ((uintptr_t)workspace & 15u) return bad(LANCIUS_ERROR_UNSUPPORTED_DTYPE);
        if (workspace_bytes < rows * (D + 2) * sizeof(float)) return bad(LANCIUS_ERROR_OVERFLOW);
        part_o = static_cast<float*>(workspace);
        part_ml = reinterpret_cast<float2*>(part_o + rows * D);
    }
    cudaStream_t st = lcu_as_stream(stream);
    g_used.store(true, std::memory_order_relaxed);
    return with_shape((int)D, hq / p.heads * b.max_new,
                      [&](auto d, auto n) {
                          if constexpr (n <= 8)
                              if (sp.cluster) return launch<d, n, true>(out, q, q_ld, hq, p, b, sp, part_o, part_ml, st);
                          return launch<d, n, false>(out, q, q_ld, hq, p, b, sp, part_o, part_ml, st);
                      });
}

}  // extern "C"
