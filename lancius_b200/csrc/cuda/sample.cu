// Drawing a token per row of logits (lcu_sample).
//
// w_i = exp((x_i - max) / t). Every filter keeps a prefix of the rank order (logit falling, index rising), so a
// row's kept set is one cut: a logit tau and a last index among the logits equal to tau. The cut is found by a
// radix search over order-preserving 32-bit keys: a histogram of 2048 bins of the current key range, the bin in
// which the count (top-k) or the mass (top-p) reaches its target, then that bin as the next range, until a bin is
// one key. Masses of bins are 64-bit fixed point, so the atomics' order does not matter: 2^44 for the largest
// weight, 2^18 tokens fit 62 bits. The draw sums weights in FP64 in a fixed order and draws in index order,
// which needs no sort.
#include "lcu_internal.h"
#include <math.h>

namespace {

constexpr int THREADS = 1024, WARPS = THREADS / 32, BINS = 2048;
constexpr double FIXED = 17592186044416.0;   // 2^44
constexpr size_t MAX_VOCAB = 262144;
typedef unsigned long long u64;

__device__ __forceinline__ float clean(float x) { return x == x ? x + 0.f : -INFINITY; }   // NaN -> -inf, -0 -> +0
// keys order like the numbers
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct Row {
    const float* x;
    int n;
    float max;
    double t;
    uint32_t tau;   // kept: key > tau, or key == tau and index <= last
    int last;
};

__device__ __forceinline__ bool kept(const Row& r, uint32_t key, int i) { return key > r.tau || (key == r.tau && i <= r.last); }
__device__ __forceinline__ double weight(const Row& r, float x) {
    if (x == r.max) return 1.0;
    const double w = exp(((double)x - (double)r.max) / r.t);
    return w > 0.0 ? w : 0.0;   // also -inf / inf
}

struct Shared {
    u64 mass[BINS];
    uint32_t count[BINS];
    u64 warp_sum[WARPS];
    double warp_mass[WARPS];
    float warp_max[WARPS];
    int warp_at[WARPS];
    int bin, found, ties;
    u64 before, in_bin, total;
};

// inclusive scan of one value per thread over the block
__device__ u64 block_scan(Shared& sh, u64 v) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 31) sh.warp_sum[warp] = v;
    __syncthreads();
    u64 add = 0;
    for (int w = 0; w < warp; w++) add += sh.warp_sum[w];
    return v + add;
}

// Moves the row's cut to the rank at which the running count (MASS = false) or mass reaches `target`; p: target =
// p * the mass of what is kept so far.
template <bool MASS>
__device__ void cut(Shared& sh, Row& r, u64 k, double p) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t lo = r.tau, hi = key_of(r.max);
    u64 before = 0;
    double target = (double)k;
    for (int round = 0;; round++) {
        const uint32_t span = hi - lo;
        const int sh_bits = max(0, 32 - __clz(span) - 11);
        __syncthreads();
        for (int i = tid; i < BINS; i += THREADS) { sh.mass[i] = 0; sh.count[i] = 0; }
        __syncthreads();
        for (int i = tid; i < r.n; i += THREADS) {
            const float x = clean(r.x[i]);
            const uint32_t key = key_of(x);
            if (key < lo || key > hi || !kept(r, key, i)) continue;
            const int bin = (hi - key) >> sh_bits;
            atomicAdd(&sh.count[bin], 1u);
            if (MASS) atomicAdd(&sh.mass[bin], (u64)__double2ll_rn(weight(r, x) * FIXED));
        }
        __syncthreads();
        u64 a = MASS ? sh.mass[2 * tid] : sh.count[2 * tid], c = MASS ? sh.mass[2 * tid + 1] : sh.count[2 * tid + 1];
        const u64 upto = block_scan(sh, a + c);
        if (tid == THREADS - 1) { sh.total = upto; sh.found = 0; }
        __syncthreads();
        if (round == 0) {
            if (MASS) target = fmax(p * (double)sh.total, 0.5);
            else if (sh.total <= k) return;
        }
        const u64 e0 = before + upto - a - c;
        if (!((double)e0 >= target) && (double)(e0 + a) >= target) { sh.bin = 2 * tid; sh.before = e0; sh.in_bin = a; sh.found = 1; }
        else if (!((double)(e0 + a) >= target) && (double)(e0 + a + c) >= target) {
            sh.bin = 2 * tid + 1; sh.before = e0 + a; sh.in_bin = c; sh.found = 1;
        }
        __syncthreads();
        if (!sh.found) return;   // the whole mass is needed (rounding of the target)
        const int bin = sh.bin;
        before = sh.before;
        hi -= (uint32_t)bin << sh_bits;
        if (sh_bits) {
            const uint32_t low = hi - ((1u << sh_bits) - 1);
            lo = low > lo && low <= hi ? low : lo;
            continue;
        }
        // one key: how many of its equals, by rising index
        const u64 ties = sh.count[bin];
        u64 keep;
        if (MASS) {
            const double each = (double)sh.in_bin / (double)ties, need = ceil((target - (double)before) / each);
            keep = need < 1 ? 1 : need > (double)ties ? ties : (u64)need;
        } else keep = k - before;
        if (keep == ties) { if (hi > r.tau) { r.tau = hi; r.last = 0x7fffffff; } return; }
        const int seg = (r.n + WARPS - 1) / WARPS, s0 = warp * seg, s1 = min(r.n, s0 + seg);
        u64 n = 0;
        for (int i = s0 + lane; i - lane < s1; i += 32) {
            const uint32_t key = i < s1 ? key_of(clean(r.x[i])) : 0;
            n += __popc(__ballot_sync(0xffffffffu, i < s1 && key == hi && kept(r, key, i)));
        }
        __syncthreads();
        if (lane == 0) sh.warp_sum[warp] = n;
        __syncthreads();
        u64 ahead = 0;
        for (int w = 0; w < warp; w++) ahead += sh.warp_sum[w];
        if (ahead < keep && ahead + n >= keep) {
            for (int i = s0 + lane; i - lane < s1; i += 32) {
                const uint32_t key = i < s1 ? key_of(clean(r.x[i])) : 0;
                const unsigned hits = __ballot_sync(0xffffffffu, i < s1 && key == hi && kept(r, key, i));
                const int c2 = __popc(hits);
                if (ahead + c2 >= keep) {
                    int skip = (int)(keep - ahead) - 1;
                    unsigned h = hits;
                    while (skip--) h &= h - 1;
                    if (lane == 0) sh.ties = i - lane + __ffs(h) - 1;
                    break;
                }
                ahead += c2;
            }
        }
        __syncthreads();
        r.tau = hi;
        r.last = sh.ties;
        return;
    }
}

__global__ void __launch_bounds__(THREADS) k_sample(int32_t* __restrict__ token, const float* __restrict__ logits, size_t ld, int n,
                                                    const float* temperature, const int32_t* top_k, const float* top_p,
                                                    const float* min_p, const float* u) {
    __shared__ Shared sh;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Row r;
    r.x = logits + (size_t)row * ld;
    r.n = n;
    float m = -INFINITY;
    int at = 0x7fffffff;
    for (int i = tid; i < n; i += THREADS) {
        const float x = clean(r.x[i]);
        if (x > m) { m = x; at = i; }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o);
        const int a2 = __shfl_xor_sync(0xffffffffu, at, o);
        if (m2 > m || (m2 == m && a2 < at)) { m = m2; at = a2; }
    }
    if (lane == 0) { sh.warp_max[warp] = m; sh.warp_at[warp] = at; }
    __syncthreads();
    for (int w = 0; w < WARPS; w++)
        if (sh.warp_max[w] > m || (sh.warp_max[w] == m && sh.warp_at[w] < at)) { m = sh.warp_max[w]; at = sh.warp_at[w]; }
    const float t = temperature ? temperature[row] : 1.f;
    if (m == -INFINITY || !(t > 0.f)) {
        if (tid == 0) token[row] = m == -INFINITY ? -1 : at;
        return;
    }
    r.max = m;
    r.t = t;
    r.tau = key_of(-INFINITY) + 1;
    r.last = 0x7fffffff;
    const float mp = min_p ? min_p[row] : 0.f;
    if (mp > 0.f) r.tau = max(r.tau, key_of(fminf(m, __double2float_ru((double)m + (double)t * log((double)fminf(mp, 1.f))) + 0.f)));
    const int k = top_k ? top_k[row] : 0;
    if (k > 0 && k < n) cut<false>(sh, r, k, 0.0);
    const float p = top_p ? top_p[row] : 1.f;
    if (p < 1.f) cut<true>(sh, r, 0, p);

    const int seg = ((n + WARPS - 1) / WARPS + 31) / 32 * 32, s0 = warp * seg, s1 = min(n, s0 + seg);
    double mass = 0.0;
    int last = -1;
    for (int i = s0 + lane; i < s1; i += 32) {
        const float x = clean(r.x[i]);
        if (kept(r, key_of(x), i)) {
            const double w = weight(r, x);
            mass += w;
            if (w > 0.0) last = i;
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        mass += __shfl_xor_sync(0xffffffffu, mass, o);
        last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
    }
    __syncthreads();
    if (lane == 0) { sh.warp_mass[warp] = mass; sh.warp_at[warp] = last; }
    __syncthreads();
    if (warp != 0) return;
    double total = 0.0;
    for (int w = 0; w < WARPS; w++) { total += sh.warp_mass[w]; last = max(last, sh.warp_at[w]); }
    const double target = (double)u[row] * total;
    double ahead = 0.0;
    int w = 0;
    for (; w < WARPS - 1; w++) {
        if (ahead + sh.warp_mass[w] > target) break;
        ahead += sh.warp_mass[w];
    }
    int drawn = last;
    const int d0 = w * seg, d1 = min(n, d0 + seg);
    bool done = false;
    int in_seg = -1;
    for (int i = d0 + lane; i - lane < d1 && !done; i += 32) {
        double wi = 0.0;
        if (i < d1) {
            const float x = clean(r.x[i]);
            if (kept(r, key_of(x), i)) wi = weight(r, x);
        }
        double c = wi;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double v = __shfl_up_sync(0xffffffffu, c, o);
            if (lane >= o) c += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, wi > 0.0 && ahead + c > target), any = __ballot_sync(0xffffffffu, wi > 0.0);
        if (hit) { drawn = i - lane + __ffs(hit) - 1; done = true; }
        else if (any) in_seg = i - lane + 31 - __clz(any);
        ahead += __shfl_sync(0xffffffffu, c, 31);
    }
    if (!done && in_seg >= 0 && w < WARPS - 1) drawn = in_seg;   // the segment's sums differ in their last bit
    if (lane == 0) token[row] = drawn;
}

lancius_error bad(lancius_error e) { lancius_set_error(e); return e; }

}  // namespace

extern "C" lancius_error lcu_sample(int32_t* token, const float* logits, size_t ld, size_t rows, size_t vocab,
                                    const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                                    const float* u, void* stream) {
    if (!rows) return LANCIUS_ERROR_OK;
    if (!token || !logits || !u) return bad(LANCIUS_ERROR_NULL_PTR);
    if (!vocab || vocab > MAX_VOCAB || ld < vocab || rows > (size_t)INT32_MAX) return bad(LANCIUS_ERROR_SHAPE_MISMATCH);
    k_sample<<<(unsigned)rows, THREADS, 0, lcu_as_stream(stream)>>>(token, logits, ld, (int)vocab, temperature, top_k, top_p, min_p, u);
    lcu_note_launch();
    return lcu_launch_status();
}
