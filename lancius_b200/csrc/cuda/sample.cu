// Drawing a token per row of logits (lcu_sample).
//
// w_i = exp((x_i - max) / t). Every filter keeps a prefix of the rank order (logit falling, index rising), so a row's kept
// set is one cut: a logit tau and a last index among the logits equal to tau. No sort is needed: a histogram of the
// logits finds the bin in which the count (top-k) or the mass (top-p) reaches its target, and the few logits of that
// bin are ranked against each other; where a bin holds more than LIST of them (many equal logits), a radix search
// over order-preserving 32-bit keys narrows it down to one key first. The draw adds weights in index order.
//
// Masses of bins are 64-bit fixed point, so the order of the atomics does not matter: 2^44 for the largest weight, and
// 2^18 tokens fit 62 bits. The draw's sums are FP64 in a fixed order, on every path. Weights are FP64: with
// FP32 ones a drawn token would differ from the exact one in about one row of a thousand.
//
// k_sample: a row is spread over a cluster of 1 to 8 CTAs that hold it in shared memory through all passes and exchange
// histograms and sums through each other's shared memory; HBM is read once. Bound by the passes' instructions and by
// the chain of barriers between them, not by HBM: of 29 us that a cluster needs for a quarter of 50021 logits a CTA with top-p,
// the load takes 4, the histogram 8, its scan 3, the list 3, the ranking 1, the draw's weights 6, the draw 1.
// 32000 logits with every filter: 8.0 us; 200 x 50021 with mixed filters: 54 us (top-p alone 84, top-k of 50 alone 34).
// k_sample_open, without filters: one pass, no part of the row kept. 64 x 131072: 20.6 us, of which the loads and
// barriers alone take 9 (as greedy rows measure them) and the FP64 pipe is busy for 6: 12 instructions a logit.
#include "lcu_internal.h"
#include <cooperative_groups.h>
#include <math.h>

namespace cg = cooperative_groups;

namespace {

constexpr int THREADS = 512, WARPS = THREADS / 32, BINS = 2048, LIST = THREADS, MAX_CLUSTER = 8;
constexpr int SMALL = 256;   // candidates that one CTA finishes alone
constexpr int BLOCK = 128;   // logits whose weights are summed as one in the draw, 4 a lane
constexpr double FIXED = 17592186044416.0;   // 2^44
constexpr size_t MAX_VOCAB = 262144;
constexpr int MAX_BLOCKS = (int)(MAX_VOCAB / MAX_CLUSTER / BLOCK);
typedef unsigned long long u64;

__device__ __forceinline__ float clean(float x) { return fmaxf(x, -INFINITY) + 0.f; }   // NaN -> -inf, -0 -> +0
// keys order like the numbers
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct Shared {
    uint32_t low[BINS], high[BINS];    // of a bin: its sum (counts in low alone)
    float warp_max[WARPS], warp_min[WARPS];
    union {
        u64 list[LIST];   // key << 32 | ~index, so that larger means an earlier rank
        double block_mass[MAX_BLOCKS];   // of the draw, when the list is done with
    };
    u64 list_mass[LIST];
    double power[16];
    u64 warp_sum[WARPS];
    double mass_of[MAX_CLUSTER];   // mass_of: written by every CTA of the cluster
    float max, min, tau;
    int at, found, bin, last;
    uint32_t listed;
    u64 slice_sum, before, in_bin, total;
};

struct Row {
    const float* x;     // this CTA's part, in shared memory, cleaned
    int padded, first;  // its length and the index of its first token
    float max, min;     // of the row, min over the finite ones
    double top, rate;   // max, 16 log2(e) / t
    const double* power;   // 2^(j/16), in shared memory
    bool fresh;         // the histogram is cleared
    float tau;          // kept: logit > tau, or logit == tau and index <= last
    int last;
};

constexpr int ALL = 0x7fffffff;
__device__ __forceinline__ bool kept(const Row& r, float x, int i) {
    return x >= r.tau && (r.last == ALL || x > r.tau || r.first + i <= r.last);
}
// Calls use(logit, index in the part) for the kept logits of this CTA's part, 4 neighbours at a time per thread. The
// part is padded with -infinity, which is never kept, to a multiple of BLOCK.
template <typename Use>
__device__ __forceinline__ void for_kept(const Row& r, Use use) {
    const float4* x4 = reinterpret_cast<const float4*>(r.x);
#pragma unroll 2
    for (int j = threadIdx.x; j < r.padded / 4; j += THREADS) {
        const float4 v = x4[j];
        if (kept(r, v.x, 4 * j)) use(v.x, 4 * j);
        if (kept(r, v.y, 4 * j + 1)) use(v.y, 4 * j + 1);
        if (kept(r, v.z, 4 * j + 2)) use(v.z, 4 * j + 2);
        if (kept(r, v.w, 4 * j + 3)) use(v.w, 4 * j + 3);
    }
}
// exp((x - top) / t), rate = 16 log2(e) / t, for weights above 2^-1022. 2^(z / 16) with z = n + f, |f| <= 1/2, is a table of
// 2^(j/16) times a polynomial (table-driven exponential, Tang 1989): 1 + f q(f), q interpolating (2^(f/16) - 1) / f at the 5
// Chebyshev nodes of [-1/2, 1/2]; relative error 9e-15. 10 FP64 instructions and a conversion.
__device__ __forceinline__ double weight_of(float x, double top, double rate, const double* power) {
    constexpr double MAGIC = 6755399441055744.0;   // 1.5 * 2^52: the sum's low bits are the rounded integer
    const double d = (double)x - top, k = fma(d, rate, MAGIC);
    const int n = __double2loint(k);
    const double f = fma(d, rate, MAGIC - k);
    double p = 1.2716049516906705e-9;
    p = fma(p, f, 1.4676387238435006e-7);
    p = fma(p, f, 1.3550807778387664e-5);
    p = fma(p, f, 9.3838479262966460e-4);
    p = fma(p, f, 4.3321698784996580e-2);
    p = fma(p, f, 1.0) * power[n & 15];
    return __hiloint2double(__double2hiint(p) + ((n & ~15) << 16), __double2loint(p));
}
__device__ __forceinline__ double weight(const Row& r, float x) { return weight_of(x, r.top, r.rate, r.power); }   // of a kept one
__device__ __forceinline__ u64 fixed_weight(const Row& r, float x) {   // times 2^44, rounded
    return (u64)__double_as_longlong(fma(weight(r, x), FIXED, 4503599627370496.0)) & 0xfffffffffffffull;
}

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
    u64 add = lane < warp ? sh.warp_sum[lane] : 0;
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1) add += __shfl_xor_sync(0xffffffffu, add, o);
    return v + __shfl_sync(0xffffffffu, add, 0);
}

__device__ __forceinline__ double scan(double v) {   // inclusive, over the warp
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
    }
    return v;
}

__device__ __forceinline__ void clear(Shared& sh) {
    for (int i = threadIdx.x; i < BINS; i += THREADS) sh.low[i] = sh.high[i] = 0;
    if (threadIdx.x == 0) sh.listed = 0;
}

// One histogram over the kept logits, of counts or masses, bin_of(x) < BINS rising with the rank (or -1: not counted), and
// the bin in which the running sum, from `before` on, reaches the target, which target_of(total) makes from the sum of
// all bins.
struct Found {
    bool any;
    int bin;
    u64 before, in_bin, total;   // sum before the bin, in it, of all bins
};
template <bool MASS, bool FEW, typename Bin, typename Target>
__device__ Found find_bin(cg::cluster_group& cl, Shared& sh, Row& r, u64 before, Bin bin_of, Target target_of) {
    const int tid = threadIdx.x, lane = tid & 31, ranks = cl.num_blocks(), rank = cl.block_rank(), slice = BINS / ranks;
    if (!r.fresh) {
        cl.sync();   // nobody reads the last histogram any more
        clear(sh);
        __syncthreads();
    }
    r.fresh = false;
    for_kept(r, [&](float x, int) {
        const int bin = bin_of(x);
        if (bin < 0) return;
        if (MASS) {   // two 32-bit atomics with a carry: shared memory has no 64-bit add
            const u64 w = fixed_weight(r, x);
            const uint32_t lo = (uint32_t)w, old = atomicAdd(&sh.low[bin], lo);
            const uint32_t hi = (uint32_t)(w >> 32) + (old + lo < old);
            if (hi) atomicAdd(&sh.high[bin], hi);
        } else {
            atomicAdd(&sh.low[bin], 1u);
        }
    });
    cl.sync();
    if (FEW) {   // each CTA adds up and scans the first THREADS bins by itself: two barriers of the cluster less
        u64 here = 0, x[MAX_CLUSTER];
#pragma unroll
        for (int c = 0; c < MAX_CLUSTER; c++) x[c] = c < ranks ? cl.map_shared_rank(&sh, min(c, ranks - 1))->low[tid] : 0;
#pragma unroll
        for (int c = 0; c < MAX_CLUSTER; c++) here += x[c];
        const u64 upto = block_scan(sh, here);
        if (tid == THREADS - 1) { sh.slice_sum = upto; sh.found = 0; }
        __syncthreads();
        const u64 total = sh.slice_sum, at = before + upto - here;
        const double target = target_of(total);
        if ((double)at < target && (double)(at + here) >= target) { sh.bin = tid; sh.before = at; sh.in_bin = here; sh.found = 1; }
        __syncthreads();
        return Found{sh.found != 0, sh.bin, sh.before, sh.in_bin, total};
    }
    // each CTA adds up its slice of the bins over the cluster and scans it, q neighbours a thread
    const int b0 = rank * slice, q = max(1, slice / THREADS);
    constexpr int PER = BINS / THREADS;
    u64 v[PER], sum = 0;
#pragma unroll
    for (int k = 0; k < PER; k++) {
        const int i = q * tid + k;
        v[k] = 0;
        if (k < q && i < slice) {
            u64 x[MAX_CLUSTER];   // the remote reads are in flight together
#pragma unroll
            for (int c = 0; c < MAX_CLUSTER; c++) {
                const Shared* o = cl.map_shared_rank(&sh, min(c, ranks - 1));
                x[c] = c < ranks ? o->low[b0 + i] + (MASS ? (u64)o->high[b0 + i] << 32 : 0) : 0;
            }
#pragma unroll
            for (int c = 0; c < MAX_CLUSTER; c++) v[k] += x[c];
        }
        sum += v[k];
    }
    const u64 upto = block_scan(sh, sum);
    if (tid == THREADS - 1) { sh.slice_sum = upto; sh.found = 0; }
    cl.sync();
    u64 slices = lane < ranks ? cl.map_shared_rank(&sh, lane % ranks)->slice_sum : 0;
    u64 ahead = lane < rank ? slices : 0;
#pragma unroll
    for (int o = MAX_CLUSTER / 2; o > 0; o >>= 1) {
        slices += __shfl_xor_sync(0xffffffffu, slices, o);
        ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
    }
    const u64 total = __shfl_sync(0xffffffffu, slices, 0);
    const double target = target_of(total);
    u64 at = before + __shfl_sync(0xffffffffu, ahead, 0) + upto - sum;
#pragma unroll
    for (int k = 0; k < PER; k++) {
        if ((double)at < target && (double)(at + v[k]) >= target) {   // one bin of one thread of one CTA
            sh.bin = b0 + q * tid + k; sh.before = at; sh.in_bin = v[k]; sh.found = 1;
        }
        at += v[k];
    }
    cl.sync();
    const Shared* o = cl.map_shared_rank(&sh, lane % ranks);
    const unsigned owners = __ballot_sync(0xffffffffu, o->found);
    o = cl.map_shared_rank(&sh, owners ? __ffs(owners) - 1 : 0);
    return Found{owners != 0, o->bin, o->before, o->in_bin, total};
}

// Puts a logit on the first CTA's list (its counter is cleared with the histogram).
__device__ __forceinline__ void put(const Row& r, Shared* lead, int i, float x, u64 mass) {
    const uint32_t to = atomicAdd(&lead->listed, 1u);
    if (to >= LIST) return;
    lead->list[to] = (u64)key_of(x) << 32 | (uint32_t)~(uint32_t)(r.first + i);
    lead->list_mass[to] = mass;
}

// All of a list is on it (cluster barrier passed): the first CTA ranks it, starting from the sum `before`, and the cut moves
// to the logit at which the sum reaches the target.
template <bool MASS>
__device__ void rank_list(cg::cluster_group& cl, Shared& sh, Row& r, u64 before, double target) {
    const int tid = threadIdx.x;
    if (cl.block_rank() == 0) {
        const int n = sh.listed;
        if (tid < n) {
            const u64 me = sh.list[tid];
            u64 ahead = before;
#pragma unroll 4
            for (int j = 0; j < n; j++)
                if (sh.list[j] > me) ahead += MASS ? sh.list_mass[j] : 1;
            const u64 w = MASS ? sh.list_mass[tid] : 1;
            if ((double)ahead < target && (double)(ahead + w) >= target) {
                sh.tau = of_key((uint32_t)(me >> 32));
                sh.last = (int)~(uint32_t)me;
            }
        }
    }
    cl.sync();
    const Shared* lead = cl.map_shared_rank(&sh, 0);
    r.tau = lead->tau;
    r.last = lead->last;
}

// Cuts within the kept logits with in(x), the sum before which is `before`. False: they are more than LIST; their number
// is in the first CTA's `listed`.
template <bool MASS, typename In>
__device__ bool finish_list(cg::cluster_group& cl, Shared& sh, Row& r, u64 before, double target, In in) {
    Shared* lead = cl.map_shared_rank(&sh, 0);
    for_kept(r, [&](float x, int i) {
        if (in(x)) put(r, lead, i, x, MASS ? fixed_weight(r, x) : 0);
    });
    cl.sync();
    if (lead->listed > LIST) return false;
    rank_list<MASS>(cl, sh, r, before, target);
    return true;
}

// The kept logits with in(x) are at most SMALL and hold all of the top k: the first CTA ranks them, cuts by k and p
// and draws. Top-p's masses are fixed point, as the list's order is anybody's; the draw's are FP64, in the order of the
// indices: it may fall on a weight that is nothing next to the largest.
template <typename In>
__device__ void finish_small(cg::cluster_group& cl, Shared& sh, const Row& r, int k, double p, double u, int32_t* token, In in) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Shared* lead = cl.map_shared_rank(&sh, 0);
    for_kept(r, [&](float x, int i) {
        if (in(x)) put(r, lead, i, x, fixed_weight(r, x));
    });
    cl.sync();
    if (cl.block_rank() != 0) return;   // only the first CTA's shared memory is used from here on
    const int n = min(sh.listed, (uint32_t)LIST);
    const bool mine = tid < n;
    const u64 me = mine ? sh.list[tid] : 0, w = mine ? sh.list_mass[tid] : 0;
    const int index = (int)~(uint32_t)me;
    u64 ahead = 0;
    int rank = 0, place = 0;   // by logit, by index
    if (mine)
        for (int j = 0; j < n; j++) {
            const u64 it = sh.list[j];
            if (it > me) { rank++; ahead += sh.list_mass[j]; }
            if ((uint32_t)it > (uint32_t)me) place++;
        }
    bool keep = mine && rank < k;
    if (p < 1.0) {
        const u64 upto = block_scan(sh, keep ? w : 0);
        if (tid == THREADS - 1) sh.total = upto;
        __syncthreads();
        keep = keep && (double)ahead < fmax(p * (double)sh.total, 0.5);
    }
    if (tid == 0) { sh.at = 0x7fffffff; sh.last = -1; }
    __syncthreads();   // the list has been read
    double* weights = reinterpret_cast<double*>(sh.list_mass);
    int* indices = reinterpret_cast<int*>(sh.list);
    if (mine) {
        weights[place] = keep ? weight(r, of_key((uint32_t)(me >> 32))) : 0.0;
        indices[place] = index;
        if (keep) atomicMax(&sh.last, index);
    }
    __syncthreads();
    const double here = mine ? weights[tid] : 0.0;
    double upto = scan(here);
    double* of_warp = reinterpret_cast<double*>(sh.warp_sum);
    if (lane == 31) of_warp[warp] = upto;
    __syncthreads();
    double total = 0.0;
#pragma unroll
    for (int i = 0; i < SMALL / 32; i++) {
        if (i < warp) upto += of_warp[i];
        total += of_warp[i];
    }
    if (here > 0.0 && upto > u * total) atomicMin(&sh.at, indices[tid]);
    __syncthreads();
    if (tid == 0) *token = sh.at < 0x7fffffff ? sh.at : sh.last;
}

// Of the kept logits equal to `value`, the one that is the keep-th by index becomes the last.
__device__ void finish_ties(cg::cluster_group& cl, Shared& sh, Row& r, float value, u64 keep) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int seg = (r.padded / 32 + WARPS - 1) / WARPS * 32, s0 = warp * seg, s1 = min(r.padded, s0 + seg);
    auto hits = [&](int i) { return __ballot_sync(0xffffffffu, r.x[i] == value && kept(r, r.x[i], i)); };
    u64 n = 0;
    for (int i = s0 + lane; i < s1; i += 32) n += __popc(hits(i));
    __syncthreads();
    if (lane == 0) sh.warp_sum[warp] = n;
    cl.sync();
    u64 ahead = 0;   // hits of the segments before this warp's
    const int mine = cl.block_rank() * WARPS + warp;
    for (int c = lane; c < mine; c += 32) ahead += cl.map_shared_rank(&sh, c / WARPS)->warp_sum[c % WARPS];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
    Shared* lead = cl.map_shared_rank(&sh, 0);
    if (ahead < keep && ahead + n >= keep) {
        for (int i = s0 + lane; i < s1; i += 32) {
            unsigned h = hits(i);
            const int c = __popc(h);
            if (ahead + c >= keep) {
                for (int skip = (int)(keep - ahead) - 1; skip > 0; skip--) h &= h - 1;
                if (lane == 0) lead->last = r.first + i - lane + __ffs(h) - 1;
                break;
            }
            ahead += c;
        }
    }
    cl.sync();
    r.tau = value;
    r.last = lead->last;
}

// Bins of equal width in the logit, down to weights of 2^-144; false where the logits' range allows none.
struct ValueBins {
    float max, per, most;
    __device__ bool make(const Row& r, int bins) {
        most = (float)(bins - 1);
        const float range = fminf(r.max - r.min, 144.f * 16 / (float)r.rate);
        max = r.max;
        per = most / range;
        return range > 0.f && range < INFINITY && per < 1e30f;
    }
    __device__ __forceinline__ int operator()(float x) const {   // rounded by adding 2^23
        return __float_as_int(fminf((max - x) * per, most) + 8388608.f) & 0xffff;
    }
};

// Moves the row's cut to the rank at which the running count (MASS = false: k) or mass (p times the mass of what is
// kept so far) is reached. With a count of few candidates it draws the token at once and returns true.
template <bool MASS>
__device__ bool cut(cg::cluster_group& cl, Shared& sh, Row& r, int k, double p, double u, int32_t* token) {
    auto first_target = [&](u64 total) { return MASS ? fmax(p * (double)total, 0.5) : (double)k; };
    // The upper few thousand logits lie apart: fewer bins hold no more than a list of them each, and one pass less over
    // the cluster finds the bin (32000 logits, top-k of 50: 8.9 us, with 2048 bins 10.2).
    const bool few = !MASS && k <= 4096;
    ValueBins bin_of;
    if (bin_of.make(r, few ? THREADS : BINS)) {
        const Found f = few ? find_bin<MASS, !MASS>(cl, sh, r, 0, bin_of, first_target)
                            : find_bin<MASS, false>(cl, sh, r, 0, bin_of, first_target);
        const int bin = f.any ? f.bin : BINS;
        if (!MASS && (f.any ? f.before + f.in_bin : f.total) <= SMALL) {
            finish_small(cl, sh, r, k, p, u, token, [&](float x) { return bin_of(x) <= bin; });
            return true;
        }
        if (!f.any) return false;   // fewer than k, or all of the mass is wanted
        if ((MASS || f.in_bin <= LIST) &&
            finish_list<MASS>(cl, sh, r, f.before, first_target(f.total), [&](float x) { return bin_of(x) == bin; }))
            return false;
    }
    uint32_t lo = key_of(r.tau), hi = key_of(r.max);
    u64 before = 0;
    double target = 0.0;
    for (bool first = true;; first = false) {   // at most 3 rounds: 32 bits, 21, 10
        const int bits = max(0, 32 - __clz(hi - lo) - 11);
        auto key_bin = [&](float x) {
            const uint32_t key = key_of(x);
            return key < lo || key > hi ? -1 : (int)((hi - key) >> bits);
        };
        const Found f = find_bin<MASS, false>(cl, sh, r, before, key_bin, [&](u64 total) { return first ? first_target(total) : target; });
        if (!f.any) return false;
        if (first) target = first_target(f.total);
        before = f.before;
        hi -= (uint32_t)f.bin << bits;
        const uint32_t low = hi - ((1u << bits) - 1);
        if (low > lo && low <= hi) lo = low;
        if ((MASS || f.in_bin <= LIST || !bits) &&
            finish_list<MASS>(cl, sh, r, before, target, [&](float x) { return key_of(x) >= lo && key_of(x) <= hi; }))
            return false;
        if (bits) continue;
        const double ties = (double)cl.map_shared_rank(&sh, 0)->listed, each = (double)f.in_bin / ties;
        const double need = MASS ? fmin(fmax(ceil((target - (double)before) / each), 1.0), ties) : target - (double)before;
        finish_ties(cl, sh, r, of_key(hi), (u64)need);
        return false;
    }
}

// v: inclusive sums by lane of what each lane has, if any; the first lane that has some and whose sum, behind `ahead`,
// passes the target (32: none); ahead moves to its start. A sum's last bits depend on its order, so a lane without
// weight may seem to pass.
__device__ __forceinline__ int first_over(double v, bool any, double& ahead, double target) {
    const unsigned over = __ballot_sync(0xffffffffu, any && ahead + v > target);
    const int at = over ? __ffs(over) - 1 : 32;
    const double x = __shfl_sync(0xffffffffu, v, max(min(at, 31) - 1, 0));
    if (at > 0 && at < 32) ahead += x;
    return at;
}
// Where no lane passes, again for the last bits, the last that has some.
__device__ __forceinline__ int or_last(int at, bool any) {
    const unsigned some = __ballot_sync(0xffffffffu, any);
    return at < 32 ? at : 31 - __clz(some);
}
// One warp draws within its CTA: mine, the inclusive sums by lane of per neighbouring blocks each; block_mass, the blocks'
// sums; lane_weights(i, w), the weights of the 4 logits of the lane in the 128 at 128 i, SUBS of which make a block.
// Returns the index in the CTA's part.
template <int SUBS, typename Weights>
__device__ __forceinline__ int draw_in_part(double mine, bool mine_any, int per, int blocks, const double* block_mass, double ahead,
                                            double target, Weights lane_weights) {
    const int lane = threadIdx.x & 31;
    int at = or_last(first_over(mine, mine_any, ahead, target), mine_any);
    const int b0 = at * per, n = min(per, blocks - b0);   // per <= 8 blocks
    const double of_block = lane < n ? block_mass[b0 + lane] : 0.0;
    int block = (b0 + or_last(first_over(scan(of_block), of_block > 0.0, ahead, target), of_block > 0.0)) * SUBS;
    double w[4];
    if (SUBS > 1) {
        double of_sub = 0.0;
#pragma unroll
        for (int s = 0; s < SUBS; s++) {
            lane_weights(block + s, w);
            double v = (w[0] + w[1]) + (w[2] + w[3]);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            if (lane == s) of_sub = v;
        }
        block += or_last(first_over(scan(of_sub), of_sub > 0.0, ahead, target), of_sub > 0.0);
    }
    lane_weights(block, w);
    const double four = (w[0] + w[1]) + (w[2] + w[3]);
    at = or_last(first_over(scan(four), four > 0.0, ahead, target), four > 0.0);
    int drawn = 0;
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (w[j] > 0.0 && !(ahead > target)) {
            drawn = j;
            ahead += w[j];
        }
    return __shfl_sync(0xffffffffu, block * BLOCK + 4 * lane + drawn, at);
}

// RESIDENT CTAs per SM: 3 take 40 registers a thread and spill 464 bytes of it, which pays as soon as there are more CTAs than
// 2 per SM hold (when first measured, 200 x 50021, mixed filters: 56.5 us, with 2 62.8; one row of 32000: 9.9 and 9.7)
template <int RESIDENT>
__global__ void __launch_bounds__(THREADS, RESIDENT) k_sample(int32_t* __restrict__ token, const float* __restrict__ logits, size_t ld,
                                                              int vocab, int part, int vec, const float* temperature,
                                                              const int32_t* top_k, const float* top_p, const float* min_p,
                                                              const float* u) {
    extern __shared__ __align__(16) float part_of_row[];
    __shared__ Shared sh;
    cg::cluster_group cl = cg::this_cluster();
    const int ranks = cl.num_blocks(), rank = cl.block_rank(), row = blockIdx.x / ranks;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Row r;
    r.x = part_of_row;
    r.first = rank * part;
    const int n = max(0, min(part, vocab - r.first));
    r.padded = (n + BLOCK - 1) / BLOCK * BLOCK;
    const float* src = logits + (size_t)row * ld + r.first;
    const float t = temperature ? temperature[row] : 1.f, mp = min_p ? min_p[row] : 0.f, p = top_p ? top_p[row] : 1.f;
    const int k = top_k ? top_k[row] : 0;
    const bool greedy = !(t > 0.f), cuts = !greedy && ((k > 0 && k < vocab) || p < 1.f);
    const double rate = 16 * 1.4426950408889634074 / (double)t;
    float m = -INFINITY, lowest = INFINITY;   // lowest of the finite ones, where a cut will want it
    auto take = [&](float x) {
        x = clean(x);
        m = fmaxf(m, x);
        if (cuts && x > -INFINITY) lowest = fminf(lowest, x);
        return x;
    };
    const int n4 = vec ? n / 4 : 0;
#pragma unroll 4
    for (int i = tid; i < n4; i += THREADS) {
        const float4 v = __ldcs(reinterpret_cast<const float4*>(src) + i);
        reinterpret_cast<float4*>(part_of_row)[i] = make_float4(take(v.x), take(v.y), take(v.z), take(v.w));
    }
#pragma unroll 4
    for (int i = 4 * n4 + tid; i < n; i += THREADS) part_of_row[i] = take(src[i]);
    for (int i = n + tid; i < r.padded; i += THREADS) part_of_row[i] = -INFINITY;
    auto reduce = [&](int width) {
        for (int o = width / 2; o > 0; o >>= 1) {
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            lowest = fminf(lowest, __shfl_xor_sync(0xffffffffu, lowest, o));
        }
    };
    reduce(32);
    if (lane == 0) { sh.warp_max[warp] = m; sh.warp_min[warp] = lowest; }
    if (tid < 16) sh.power[tid] = exp2((double)tid / 16);
    if (cuts) clear(sh);
    __syncthreads();
    m = sh.warp_max[lane % WARPS];
    lowest = sh.warp_min[lane % WARPS];
    reduce(WARPS);
    if (tid == 0) { sh.max = m; sh.min = lowest; sh.at = 0x7fffffff; }
    cl.sync();
    m = cl.map_shared_rank(&sh, lane % ranks)->max;
    lowest = cl.map_shared_rank(&sh, lane % ranks)->min;
    reduce(MAX_CLUSTER);
    if (m == -INFINITY || greedy) {
        if (m > -INFINITY) {   // the first place of the largest
            int at = 0x7fffffff;
            for (int i = tid; i < r.padded; i += THREADS)
                if (r.x[i] == m) { at = r.first + i; break; }
            at = __reduce_min_sync(0xffffffffu, at);
            if (lane == 0 && at < 0x7fffffff) atomicMin(&cl.map_shared_rank(&sh, 0)->at, at);
        }
        cl.sync();
        if (rank == 0 && tid == 0) token[row] = m == -INFINITY ? -1 : sh.at;
        return;
    }
    if (m == INFINITY) {   // the infinite ones share the mass: as logits of 0 among -infinity
        for (int i = tid; i < r.padded; i += THREADS) part_of_row[i] = r.x[i] == INFINITY ? 0.f : -INFINITY;
        m = lowest = 0.f;
        __syncthreads();
    }
    r.max = m;
    r.min = lowest;
    r.top = m;
    r.fresh = true;
    r.rate = rate;
    r.power = sh.power;
    // What weighs less than 2^-1000 is not kept. Rounded up, so that far from zero no logit next to the largest leaves the
    // exponent's range.
    r.tau = fmaxf(__double2float_ru(r.top - (1000.0 * 0.69314718055994530942) * (double)t), -3.4028235e38f);
    r.last = ALL;
    if (mp > 0.f && t < INFINITY) {
        r.tau = fmaxf(r.tau, fminf(m, __double2float_ru((double)m + (double)t * log((double)fminf(mp, 1.f))) + 0.f));
    }
    r.min = fmaxf(r.min, r.tau);
    if (k > 0 && k < vocab && cut<false>(cl, sh, r, k, p, u[row], token + row)) return;
    if (p < 1.f) cut<true>(cl, sh, r, 0, fmaxf(p, 1e-30f), 0.0, nullptr);   // rank 0 always stays

    // the draw: sums of blocks of 128 logits, the CTA in which u falls, the block, the logit
    auto lane_weights = [&](int block, double (&w)[4]) {   // this lane's 4 of a block
        const int i = block * BLOCK + 4 * lane;
        const float4 v = *reinterpret_cast<const float4*>(r.x + i);
        const bool k0 = kept(r, v.x, i), k1 = kept(r, v.y, i + 1), k2 = kept(r, v.z, i + 2), k3 = kept(r, v.w, i + 3);
        w[0] = w[1] = w[2] = w[3] = 0.0;
        if (!__any_sync(0xffffffffu, k0 || k1 || k2 || k3)) return;
        w[0] = k0 ? weight(r, fmaxf(v.x, r.tau)) : 0.0;   // without branches
        w[1] = k1 ? weight(r, fmaxf(v.y, r.tau)) : 0.0;
        w[2] = k2 ? weight(r, fmaxf(v.z, r.tau)) : 0.0;
        w[3] = k3 ? weight(r, fmaxf(v.w, r.tau)) : 0.0;
    };
    const int blocks = r.padded / BLOCK;
    for (int b = warp; b < blocks; b += WARPS) {
        double w[4];
        lane_weights(b, w);
        double v = (w[0] + w[1]) + (w[2] + w[3]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == 0) sh.block_mass[b] = v;
    }
    __syncthreads();
    double mine = 0.0;   // of this lane's blocks: blocks / 32 neighbours each
    bool mine_any = false;
    const int per = (blocks + 31) / 32;
    if (warp == 0) {
        for (int k = 0; k < per; k++)
            if (lane * per + k < blocks) mine += sh.block_mass[lane * per + k];
        mine_any = mine > 0.0;
        mine = scan(mine);
        const double here = __shfl_sync(0xffffffffu, mine, 31);
        if (lane < ranks) cl.map_shared_rank(&sh, lane)->mass_of[rank] = here;
    }
    cl.sync();
    double of_cta = lane < ranks ? sh.mass_of[lane] : 0.0;
    const bool cta_any = of_cta > 0.0;
    of_cta = scan(of_cta);
    const double total = __shfl_sync(0xffffffffu, of_cta, 31), target = (double)u[row] * total;
    double ahead = 0.0;
    const int owner = first_over(of_cta, cta_any, ahead, target);
    if (owner >= ranks) {   // u >= 1, or the sums' last bits: the last kept token
        int last = -1;
        for_kept(r, [&](float, int i) { last = max(last, r.first + i); });
        last = __reduce_max_sync(0xffffffffu, last);
        __syncthreads();
        if (tid == 0) sh.last = -1;
        cl.sync();
        if (lane == 0) atomicMax(&cl.map_shared_rank(&sh, 0)->last, last);
        cl.sync();
        if (rank == 0 && tid == 0) token[row] = sh.last;
        return;
    }
    if (owner == rank && warp == 0) {
        const int at = draw_in_part<1>(mine, mine_any, per, blocks, sh.block_mass, ahead, target, lane_weights);
        if (lane == 0) token[row] = r.first + at;
    }
}

// Without filters: one pass. Each warp takes blocks of 256 logits (128: 25.6 us for 64 x 131072, 256: 20.6, 512: the same, and
// slower rows of 32000), whose weights are summed relative to the block's own maximum; the sums are brought to the
// row's maximum when that is known, and the drawn block's logits are read again.
// Nothing of a row stays in shared memory but a maximum and a sum per block, so twice as many CTAs run as above.
constexpr int OPEN_THREADS = 256, OPEN_WARPS = OPEN_THREADS / 32, OPEN_SUBS = 2, OPEN_BLOCK = OPEN_SUBS * BLOCK;
constexpr int OPEN_MOST = 32768;   // logits of a CTA

__global__ void __launch_bounds__(OPEN_THREADS, 4) k_sample_open(int32_t* __restrict__ token, const float* __restrict__ logits,
                                                                 size_t ld, int vocab, int part, int vec, const float* temperature,
                                                                 const float* u) {
    __shared__ double block_mass[OPEN_MOST / OPEN_BLOCK], power[16], mass_here;
    __shared__ float block_max[OPEN_MOST / OPEN_BLOCK], warp_max[OPEN_WARPS], max_here;
    __shared__ int first_here;
    cg::cluster_group cl = cg::this_cluster();
    const int ranks = cl.num_blocks(), rank = cl.block_rank(), row = blockIdx.x / ranks, first = rank * part;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = max(0, min(part, vocab - first)), blocks = (n + OPEN_BLOCK - 1) / OPEN_BLOCK;
    const float* src = logits + (size_t)row * ld + first;
    const float t = temperature ? temperature[row] : 1.f;
    const double rate = 16 * 1.4426950408889634074 / (double)t;
    const bool greedy = !(t > 0.f);
    if (tid < 16) power[tid] = exp2((double)tid / 16);
    if (tid == 0) first_here = ALL;
    __syncthreads();
    auto fetch = [&](int block, float (&x)[4], bool in_order) {   // a block's logits; in order: 4 neighbours a lane
        const int i = block * BLOCK + 4 * lane;
        if (vec && i + 3 < n) {
            const float4 v = *reinterpret_cast<const float4*>(src + i);
            x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int k = vec || in_order ? i + j : block * BLOCK + 32 * j + lane;
                x[j] = k < n ? src[k] : -INFINITY;
            }
        }
    };
    const float reach = 693.14718f * t;   // to 2^-1000, rounded up where it is subtracted
    constexpr float LOWEST = -3.4028235e38f;
    // In two steps, as logits may be further apart than FP32 reaches; from where one of them is infinite they are not.
    const float half_reach = 346.57359f * t;
    auto nothing_below = [&](float top) { return fmaxf(__fsub_ru(__fsub_ru(top, half_reach), half_reach), LOWEST); };
    // Weights relative to top, the largest or infinite: then the infinite ones share the mass. What lies below `nothing`
    // weighs as much as that, or with to_zero 0.
    auto lane_weights = [&](const float (&x)[4], float top, float nothing, bool to_zero, double (&w)[4]) {
        if (top == INFINITY) {
#pragma unroll
            for (int j = 0; j < 4; j++) w[j] = x[j] == INFINITY ? 1.0 : 0.0;
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                w[j] = weight_of(fmaxf(x[j], nothing), top, rate, power);
                if (to_zero && !(x[j] >= nothing)) w[j] = 0.0;
            }
        }
    };
    float m = -INFINITY;
    for (int b = warp; b < blocks; b += OPEN_WARPS) {
        float x[OPEN_SUBS][4], top = -INFINITY;
#pragma unroll
        for (int s = 0; s < OPEN_SUBS; s++) fetch(b * OPEN_SUBS + s, x[s], false);
#pragma unroll
        for (int s = 0; s < OPEN_SUBS; s++) top = fmaxf(top, fmaxf(fmaxf(x[s][0], x[s][1]), fmaxf(x[s][2], x[s][3])));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        double v = 0.0;
        if (!greedy && top > -INFINITY) {
            const float nothing = nothing_below(top);
            auto add = [&](bool to_zero) {
#pragma unroll
                for (int s = 0; s < OPEN_SUBS; s++) {
                    double w[4];
                    lane_weights(x[s], top, nothing, to_zero, w);
                    v += (w[0] + w[1]) + (w[2] + w[3]);
                }
            };
            if (reach < INFINITY && top - nothing >= 0.9f * reach) add(false);   // 2^-900 is lost in a sum with the largest's 1
            else add(true);   // hot, or so far from zero that `nothing` was rounded far up
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        }
        if (lane == 0) { block_max[b] = top; block_mass[b] = v; }
        m = fmaxf(m, top);
    }
    if (lane == 0) warp_max[warp] = m;
    __syncthreads();
    m = warp_max[lane % OPEN_WARPS];
#pragma unroll
    for (int o = OPEN_WARPS / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (tid == 0) max_here = m;
    cl.sync();
    m = *cl.map_shared_rank(&max_here, lane % ranks);
#pragma unroll
    for (int o = MAX_CLUSTER / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    // of this CTA's blocks: per neighbours a lane of the first warp
    double mine = 0.0;
    bool mine_any = false;
    const int per = (blocks + 31) / 32;
    if (warp == 0) {
        int at = ALL;   // the first block that holds the row's maximum
        const float nothing = nothing_below(m);
        for (int k = 0; k < per; k++) {
            const int b = lane * per + k;
            if (b >= blocks) break;
            const float top = block_max[b];
            if (top == m) at = min(at, b);
            double v = 0.0;
            if (!greedy && m == INFINITY) v = top == m ? block_mass[b] : 0.0;
            else if (!greedy && top >= nothing) v = block_mass[b] * weight_of(top, m, rate, power);
            block_mass[b] = v;
            mine += v;
        }
        mine_any = mine > 0.0;
        mine = scan(mine);
        if (lane == 31) mass_here = mine;
        if (greedy && m > -INFINITY) {
            at = __reduce_min_sync(0xffffffffu, at);
            if (at < ALL) {
                int where = ALL;
                for (int s = 0; s < OPEN_SUBS; s++) {
                    float y[4];
                    fetch(at * OPEN_SUBS + s, y, true);
                    const int j = y[0] == m ? 0 : y[1] == m ? 1 : y[2] == m ? 2 : y[3] == m ? 3 : ALL;
                    if (j < ALL) where = min(where, BLOCK * s + 4 * lane + j);
                }
                where = __reduce_min_sync(0xffffffffu, where);
                if (lane == 0) first_here = first + at * OPEN_BLOCK + where;
            }
        }
    }
    cl.sync();
    if (warp == 0) {
        if (m == -INFINITY || greedy) {
            const int at = __reduce_min_sync(0xffffffffu, *cl.map_shared_rank(&first_here, lane % ranks));
            if (rank == 0 && lane == 0) token[row] = m == -INFINITY ? -1 : at;
        } else {
            double of_cta = lane < ranks ? *cl.map_shared_rank(&mass_here, lane % ranks) : 0.0;
            const bool cta_any = of_cta > 0.0;
            of_cta = scan(of_cta);
            const double total = __shfl_sync(0xffffffffu, of_cta, 31), target = (double)u[row] * total;
            double ahead = 0.0;
            // u >= 1 draws from the last that has any, and there the last
            const int owner = or_last(first_over(of_cta, cta_any, ahead, target), cta_any);
            if (owner == rank) {
                const int at = draw_in_part<OPEN_SUBS>(mine, mine_any, per, blocks, block_mass, ahead, target, [&](int block, double (&w)[4]) {
                    float y[4];
                    fetch(block, y, true);
                    lane_weights(y, m, nothing_below(m), true, w);
                });
                if (lane == 0) token[row] = first + at;
            }
        }
    }
    cl.sync();   // nobody leaves while its shared memory is read
}

lancius_error bad(lancius_error e) { lancius_set_error(e); return e; }

// CTAs per row. With filters parts of at most 16384 logits, so that two CTAs fit on an SM (three with 12544), without them of OPEN_MOST; for few
// rows up to 8 with at least 2048, as long as all CTAs run at once.
int cluster_of(size_t rows, size_t vocab, bool open) {
    const size_t resident = (open ? 4 : 2) * LCU_SMS, most = open ? OPEN_MOST : 16384;
    int c = 1;
    while (c < MAX_CLUSTER && vocab > most * c) c *= 2;
    while (c < MAX_CLUSTER && rows * c * 2 <= resident && vocab >= 4096 * (size_t)c) c *= 2;
    return c;
}

}  // namespace

extern "C" lancius_error lcu_sample(int32_t* token, const float* logits, size_t ld, size_t rows, size_t vocab,
                                    const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                                    const float* u, void* stream) {
    if (!rows) return LANCIUS_ERROR_OK;
    if (!token || !logits || !u) return bad(LANCIUS_ERROR_NULL_PTR);
    if (!vocab || vocab > MAX_VOCAB || ld < vocab || rows > (size_t)INT32_MAX / MAX_CLUSTER) return bad(LANCIUS_ERROR_SHAPE_MISMATCH);
    const bool open = !top_k && !top_p && !min_p;
    const int c = cluster_of(rows, vocab, open);
    const size_t part = ((vocab + c - 1) / c + 3) / 4 * 4;
    const int vec = (uintptr_t)logits % 16 == 0 && ld % 4 == 0;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = c;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(rows * c));
    cfg.blockDim = dim3(open ? OPEN_THREADS : THREADS);
    cfg.stream = lcu_as_stream(stream);
    cfg.attrs = at;
    cfg.numAttrs = 1;
    cudaError_t ce;
    if (open) {
        ce = cudaLaunchKernelEx(&cfg, k_sample_open, token, logits, ld, (int)vocab, (int)part, vec, temperature, u);
    } else {
        cfg.dynamicSmemBytes = (part + BLOCK - 1) / BLOCK * BLOCK * sizeof(float);   // whole blocks are read
        auto launch = [&](auto kernel, std::atomic<unsigned long long>& allowed, int most) {
            const cudaError_t e = lcu_allow_smem(allowed, kernel, most);
            return e != cudaSuccess ? e : cudaLaunchKernelEx(&cfg, kernel, token, logits, ld, (int)vocab, (int)part, vec, temperature,
                                                             top_k, top_p, min_p, u);
        };
        static std::atomic<unsigned long long> allowed2{0}, allowed3{0};
        constexpr size_t THIRD = (228 * 1024) / 3 - 1024 - sizeof(Shared);   // of an SM's shared memory
        ce = rows * c > 2 * LCU_SMS && cfg.dynamicSmemBytes <= THIRD
                 ? launch(k_sample<3>, allowed3, (int)THIRD)
                 : launch(k_sample<2>, allowed2, (int)(MAX_VOCAB / MAX_CLUSTER * sizeof(float)));
    }
    if (ce != cudaSuccess) {
        cudaGetLastError();
        return lcu_check_cuda(ce);
    }
    lcu_note_launch();
    return lcu_launch_status();
}
