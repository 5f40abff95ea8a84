// Drawing a token per row of logits (lcu_sample).
//
// w_i = exp((x_i - max) / t). Every filter keeps a prefix of the rank order (logit falling, index rising), so a row's kept
// set is one cut: a logit tau and a last index among the logits equal to tau. No sort is needed: a histogram of the
// logits finds the bin in which the count (top-k) or the mass (top-p) reaches its target, and the few logits of that
// bin are ranked against each other; where a bin holds more than LIST of them (many equal logits), a radix search
// over order-preserving 32-bit keys narrows it down to one key first. The draw adds weights in index order.
//
// Masses of bins are 64-bit fixed point, so the order of the atomics does not matter: 2^44 for the largest weight, and
// 2^18 tokens fit 62 bits. The draw's sums are FP64 in a fixed order. Weights are FP64: with FP32 ones a drawn token
// would differ from the exact one in about one row of a thousand.
//
// Bound: HBM for large batches (each logit read once), the length of the chain of passes for small ones. A row is
// spread over a cluster of 1 to 8 CTAs that hold it in shared memory through all passes and exchange histograms and
// sums through each other's shared memory.
#include "lcu_internal.h"
#include <cooperative_groups.h>
#include <math.h>

namespace cg = cooperative_groups;

namespace {

constexpr int THREADS = 512, WARPS = THREADS / 32, BINS = 2048, LIST = THREADS, MAX_CLUSTER = 8;
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

struct Shared {
    u64 mass[BINS];
    uint32_t count[BINS];
    float warp_max[WARPS], warp_min[WARPS];
    u64 list[LIST], list_mass[LIST];   // key << 32 | ~index, so that larger means an earlier rank
    double power[16];
    u64 warp_sum[WARPS];
    double block_mass[MAX_BLOCKS], mass_here;
    float max, min;
    int at, found, bin, last;
    uint32_t listed, members, tau;
    u64 before, in_bin, total, ties;
};

struct Row {
    const float* x;     // this CTA's part, in shared memory, cleaned
    int n, first;       // its length and the index of its first token
    float max, min;     // of the row, min over the finite ones
    double top, rate;   // max, log2(e) / t
    float nothing;      // weights are 0 below this logit
    const double* power;   // 2^(j/16), in shared memory
    uint32_t tau;       // kept: key > tau, or key == tau and index <= last
    int last;
};

__device__ __forceinline__ bool kept(const Row& r, uint32_t key, int i) { return key > r.tau || (key == r.tau && r.first + i <= r.last); }
// exp((x - max) / t) as 2^z, z = n / 16 + f, |f| <= 1/32: a table of 2^(j/16) times the Taylor series of 2^f to f^6
// (table-driven exponential, Tang 1989); the series' remainder is 5e-16. 13 FP64 instructions, where the library's
// exp and a division took 124 of all kinds. Below 2^-1000 the
// weight is 0.
__device__ __forceinline__ double weight(const Row& r, float x) {
    if (!(x >= r.nothing)) return 0.0;
    const double z = ((double)x - r.top) * r.rate;
    constexpr double MAGIC = 6755399441055744.0;   // 1.5 * 2^52: the sum's low bits are the rounded integer
    const double k = fma(z, 16.0, MAGIC);
    const int n = __double2loint(k);
    const double f = fma(k - MAGIC, -0.0625, z);
    double p = 1.5403530393381609954e-4;           // ln2^i / i!
    p = fma(p, f, 1.3333558146428443423e-3);
    p = fma(p, f, 9.6181291076284771620e-3);
    p = fma(p, f, 5.5504108664821579953e-2);
    p = fma(p, f, 2.4022650695910071233e-1);
    p = fma(p, f, 6.9314718055994530942e-1);
    p = fma(p, f, 1.0) * r.power[n & 15];
    return __hiloint2double(__double2hiint(p) + ((n >> 4) << 20), __double2loint(p));
}
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
    u64 add = 0;
    for (int w = 0; w < warp; w++) add += sh.warp_sum[w];
    return v + add;
}

// One histogram over the kept logits, bin_of(x, key) < BINS rising with the rank (or -1: not counted), and the bin in
// which the running sum reaches the target: sh.bin, sh.before (sum before the bin, starting at `before`),
// sh.in_bin, sh.members, sh.found. The target is made by target_of(total) from the sum of all bins.
template <bool MASS, typename Bin, typename Target>
__device__ void find_bin(cg::cluster_group& cl, Shared& sh, const Row& r, u64 before, Bin bin_of, Target target_of) {
    const int tid = threadIdx.x, ranks = cl.num_blocks(), slice = BINS / ranks;
    cl.sync();   // nobody reads the last histogram any more
    for (int i = tid; i < BINS; i += THREADS) { sh.mass[i] = 0; sh.count[i] = 0; }
    if (tid == 0) { sh.found = 0; sh.listed = 0; }
    __syncthreads();
    for (int i = tid; i < r.n; i += THREADS) {
        const float x = r.x[i];
        const uint32_t key = key_of(x);
        if (!kept(r, key, i)) continue;
        const int bin = bin_of(x, key);
        if (bin < 0) continue;
        atomicAdd(&sh.count[bin], 1u);
        if (MASS) atomicAdd(&sh.mass[bin], fixed_weight(r, x));
    }
    cl.sync();
    if (ranks > 1) {   // each CTA adds up its slice of the bins, in place: nobody else reads that slice of its own
        const int b0 = cl.block_rank() * slice;
        for (int i = b0 + tid; i < b0 + slice; i += THREADS) {
            uint32_t c = 0;
            u64 m = 0;
#pragma unroll
            for (int k = 0; k < MAX_CLUSTER; k++)   // unrolled: the remote reads are in flight together
                if (k < ranks) {
                    const Shared* o = cl.map_shared_rank(&sh, k);
                    c += o->count[i];
                    if (MASS) m += o->mass[i];
                }
            sh.count[i] = c;
            sh.mass[i] = m;
        }
        cl.sync();
    }
    // every CTA scans all bins
    constexpr int PER = BINS / THREADS;
    u64 v[PER], sum = 0;
    uint32_t c[PER];
    const Shared* owner = cl.map_shared_rank(&sh, PER * tid / slice);
#pragma unroll
    for (int k = 0; k < PER; k++) {
        c[k] = owner->count[PER * tid + k];
        v[k] = MASS ? owner->mass[PER * tid + k] : c[k];
        sum += v[k];
    }
    const u64 upto = block_scan(sh, sum);
    if (tid == THREADS - 1) sh.total = upto;
    __syncthreads();
    const double target = target_of(sh.total);
    u64 at = before + upto - sum;
#pragma unroll
    for (int k = 0; k < PER; k++) {
        if ((double)at < target && (double)(at + v[k]) >= target) {   // one bin of one thread
            sh.bin = PER * tid + k; sh.before = at; sh.in_bin = v[k]; sh.members = c[k]; sh.found = 1;
        }
        at += v[k];
    }
    __syncthreads();
}

// The kept logits with in(x, key) are at most LIST: ranks them and moves the cut to the one at which the sum reaches the
// target.
template <bool MASS, typename In>
__device__ void finish_list(cg::cluster_group& cl, Shared& sh, Row& r, double target, In in) {
    const int tid = threadIdx.x;
    const u64 before = sh.before;
    Shared* lead = cl.map_shared_rank(&sh, 0);   // its counter was zeroed before the histogram
    for (int i = tid; i < r.n; i += THREADS) {
        const float x = r.x[i];
        const uint32_t key = key_of(x);
        if (!kept(r, key, i) || !in(x, key)) continue;
        const uint32_t to = atomicAdd(&lead->listed, 1u);
        if (to >= LIST) continue;
        lead->list[to] = (u64)key << 32 | (uint32_t)~(uint32_t)(r.first + i);
        if (MASS) lead->list_mass[to] = fixed_weight(r, x);
    }
    cl.sync();
    if (cl.block_rank() == 0) {
        const int n = min(sh.listed, (uint32_t)LIST);
        if (tid < n) {
            const u64 me = sh.list[tid];
            u64 ahead = before;
            for (int j = 0; j < n; j++)
                if (sh.list[j] > me) ahead += MASS ? sh.list_mass[j] : 1;
            const u64 w = MASS ? sh.list_mass[tid] : 1;
            if ((double)ahead < target && (double)(ahead + w) >= target) { sh.tau = (uint32_t)(me >> 32); sh.last = (int)~(uint32_t)me; }
        }
    }
    cl.sync();
    r.tau = lead->tau;
    r.last = lead->last;
}

// Of the kept logits equal to `key`, the one that is the keep-th by index becomes the last.
__device__ void finish_ties(cg::cluster_group& cl, Shared& sh, Row& r, uint32_t key, u64 keep) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int seg = ((r.n + WARPS - 1) / WARPS + 31) / 32 * 32, s0 = warp * seg, s1 = min(r.n, s0 + seg);
    auto hits = [&](int i) {
        const uint32_t k = i < s1 ? key_of(r.x[i]) : 0;
        return __ballot_sync(0xffffffffu, i < s1 && k == key && kept(r, k, i));
    };
    u64 n = 0;
    for (int i = s0 + lane; i - lane < s1; i += 32) n += __popc(hits(i));
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
        for (int i = s0 + lane; i - lane < s1; i += 32) {
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
    r.tau = key;
    r.last = lead->last;
}

// Moves the row's cut to the rank at which the running count (MASS = false: k) or mass (p times the mass of what is
// kept so far) is reached.
template <bool MASS>
__device__ void cut(cg::cluster_group& cl, Shared& sh, Row& r, int k, double p) {
    double target = k;
    auto first_target = [&](u64 total) { return MASS ? fmax(p * (double)total, 0.5) : (double)k; };
    // bins of equal width in the logit, down to weights of e^-100
    const float range = fminf(r.max - r.min, 144.f / (float)r.rate);
    if (range > 0.f && range < INFINITY) {
        const float per = (BINS - 1) / range;
        auto bin_of = [&](float x, uint32_t) { return min(BINS - 1, __float2int_rz((r.max - x) * per)); };
        find_bin<MASS>(cl, sh, r, 0, bin_of, first_target);
        if (!sh.found) return;   // fewer than k, or all of the mass is wanted
        if (sh.members <= LIST) {
            target = first_target(sh.total);
            const int bin = sh.bin;
            finish_list<MASS>(cl, sh, r, target, [&](float x, uint32_t key) { return bin_of(x, key) == bin; });
            return;
        }
    }
    uint32_t lo = r.tau, hi = key_of(r.max);
    u64 before = 0;
    for (bool first = true;; first = false) {   // at most 3 rounds: 32 bits, 21, 10
        const int bits = max(0, 32 - __clz(hi - lo) - 11);
        auto bin_of = [&](float, uint32_t key) { return key < lo || key > hi ? -1 : (int)((hi - key) >> bits); };
        find_bin<MASS>(cl, sh, r, before, bin_of, [&](u64 total) { return first ? first_target(total) : target; });
        if (!sh.found) return;
        if (first) target = first_target(sh.total);
        before = sh.before;
        hi -= (uint32_t)sh.bin << bits;
        const uint32_t low = hi - ((1u << bits) - 1);
        if (low > lo && low <= hi) lo = low;
        if (sh.members <= LIST) {
            finish_list<MASS>(cl, sh, r, target, [&](float, uint32_t key) { return key >= lo && key <= hi; });
            return;
        }
        if (bits) continue;
        const double ties = (double)sh.members, each = (double)sh.in_bin / ties;
        const double need = MASS ? fmin(fmax(ceil((target - (double)before) / each), 1.0), ties) : target - (double)before;
        finish_ties(cl, sh, r, hi, (u64)need);
        return;
    }
}

__global__ void __launch_bounds__(THREADS, 2) k_sample(int32_t* __restrict__ token, const float* __restrict__ logits, size_t ld, int vocab,
                                                    int part, int vec, const float* temperature, const int32_t* top_k,
                                                    const float* top_p, const float* min_p, const float* u) {
    extern __shared__ __align__(16) float part_of_row[];
    __shared__ Shared sh;
    cg::cluster_group cl = cg::this_cluster();
    const int ranks = cl.num_blocks(), rank = cl.block_rank(), row = blockIdx.x / ranks;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Row r;
    r.x = part_of_row;
    r.first = rank * part;
    r.n = max(0, min(part, vocab - r.first));
    const float* src = logits + (size_t)row * ld + r.first;
    const float t = temperature ? temperature[row] : 1.f, mp = min_p ? min_p[row] : 0.f, p = top_p ? top_p[row] : 1.f;
    const int k = top_k ? top_k[row] : 0;
    const bool greedy = !(t > 0.f), cuts = !greedy && ((k > 0 && k < vocab) || p < 1.f);
    float m = -INFINITY, lowest = INFINITY;   // lowest of the finite ones, where a cut will want it
    auto take = [&](float x) {
        x = clean(x);
        m = fmaxf(m, x);
        if (cuts && x > -INFINITY) lowest = fminf(lowest, x);
        return x;
    };
    const int n4 = vec ? r.n / 4 : 0;
#pragma unroll 4
    for (int i = tid; i < n4; i += THREADS) {
        const float4 v = __ldcs(reinterpret_cast<const float4*>(src) + i);
        reinterpret_cast<float4*>(part_of_row)[i] = make_float4(take(v.x), take(v.y), take(v.z), take(v.w));
    }
#pragma unroll 4
    for (int i = 4 * n4 + tid; i < r.n; i += THREADS) part_of_row[i] = take(src[i]);
    auto reduce = [&](int width) {
        for (int o = width / 2; o > 0; o >>= 1) {
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            lowest = fminf(lowest, __shfl_xor_sync(0xffffffffu, lowest, o));
        }
    };
    reduce(32);
    if (lane == 0) { sh.warp_max[warp] = m; sh.warp_min[warp] = lowest; }
    if (tid < 16) sh.power[tid] = exp2((double)tid / 16);
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
            for (int i = tid; i < r.n; i += THREADS)
                if (r.x[i] == m) { at = r.first + i; break; }
            at = __reduce_min_sync(0xffffffffu, at);
            if (lane == 0 && at < 0x7fffffff) atomicMin(&cl.map_shared_rank(&sh, 0)->at, at);
        }
        cl.sync();
        if (rank == 0 && tid == 0) token[row] = m == -INFINITY ? -1 : sh.at;
        return;
    }
    if (m == INFINITY) {   // the infinite ones share the mass: as logits of 0 among -infinity
        for (int i = tid; i < r.n; i += THREADS) part_of_row[i] = r.x[i] == INFINITY ? 0.f : -INFINITY;
        m = lowest = 0.f;
        __syncthreads();
    }
    r.max = m;
    r.min = lowest;
    r.top = m;
    r.rate = 1.4426950408889634074 / (double)t;
    r.power = sh.power;
    r.nothing = fmaxf((float)(r.top - 1000.0 / r.rate), -3.4028235e38f);
    r.tau = key_of(-INFINITY) + 1;
    r.last = 0x7fffffff;
    if (mp > 0.f) {
        const float least = fminf(m, __double2float_ru((double)m + (double)t * log((double)fminf(mp, 1.f))) + 0.f);
        r.tau = max(r.tau, key_of(least));
        r.min = fmaxf(r.min, least);
    }
    if (k > 0 && k < vocab) cut<false>(cl, sh, r, k, 0.0);
    if (p < 1.f) cut<true>(cl, sh, r, 0, p);
    const bool all = r.tau == key_of(-INFINITY) + 1 && r.last == 0x7fffffff;

    // the draw: sums of blocks of 128 logits, the CTA in which u falls, the block, the logit
    auto kept_weight = [&](int i, float x) { return all || kept(r, key_of(x), i) ? weight(r, x) : 0.0; };
    auto lane_weights = [&](int block, double (&w)[4]) {   // this lane's 4 of a block; past the end: 0
        const int i = block * BLOCK + 4 * lane;
        const float4 v = *reinterpret_cast<const float4*>(r.x + i);
        w[0] = i < r.n ? kept_weight(i, v.x) : 0.0;
        w[1] = i + 1 < r.n ? kept_weight(i + 1, v.y) : 0.0;
        w[2] = i + 2 < r.n ? kept_weight(i + 2, v.z) : 0.0;
        w[3] = i + 3 < r.n ? kept_weight(i + 3, v.w) : 0.0;
    };
    auto scan = [&](double v) {   // inclusive, over the warp
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double x = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += x;
        }
        return v;
    };
    // v: inclusive sums by lane of what each lane has, if any; the first lane that has some and whose sum, behind `ahead`,
    // passes the target (32: none); ahead moves to its start. A sum's last bits depend on its order, so a lane without
    // weight may seem to pass.
    auto first_over = [&](double v, bool any, double& ahead, double target) {
        const unsigned over = __ballot_sync(0xffffffffu, any && ahead + v > target);
        const int at = over ? __ffs(over) - 1 : 32;
        const double x = __shfl_sync(0xffffffffu, v, max(min(at, 31) - 1, 0));
        if (at > 0 && at < 32) ahead += x;
        return at;
    };
    const int blocks = (r.n + BLOCK - 1) / BLOCK;
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
        if (lane == 31) sh.mass_here = mine;
    }
    cl.sync();
    double of_cta = lane < ranks ? cl.map_shared_rank(&sh, lane % ranks)->mass_here : 0.0;
    const bool cta_any = of_cta > 0.0;
    of_cta = scan(of_cta);
    const double total = __shfl_sync(0xffffffffu, of_cta, 31), target = (double)u[row] * total;
    double ahead = 0.0;
    const int owner = first_over(of_cta, cta_any, ahead, target);
    if (owner >= ranks) {   // u >= 1, or the sums' last bits: the last kept token that weighs anything
        int last = -1;
        for (int i = tid; i < r.n; i += THREADS)
            if (kept(r, key_of(r.x[i]), i) && weight(r, r.x[i]) > 0.0) last = r.first + i;
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
        // where no lane passes, again for the last bits, the last that has some is taken
        auto or_last = [&](int at, bool any) {
            const unsigned some = __ballot_sync(0xffffffffu, any);
            return at < 32 ? at : 31 - __clz(some);
        };
        int at = or_last(first_over(mine, mine_any, ahead, target), mine_any);
        const int b0 = at * per, n = min(per, blocks - b0);   // per <= 8 blocks
        const double of_block = lane < n ? sh.block_mass[b0 + lane] : 0.0;
        const int block = b0 + or_last(first_over(scan(of_block), of_block > 0.0, ahead, target), of_block > 0.0);
        double w[4];
        lane_weights(block, w);
        const double four = (w[0] + w[1]) + (w[2] + w[3]);
        at = or_last(first_over(scan(four), four > 0.0, ahead, target), four > 0.0);
        if (lane == at) {
            int drawn = -1;
            for (int j = 0; j < 4; j++)
                if (w[j] > 0.0) {
                    drawn = j;
                    ahead += w[j];
                    if (ahead > target) break;
                }
            token[row] = r.first + block * BLOCK + 4 * lane + drawn;
        }
    }
    cl.sync();   // nobody leaves while its shared memory is read
}

lancius_error bad(lancius_error e) { lancius_set_error(e); return e; }

// CTAs per row: parts of at most 16384 logits, so that two CTAs fit on an SM, and for few rows up to 8 with at least 2048
int cluster_of(size_t rows, size_t vocab) {
    int c = 1;
    while (c < MAX_CLUSTER && vocab > 16384 * (size_t)c) c *= 2;
    while (c < MAX_CLUSTER && rows * c * 2 <= 2 * LCU_SMS && vocab >= 4096 * (size_t)c) c *= 2;
    return c;
}

}  // namespace

extern "C" lancius_error lcu_sample(int32_t* token, const float* logits, size_t ld, size_t rows, size_t vocab,
                                    const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                                    const float* u, void* stream) {
    if (!rows) return LANCIUS_ERROR_OK;
    if (!token || !logits || !u) return bad(LANCIUS_ERROR_NULL_PTR);
    if (!vocab || vocab > MAX_VOCAB || ld < vocab || rows > (size_t)INT32_MAX / MAX_CLUSTER) return bad(LANCIUS_ERROR_SHAPE_MISMATCH);
    const int c = cluster_of(rows, vocab);
    const size_t part = ((vocab + c - 1) / c + 3) / 4 * 4, space = (part + BLOCK - 1) / BLOCK * BLOCK;   // whole blocks are read
    cudaError_t ce = cudaFuncSetAttribute(k_sample, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(MAX_VOCAB / MAX_CLUSTER * sizeof(float)));
    if (ce != cudaSuccess) return lcu_check_cuda(ce);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = c;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(rows * c));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = space * sizeof(float);
    cfg.stream = lcu_as_stream(stream);
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const int vec = (uintptr_t)logits % 16 == 0 && ld % 4 == 0;
    ce = cudaLaunchKernelEx(&cfg, k_sample, token, logits, ld, (int)vocab, (int)part, vec, temperature, top_k, top_p, min_p, u);
    if (ce != cudaSuccess) {
        cudaGetLastError();
        return lcu_check_cuda(ce);
    }
    lcu_note_launch();
    return lcu_launch_status();
}
