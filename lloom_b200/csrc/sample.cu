// The next token of every row of logits: temperature, top-k, top-p (nucleus) and min-p filters and a draw from a given uniform number.
//
//   w_i = exp((l_i - max) / T); tokens in the order (logit falling, index rising); kept: the shortest of three prefixes of it -- the first
//   K, the first whose weights reach P times those of the first K, those with w_i >= min_p; drawn: of the kept ones, by rising index, the
//   first whose running sum of weights exceeds u times their sum.
//
// A cluster of CTAs has a row: it is read once, stays in shared memory, and everything after works there.  A filter's border is found by
// a histogram over 2048 buckets of (max - l) / T, 1/64 wide, then within the bucket that holds it: by further histograms over the bits of the
// logits while it has more than 256 tokens, else by ranking them against one another; equal logits by index.  No sort of the row.
//
// Weights are summed as integers, in units of 2^-43 of the largest weight: the sums are exact, so that they depend neither on
// the split of a row nor on the order of atomics, and borders fall where 64-bit arithmetic puts them.  (In 32 bits a running sum over
// 100,000 tokens is off by more than a token's share of it.)  Tokens below 2^-44 of the largest weight count as zero.
// exp: table of 2^(-j/32) and a polynomial (table-driven, after Tang 1989) in 64-bit arithmetic, relative error below 1e-14.
//
// Bound by latency for a few rows (a launch, one read of DRAM, a handful of cluster barriers), by the 64-bit pipe and the read for many.
#include <mutex>

#include "abi.h"
#include "common.cuh"
#include "forward.h"

namespace lloom {

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBuckets = 2048, kPerThread = kBuckets / kThreads;
constexpr int kList = 256;       // tokens that are ranked against one another
constexpr int kMaxCluster = 8;
constexpr double kUnit = 8796093022208.0;  // 2^43
constexpr int kMaxChunk = LLOOM_B200_MAX_VOCAB / kMaxCluster;  // logits of a CTA

struct SampleParams {
    const void *logits;
    int type;
    int64_t ld;
    int vocab, chunk;  // chunk: logits per CTA
    const float *u, *temperature, *top_p, *min_p;  // per row; null: the number beside it (u: never null)
    const int *top_k;
    double temperature_all, top_p_all, min_p_all;
    int top_k_all;
    int64_t *ids;
    float *probs;
};

struct Border {  // the last kept token of a prefix: (key, index)
    uint32_t key, index;
};

struct Found {
    int bucket;
    uint32_t count, before;          // tokens in it and in front of it
    unsigned long long weight_before, total;
};

struct Shared {
    uint32_t count[kBuckets];  // read by the cluster's other CTAs, cleared behind a barrier of its own
    unsigned long long weight[kBuckets];
    double table[32];
    unsigned long long warp_w[kWarps];
    uint32_t warp_c[kWarps];
    // read by the other CTAs too; two of each, used in turn: what one exchange leaves is rewritten only behind the barrier of the next
    float max;
    uint2 range[2];
    uint32_t list_n[2];
    uint2 list[2][kList];
    unsigned long long sum[2];
    // this CTA's own
    uint2 all[kList];
    unsigned long long all_w[kList];
    Found found;
    Border border;
    unsigned long long target;
    uint32_t flag;
};

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_addr(const void *p, int rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ uint32_t peer_u32(const void *p, int rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(peer_addr(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ unsigned long long peer_u64(const void *p, int rank) {
    unsigned long long v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(peer_addr(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ uint4 peer_v4(const void *p, int rank) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(peer_addr(p, rank)) : "memory");
    return v;
}

// Bits of a logit in an order in which larger logits come first.  -0 counts as 0.
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t b = __float_as_uint(__fadd_rn(l, 0.0f));
    return (b & 0x80000000u) ? b : ~b & 0x7fffffffu;
}

struct Row {
    const float *logits;  // this CTA's, in shared memory
    int count, first;     // how many, index of the first
    int run;              // logits per thread, one after the other (odd: the threads of a warp read different banks)
    int ctas, rank;
    float max;
    double inv_t;
    __device__ __forceinline__ double depth(float l) const { return l == max ? 0.0 : ((double)max - (double)l) * inv_t; }
    __device__ __forceinline__ int bucket(float l) const {
        const double d = depth(l) * 64.0;
        return d < (double)(kBuckets - 1) ? (int)d : kBuckets - 1;  // NaN: the last
    }
};

// exp(-y), y >= 0; 0 from y = 32 on (beyond every weight that counts) and for NaN
__device__ __forceinline__ double exp_neg(double y, const double *table) {
    if (!(y < 32.0)) return 0.0;
    const double t = y * 46.166241308446828384;  // 32 / ln 2
    const int n = __double2int_rn(t);
    const double z = (t - (double)n) * 0.021660849392498290;  // ln 2 / 32
    double p = fma(z, -1.0 / 120.0, 1.0 / 24.0);
    p = fma(z, p, -1.0 / 6.0);
    p = fma(z, p, 0.5);
    p = fma(z, p, -1.0);
    p = fma(z, p, 1.0);
    p *= table[n & 31];
    return __hiloint2double(__double2hiint(p) - ((n >> 5) << 20), __double2loint(p));  // n / 32 <= 47: far from subnormal
}
__device__ __forceinline__ unsigned long long fixed_weight(double w) { return __double2ull_rn(w * kUnit); }

// share * total for 0 <= share < 1, exactly, rounded down or up to a whole number
__device__ __forceinline__ unsigned long long part_of(double share, unsigned long long total, bool up) {
    const unsigned long long bits = (unsigned long long)__double_as_longlong(share);
    const int exponent = (int)(bits >> 52) & 0x7ff, shift = 1075 - (exponent ? exponent : 1);  // share = mantissa / 2^shift, shift >= 53
    const unsigned long long mantissa = (bits & 0xfffffffffffffull) | (exponent ? 1ull << 52 : 0ull);
    const unsigned __int128 product = (unsigned __int128)mantissa * total;
    if (shift >= 128) return up && product ? 1ull : 0ull;
    const unsigned __int128 whole = product >> shift;
    return (unsigned long long)whole + (up && (whole << shift) != product ? 1ull : 0ull);
}

// f(logit, index) over this thread's tokens
template <class F>
__device__ __forceinline__ void each_token(const Row &row, F f) {
    const int begin = threadIdx.x * row.run, end = min(begin + row.run, row.count);
    for (int i = begin; i < end; ++i) f(row.logits[i], (uint32_t)(row.first + i));
}
__device__ __forceinline__ bool within(uint32_t key, uint32_t index, const Border &b) { return key < b.key || (key == b.key && index <= b.index); }

// Exclusive prefix sums over the CTA's threads, and the totals
__device__ __forceinline__ void block_scan(Shared &s, uint32_t c, unsigned long long w, uint32_t &c_before, unsigned long long &w_before,
                                           uint32_t &c_total, unsigned long long &w_total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t ci = c;
    unsigned long long wi = w;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const uint32_t cu = __shfl_up_sync(0xffffffffu, ci, off);
        const unsigned long long wu = __shfl_up_sync(0xffffffffu, wi, off);
        if (lane >= off) {
            ci += cu;
            wi += wu;
        }
    }
    __syncthreads();  // the last call's sums have been read
    if (lane == 31) {
        s.warp_c[warp] = ci;
        s.warp_w[warp] = wi;
    }
    __syncthreads();
    c_before = ci - c;
    w_before = wi - w;
    c_total = 0;
    w_total = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
        if (i < warp) {
            c_before += s.warp_c[i];
            w_before += s.warp_w[i];
        }
        c_total += s.warp_c[i];
        w_total += s.warp_w[i];
    }
}

// What a selection looks for: the K-th token, or the first at which the weights reach a share of their sum
struct Goal {
    bool by_weight;
    uint32_t k;
    double share;
};

// Adds up the CTAs' histograms and finds the bucket that the goal falls into: s.found, for all threads (bucket -1: none).  What lies in front
// of the first bucket counts too.  set_target: the goal's share of the sum of all weights becomes s.target.
__device__ void find_bucket(Shared &s, const Row &row, const Goal &goal, uint32_t count_before, unsigned long long weight_before, bool set_target) {
    uint32_t c[kPerThread] = {};
    unsigned long long w[kPerThread] = {};
    const int b0 = threadIdx.x * kPerThread;
    static_assert(kPerThread == 4, "vector loads of a thread's buckets");
    for (int q = 0; q < row.ctas; ++q) {
        const uint4 v = peer_v4(&s.count[b0], q);
        c[0] += v.x;
        c[1] += v.y;
        c[2] += v.z;
        c[3] += v.w;
        if (goal.by_weight) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint4 t = peer_v4(&s.weight[b0 + 2 * i], q);
                w[2 * i] += (unsigned long long)t.x | ((unsigned long long)t.y << 32);
                w[2 * i + 1] += (unsigned long long)t.z | ((unsigned long long)t.w << 32);
            }
        }
    }
    uint32_t cb, ct;
    unsigned long long wb, wt;
    block_scan(s, c[0] + c[1] + c[2] + c[3], w[0] + w[1] + w[2] + w[3], cb, wb, ct, wt);
    if (threadIdx.x == 0) {
        s.found.bucket = -1;
        if (set_target) {
            const unsigned long long t = goal.share > 0.0 ? part_of(goal.share, wt, true) : 0ull;
            s.target = t > 0 ? t : 1ull;
        }
    }
    __syncthreads();
    cb += count_before;
    wb += weight_before;
    const unsigned long long target = s.target;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
        const bool here = goal.by_weight ? wb < target && target <= wb + w[i] : cb < goal.k && goal.k <= cb + c[i];
        if (here) {
            s.found.bucket = b0 + i;
            s.found.count = c[i];
            s.found.before = cb;
            s.found.weight_before = wb;
        }
        cb += c[i];
        wb += w[i];
    }
    __syncthreads();
}

__device__ __forceinline__ void clear_histogram(Shared &s, bool weights, bool &used) {
    if (used) cluster_sync();  // the others have read the last one
    used = true;
    for (int i = threadIdx.x; i < kBuckets; i += kThreads) {
        s.count[i] = 0;
        if (weights) s.weight[i] = 0;
    }
    __syncthreads();
}

// The border of a prefix of the tokens within `limit` (all threads get it).  `turn`: which of the exchanged buffers is next; `used`: whether
// the histogram has been.
// Returns false where the border lies among tokens without weight, which no draw can reach: nothing is cut off then.
__device__ bool find_border(Shared &s, const Row &row, const Goal &goal, const Border &limit, int &turn, bool &used, Border &border) {
    // ---- buckets of (max - l) / T ----
    int h;
    clear_histogram(s, goal.by_weight, used);
    each_token(row, [&](float l, uint32_t index) {
        if (!within(key_of(l), index, limit)) return;
        const int b = row.bucket(l);
        atomicAdd(&s.count[b], 1u);
        if (goal.by_weight) {
            const unsigned long long w = fixed_weight(exp_neg(row.depth(l), s.table));
            if (w) atomicAdd(&s.weight[b], w);
        }
    });
    cluster_sync();
    find_bucket(s, row, goal, 0, 0, goal.by_weight);
    const int bucket = s.found.bucket;
    if (bucket < 0 || bucket == kBuckets - 1) return false;
    uint32_t count = s.found.count, before = s.found.before;
    unsigned long long weight_before = s.found.weight_before;
    uint32_t lo = 0, hi = 0xffffffffu;
    auto candidate = [&](float l, uint32_t key, uint32_t index) {
        return key >= lo && key <= hi && within(key, index, limit) && row.bucket(l) == bucket;
    };
    // ---- narrower and narrower ranges of the logits' bits ----
    if (count > kList) {
        uint32_t least = 0xffffffffu, most = 0;
        each_token(row, [&](float l, uint32_t index) {
            const uint32_t key = key_of(l);
            if (!candidate(l, key, index)) return;
            least = min(least, key);
            most = max(most, key);
        });
        least = __reduce_min_sync(0xffffffffu, least);
        most = __reduce_max_sync(0xffffffffu, most);
        h = turn & 1;
        ++turn;
        if (threadIdx.x == 0) s.range[h] = make_uint2(0xffffffffu, 0u);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) {
            atomicMin(&s.range[h].x, least);
            atomicMax(&s.range[h].y, most);
        }
        cluster_sync();
        lo = 0xffffffffu;
        hi = 0;
        for (int q = 0; q < row.ctas; ++q) {
            lo = min(lo, peer_u32(&s.range[h].x, q));
            hi = max(hi, peer_u32(&s.range[h].y, q));
        }
    }
    while (count > kList && lo < hi) {
        const uint32_t span = hi - lo;
        const int shift = span < (uint32_t)kBuckets ? 0 : 32 - __clz(span) - 11;
        clear_histogram(s, goal.by_weight, used);
        each_token(row, [&](float l, uint32_t index) {
            const uint32_t key = key_of(l);
            if (!candidate(l, key, index)) return;
            const int b = (int)((key - lo) >> shift);
            atomicAdd(&s.count[b], 1u);
            if (goal.by_weight) atomicAdd(&s.weight[b], fixed_weight(exp_neg(row.depth(l), s.table)));
        });
        cluster_sync();
        find_bucket(s, row, goal, before, weight_before, false);
        if (s.found.bucket < 0) return false;
        count = s.found.count;
        before = s.found.before;
        weight_before = s.found.weight_before;
        lo += (uint32_t)s.found.bucket << shift;
        hi = min(hi, lo + ((1u << shift) - 1u));
    }
    if (count <= kList) {
        // ---- the few that are left: every CTA collects them all and ranks them ----
        h = turn & 1;
        ++turn;
        if (threadIdx.x == 0) s.list_n[h] = 0;
        __syncthreads();
        each_token(row, [&](float l, uint32_t index) {
            const uint32_t key = key_of(l);
            if (candidate(l, key, index)) s.list[h][atomicAdd(&s.list_n[h], 1u)] = make_uint2(key, index);
        });
        cluster_sync();
        uint32_t at = 0;
        for (int q = 0; q < row.ctas; ++q) {
            const uint32_t n = peer_u32(&s.list_n[h], q);
            for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
                const unsigned long long e = peer_u64(&s.list[h][i], q);
                const uint32_t key = (uint32_t)e;
                s.all[at + i] = make_uint2(key, (uint32_t)(e >> 32));
                const float l = __uint_as_float((key & 0x80000000u) ? key : ~key & 0x7fffffffu);
                s.all_w[at + i] = goal.by_weight ? fixed_weight(exp_neg(row.depth(l), s.table)) : 0ull;
            }
            at += n;
        }
        __syncthreads();
        if (threadIdx.x < count) {
            const uint2 me = s.all[threadIdx.x];
            uint32_t rank = before;
            unsigned long long sum = weight_before;
            for (uint32_t i = 0; i < count; ++i) {
                const uint2 e = s.all[i];
                if (e.x < me.x || (e.x == me.x && e.y < me.y)) {
                    ++rank;
                    sum += s.all_w[i];
                }
            }
            const bool here = goal.by_weight ? sum < s.target && s.target <= sum + s.all_w[threadIdx.x] : rank + 1 == goal.k;
            if (here) s.border = {me.x, me.y};
        }
        __syncthreads();
        border = s.border;
        return true;
    }
    // ---- more equal logits than that: the n-th of them by index ----
    const float l = __uint_as_float((lo & 0x80000000u) ? lo : ~lo & 0x7fffffffu);
    uint32_t nth;
    if (goal.by_weight) {
        const unsigned long long w = fixed_weight(exp_neg(row.depth(l), s.table));
        nth = (uint32_t)((s.target - weight_before + w - 1) / w);  // w > 0: the target lies among these tokens' weights
    } else {
        nth = goal.k - before;
    }
    uint32_t mine = 0;
    each_token(row, [&](float v, uint32_t index) {
        const uint32_t key = key_of(v);
        if (key == lo && candidate(v, key, index)) ++mine;
    });
    uint32_t ahead, total;
    unsigned long long unused_a, unused_b;
    block_scan(s, mine, 0ull, ahead, unused_a, total, unused_b);
    h = turn & 1;
    ++turn;
    if (threadIdx.x == 0) {
        s.list_n[h] = total;
        s.flag = 0xffffffffu;
    }
    cluster_sync();
    for (int q = 0; q < row.rank; ++q) ahead += peer_u32(&s.list_n[h], q);
    if (ahead < nth && nth <= ahead + mine) {
        uint32_t left = nth - ahead;
        each_token(row, [&](float v, uint32_t index) {
            const uint32_t key = key_of(v);
            if (key == lo && candidate(v, key, index) && --left == 0) s.flag = index;
        });
    }
    // (list_n's other half: the CTA that has it tells the others)
    h = turn & 1;
    ++turn;
    __syncthreads();
    if (threadIdx.x == 0) s.list_n[h] = s.flag;
    cluster_sync();
    uint32_t index = 0xffffffffu;
    for (int q = 0; q < row.ctas; ++q) index = min(index, peer_u32(&s.list_n[h], q));
    border = {lo, index};
    return true;
}

__device__ __forceinline__ float load_logit(const void *p, int type, int64_t i) {
    float l;
    if (type == LLOOM_F32) l = __ldg(reinterpret_cast<const float *>(p) + i);
    else if (type == LLOOM_F16) l = __half2float(__ldg(reinterpret_cast<const __half *>(p) + i));
    else l = __bfloat162float(__ldg(reinterpret_cast<const __nv_bfloat16 *>(p) + i));
    return l == l ? l : -INFINITY;
}

__global__ void __launch_bounds__(kThreads) sample_kernel(const __grid_constant__ SampleParams p, int ctas) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    Shared &s = *reinterpret_cast<Shared *>(smem_raw);
    float *logits = reinterpret_cast<float *>(smem_raw + (sizeof(Shared) + 15) / 16 * 16);
    const int64_t b = blockIdx.x / ctas;
    Row row;
    row.ctas = ctas;
    row.rank = blockIdx.x - (int)b * ctas;
    row.logits = logits;
    row.first = min(row.rank * p.chunk, p.vocab);
    row.count = min(p.chunk, p.vocab - row.first);
    row.run = ((p.chunk + kThreads - 1) / kThreads) | 1;
    int turn = 0;
    bool used = false;
    launch_dependents();
    if (threadIdx.x < 32) s.table[threadIdx.x] = exp2(-(double)threadIdx.x / 32.0);
    wait_predecessor();
    // ---- the row, and its largest logit ----
    float top = -INFINITY;
    for (int i = threadIdx.x; i < row.count; i += kThreads) {
        const float l = load_logit(p.logits, p.type, b * p.ld + row.first + i);
        logits[i] = l;
        top = fmaxf(top, l);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    if ((threadIdx.x & 31) == 0) s.warp_c[threadIdx.x >> 5] = __float_as_uint(top);
    __syncthreads();
    for (int i = 0; i < kWarps; ++i) top = fmaxf(top, __uint_as_float(s.warp_c[i]));
    if (threadIdx.x == 0) s.max = top;
    cluster_sync();
    for (int q = 0; q < ctas; ++q) top = fmaxf(top, __uint_as_float(peer_u32(&s.max, q)));
    row.max = top;
    // ---- settings ----
    const double temperature = p.temperature ? (double)p.temperature[b] : p.temperature_all;
    const bool greedy = !(temperature > 0.0);
    row.inv_t = greedy ? 0.0 : 1.0 / temperature;
    const int top_k = p.top_k ? p.top_k[b] : p.top_k_all;
    const double top_p = p.top_p ? (double)p.top_p[b] : p.top_p_all, min_p = p.min_p ? (double)p.min_p[b] : p.min_p_all;
    Border limit = {0xffffffffu, 0xffffffffu};
    if (top > -INFINITY) {
        Border at;
        if (!greedy && top_k > 0 && top_k < p.vocab && find_border(s, row, Goal{false, (uint32_t)top_k, 0.0}, limit, turn, used, at)) limit = at;
        if (!greedy && top_p < 1.0 && find_border(s, row, Goal{true, 0u, top_p}, limit, turn, used, at)) limit = at;
    }
    // ---- the draw ----
    unsigned long long mine = 0;
    auto weight = [&](float l, uint32_t index) -> unsigned long long {
        if (l == -INFINITY || !within(key_of(l), index, limit)) return 0ull;
        if (greedy) return l == row.max ? 1ull : 0ull;
        const double w = exp_neg(row.depth(l), s.table);
        return w >= min_p || l == row.max || !(min_p > 0.0) ? fixed_weight(w) : 0ull;
    };
    each_token(row, [&](float l, uint32_t index) { mine += weight(l, index); });
    uint32_t unused_a, unused_b;
    unsigned long long ahead, total;
    block_scan(s, 0u, mine, unused_a, ahead, unused_b, total);
    const int h = turn & 1;
    if (threadIdx.x == 0) s.sum[h] = total;
    cluster_sync();
    unsigned long long all = 0;
    for (int q = 0; q < ctas; ++q) {
        const unsigned long long t = peer_u64(&s.sum[h], q);
        if (q < row.rank) ahead += t;
        all += t;
    }
    if (all == 0) {  // nothing above -inf
        if (row.rank == 0 && threadIdx.x == 0) {
            p.ids[b] = -1;
            if (p.probs) p.probs[b] = 0.0f;
        }
    } else {
        const double u = (double)p.u[b];
        const unsigned long long t = greedy || !(u > 0.0) ? 0ull : u < 1.0 ? part_of(u, all, false) : all - 1;
        if (ahead <= t && t < ahead + mine) {
            unsigned long long sum = ahead;
            bool found = false;
            each_token(row, [&](float l, uint32_t index) {
                sum += weight(l, index);
                if (!found && sum > t) {
                    found = true;
                    p.ids[b] = (int64_t)index;
                    if (p.probs) p.probs[b] = greedy ? 1.0f : (float)(exp_neg(row.depth(l), s.table) * kUnit / (double)all);
                }
            });
        }
    }
    cluster_sync();  // the others may still read this CTA's memory
}

struct SmemOnce {
    std::mutex mu;
    bool done[64] = {false};
};

}  // namespace

int sample(const void *logits, int type, int64_t batch, int64_t vocab, int64_t ld, const float *u, const float *temperature, double temperature_all,
           const int *top_k, int64_t top_k_all, const float *top_p, double top_p_all, const float *min_p, double min_p_all, int64_t *ids,
           float *probs, void *stream, bool overlap) {
    if (!elem_type_ok(type)) return LLOOM_ERR_DTYPE;
    if (batch <= 0 || vocab <= 0 || ld < vocab || vocab > LLOOM_B200_MAX_VOCAB || batch > (1 << 24)) return LLOOM_ERR_SHAPE;
    if (!logits || !u || !ids) return LLOOM_ERR_NULL;
    const uintptr_t es = type == LLOOM_F32 ? 4 : 2;
    if (!aligned(logits, es) || !aligned(u, 4) || !aligned(ids, 8) || !aligned(probs, 4) || !aligned(temperature, 4) || !aligned(top_k, 4) ||
        !aligned(top_p, 4) || !aligned(min_p, 4))
        return LLOOM_ERR_ALIGN;
    if ((!temperature && !(temperature_all >= 0.0)) || (!top_k && top_k_all < 0) || (!top_p && !(top_p_all >= 0.0 && top_p_all <= 1.0)) ||
        (!min_p && !(min_p_all >= 0.0 && min_p_all <= 1.0)))
        return LLOOM_ERR_VALUE;
    DeviceInfo di;
    int rc = device_info(di);
    if (rc != LLOOM_OK) return rc;
    SampleParams p = {};
    p.logits = logits;
    p.type = type;
    p.ld = ld;
    p.vocab = (int)vocab;
    p.u = u;
    p.temperature = temperature;
    p.top_k = top_k;
    p.top_p = top_p;
    p.min_p = min_p;
    p.temperature_all = temperature_all;
    p.top_k_all = (int)(top_k_all < vocab ? top_k_all : 0);
    p.top_p_all = top_p_all;
    p.min_p_all = min_p_all;
    p.ids = ids;
    p.probs = probs;
    int ctas = 1;
    while (ctas < kMaxCluster && vocab > (int64_t)ctas * 4096) ctas *= 2;
    p.chunk = (int)((vocab + ctas - 1) / ctas);
    const int smem = (int)((sizeof(Shared) + 15) / 16 * 16) + p.chunk * 4;
    static SmemOnce once;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || dev < 0 || dev >= 64) return LLOOM_ERR_DEVICE;
    {
        static_assert(sizeof(Shared) + 16 + kMaxChunk * 4 <= 227 * 1024, "shared memory");
        std::lock_guard<std::mutex> lock(once.mu);
        if (!once.done[dev]) {
            e = cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, di.max_smem_optin);
            if (e != cudaSuccess) return launch_status(e);
            once.done[dev] = true;
        }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(batch * ctas));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap ? 2 : 1;
    return launch_status(cudaLaunchKernelEx(&cfg, sample_kernel, p, ctas));
}

}  // namespace lloom

using namespace lloom;

extern "C" int lloom_b200_sample(const void *logits, int type, int64_t batch, int64_t vocab, int64_t ld, const float *u, const float *temperature,
                                 double temperature_all, const int *top_k, int64_t top_k_all, const float *top_p, double top_p_all,
                                 const float *min_p, double min_p_all, int64_t *ids, float *probs, void *stream) {
    return sample(logits, type, batch, vocab, ld, u, temperature, temperature_all, top_k, top_k_all, top_p, top_p_all, min_p, min_p_all, ids,
                  probs, stream, launch_overlap() > 0);
}
