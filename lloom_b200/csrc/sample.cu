// The next token of every row of logits: temperature, top-k, top-p (nucleus) and min-p filters and a draw from a given uniform number.
//
//   w_i = exp((l_i - max) / T); tokens in the order (logit falling, index rising); kept: the shortest of three prefixes of it -- the first
//   K, the first whose weights reach P times those of the first K, those with w_i >= min_p; drawn: of the kept ones, by rising index, the
//   first whose running sum of weights exceeds u times their sum.
//
// A cluster of CTAs has a row: it is read once, stays in shared memory, and everything after works there.  A filter's border is found by
// a histogram over 2048 buckets of (max - l) / T, 1/64 wide, then within the bucket that holds it: by further histograms over the bits of the
// logits while it has more than 512 tokens, else by sorting these; equal logits by index.  Where all tokens up to the border are no more
// than 256, the draw needs these alone.  No sort of the row.  (With 256 sorted by counting, 16 rows of 128256 at temperatures up to 1.5, whose
// border buckets have 300 to 500 tokens, took 59 us instead of 41.)
//
// Weights are summed as integers, in units of 2^-43 of the largest weight: the sums are exact, so that they depend neither on
// the split of a row nor on the order of atomics, and borders fall where 64-bit arithmetic puts them.  (In 32 bits a running sum over
// 100,000 tokens is off by more than a token's share of it.)  Tokens below 2^-44 of the largest weight count as zero.
// exp in 64-bit arithmetic: the difference to the maximum times 1 / (T ln 2) is split into a whole number, the exponent, and the rest, a polynomial of
// degree 9; relative error below 3e-14 at every temperature and size of the logits.
//
// Bound by latency for a few rows: a launch, one read of DRAM, six to eight cluster barriers of about a microsecond with short passes between
// them (1 x 128256 f32 with all filters 15.4 us, 7 x 50257 bf16 with top-p 33).  For many rows by instruction issue and barriers
// (issue slots 54 % taken, the 64-bit pipe 10 %, shared memory's 25 %; half of the instructions are per logit, half per CTA): 64 x 128256 f32, 33 MB,
// settings of their own, 70 us.
// There a row read from L2 in every pass by fewer CTAs, all rows at once, was faster for alike rows (75 us for 85) and slower for unlike ones (126 for 84).
#include <mutex>
#include <type_traits>

#include "abi.h"
#include "common.cuh"
#include "forward.h"

namespace lloom {

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBuckets = 2048;
constexpr int kList = 256;       // tokens that the draw needs alone: every one up to the border
constexpr int kLast = kThreads;  // tokens of the border's bucket that are sorted
constexpr int kMaxCluster = 8;
constexpr int kMaxChunk = LLOOM_B200_MAX_VOCAB / kMaxCluster;  // logits of a CTA
constexpr double kLeastTemperature = 7.5231638452626401e-37;  // 2^-120: 2^896 / T stays finite
constexpr int kSpan = 128;                 // logits that a warp looks at together: four per lane
constexpr double kUnit = 8796093022208.0;  // 2^43: the largest weight

struct SampleParams {
    const void *logits;
    int type;
    int64_t ld;
    int vocab, chunk, share;  // chunk: logits per CTA; share: places per warp for them
    const float *u, *temperature, *top_p, *min_p;  // per row; null: the number beside it (u: never null)
    const int *top_k;
    double temperature_all, top_p_all, min_p_all;
    int top_k_all;
    int64_t *ids;
    float *probs;
};

struct Border {  // the last token of a prefix: (key, index)
    uint32_t key, index;
};

struct Shared {
    // a histogram of tokens, or of weights (bits 0-14, 15-29 and the rest, each summed on its own); read by the cluster's other CTAs, cleared behind a barrier of its own
    // (the draw uses the place for kept logits that wait for their weights)
    union {
        struct {
            uint32_t low[kBuckets], mid[kBuckets], high[kBuckets];
        };
        struct {
            float batch[kWarps][2 * kSpan];
            uint16_t place[kWarps][2 * kSpan];  // (kMaxChunk < 2^16)
        };
        struct {  // (`low` and `high` stay free in the draw from a list)
            uint32_t low_[kBuckets];
            struct alignas(16) {
                uint2 token;  // (index, key): in order as one number
                unsigned long long weight;
            } list[kLast];
            unsigned long long exchange[2][kThreads];
        };
    };
    unsigned long long warp_w[kWarps];
    unsigned long long half_w[kList];
    uint32_t half_n[kList];
    unsigned long long part_total;  // of all histograms over this CTA's share of the buckets
    // read by the other CTAs too; two of each, used in turn: what one exchange leaves is rewritten only behind the barrier of the next
    float max;
    uint2 range[2];
    uint32_t listed[2], last_n[2];  // listed: lengths of the lists, of `last` in the upper half (a CTA has fewer than 2^16 tokens)
    uint2 upto[2][kList], last[2][kLast];
    unsigned long long sum[2];
    // this CTA's own
    unsigned long long before, target, total;
    uint2 own[kWarps];
    int bucket;
    Border border;
    uint32_t flag;
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
    cluster_arrive();
    cluster_wait();
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

// Bits of a logit in an order in which larger logits come first (-0 counts as 0), and back
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t b = __float_as_uint(__fadd_rn(l, 0.0f));
    return (b & 0x80000000u) ? b : ~b & 0x7fffffffu;
}
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? key : ~key & 0x7fffffffu); }

struct Row {
    const float *logits;  // this CTA's, in shared memory; -infinity around them, where a warp's share is not full
    int first;            // index of logits[0] in the row (that of the first logit, less the padding in front of it)
    int begin, end;       // indices of this CTA's
    int share;            // logits per warp, a multiple of kSpan
    unsigned long long *part;  // this CTA's, in shared memory: running sums of all histograms over its share of the buckets
    int ctas, rank;
    float max;            // finite
    double wide_max, slope; // the maximum as widen() has it; slope * (wide_max - widen(l)) = (max - l) / T / ln 2
    float bucket_scale;   // 64 / T, finite
    double least;         // min_p in units of 2^-43

    // (max - l) / T in 1/64, rounded to a bucket; the last one from 32 on, where weights are zero.  Every step keeps the order of the
    // logits, so that a bucket is a range of them; 32 bits will do.
    __device__ __forceinline__ float depth(float l) const { return __fmul_rn(__fsub_rn(max, l), bucket_scale); }
    __device__ __forceinline__ int bucket(float l) const { return (int)(__float_as_uint(__fadd_rn(fminf(depth(l), (float)(kBuckets - 1)), 8388608.0f)) & 0x7fffffu); }
    // l * 2^-896, exactly, subnormal ones too: its bits, moved to the places of a double's
    static __device__ __forceinline__ double widen(float l) {
        const uint32_t bits = __float_as_uint(l);
        return __hiloint2double((int)(((int)bits >> 3) & 0x8fffffff), (int)(bits << 29));
    }
    // exp(-(max - l) / T) in units of 2^-43, for tokens with `counts`: 2^-n by the exponent, 2^-z, |z| <= 1/2, by a polynomial fitted at
    // Chebyshev nodes (2e-14).  No conversions (eight cycles a warp; a multiply-add takes two) and no table (a random look-up in shared memory
    // costs more than the five multiply-adds it would save): whole numbers are read from sums with 1.5 * 2^52.
    // The difference comes first, then the factor: for n + z = 46 at most (`counts`) the two roundings are off by 46 * 2^-52, whatever the logits'
    // size, and the maximum's own weight is that of 0.  (Two products, of the maximum and of the logit, would each be rounded at the size of max / T.)
    __device__ __forceinline__ bool counts(float l) const { return depth(l) < (float)(kBuckets - 1) - 0.5f; }
    __device__ __forceinline__ double units(float l) const {
        constexpr double magic = 6755399441055744.0;
        const double below = wide_max - widen(l), m = fma(below, slope, magic), z = fma(below, slope, magic - m);
        double p = fma(z, -1.0205905407077635e-07 * kUnit, 1.3259645243921192e-06 * kUnit);
        p = fma(z, p, -1.5252672924891586e-05 * kUnit);
        p = fma(z, p, 0.00015403433751254647 * kUnit);
        p = fma(z, p, -0.0013333558200794562 * kUnit);
        p = fma(z, p, 0.0096181291939343126 * kUnit);
        p = fma(z, p, -0.05550410866465167 * kUnit);
        p = fma(z, p, 0.24022650695640341 * kUnit);
        p = fma(z, p, -0.69314718055994617 * kUnit);
        p = fma(z, p, 1.0000000000000135 * kUnit);
        return __hiloint2double(__double2hiint(p) - (__double2loint(m) << 20), __double2loint(p));
    }
    // The same as a whole number, 0 below min_p
    __device__ __forceinline__ unsigned long long weight(float l) const {
        const double w = units(l);
        return counts(l) && (w >= least || l == max) ? whole(w) : 0ull;
    }
    static __device__ __forceinline__ unsigned long long whole(double w) {
        return (unsigned long long)__double_as_longlong(w + 4503599627370496.0) - 0x4330000000000000ull;  // + 2^52
    }
};

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

// f(four logits, index of the first) over the warp's share, a span at a time: all lanes call it
template <class F>
__device__ __forceinline__ void each_span(const Row &row, F f) {
    const int begin = (threadIdx.x >> 5) * row.share + (threadIdx.x & 31) * 4, end = ((threadIdx.x >> 5) + 1) * row.share;
#pragma unroll 1
    for (int i = begin; i < end; i += kSpan) {
        const float4 v = *reinterpret_cast<const float4 *>(row.logits + i);
        const float l[4] = {v.x, v.y, v.z, v.w};
        f(l, row.first + i);
    }
}
// f(logit, index) over this lane's logits whose depth is at most `most`
template <class F>
__device__ __forceinline__ void each_near(const Row &row, float most, F f) {
    each_span(row, [&](const float (&l)[4], int index) {
        bool near[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) near[j] = row.depth(l[j]) <= most;
        if (near[0] || near[1] || near[2] || near[3]) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (near[j]) f(l[j], (uint32_t)(index + j));
        }
    });
}
__device__ __forceinline__ bool within(uint32_t key, uint32_t index, const Border &b) { return key < b.key || (key == b.key && index <= b.index); }

// The warp's tokens that pass a cheap test, gathered until f can have four of them in every lane: f(logits, indices, which of the four there
// are), called by all lanes.  What follows for a token that counts (keys, lists, 64-bit weights) takes ten times the test's instructions.
struct Gather {
    float *logit;  // of the warp: room for two spans
    uint16_t *place;
    int waiting = 0;
    __device__ __forceinline__ Gather(Shared &s) : logit(s.batch[threadIdx.x >> 5]), place(s.place[threadIdx.x >> 5]) {}
    template <class F>
    __device__ __forceinline__ void add(const Row &row, const float (&l)[4], int index, const bool (&take)[4], F f) {
        if (!__any_sync(0xffffffffu, take[0] || take[1] || take[2] || take[3])) return;
        const unsigned below = (1u << (threadIdx.x & 31)) - 1u;
        int at = waiting;  // (a population count takes a warp eight cycles)
#pragma unroll
        for (int j = 0; j < 4; ++j) at += __popc(__ballot_sync(0xffffffffu, take[j]) & below);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (take[j]) {
                logit[at] = l[j];
                place[at] = (uint16_t)(index + j - row.first);
                ++at;
            }
        waiting = __shfl_sync(0xffffffffu, at, 31);
        __syncwarp();
        if (waiting >= kSpan) some(row, kSpan, f);
    }
    template <class F>
    __device__ __forceinline__ void finish(const Row &row, F f) {
        if (waiting > 0) some(row, waiting, f);
    }
    template <class F>
    __device__ __forceinline__ void some(const Row &row, int n, F f) {  // the last n, at most a span
        waiting -= n;
        float l[4];
        uint32_t index[4];
        bool there[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = 32 * j + (threadIdx.x & 31);
            there[j] = i < n;
            l[j] = there[j] ? logit[waiting + i] : -INFINITY;
            index[j] = (uint32_t)row.first + (there[j] ? place[waiting + i] : 0u);
        }
        __syncwarp();
        f(l, index, there);
    }
};

// Exclusive prefix sum over the CTA's threads, and the total
__device__ __forceinline__ void block_scan(Shared &s, unsigned long long w, unsigned long long &before, unsigned long long &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long wi = w;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const unsigned long long up = __shfl_up_sync(0xffffffffu, wi, off);
        if (lane >= off) wi += up;
    }
    __syncthreads();  // the last call's sums have been read
    if (lane == 31) s.warp_w[warp] = wi;
    __syncthreads();
    before = wi - w;
    total = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
        const unsigned long long v = s.warp_w[i];
        if (i < warp) before += v;
        total += v;
    }
}

// What a selection looks for: the K-th token, or the first at which the weights reach a share of their sum
struct Goal {
    bool by_weight;
    double share;
};

// To a histogram's bucket, of tokens or of weights.  Predicated, not branched around: a branch per token kept the arithmetic of four tokens
// from running side by side.
__device__ __forceinline__ void add_nonzero(uint32_t *p, uint32_t v) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %1, 0;\n\t@p red.shared.add.u32 [%0], %1;\n\t}\n" ::"r"(smem_u32(p)), "r"(v) : "memory");
}
__device__ __forceinline__ void add_tokens(Shared &s, int b, uint32_t n) { add_nonzero(&s.low[b], n); }
// A CTA has fewer than 2^16 tokens, so that none of the three sums overflows.  (Shared memory has no 64-bit addition: a loop of compare-and-
// swaps took 75 to 370 cycles a warp; two words with a carry between them wait for the first one's answer.)
__device__ __forceinline__ void add_weight(Shared &s, int b, unsigned long long w) {
    static_assert(kMaxChunk < (1 << 16), "sums of 16-bit pieces");
    add_nonzero(&s.low[b], (uint32_t)w & 0x7fffu);
    add_nonzero(&s.mid[b], (uint32_t)(w >> 15) & 0x7fffu);
    add_nonzero(&s.high[b], (uint32_t)(w >> 30));
}

// Adds up the CTAs' histograms and finds the bucket in which the sum reaches s.target: s.bucket (-1: none) and s.before, the sum in front of
// it (`before` in front of the first), for all threads.  set_target: a share of the sum of all weights becomes the target first.
// Every CTA adds up its share of the buckets for the others: reading all of all histograms everywhere took 6 us of a row's 32.
__device__ void find_bucket(Shared &s, const Row &row, const Goal &goal, unsigned long long before, bool set_target) {
    const int share = kBuckets / row.ctas, lane = threadIdx.x & 31;
    {  // four buckets of one CTA's histogram per thread, neighbouring threads the same of the others'
        static_assert(kBuckets == 4 * kThreads, "a thread has one piece");
        const int q = threadIdx.x & (row.ctas - 1), b = threadIdx.x / row.ctas * 4;
        const int at = row.rank * share + b;
        const uint4 lo = peer_v4(&s.low[at], q);
        unsigned long long w[4] = {lo.x, lo.y, lo.z, lo.w};
        if (goal.by_weight) {
            const uint4 mid = peer_v4(&s.mid[at], q), hi = peer_v4(&s.high[at], q);
            w[0] += ((unsigned long long)mid.x << 15) + ((unsigned long long)hi.x << 30);
            w[1] += ((unsigned long long)mid.y << 15) + ((unsigned long long)hi.y << 30);
            w[2] += ((unsigned long long)mid.z << 15) + ((unsigned long long)hi.z << 30);
            w[3] += ((unsigned long long)mid.w << 15) + ((unsigned long long)hi.w << 30);
        }
        for (int off = 1; off < row.ctas; off <<= 1)
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] += __shfl_xor_sync(0xffffffffu, w[j], off);
        if (q == 0)
#pragma unroll
            for (int j = 0; j < 4; ++j) row.part[b + j] = w[j];
    }
    __syncthreads();
    {  // running sums of the share
        const int per = (share + kThreads - 1) / kThreads, b0 = threadIdx.x * per;
        unsigned long long mine = 0, ahead, total;
        for (int i = 0; i < per; ++i) mine += b0 + i < share ? row.part[b0 + i] : 0ull;
        block_scan(s, mine, ahead, total);
        for (int i = 0; i < per; ++i)
            if (b0 + i < share) {
                const unsigned long long w = row.part[b0 + i];
                ahead += w;
                row.part[b0 + i] = ahead;
            }
        if (threadIdx.x == 0) s.part_total = total;
    }
    cluster_sync();
    unsigned long long sum = lane < row.ctas ? peer_u64(&s.part_total, lane) : 0ull;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const unsigned long long up = __shfl_up_sync(0xffffffffu, sum, off);
        if (lane >= off) sum += up;
    }
    const unsigned long long total = __shfl_sync(0xffffffffu, sum, 31);
    if (threadIdx.x == 0) {
        s.bucket = -1;
        if (set_target) {
            const unsigned long long t = goal.share > 0.0 ? part_of(goal.share, total, true) : 0ull;
            s.target = t > 0 ? t : 1ull;
        }
    }
    __syncthreads();
    const unsigned long long target = s.target;
    const unsigned reached = __ballot_sync(0xffffffffu, target <= before + sum);
    if (target > before && reached) {
        const int owner = __ffs(reached) - 1;
        const unsigned long long from = before + (owner ? __shfl_sync(0xffffffffu, sum, owner - 1) : 0ull);
        for (int i = threadIdx.x; i < share; i += kThreads) {
            const unsigned long long up_to = from + peer_u64(&row.part[i], owner), in_front = i ? from + peer_u64(&row.part[i - 1], owner) : from;
            if (in_front < target && target <= up_to) {
                s.bucket = owner * share + i;
                s.before = in_front;
            }
        }
    }
    __syncthreads();
}

__device__ __forceinline__ void clear_histogram(Shared &s, bool weights, bool &used) {
    if (used) cluster_sync();  // the others have read the last one
    used = true;
    for (int i = threadIdx.x; i < kBuckets; i += kThreads) {
        s.low[i] = 0;
        if (weights) s.mid[i] = s.high[i] = 0;
    }
    __syncthreads();
}

// The cluster's lists (of up to kLast tokens in all) as one: s.list.  A warp per CTA that has one; n: how many the lane's has.
template <bool WEIGHTS>
__device__ __forceinline__ void collect(Shared &s, const Row &row, uint32_t n, const uint2 *of) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t at = __reduce_add_sync(0xffffffffu, lane < warp ? n : 0u), mine = __shfl_sync(0xffffffffu, n, warp);
    if (warp < row.ctas)
        for (uint32_t i = lane; i < mine; i += 32) {
            const unsigned long long e = peer_u64(of + i, warp);
            s.list[at + i].token = make_uint2((uint32_t)(e >> 32), (uint32_t)e);
            if constexpr (WEIGHTS) s.list[at + i].weight = row.counts(logit_of((uint32_t)e)) ? Row::whole(row.units(logit_of((uint32_t)e))) : 0ull;
        }
    __syncthreads();
}
// One value per thread of the first n to rising order (bitonic; those behind bring the largest value).  Warps behind all n only keep step.
__device__ __forceinline__ unsigned long long sort_threads(Shared &s, unsigned long long v, uint32_t n) {
    int turn = 0;
    const bool busy = (threadIdx.x & ~31u) < n || (threadIdx.x & ~31u) < (1u << (32 - __clz(n - 1)));
    auto step = [&](unsigned size, unsigned stride, unsigned long long other) {
        return (((threadIdx.x & size) == 0) == ((threadIdx.x & stride) == 0)) == (other < v) ? other : v;
    };
    for (unsigned size = 2; size < 2 * n; size <<= 1) {
        for (unsigned stride = size >> 1; stride >= 32; stride >>= 1) {
            if (busy) s.exchange[turn][threadIdx.x] = v;
            __syncthreads();
            if (busy) v = step(size, stride, s.exchange[turn][threadIdx.x ^ stride]);
            turn ^= 1;
        }
        if (busy)
            for (unsigned stride = min(size >> 1, 16u); stride > 0; stride >>= 1) v = step(size, stride, __shfl_xor_sync(0xffffffffu, v, stride));
    }
    return v;
}
// How many of the list's tokens come before the thread's own (list[threadIdx.x % kList]), and their weights; two threads share a token, and
// the second half's answer is no use
__device__ __forceinline__ uint32_t rank_in_list(Shared &s, uint32_t n, unsigned long long &sum) {
    static_assert(kThreads == 2 * kList, "two threads per token");
    const uint32_t own = threadIdx.x & (kList - 1), half = threadIdx.x / kList, begin = half ? n / 2 : 0, end = half ? n : n / 2;
    uint32_t rank = 0;
    sum = 0;
    if (own < n) {
        auto order = [](const uint4 &e) { return ((unsigned long long)e.y << 32) | e.x; };
        const uint4 *list = reinterpret_cast<const uint4 *>(s.list);
        const unsigned long long me = order(list[own]);
#pragma unroll 4
        for (uint32_t i = begin; i < end; ++i) {
            const uint4 e = list[i];
            if (order(e) < me) {
                ++rank;
                sum += (unsigned long long)e.z | ((unsigned long long)e.w << 32);
            }
        }
        if (half) {
            s.half_n[own] = rank;
            s.half_w[own] = sum;
        }
    }
    __syncthreads();
    if (!half && own < n) {
        rank += s.half_n[own];
        sum += s.half_w[own];
    }
    __syncthreads();
    return rank;
}

enum Selected {
    kNothing,  // the border lies among tokens without weight, which no draw can reach: nothing is cut off
    kBorder,   // the border
    kListed    // every token up to the border, and a few behind it, is in the first CTA's list
};

// Looks for the goal (s.target: in tokens, or set here from its share) among the tokens within `limit`.  `turn`: which of the exchanged
// buffers is next; `used`: whether the histogram has been; `listed`: length of the list.  LIMITED: `limit` is one.  final: no other border comes
// behind this one; `sum` is then the lane's part of the weights of its warp's tokens up to the border (kBorder).
template <bool LIMITED>
__device__ Selected find_border(Shared &s, const Row &row, const Goal &goal, const Border &limit, bool final, int &turn, bool &used, Border &border,
                                uint32_t &listed, unsigned long long &sum) {
    auto inside = [&](float l, uint32_t index) { return !LIMITED || within(key_of(l), index, limit); };
    // ---- buckets of (max - l) / T ----
    clear_histogram(s, goal.by_weight, used);
    if (goal.by_weight) {
        each_span(row, [&](const float (&l)[4], int index) {
            unsigned long long w[4];
            int b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const double units = row.units(l[j]);
                b[j] = row.bucket(l[j]);
                w[j] = row.counts(l[j]) && inside(l[j], (uint32_t)(index + j)) ? Row::whole(units) : 0ull;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) add_weight(s, b[j], w[j]);
        });
    } else {
        each_span(row, [&](const float (&l)[4], int index) {
#pragma unroll
            for (int j = 0; j < 4; ++j) add_tokens(s, row.bucket(l[j]), row.counts(l[j]) && inside(l[j], (uint32_t)(index + j)) ? 1u : 0u);
        });
    }
    cluster_sync();
    find_bucket(s, row, goal, 0, goal.by_weight);
    const int bucket = s.bucket;
    if (bucket < 0 || bucket == kBuckets - 1) return kNothing;
    unsigned long long before = s.before;
    uint32_t lo = 0, hi = 0xffffffffu;  // keys that the border may have
    auto candidate = [&](float l, uint32_t key, uint32_t index) {
        return key >= lo && key <= hi && within(key, index, limit) && row.bucket(l) == bucket;
    };
    // the largest depths that round to the bucket, and to the one in front of it
    const float most = (bucket & 1) ? __uint_as_float(__float_as_uint((float)bucket + 0.5f) - 1u) : (float)bucket + 0.5f;
    const float most_front = bucket == 0 ? -1.0f : (bucket & 1) ? (float)bucket - 0.5f : __uint_as_float(__float_as_uint((float)bucket - 0.5f) - 1u);
    const int lane = threadIdx.x & 31;
    bool ranged = false, ranked = false;
    for (;;) {
        // ---- the tokens that are left (and, the first time, all in front of them), if they are few ----
        const int h = turn & 1;
        ++turn;
        if (threadIdx.x == 0) s.listed[h] = 0;
        __syncthreads();
        // while the longer list has room; counted tokens in front say beforehand whether it has
        const bool all_few = !ranged && (goal.by_weight || before < kList);
        bool open = all_few;
        unsigned long long front = 0;  // weights of tokens in the buckets in front
        auto look = [&](const float (&l)[4], const uint32_t (&index)[4], const bool (&there)[4]) {
            unsigned here[4], ahead[4];
            uint32_t key[4], n_here = 0, n_ahead = 0;
            unsigned long long w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = final && !ranged ? row.weight(l[j]) : 0ull;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool in_front = row.depth(l[j]) <= most_front, in = there[j] && inside(l[j], index[j]);
                key[j] = key_of(l[j]);
                here[j] = __ballot_sync(0xffffffffu, in && !in_front && key[j] >= lo && key[j] <= hi);
                ahead[j] = __ballot_sync(0xffffffffu, in && in_front);
                n_here += __popc(here[j]);
                n_ahead += __popc(ahead[j]);
                front += in && in_front ? w[j] : 0ull;
            }
            // places for the warp's tokens at once
            const uint32_t n_upto = open ? n_here + n_ahead : 0u, n = n_here << 16 | n_upto;
            if (n == 0) return;
            uint32_t at = 0;
            if (lane == 0) at = atomicAdd(&s.listed[h], n);
            at = __shfl_sync(0xffffffffu, at, 0);
            uint32_t last = at >> 16, upto = at & 0xffffu;
            open = open && upto + n_upto <= kList;
            const unsigned below = (1u << lane) - 1u;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const unsigned all = here[j] | ahead[j];
                const uint32_t to_last = last + __popc(here[j] & below), to_upto = upto + __popc(all & below);
                if ((here[j] >> lane & 1u) && to_last < kLast) s.last[h][to_last] = make_uint2(key[j], index[j]);
                if (n_upto && (all >> lane & 1u) && to_upto < kList) s.upto[h][to_upto] = make_uint2(key[j], index[j]);
                last += __popc(here[j]);
                upto += __popc(all);
            }
        };
        Gather near(s);
        each_span(row, [&](const float (&l)[4], int index) {
            bool take[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float d = row.depth(l[j]);
                take[j] = d <= most && (d > most_front || open || (final && !ranged));
            }
            near.add(row, l, index, take, look);
        });
        near.finish(row, look);
        if (final && !ranged) sum = front;
        cluster_sync();
        const uint32_t of = lane < row.ctas ? peer_u32(&s.listed[h], lane) : 0u, upto_of = of & 0xffffu, last_of = of >> 16;
        const uint32_t upto_n = __reduce_add_sync(0xffffffffu, upto_of), last_n = __reduce_add_sync(0xffffffffu, last_of);
        if (all_few && upto_n <= kList) {
            if (row.rank == 0) collect<true>(s, row, upto_of, s.upto[h]);
            listed = upto_n;
            return kListed;
        }
        if (last_n <= kLast) {
            if (threadIdx.x < kWarps) s.own[threadIdx.x] = make_uint2(0u, 0u);
            collect<false>(s, row, last_of, s.last[h]);
            auto order = [](uint2 t) { return ((unsigned long long)t.y << 32) | t.x; };
            const bool has = threadIdx.x < last_n;
            const unsigned long long me = sort_threads(s, has ? order(s.list[threadIdx.x].token) : ~0ull, last_n);
            const uint32_t key = (uint32_t)(me >> 32), index = (uint32_t)me;
            const float l = logit_of(key);
            const double units = row.units(l);
            const unsigned long long w = has && row.counts(l) ? Row::whole(units) : 0ull, mine = goal.by_weight ? w : has ? 1ull : 0ull;
            unsigned long long from, all;
            block_scan(s, mine, from, all);
            from += before;
            if (from < s.target && s.target <= from + mine) s.border = {key, index};
            __syncthreads();
            border = s.border;
            if (!final) return kBorder;
            if (!ranged) {  // the warps' own of the list, up to the border, in two pieces
                const uint32_t at = index - (uint32_t)row.first;
                if (has && index >= (uint32_t)row.begin && index < (uint32_t)row.end && within(key, index, border) && (units >= row.least || l == row.max)) {
                    atomicAdd(&s.own[at / (uint32_t)row.share].x, (uint32_t)w & 0x3fffffu);
                    atomicAdd(&s.own[at / (uint32_t)row.share].y, (uint32_t)(w >> 22));
                }
                __syncthreads();
                if (lane == 0) sum += s.own[threadIdx.x >> 5].x + ((unsigned long long)s.own[threadIdx.x >> 5].y << 22);
                return kBorder;
            }
            ranked = true;
            break;
        }
        // ---- else narrower and narrower ranges of the logits' bits ----
        if (!ranged) {
            ranged = true;
            uint32_t low_key = 0xffffffffu, high_key = 0;
            each_near(row, most, [&](float l, uint32_t index) {
                const uint32_t key = key_of(l);
                if (!candidate(l, key, index)) return;
                low_key = min(low_key, key);
                high_key = max(high_key, key);
            });
            low_key = __reduce_min_sync(0xffffffffu, low_key);
            high_key = __reduce_max_sync(0xffffffffu, high_key);
            const int g = turn & 1;
            ++turn;
            if (threadIdx.x == 0) s.range[g] = make_uint2(0xffffffffu, 0u);
            __syncthreads();
            if ((threadIdx.x & 31) == 0) {
                atomicMin(&s.range[g].x, low_key);
                atomicMax(&s.range[g].y, high_key);
            }
            cluster_sync();
            lo = 0xffffffffu;
            hi = 0;
            for (int q = 0; q < row.ctas; ++q) {
                lo = min(lo, peer_u32(&s.range[g].x, q));
                hi = max(hi, peer_u32(&s.range[g].y, q));
            }
        }
        if (lo >= hi) break;
        const uint32_t span = hi - lo;
        const int shift = span < (uint32_t)kBuckets ? 0 : 32 - __clz(span) - 11;
        clear_histogram(s, goal.by_weight, used);
        each_near(row, most, [&](float l, uint32_t index) {
            const uint32_t key = key_of(l);
            if (!candidate(l, key, index)) return;
            const int b = (int)((key - lo) >> shift);
            if (goal.by_weight) add_weight(s, b, Row::whole(row.units(l)));
            else add_tokens(s, b, 1u);
        });
        cluster_sync();
        find_bucket(s, row, goal, before, false);
        if (s.bucket < 0) return kNothing;
        before = s.before;
        lo += (uint32_t)s.bucket << shift;
        hi = min(hi, lo + ((1u << shift) - 1u));
    }
    // The border bucket's tokens, where they are too many for a list
    auto add_bucket = [&] {
        if (final)
            each_near(row, most, [&](float l, uint32_t index) {
                if (row.bucket(l) == bucket && inside(l, index) && within(key_of(l), index, border)) sum += row.weight(l);
            });
        return kBorder;
    };
    if (ranked) return add_bucket();
    // ---- more equal logits than are ranked: the n-th of them by index ----
    unsigned long long nth = s.target - before;
    if (goal.by_weight) {
        const unsigned long long w = Row::whole(row.units(logit_of(lo)));
        nth = (nth + w - 1) / w;  // w > 0: the target lies among these tokens' weights
    }
    uint32_t mine = 0;
    each_near(row, most, [&](float v, uint32_t index) {
        const uint32_t key = key_of(v);
        if (key == lo && candidate(v, key, index)) ++mine;
    });
    mine = __reduce_add_sync(0xffffffffu, mine);  // of the warp, whose tokens are neighbours
    unsigned long long ahead, total;
    block_scan(s, lane == 0 ? mine : 0u, ahead, total);
    ahead = __shfl_sync(0xffffffffu, ahead, 0);
    int h = turn & 1;
    ++turn;
    if (threadIdx.x == 0) {
        s.last_n[h] = (uint32_t)total;
        s.flag = 0xffffffffu;
    }
    cluster_sync();
    for (int q = 0; q < row.rank; ++q) ahead += peer_u32(&s.last_n[h], q);
    if (ahead < nth && nth <= ahead + mine) {  // whole warps
        uint32_t left = (uint32_t)(nth - ahead);
        each_span(row, [&](const float (&l)[4], int index) {
            uint32_t n = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t key = key_of(l[j]);
                n += key == lo && candidate(l[j], key, (uint32_t)(index + j)) ? 1u : 0u;
            }
            uint32_t run = n;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const uint32_t up = __shfl_up_sync(0xffffffffu, run, off);
                if (lane >= off) run += up;
            }
            uint32_t k = run - n;  // in front of this lane's, in the span
            for (int j = 0; j < 4; ++j) {
                const uint32_t key = key_of(l[j]);
                if (key == lo && candidate(l[j], key, (uint32_t)(index + j)) && ++k == left) s.flag = (uint32_t)(index + j);
            }
            const uint32_t in_span = __shfl_sync(0xffffffffu, run, 31);
            left = left > in_span ? left - in_span : 0u;  // 0: found (k starts from 1)
        });
    }
    h = turn & 1;
    ++turn;
    __syncthreads();
    if (threadIdx.x == 0) s.last_n[h] = s.flag;  // the CTA that has it tells the others
    cluster_sync();
    uint32_t index = 0xffffffffu;
    for (int q = 0; q < row.ctas; ++q) index = min(index, peer_u32(&s.last_n[h], q));
    border = {lo, index};
    return add_bucket();
}

__device__ __forceinline__ float clean(float l) { return l == l ? l : -INFINITY; }

// This CTA's logits to shared memory as f32, NaN as -infinity; the largest.  16-byte loads between the first and the last 16-byte
// boundary; `out` is placed so that what they bring is stored in 16 bytes too.
template <class T>
__device__ __forceinline__ float load_logits(const T *in, int count, float *out) {
    constexpr int V = 16 / sizeof(T);
    float top = -INFINITY;
    const int head = min(count, (int)((16 - (reinterpret_cast<uintptr_t>(in) & 15)) & 15) / (int)sizeof(T));
    const int vectors = (count - head) / V, tail = head + vectors * V;
    auto one = [&](int i) {
        float l;
        if constexpr (sizeof(T) == 4) l = __ldg(in + i);
        else if constexpr (std::is_same_v<T, __half>) l = __half2float(__ldg(in + i));
        else l = __bfloat162float(__ldg(in + i));
        l = clean(l);
        out[i] = l;
        top = fmaxf(top, l);
    };
    if ((int)threadIdx.x < head) one(threadIdx.x);
    if (tail + (int)threadIdx.x < count) one(tail + threadIdx.x);
    const uint4 *v4 = reinterpret_cast<const uint4 *>(in + head);
    constexpr int kBatch = 8;  // loads in flight per thread
    for (int i = threadIdx.x; i < vectors; i += kThreads * kBatch) {
        uint4 v[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
            if (i + j * kThreads < vectors) v[j] = __ldg(v4 + i + j * kThreads);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            if (i + j * kThreads >= vectors) break;
            const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
            float l[V];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (sizeof(T) == 4) {
                    l[e] = clean(__uint_as_float(w[e]));
                } else if constexpr (std::is_same_v<T, __half>) {
                    l[2 * e] = clean(f16_bits_to_f32(w[e] & 0xffffu));
                    l[2 * e + 1] = clean(f16_bits_to_f32(w[e] >> 16));
                } else {
                    l[2 * e] = clean(__uint_as_float(w[e] << 16));
                    l[2 * e + 1] = clean(__uint_as_float(w[e] & 0xffff0000u));
                }
            }
            float4 *dst = reinterpret_cast<float4 *>(out + head + (i + j * kThreads) * V);
#pragma unroll
            for (int e = 0; e < V / 4; ++e) dst[e] = make_float4(l[4 * e], l[4 * e + 1], l[4 * e + 2], l[4 * e + 3]);
#pragma unroll
            for (int e = 0; e < V; ++e) top = fmaxf(top, l[e]);
        }
    }
    return top;
}

__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ SampleParams p, int ctas) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    Shared &s = *reinterpret_cast<Shared *>(smem_raw);
    const int64_t b = blockIdx.x / ctas;
    const int lane = threadIdx.x & 31;
    Row row;
    row.ctas = ctas;
    row.rank = blockIdx.x - (int)b * ctas;
    const int first = min(row.rank * p.chunk, p.vocab), count = min(p.chunk, p.vocab - first);
    row.share = p.share;
    int turn = 0;
    bool used = false;
    launch_dependents();
    wait_predecessor();
    // ---- the row, and its largest logit ----
    const int64_t start = b * p.ld + first;
    const uintptr_t address = reinterpret_cast<uintptr_t>(p.logits) + (uintptr_t)start * (p.type == LLOOM_F32 ? 4 : 2);
    const int head = (int)((16 - (address & 15)) & 15) / (p.type == LLOOM_F32 ? 4 : 2);  // logits in front of a 16-byte boundary
    row.part = reinterpret_cast<unsigned long long *>(smem_raw + (sizeof(Shared) + 15) / 16 * 16);
    float *padded = reinterpret_cast<float *>(row.part + kBuckets / ctas);
    const int pad = (4 - head) & 3;
    row.logits = padded;
    row.first = first - pad;
    row.begin = first;
    row.end = first + count;
    if ((int)threadIdx.x < pad) padded[threadIdx.x] = -INFINITY;
    for (int i = pad + count + threadIdx.x; i < kWarps * p.share; i += kThreads) padded[i] = -INFINITY;
    float top = p.type == LLOOM_F32   ? load_logits(reinterpret_cast<const float *>(p.logits) + start, count, padded + pad)
                : p.type == LLOOM_F16 ? load_logits(reinterpret_cast<const __half *>(p.logits) + start, count, padded + pad)
                                      : load_logits(reinterpret_cast<const __nv_bfloat16 *>(p.logits) + start, count, padded + pad);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    if (lane == 0) s.low[threadIdx.x >> 5] = __float_as_uint(top);
    __syncthreads();
    for (int i = 0; i < kWarps; ++i) top = fmaxf(top, __uint_as_float(s.low[i]));
    if (threadIdx.x == 0) s.max = top;
    cluster_sync();
    for (int q = 0; q < ctas; ++q) top = fmaxf(top, __uint_as_float(peer_u32(&s.max, q)));
    if (top == INFINITY) {  // these alone count, and all the same
        for (int i = threadIdx.x; i < kWarps * p.share; i += kThreads) padded[i] = padded[i] == INFINITY ? 0.0f : -INFINITY;
        top = 0.0f;
        __syncthreads();
    }
    row.max = top;
    // ---- settings ----
    const double temperature = p.temperature ? (double)p.temperature[b] : p.temperature_all;
    const bool greedy = !(temperature >= kLeastTemperature);
    const double inv_t = greedy ? 0.0 : 1.0 / temperature;
    const double per_logit = inv_t * 1.4426950408889634074;  // 1 / ln 2 / T
    row.wide_max = Row::widen(top);
    row.slope = per_logit * 5.2829453113566525e+269;  // 2^896
    row.bucket_scale = (float)(inv_t * 64.0);
    const int top_k = p.top_k ? p.top_k[b] : p.top_k_all;
    const double top_p = p.top_p ? (double)p.top_p[b] : p.top_p_all, min_p = p.min_p ? (double)p.min_p[b] : p.min_p_all;
    row.least = min_p > 0.0 ? min_p * kUnit : 0.0;
    const double u = (double)p.u[b];
    const bool by_k = !greedy && top_k > 0 && top_k < p.vocab, by_p = !greedy && top_p < 1.0;
    Border limit = {0xffffffffu, 0xffffffffu};
    bool limited = false, summed = false;
    uint32_t listed = 0;
    unsigned long long mine = 0;  // the lane's part of its warp's kept weights
    Selected got = kNothing;
    if (top > -INFINITY && by_k) {
        if (threadIdx.x == 0) s.target = (unsigned long long)top_k;  // behind the barriers of clear_histogram for the others
        Border at;
        got = find_border<false>(s, row, Goal{false, 0.0}, limit, !by_p, turn, used, at, listed, mine);
        if (got == kBorder) {
            limit = at;
            limited = true;
            summed = !by_p;
        }
    }
    const bool listed_by_k = got == kListed;
    if (top > -INFINITY && by_p && !listed_by_k) {
        const Goal goal{true, top_p};
        Border at;
        got = limited ? find_border<true>(s, row, goal, limit, true, turn, used, at, listed, mine)
                      : find_border<false>(s, row, goal, limit, true, turn, used, at, listed, mine);
        if (got == kBorder) {
            limit = at;
            limited = true;
            summed = true;
        }
    }
    auto pick = [&](unsigned long long all) { return greedy || !(u > 0.0) ? 0ull : u < 1.0 ? part_of(u, all, false) : all - 1; };
    auto write = [&](uint32_t index, double units, unsigned long long all) {
        p.ids[b] = (int64_t)index;
        if (p.probs) p.probs[b] = greedy ? 1.0f : (float)(units / (double)all);
    };
    if (got == kListed) {
        // ---- the draw from the list: its first CTA does it ----
        if (row.rank == 0) {
            unsigned long long from;
            const uint32_t rank = rank_in_list(s, listed, from);
            const bool has = threadIdx.x < listed;
            uint2 me = make_uint2(0u, 0u);
            if (has) {
                me = s.list[threadIdx.x].token;
                if (listed_by_k && rank + 1 == (uint32_t)top_k) s.total = from + s.list[threadIdx.x].weight;
            }
            __syncthreads();
            if (listed_by_k && threadIdx.x == 0) {
                const unsigned long long t = !by_p ? s.total : top_p > 0.0 ? part_of(top_p, s.total, true) : 0ull;
                s.target = t > 0 ? t : 1ull;
            }
            __syncthreads();
            // kept: fewer than K in front, and less weight in front than the target
            if (has) {
                const unsigned long long w = s.list[threadIdx.x].weight;
                const float l = logit_of(me.y);
                const bool keep = (!listed_by_k || rank < (uint32_t)top_k) && from < s.target && (row.units(l) >= row.least || l == row.max);
                s.low[threadIdx.x] = (uint32_t)(keep ? w : 0ull);  // (the histogram has been read)
                s.high[threadIdx.x] = (uint32_t)((keep ? w : 0ull) >> 32);
            }
            __syncthreads();
            if (has) {
                auto kept = [&](uint32_t i) { return (unsigned long long)s.low[i] | ((unsigned long long)s.high[i] << 32); };
                unsigned long long ahead = 0, all = 0;
#pragma unroll 4
                for (uint32_t i = 0; i < listed; ++i) {
                    const unsigned long long w = kept(i);
                    all += w;
                    ahead += s.list[i].token.x < me.x ? w : 0ull;
                }
                const unsigned long long t = pick(all);
                if (ahead <= t && t < ahead + kept(threadIdx.x)) write(me.x, row.units(logit_of(me.y)), all);
            }
        }
        cluster_sync();  // the others' lists are read no more
        return;
    }
    // ---- the draw from all of the row ----
    auto weight = [&](float l, uint32_t index) -> unsigned long long {
        if (greedy) return l == row.max ? 1ull : 0ull;
        const unsigned long long w = row.weight(l);
        return !limited || within(key_of(l), index, limit) ? w : 0ull;
    };
    unsigned long long ahead, total;
    if (top > -INFINITY && !summed) {
        if (greedy) {
            each_near(row, 0.0f, [&](float l, uint32_t) { mine += l == row.max ? 1ull : 0ull; });
        } else if (limited) {
            mine = 0;
            auto add = [&](const float (&l)[4], const uint32_t (&)[4], const bool (&there)[4]) {
#pragma unroll
                for (int j = 0; j < 4; ++j) mine += there[j] ? row.weight(l[j]) : 0ull;
            };
            Gather kept(s);
            each_span(row, [&](const float (&l)[4], int index) {
                bool take[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) take[j] = within(key_of(l[j]), (uint32_t)(index + j), limit);
                kept.add(row, l, index, take, add);
            });
            kept.finish(row, add);
        } else {
            mine = 0;
            each_span(row, [&](const float (&l)[4], int) {
                unsigned long long w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = row.weight(l[j]);
                mine += w[0] + w[1] + w[2] + w[3];
            });
        }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, off);
    block_scan(s, lane == 0 ? mine : 0ull, ahead, total);
    ahead = __shfl_sync(0xffffffffu, ahead, 0);
    const int h = turn & 1;
    if (threadIdx.x == 0) s.sum[h] = total;
    cluster_sync();
    unsigned long long all = 0;
    for (int q = 0; q < ctas; ++q) {
        const unsigned long long t = peer_u64(&s.sum[h], q);
        if (q < row.rank) ahead += t;
        all += t;
    }
    __syncthreads();
    cluster_arrive();  // this CTA reads the others' memory no more
    if (all == 0) {  // nothing above -inf
        if (row.rank == 0 && threadIdx.x == 0) {
            p.ids[b] = -1;
            if (p.probs) p.probs[b] = 0.0f;
        }
    } else {
        const unsigned long long t = pick(all);
        // One warp of the cluster has the token among its own: its CTA looks through these again, four per thread.
        if (threadIdx.x == 0) s.flag = kWarps;
        __syncthreads();
        if (lane == 0 && ahead <= t && t < ahead + mine) {
            s.flag = threadIdx.x >> 5;
            s.before = ahead;
        }
        __syncthreads();
        const int found = (int)s.flag;
        if (found < kWarps) {
            unsigned long long sum = s.before;
            for (int i0 = 0; i0 < row.share; i0 += 4 * kThreads) {
                const int i = i0 + 4 * threadIdx.x, at = found * row.share + i;
                unsigned long long own[4] = {}, run = 0, in_front, part;
                float l[4];
                if (i < row.share) {
                    const float4 v = *reinterpret_cast<const float4 *>(row.logits + at);
                    l[0] = v.x;
                    l[1] = v.y;
                    l[2] = v.z;
                    l[3] = v.w;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        own[j] = weight(l[j], (uint32_t)(row.first + at + j));
                        run += own[j];
                    }
                }
                block_scan(s, run, in_front, part);
                in_front += sum;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (own[j] && in_front <= t && t < in_front + own[j])
                        write((uint32_t)(row.first + at + j), greedy ? 1.0 : row.units(l[j]), all);
                    in_front += own[j];
                }
                sum += part;
            }
        }
    }
    cluster_wait();  // nor they this one's
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
    // CTAs to a row: up to eight with more than 2048 logits each; half as many while there are more CTAs than SMs and a part of the row twice as
    // long still leaves room for another CTA on the SM: half of a CTA's work does not depend on how many logits it has.  us by 8 / 4 / 2 / 1 CTAs:
    // 7 x 50257 31 / 35 / 46; 19 x 128256 40 / 46; 19 x 32000 31 / 26 / 31 / 42; 30 x 50257 35 / 31 / 37; 37 x 50257 54 / 40 / 37; 64 x 32000 55 / 36 / 34 / 42; 64 x 128256 85 / 79 (alike rows; others level);
    // 300 x 8000 179 / 87 / 52 / 42; 1000 x 32000 673 / 353 / 232 / 239.
    auto share = [&](int ctas) { return (((vocab + ctas - 1) / ctas + 3 + kWarps - 1) / kWarps + kSpan - 1) / kSpan * kSpan; };
    auto bytes = [&](int ctas) { return (int64_t)((sizeof(Shared) + 15) / 16 * 16) + kBuckets / ctas * 8 + kWarps * share(ctas) * 4; };
    int ctas = 1;
    while (ctas < kMaxCluster && vocab > (int64_t)ctas * 4096) ctas *= 2;
    while (ctas > 1 && batch * ctas > di.sm_count && 2 * (bytes(ctas / 2) + di.smem_reserved) <= di.smem_per_sm) ctas /= 2;
    p.chunk = (int)((vocab + ctas - 1) / ctas);
    p.share = (int)share(ctas);
    const int smem = (int)bytes(ctas);
    static SmemOnce once;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || dev < 0 || dev >= 64) return LLOOM_ERR_DEVICE;
    {
        static_assert(sizeof(Shared) + 16 + kBuckets / kMaxCluster * 8 + (kMaxChunk + 3 + kWarps * kSpan) * 4 <= 227 * 1024, "shared memory");
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
