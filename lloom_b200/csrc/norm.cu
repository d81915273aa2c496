// RMS norm of a hidden state with the residual's addition in front and, behind it, the 8-bit activation blocks that the
// products read:
//
//   h = T(x + r)                                  the residual stream, rounded to its element type T
//   inv = f32(1 / sqrt(sum(h * h) / k + eps))     the sum and everything up to inv in 64 bits
//   y = f32(f32(h * inv) * w)                     stored as T, or as Q8_0 / Q8_K blocks of these f32 values
//
// Squares of f32 values are exact in 64 bits and their sum is off by 1e-16.  How a row is split over threads (which depends on the batch and on
// alignment) changes the last bits of the sum in one row of three, and inv, and with it codes of the 8-bit blocks, only where 1 / sqrt lies within a few
// units of 2^-53 of the middle between two f32 values: about one row in 10^8.
//
// Bound by memory (x and r read once, h and y written once: the row stays in registers between the sum and the output) or,
// for a few rows, by the latency of one launch, two loads and a reduction over the row.
#include "abi.h"
#include "common.cuh"
#include "forward.h"
#include "gemv_params.h"
#include "quantize_act.cuh"

namespace lloom {

namespace {

struct NormParams {
    const void *x, *r, *w;  // r may be null
    void *h, *y;            // h: null exactly when r is
    int w_type, y_type;     // y_type: x's own, LLOOM_Q8_0 or LLOOM_Q8_K
    int lanes;              // threads on a row where they are fewer than a warp's, else 0: the CTA's threads
    int64_t m, ldx, ldr;
    int k;
    double per_k, eps;  // per_k: 1 / k
};

__device__ __forceinline__ float load_one(const void *p, int type, int64_t i) {
    if (type == LLOOM_F32) return __ldg(reinterpret_cast<const float *>(p) + i);
    if (type == LLOOM_F16) return __half2float(__ldg(reinterpret_cast<const __half *>(p) + i));
    return __bfloat162float(__ldg(reinterpret_cast<const __nv_bfloat16 *>(p) + i));
}
// How the pieces of a row lie
enum Pieces {
    kAnywhere,  // element by element
    kEdges,     // on 16-byte boundaries, the first and the last one partly outside of the row
    kWhole      // on 16-byte boundaries, all of them inside
};
__device__ __forceinline__ uint32_t pack_halves(int type, float a, float b) {
    if (type == LLOOM_F16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Elements e .. e + 7 of a row, as they lie in memory: halves in four registers, so that more rows are in flight
template <int TYPE>
struct Piece {
    static constexpr int kWords = TYPE == LLOOM_F32 ? 8 : 4;
    uint32_t w[kWords];
    __device__ __forceinline__ void put(const float (&v)[8]) {
        if constexpr (TYPE == LLOOM_F32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = pack_halves(TYPE, v[2 * i], v[2 * i + 1]);
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        if constexpr (TYPE == LLOOM_F32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = TYPE == LLOOM_F16 ? f16_bits_to_f32(w[i] & 0xffffu) : __uint_as_float(w[i] << 16);
                v[2 * i + 1] = TYPE == LLOOM_F16 ? f16_bits_to_f32(w[i] >> 16) : __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0u;
    }
    // from and to the row that starts at element `row` of p; zeros outside of 0 .. k - 1
    template <int PIECES>
    __device__ __forceinline__ void load(const void *p, int64_t row, int e, int k) {
        if (PIECES == kWhole || (PIECES == kEdges && e >= 0 && e + 8 <= k)) {
            const uint4 *q = reinterpret_cast<const uint4 *>(reinterpret_cast<const uint8_t *>(p) + (row + e) * (kWords / 2));
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i) {
                const uint4 t = __ldg(q + i);
                w[4 * i] = t.x;
                w[4 * i + 1] = t.y;
                w[4 * i + 2] = t.z;
                w[4 * i + 3] = t.w;
            }
        } else {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = e + i >= 0 && e + i < k ? load_one(p, TYPE, row + e + i) : 0.0f;
            put(v);
        }
    }
    template <int PIECES>
    __device__ __forceinline__ void store(void *p, int64_t row, int e, int k) const {
        if (PIECES == kWhole || (PIECES == kEdges && e >= 0 && e + 8 <= k)) {
            uint4 *q = reinterpret_cast<uint4 *>(reinterpret_cast<uint8_t *>(p) + (row + e) * (kWords / 2));
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i) q[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        } else {
            float v[8];
            get(v);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (e + i >= 0 && e + i < k) store_y(p, TYPE, row + e + i, v[i]);
        }
    }
};

template <int X_TYPE>
__device__ __forceinline__ float round_to(float v) {
    if (X_TYPE == LLOOM_F16) return __half2float(__float2half_rn(v));
    if (X_TYPE == LLOOM_BF16) return __bfloat162float(__float2bfloat16_rn(v));
    return v;
}

// x becomes h = x + r, which is stored, where there is a residual; its squares are added
template <int X_TYPE, int PIECES>
__device__ __forceinline__ void stream_piece(const NormParams &p, int64_t row, int e, bool live, Piece<X_TYPE> &x, const Piece<X_TYPE> &r, double (&sum)[2]) {
    float v[8];
    x.get(v);
    if (p.r && live) {
        float u[8];
        r.get(u);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = round_to<X_TYPE>(__fadd_rn(v[i], u[i]));
        x.put(v);
        x.template store<PIECES>(p.h, row * p.k, e, p.k);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i & 1] = fma((double)v[i], (double)v[i], sum[i & 1]);
}

// 1 / sqrt(a), rounded to f32: Newton's iteration in 64 bits from the 32-bit approximation (2^-21, then below 2^-41, then 2^-53) where that one
// is in range.  A row waits for this between its loads and its output, and the square root and the division take three times as long.
__device__ __forceinline__ float inverse_root(double a) {
    if (!(a > 1e-30 && a < 1e30)) return (float)(1.0 / sqrt(a));
    double y = (double)rsqrtf((float)a);
    const double half = 0.5 * a;
    y = y * fma(-half * y, y, 1.5);
    y = y * fma(-half * y, y, 1.5);
    return (float)y;
}

// An octet of weights, which lie like the row only where that starts on a boundary
template <int PIECES>
__device__ __forceinline__ void weight_octet(const NormParams &p, int e, float (&w)[8]) {
    if (PIECES == kWhole) {
        load8(p.w, p.w_type, e, w);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = e + i >= 0 && e + i < p.k ? load_one(p.w, p.w_type, e + i) : 0.0f;
    }
}

// y of an octet from h and w; all lanes of a warp, `live` says whose octet lies in a row
template <int X_TYPE, int PIECES>
__device__ __forceinline__ void output_octet(const NormParams &p, int64_t row, int e, bool live, float inv, float (&v)[8]) {
    float w[8];
    if (live) weight_octet<PIECES>(p, e, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = live ? __fmul_rn(__fmul_rn(v[i], inv), w[i]) : 0.0f;
    if (p.y_type == LLOOM_Q8_K) {  // a warp has a 256-element block
        uint32_t lo, hi;
        float d;
        int sum16;
        const int lane = threadIdx.x & 31;
        q8k_quantize_warp(v, lane, lo, hi, d, sum16);
        if (!live) return;
        uint8_t *dst = reinterpret_cast<uint8_t *>(p.y) + (row * (p.k / QK_K) + e / QK_K) * Q8K_BYTES;
        uint32_t *q = reinterpret_cast<uint32_t *>(dst + 4 + lane * 8);
        q[0] = lo;
        q[1] = hi;
        if ((lane & 1) == 0) reinterpret_cast<short *>(dst + 4 + QK_K)[lane >> 1] = (short)sum16;
        if (lane == 0) *reinterpret_cast<float *>(dst) = d;
    } else if (p.y_type == LLOOM_Q8_0) {  // four lanes have a 32-element block
        uint32_t lo, hi;
        unsigned short d16;
        q8_0_quantize_quad(v, lo, hi, d16);
        if (!live) return;
        uint8_t *dst = reinterpret_cast<uint8_t *>(p.y) + (row * (p.k / QK8_0) + e / QK8_0) * Q8_0_BYTES;
        const int part = (e / 8) & 3;
        if (part == 0) *reinterpret_cast<unsigned short *>(dst) = d16;
        unsigned short *q = reinterpret_cast<unsigned short *>(dst + 2 + part * 8);
        q[0] = (unsigned short)(lo & 0xffffu);
        q[1] = (unsigned short)(lo >> 16);
        q[2] = (unsigned short)(hi & 0xffffu);
        q[3] = (unsigned short)(hi >> 16);
    } else if (live) {
        Piece<X_TYPE> y;
        y.put(v);
        y.template store<PIECES>(p.y, row * p.k, e, p.k);
    }
}

// OCTETS: eight-element pieces a thread keeps in registers; 0: any number, read again from h (or x) for the output.
// PIECES: kEdges where the rows of x, r, h and y lie alike modulo 16 bytes, kWhole where they start there, k is a multiple of eight and the weights
// start there too.
template <int X_TYPE, int OCTETS, int PIECES>
__global__ void __launch_bounds__(OCTETS == 2 && X_TYPE != LLOOM_F32 ? 512 : 1024, OCTETS == 1 ? 2 : OCTETS == 2 && X_TYPE != LLOOM_F32 ? 3 : 1) rms_norm_kernel(const __grid_constant__ NormParams p) {
    __shared__ double part[32];
    launch_dependents();
    wait_predecessor();  // everything read or written here may be the predecessor's
    const int lanes = p.lanes ? p.lanes : (int)blockDim.x, t = p.lanes ? (int)threadIdx.x % p.lanes : (int)threadIdx.x;
    const int64_t row = p.lanes ? (int64_t)blockIdx.x * (blockDim.x / p.lanes) + threadIdx.x / p.lanes : (int64_t)blockIdx.x;
    const bool has_row = row < p.m;
    // elements in front of the row that its first piece would reach into
    constexpr int size = X_TYPE == LLOOM_F32 ? 4 : 2;
    const int pad = PIECES == kEdges ? (int)((reinterpret_cast<uintptr_t>(p.x) + (uintptr_t)(row * p.ldx) * size) & 15) / size : 0;
    const int e0 = t * 8 - pad, step = lanes * 8;
    constexpr int N = OCTETS > 0 ? OCTETS : 1;
    Piece<X_TYPE> h[N];
    double sums[2] = {0.0, 0.0};
    if constexpr (OCTETS > 0) {
        Piece<X_TYPE> r[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = e0 + i * step;
            if (has_row && e < p.k) {
                h[i].template load<PIECES>(p.x, row * p.ldx, e, p.k);
                if (p.r) r[i].template load<PIECES>(p.r, row * p.ldr, e, p.k);
            } else {
                h[i].zero();
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) stream_piece<X_TYPE, PIECES>(p, row, e0 + i * step, has_row && e0 + i * step < p.k, h[i], r[i], sums);
    } else {
        for (int e = e0; e < p.k; e += step) {
            Piece<X_TYPE> r;
            h[0].template load<PIECES>(p.x, row * p.ldx, e, p.k);
            if (p.r) r.template load<PIECES>(p.r, row * p.ldr, e, p.k);
            stream_piece<X_TYPE, PIECES>(p, row, e, true, h[0], r, sums);
        }
    }
    double sum = sums[0] + sums[1];
    for (int off = (lanes < 32 ? lanes : 32) / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (lanes > 32) {
        const int warps = blockDim.x >> 5;
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
        __syncthreads();
        double all[4] = {0.0, 0.0, 0.0, 0.0};
        for (int i = 0; i < warps; i += 4)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j < warps) all[j] += part[i + j];
        sum = (all[0] + all[1]) + (all[2] + all[3]);
    }
    const float inv = inverse_root(sum * p.per_k + p.eps);
    const int warp_e = e0 - (lanes < 32 ? t : t & 31) * 8;  // of the warp's first lane on the row
    if constexpr (OCTETS > 0) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (warp_e + i * step < p.k) {
                float v[8];
                h[i].get(v);
                output_octet<X_TYPE, PIECES>(p, row, e0 + i * step, has_row && e0 + i * step < p.k, inv, v);
            }
    } else {
        for (int e = e0, we = warp_e; we < p.k; e += step, we += step) {
            const bool live = e < p.k;
            float v[8];
            if (live) {
                // plain loads: h was written by this thread a moment ago
                const void *src = p.r ? p.h : p.x;
                const int64_t base = row * (p.r ? (int64_t)p.k : p.ldx) + e;
                for (int i = 0; i < 8; ++i) {
                    if (e + i < 0 || e + i >= p.k) v[i] = 0.0f;
                    else if (X_TYPE == LLOOM_F32) v[i] = reinterpret_cast<const volatile float *>(src)[base + i];
                    else {
                        const unsigned short b = reinterpret_cast<const volatile unsigned short *>(src)[base + i];
                        v[i] = X_TYPE == LLOOM_F16 ? f16_bits_to_f32(b) : __uint_as_float((uint32_t)b << 16);
                    }
                }
            }
            output_octet<X_TYPE, PIECES>(p, row, e, live, inv, v);
        }
    }
}

using NormKernel = void (*)(NormParams);
template <int X_TYPE, int PIECES>
NormKernel norm_kernel(int octets) {
    switch (octets) {
    case 1: return rms_norm_kernel<X_TYPE, 1, PIECES>;
    case 2: return rms_norm_kernel<X_TYPE, 2, PIECES>;
    case 4: return rms_norm_kernel<X_TYPE, 4, PIECES>;
    }
    return rms_norm_kernel<X_TYPE, 0, PIECES>;
}
template <int X_TYPE>
NormKernel norm_kernel(int octets, int pieces) {
    return pieces == kWhole ? norm_kernel<X_TYPE, kWhole>(octets) : pieces == kEdges ? norm_kernel<X_TYPE, kEdges>(octets) : norm_kernel<X_TYPE, kAnywhere>(octets);
}

// Activation blocks back to the values they stand for, eight elements per thread
__global__ void __launch_bounds__(256) dequantize_act_kernel(int dtype, const uint8_t *__restrict__ blocks, int64_t elems, float *__restrict__ out) {
    launch_dependents();
    wait_predecessor();
    const int64_t e = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * 8;
    if (e >= elems) return;
    const bool q8k = dtype == LLOOM_Q8_K;
    const uint8_t *blk = blocks + (q8k ? e / QK_K * Q8K_BYTES : e / QK8_0 * Q8_0_BYTES);
    const float d = q8k ? *reinterpret_cast<const float *>(blk) : f16_bits_to_f32(*reinterpret_cast<const unsigned short *>(blk));
    const unsigned short *q = reinterpret_cast<const unsigned short *>(blk + (q8k ? 4 + (e & (QK_K - 1)) : 2 + (e & (QK8_0 - 1))));
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = q[i];
        v[2 * i] = __fmul_rn((float)(int8_t)(w & 0xff), d);
        v[2 * i + 1] = __fmul_rn((float)(int8_t)(w >> 8), d);
    }
    reinterpret_cast<float4 *>(out + e)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4 *>(out + e)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

}  // namespace

int rms_norm(const void *x, const void *residual, const void *weight, int x_type, int w_type, double eps, int64_t m, int64_t k, int64_t ldx,
             int64_t ldr, void *h, void *y, int y_type, void *stream, bool overlap) {
    const bool blocks = y_type == LLOOM_Q8_0 || y_type == LLOOM_Q8_K;
    if (!elem_type_ok(x_type) || !elem_type_ok(w_type) || (!blocks && y_type != x_type)) return LLOOM_ERR_DTYPE;
    if (m <= 0 || k <= 0 || m > 0x7fffffff || k > (1 << 24) || ldx < k || (residual && (ldr < k || (h == residual && ldr != k)))) return LLOOM_ERR_SHAPE;
    if (blocks && k % lloom_b200_block_elems(y_type) != 0) return LLOOM_ERR_SHAPE;
    if (!x || !weight || !y || (residual && !h)) return LLOOM_ERR_NULL;
    const int64_t es = elem_bytes(x_type), ws = elem_bytes(w_type);
    if (!aligned(x, es) || !aligned(weight, ws) || !aligned(y, blocks ? 4 : es) || (residual && (!aligned(residual, es) || !aligned(h, es))))
        return LLOOM_ERR_ALIGN;
    NormParams p = {};
    p.x = x;
    p.r = residual;
    p.w = weight;
    p.h = h;
    p.y = y;
    p.w_type = w_type;
    p.y_type = y_type;
    p.m = m;
    p.k = (int)k;
    p.ldx = ldx;
    p.ldr = ldr;
    p.per_k = 1.0 / (double)k;
    p.eps = eps;
    // rows alike modulo 16 bytes: one start, and one distance between rows (or distances that are multiples of 16 bytes)
    auto phase = [](const void *q) { return (uintptr_t)q & 15; };
    const bool steps = (ldx - k) * es % 16 == 0 && (!residual || (ldr - k) * es % 16 == 0);
    const bool wide = blocks ? phase(x) == 0 && ldx * es % 16 == 0 && (!residual || (phase(residual) == 0 && phase(h) == 0 && ldr * es % 16 == 0))
                             : steps && phase(y) == phase(x) && (!residual || (phase(residual) == phase(x) && phase(h) == phase(x)));
    // Threads: a piece each and a row per CTA, so that a row alone waits for memory once.  Many rows of halves: two pieces each, in 40 registers, so
    // that six rows of 4096 are in flight on an SM instead of four.  us of a call in a captured chain with changing inputs, two pieces / one, bf16 with a
    // residual: 2048 x 4096 13.0 / 16.0, 1024 x 4096 8.3 / 9.4, 592 x 4096 6.7 / 6.1, 2048 x 2048 7.9 / 8.5, 2048 x 8192 24.5 / 37.9.  (With
    // f32 four rows in flight are enough: 22.7 us are 5.9 TB/s.)  Rows of up to 32 pieces share a CTA of 256 threads.
    const int pieces = !wide ? kAnywhere : phase(x) == 0 && phase(weight) == 0 && k % 8 == 0 && ldx * es % 16 == 0 ? kWhole : kEdges;
    const int64_t octets = (k + 7) / 8 + (pieces == kEdges ? 1 : 0);
    const bool pairs = x_type != LLOOM_F32 && m >= 592 && octets > 64 && octets <= 1024;
    const int per = pairs ? 2 : octets <= 1024 ? 1 : octets <= (x_type == LLOOM_F32 ? 2048 : 1024) ? 2 : octets <= 4096 ? 4 : 0;
    const int64_t threads = per ? (octets + per - 1) / per : 1024;
    p.lanes = threads > 32 ? 0 : threads <= 8 ? 8 : threads <= 16 ? 16 : 32;
    const unsigned block = p.lanes ? 256 : (unsigned)((threads + 31) / 32 * 32);
    const unsigned grid = p.lanes ? (unsigned)ceil_div64(m, 256 / p.lanes) : (unsigned)m;
    auto kern = x_type == LLOOM_F32 ? norm_kernel<LLOOM_F32>(per, pieces) : x_type == LLOOM_F16 ? norm_kernel<LLOOM_F16>(per, pieces) : norm_kernel<LLOOM_BF16>(per, pieces);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap ? 1 : 0;
    return launch_status(cudaLaunchKernelEx(&cfg, kern, p));
}

int dequantize_act(int act_dtype, const void *act_blocks, int64_t elem_count, float *out, void *stream, bool overlap) {
    if (act_dtype != LLOOM_Q8_0 && act_dtype != LLOOM_Q8_K) return LLOOM_ERR_DTYPE;
    if (elem_count <= 0 || elem_count % lloom_b200_block_elems(act_dtype) != 0 || elem_count / 8 / 256 >= 0x7fffffff) return LLOOM_ERR_SHAPE;
    if (!act_blocks || !out) return LLOOM_ERR_NULL;
    if (!aligned(act_blocks, 4) || !aligned(out, 16)) return LLOOM_ERR_ALIGN;
    return launch_status(launch_early(dequantize_act_kernel, (unsigned)ceil_div64(elem_count / 8, 256), 256, 0, overlap, (cudaStream_t)stream,
                                      act_dtype, (const uint8_t *)act_blocks, elem_count, out));
}

}  // namespace lloom

using namespace lloom;

extern "C" {

int lloom_b200_rms_norm(const void *x, const void *residual, const void *weight, int x_type, int w_type, double eps, int64_t m, int64_t k,
                        int64_t ldx, int64_t ldr, void *h, void *y, int y_type, void *stream) {
    return rms_norm(x, residual, weight, x_type, w_type, eps, m, k, ldx, ldr, h, y, y_type, stream, launch_overlap() > 0);
}

int lloom_b200_dequantize_act(int act_dtype, const void *act_blocks, int64_t elem_count, float *out, void *stream) {
    return dequantize_act(act_dtype, act_blocks, elem_count, out, stream, launch_overlap() > 0);
}

}  // extern "C"
