// RMS norm of a hidden state with the residual's addition in front and, behind it, the 8-bit activation blocks that the
// products read:
//
//   h = T(x + r)                                  the residual stream, rounded to its element type T
//   inv = f32(1 / sqrt(sum(h * h) / k + eps))     the sum and everything up to inv in 64 bits
//   y = f32(f32(h * inv) * w)                     stored as T, or as Q8_0 / Q8_K blocks of these f32 values
//
// Squares of f32 values are exact in 64 bits and their sum is off by 1e-16, so that inv, and with it every code of the 8-bit
// blocks, is a function of the inputs and not of how the row was split over threads.
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
    int x_type, w_type, y_type;  // y_type: x_type's own, LLOOM_Q8_0 or LLOOM_Q8_K
    int vec;                // rows and weights start on 16 bytes and k is a multiple of 8
    int64_t m, ldx, ldr;
    int k;
    double eps;
};

// elements e .. e + 7 of a row, zeros past its end
__device__ __forceinline__ void load_octet(const void *p, int type, int64_t row, int e, int k, int vec, float (&v)[8]) {
    if (vec) {
        load8(p, type, row + e, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = 0.0f;
        if (e + i >= k) continue;
        const int64_t at = row + e + i;
        if (type == LLOOM_F32) v[i] = __ldg(reinterpret_cast<const float *>(p) + at);
        else if (type == LLOOM_F16) v[i] = __half2float(__ldg(reinterpret_cast<const __half *>(p) + at));
        else v[i] = __bfloat162float(__ldg(reinterpret_cast<const __nv_bfloat16 *>(p) + at));
    }
}

__device__ __forceinline__ uint32_t pack_halves(int type, float a, float b) {
    if (type == LLOOM_F16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ void store_octet(void *p, int type, int64_t row, int e, int k, int vec, const float (&v)[8]) {
    if (!vec) {
        for (int i = 0; i < 8 && e + i < k; ++i) store_y(p, type, row + e + i, v[i]);
    } else if (type == LLOOM_F32) {
        float4 *q = reinterpret_cast<float4 *>(reinterpret_cast<float *>(p) + row + e);
        q[0] = make_float4(v[0], v[1], v[2], v[3]);
        q[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *reinterpret_cast<uint4 *>(reinterpret_cast<unsigned short *>(p) + row + e) =
            make_uint4(pack_halves(type, v[0], v[1]), pack_halves(type, v[2], v[3]), pack_halves(type, v[4], v[5]), pack_halves(type, v[6], v[7]));
    }
}

__device__ __forceinline__ float round_to(int type, float v) {
    if (type == LLOOM_F16) return __half2float(__float2half_rn(v));
    if (type == LLOOM_BF16) return __bfloat162float(__float2bfloat16_rn(v));
    return v;
}

// The stream's elements h of an octet; stored if there is a residual
__device__ __forceinline__ void stream_octet(const NormParams &p, int64_t row, int e, float (&v)[8]) {
    load_octet(p.x, p.x_type, row * p.ldx, e, p.k, p.vec, v);
    if (!p.r) return;
    float r[8];
    load_octet(p.r, p.x_type, row * p.ldr, e, p.k, p.vec, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = round_to(p.x_type, __fadd_rn(v[i], r[i]));
    store_octet(p.h, p.x_type, row * p.k, e, p.k, p.vec, v);
}

__device__ __forceinline__ void square_sum(const float (&v)[8], double &sum) {
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fma((double)v[i], (double)v[i], sum);
}

// y of an octet from h; all lanes of a warp, `live` says whose octet lies in the row
__device__ __forceinline__ void output_octet(const NormParams &p, int64_t row, int e, bool live, float inv, float (&v)[8]) {
    float w[8];
    if (live) load_octet(p.w, p.w_type, 0, e, p.k, p.vec, w);
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
        store_octet(p.y, p.y_type, row * p.k, e, p.k, p.vec, v);
    }
}

// blockDim.x threads on a row (whole warps; blockDim.y rows per CTA, more than one only where a warp has a row to itself).
// OCTETS: eight-element pieces a thread keeps in registers; 0: any number, read again from h (or x) for the output.
template <int OCTETS>
__global__ void __launch_bounds__(1024) rms_norm_kernel(const __grid_constant__ NormParams p) {
    __shared__ double part[32];
    launch_dependents();
    wait_predecessor();  // everything read or written here may be the predecessor's
    const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (row >= p.m) return;  // whole warps, and only where no one waits for them
    const int warp_e = (threadIdx.x & ~31) * 8, e0 = threadIdx.x * 8, step = blockDim.x * 8;
    constexpr int N = OCTETS > 0 ? OCTETS : 1;
    float v[N][8];
    double sum = 0.0;
    if constexpr (OCTETS > 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = e0 + i * step;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
            if (e < p.k) stream_octet(p, row, e, v[i]);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) square_sum(v[i], sum);
    } else {
        for (int e = e0; e < p.k; e += step) {
            stream_octet(p, row, e, v[0]);
            square_sum(v[0], sum);
        }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (blockDim.x > 32) {
        const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0) part[threadIdx.x >> 5] = sum;
        __syncthreads();
        sum = lane < warps ? part[lane] : 0.0;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    }
    const float inv = (float)(1.0 / sqrt(sum / (double)p.k + p.eps));
    if constexpr (OCTETS > 0) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (warp_e + i * step < p.k) output_octet(p, row, e0 + i * step, e0 + i * step < p.k, inv, v[i]);
    } else {
        for (int e = e0, we = warp_e; we < p.k; e += step, we += step) {
            const bool live = e < p.k;
            if (live) {
                // plain loads: h was written by this thread a moment ago
                const void *src = p.r ? p.h : p.x;
                const int64_t base = row * (p.r ? (int64_t)p.k : p.ldx) + e;
                for (int i = 0; i < 8; ++i) {
                    if (e + i >= p.k) v[0][i] = 0.0f;
                    else if (p.x_type == LLOOM_F32) v[0][i] = reinterpret_cast<const volatile float *>(src)[base + i];
                    else {
                        const unsigned short b = reinterpret_cast<const volatile unsigned short *>(src)[base + i];
                        v[0][i] = p.x_type == LLOOM_F16 ? f16_bits_to_f32(b) : __uint_as_float((uint32_t)b << 16);
                    }
                }
            }
            output_octet(p, row, e, live, inv, v[0]);
        }
    }
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
    if (m <= 0 || k <= 0 || m > 0x7fffffff || k > (1 << 24) || ldx < k || (residual && ldr < k)) return LLOOM_ERR_SHAPE;
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
    p.x_type = x_type;
    p.w_type = w_type;
    p.y_type = y_type;
    p.m = m;
    p.k = (int)k;
    p.ldx = ldx;
    p.ldr = ldr;
    p.eps = eps;
    p.vec = k % 8 == 0 && aligned(x, 16) && ldx * es % 16 == 0 && aligned(weight, 16) && (blocks || aligned(y, 16)) &&
            (!residual || (aligned(residual, 16) && ldr * es % 16 == 0 && aligned(h, 16)));
    // One octet per thread and a row per CTA; rows of up to 256 elements get a warp, eight of them in a CTA.
    const int64_t octets = (k + 7) / 8;
    int threads = 32, rows = 8;
    if (octets > 32) {
        rows = 1;
        threads = octets >= 1024 ? 1024 : (int)((octets + 31) / 32 * 32);
    }
    const int64_t per = (octets + threads - 1) / threads;
    const dim3 grid((unsigned)((m + rows - 1) / rows));
    auto kern = per == 1 ? rms_norm_kernel<1> : per == 2 ? rms_norm_kernel<2> : per <= 4 ? rms_norm_kernel<4> : rms_norm_kernel<0>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads, (unsigned)rows);
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
