// Microscaled 4-bit floating point (OCP MX: E2M1 elements, one E8M0 scale per 32 along a row): quantisation, the block format
// of files, and the product y = x . W^T with both sides in this format on the tensor cores' block-scaled instructions.
//
//   quantisation   e = clamp(floor(log2 max|v|) - 2, -127, 127) per 32 elements; code = v / 2^e rounded to the nearest of
//                  0, .5, 1, 1.5, 2, 3, 4, 6 (ties to the even code), beyond 6 to 6.  The division is exact.  A block with a NaN or an
//                  infinity gets the scale NaN (255): its row's outputs are NaN.
//   product        y[m][n] = sum over blocks of 2^(ea + ew) * sum of a_i * w_i: exact products, sums in f32 inside the tensor
//                  core (tcgen05.mma kind::mxf4, 64 elements of K per instruction, one scale per 32).
//
// Operand image: what the MMA reads, ready-made in global memory, so that a stage is one bulk copy per side.  Rows in tiles of T
// (128 for weights; for activations as many as a CTA takes), K in units of 256 elements:
//   unit (tile, u)   T x 128 bytes of codes, K-major, 16-byte chunks (one block each) XOR-swizzled within groups of eight rows,
//                    then per 128 rows two scale atoms of 512 bytes (128 elements of K each): scale of row r, block b at
//                    (r % 32) * 16 + (r / 32) * 4 + b, the order in which tcgen05.cp spreads them over tensor memory.
// 4.25 bits an element; K is padded to 256 and rows to the tile with zeros.  Activations for pairs of CTAs: a unit is two parts, each with the
// codes of half of the rows and the scales of all, so that a CTA of the pair copies one piece.
//
// Bound by: one row of small matrices, the latency of one launch and a chain of copy, products, reduction ([1024, 4096] 4.3 us); a few rows of large
// ones, reading the weights (8 x [14336, 4096] 7.4 us, 31 MB: 4.2 TB/s with all of start and end); many rows, the tensor cores and
// what L2 gives an SM (2048 x [14336, 4096] 51 us, 4.7 PFLOP/s, the tensor pipe 75 % busy; 73 with the quantizer and from new inputs; 512 x [4096, 14336]
// 26 us: 2.3).  Quantizing 512 x 4096 bf16 takes
// 2.4 us, reading the values back as f32 4.3.
#include <algorithm>
#include <mutex>

#include "abi.h"
#include "common.cuh"
#include "forward.h"
#include "gemv_params.h"
#include "quantize_act.cuh"
#include "tcgen05.cuh"

namespace lloom {

LLOOM_TU_REGISTER()

namespace {

constexpr int kMxBlock = 32, kMxUnit = 256, kMxBlockBytes = 17;
constexpr int kMxTile = 128;  // weight rows per tile: the MMA's M

__host__ __device__ constexpr int mx_scale_bytes(int rows) { return (rows + 127) / 128 * 1024; }
__host__ __device__ constexpr int mx_unit_bytes(int rows, int parts = 1) { return rows * 128 + parts * mx_scale_bytes(rows); }
__host__ __device__ inline int64_t mx_units(int64_t k) { return (k + kMxUnit - 1) / kMxUnit; }
// offsets inside a unit of T rows: 16-byte chunk `c` (block of the unit) of row r, and the scale of that block
__host__ __device__ inline int mx_chunk_offset(int r, int c) { return (r >> 3) * 1024 + (r & 7) * 128 + ((c ^ (r & 7)) << 4); }
__host__ __device__ inline int mx_scale_offset(int rows, int r, int c) {  // rows: of codes in front of the scales
    return rows * 128 + (r >> 7) * 1024 + (c >> 2) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (c & 3);
}

// ---- quantisation ----

// The larger one, or NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// Four lanes share a block, eight elements each: the lane's codes (element i in bits 4i ..) and the block's scale byte.
__device__ __forceinline__ uint32_t mx_quantize_quad(const float (&v)[8], uint32_t &scale) {
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max_nan(amax, fabsf(v[i]));
    amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const uint32_t field = __float_as_uint(amax) >> 23;  // 255: infinity or NaN
    scale = field == 255u ? 255u : field > 2u ? field - 2u : 0u;
    if (field == 255u) return 0u;
    const float inv = __uint_as_float((254u - scale) << 23);  // 2^-e
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = __fmul_rn(v[i], inv);
    uint32_t codes;
    asm("{\n"
        ".reg .b8 a, b, c, d;\n"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
        "mov.b32 %0, {a, b, c, d};\n"
        "}\n"
        : "=r"(codes)
        : "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]));
    return codes;
}

// Codes (128 bytes) and scales of one unit of row r of a tile, by a warp with elements 8 lane .. 8 lane + 7 in v.
__device__ __forceinline__ void mx_store_unit(const float (&v)[8], uint8_t *unit, int T, int parts, int r, int lane) {
    uint32_t scale;
    const uint32_t codes = mx_quantize_quad(v, scale);
    const int rows = parts == 2 ? T / 2 : T, part = parts == 2 && r >= rows ? 1 : 0, part_bytes = rows * 128 + mx_scale_bytes(T);
    *reinterpret_cast<uint32_t *>(unit + part * part_bytes + mx_chunk_offset(r - part * rows, lane >> 2) + (lane & 3) * 4) = codes;
    if ((lane & 3) == 0) {
        uint8_t *at = unit + mx_scale_offset(rows, r, lane >> 2);
        *at = (uint8_t)scale;
        if (parts == 2) at[part_bytes] = (uint8_t)scale;
    }
}

// Rows of x to the image of tiles of T rows: a warp has two units of a row, `across` warps of a CTA lie along it.  Rows from m to the
// end of the last tile and elements past k are zeros.  trigger: the stream's next kernel may start; not behind a kernel that writes weights,
// which later kernels read without waiting.
constexpr int kQuantUnits = 2;
template <int X_TYPE>
__global__ void __launch_bounds__(256) mx_quantize_kernel(const void *__restrict__ x, int m, int k, int units, int T, int parts, int rows,
                                                          int across, uint8_t *__restrict__ image, int trigger) {
    if (trigger) launch_dependents();
    wait_predecessor();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = (int)blockIdx.x * (8 / across) + warp / across, u0 = ((int)blockIdx.y * across + warp % across) * kQuantUnits;
    if (row >= rows || u0 >= units) return;  // whole warp
    const int64_t from = (int64_t)row * k + u0 * kMxUnit + lane * 8;
    const int left = row < m ? k - (u0 * kMxUnit + lane * 8) : 0;  // elements of the row from there
    float v[kQuantUnits][8];
#pragma unroll
    for (int j = 0; j < kQuantUnits; ++j) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] = 0.0f;
        if (j * kMxUnit < left) load8(x, X_TYPE, from + j * kMxUnit, v[j]);
    }
    const int tile = row / T;
    uint8_t *unit = image + ((int64_t)tile * units + u0) * mx_unit_bytes(T, parts);
#pragma unroll
    for (int j = 0; j < kQuantUnits; ++j)
        if (u0 + j < units) mx_store_unit(v[j], unit + (int64_t)j * mx_unit_bytes(T, parts), T, parts, row - tile * T, lane);
}

// A file's 17-byte blocks (scale, then elements 0..15 in the low and 16..31 in the high halves of 16 bytes) to the weight image,
// a thread per block of the padded matrix, and back.
__global__ void __launch_bounds__(256) mx_from_blocks_kernel(const uint8_t *__restrict__ blocks, int64_t n, int kb, int units, int64_t total,
                                                             uint8_t *__restrict__ image) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= total) return;
    const int per_row = units * 8;
    const int64_t row = i / per_row;
    const int b = (int)(i - row * per_row), c = b & 7;
    uint32_t w[4] = {0, 0, 0, 0}, scale = 0;
    if (row < n && b < kb) {
        const uint8_t *blk = blocks + (row * kb + b) * kMxBlockBytes;
        scale = __ldg(blk);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const uint32_t q = __ldg(blk + 1 + j);
            w[j >> 3] |= (q & 15u) << (4 * (j & 7));
            w[2 + (j >> 3)] |= (q >> 4) << (4 * (j & 7));
        }
    }
    const int r = (int)(row % kMxTile);
    uint8_t *unit = image + (row / kMxTile * units + (b >> 3)) * (int64_t)mx_unit_bytes(kMxTile);
    *reinterpret_cast<uint4 *>(unit + mx_chunk_offset(r, c)) = make_uint4(w[0], w[1], w[2], w[3]);
    unit[mx_scale_offset(kMxTile, r, c)] = (uint8_t)scale;
}

__global__ void __launch_bounds__(256) mx_to_blocks_kernel(const uint8_t *__restrict__ image, int64_t n, int kb, int units, uint8_t *__restrict__ blocks) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n * kb) return;
    const int64_t row = i / kb;
    const int b = (int)(i - row * kb), c = b & 7, r = (int)(row % kMxTile);
    const uint8_t *unit = image + (row / kMxTile * units + (b >> 3)) * (int64_t)mx_unit_bytes(kMxTile);
    const uint4 q = *reinterpret_cast<const uint4 *>(unit + mx_chunk_offset(r, c));
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    uint8_t *blk = blocks + i * kMxBlockBytes;
    blk[0] = unit[mx_scale_offset(kMxTile, r, c)];
#pragma unroll
    for (int j = 0; j < 16; ++j)
        blk[1 + j] = (uint8_t)(((w[j >> 3] >> (4 * (j & 7))) & 15u) | (((w[2 + (j >> 3)] >> (4 * (j & 7))) & 15u) << 4));
}

// A code's value times the scale: its exponent (bias 1) and mantissa bits, moved to the places of f16's, read as the value times 2^-14.
__device__ __forceinline__ float mx_value(uint32_t code, float d) {
    const uint32_t half = ((code & 7u) << 9) | ((code & 8u) << 12);
    return __fmul_rn(__half2float(__ushort_as_half((unsigned short)half)) * 16384.0f, d);
}

// Image to values: a warp has two units of a row, as in the quantizer.  2^e of the smallest scale is subnormal: products with it are exact all
// the same.
template <bool F16>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const uint8_t *__restrict__ image, int n, int k, int units, int across, void *__restrict__ out) {
    launch_dependents();
    wait_predecessor();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = (int)blockIdx.x * (8 / across) + warp / across, u0 = ((int)blockIdx.y * across + warp % across) * kQuantUnits;
    if (row >= n) return;
    const int r = row % kMxTile, c = lane >> 2;
    const uint8_t *unit = image + ((int64_t)(row / kMxTile) * units + u0) * mx_unit_bytes(kMxTile);
    const int chunk = mx_chunk_offset(r, c) + (lane & 3) * 4, scale = mx_scale_offset(kMxTile, r, c);
    uint32_t q[kQuantUnits], s[kQuantUnits];
#pragma unroll
    for (int j = 0; j < kQuantUnits; ++j) {
        const bool in = (u0 + j) * kMxUnit + lane * 8 < k;
        q[j] = in ? __ldg(reinterpret_cast<const uint32_t *>(unit + j * mx_unit_bytes(kMxTile) + chunk)) : 0u;
        s[j] = in ? __ldg(unit + j * mx_unit_bytes(kMxTile) + scale) : 0u;
    }
#pragma unroll
    for (int j = 0; j < kQuantUnits; ++j) {
        const int e = (u0 + j) * kMxUnit + lane * 8;
        if (e >= k) continue;
        const float d = s[j] == 255u ? __uint_as_float(0x7fc00000u) : s[j] == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(s[j] << 23);
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = mx_value(q[j] >> (4 * i), d);
        if (F16) {
            uint32_t h[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __half2 t = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                h[i] = *reinterpret_cast<const uint32_t *>(&t);
            }
            *reinterpret_cast<uint4 *>(reinterpret_cast<__half *>(out) + (int64_t)row * k + e) = make_uint4(h[0], h[1], h[2], h[3]);
        } else {
            float4 *o = reinterpret_cast<float4 *>(reinterpret_cast<float *>(out) + (int64_t)row * k + e);
            o[0] = make_float4(v[0], v[1], v[2], v[3]);
            o[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
    }
}

// ---- product ----

// Shared-memory matrix descriptor, high words: 128-byte swizzle with eight-row groups 1024 bytes apart (codes; the same as for
// 16-bit operands: rows of 128 bytes), and no swizzle with groups of 8 x 16 bytes 128 apart (scale atoms).
constexpr uint32_t kDescHiScales = (128u >> 4) | (1u << 14);

// D[128 x N] (+)= A[128 x 64] . B[N x 64]^T, E2M1, a scale per 32: `ids` = which half of the scale words (0 or 2) in the
// descriptor's fields.  Only the low descriptor words change from step to step.
__device__ __forceinline__ void umma_mxf4(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        ".reg .b64 da, db;\n\t"
        "setp.ne.b32 p, %7, 0;\n\t"
        "mov.b64 da, {%1, %3};\n\t"
        "mov.b64 db, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], da, db, %4, [%5], [%6], p;\n\t"
        "}\n" ::"r"(d),
        "r"(a_lo), "r"(b_lo), "r"(kUmmaDescHiSw128), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
// A scale atom (32 x 16 bytes) to four columns of tensor memory, in all four lane quarters.  In order with the MMAs that this
// thread issues before and after.
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t smem_lo) {
    asm volatile(
        "{\n\t"
        ".reg .b64 d;\n\t"
        "mov.b64 d, {%1, %2};\n\t"
        "tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], d;\n\t"
        "}\n" ::"r"(tmem),
        "r"(smem_lo), "r"(kDescHiScales)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr));
}

constexpr int kMxMaxStages = 12;
constexpr int kMxQuantWarps = 8;              // quantize in the prologue; the first four are the epilogue
constexpr int kMxThreads = 32 * (kMxQuantWarps + 2);  // and one warp copies, one issues MMAs

struct MxParams {
    const uint8_t *w, *a;  // images: weights (tiles of 128 rows), activations (tiles of bn rows)
    const void *x;         // or the activations themselves, which this kernel quantizes (a tile of 16 rows)
    int x_type;
    void *y;
    int y_type;
    int64_t ldy;
    int m, n, k, units;
    int bn, m_tiles;       // activation rows per tile (a multiple of 16, at most 256: the MMA's N)
    int split;             // CTAs of a cluster, which share the units of a tile
    int stages, stage_bytes;
    int resident;          // bytes in front of the stages: the CTA's part of K of all activations, where it quantizes them
    int tmem_cols;
    int wide;              // four outputs of a row may be stored together
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float4 ld_cluster4(uint32_t smem, int rank) {
    float4 v;
    asm volatile(
        "{\n\t"
        ".reg .b32 r;\n\t"
        "mapa.shared::cluster.u32 r, %4, %5;\n\t"
        "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [r];\n\t"
        "}\n"
        : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
        : "r"(smem), "r"(rank)
        : "memory");
    return v;
}
__device__ __forceinline__ void put4(float *y, const float4 &v) { *reinterpret_cast<float4 *>(y) = v; }
__device__ __forceinline__ void put4(__half *y, const float4 &v) {
    const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    *reinterpret_cast<uint2 *>(y) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}
__device__ __forceinline__ void put4(__nv_bfloat16 *y, const float4 &v) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2 *>(y) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}

// After a wait that ran out: the copies that a thread has started, `issued` stages in turn, end or run out of time themselves
__device__ __forceinline__ void drain(uint64_t *full, int issued, int stages) {
    for (int i = max(issued - stages, 0); i < issued; ++i)
        if (!mbar_wait(&full[i % stages], (uint32_t)(i / stages) & 1u)) break;
}

// One 128 x bn tile per cluster; its CTAs take equal parts of K, and the parts' sums meet in shared memory in a fixed order.
// QUANTIZE: up to sixteen activation rows, which every CTA quantizes itself, its part of K, while the first weights are on their way: one launch
// instead of two.
// Ends in every case: waits are bounded, and a CTA that gave up still meets the others.
template <bool QUANTIZE>
__global__ void __launch_bounds__(kMxThreads, 1) mx_gemm_kernel(const __grid_constant__ MxParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *ring = smem + (QUANTIZE ? p.resident : 0);
    uint64_t *full = reinterpret_cast<uint64_t *>(ring + p.stages * p.stage_bytes), *empty = full + kMxMaxStages, *done = empty + kMxMaxStages;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(done + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile = blockIdx.x / p.split, rank = blockIdx.x - tile * p.split;
    const int mt = tile % p.m_tiles, nt = tile / p.m_tiles;
    const int u0 = (int)((int64_t)p.units * rank / p.split), u1 = (int)((int64_t)p.units * (rank + 1) / p.split);
    const int count = u1 - u0;
    constexpr int kABytes = mx_unit_bytes(kMxTile), kQuantUnit = mx_unit_bytes(16);
    const int b_bytes = QUANTIZE ? 0 : mx_unit_bytes(p.bn);
    int issued = 0;  // stages that this thread has started to fill

    launch_dependents();
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(done, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    __syncthreads();
    if (warp == kMxQuantWarps) {
        // ---- operand tiles ----
        if (lane == 0) {
            const uint8_t *w = p.w + ((int64_t)nt * p.units + u0) * kABytes, *a = p.a + ((int64_t)mt * p.units + u0) * b_bytes;
            const int first = count < p.stages ? count : p.stages;
            for (int i = 0; i < first; ++i) {
                mbar_arrive_expect_tx(&full[i], (uint32_t)(kABytes + b_bytes));
                bulk_g2s(ring + i * p.stage_bytes, w + (int64_t)i * kABytes, kABytes, &full[i]);
            }
            issued = first;
            wait_predecessor();  // the activation image is there
            if (!QUANTIZE)
                for (int i = 0; i < first; ++i) bulk_g2s(ring + i * p.stage_bytes + kABytes, a + (int64_t)i * b_bytes, (uint32_t)b_bytes, &full[i]);
            int s = 0;
            uint32_t par = 0;
            for (int i = first; i < count; ++i) {
                if (!mbar_wait_abortable<0>(&empty[s], par, abort_flag)) break;
                mbar_arrive_expect_tx(&full[s], (uint32_t)(kABytes + b_bytes));
                bulk_g2s(ring + s * p.stage_bytes, w + (int64_t)i * kABytes, kABytes, &full[s]);
                if (!QUANTIZE) bulk_g2s(ring + s * p.stage_bytes + kABytes, a + (int64_t)i * b_bytes, (uint32_t)b_bytes, &full[s]);
                ++issued;
                if (++s == p.stages) {
                    s = 0;
                    par ^= 1;
                }
            }
        }
        __syncwarp();
    } else if (warp == kMxQuantWarps + 1) {
        // ---- MMA ----
        // Tensor memory is taken only once the kernel before has finished: one that has yet to take all of it may still be starting.
        wait_predecessor();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)p.tmem_cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        asm volatile("bar.sync 1, %0;" ::"n"(32 * (kMxQuantWarps + 1)) : "memory");  // with the quantizing and the epilogue warps
        const uint32_t tmem = *tmem_slot;
        if (elect_one()) {
            const uint32_t sfa = tmem + (uint32_t)((p.bn + 31) / 32 * 32), sfb = sfa + 8;
            const int groups = (p.bn + 127) / 128;
            // E2M1 both, E8M0 scales, K-major both, N, M = 128
            const uint32_t idesc = (1u << 7) | (1u << 10) | ((uint32_t)(p.bn >> 3) << 17) | (1u << 23) | (1u << 27);
            const uint32_t base = smem_u32(ring);
            bool ok = true;
            int s = 0;
            uint32_t par = 0;
            for (int i = 0; i < count; ++i) {
                ok = mbar_wait_abortable<0>(&full[s], par, abort_flag);
                if (!ok) break;
                tc_fence_after();
                const uint32_t at = base + (uint32_t)(s * p.stage_bytes), bt = QUANTIZE ? smem_u32(smem) + (uint32_t)(i * kQuantUnit) : at + kABytes;
                const uint32_t sa = umma_desc_lo(at + kMxTile * 128, 128), sb = umma_desc_lo(bt + (uint32_t)p.bn * 128, 128);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    copy_scales(sfa + 4 * j, sa + j * (512 >> 4));
                    copy_scales(sfb + 8 * j, sb + j * (512 >> 4));
                    if (!QUANTIZE && groups == 2) copy_scales(sfb + 8 * j + 4, sb + (1024 >> 4) + j * (512 >> 4));
                }
                const uint32_t a_lo = umma_desc_lo(at, 16), b_lo = umma_desc_lo(bt, 16);
#pragma unroll
                for (int j = 0; j < 4; ++j) {  // 64 elements: 32 bytes along the swizzled rows
                    const uint32_t ids = (j & 1) ? (2u << 4) | (2u << 29) : 0u;
                    umma_mxf4(tmem, a_lo + 2 * j, b_lo + 2 * j, idesc | ids, sfa + 4 * (j >> 1), sfb + 8 * (j >> 1), i > 0 || j > 0 ? 1u : 0u);
                }
                umma_commit(&empty[s]);
                if (++s == p.stages) {
                    s = 0;
                    par ^= 1;
                }
            }
            umma_commit(done);
        }
        __syncwarp();
    } else {
        wait_predecessor();  // the time limit of the wait for the sums counts from here
        if (QUANTIZE) {
            // a warp takes (row, unit) after (row, unit), four at a time
            const int items = p.m * count;
            for (int i0 = warp; i0 < items; i0 += 4 * kMxQuantWarps) {
                float v[4][8];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int i = i0 + j * kMxQuantWarps, r = i / count, e = (u0 + i - r * count) * kMxUnit + lane * 8;
#pragma unroll
                    for (int q = 0; q < 8; ++q) v[j][q] = 0.0f;
                    if (i < items && e < p.k) load8(p.x, p.x_type, (int64_t)r * p.k + e, v[j]);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int i = i0 + j * kMxQuantWarps, r = i / count;
                    if (i < items) mx_store_unit(v[j], smem + (i - r * count) * kQuantUnit, 16, 1, r, lane);
                }
            }
            fence_proxy_async();  // the tensor cores read what was written here
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * (kMxQuantWarps + 1)) : "memory");
    }
    // ---- epilogue ----
    if (warp < 4) {
        const bool ok = mbar_wait_abortable<64>(done, 0, abort_flag);
        tc_fence_after();
        const uint32_t tmem = *tmem_slot + ((uint32_t)(warp * 32) << 16);
        if (ok) {
            float *part = reinterpret_cast<float *>(smem);  // [bn][128]; every copy and MMA has finished with the memory
            for (int c0 = 0; c0 < p.bn; c0 += 16) {
                uint32_t v[16];
                tmem_ld16(tmem + (uint32_t)c0, v);
                tmem_ld_wait();
                loaded(v);
#pragma unroll
                for (int j = 0; j < 16; ++j) part[(c0 + j) * kMxTile + warp * 32 + lane] = __uint_as_float(v[j]);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {  // what is in flight ends first
        if (warp == kMxQuantWarps && lane == 0) drain(full, issued, p.stages);
        if (warp == kMxQuantWarps + 1) mbar_wait(done, 0);
        __syncthreads();
    }
    if (warp == kMxQuantWarps + 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot), "r"((uint32_t)p.tmem_cols));
    }
    if (p.split > 1) {
        __syncwarp();
        cluster_arrive();
        cluster_wait();
    }
    {
        const int rows = min(p.bn, p.m - mt * p.bn);
        const int c0 = rows * rank / p.split, c1 = rows * (rank + 1) / p.split;
        const uint32_t part = smem_u32(smem);
        const int64_t n = (int64_t)nt * kMxTile + 4 * lane;
        with_y_type(p.y, p.y_type, [&](auto *y) {
            // a warp per row of outputs, four per lane (straight from tensor memory a store has 32: 14336 outputs of 128 rows took 3 us longer)
            for (int c = c0 + warp; c < c1; c += kMxThreads / 32) {
                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
                for (int q = 0; q < p.split; ++q) {
                    const float4 v = ld_cluster4(part + 16u * (uint32_t)(c * (kMxTile / 4) + lane), q);
                    sum.x += v.x;
                    sum.y += v.y;
                    sum.z += v.z;
                    sum.w += v.w;
                }
                auto *out = y + ((int64_t)mt * p.bn + c) * p.ldy + n;
                if (p.wide && n + 4 <= p.n) {
                    put4(out, sum);
                } else {
                    if (n < p.n) put_y(out, 0, sum.x);
                    if (n + 1 < p.n) put_y(out, 1, sum.y);
                    if (n + 2 < p.n) put_y(out, 2, sum.z);
                    if (n + 3 < p.n) put_y(out, 3, sum.w);
                }
            }
        });
    }
    if (p.split > 1) {
        cluster_arrive();
        cluster_wait();  // the others may still read this CTA's part
    }
}

// ---- product of many rows: pairs of CTAs ----
// Two CTAs on neighbouring SMs compute a 256 x bn tile with one instruction (cta_group::2): each has 128 rows of weights and of the
// accumulator and half of the activation rows, so that a stage brings 35 KB per CTA where one alone would load 50 for the same work: bulk copies
// from L2 run at 69 bytes a clock and SM, and a stage of bn = 240 takes the tensor cores 480 clocks.  Persistent: the pairs walk the
// tiles, and with two accumulators in tensor memory the stores of one tile run under the next one's products.
// The first CTA of a pair issues the MMAs of both, and both CTAs' copies complete on its barriers, which takes TMA's tensor copies: untiled ones
// may only signal their own CTA, and passing that on by a thread (wait, arrive across the cluster) cost a microsecond a stage, four times
// the stage's work.  The maps see an image as rows of 128 bytes.
constexpr int kPairMaxBn = 240;  // two accumulators and the scales fill the 512 columns
constexpr int kPairStages = 12;
constexpr int kPairEpiWarps = 8;
constexpr int kPairThreads = 32 * (kPairEpiWarps + 2);

struct MxPairParams {
    CUtensorMap w, a;  // boxes of a unit's rows of 128 bytes: of weights; of one part of the activations
    void *y;
    int y_type;
    int64_t ldy;
    int m, n, units;
    int bn, m_tiles, n_tiles;  // n_tiles of 128 rows; a pair takes two
    int stages, stage_bytes;
};

__device__ __forceinline__ uint32_t mapa(uint32_t smem, int rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem), "r"(rank));
    return r;
}
// Rows `row` .. of a map's box to this CTA's shared memory; `bar`: of either CTA of the pair
__device__ __forceinline__ void copy_rows(void *dst, const CUtensorMap *map, int row, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(0), "r"(row), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void umma2_mxf4(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        ".reg .b64 da, db;\n\t"
        "setp.ne.b32 p, %7, 0;\n\t"
        "mov.b64 da, {%1, %3};\n\t"
        "mov.b64 db, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], da, db, %4, [%5], [%6], p;\n\t"
        "}\n" ::"r"(d),
        "r"(a_lo), "r"(b_lo), "r"(kUmmaDescHiSw128), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
// In both CTAs, from each one's own shared memory
__device__ __forceinline__ void copy_scales2(uint32_t tmem, uint32_t smem_lo) {
    asm volatile(
        "{\n\t"
        ".reg .b64 d;\n\t"
        "mov.b64 d, {%1, %2};\n\t"
        "tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], d;\n\t"
        "}\n" ::"r"(tmem),
        "r"(smem_lo), "r"(kDescHiScales)
        : "memory");
}
// Arrives at the barrier of this address in both CTAs once the MMAs issued so far have finished
__device__ __forceinline__ void umma2_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                 "h"((unsigned short)3)
                 : "memory");
}

__global__ void __launch_bounds__(kPairThreads, 1) mx_gemm_pair_kernel(const __grid_constant__ MxPairParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + p.stages * p.stage_bytes), *empty = full + kPairStages;
    uint64_t *acc_full = empty + kPairStages, *acc_empty = acc_full + 2, *drained = acc_empty + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drained + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x & 1;
    const int tiles = (p.n_tiles + 1) / 2 * p.m_tiles, first = blockIdx.x >> 1, step = gridDim.x >> 1;
    constexpr int kABytes = mx_unit_bytes(kMxTile);
    const int half = p.bn / 2 * 128, part_bytes = half + mx_scale_bytes(p.bn), part_rows = part_bytes / 128;
    int issued = 0;
    bool issuer = false;

    launch_dependents();
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&full[s], 1);  // the first CTA's are used: both CTAs' copies
            mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], 2 * kPairEpiWarps);
        }
        mbar_init(drained, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == kPairEpiWarps + 1) {
        wait_predecessor();  // see mx_gemm_kernel
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    wait_predecessor();

    if (warp == kPairEpiWarps) {
        // ---- operand tiles ----
        if (lane == 0) {
            bool ok = true;
            int s = 0, fill = 0;
            uint32_t par = 1;
            const uint32_t full0 = mapa(smem_u32(full), 0);
            for (int t = first; t < tiles && ok; t += step) {
                const int mt = t % p.m_tiles, nt = min(t / p.m_tiles * 2 + rank, p.n_tiles - 1);  // an odd last tile: once more, not stored
                int w = nt * p.units * (kABytes / 128), a = (mt * p.units * 2 + rank) * part_rows;  // rows of 128 bytes
                for (int u = 0; u < p.units; ++u) {
                    if (fill >= p.stages) {
                        ok = mbar_wait_abortable<0>(&empty[s], par, abort_flag);
                        if (!ok) break;
                    } else {
                        ++fill;
                    }
                    uint8_t *dst = smem + s * p.stage_bytes;
                    const uint32_t bar = full0 + 8u * (uint32_t)s;
                    if (rank == 0) mbar_arrive_expect_tx(&full[s], (uint32_t)(2 * (kABytes + part_bytes)));
                    copy_rows(dst, &p.w, w, bar);
                    copy_rows(dst + kABytes, &p.a, a, bar);
                    ++issued;
                    w += kABytes / 128;
                    a += 2 * part_rows;
                    if (++s == p.stages) {
                        s = 0;
                        par ^= 1;
                    }
                }
            }
        }
        __syncwarp();
    } else if (warp == kPairEpiWarps + 1) {
        // ---- MMA, for both CTAs ----
        issuer = rank == 0 && elect_one();
        if (issuer) {
            const int groups = (p.bn + 127) / 128;
            const uint32_t sfa = tmem + 2 * (uint32_t)p.bn, sfb = sfa + 8;
            const uint32_t idesc = (1u << 7) | (1u << 10) | ((uint32_t)(p.bn >> 3) << 17) | (1u << 23) | (2u << 27);
            const uint32_t base = smem_u32(smem);
            bool ok = true;
            int s = 0, acc = 0;
            uint32_t par = 0, acc_par = 1;
            for (int t = first; t < tiles && ok; t += step) {
                ok = mbar_wait_abortable<0>(&acc_empty[acc], acc_par, abort_flag);
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = tmem + (uint32_t)(acc * p.bn);
                for (int u = 0; u < p.units; ++u) {
                    ok = mbar_wait_abortable<0>(&full[s], par, abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t at = base + (uint32_t)(s * p.stage_bytes), bt = at + kABytes;
                    const uint32_t sa = umma_desc_lo(at + kMxTile * 128, 128), sb = umma_desc_lo(bt + (uint32_t)half, 128);
                    const uint32_t a_lo = umma_desc_lo(at, 16), b_lo = umma_desc_lo(bt, 16);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        copy_scales2(sfa + 4 * j, sa + j * (512 >> 4));
                        copy_scales2(sfb + 8 * j, sb + j * (512 >> 4));
                        if (groups == 2) copy_scales2(sfb + 8 * j + 4, sb + (1024 >> 4) + j * (512 >> 4));
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t ids = (j & 1) ? (2u << 4) | (2u << 29) : 0u;
                        umma2_mxf4(d, a_lo + 2 * j, b_lo + 2 * j, idesc | ids, sfa + 4 * (j >> 1), sfb + 8 * (j >> 1), u > 0 || j > 0 ? 1u : 0u);
                    }
                    umma2_commit(&empty[s]);
                    if (++s == p.stages) {
                        s = 0;
                        par ^= 1;
                    }
                }
                umma2_commit(&acc_full[acc]);
                if (acc == 1) acc_par ^= 1;
                acc ^= 1;
            }
        }
        __syncwarp();
    } else {
        // ---- epilogue: a warp has 32 rows of weights and about half of the columns ----
        const int q = warp & 3, c_mid = (p.bn / 2 + 15) / 16 * 16;
        const int c_begin = warp < 4 ? 0 : c_mid, c_end = warp < 4 ? c_mid : p.bn;
        const uint32_t empty0 = mapa(smem_u32(acc_empty), 0);
        bool ok = true;
        int acc = 0;
        uint32_t par = 0;
        for (int t = first; t < tiles && ok; t += step) {
            ok = mbar_wait_abortable<64>(&acc_full[acc], par, abort_flag);
            if (!ok) break;
            tc_fence_after();
            const int mt = t % p.m_tiles;
            const int64_t n = ((int64_t)(t / p.m_tiles) * 2 + rank) * kMxTile + q * 32 + lane;
            const uint32_t from = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * p.bn);
            with_y_type(p.y, p.y_type, [&](auto *y) {
                for (int c = c_begin; c < c_end; c += 16) {
                    uint32_t v[16];
                    tmem_ld16(from + (uint32_t)c, v);
                    tmem_ld_wait();
                    loaded(v);
                    const int row = mt * p.bn + c, left = n < p.n ? p.m - row : 0;
                    auto *at = y + (int64_t)row * p.ldy + n;
                    if (left >= 16) {
#pragma unroll
                        for (int j = 0; j < 16; ++j, at += p.ldy) put_y(at, 0, __uint_as_float(v[j]));
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; ++j, at += p.ldy)
                            if (j < left) put_y(at, 0, __uint_as_float(v[j]));
                    }
                }
            });
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(empty0 + 8u * (uint32_t)acc);
            if (acc == 1) par ^= 1;
            acc ^= 1;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {  // what is in flight ends first; the second CTA's copies, which arrive at the first one's barriers, have a millisecond
        if (rank == 0 && warp == kPairEpiWarps && lane == 0) drain(full, issued, p.stages);
        if (issuer) {
            umma2_commit(drained);
            mbar_wait(drained, 0);
        }
        if (rank == 1 && warp == kPairEpiWarps)
            for (int i = 0; i < 1000; ++i) __nanosleep(1000);
        __syncthreads();
    }
    cluster_arrive();
    cluster_wait();  // neither reads the other's memory, or computes into it, any more
    if (warp == kPairEpiWarps + 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
    }
}

// Activation rows in `count` equal tiles, each a multiple of 16
struct MxTiles {
    int bn, count;
};
MxTiles mx_tiles(int64_t m, int64_t count) {
    MxTiles t;
    t.count = (int)count;
    t.bn = (int)((m + count - 1) / count + 15) / 16 * 16;
    return t;
}

int mx_check(int64_t m, int64_t n, int64_t k) {
    if (m <= 0 || n <= 0 || k <= 0 || k % kMxBlock != 0) return LLOOM_ERR_SHAPE;
    if (m > (1 << 24) || n > (1 << 30) || k > (1 << 24)) return LLOOM_ERR_SHAPE;
    return LLOOM_OK;
}

int64_t mx_image_bytes(int64_t rows, int64_t k, int T, int parts = 1) { return (rows + T - 1) / T * mx_units(k) * mx_unit_bytes(T, parts); }

// CTAs of eight warps over rows of units, kQuantUnits to a warp: `across` of a CTA's warps lie along a row
dim3 mx_row_grid(int64_t rows, int64_t units, int &across) {
    for (across = 1; across < 8 && across * kQuantUnits < units; across *= 2) {}
    return dim3((unsigned)ceil_div64(rows, 8 / across), (unsigned)ceil_div64(units, kQuantUnits * across));
}

int launch_mx_quantize(const void *x, int x_type, int64_t m, int64_t k, int T, int parts, uint8_t *image, bool trigger, bool overlap,
                       cudaStream_t stream) {
    const int64_t rows = (m + T - 1) / T * T, units = mx_units(k);
    if (rows > 0x7fffffff) return LLOOM_ERR_SHAPE;
    int across;
    const dim3 grid = mx_row_grid(rows, units, across);
    if (grid.y > 65535) return LLOOM_ERR_SHAPE;
    auto kern = x_type == LLOOM_F32   ? mx_quantize_kernel<LLOOM_F32>
                : x_type == LLOOM_F16 ? mx_quantize_kernel<LLOOM_F16>
                                      : mx_quantize_kernel<LLOOM_BF16>;
    return launch_status(launch_early(kern, grid, 256, 0, overlap, stream, x, (int)m, (int)k, (int)units, T, parts, (int)rows, across, image,
                                      trigger ? 1 : 0));
}

// Tiles for pairs of CTAs: of the widths that fit, the one with the least time over the rounds that the pairs make, a unit of K taking
// 2 bn clocks of the tensor cores or its bytes at 69 per clock.
MxTiles mx_pair_tiles(int64_t m, int64_t n, int pairs) {
    const int64_t n_pairs = (n + 2 * kMxTile - 1) / (2 * kMxTile);
    MxTiles best = {0, 0};
    double least = 0;
    const int64_t fewest = (m + kPairMaxBn - 1) / kPairMaxBn;
    for (int64_t count = fewest; count < fewest + 8 && count <= (m + 63) / 64; ++count) {
        const MxTiles t = mx_tiles(m, count);
        const double clocks = 2.0 * t.bn, bytes = (mx_unit_bytes(kMxTile) + t.bn * 64 + mx_scale_bytes(t.bn)) / 69.0;
        const double time = (double)((n_pairs * t.count + pairs - 1) / pairs) * (clocks > bytes ? clocks : bytes);
        if (best.count == 0 || time < least) {
            best = t;
            least = time;
        }
    }
    return best;
}

// The three rules, with both sides measured (us a call on a B200, bf16 in and out, weights [n, k]):
//   pairs of CTAs past 128 rows, if K is short or they have tiles for half of the SMs: their own K is not split.  Split / pairs:
//     [1024, 4096] 128 rows 9.2 / 10.4, 192 10.8 / 10.5, 256 12.5 / 10.8; [4096, 4096] 128 10.9 / 10.8, 192 12.6 / 11.1;
//     [14336, 4096] 96 11.6 / 12.3, 128 12.8 / 12.2, 256 17.7 / 16.5; [4096, 14336] 128 15.8 / 22.2, 384 22.7 / 25.0; [8192, 8192] 384 21.5 / 19.8
//   split: K over as many CTAs of a cluster, up to eight, as there are SMs for, one unit at least to each.
//   quantize: the quantizer in the product's prologue where a CTA has up to 32 (row, unit of K) pairs to do, four to a warp: beyond, all CTAs
//     repeating the work costs more than a launch.  In the prologue / in a launch of its own: 1 x [1024, 4096] 4.5 / 5.9, 16 x [1024, 4096] (32) 5.9 / 6.3,
//     8 x [4096, 4096] (32) 6.9 / 7.0, 16 x [4096, 4096] (64) 8.8 / 7.2, 1 x [14336, 4096] (16) 6.7 / 7.7, 4 x [14336, 4096] (64) 9.3 / 8.0
struct MxPlan {
    bool pairs, quantize;
    MxTiles tiles;
    int split;
};
MxPlan mx_plan(int64_t m, int64_t n, int64_t k, int sms) {
    MxPlan pl;
    const int64_t units = mx_units(k);
    pl.tiles = mx_pair_tiles(m, n, sms / 2);
    const int64_t pair_tiles = (n + 2 * kMxTile - 1) / (2 * kMxTile) * pl.tiles.count;
    pl.pairs = m > 128 && (units <= 32 || pair_tiles * 4 >= sms);
    if (!pl.pairs) pl.tiles = mx_tiles(m, (m + 255) / 256);
    const int64_t tiles = (n + kMxTile - 1) / kMxTile * pl.tiles.count;
    for (pl.split = 1; pl.split < 8 && tiles * pl.split * 2 <= sms && units >= pl.split * 2; pl.split *= 2) {}
    const int64_t part = (units + pl.split - 1) / pl.split;
    pl.quantize = m <= 16 && m * part <= 32;
    return pl;
}
// Bytes of the activation image, whatever the device's plan: the largest of all tile widths
int64_t mx_act_bytes(int64_t m, int64_t k) {
    int64_t most = 0;
    for (int T = 16; T <= 256; T += 16) most = std::max(most, (m + T - 1) / T * mx_unit_bytes(T, 2));
    return most * mx_units(k);
}

struct MxSmemOnce {
    std::mutex mu;
    bool done[64] = {false};
};

template <class Params>
int launch_mx_gemm(void (*kern)(Params), MxSmemOnce &once, const Params &p, int stages, int ctas, int cluster, int threads, bool early, cudaStream_t stream) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || dev < 0 || dev >= 64) return LLOOM_ERR_DEVICE;
    const int smem = stages + 256 + 1024;
    {
        std::lock_guard<std::mutex> lock(once.mu);
        if (!once.done[dev]) {
            e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
            if (e != cudaSuccess) return launch_status(e);
            once.done[dev] = true;
        }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = early ? 2 : 1;
    return launch_status(cudaLaunchKernelEx(&cfg, kern, p));
}

}  // namespace

int mx_forward(const void *image, const void *x, int x_type, void *y, int y_type, int64_t m, int64_t n, int64_t k, int64_t ldy, void *workspace,
               int64_t workspace_bytes, void *stream, bool overlap) {
    int rc = mx_check(m, n, k);
    if (rc != LLOOM_OK) return rc;
    if (!elem_type_ok(x_type) || !elem_type_ok(y_type)) return LLOOM_ERR_DTYPE;
    if (ldy < n) return LLOOM_ERR_SHAPE;
    if (!image || !x || !y) return LLOOM_ERR_NULL;
    if (!workspace || workspace_bytes < lloom_b200_mx_workspace_bytes(m, n, k)) return LLOOM_ERR_WORKSPACE;
    if (!aligned(workspace, 256) || !aligned(image, 256) || !aligned(x, 16) || !aligned(y, elem_bytes(y_type))) return LLOOM_ERR_ALIGN;
    DeviceInfo di;
    rc = device_info(di);
    if (rc != LLOOM_OK) return rc;
    const MxPlan pl = mx_plan(m, n, k, di.sm_count);
    const MxTiles t = pl.tiles;
    // The product may start while the quantizer runs; the quantizer itself (or the product that does its work) starts under the kernel in front
    // only if the weights are in place.
    if (!pl.quantize) {
        rc = launch_mx_quantize(x, x_type, m, k, t.bn, pl.pairs ? 2 : 1, (uint8_t *)workspace, true, overlap, (cudaStream_t)stream);
        if (rc != LLOOM_OK) return rc;
    }
    const int64_t n_tiles = (n + kMxTile - 1) / kMxTile;
    const int units = (int)mx_units(k);
    if (pl.pairs) {
        static MxSmemOnce once;
        MxPairParams p = {};
        const int64_t w_rows = mx_image_bytes(n, k, kMxTile) / 128, a_rows = mx_image_bytes(m, k, t.bn, 2) / 128;
        if (w_rows > 0x7fffffff || a_rows > 0x7fffffff) return LLOOM_ERR_SHAPE;  // 256 GB
        if (!encode_rows_map(p.w, image, w_rows, 128, 128, mx_unit_bytes(kMxTile) / 128) ||
            !encode_rows_map(p.a, workspace, a_rows, 128, 128, mx_unit_bytes(t.bn, 2) / 256))
            return LLOOM_ERR_DEVICE;
        p.y = y;
        p.y_type = y_type;
        p.ldy = ldy;
        p.m = (int)m;
        p.n = (int)n;
        p.units = units;
        p.bn = t.bn;
        p.m_tiles = t.count;
        p.n_tiles = (int)n_tiles;
        p.stage_bytes = mx_unit_bytes(kMxTile) + t.bn * 64 + mx_scale_bytes(t.bn);
        p.stages = (di.max_smem_optin - 256 - 1024) / p.stage_bytes;
        if (p.stages > kPairStages) p.stages = kPairStages;
        const int64_t tiles = (n_tiles + 1) / 2 * t.count;
        if (tiles > 0x3fffffff) return LLOOM_ERR_SHAPE;
        const int pairs = (int)(tiles < di.sm_count / 2 ? tiles : di.sm_count / 2);
        return launch_mx_gemm(mx_gemm_pair_kernel, once, p, p.stages * p.stage_bytes, 2 * pairs, 2, kPairThreads, true, (cudaStream_t)stream);
    }
    static MxSmemOnce once, once_quantize;
    MxParams p = {};
    p.w = (const uint8_t *)image;
    p.a = (const uint8_t *)workspace;
    p.x = x;
    p.x_type = x_type;
    p.y = y;
    p.y_type = y_type;
    p.ldy = ldy;
    p.m = (int)m;
    p.n = (int)n;
    p.k = (int)k;
    p.units = units;
    p.bn = t.bn;
    p.m_tiles = t.count;
    p.split = pl.split;
    p.wide = ldy % 4 == 0 && aligned(y, 4 * elem_bytes(y_type));
    const int64_t ctas = n_tiles * t.count * p.split;
    if (ctas > 0x7fffffff) return LLOOM_ERR_SHAPE;
    p.resident = pl.quantize ? (units + p.split - 1) / p.split * mx_unit_bytes(16) : 0;
    p.stage_bytes = mx_unit_bytes(kMxTile) + (pl.quantize ? 0 : mx_unit_bytes(t.bn));
    p.stages = (di.max_smem_optin - 256 - 1024 - p.resident) / p.stage_bytes;
    if (p.stages > kMxMaxStages) p.stages = kMxMaxStages;
    const int cols = (t.bn + 31) / 32 * 32 + 24;
    for (p.tmem_cols = 32; p.tmem_cols < cols; p.tmem_cols *= 2) {}
    const int smem = p.resident + p.stages * p.stage_bytes;
    return pl.quantize ? launch_mx_gemm(mx_gemm_kernel<true>, once_quantize, p, smem, (int)ctas, p.split, kMxThreads, overlap, (cudaStream_t)stream)
                       : launch_mx_gemm(mx_gemm_kernel<false>, once, p, smem, (int)ctas, p.split, kMxThreads, true, (cudaStream_t)stream);
}

int mx_quantize(const void *x, int x_type, int64_t rows, int64_t k, void *image, int64_t image_bytes, void *stream, bool overlap) {
    const int rc = mx_check(1, rows, k);
    if (rc != LLOOM_OK) return rc;
    if (!elem_type_ok(x_type)) return LLOOM_ERR_DTYPE;
    if (!x || !image) return LLOOM_ERR_NULL;
    if (image_bytes < mx_image_bytes(rows, k, kMxTile)) return LLOOM_ERR_WORKSPACE;
    if (!aligned(x, 16) || !aligned(image, 256)) return LLOOM_ERR_ALIGN;
    return launch_mx_quantize(x, x_type, rows, k, kMxTile, 1, (uint8_t *)image, false, overlap, (cudaStream_t)stream);
}

int mx_dequantize(const void *image, int64_t rows, int64_t k, void *out, bool f16, void *stream, bool overlap) {
    const int rc = mx_check(1, rows, k);
    if (rc != LLOOM_OK) return rc;
    if (!image || !out) return LLOOM_ERR_NULL;
    if (!aligned(image, 256) || !aligned(out, 16)) return LLOOM_ERR_ALIGN;
    int across;
    const dim3 grid = mx_row_grid(rows, mx_units(k), across);
    if (grid.y > 65535) return LLOOM_ERR_SHAPE;
    return launch_status(launch_early(f16 ? mx_dequantize_kernel<true> : mx_dequantize_kernel<false>, grid, 256, 0, overlap, (cudaStream_t)stream,
                                      (const uint8_t *)image, (int)rows, (int)k, (int)mx_units(k), across, out));
}

}  // namespace lloom

using namespace lloom;

extern "C" {

int64_t lloom_b200_mx_image_bytes(int64_t rows, int64_t k) { return mx_check(1, rows, k) != LLOOM_OK ? 0 : mx_image_bytes(rows, k, kMxTile); }

int64_t lloom_b200_mx_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    return mx_check(m, n, k) != LLOOM_OK ? 0 : mx_act_bytes(m, k);
}

int lloom_b200_mx_quantize(const void *x, int x_type, int64_t rows, int64_t k, void *image, int64_t image_bytes, void *stream) {
    return mx_quantize(x, x_type, rows, k, image, image_bytes, stream, launch_overlap() > 0);
}

int lloom_b200_mx_from_blocks(const void *blocks, int64_t rows, int64_t k, void *image, int64_t image_bytes, void *stream) {
    const int rc = mx_check(1, rows, k);
    if (rc != LLOOM_OK) return rc;
    if (!blocks || !image) return LLOOM_ERR_NULL;
    if (image_bytes < mx_image_bytes(rows, k, kMxTile)) return LLOOM_ERR_WORKSPACE;
    if (!aligned(image, 256)) return LLOOM_ERR_ALIGN;
    const int64_t total = (rows + kMxTile - 1) / kMxTile * kMxTile * mx_units(k) * 8, grid = ceil_div64(total, 256);
    if (grid > 0x7fffffff) return LLOOM_ERR_SHAPE;
    mx_from_blocks_kernel<<<(unsigned)grid, 256, 0, (cudaStream_t)stream>>>((const uint8_t *)blocks, rows, (int)(k / kMxBlock), (int)mx_units(k),
                                                                            total, (uint8_t *)image);
    return launch_status(cudaGetLastError());
}

int lloom_b200_mx_to_blocks(const void *image, int64_t rows, int64_t k, void *blocks, void *stream) {
    const int rc = mx_check(1, rows, k);
    if (rc != LLOOM_OK) return rc;
    if (!blocks || !image) return LLOOM_ERR_NULL;
    if (!aligned(image, 256)) return LLOOM_ERR_ALIGN;
    const int64_t grid = ceil_div64(rows * (k / kMxBlock), 256);
    if (grid > 0x7fffffff) return LLOOM_ERR_SHAPE;
    mx_to_blocks_kernel<<<(unsigned)grid, 256, 0, (cudaStream_t)stream>>>((const uint8_t *)image, rows, (int)(k / kMxBlock), (int)mx_units(k),
                                                                          (uint8_t *)blocks);
    return launch_status(cudaGetLastError());
}

int lloom_b200_mx_dequantize(const void *image, int64_t rows, int64_t k, void *out, int out_is_f16, void *stream) {
    return mx_dequantize(image, rows, k, out, out_is_f16 != 0, stream, launch_overlap() > 0);
}

int lloom_b200_mx_fwd(const void *image, const void *x, int x_type, void *y, int y_type, int64_t m, int64_t n, int64_t k, int64_t ldy,
                      void *workspace, int64_t workspace_bytes, void *stream) {
    return mx_forward(image, x, x_type, y, y_type, m, n, k, ldy, workspace, workspace_bytes, stream, launch_overlap() > 0);
}

}  // extern "C"
