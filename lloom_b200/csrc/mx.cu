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
// 4.25 bits an element; K is padded to 256 and rows to the tile with zeros.
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
__host__ __device__ constexpr int mx_unit_bytes(int rows) { return rows * 128 + mx_scale_bytes(rows); }
__host__ __device__ inline int64_t mx_units(int64_t k) { return (k + kMxUnit - 1) / kMxUnit; }
// offsets inside a unit of T rows: 16-byte chunk `c` (block of the unit) of row r, and the scale of that block
__host__ __device__ inline int mx_chunk_offset(int r, int c) { return (r >> 3) * 1024 + (r & 7) * 128 + ((c ^ (r & 7)) << 4); }
__host__ __device__ inline int mx_scale_offset(int T, int r, int c) {
    return T * 128 + (r >> 7) * 1024 + (c >> 2) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (c & 3);
}

// ---- quantisation ----

// Four lanes share a block, eight elements each: the lane's codes (element i in bits 4i ..) and the block's scale byte.
__device__ __forceinline__ uint32_t mx_quantize_quad(const float (&v)[8], uint32_t &scale) {
    uint32_t top = 0;  // of the magnitudes' bits, so that an infinity or a NaN is the largest
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t field = top >> 23;
    scale = field == 255u ? 255u : field > 2u ? field - 2u : 0u;
    if (field == 255u) return 0u;
    const float inv = __uint_as_float((254u - scale) << 23);  // 2^-e
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t two;
        asm("{\n"
            ".reg .b8 t;\n"
            "cvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n"
            "cvt.u32.u8 %0, t;\n"
            "}\n"
            : "=r"(two)
            : "f"(__fmul_rn(v[2 * i], inv)), "f"(__fmul_rn(v[2 * i + 1], inv)));
        codes |= two << (8 * i);
    }
    return codes;
}

// One warp per (row, unit): 256 elements to 128 bytes of codes and eight scales of the image of tiles of T rows.  Rows from m to
// the end of the last tile and elements past k are zeros.  trigger: the stream's next kernel may start; not behind a kernel that
// writes weights, which later kernels read without waiting.
__global__ void __launch_bounds__(256) mx_quantize_kernel(const void *__restrict__ x, int x_type, int64_t m, int k, int units, int T, int64_t rows,
                                                          uint8_t *__restrict__ image, int trigger) {
    if (trigger) launch_dependents();
    wait_predecessor();
    const int lane = threadIdx.x & 31;
    const int64_t item = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    const int64_t row = item / units;
    const int u = (int)(item - row * units);
    if (row >= rows) return;  // whole warp
    const int e = u * kMxUnit + lane * 8;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    if (row < m && e < k) load8(x, x_type, row * k + e, v);
    uint32_t scale;
    const uint32_t codes = mx_quantize_quad(v, scale);
    const int64_t tile = row / T;
    const int r = (int)(row - tile * T);
    uint8_t *unit = image + (tile * units + u) * mx_unit_bytes(T);
    *reinterpret_cast<uint32_t *>(unit + mx_chunk_offset(r, lane >> 2) + (lane & 3) * 4) = codes;
    // the scales of four blocks make a word: lanes 0, 4, 8, 12 and 16, 20, 24, 28
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) word |= __shfl_sync(0xffffffffu, scale, (lane & 16) + 4 * i) << (8 * i);
    if ((lane & 15) == 0) *reinterpret_cast<uint32_t *>(unit + mx_scale_offset(T, r, lane >> 2)) = word;
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

// Eight elements per thread.  2^e of the smallest scales is subnormal: the product with an element's value is exact all the same.
template <bool F16>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const uint8_t *__restrict__ image, int64_t n, int k, int units, void *__restrict__ out) {
    launch_dependents();
    wait_predecessor();
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int per_row = k / 8;
    const int64_t row = i / per_row;
    if (row >= n) return;
    const int e = (int)(i - row * per_row) * 8, b = e / kMxBlock, c = b & 7, r = (int)(row % kMxTile);
    const uint8_t *unit = image + (row / kMxTile * units + (b >> 3)) * (int64_t)mx_unit_bytes(kMxTile);
    const uint32_t q = *reinterpret_cast<const uint32_t *>(unit + mx_chunk_offset(r, c) + ((e >> 3) & 3) * 4);
    const uint32_t s = unit[mx_scale_offset(kMxTile, r, c)];
    const float d = s == 255u ? __uint_as_float(0x7fc00000u) : s == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(s << 23);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t code = (q >> (4 * j)) & 15u, m = code & 7u;
        // twice the magnitude: 0, 1, 2, 3, 4, 6, 8, 12
        const uint32_t twice = m < 4u ? m : m == 4u ? 4u : m == 5u ? 6u : m == 6u ? 8u : 12u;
        const float a = 0.5f * (float)twice;
        v[j] = __fmul_rn(code & 8u ? -a : a, d);
    }
    if (F16) {
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __half2 t = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
            h[j] = *reinterpret_cast<const uint32_t *>(&t);
        }
        *reinterpret_cast<uint4 *>(reinterpret_cast<__half *>(out) + row * k + e) = make_uint4(h[0], h[1], h[2], h[3]);
    } else {
        float4 *o = reinterpret_cast<float4 *>(reinterpret_cast<float *>(out) + row * k + e);
        o[0] = make_float4(v[0], v[1], v[2], v[3]);
        o[1] = make_float4(v[4], v[5], v[6], v[7]);
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
constexpr int kMxThreads = 192;  // warps 0-3 epilogue, 4 copies, 5 MMA

struct MxParams {
    const uint8_t *w, *a;  // images: weights (tiles of 128 rows), activations (tiles of bn rows)
    void *y;
    int y_type;
    int64_t ldy;
    int m, n, units;
    int bn, m_tiles;       // activation rows per tile (a multiple of 16, at most 256: the MMA's N)
    int split;             // CTAs of a cluster, which share the units of a tile
    int stages, stage_bytes;
    int tmem_cols;
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float ld_cluster(uint32_t smem, int rank) {
    float v;
    asm volatile(
        "{\n\t"
        ".reg .b32 r;\n\t"
        "mapa.shared::cluster.u32 r, %1, %2;\n\t"
        "ld.shared::cluster.f32 %0, [r];\n\t"
        "}\n"
        : "=f"(v)
        : "r"(smem), "r"(rank)
        : "memory");
    return v;
}

// One 128 x bn tile per cluster; its CTAs take equal parts of K, and the parts' sums meet in shared memory in a fixed order.
// Ends in every case: waits are bounded, and a CTA that gave up still meets the others.
__global__ void __launch_bounds__(kMxThreads, 1) mx_gemm_kernel(const __grid_constant__ MxParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + p.stages * p.stage_bytes), *empty = full + kMxMaxStages, *done = empty + kMxMaxStages;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(done + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile = blockIdx.x / p.split, rank = blockIdx.x - tile * p.split;
    const int mt = tile % p.m_tiles, nt = tile / p.m_tiles;
    const int u0 = (int)((int64_t)p.units * rank / p.split), u1 = (int)((int64_t)p.units * (rank + 1) / p.split);
    const int count = u1 - u0;
    constexpr int kABytes = mx_unit_bytes(kMxTile);
    const int b_bytes = mx_unit_bytes(p.bn);

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
    if (warp == 4) {
        // ---- operand tiles ----
        if (lane == 0) {
            const uint8_t *w = p.w + ((int64_t)nt * p.units + u0) * kABytes, *a = p.a + ((int64_t)mt * p.units + u0) * b_bytes;
            const int first = count < p.stages ? count : p.stages;
            for (int i = 0; i < first; ++i) {
                mbar_arrive_expect_tx(&full[i], (uint32_t)(kABytes + b_bytes));
                bulk_g2s(smem + i * p.stage_bytes, w + (int64_t)i * kABytes, kABytes, &full[i]);
            }
            wait_predecessor();  // the activation image is there
            for (int i = 0; i < first; ++i) bulk_g2s(smem + i * p.stage_bytes + kABytes, a + (int64_t)i * b_bytes, (uint32_t)b_bytes, &full[i]);
            int s = 0;
            uint32_t par = 0;
            for (int i = first; i < count; ++i) {
                if (!mbar_wait_abortable<32>(&empty[s], par, abort_flag)) break;
                mbar_arrive_expect_tx(&full[s], (uint32_t)(kABytes + b_bytes));
                bulk_g2s(smem + s * p.stage_bytes, w + (int64_t)i * kABytes, kABytes, &full[s]);
                bulk_g2s(smem + s * p.stage_bytes + kABytes, a + (int64_t)i * b_bytes, (uint32_t)b_bytes, &full[s]);
                if (++s == p.stages) {
                    s = 0;
                    par ^= 1;
                }
            }
        }
        __syncwarp();
    } else if (warp == 5) {
        // ---- MMA ----
        // Tensor memory is taken only once the kernel before has finished: one that has yet to take all of it may still be starting.
        wait_predecessor();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)p.tmem_cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        asm volatile("bar.sync 1, 160;" ::: "memory");  // with the epilogue warps
        const uint32_t tmem = *tmem_slot;
        if (elect_one()) {
            const uint32_t sfa = tmem + (uint32_t)((p.bn + 31) / 32 * 32), sfb = sfa + 8;
            const int groups = (p.bn + 127) / 128;
            // E2M1 both, E8M0 scales, K-major both, N, M = 128
            const uint32_t idesc = (1u << 7) | (1u << 10) | ((uint32_t)(p.bn >> 3) << 17) | (1u << 23) | (1u << 27);
            const uint32_t base = smem_u32(smem);
            bool ok = true;
            int s = 0;
            uint32_t par = 0;
            for (int i = 0; i < count; ++i) {
                ok = mbar_wait_abortable<0>(&full[s], par, abort_flag);
                if (!ok) break;
                tc_fence_after();
                const uint32_t at = base + (uint32_t)(s * p.stage_bytes), bt = at + kABytes;
                const uint32_t sa = umma_desc_lo(at + kMxTile * 128, 128), sb = umma_desc_lo(bt + (uint32_t)p.bn * 128, 128);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    copy_scales(sfa + 4 * j, sa + j * (512 >> 4));
                    for (int g = 0; g < groups; ++g) copy_scales(sfb + (uint32_t)(j * 4 * groups + 4 * g), sb + (uint32_t)((g * 1024 + j * 512) >> 4));
                }
                const uint32_t a_lo = umma_desc_lo(at, 16), b_lo = umma_desc_lo(bt, 16);
#pragma unroll
                for (int j = 0; j < 4; ++j) {  // 64 elements: 32 bytes along the swizzled rows
                    const uint32_t ids = (j & 1) ? (2u << 4) | (2u << 29) : 0u;
                    umma_mxf4(tmem, a_lo + 2 * j, b_lo + 2 * j, idesc | ids, sfa + 4 * (j >> 1), sfb + (uint32_t)((j >> 1) * 4 * groups),
                              i > 0 || j > 0 ? 1u : 0u);
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
    }
    // ---- epilogue ----
    if (warp < 4) {
        wait_predecessor();  // the time limit of the wait below counts from here
        asm volatile("bar.sync 1, 160;" ::: "memory");
        const bool ok = mbar_wait_abortable<64>(done, 0, abort_flag);
        tc_fence_after();
        const uint32_t tmem = *tmem_slot + ((uint32_t)(warp * 32) << 16);
        const int r = warp * 32 + lane;
        const int64_t n = (int64_t)nt * kMxTile + r;
        if (!ok) {
            // nothing to read or store
        } else if (p.split == 1) {
            for (int c0 = 0; c0 < p.bn; c0 += 16) {
                uint32_t v[16];
                tmem_ld16(tmem + (uint32_t)c0, v);
                tmem_ld_wait();
                loaded(v);
                const int left = p.m - (mt * p.bn + c0);  // rows of x
                if (n < p.n)
                    with_y_type(p.y, p.y_type, [&](auto *y) {
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (j < left) put_y(y, ((int64_t)mt * p.bn + c0 + j) * p.ldy + n, __uint_as_float(v[j]));
                    });
            }
        } else {
            float *part = reinterpret_cast<float *>(smem);  // [bn][128]; every copy and MMA has finished with the stages
            for (int c0 = 0; c0 < p.bn; c0 += 16) {
                uint32_t v[16];
                tmem_ld16(tmem + (uint32_t)c0, v);
                tmem_ld_wait();
                loaded(v);
#pragma unroll
                for (int j = 0; j < 16; ++j) part[(c0 + j) * kMxTile + r] = __uint_as_float(v[j]);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 5) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot), "r"((uint32_t)p.tmem_cols));
    }
    if (p.split > 1) {
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        const int rows = min(p.bn, p.m - mt * p.bn);
        const int c0 = rows * rank / p.split, c1 = rows * (rank + 1) / p.split;
        const uint32_t part = smem_u32(smem);
        with_y_type(p.y, p.y_type, [&](auto *y) {
            for (int i = c0 * kMxTile + threadIdx.x; i < c1 * kMxTile; i += kMxThreads) {
                const int64_t n = (int64_t)nt * kMxTile + (i & (kMxTile - 1));
                float sum = 0.0f;
                for (int q = 0; q < p.split; ++q) sum += ld_cluster(part + 4u * (uint32_t)i, q);
                if (n < p.n) put_y(y, ((int64_t)mt * p.bn + (i >> 7)) * p.ldy + n, sum);
            }
        });
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
constexpr int kPairStages = 6;
constexpr int kPairEpiWarps = 8;
constexpr int kPairThreads = 32 * (kPairEpiWarps + 2);

struct MxPairParams {
    CUtensorMap w, codes, scales;  // boxes of a unit's rows of 128 bytes: of weights; of half of the activations' codes; of their scales
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
    uint64_t *acc_full = empty + kPairStages, *acc_empty = acc_full + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + 2);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x & 1;
    const int tiles = (p.n_tiles + 1) / 2 * p.m_tiles, first = blockIdx.x >> 1, step = gridDim.x >> 1;
    constexpr int kABytes = mx_unit_bytes(kMxTile);
    const int half = p.bn / 2 * 128, scales = mx_scale_bytes(p.bn), unit_rows = p.bn + scales / 128;

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
                int w = nt * p.units * (kABytes / 128), a = mt * p.units * unit_rows;  // rows of 128 bytes
                for (int u = 0; u < p.units; ++u) {
                    if (fill >= p.stages) {
                        ok = mbar_wait_abortable<0>(&empty[s], par, abort_flag);
                        if (!ok) break;
                    } else {
                        ++fill;
                    }
                    uint8_t *dst = smem + s * p.stage_bytes;
                    const uint32_t bar = full0 + 8u * (uint32_t)s;
                    if (rank == 0) mbar_arrive_expect_tx(&full[s], (uint32_t)(2 * (kABytes + half + scales)));
                    copy_rows(dst, &p.w, w, bar);
                    copy_rows(dst + kABytes, &p.codes, a + rank * (p.bn / 2), bar);
                    copy_rows(dst + kABytes + half, &p.scales, a + p.bn, bar);
                    w += kABytes / 128;
                    a += unit_rows;
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
        if (rank == 0 && elect_one()) {
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
                    const int row = mt * p.bn + c, left = p.m - row;
                    auto *at = y + (int64_t)row * p.ldy + n;
                    if (n < p.n) {
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (j < left) put_y(at + (int64_t)j * p.ldy, 0, __uint_as_float(v[j]));
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

int64_t mx_image_bytes(int64_t rows, int64_t k, int T) { return (rows + T - 1) / T * mx_units(k) * mx_unit_bytes(T); }

int launch_mx_quantize(const void *x, int x_type, int64_t m, int64_t k, int T, uint8_t *image, bool trigger, bool overlap,
                       cudaStream_t stream) {
    const int64_t rows = (m + T - 1) / T * T, grid = ceil_div64(rows * mx_units(k), 8);
    if (grid > 0x7fffffff) return LLOOM_ERR_SHAPE;
    return launch_status(launch_early(mx_quantize_kernel, (unsigned)grid, 256, 0, overlap, stream, x, x_type, m, (int)k, (int)mx_units(k), T, rows,
                                      image, trigger ? 1 : 0));
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

struct MxPlan {
    bool pairs;
    MxTiles tiles;
};
MxPlan mx_plan(int64_t m, int64_t n, int64_t k, int sms) {
    MxPlan pl;
    pl.pairs = m > 128;
    pl.tiles = pl.pairs ? mx_pair_tiles(m, n, sms / 2) : mx_tiles(m, (m + 255) / 256);
    return pl;
}
// Bytes of the activation image, whatever the device's plan: the largest of all tile widths
int64_t mx_act_bytes(int64_t m, int64_t k) {
    int64_t most = 0;
    for (int T = 16; T <= 256; T += 16) most = std::max(most, (m + T - 1) / T * mx_unit_bytes(T));
    return most * mx_units(k);
}

struct MxSmemOnce {
    std::mutex mu;
    bool done[64] = {false};
};

template <class Params>
int launch_mx_gemm(void (*kern)(Params), MxSmemOnce &once, const Params &p, int ctas, int cluster, int threads, cudaStream_t stream) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || dev < 0 || dev >= 64) return LLOOM_ERR_DEVICE;
    const int smem = p.stages * p.stage_bytes + 256 + 1024;
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
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
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
    // The product starts on the weights while this kernel runs, so it is not launched early itself unless they are in place.
    rc = launch_mx_quantize(x, x_type, m, k, t.bn, (uint8_t *)workspace, true, overlap, (cudaStream_t)stream);
    if (rc != LLOOM_OK) return rc;
    const int64_t n_tiles = (n + kMxTile - 1) / kMxTile;
    const int units = (int)mx_units(k);
    if (pl.pairs) {
        static MxSmemOnce once;
        MxPairParams p = {};
        const int64_t w_rows = mx_image_bytes(n, k, kMxTile) / 128, a_rows = mx_image_bytes(m, k, t.bn) / 128;
        if (w_rows > 0x7fffffff || a_rows > 0x7fffffff) return LLOOM_ERR_SHAPE;  // 256 GB
        if (!encode_rows_map(p.w, image, w_rows, 128, 128, mx_unit_bytes(kMxTile) / 128) || !encode_rows_map(p.codes, workspace, a_rows, 128, 128, t.bn / 2) ||
            !encode_rows_map(p.scales, workspace, a_rows, 128, 128, mx_scale_bytes(t.bn) / 128))
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
        return launch_mx_gemm(mx_gemm_pair_kernel, once, p, 2 * pairs, 2, kPairThreads, (cudaStream_t)stream);
    }
    static MxSmemOnce once;
    MxParams p = {};
    p.w = (const uint8_t *)image;
    p.a = (const uint8_t *)workspace;
    p.y = y;
    p.y_type = y_type;
    p.ldy = ldy;
    p.m = (int)m;
    p.n = (int)n;
    p.units = units;
    p.bn = t.bn;
    p.m_tiles = t.count;
    const int64_t tiles = n_tiles * t.count;
    p.split = 1;
    while (p.split < 8 && tiles * p.split * 2 <= di.sm_count && p.units >= p.split * 2) p.split *= 2;
    if (tiles * p.split > 0x7fffffff) return LLOOM_ERR_SHAPE;
    p.stage_bytes = mx_unit_bytes(kMxTile) + mx_unit_bytes(t.bn);
    p.stages = (di.max_smem_optin - 256 - 1024) / p.stage_bytes;
    if (p.stages > kMxMaxStages) p.stages = kMxMaxStages;
    const int cols = (t.bn + 31) / 32 * 32 + 8 + 8 * ((t.bn + 127) / 128);
    for (p.tmem_cols = 32; p.tmem_cols < cols; p.tmem_cols *= 2) {}
    return launch_mx_gemm(mx_gemm_kernel, once, p, (int)(tiles * p.split), p.split, kMxThreads, (cudaStream_t)stream);
}

int mx_quantize(const void *x, int x_type, int64_t rows, int64_t k, void *image, int64_t image_bytes, void *stream, bool overlap) {
    const int rc = mx_check(1, rows, k);
    if (rc != LLOOM_OK) return rc;
    if (!elem_type_ok(x_type)) return LLOOM_ERR_DTYPE;
    if (!x || !image) return LLOOM_ERR_NULL;
    if (image_bytes < mx_image_bytes(rows, k, kMxTile)) return LLOOM_ERR_WORKSPACE;
    if (!aligned(x, 16) || !aligned(image, 256)) return LLOOM_ERR_ALIGN;
    return launch_mx_quantize(x, x_type, rows, k, kMxTile, (uint8_t *)image, false, overlap, (cudaStream_t)stream);
}

int mx_dequantize(const void *image, int64_t rows, int64_t k, void *out, bool f16, void *stream, bool overlap) {
    const int rc = mx_check(1, rows, k);
    if (rc != LLOOM_OK) return rc;
    if (!image || !out) return LLOOM_ERR_NULL;
    if (!aligned(image, 256) || !aligned(out, 16)) return LLOOM_ERR_ALIGN;
    const int64_t grid = ceil_div64(rows * (k / 8), 256);
    if (grid > 0x7fffffff) return LLOOM_ERR_SHAPE;
    return launch_status(launch_early(f16 ? mx_dequantize_kernel<true> : mx_dequantize_kernel<false>, (unsigned)grid, 256, 0, overlap,
                                      (cudaStream_t)stream, (const uint8_t *)image, rows, (int)k, (int)mx_units(k), out));
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
