// 8-bit floating point with a power-of-two scale for each block of 128: casts and the scaled matrix product.
//
// A value x of block b is held as q 2^e(b): e is the smallest integer >= -126 with amax(b) <= fmax 2^e over the
// block's finite values (fmax 448 for e4m3, 57344 for e5m2; e = 0 for a block of zeros), q = x 2^-e rounded to
// the nearest 8-bit value (ties to even).  Scales are bytes e + 127, the form the tensor core's block-scaled
// MMA takes (UE8M0), so products need no scaling pass: the hardware multiplies each 32-element dot product by
// 2^(ea + eb) and accumulates in FP32.  A power of two costs no precision against an arbitrary FP32 scale: it
// moves the block inside the format's exponent range and rounds nothing.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <stdexcept>
#include <string>

#include "kernels.h"

namespace sy {

namespace {

// ------------------------------------------------------------------ casts

__device__ __forceinline__ float load_f(const float* p) { return *p; }
__device__ __forceinline__ float load_f(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_f(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void store_f(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_f(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_f(__half* p, float v) { *p = __float2half_rn(v); }

__device__ __forceinline__ void unpack(uint4 u, const __nv_bfloat16*, float* v) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void unpack(uint4 u, const __half*, float* v) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void unpack(uint4 u, const float*, float* v) {
    v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y), v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
}

// 16 consecutive values of a row from column c; columns at and past `cols` read as zero.
template <class T>
__device__ __forceinline__ void load16(const T* row, int c, int cols, bool vec, float* v) {
    if (vec && c + 16 <= cols) {
        constexpr int kPer = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 16 / kPer; i++)
            unpack(__ldg(reinterpret_cast<const uint4*>(row + c) + i), row, v + i * kPer);
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = c + i < cols ? load_f(row + c + i) : 0.0f;
    }
}

// |v| of finite values, 0 for the others
__device__ __forceinline__ float finite_size(float v) {
    const float a = fabsf(v);
    return a <= 3.402823466e38f ? a : 0.0f;
}

// Smallest e >= -126 with amax <= fmax 2^e.  fmax = 0.875 * 2^top (top 9 for e4m3, 16 for e5m2), so with
// amax = f 2^x, f in [0.5, 1): e = x - top, plus one where f > 0.875.
__device__ __forceinline__ int block_exponent(float amax, int top) {
    if (amax == 0.0f) return 0;
    int x;
    const float f = frexpf(amax, &x);
    return max(x - top + (f > 0.875f ? 1 : 0), -126);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

template <bool E5M2>
__device__ __forceinline__ uint32_t cvt2(float lo, float hi) {
    uint16_t r;
    if (E5M2)
        asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    else
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// The conversion saturates: an infinity, which no scale brings into range, becomes the format's infinity
// (e5m2) or, as e4m3 has none, NaN.
template <bool E5M2>
__device__ __forceinline__ uint32_t cvt4(const float* v, float s) {
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = v[i] * s;
    uint32_t w = cvt2<E5M2>(x[0], x[1]) | cvt2<E5M2>(x[2], x[3]) << 16;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (isinf(v[i])) {
            const uint32_t b = (E5M2 ? 0x7cu : 0x7fu) | (v[i] < 0.0f ? 0x80u : 0u);
            w = (w & ~(0xffu << (8 * i))) | b << (8 * i);
        }
    return w;
}

struct CastParams {
    const void* x;
    long pitch;          // elements between rows of x
    int rows, cols;
    uint8_t *q, *scale, *qt, *scale_t;
    int qp, sp, qtp, stp;   // row pitches in bytes: q, scale, and of the transposed copies
    int vec;             // rows of x are 16-byte aligned
    int block_rows;      // 1 or 128
};

// Blocks of 1 x 128 without the transposed copy: eight threads per block, 16 values each, the block's maximum
// by three shuffles.  One read, one write, no shared memory.
template <class T, bool E5M2>
__global__ void __launch_bounds__(256) cast_rows_kernel(CastParams p) {
    const uint32_t kb = (p.cols + 127) / 128;
    const uint32_t unit = blockIdx.x * 32u + (threadIdx.x >> 3);
    const uint32_t row = unit / kb, b = unit - row * kb;
    const bool live = row < (uint32_t)p.rows;
    const int c = b * 128 + (threadIdx.x & 7) * 16;
    float v[16];
    if (live)
        load16(static_cast<const T*>(p.x) + row * p.pitch, c, p.cols, p.vec, v);
    else
        for (int i = 0; i < 16; i++) v[i] = 0.0f;
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i++) amax = fmaxf(amax, finite_size(v[i]));
#pragma unroll
    for (int o = 4; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (!live) return;
    const int e = block_exponent(amax, E5M2 ? 16 : 9);
    const float s = pow2(-e);
    if (c < p.qp) {
        uint4 w;
        w.x = cvt4<E5M2>(v, s), w.y = cvt4<E5M2>(v + 4, s), w.z = cvt4<E5M2>(v + 8, s), w.w = cvt4<E5M2>(v + 12, s);
        *reinterpret_cast<uint4*>(p.q + (long)row * p.qp + c) = w;
    }
    if ((threadIdx.x & 7) == 0) p.scale[(long)row * p.sp + b] = (uint8_t)(e + 127);
}

// One CTA per 128 x 128 tile, for blocks of 128 x 128 and for the transposed copy: x is read once, both
// orientations leave from registers.  Thread t holds columns 16 (t % 8) .. + 15 of the four rows 4 (t / 8) ..
// + 3, so the four bytes of a transposed word are its own.  The transposed bytes pass through shared memory:
// word (column, row / 4) at column * 32 + (row / 4 ^ 4 (column / 16)), where the 32 lanes of a store and the
// 16-byte groups of a read fall into different banks.
template <class T, bool E5M2>
__global__ void __launch_bounds__(256) cast_tile_kernel(CastParams p) {
    __shared__ uint32_t smax[128];            // column maxima (bits of non-negative floats order as integers)
    __shared__ uint32_t smax_tile;
    __shared__ __align__(16) uint32_t tile[128 * 32];
    const int t = threadIdx.x, seg = t & 7, rw = t >> 3;
    const int b = blockIdx.x % ((p.cols + 127) / 128), rb = blockIdx.x / ((p.cols + 127) / 128);
    const int c = b * 128 + seg * 16, r0 = rb * 128 + rw * 4;
    constexpr int kTop = E5M2 ? 16 : 9;
    if (t < 128) smax[t] = 0;
    if (t == 0) smax_tile = 0;
    float v[4][16];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (r0 + i < p.rows)
            load16(static_cast<const T*>(p.x) + (r0 + i) * p.pitch, c, p.cols, p.vec, v[i]);
        else
#pragma unroll
            for (int j = 0; j < 16; j++) v[i][j] = 0.0f;
    }
    __syncthreads();
    float rmax[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        rmax[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < 16; j++) rmax[i] = fmaxf(rmax[i], finite_size(v[i][j]));
#pragma unroll
        for (int o = 4; o; o >>= 1) rmax[i] = fmaxf(rmax[i], __shfl_xor_sync(0xffffffffu, rmax[i], o));
    }
    int e_tile = 0;
    if (p.block_rows == 128) {
        if (seg == 0)
            atomicMax(&smax_tile, __float_as_uint(fmaxf(fmaxf(rmax[0], rmax[1]), fmaxf(rmax[2], rmax[3]))));
        __syncthreads();
        e_tile = block_exponent(__uint_as_float(smax_tile), kTop);
        if (t == 0) {
            p.scale[(long)rb * p.sp + b] = (uint8_t)(e_tile + 127);
            if (p.qt) p.scale_t[(long)b * p.stp + rb] = (uint8_t)(e_tile + 127);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (r0 + i >= p.rows) continue;
        const int e = p.block_rows == 128 ? e_tile : block_exponent(rmax[i], kTop);
        const float s = pow2(-e);
        if (c < p.qp) {
            uint4 w;
            w.x = cvt4<E5M2>(v[i], s), w.y = cvt4<E5M2>(v[i] + 4, s), w.z = cvt4<E5M2>(v[i] + 8, s),
            w.w = cvt4<E5M2>(v[i] + 12, s);
            *reinterpret_cast<uint4*>(p.q + (long)(r0 + i) * p.qp + c) = w;
        }
        if (p.block_rows == 1 && seg == 0) p.scale[(long)(r0 + i) * p.sp + b] = (uint8_t)(e + 127);
    }
    if (!p.qt) return;
    if (p.block_rows == 1) {
#pragma unroll
        for (int j = 0; j < 16; j++) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) m = fmaxf(m, finite_size(v[i][j]));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
            if ((t & 31) < 8) atomicMax(&smax[seg * 16 + j], __float_as_uint(m));
        }
        __syncthreads();
        if (t < 128 && b * 128 + t < p.cols)
            p.scale_t[(long)(b * 128 + t) * p.stp + rb] =
                (uint8_t)(block_exponent(__uint_as_float(smax[t]), kTop) + 127);
    }
#pragma unroll
    for (int j = 0; j < 16; j++) {
        const int e = p.block_rows == 128 ? e_tile : block_exponent(__uint_as_float(smax[seg * 16 + j]), kTop);
        const float col[4] = {v[0][j], v[1][j], v[2][j], v[3][j]};
        tile[(seg * 16 + j) * 32 + (rw ^ (seg << 2))] = cvt4<E5M2>(col, pow2(-e));
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int idx = t + i * 256, col = idx >> 3, chunk = idx & 7;
        if (b * 128 + col < p.cols && rb * 128 + chunk * 16 < p.qtp)
            *reinterpret_cast<uint4*>(p.qt + (long)(b * 128 + col) * p.qtp + rb * 128 + chunk * 16) =
                reinterpret_cast<const uint4*>(tile)[col * 8 + (chunk ^ (col >> 4))];
    }
}

// UE8M0: 2^(s - 127); 0 is 2^-127 (a subnormal float), 255 is NaN
__device__ __forceinline__ float scale_value(uint32_t s) {
    return __uint_as_float(s == 0 ? 0x00400000u : s == 255 ? 0x7fffffffu : s << 23);
}

template <class T, bool E5M2>
__global__ void __launch_bounds__(256)
    uncast_kernel(const uint8_t* q, const uint8_t* scale, int rows, int cols, int qp, int sp, int row_shift, T* out,
                  long pitch, int vec) {
    const uint32_t per = (cols + 15) / 16;
    const uint32_t unit = blockIdx.x * 256u + threadIdx.x;
    const uint32_t row = unit / per;
    const int c = (unit - row * per) * 16;
    if (row >= (uint32_t)rows) return;
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(q + (long)row * qp + c));
    const float s = scale_value(__ldg(scale + (long)(row >> row_shift) * sp + (c >> 7)));
    const uint32_t word[4] = {w.x, w.y, w.z, w.w};
    __align__(16) T o[16];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const __nv_fp8x2_storage_t pair = (__nv_fp8x2_storage_t)(word[i >> 1] >> (16 * (i & 1)));
        const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(pair, E5M2 ? __NV_E5M2 : __NV_E4M3)));
        store_f(&o[2 * i], f.x * s);
        store_f(&o[2 * i + 1], f.y * s);
    }
    T* dst = out + row * pitch + c;
    if (vec && c + 16 <= cols) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); i++)
            reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(o)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++)
            if (c + i < cols) dst[i] = o[i];
    }
}

// ------------------------------------------------------------------ product

constexpr int kTileRows = 128, kBlockK = 128;
constexpr int kScaleSlots = 4;   // groups of four K blocks whose scale words are in flight
// Warps: 0, 8 and 9 TMA, 1 MMA, 2 scales, 3 MMA-side waits, 4-7 epilogue.
constexpr int kThreads = 320, kProducers = 3;
constexpr int kStageBar = 1;     // named barrier: a stage is loaded (the waiting warp and the MMA warp)

struct ProductParams {
    int rows[2];                 // [0] the MMA's M side, [1] its N side
    const uint8_t* scale[2];
    int sp[2], shift[2];         // scale pitch in bytes; log2 of the rows that share a scale
    int kblocks;
    int tiles_m, tiles_n, splits;
    uint32_t idesc;
    void* out;
    long pitch;
    int out_type, accumulate, swap, vec;   // swap: M side indexes the output's columns
    int* status;
};

template <int BN>
struct ProductShape {
    static constexpr int kScaleRows = (BN + 127) / 128;              // N-side scale atoms of 128 rows
    static constexpr int kStageBytes = (kTileRows + BN) * kBlockK;
    static constexpr int kStages = BN == 256 ? 4 : BN == 128 ? 6 : 8;
    static constexpr int kScaleBytes = 512 * (1 + kScaleRows);
    static constexpr int kScaleCols = 4 * (1 + kScaleRows);
    static constexpr int kCols = BN + kScaleSlots * kScaleCols;
    static constexpr int kTmemCols = kCols <= 64 ? 64 : kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
    static constexpr int kBarriers = 2 * kStages + 2 * kScaleSlots + 1;
    static constexpr int kSmem = 1024 + kStages * kStageBytes + kScaleSlots * kScaleBytes + kBarriers * 8 + 16;
    // the split sum's partial tile lies over the stages: BN columns of 129 floats
    static_assert(BN * 129 * 4 <= kStages * kStageBytes, "partial tile exceeds the stages");
};

__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer_addr(addr, rank)) : "memory");
    return v;
}

__device__ __forceinline__ void put(const ProductParams& p, int i, int j, float v) {
    const long at = p.swap ? j * p.pitch + i : i * p.pitch + j;
    if (p.out_type == kTypeF32) {
        float* o = static_cast<float*>(p.out) + at;
        *o = p.accumulate ? *o + v : v;
    } else if (p.out_type == kTypeBF16) {
        static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
    } else {
        static_cast<__half*>(p.out)[at] = __float2half_rn(v);
    }
}

// 32 consecutive columns of output row i in 16-byte pieces
__device__ __forceinline__ void put_row32(const ProductParams& p, int i, int j, const float* v) {
    if (p.out_type == kTypeF32) {
        float4* o = reinterpret_cast<float4*>(static_cast<float*>(p.out) + i * p.pitch + j);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            float4 f = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
            if (p.accumulate) {
                const float4 c = o[k];
                f.x += c.x, f.y += c.y, f.z += c.z, f.w += c.w;
            }
            o[k] = f;
        }
        return;
    }
    uint4* o = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + i * p.pitch + j);
#pragma unroll
    for (int k = 0; k < 4; k++) {
        uint32_t w[4];
#pragma unroll
        for (int l = 0; l < 4; l++) {
            const float a = v[8 * k + 2 * l], b = v[8 * k + 2 * l + 1];
            if (p.out_type == kTypeBF16) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
                w[l] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __half2 h = __floats2half2_rn(a, b);
                w[l] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        o[k] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// c = a b^T on 128 x BN tiles, one CTA per tile and K split.  Both operands stream through shared memory in
// blocks of 128 along K (one scale per row and block, 128-byte swizzled rows); one warp issues four
// 128 x BN x 32 block-scaled MMAs per block and touches no shared memory itself: a warp that has MMAs in flight
// waits ~1,200 cycles for any shared-memory access, an mbarrier wait included, so another warp does its waiting.  A warp gathers the rows' scale words (four K blocks each) into
// 512-byte atoms, which the MMA thread copies to TMEM ahead of the MMAs that use them.  K splits form a cluster:
// each CTA leaves its partial tile in its shared memory and sums a share of the tile over the cluster in rank
// order, so the result does not depend on timing and no workspace is needed.
template <int BN>
__global__ void __launch_bounds__(kThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                   const ProductParams p) {
    using S = ProductShape<BN>;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    uint8_t* ssm = smem + S::kStages * S::kStageBytes;
    uint64_t* bars = reinterpret_cast<uint64_t*>(ssm + kScaleSlots * S::kScaleBytes);
    uint64_t *full = bars, *empty = bars + S::kStages, *sfull = bars + 2 * S::kStages, *sempty = sfull + kScaleSlots;
    uint64_t* done = sempty + kScaleSlots;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // tile order: bands of 12 row tiles, so that the CTAs of a wave share rows of both operands in L2
    const int band = 12 * p.tiles_n, in_band = blockIdx.x % band, m_first = blockIdx.x / band * 12;
    const int band_m = min(12, p.tiles_m - m_first);
    const int m0 = (m_first + in_band % band_m) * kTileRows, n0 = in_band / band_m * BN;
    const int split = blockIdx.y;
    const int k0 = (int)((long)p.kblocks * split / p.splits), k1 = (int)((long)p.kblocks * (split + 1) / p.splits);

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < kScaleSlots; s++) {
            mbar_init(&sfull[s], 32);
            mbar_init(&sempty[s], 1);
        }
        mbar_init(done, 1);
        fence_barrier_init();
    }
    if (warp == 3) {
        tmem_alloc(tmem_slot, S::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0 || warp >= 8) {
        // The producers take turns.  A wait after a bulk copy holds a thread for ~1,000 cycles, whatever it waits for, more
        // than a stage's copies or MMAs take.  The first stages are free and need no wait.
        if (lane == 0) {
            const int mine = warp ? warp - 7 : 0;
            int i = mine;
            for (; i < k1 - k0; i += kProducers) {
                const int s = i % S::kStages;
                if (i >= S::kStages && !mbar_wait(&empty[s], ((i / S::kStages) & 1) ^ 1, p.status, kStatusWait)) break;
                uint8_t* st = smem + s * S::kStageBytes;
                mbar_arrive_expect_tx(&full[s], S::kStageBytes);
                tma_load_2d(st, &tm_a, &full[s], (k0 + i) * kBlockK, m0);
                tma_load_2d(st + kTileRows * kBlockK, &tm_b, &full[s], (k0 + i) * kBlockK, n0);
            }
            // No copy is in flight when the CTA ends, even after a wait that gave up.  Only the last use of a stage is
            // waited for: the barrier of an earlier one may have moved on by two phases.
            for (int j = mine; j < min(i, k1 - k0); j += kProducers)
                if (j + S::kStages >= k1 - k0) mbar_wait(&full[j % S::kStages], (j / S::kStages) & 1, p.status, kStatusWait);
        }
    } else if (warp == 3) {
        // every wait of the MMA side; after one that gave up the hand-offs go on, so that every warp finishes
        bool live = true;
        for (int i = 0, group = 0; i < k1 - k0; i++) {
            const int s = i % S::kStages, kb = k0 + i;
            if (live && (i == 0 || (kb & 3) == 0))
                live = mbar_wait(&sfull[group % kScaleSlots], (group / kScaleSlots) & 1, p.status, kStatusWait);
            if (live) live = mbar_wait(&full[s], (i / S::kStages) & 1, p.status, kStatusWait);
            if ((kb & 3) == 3) group++;
            named_bar_sync(kStageBar, 64);
        }
    } else if (warp == 1) {
        const uint32_t st0 = smem_u32(smem), sc0 = smem_u32(ssm);
        int group = 0;
        for (int i = 0; i < k1 - k0; i++) {
            const int s = i % S::kStages, kb = k0 + i, slot = group % kScaleSlots;
            const uint32_t tsc = tmem + BN + slot * S::kScaleCols;
            named_bar_sync(kStageBar, 64);   // stage (and its scales) loaded
            tc_fence_after();
            if (i == 0 || (kb & 3) == 0)
#pragma unroll
                for (int a = 0; a < 1 + S::kScaleRows; a++)
                    tmem_cp_scales_elect(tsc + 4 * a,
                                         smem_desc(sc0 + slot * S::kScaleBytes + a * 512, 0, 128, kLayoutNone));
            const uint64_t da = smem_desc(st0 + s * S::kStageBytes, 0, 1024, kLayoutSw128);
            const uint64_t db = smem_desc(st0 + s * S::kStageBytes + kTileRows * kBlockK, 0, 1024, kLayoutSw128);
            const uint32_t idesc = p.idesc | (uint32_t)(kb & 3) << 4 | (uint32_t)(kb & 3) << 29;
#pragma unroll
            for (int k = 0; k < kBlockK / 32; k++)
                mma_mxf8_elect(tmem, da + 2 * k, db + 2 * k, idesc, tsc, tsc + 4, (i | k) != 0);
            mma_commit_elect(&empty[s]);
            if ((kb & 3) == 3) {
                mma_commit_elect(&sempty[slot]);
                group++;
            }
        }
        mma_commit_elect(done);
    } else if (warp == 2) {
        // lane l gathers rows l, l + 32, l + 64, l + 96: the four words of 16-byte row l of the atom
        const int g0 = k0 >> 2, g1 = (k1 + 3) >> 2;
        for (int g = g0; g < g1; g++) {
            const int i = g - g0, slot = i % kScaleSlots;
            uint4 w[1 + S::kScaleRows];
#pragma unroll
            for (int a = 0; a < 1 + S::kScaleRows; a++) {
                const int side = a > 0, first = side ? n0 + (a - 1) * 128 : m0;
                uint32_t x[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int r = first + lane + 32 * j;
                    x[j] = r < p.rows[side]
                               ? __ldg(reinterpret_cast<const uint32_t*>(
                                           p.scale[side] + (long)(r >> p.shift[side]) * p.sp[side]) + g)
                               : 0u;
                }
                w[a] = make_uint4(x[0], x[1], x[2], x[3]);
            }
            if (!mbar_wait(&sempty[slot], ((i / kScaleSlots) & 1) ^ 1, p.status, kStatusWait)) break;
#pragma unroll
            for (int a = 0; a < 1 + S::kScaleRows; a++)
                *reinterpret_cast<uint4*>(ssm + slot * S::kScaleBytes + a * 512 + lane * 16) = w[a];
            fence_proxy_async();
            mbar_arrive(&sfull[slot]);
        }
    }
    __syncwarp();
    if (warp >= 4 && warp < 8) {
        const int q = warp & 3, r = q * 32 + lane, i = m0 + r;
        mbar_wait(done, 0, p.status, kStatusWait);
        tc_fence_after();
        float* part = reinterpret_cast<float*>(smem);
#pragma unroll 1
        for (int c = 0; c < BN; c += 32) {
            float v[32];
            if (BN % 32 == 0) {
                tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + c, v);
            } else {
                tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + c, v);
            }
            constexpr int kPer = BN % 32 == 0 ? 32 : 16;
            if (p.splits > 1) {
#pragma unroll
                for (int k = 0; k < kPer; k++) part[(c + k) * 129 + r] = v[k];
            } else if (i < p.rows[0]) {
                const int j = n0 + c;
                if (kPer == 32 && p.vec && j + 32 <= p.rows[1]) {
                    put_row32(p, i, j, v);
                } else {
#pragma unroll
                    for (int k = 0; k < kPer; k++)
                        if (j + k < p.rows[1]) put(p, i, j + k, v[k]);
                }
            }
        }
        tc_fence_before();
    }
    if (p.splits > 1) {
        cluster_sync_all();
        const int share = kTileRows / p.splits, first = split * share;
        const uint32_t part = smem_u32(smem);
        for (int idx = threadIdx.x; idx < share * BN; idx += kThreads) {
            const int r = first + (p.swap ? idx % share : idx / BN), c = p.swap ? idx / share : idx % BN;
            if (m0 + r >= p.rows[0] || n0 + c >= p.rows[1]) continue;
            float v = 0.0f;
            for (int s = 0; s < p.splits; s++) v += ld_cluster(part + (c * 129 + r) * 4, s);
            put(p, m0 + r, n0 + c, v);
        }
        cluster_sync_all();   // a peer may still read this CTA's partial tile
    } else {
        __syncthreads();
    }
    if (warp == 3) {
        tc_fence_after();
        tmem_dealloc(tmem, S::kTmemCols);
    }
}

__global__ void fill_zero_kernel(ProductParams p) {
    const long n = (long)p.rows[0] * p.rows[1];
    for (long i = blockIdx.x * (long)blockDim.x + threadIdx.x; i < n; i += (long)gridDim.x * blockDim.x)
        put(p, (int)(i / p.rows[1]), (int)(i % p.rows[1]), 0.0f);
}

struct Plan {
    int swap, bn, splits;
};

// Tile width, K splits and which operand takes the MMA's 128-row side, by an estimate of the time: a wave of
// CTAs takes a fixed start and end plus, per K block, the longer of its MMAs and of its share of the copies.
Plan plan_product(int m, int n, int kblocks, int sms) {
    Plan best{0, 256, 1};
    double least = 1e30;
    for (int swap = 0; swap < 2; swap++)
        for (int bn : {16, 32, 64, 128, 256})
            for (int splits : {1, 2, 4, 8}) {
                if (splits > 1 && kblocks < 2 * splits) continue;
                const long mt = ((swap ? n : m) + 127L) / 128, nt = ((swap ? m : n) + bn - 1L) / bn;
                const long ctas = mt * nt * splits, waves = (ctas + sms - 1) / sms;
                const double load = (kTileRows + bn) * kBlockK / 100.0 * std::min(1.0, (double)ctas / sms + 0.3);
                const double block = std::max(load, bn * 0.55);   // ns
                const double t = waves * (2500.0 + (splits > 1 ? 800.0 + 4.0 * bn : 6.0 * bn) +
                                          block * ((kblocks + splits - 1) / splits));
                if (t < least) {
                    least = t;
                    best = Plan{swap, bn, splits};
                }
            }
    return best;
}

CUtensorMap operand_map(const uint8_t* q, int rows, int k, int box_rows) {
    CUtensorMap map;
    cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)((k + 15) / 16 * 16)};
    cuuint32_t box[2] = {(cuuint32_t)kBlockK, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r = tensor_map_encoder()(
        &map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(q), dims, strides, box, estr,
        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) throw std::runtime_error("cuTensorMapEncodeTiled failed: " + std::to_string((int)r));
    return map;
}

template <int BN>
void launch_product(const CUtensorMap& ta, const CUtensorMap& tb, const ProductParams& p, cudaStream_t stream) {
    using S = ProductShape<BN>;
    static PerDeviceOnce once;
    once_per_device(once, [] { set_max_dynamic_smem(product_kernel<BN>, S::kSmem, "product_kernel"); });
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(p.tiles_m * p.tiles_n, p.splits);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = S::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = p.splits;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, product_kernel<BN>, ta, tb, p);
    launch_check("product_kernel");
}

template <class T>
void launch_cast(const CastParams& p, bool e5m2, cudaStream_t stream) {
    const long kb = (p.cols + 127) / 128;
    if (p.block_rows == 1 && !p.qt) {
        const unsigned blocks = (unsigned)((p.rows * kb + 31) / 32);
        if (e5m2)
            cast_rows_kernel<T, true><<<blocks, 256, 0, stream>>>(p);
        else
            cast_rows_kernel<T, false><<<blocks, 256, 0, stream>>>(p);
    } else {
        const unsigned blocks = (unsigned)((p.rows + 127L) / 128 * kb);
        if (e5m2)
            cast_tile_kernel<T, true><<<blocks, 256, 0, stream>>>(p);
        else
            cast_tile_kernel<T, false><<<blocks, 256, 0, stream>>>(p);
    }
    launch_check("fp8 cast kernel");
}

template <class T>
void launch_uncast(const uint8_t* q, const uint8_t* scale, int rows, int cols, bool e5m2, int row_shift, T* out,
                   long pitch, cudaStream_t stream) {
    const int vec = reinterpret_cast<uintptr_t>(out) % 16 == 0 && pitch * sizeof(T) % 16 == 0;
    const unsigned blocks = (unsigned)((rows * ((cols + 15L) / 16) + 255) / 256);
    const int qp = (int)fp8_pitch(cols), sp = (int)fp8_scale_pitch(cols);
    if (e5m2)
        uncast_kernel<T, true><<<blocks, 256, 0, stream>>>(q, scale, rows, cols, qp, sp, row_shift, out, pitch, vec);
    else
        uncast_kernel<T, false><<<blocks, 256, 0, stream>>>(q, scale, rows, cols, qp, sp, row_shift, out, pitch, vec);
    launch_check("fp8 uncast kernel");
}

}  // namespace

void fp8_quantize(const void* x, int x_type, long x_pitch, int rows, int cols, bool e5m2, int block_rows, uint8_t* q,
                  uint8_t* scale, uint8_t* qt, uint8_t* scale_t, cudaStream_t stream) {
    if (rows == 0 || cols == 0) return;
    const int elem = x_type == kTypeF32 ? 4 : 2;
    CastParams p{x, x_pitch, rows, cols, q, scale, qt, scale_t, (int)fp8_pitch(cols), (int)fp8_scale_pitch(cols),
                 (int)fp8_pitch(rows), (int)fp8_scale_pitch(rows),
                 reinterpret_cast<uintptr_t>(x) % 16 == 0 && x_pitch * elem % 16 == 0, block_rows};
    if (x_type == kTypeF32)
        launch_cast<float>(p, e5m2, stream);
    else if (x_type == kTypeBF16)
        launch_cast<__nv_bfloat16>(p, e5m2, stream);
    else
        launch_cast<__half>(p, e5m2, stream);
}

void fp8_dequantize(const uint8_t* q, const uint8_t* scale, int rows, int cols, bool e5m2, int block_rows, void* out,
                    int out_type, long out_pitch, cudaStream_t stream) {
    if (rows == 0 || cols == 0) return;
    const int shift = block_rows == 128 ? 7 : 0;
    if (out_type == kTypeF32)
        launch_uncast(q, scale, rows, cols, e5m2, shift, static_cast<float*>(out), out_pitch, stream);
    else if (out_type == kTypeBF16)
        launch_uncast(q, scale, rows, cols, e5m2, shift, static_cast<__nv_bfloat16*>(out), out_pitch, stream);
    else
        launch_uncast(q, scale, rows, cols, e5m2, shift, static_cast<__half*>(out), out_pitch, stream);
}

void fp8_matmul(const Fp8Operand& a, const Fp8Operand& b, int k, void* out, int out_type, long out_pitch,
                bool accumulate, int* status, cudaStream_t stream) {
    if (a.rows == 0 || b.rows == 0) return;
    const int elem = out_type == kTypeF32 ? 4 : 2;
    ProductParams p{};
    p.out = out;
    p.pitch = out_pitch;
    p.out_type = out_type;
    p.accumulate = accumulate;
    p.status = status;
    p.kblocks = (k + kBlockK - 1) / kBlockK;
    p.rows[0] = a.rows, p.rows[1] = b.rows;
    if (k == 0) {
        if (accumulate) return;
        fill_zero_kernel<<<256, 256, 0, stream>>>(p);
        launch_check("fill_zero_kernel");
        return;
    }
    const Plan plan = plan_product(a.rows, b.rows, p.kblocks, device_sms());
    const Fp8Operand& left = plan.swap ? b : a;
    const Fp8Operand& right = plan.swap ? a : b;
    const Fp8Operand* side[2] = {&left, &right};
    for (int s = 0; s < 2; s++) {
        p.rows[s] = side[s]->rows;
        p.scale[s] = side[s]->scale;
        p.sp[s] = (int)fp8_scale_pitch(k);
        p.shift[s] = side[s]->block_rows == 128 ? 7 : 0;
    }
    p.swap = plan.swap;
    p.splits = plan.splits;
    p.tiles_m = (left.rows + kTileRows - 1) / kTileRows;
    p.tiles_n = (right.rows + plan.bn - 1) / plan.bn;
    p.idesc = idesc_mxf8(plan.bn, left.e5m2, right.e5m2);
    p.vec = !plan.swap && reinterpret_cast<uintptr_t>(out) % 16 == 0 && out_pitch * elem % 16 == 0;
    const CUtensorMap ta = operand_map(left.q, left.rows, k, kTileRows);
    const CUtensorMap tb = operand_map(right.q, right.rows, k, plan.bn);
    switch (plan.bn) {
        case 16: launch_product<16>(ta, tb, p, stream); break;
        case 32: launch_product<32>(ta, tb, p, stream); break;
        case 64: launch_product<64>(ta, tb, p, stream); break;
        case 128: launch_product<128>(ta, tb, p, stream); break;
        default: launch_product<256>(ta, tb, p, stream); break;
    }
}

}  // namespace sy
