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
#include <type_traits>

#include "kernels.h"

namespace sy {

namespace {

// ------------------------------------------------------------------ casts

__device__ __forceinline__ void store_f(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_f(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_f(__half* p, float v) { *p = __float2half_rn(v); }

// 16 values of a row as they are stored, so that 16-bit types take 8 registers
template <class T>
struct Raw16 {
    static constexpr int kWords = 4 * sizeof(T);
    uint32_t w[kWords];

    // from column c; columns at and past `cols` read as zero
    __device__ __forceinline__ void load(const T* row, int c, int cols, bool vec) {
        if (vec && c + 16 <= cols) {
#pragma unroll
            for (int i = 0; i < kWords / 4; i++) {
                const uint4 u = __ldg(reinterpret_cast<const uint4*>(row + c) + i);
                w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
            }
        } else if (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 16; i++)
                w[i % kWords] = c + i < cols ? __ldg(reinterpret_cast<const uint32_t*>(row) + c + i) : 0u;
        } else {
            const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const uint32_t a = c + 2 * i < cols ? __ldg(p + c + 2 * i) : 0;
                const uint32_t b = c + 2 * i + 1 < cols ? __ldg(p + c + 2 * i + 1) : 0;
                w[i] = a | b << 16;
            }
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kWords; i++) w[i] = 0;
    }
    __device__ __forceinline__ float get(int i) const;

    // infinities become NaN, which maxima pass over
    __device__ __forceinline__ void drop_infinities() {
        constexpr uint32_t kInf = sizeof(T) == 4 ? 0x7f800000u : std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
#pragma unroll
        for (int i = 0; i < kWords; i++) {
            if (sizeof(T) == 4) {
                w[i] |= (w[i] & 0x7fffffffu) == kInf;
            } else {
                w[i] |= (w[i] & 0x7fffu) == kInf;
                w[i] |= (uint32_t)((w[i] >> 16 & 0x7fffu) == kInf) << 16;
            }
        }
    }
};
template <>
__device__ __forceinline__ float Raw16<float>::get(int i) const {
    return __uint_as_float(w[i]);
}
template <>
__device__ __forceinline__ float Raw16<__nv_bfloat16>::get(int i) const {
    return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
}
template <>
__device__ __forceinline__ float Raw16<__half>::get(int i) const {
    return __half2float(__ushort_as_half((uint16_t)(i & 1 ? w[i >> 1] >> 16 : w[i >> 1])));
}

// Smallest e >= -126 with amax <= fmax 2^e.  fmax = 0.875 * 2^top (top 9 for e4m3, 16 for e5m2), so with
// amax = f 2^x, f in [0.5, 1): e = x - top, plus one where f > 0.875.  Read off the bits; a subnormal amax ends at -126.
__device__ __forceinline__ int block_exponent(float amax, int top) {
    const int bits = __float_as_int(amax);
    return amax == 0.0f ? 0 : max((bits >> 23) - 126 - top + ((bits & 0x7fffff) > 0x600000), -126);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

template <bool E5M2>
__device__ __forceinline__ uint32_t cvt4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    if (E5M2) {
        asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    } else {
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    }
    return (uint32_t)lo | (uint32_t)hi << 16;
}
// 16 values times s as 16 bytes
template <bool E5M2, class T>
__device__ __forceinline__ uint4 cvt16(const Raw16<T>& v, float s) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
        w[i] = cvt4<E5M2>(v.get(4 * i) * s, v.get(4 * i + 1) * s, v.get(4 * i + 2) * s, v.get(4 * i + 3) * s);
    return make_uint4(w[0], w[1], w[2], w[3]);
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

// Sizes of 16-bit values are compared as integers, two at a time: the bits without the sign, those of infinities and NaN
// (`special`: there are some) taken as 0.  8192 x 4096 bf16 both ways 31 us, with FP32 comparisons 35: issue slots are 55 %
// used, L1 64 %, DRAM 36 %; 80 registers leave 24 warps per SM to hide the loads.
template <class T>
__device__ __forceinline__ uint32_t sizes2(uint32_t w, bool special) {
    constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    w &= 0x7fff7fffu;
    if (special) {
        if ((w & 0xffffu) >= kInf) w &= 0xffff0000u;
        if (w >> 16 >= kInf) w &= 0xffffu;
    }
    return w;
}
template <class T>
__device__ __forceinline__ float size_value(uint32_t bits) {
    return std::is_same<T, __half>::value ? __half2float(__ushort_as_half((uint16_t)bits)) : __uint_as_float(bits << 16);
}

// An infinity, which no scale brings into range, becomes NaN in e4m3, which has no infinity, and stays one in e5m2: there
// the blocks that held one get its bytes here, from a second look at 16 values of x.
template <class T>
__device__ __noinline__ void restore_infinities(const CastParams& p, int row, int c, uint8_t* q, int step) {
    const T* x = static_cast<const T*>(p.x) + row * p.pitch;
    for (int j = c; j < min(c + 16, p.cols); j++) {
        const float v = (float)x[j];
        if (isinf(v)) q[(j - c) * step] = v < 0.0f ? 0xfc : 0x7c;
    }
}

// Blocks of 1 x 128 without the transposed copy: eight threads per block, 16 values each, the block's maximum
// by three shuffles.  One read, one write, no shared memory.
template <class T, bool E5M2>
__global__ void __launch_bounds__(256) cast_rows_kernel(CastParams p) {
    const uint32_t kb = (p.cols + 127) / 128;
    const uint32_t unit = blockIdx.x * 32u + (threadIdx.x >> 3);
    const uint32_t row = unit / kb, b = unit - row * kb;
    const bool live = row < (uint32_t)p.rows;
    const int c = b * 128 + (threadIdx.x & 7) * 16;
    Raw16<T> v;
    if (live)
        v.load(static_cast<const T*>(p.x) + row * p.pitch, c, p.cols, p.vec);
    else
        v.zero();
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i++) amax = fmaxf(amax, fabsf(v.get(i)));
#pragma unroll
    for (int o = 4; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const bool inf = isinf(amax);
    if (__any_sync(0xffffffffu, inf)) {
        v.drop_infinities();
        amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i++) amax = fmaxf(amax, fabsf(v.get(i)));
#pragma unroll
        for (int o = 4; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    }
    if (!live) return;
    const int e = block_exponent(amax, E5M2 ? 16 : 9);
    if (c < p.qp) {
        uint8_t* q = p.q + (long)row * p.qp + c;
        *reinterpret_cast<uint4*>(q) = cvt16<E5M2>(v, pow2(-e));
        if (E5M2 && inf) restore_infinities<T>(p, row, c, q, 1);
    }
    if ((threadIdx.x & 7) == 0) p.scale[(long)row * p.sp + b] = (uint8_t)(e + 127);
}

// One CTA per 128 x 128 tile, for blocks of 128 x 128 and for the transposed copy: x is read once, both
// orientations leave from registers.  Thread t holds columns 16 (t % 8) .. + 15 of the four rows 4 (t / 8) ..
// + 3, so the four bytes of a transposed word are its own.  The transposed bytes pass through shared memory:
// word (column, row / 4) at column * 32 + (row / 4 ^ 4 (column / 16)), where the 32 lanes of a store and the
// 16-byte groups of a read fall into different banks.
template <class T, bool E5M2>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 3 : 2) cast_tile_kernel(CastParams p) {
    __shared__ float cmax[8][128], cscale[128];   // column maxima of each warp's 16 rows; the columns' scales
    __shared__ float tmax[8];
    __shared__ __align__(16) uint32_t tile[128 * 32];
    const int t = threadIdx.x, seg = t & 7, rw = t >> 3, warp = t >> 5;
    const int kb = (p.cols + 127) / 128, rb = blockIdx.x / kb, b = blockIdx.x - rb * kb;
    const int c = b * 128 + seg * 16, r0 = rb * 128 + rw * 4;
    constexpr int kTop = E5M2 ? 16 : 9;
    Raw16<T> v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (r0 + i < p.rows)
            v[i].load(static_cast<const T*>(p.x) + (r0 + i) * p.pitch, c, p.cols, p.vec);
        else
            v[i].zero();
    }
    bool inf;                                  // (16-bit types: or NaN)
    float rmax[4];
    uint32_t col[8] = {};                      // 16-bit types: column maxima
    if constexpr (sizeof(T) == 2) {
        uint32_t rows[2];                      // row maxima, two rows per word
        auto maxima = [&](bool special) {
            uint32_t m[4] = {};
#pragma unroll
            for (int k = 0; k < 8; k++) {
                col[k] = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t a = sizes2<T>(v[i].w[k], special);
                    m[i] = __vmaxu2(m[i], a);
                    col[k] = __vmaxu2(col[k], a);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; i++)
                rows[i] = __vmaxu2(__byte_perm(m[2 * i], m[2 * i + 1], 0x5410), __byte_perm(m[2 * i], m[2 * i + 1], 0x7632));
        };
        maxima(false);
        constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
        const uint32_t all = __vmaxu2(rows[0], rows[1]);
        inf = __syncthreads_or((all & 0xffffu) >= kInf || all >> 16 >= kInf);
        if (inf) {
            maxima(true);
#pragma unroll
            for (int i = 0; i < 4; i++) v[i].drop_infinities();
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
#pragma unroll
            for (int o = 4; o; o >>= 1) rows[i] = __vmaxu2(rows[i], __shfl_xor_sync(0xffffffffu, rows[i], o));
            rmax[2 * i] = size_value<T>(rows[i] & 0xffffu), rmax[2 * i + 1] = size_value<T>(rows[i] >> 16);
        }
    } else {
        float size = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 16; j++) size = fmaxf(size, fabsf(v[i].get(j)));
        inf = __syncthreads_or(isinf(size));
        if (inf)
#pragma unroll
            for (int i = 0; i < 4; i++) v[i].drop_infinities();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            rmax[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; j++) rmax[i] = fmaxf(rmax[i], fabsf(v[i].get(j)));
#pragma unroll
            for (int o = 4; o; o >>= 1) rmax[i] = fmaxf(rmax[i], __shfl_xor_sync(0xffffffffu, rmax[i], o));
        }
    }
    int e_tile = 0;
    if (p.block_rows == 128) {
        float m = fmaxf(fmaxf(rmax[0], rmax[1]), fmaxf(rmax[2], rmax[3]));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
        if ((t & 31) == 0) tmax[warp] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; w++) m = fmaxf(m, tmax[w]);
        e_tile = block_exponent(m, kTop);
        if (t == 0) {
            p.scale[(long)rb * p.sp + b] = (uint8_t)(e_tile + 127);
            if (p.qt) p.scale_t[(long)b * p.stp + rb] = (uint8_t)(e_tile + 127);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (r0 + i >= p.rows) continue;
        const int e = p.block_rows == 128 ? e_tile : block_exponent(rmax[i], kTop);
        if (c < p.qp) {
            uint8_t* q = p.q + (long)(r0 + i) * p.qp + c;
            *reinterpret_cast<uint4*>(q) = cvt16<E5M2>(v[i], pow2(-e));
            if (E5M2 && inf) restore_infinities<T>(p, r0 + i, c, q, 1);
        }
        if (p.block_rows == 1 && seg == 0) p.scale[(long)(r0 + i) * p.sp + b] = (uint8_t)(e + 127);
    }
    if (!p.qt) return;
    if (p.block_rows == 1) {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int k = 0; k < 8; k++) {
                col[k] = __vmaxu2(col[k], __shfl_xor_sync(0xffffffffu, col[k], 8));
                col[k] = __vmaxu2(col[k], __shfl_xor_sync(0xffffffffu, col[k], 16));
                if ((t & 31) < 8) reinterpret_cast<uint32_t*>(cmax[warp])[seg * 8 + k] = col[k];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 16; j++) {
                float m = 0.0f;   // which NaN does not displace: a column without a finite value is one of zeros
#pragma unroll
                for (int i = 0; i < 4; i++) m = fmaxf(m, fabsf(v[i].get(j)));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                if ((t & 31) < 8) cmax[warp][seg * 16 + j] = m;
            }
        }
        __syncthreads();
        if (t < 128) {
            float m;
            if constexpr (sizeof(T) == 2) {
                uint32_t most = 0;
#pragma unroll
                for (int w = 0; w < 8; w++) most = __vmaxu2(most, reinterpret_cast<const uint32_t*>(cmax[w])[t >> 1]);
                m = size_value<T>(t & 1 ? most >> 16 : most & 0xffffu);
            } else {
                m = cmax[0][t];
#pragma unroll
                for (int w = 1; w < 8; w++) m = fmaxf(m, cmax[w][t]);
            }
            const int e = block_exponent(m, kTop);
            cscale[t] = pow2(-e);
            if (b * 128 + t < p.cols) p.scale_t[(long)(b * 128 + t) * p.stp + rb] = (uint8_t)(e + 127);
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < 16; j++) {
        const float s = p.block_rows == 128 ? pow2(-e_tile) : cscale[seg * 16 + j];
        tile[(seg * 16 + j) * 32 + (rw ^ (seg << 2))] =
            cvt4<E5M2>(v[0].get(j) * s, v[1].get(j) * s, v[2].get(j) * s, v[3].get(j) * s);
    }
    if (E5M2 && inf)
        for (int i = 0; i < 4; i++)
            if (r0 + i < p.rows)
                restore_infinities<T>(p, r0 + i, c,
                                      reinterpret_cast<uint8_t*>(tile + seg * 16 * 32 + (rw ^ (seg << 2))) + i, 128);
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
    if (!vec) {
        // rows of the output start anywhere: lanes take consecutive values, 512 columns of a row per warp
        const uint32_t warps = (cols + 511) / 512, w = blockIdx.x * 8u + (threadIdx.x >> 5), row = w / warps;
        if (row >= (uint32_t)rows) return;
        const int c0 = (w - row * warps) * 512 + (threadIdx.x & 31);
        const uint8_t* src = q + (long)row * qp;
        const uint8_t* sc = scale + (long)(row >> row_shift) * sp;
#pragma unroll 4
        for (int c = c0; c < min(cols, c0 + 512); c += 32) {
            const __half_raw h = __nv_cvt_fp8_to_halfraw(__ldg(src + c), E5M2 ? __NV_E5M2 : __NV_E4M3);
            store_f(out + row * pitch + c, __half2float(__half(h)) * scale_value(__ldg(sc + (c >> 7))));
        }
        return;
    }
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
    if (c + 16 <= cols) {
        const uint32_t* w8 = reinterpret_cast<const uint32_t*>(o);
        if (vec == 2) {   // whole 32-byte sectors
#pragma unroll
            for (int i = 0; i < 4 * (int)sizeof(T); i += 8)
                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(
                                 reinterpret_cast<uint32_t*>(dst) + i),
                             "r"(w8[i]), "r"(w8[i + 1]), "r"(w8[i + 2]), "r"(w8[i + 3]), "r"(w8[i + 4]), "r"(w8[i + 5]),
                             "r"(w8[i + 6]), "r"(w8[i + 7])
                             : "memory");
            return;
        }
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
// Warps: 0, 8 and 9 TMA, 1 MMA, 2 scales, 3 MMA-side waits, 4-7 (and 10-13 where the tile has 128 columns) epilogue.
constexpr int kProducers = 3;
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
    int segment;                 // blocks of K per accumulator
    int* status;
};

// The tensor core's FP32 accumulator cuts off what an addition (an MMA, 32 products) has below its last place: sums of one
// sign come out low by half a place per addition, 3e-5 to 1.2e-4 after 4,096 of them.  So accumulators end after kSegment
// blocks of K (64 additions, 2e-6) and are added in registers, rounded to nearest.  16-bit results take up to kWhole
// blocks in one (128 additions, 4e-6; half a step of f16 is 2.4e-4 at least), which spares the registers: 4096^3 into
// bf16 59 us, into FP32 in segments 68; with a longer K segments cost them little (8192^3 423 and 429 us).
constexpr int kSegment = 16, kWhole = 32;

template <int BN>
struct ProductShape {
    static constexpr int kScaleRows = (BN + 127) / 128;              // N-side scale atoms of 128 rows
    static constexpr int kStageBytes = (kTileRows + BN) * kBlockK;
    static constexpr int kStages = BN >= 128 ? 6 : 8;
    static constexpr int kScaleBytes = 512 * (1 + kScaleRows);
    static constexpr int kScaleCols = 4 * (1 + kScaleRows);
    // epilogue threads hold their sums in registers: 64 columns each at most (128 spill 680 bytes)
    static constexpr int kGroups = BN > 64 ? 2 : 1, kPart = BN / kGroups;
    static constexpr int kThreads = 320 + 128 * (kGroups - 1);
    static constexpr int kCols = 2 * BN + kScaleSlots * kScaleCols;
    static constexpr int kTmemCols = kCols <= 64 ? 64 : kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
    static constexpr int kBarriers = 2 * kStages + 2 * kScaleSlots + 4;
    static constexpr int kSmem = 1024 + kStages * kStageBytes + kScaleSlots * kScaleBytes + kBarriers * 8 + 16;
    // the split sum's partial tile lies over the stages; its row pitch spreads eight rows over all banks
    static constexpr int kPartPitch = BN + 4;
    static_assert(kTileRows * kPartPitch * 4 <= kStages * kStageBytes, "partial tile exceeds the stages");
};

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
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

// two values in the output's 16-bit type
__device__ __forceinline__ uint32_t pack2(const ProductParams& p, float a, float b) {
    if (p.out_type == kTypeBF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// N consecutive columns of output row i in 16-byte pieces (8 for N = 4 values of 16 bits)
template <int N>
__device__ __forceinline__ void put_row(const ProductParams& p, int i, int j, const float* v) {
    if (p.out_type == kTypeF32) {
        float4* o = reinterpret_cast<float4*>(static_cast<float*>(p.out) + i * p.pitch + j);
#pragma unroll
        for (int k = 0; k < N / 4; k++) {
            float4 f = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
            if (p.accumulate) {
                const float4 c = o[k];
                f.x += c.x, f.y += c.y, f.z += c.z, f.w += c.w;
            }
            o[k] = f;
        }
        return;
    }
    uint32_t w[N / 2];
#pragma unroll
    for (int k = 0; k < N / 2; k++) w[k] = pack2(p, v[2 * k], v[2 * k + 1]);
    uint16_t* o = static_cast<uint16_t*>(p.out) + i * p.pitch + j;
    if (N == 4)
        *reinterpret_cast<uint2*>(o) = make_uint2(w[0], w[1]);
    else
#pragma unroll
        for (int k = 0; k < N / 8; k++)
            reinterpret_cast<uint4*>(o)[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
}

// Output rows of any alignment: a warp leaves 32 rows x 128 bytes (64 columns of 16 bits, 32 of FP32) in shared memory, a
// row per lane, and writes them with its lanes along the rows.  (Lanes along the columns write a 3000 x 3001 output in
// 103 us; rows 8 us.)
constexpr int kRaggedPitch = 144;    // bytes; 16-byte accesses of eight rows fall into different banks
constexpr int kRaggedBytes = 32 * kRaggedPitch;

// 16 columns of this lane's row, the `at`-th 16 of the buffer
template <bool F32>
__device__ __forceinline__ void ragged_put(const ProductParams& p, uint8_t* buf, int at, const float* v) {
    uint4* to = reinterpret_cast<uint4*>(buf + (threadIdx.x & 31) * kRaggedPitch + at * (F32 ? 64 : 32));
    if (F32) {
#pragma unroll
        for (int k = 0; k < 4; k++)
            to[k] = make_uint4(__float_as_uint(v[4 * k]), __float_as_uint(v[4 * k + 1]), __float_as_uint(v[4 * k + 2]),
                               __float_as_uint(v[4 * k + 3]));
    } else {
#pragma unroll
        for (int k = 0; k < 2; k++)
            to[k] = make_uint4(pack2(p, v[8 * k], v[8 * k + 1]), pack2(p, v[8 * k + 2], v[8 * k + 3]),
                               pack2(p, v[8 * k + 4], v[8 * k + 5]), pack2(p, v[8 * k + 6], v[8 * k + 7]));
    }
}

// the buffer's first `cols` columns to rows row0 .. row0 + 31, columns from j on
template <bool F32>
__device__ __forceinline__ void ragged_flush(const ProductParams& p, const uint8_t* buf, int row0, int j, int cols) {
    const int lane = threadIdx.x & 31, n = min(32, p.rows[0] - row0);
    cols = min(cols, p.rows[1] - j);
    __syncwarp();
    if (F32) {
        float* o = static_cast<float*>(p.out) + row0 * p.pitch + j + lane;
        if (lane < cols)
            for (int k0 = 0; k0 < n; k0 += 8) {
                float old[8];
#pragma unroll
                for (int k = 0; k < 8; k++) old[k] = p.accumulate && k0 + k < n ? o[(k0 + k) * p.pitch] : 0.0f;
#pragma unroll
                for (int k = 0; k < 8; k++)
                    if (k0 + k < n)
                        o[(k0 + k) * p.pitch] =
                            old[k] + *reinterpret_cast<const float*>(buf + (k0 + k) * kRaggedPitch + 4 * lane);
            }
    } else {
        uint16_t* o = static_cast<uint16_t*>(p.out) + row0 * p.pitch + j + lane;
        const uint16_t* from = reinterpret_cast<const uint16_t*>(buf) + lane;
#pragma unroll 4
        for (int k = 0; k < n; k++) {
            if (lane < cols) o[k * p.pitch] = from[k * (kRaggedPitch / 2)];
            if (lane + 32 < cols) o[k * p.pitch + 32] = from[k * (kRaggedPitch / 2) + 32];
        }
    }
    __syncwarp();
}

// The scale words (four K blocks, group g) of rows r, r + 32, r + 64 and r + 96 of an operand: 16-byte row r % 32 of a
// 512-byte atom.  Rows past the operand's end get the smallest scale; their products are zero.
__device__ __forceinline__ uint4 scale_words(const ProductParams& p, int side, int r, int g) {
    uint32_t x[4];
#pragma unroll
    for (int j = 0; j < 4; j++)
        x[j] = r + 32 * j < p.rows[side]
                   ? __ldg(reinterpret_cast<const uint32_t*>(p.scale[side] +
                                                             (long)((r + 32 * j) >> p.shift[side]) * p.sp[side]) + g)
                   : 0u;
    return make_uint4(x[0], x[1], x[2], x[3]);
}

// c = a b^T on 128 x BN tiles, one CTA per tile and K split.  Both operands stream through shared memory in
// blocks of 128 along K (one scale per row and block, 128-byte swizzled rows); one warp issues four
// 128 x BN x 32 block-scaled MMAs per block and touches no shared memory itself: a warp that has MMAs in flight
// waits ~1,200 cycles for any shared-memory access, an mbarrier wait included, so another warp does its waiting.
// A warp gathers the rows' scale words (four K blocks each) into 512-byte atoms, which the MMA thread copies to TMEM
// ahead of the MMAs that use them.  Two accumulators in TMEM take turns, one per segment of K.  K splits form a cluster:
// each CTA leaves its partial tile in its shared memory and sums a share of the tile over the cluster in rank
// order, so the result does not depend on timing and no workspace is needed.
// 1 x 4096 x 4096 takes 14 us with the weights in DRAM (floor 2.6): latency of set-up, one pass and the cluster's sum.
template <int BN>
__global__ void __launch_bounds__(ProductShape<BN>::kThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                   const ProductParams p) {
    using S = ProductShape<BN>;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    uint8_t* ssm = smem + S::kStages * S::kStageBytes;
    uint64_t* bars = reinterpret_cast<uint64_t*>(ssm + kScaleSlots * S::kScaleBytes);
    uint64_t *full = bars, *empty = bars + S::kStages, *sfull = bars + 2 * S::kStages, *sempty = sfull + kScaleSlots;
    uint64_t *tfull = sempty + kScaleSlots, *tempty = tfull + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
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
        for (int s = 0; s < 2; s++) {
            mbar_init(&tfull[s], 1);
            mbar_init(&tempty[s], 128 * S::kGroups);
        }
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

    if (warp == 0 || warp == 8 || warp == 9) {
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
            if (i % p.segment == 0) {
                const int acc = i / p.segment;
                if (live) live = mbar_wait(&tempty[acc & 1], ((acc >> 1) & 1) ^ 1, p.status, kStatusWait);
            }
            if (live && (i == 0 || (kb & 3) == 0))
                live = mbar_wait(&sfull[group % kScaleSlots], (group / kScaleSlots) & 1, p.status, kStatusWait);
            if (live) live = mbar_wait(&full[s], (i / S::kStages) & 1, p.status, kStatusWait);
            if ((kb & 3) == 3) group++;
            named_bar_sync(kStageBar, 64);
        }
    } else if (warp == 1) {
        const uint32_t st0 = smem_u32(smem), sc0 = smem_u32(ssm);
        int group = 0, acc = 0, in_segment = 0;
        for (int i = 0; i < k1 - k0; i++) {
            const int s = i % S::kStages, kb = k0 + i, slot = group % kScaleSlots;
            const uint32_t tsc = tmem + 2 * BN + slot * S::kScaleCols, d = tmem + (acc & 1) * BN;
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
                mma_mxf8_elect(d, da + 2 * k, db + 2 * k, idesc, tsc, tsc + 4, (in_segment | k) != 0);
            mma_commit_elect(&empty[s]);
            if ((kb & 3) == 3) {
                mma_commit_elect(&sempty[slot]);
                group++;
            }
            if (++in_segment == p.segment || i + 1 == k1 - k0) {
                mma_commit_elect(&tfull[acc & 1]);
                acc++;
                in_segment = 0;
            }
        }
    } else if (warp == 2) {
        const int g0 = k0 >> 2, g1 = (k1 + 3) >> 2;
        for (int g = g0; g < g1; g++) {
            const int i = g - g0, slot = i % kScaleSlots;
            uint4 w[1 + S::kScaleRows];
#pragma unroll
            for (int a = 0; a < 1 + S::kScaleRows; a++)
                w[a] = scale_words(p, a > 0, (a > 0 ? n0 + (a - 1) * 128 : m0) + lane, g);
            if (!mbar_wait(&sempty[slot], ((i / kScaleSlots) & 1) ^ 1, p.status, kStatusWait)) break;
#pragma unroll
            for (int a = 0; a < 1 + S::kScaleRows; a++)
                *reinterpret_cast<uint4*>(ssm + slot * S::kScaleBytes + a * 512 + lane * 16) = w[a];
            fence_proxy_async();
            mbar_arrive(&sfull[slot]);
        }
    }
    __syncwarp();
    if ((warp >= 4 && warp < 8) || warp >= 10) {
        constexpr int kPart = S::kPart;
        const int q = warp & 3, r = q * 32 + lane, i = m0 + r, group = warp >= 10, c_first = group * kPart;
        float sum[kPart];
        const int segments = (k1 - k0 + p.segment - 1) / p.segment;
        bool ok = true;
#pragma unroll 1
        for (int g = 0; g < segments; g++) {
            if (ok) ok = mbar_wait(&tfull[g & 1], (g >> 1) & 1, p.status, kStatusWait);
            __syncwarp();   // lanes come from their own polls
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < kPart; c += 16) {
                float w[16];
                tmem_ld16(tmem + (g & 1) * BN + ((uint32_t)(q * 32) << 16) + c_first + c, w);
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    sum[c + k] = g ? sum[c + k] + w[k] : w[k];
                    asm volatile("" : "+f"(sum[c + k]));   // before the next load: registers are short
                }
            }
            tc_fence_before();
            mbar_arrive(&tempty[g & 1]);
        }
        float* part = reinterpret_cast<float*>(smem);
        constexpr int kPer = BN % 32 == 0 ? 32 : 16;
#pragma unroll 1
        for (int c = c_first; c < c_first + kPart; c += kPer) {
            const float* v = sum;   // columns from c on
            __syncwarp();
            if (p.splits > 1) {
#pragma unroll
                for (int k = 0; k < kPer; k += 4)
                    *reinterpret_cast<float4*>(part + r * S::kPartPitch + c + k) =
                        make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
            } else {
                const int j = n0 + c;
                if (p.swap) {   // lanes run along the output's rows already
#pragma unroll
                    for (int k = 0; k < kPer; k++)
                        if (i < p.rows[0] && j + k < p.rows[1]) put(p, i, j + k, v[k]);
                } else if (kPer == 32 && p.vec && j + 32 <= p.rows[1]) {
                    if (i < p.rows[0]) put_row<kPer>(p, i, j, v);
                } else {
                    // the stages are used up: their memory serves for the rows
                    uint8_t* buf = smem + (4 * group + q) * kRaggedBytes;
                    if (p.out_type == kTypeF32) {
                        for (int k = 0; k < kPer; k += 16) ragged_put<true>(p, buf, k >> 4, v + k);
                        ragged_flush<true>(p, buf, m0 + q * 32, j, kPer);
                    } else {
                        for (int k = 0; k < kPer; k += 16) ragged_put<false>(p, buf, k >> 4, v + k);
                        ragged_flush<false>(p, buf, m0 + q * 32, j, kPer);
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < kPart - kPer; k++) sum[k] = sum[k + kPer];
        }
    }
    if (p.splits > 1) {
        cluster_sync_all();
        const int share = kTileRows / p.splits, first = split * share;
        const uint32_t part = smem_u32(smem);
        for (int u = threadIdx.x; u < share * BN / 4; u += S::kThreads) {
            // lanes along the output's rows
            const int r = first + (p.swap ? u % share : u / (BN / 4)), c = (p.swap ? u / share : u % (BN / 4)) * 4;
            if (m0 + r >= p.rows[0] || n0 + c >= p.rows[1]) continue;
            const uint32_t from = part + (r * S::kPartPitch + c) * 4;
            float4 f[8];
#pragma unroll
            for (int s = 0; s < 8; s++)
                if (s < p.splits) f[s] = ld_cluster4(peer_addr(from, s));
            float v[4] = {f[0].x, f[0].y, f[0].z, f[0].w};
#pragma unroll
            for (int s = 1; s < 8; s++)
                if (s < p.splits) v[0] += f[s].x, v[1] += f[s].y, v[2] += f[s].z, v[3] += f[s].w;
            if (p.vec && n0 + c + 4 <= p.rows[1])
                put_row<4>(p, m0 + r, n0 + c, v);
            else
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (n0 + c + k < p.rows[1]) put(p, m0 + r, n0 + c + k, v[k]);
        }
        cluster_sync_all();   // a peer may still read this CTA's partial tile
    } else {
        __syncthreads();
    }
    __syncwarp();
    if (warp == 3) {
        tc_fence_after();
        tmem_dealloc(tmem, S::kTmemCols);
    }
}

// The same product for many tiles: persistent CTAs, two accumulators in TMEM, so that the epilogue warps drain one
// while the other fills (two of 256 columns and the scales exceed TMEM's 512).  Where an accumulator may not take the
// whole K (kSegment, kWhole) its sums are added in registers, at most 80 per thread of three groups of epilogue warps
// (two groups end at 192 columns: 8192^3 into FP32 512 us, three 438; a weight gradient of 4096 x 1000 over 16,384, whose
// 240-column tiles make one wave, 82 us and 66).
// Warps: 0 TMA, 1 MMA, 2 scales, 3 waits, from 4 on epilogue, the last a second TMA warp where nothing is segmented.
enum WideKind { kWhole16, kSegments16, kSegmentsF32 };
__host__ __device__ constexpr int epilogue_groups(WideKind kind) { return kind == kWhole16 ? 2 : 3; }
constexpr int wide_threads(WideKind kind) { return kind == kWhole16 ? 416 : 512; }

template <int BN, bool RAGGED>
struct WideShape {
    static constexpr int kScaleRows = (BN + 127) / 128;
    static constexpr int kStageBytes = (kTileRows + BN) * kBlockK;
    static constexpr int kScaleBytes = 512 * (1 + kScaleRows), kScaleCols = 4 * (1 + kScaleRows);
    static constexpr int kSlots = BN > 224 ? 2 : kScaleSlots;
    static constexpr int kRagged = RAGGED ? 8 * kRaggedBytes : 0;   // of the eight epilogue warps
    static constexpr int kStages = (227 * 1024 - 2048 - kSlots * kScaleBytes - kRagged) / kStageBytes;
    static constexpr int kCols = 2 * BN + kSlots * kScaleCols;
    static constexpr int kBarriers = 2 * kStages + 2 * kSlots + 4;
    static constexpr int kSmem = 1024 + kStages * kStageBytes + kSlots * kScaleBytes + kBarriers * 8 + 16 + kRagged;
    static_assert(kCols <= 512 && kSmem <= 227 * 1024, "tile too wide");
};

template <int BN, WideKind KIND, bool RAGGED>
__global__ void __launch_bounds__(wide_threads(KIND), 1)
    product_wide_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                        const ProductParams p) {
    using S = WideShape<BN, RAGGED>;
    constexpr bool F32 = KIND == kSegmentsF32, SEGMENTS = KIND != kWhole16;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    uint8_t* ssm = smem + S::kStages * S::kStageBytes;
    uint8_t* ragged = ssm + S::kSlots * S::kScaleBytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(ragged + S::kRagged);
    uint64_t *empty = full + S::kStages, *sfull = empty + S::kStages, *sempty = sfull + S::kSlots;
    uint64_t *tfull = sempty + S::kSlots, *tempty = tfull + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles = p.tiles_m * p.tiles_n, kb = p.kblocks;
    const int mine = (tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;   // tiles of this CTA
    auto place = [&](int t, int& m0, int& n0) {
        const int tile = blockIdx.x + t * gridDim.x, band = 12 * p.tiles_n, in_band = tile % band;
        const int first = tile / band * 12, band_m = min(12, p.tiles_m - first);
        m0 = (first + in_band % band_m) * kTileRows, n0 = in_band / band_m * BN;
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < S::kSlots; s++) {
            mbar_init(&sfull[s], 32);
            mbar_init(&sempty[s], 1);
        }
        for (int s = 0; s < 2; s++) {
            mbar_init(&tfull[s], 1);
            mbar_init(&tempty[s], epilogue_groups(KIND) * 128);
        }
        fence_barrier_init();
    }
    if (warp == 3) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0 || (!SEGMENTS && warp == 12)) {
        if (lane == 0) {
            const int total = mine * kb;
            bool ok = true;
            for (int t = 0, n = 0; ok && t < mine; t++) {
                int m0, n0;
                place(t, m0, n0);
                for (int k = 0; k < kb; k++, n++) {
                    if (!SEGMENTS && (n & 1) != (warp == 12)) continue;
                    const int s = n % S::kStages;
                    if (n >= S::kStages &&
                        !(ok = mbar_wait(&empty[s], ((n / S::kStages) & 1) ^ 1, p.status, kStatusWait)))
                        break;
                    uint8_t* st = smem + s * S::kStageBytes;
                    mbar_arrive_expect_tx(&full[s], S::kStageBytes);
                    tma_load_2d(st, &tm_a, &full[s], k * kBlockK, m0);
                    tma_load_2d(st + kTileRows * kBlockK, &tm_b, &full[s], k * kBlockK, n0);
                    if (n + S::kStages >= total)   // no copy is in flight when the CTA ends
                        mbar_wait(&full[s], (n / S::kStages) & 1, p.status, kStatusWait);
                }
            }
        }
    } else if (warp == 3) {
        bool live = true;
        for (int t = 0, n = 0, group = 0, acc = 0; t < mine; t++)
            for (int k = 0; k < kb; k++, n++) {
                if (k == 0 || (SEGMENTS && k % kSegment == 0)) {
                    if (live) live = mbar_wait(&tempty[acc & 1], ((acc >> 1) & 1) ^ 1, p.status, kStatusWait);
                    acc++;
                }
                if ((k & 3) == 0) {
                    if (live) live = mbar_wait(&sfull[group % S::kSlots], (group / S::kSlots) & 1, p.status, kStatusWait);
                    group++;
                }
                if (live) live = mbar_wait(&full[n % S::kStages], (n / S::kStages) & 1, p.status, kStatusWait);
                named_bar_sync(kStageBar, 64);
            }
    } else if (warp == 1) {
        const uint32_t st0 = smem_u32(smem), sc0 = smem_u32(ssm);
        for (int t = 0, n = 0, group = 0, acc = 0; t < mine; t++)
            for (int k = 0; k < kb; k++, n++) {
                const int s = n % S::kStages, slot = group % S::kSlots;
                const uint32_t tsc = tmem + 2 * BN + slot * S::kScaleCols, d = tmem + (acc & 1) * BN;
                named_bar_sync(kStageBar, 64);
                tc_fence_after();
                if ((k & 3) == 0)
#pragma unroll
                    for (int a = 0; a < 1 + S::kScaleRows; a++)
                        tmem_cp_scales_elect(tsc + 4 * a,
                                             smem_desc(sc0 + slot * S::kScaleBytes + a * 512, 0, 128, kLayoutNone));
                const uint64_t da = smem_desc(st0 + s * S::kStageBytes, 0, 1024, kLayoutSw128);
                const uint64_t db = smem_desc(st0 + s * S::kStageBytes + kTileRows * kBlockK, 0, 1024, kLayoutSw128);
                const uint32_t idesc = p.idesc | (uint32_t)(k & 3) << 4 | (uint32_t)(k & 3) << 29;
                const int in_segment = SEGMENTS ? k % kSegment : k;
#pragma unroll
                for (int i = 0; i < kBlockK / 32; i++)
                    mma_mxf8_elect(d, da + 2 * i, db + 2 * i, idesc, tsc, tsc + 4, (in_segment | i) != 0);
                mma_commit_elect(&empty[s]);
                if ((k & 3) == 3 || k + 1 == kb) {
                    mma_commit_elect(&sempty[slot]);
                    group++;
                }
                if (k + 1 == kb || (SEGMENTS && in_segment + 1 == kSegment)) {
                    mma_commit_elect(&tfull[acc & 1]);
                    acc++;
                }
            }
    } else if (warp == 2) {
        bool ok = true;
        for (int t = 0, group = 0; ok && t < mine; t++) {
            int first[2];
            place(t, first[0], first[1]);
            for (int g = 0; g < (kb + 3) / 4; g++, group++) {
                const int slot = group % S::kSlots;
                uint4 w[1 + S::kScaleRows];
#pragma unroll
                for (int a = 0; a < 1 + S::kScaleRows; a++)
                    w[a] = scale_words(p, a > 0, first[a > 0] + (a > 0 ? a - 1 : 0) * 128 + lane, g);
                if (!(ok = mbar_wait(&sempty[slot], ((group / S::kSlots) & 1) ^ 1, p.status, kStatusWait))) break;
#pragma unroll
                for (int a = 0; a < 1 + S::kScaleRows; a++)
                    *reinterpret_cast<uint4*>(ssm + slot * S::kScaleBytes + a * 512 + lane * 16) = w[a];
                fence_proxy_async();
                mbar_arrive(&sfull[slot]);
            }
        }
    } else {
        constexpr int kPart = (BN / epilogue_groups(KIND) + 15) / 16 * 16;   // columns of a warp, the last group's fewer
        const int r = (warp & 3) * 32 + lane, c_first = ((warp - 4) >> 2) * kPart, c_end = min(BN, c_first + kPart);
        const uint32_t quarter = (uint32_t)((warp & 3) * 32) << 16;
        bool ok = true;
        int acc = 0;
        for (int t = 0; t < mine; t++) {
            int m0, n0;
            place(t, m0, n0);
            const int i = m0 + r;
            uint8_t* buf = ragged + (warp - 4) * kRaggedBytes;
            // Four pieces of 16 bytes from column c on, those inside the warp's part and the output: transposed between the
            // lanes, so that a store covers 64 bytes of eight rows.  Columns come in whole pieces.
            auto emit_pieces = [&](int c, uint4* q) {
                constexpr int kPer = F32 ? 4 : 8;      // values per piece
                const int row0 = i & ~3, j = n0 + c + kPer * (lane & 3);
                transpose_pieces(q);
                if (j >= p.rows[1] || j - n0 >= c_end) return;
                if (F32) {
                    float4* o = reinterpret_cast<float4*>(static_cast<float*>(p.out) + row0 * p.pitch + j);
                    float4 old[4];
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        old[k] = p.accumulate && row0 + k < p.rows[0] ? o[k * p.pitch / 4] : make_float4(0, 0, 0, 0);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const float4 f = *reinterpret_cast<const float4*>(&q[k]);
                        if (row0 + k < p.rows[0])
                            o[k * p.pitch / 4] =
                                make_float4(f.x + old[k].x, f.y + old[k].y, f.z + old[k].z, f.w + old[k].w);
                    }
                } else {
                    uint16_t* o = static_cast<uint16_t*>(p.out) + row0 * p.pitch + j;
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        if (row0 + k < p.rows[0]) *reinterpret_cast<uint4*>(o + k * p.pitch) = q[k];
                }
            };
            if constexpr (SEGMENTS) {
                float sum[kPart] = {};
                const int segments = (kb + kSegment - 1) / kSegment;
                for (int g = 0; g < segments; g++, acc++) {
                    if (ok) ok = mbar_wait(&tfull[acc & 1], (acc >> 1) & 1, p.status, kStatusWait);
                    __syncwarp();
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < kPart; c += 16) {
                        if (c_first + c >= c_end) break;
                        float v[16];
                        tmem_ld16(tmem + (acc & 1) * BN + quarter + c_first + c, v);
#pragma unroll
                        for (int k = 0; k < 16; k++) {
                            sum[c + k] += v[k];
                            asm volatile("" : "+f"(sum[c + k]));   // before the next load: registers are short
                        }
                    }
                    tc_fence_before();
                    mbar_arrive(&tempty[acc & 1]);
                }
                constexpr int kEmit = F32 ? 16 : 32;   // four pieces of 16 bytes
                uint32_t word[F32 ? 1 : kPart / 2];
                if constexpr (!F32) {
#pragma unroll
                    for (int k = 0; k < kPart / 2; k++) {
                        word[k] = pack2(p, sum[2 * k], sum[2 * k + 1]);
                        asm volatile("" : "+r"(word[k]));   // here and now: half the registers
                    }
                }
#pragma unroll
                for (int c = 0; c < kPart; c += kEmit) {
                    const int j = n0 + c_first + c;
                    if (c_first + c >= c_end || j >= p.rows[1]) break;
                    if constexpr (!F32) {
                        uint32_t w[16];
#pragma unroll
                        for (int k = 0; k < 16; k++) w[k] = c / 2 + k < kPart / 2 ? word[(c / 2 + k) % (kPart / 2)] : 0u;
                        if (!p.swap) {
                            uint4 q[4];
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                q[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
                            emit_pieces(c_first + c, q);
                        } else if (i < p.rows[0]) {   // lanes run along the output's rows, which may start anywhere
                            uint16_t* o = static_cast<uint16_t*>(p.out) + j * p.pitch + i;
                            const int n = min(c_end - c_first - c, p.rows[1] - j);
#pragma unroll
                            for (int k = 0; k < 32; k++) {
                                asm volatile("" : "+l"(o));   // addresses as they are needed
                                if (k < n) *o = (uint16_t)(w[k / 2] >> 16 * (k & 1));
                                o += p.pitch;
                            }
                        }
                    } else if (!p.swap) {
                        emit_pieces(c_first + c, reinterpret_cast<uint4*>(sum + c));
                    } else if (i < p.rows[0]) {   // lanes run along the output's rows, which may start anywhere
                        float* o = static_cast<float*>(p.out) + j * p.pitch + i;
#pragma unroll
                        for (int h = 0; h < 16; h += 8) {
                            float old[8];
                            asm volatile("" : "+l"(o));   // addresses as they are needed: the sums fill the registers
                            const float* from = o;
#pragma unroll
                            for (int k = 0; k < 8; k++, from += p.pitch)
                                old[k] = p.accumulate && j + h + k < p.rows[1] ? *from : 0.0f;
#pragma unroll
                            for (int k = 0; k < 8; k++, o += p.pitch)
                                if (j + h + k < p.rows[1]) *o = sum[c + h + k] + old[k];
                        }
                    }
                }
            } else {
                if (ok) ok = mbar_wait(&tfull[acc & 1], (acc >> 1) & 1, p.status, kStatusWait);
                __syncwarp();
                tc_fence_after();
                const uint32_t d = tmem + (acc & 1) * BN + quarter + c_first;
                if (!RAGGED) {
#pragma unroll 1
                    for (int c = 0; c < c_end - c_first && n0 + c_first + c < p.rows[1]; c += 32) {
                        float v[32];
                        uint4 q[4];
                        __syncwarp();
                        tmem_ld16(d + c, v);
                        if (c + 16 < c_end - c_first) tmem_ld16(d + c + 16, v + 16);
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            uint32_t w[4];
#pragma unroll
                            for (int l = 0; l < 4; l++) w[l] = pack2(p, v[8 * k + 2 * l], v[8 * k + 2 * l + 1]);
                            q[k] = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                        emit_pieces(c_first + c, q);
                    }
                } else {
#pragma unroll 1
                    for (int c = 0; c < c_end - c_first && n0 + c_first + c < p.rows[1]; c += 64) {
                        const int some = min(64, c_end - c_first - c);
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            if (16 * k < some) {
                                float v[16];
                                tmem_ld16(d + c + 16 * k, v);
                                ragged_put<false>(p, buf, k, v);
                            }
                        ragged_flush<false>(p, buf, i & ~31, n0 + c_first + c, some);
                    }
                }
                tc_fence_before();
                mbar_arrive(&tempty[acc & 1]);
                acc++;
            }
        }
    }
    __syncwarp();
    __syncthreads();
    if (warp == 3) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

__global__ void fill_zero_kernel(ProductParams p) {
    const long n = (long)p.rows[0] * p.rows[1];
    for (long i = blockIdx.x * (long)blockDim.x + threadIdx.x; i < n; i += (long)gridDim.x * blockDim.x)
        put(p, (int)(i / p.rows[1]), (int)(i % p.rows[1]), 0.0f);
}

struct Plan {
    int swap, bn, splits, wide;
};

// Tile width, K splits, the operand on the MMA's 128-row side and the kernel, by an estimate of the time in ns.
Plan plan_product(int m, int n, int kblocks, bool f32, bool vec, int sms) {
    Plan best{0, 128, 1, 0};
    double least = 1e30;
    auto offer = [&](double t, const Plan& p) {
        if (t < least) least = t, best = p;
    };
    // A block of K is bound by shared memory, which every operand byte passes once in and once out, 128 bytes per cycle
    // (measured at 8192^3: 281 ns for 128 columns, 357 for 192, 372 for 224; its MMAs take 135, 202 and 236).
    auto block = [](int bn) { return (kTileRows + bn) * kBlockK * 2 / 240.0; };
    for (int swap = 0; swap < 2; swap++)
        for (int bn : {16, 32, 64, 128})
            for (int splits : {1, 2, 4, 8}) {
                if (splits > 1 && kblocks < 2 * splits) continue;
                const long mt = ((swap ? n : m) + 127L) / 128, nt = ((swap ? m : n) + bn - 1L) / bn;
                const long waves = (mt * nt * splits + sms - 1) / sms;
                offer(waves * (4000.0 + (swap ? 20.0 : 8.0) * bn + (splits > 1 ? 1500.0 + 20.0 * bn : 0.0) +
                               block(bn) * ((kblocks + splits - 1) / splits)),
                      Plan{swap, bn, splits, 0});
            }
    // Segmented outputs whose rows are not whole 16-byte pieces leave with the lanes along them, as the M side.
    const bool segments = f32 || kblocks > kWhole;
    for (int swap = segments && !vec; swap <= (int)segments; swap++)
        for (int bn : {128, 192, 224, 240}) {
            const long tiles = ((swap ? n : m) + 127L) / 128 * (((swap ? m : n) + bn - 1L) / bn);
            const long waves = (tiles + sms - 1) / sms;
            offer(4000.0 + 8.0 * bn + waves * std::max(block(bn) * kblocks, 8.0 * bn), Plan{swap, bn, 1, 1});
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
    cfg.blockDim = dim3(S::kThreads);
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

template <int BN, WideKind KIND, bool RAGGED>
void launch_wide(const CUtensorMap& ta, const CUtensorMap& tb, const ProductParams& p, cudaStream_t stream) {
    using S = WideShape<BN, RAGGED>;
    static PerDeviceOnce once;
    once_per_device(
        once, [] { set_max_dynamic_smem(product_wide_kernel<BN, KIND, RAGGED>, S::kSmem, "product_wide_kernel"); });
    const int grid = std::min(p.tiles_m * p.tiles_n, device_sms());
    product_wide_kernel<BN, KIND, RAGGED><<<grid, wide_threads(KIND), S::kSmem, stream>>>(ta, tb, p);
    launch_check("product_wide_kernel");
}

template <int BN>
void launch_wide(const CUtensorMap& ta, const CUtensorMap& tb, const ProductParams& p, cudaStream_t stream) {
    if (p.out_type == kTypeF32) return launch_wide<BN, kSegmentsF32, false>(ta, tb, p, stream);
    if (p.kblocks > kWhole) return launch_wide<BN, kSegments16, false>(ta, tb, p, stream);
    if (p.vec)
        launch_wide<BN, kWhole16, false>(ta, tb, p, stream);
    else
        launch_wide<BN, kWhole16, true>(ta, tb, p, stream);
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
    const uintptr_t align = reinterpret_cast<uintptr_t>(out) | (uintptr_t)(pitch * sizeof(T));
    const int vec = align % 32 == 0 ? 2 : align % 16 == 0 ? 1 : 0;   // what the output's rows start on: 32, 16 bytes
    const unsigned blocks = vec ? (unsigned)((rows * ((cols + 15L) / 16) + 255) / 256)
                                : (unsigned)((rows * ((cols + 511L) / 512) + 7) / 8);
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
    // whole 16-byte pieces of the output's rows
    const bool vec = reinterpret_cast<uintptr_t>(out) % 16 == 0 && out_pitch * elem % 16 == 0 &&
                     (long)b.rows * elem % 16 == 0;
    const Plan plan = plan_product(a.rows, b.rows, p.kblocks, out_type == kTypeF32, vec, device_sms());
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
    p.vec = vec && !plan.swap;
    p.segment = out_type == kTypeF32 || p.kblocks > kWhole * p.splits ? kSegment : kWhole;
    const CUtensorMap ta = operand_map(left.q, left.rows, k, kTileRows);
    const CUtensorMap tb = operand_map(right.q, right.rows, k, plan.bn);
    switch (plan.wide ? 1000 + plan.bn : plan.bn) {
        case 16: launch_product<16>(ta, tb, p, stream); break;
        case 32: launch_product<32>(ta, tb, p, stream); break;
        case 64: launch_product<64>(ta, tb, p, stream); break;
        case 128: launch_product<128>(ta, tb, p, stream); break;
        case 1128: launch_wide<128>(ta, tb, p, stream); break;
        case 1192: launch_wide<192>(ta, tb, p, stream); break;
        case 1224: launch_wide<224>(ta, tb, p, stream); break;
        default: launch_wide<240>(ta, tb, p, stream); break;
    }
}

}  // namespace sy
