// Orthogonalisation of an update by Newton-Schulz products, and the Muon optimizer step built on it
// (K. Jordan et al., "Muon: an optimizer for hidden layers in neural networks", 2024).
//
// X0 = U / |U|_F, with U transposed where it has more rows than columns (X is r x c, r <= c); then, `steps` times,
//   A = X X^T,  B = b A + c A^2,  X <- a X + B X,      (a, b, c) = (3.4445, -4.7750, 2.0315),
// which drives the singular values of X towards 1.
//
// The products run on the tensor cores in fp16 with FP32 accumulation.  fp16 carries TF32's 11 significant bits
// at twice TF32's rate; its range is enough because every matrix here is bounded: the singular values of X stay
// below 1.203 (the maximum of the quintic on [0, 1.203]), so |X| <= 1.203, |A| <= 1.447 and |B| <= 2.807 (the
// largest |b l + c l^2| for l in [0, 1.447]).  X is held times 2^p, p = min(15, log2 sqrt(r c)), which puts its
// entries near 1, A and B times 2^14; all factors are powers of two.  Where the caller wants FP32 accuracy every
// operand is a pair hi + lo of fp16 values (22 bits) and each product is hi hi + hi lo + lo hi.
//
// Operands are kept as tiles of 64 columns in the swizzled form the tensor core reads (128-byte rows, 16-byte chunks
// XOR-ed with row % 8), so that the same X tile serves as a K-major operand of X X^T and as an MN-major operand of
// B X.  Matrices of at most 128 rows (of X) run on chip, one cluster each; larger ones run as tiles of all
// matrices of the call in one persistent cooperative kernel.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <stdexcept>
#include <string>
#include <vector>

#include "kernels.h"

namespace sy {

namespace {

constexpr float kNsA = 3.4445f, kNsB = -4.7750f, kNsC = 2.0315f;
constexpr int kTile = 128, kChunk = 64;             // output tile; columns of an operand tile
constexpr int kTileBytes = kTile * kChunk * 2;      // 16 KB
constexpr int kGramExp = 14;                        // A and B are held times 2^14
constexpr int kMaxJobs = 32;                        // matrices per launch (kernel parameters hold the table)

// One matrix as the caller has it.
struct Source {
    const void* in;             // orthogonalisation: U;  Muon: grad
    float *weight, *momentum;   // Muon
    void* out;                  // orthogonalisation
    long in_pitch, out_pitch;
    int r, c;                   // X is r x c
    int tall;                   // X is U transposed
    int p;                      // X is held times 2^p
    int in_type, out_type;
    float rate;                 // Muon: factor of O in the update
    int mode;                   // how U (and the momentum) is read
};

struct Settings {
    int steps, nesterov;
    float lr, momentum, decay, grad_scale;
    int* status;
};

// byte offset of element (row, col) in a matrix of 128 x 64 tiles, `cb` tiles per row of tiles
__device__ __forceinline__ long tile_offset(int row, int col, int cb) {
    return ((long)(row >> 7) * cb + (col >> 6)) * kTileBytes + (row & 127) * 128 +
           ((((col & 63) >> 3) ^ (row & 7)) << 4) + (col & 7) * 2;
}

__device__ __forceinline__ void split_half(float v, __half& hi, __half& lo) {
    hi = __float2half_rn(v);
    lo = __float2half_rn(v - __half2float(hi));
}

// How four consecutive values of a matrix are read: one access where its rows are aligned and a multiple of four long,
// otherwise value by value.
enum { kWide32, kWide16, kAny32, kAny16 };

// Up to four consecutive values from `at` (the first n; the rest are zero; the wide modes see multiples of four only).
// Without branches, so that a thread's loads overlap: a lane with nothing to read takes the first value.  Past L1:
// Muon's momentum may just have been written by another SM.
template <int MODE>
__device__ __forceinline__ float4 load_u4(const void* in, int type, long at, int n) {
    float v[4];
    if (MODE == kWide32) {
        const float4 f = __ldcg(reinterpret_cast<const float4*>(static_cast<const float*>(in) + (n > 0 ? at : 0)));
        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    } else if (MODE == kAny32) {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = __ldcg(static_cast<const float*>(in) + (i < n ? at + i : 0));
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(in);
        uint32_t h[4];
        if (MODE == kWide16) {
            const uint2 u = __ldcg(reinterpret_cast<const uint2*>(p + (n > 0 ? at : 0)));
            h[0] = u.x & 0xffff, h[1] = u.x >> 16, h[2] = u.y & 0xffff, h[3] = u.y >> 16;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) h[i] = __ldcg(p + (i < n ? at + i : 0));
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
            v[i] = type == kTypeBF16 ? __uint_as_float(h[i] << 16) : __half2float(__ushort_as_half((uint16_t)h[i]));
    }
    return make_float4(n > 0 ? v[0] : 0.0f, n > 1 ? v[1] : 0.0f, n > 2 ? v[2] : 0.0f, n > 3 ? v[3] : 0.0f);
}

// Muon's direction from the (scaled) gradient g and the new momentum m
__device__ __forceinline__ float direction(const Settings& q, float g, float m) {
    return q.nesterov ? q.grad_scale * g + q.momentum * m : m;
}

// The momentum step of up to four values at `at`; v: the gradient, then the direction.
template <int MODE>
__device__ __forceinline__ void update_momentum(const Settings& q, const Source& j, long at, int n, float* v,
                                                const float4& old) {
    float w[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
    for (int k = 0; k < 4; k++) {
        w[k] = q.momentum * w[k] + q.grad_scale * v[k];
        v[k] = direction(q, v[k], w[k]);
    }
    if (MODE == kWide32) {
        if (n > 0) *reinterpret_cast<float4*>(j.momentum + at) = make_float4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (k < n) j.momentum[at + k] = w[k];
    }
}

// U after the momentum step: up to four values
template <int MODE>
__device__ __forceinline__ float4 load_direction4(const Settings& q, const Source& j, long at, int n) {
    float4 g = load_u4<MODE>(j.in, j.in_type, at, n);
    if ((MODE == kWide32 || MODE == kAny32) && j.weight) {
        const float4 m = load_u4<MODE>(j.momentum, kTypeF32, at, n);
        g.x = direction(q, g.x, m.x), g.y = direction(q, g.y, m.y);
        g.z = direction(q, g.z, m.z), g.w = direction(q, g.w, m.w);
    }
    return g;
}

// 2^p / |U| as two floats, applied one after the other (their product may leave the range of a float); 0 for |U| = 0
// and NaN for a norm that is not finite.
struct Scale {
    float a, b;
    __device__ __forceinline__ float operator()(float v) const { return v * a * b; }
};
__device__ __forceinline__ Scale scale_of(double sum_of_squares, int p) {
    if (sum_of_squares == 0.0) return Scale{0.0f, 0.0f};
    if (!(sum_of_squares <= 1.7e308)) return Scale{__int_as_float(0x7fffffff), 1.0f};
    const double s = exp2((double)p) / sqrt(sum_of_squares);
    int e;
    frexp(s, &e);
    return Scale{exp2f((float)(e / 2)), (float)(s * exp2((double)-(e / 2)))};
}

__device__ __forceinline__ void pack8(const float* v, uint4& hi, uint4& lo) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int m = 0; m < 4; m++) {
        __half2 a, b;
        split_half(v[2 * m], a.x, b.x);
        split_half(v[2 * m + 1], a.y, b.y);
        h[m] = *reinterpret_cast<const uint32_t*>(&a);
        l[m] = *reinterpret_cast<const uint32_t*>(&b);
    }
    hi = make_uint4(h[0], h[1], h[2], h[3]);
    lo = make_uint4(l[0], l[1], l[2], l[3]);
}

// 16 consecutive values of O (X's orientation) per lane, from column `col` of row row0 + lane: the output, or the weight
// update.  Called by a whole warp.  Where X is U the block is transposed between the lanes first, so that a warp's
// accesses run along the rows of the output for any pitch and alignment; where X is U transposed they do already.
// The old weights are all loaded before the first is stored, so that the loads overlap.
__device__ __forceinline__ void finish16(const Settings& q, const Source& j, int row0, int col, float* v, bool& bad) {
    const int lane = threadIdx.x & 31;
    long at, step;
    int n;                           // valid values of this lane
    if (j.tall) {
        const int row = row0 + lane;
        at = (long)col * j.out_pitch + row, step = j.out_pitch;
        n = row < j.r ? min(16, j.c - col) : 0;
    } else {
        transpose16(v, lane);
        const int row = row0 + (lane & 16);
        col += lane & 15;
        at = (long)row * j.out_pitch + col, step = j.out_pitch;
        n = col < j.c ? min(16, j.r - row) : 0;
    }
    if (j.weight) {
        float w[16];
        const float keep = 1.0f - q.lr * q.decay;
#pragma unroll
        for (int k = 0; k < 16; k++) w[k] = k < n ? j.weight[at + k * step] : 0.0f;
#pragma unroll
        for (int k = 0; k < 16; k++) {
            w[k] = w[k] * keep - j.rate * v[k];
            if (k < n) {
                bad |= !(fabsf(w[k]) <= 3.402823466e38f);
                j.weight[at + k * step] = w[k];
            }
        }
    } else if (j.out_type == kTypeF32) {
        float* o = static_cast<float*>(j.out) + at;
#pragma unroll
        for (int k = 0; k < 16; k++)
            if (k < n) o[k * step] = v[k];
    } else {
        uint16_t* o = static_cast<uint16_t*>(j.out) + at;
#pragma unroll
        for (int k = 0; k < 16; k++)
            if (k < n)
                o[k * step] = j.out_type == kTypeBF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v[k]))
                                                      : __half_as_ushort(__float2half_rn(v[k]));
    }
}

// The same out of line, for the tiled kernel: it runs in the last iteration only, and inlined it crowds the instruction
// cache of the others.  Returns whether a new weight is not finite.
struct Values16 {
    float v[16];
};
__device__ __noinline__ bool finish16_far(const Settings& q, const Source& j, int row0, int col, Values16 values) {
    bool bad = false;
    finish16(q, j, row0, col, values.v, bad);
    return bad;
}

// A report that is there already, of a wait that gave up above all, is kept.
__device__ __forceinline__ void report_not_finite(int* status) { atomicCAS(status, 0, kStatusNonFinite); }

// ------------------------------------------------------------------ short matrices: one cluster each
//
// A matrix of at most 128 rows (of X) stays on chip for the whole call.  The CTAs of a cluster hold a slab of
// columns each, in shared memory as operand tiles of `rows` x 64 (rows = r rounded up to 16).  Per iteration every
// CTA forms X X^T over its columns, the cluster sums the partial products (each CTA a share of the rows, in rank
// order) and hands every CTA the whole of A; A^2, B and B X are then local.  Three products and two cluster
// barriers per iteration instead of three launches, and U is read and O written once.
// The MMA always takes 128 rows: those past `rows` read whatever follows the tile in shared memory and land in
// accumulator rows that nothing reads.

constexpr int kSlabThreads = 512;
// TMEM columns: the products of A and a round of columns of B X; for pairs each with as many for the cross products,
// whose additions would otherwise truncate the hi hi sums twice as often.
__host__ __device__ constexpr int slab_gram_cols(bool split) { return split ? 256 : 128; }
__host__ __device__ constexpr int slab_round(bool split) { return split ? 128 : 384; }
constexpr int kMaxSmem = 227 * 1024, kMaxSlabSmem = kMaxSmem - 1024;   // per CTA; dynamic, beside the static arrays

struct SlabJob : Source {
    int rows;                        // r rounded up to 16
    int width;                       // columns per CTA, a multiple of 64
    int first, ranks;                // its CTAs, all of one cluster
};
template <int N>
struct SlabJobs : Settings {
    int count;
    SlabJob job[N];
};

__host__ __device__ constexpr int slab_x_bytes(int rows, int width) { return width / 64 * rows * 128; }   // one half
__host__ __device__ constexpr int slab_a_bytes(int rows) { return (rows + 63) / 64 * rows * 128; }
__host__ __device__ constexpr int slab_part_bytes(int rows) { return rows * (rows + 4) * 4; }
int slab_smem(int rows, int width, int ranks, bool split) {
    const int tiles = (slab_x_bytes(rows, width) + slab_a_bytes(rows)) * (split ? 2 : 1);
    // the last operand tile may be read for 128 rows
    return 1024 + std::max(tiles + (ranks > 1 ? slab_part_bytes(rows) : 0), tiles - rows * 128 + 128 * 128);
}

__device__ __forceinline__ float4 peer_load4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}
__device__ __forceinline__ void peer_store4(uint32_t addr, uint4 v) {
    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                 : "memory");
}
__device__ __forceinline__ double peer_load_d(uint32_t addr) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
    return v;
}

// byte offset of element (row, col) in slab tiles
__device__ __forceinline__ int slab_offset(int row, int col, int rows) {
    return (col >> 6) * rows * 128 + row * 128 + ((((col & 63) >> 3) ^ (row & 7)) << 4) + (col & 7) * 2;
}

// 16 consecutive columns (a multiple of 16) of a row: value of hi + lo
template <bool SPLIT>
__device__ __forceinline__ void slab_read16(const uint8_t* hi, int lo, int row, int col, int rows, float* v) {
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const uint8_t* p = hi + slab_offset(row, col + 8 * k, rows);
        const uint4 h = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
        for (int l = 0; l < 4; l++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[l]));
            v[8 * k + 2 * l] = f.x, v[8 * k + 2 * l + 1] = f.y;
        }
        if (SPLIT) {
            const uint4 g = *reinterpret_cast<const uint4*>(p + lo);
            const uint32_t x[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
            for (int l = 0; l < 4; l++) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x[l]));
                v[8 * k + 2 * l] += f.x, v[8 * k + 2 * l + 1] += f.y;
            }
        }
    }
}

template <bool SPLIT>
__device__ __forceinline__ void slab_write16(uint8_t* hi, int lo, int row, int col, int rows, const float* v) {
#pragma unroll
    for (int k = 0; k < 2; k++) {
        uint8_t* p = hi + slab_offset(row, col + 8 * k, rows);
        uint4 h, l;
        pack8(v + 8 * k, h, l);
        *reinterpret_cast<uint4*>(p) = h;
        if (SPLIT) *reinterpret_cast<uint4*>(p + lo) = l;
    }
}

// D += A B over 16 K elements of operands held as hi (+ lo at byte distance `a_lo`, `b_lo`); the cross products go to the
// accumulator 128 columns on.
template <bool SPLIT>
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t a_lo, uint64_t b, uint64_t b_lo, uint32_t idesc,
                                         bool accumulate) {
    mma_f16(d, a, b, idesc, accumulate);
    if (SPLIT) {
        mma_f16(d + 128, a, b + b_lo, idesc, accumulate);
        mma_f16(d + 128, a + a_lo, b, idesc, 1);
    }
}
template <bool SPLIT>
__device__ __forceinline__ void load_pair16(uint32_t d, float* v) {
    tmem_ld16(d, v);
    if (SPLIT) {
        float w[16];
        tmem_ld16(d + 128, w);
#pragma unroll
        for (int k = 0; k < 16; k++) v[k] += w[k];
    }
}

// The part of U that a CTA of the cluster path reads: units of four values along U's contiguous axis (X's columns, or
// its rows when tall), zero outside the matrix.
struct SlabUnits {
    int col0, per, count, live_across, live_along, tall;
    float per_inv;
    __device__ SlabUnits(const SlabJob& j, int col0, int cols, int tiles) : col0(col0), tall(j.tall) {
        per = (j.tall ? j.rows : tiles * 64) / 4;
        count = (j.tall ? cols : j.rows) * per;
        live_across = j.tall ? cols : j.r, live_along = j.tall ? j.r : cols;
        per_inv = 1.0f / per;
    }
    // values of unit u that exist, and where they are; line and k: its place across and along
    __device__ int locate(int u, long pitch, int& line, int& k, long& at) const {
        line = fast_div(u, per_inv), k = (u - line * per) * 4;
        at = (tall ? col0 + line : (long)line) * pitch + (tall ? k : col0 + k);
        return u < count && line < live_across ? live_along - k : 0;
    }
};

// Momentum and this thread's part of |U|^2 (double: no scale of the gradient overflows or loses terms).  d: the last
// four units, which are all of this thread's where the slab is small.
template <int MODE>
__device__ __forceinline__ double slab_norm(const Settings& q, const SlabJob& j, const SlabUnits& units, float4* d) {
    double s = 0.0;
    for (int base = threadIdx.x; base < units.count; base += 4 * kSlabThreads) {
        float4 g[4], m[4];
        long at[4];
        int n[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            int line, k;
            n[i] = units.locate(base + i * kSlabThreads, j.in_pitch, line, k, at[i]);
            g[i] = load_u4<MODE>(j.in, j.in_type, at[i], n[i]);
            if ((MODE == kWide32 || MODE == kAny32) && j.weight) m[i] = load_u4<MODE>(j.momentum, kTypeF32, at[i], n[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float v[4] = {g[i].x, g[i].y, g[i].z, g[i].w};
            if ((MODE == kWide32 || MODE == kAny32) && j.weight) update_momentum<MODE>(q, j, at[i], n[i], v, m[i]);
#pragma unroll
            for (int k = 0; k < 4; k++) s += (double)v[k] * v[k];
            d[i] = make_float4(v[0], v[1], v[2], v[3]);
        }
    }
    return s;
}

// X0 = U / |U| times 2^p
template <int MODE, bool SPLIT>
__device__ __forceinline__ void slab_pack(const Settings& q, const SlabJob& j, const SlabUnits& units, const Scale& scale,
                                          uint8_t* x, int x_lo, float4* d) {
    const int rows = j.rows;
    for (int base = threadIdx.x; base < units.count; base += 4 * kSlabThreads) {
        if (units.count > 4 * kSlabThreads)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                int line, k;
                long at;
                const int n = units.locate(base + i * kSlabThreads, j.in_pitch, line, k, at);
                d[i] = load_direction4<MODE>(q, j, at, n);
            }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            int line, k0;
            long at;
            units.locate(base + i * kSlabThreads, j.in_pitch, line, k0, at);
            if (base + i * kSlabThreads >= units.count) continue;
            const float v[4] = {d[i].x, d[i].y, d[i].z, d[i].w};
            __half hi[4], lo[4];
#pragma unroll
            for (int k = 0; k < 4; k++) split_half(scale(v[k]), hi[k], lo[k]);
            if (j.tall) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    *reinterpret_cast<__half*>(x + slab_offset(k0 + k, line, rows)) = hi[k];
                    if (SPLIT) *reinterpret_cast<__half*>(x + x_lo + slab_offset(k0 + k, line, rows)) = lo[k];
                }
            } else {
                uint8_t* p = x + slab_offset(line, k0, rows);
                *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(hi);
                if (SPLIT) *reinterpret_cast<uint2*>(p + x_lo) = *reinterpret_cast<const uint2*>(lo);
            }
        }
    }
}

template <bool SPLIT, int N>
__global__ void __launch_bounds__(kSlabThreads, 1) slab_kernel(const __grid_constant__ SlabJobs<N> q) {
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t bar;
    __shared__ uint32_t tmem_slot;
    __shared__ double red[kSlabThreads / 32], norm;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int index = 0;
    while (index < q.count && (int)blockIdx.x >= q.job[index].first + q.job[index].ranks) index++;
    if (index == q.count || (int)blockIdx.x < q.job[index].first) {
        // a cluster's CTA without a matrix takes part in its barriers
        for (int i = 0; i < 2 + 2 * q.steps; i++) cluster_sync_all();
        return;
    }
    const SlabJob& j = q.job[index];
    const int ranks = j.ranks, rank = blockIdx.x - j.first;
    const uint32_t peer0 = cluster_rank() - rank;                  // the matrix's first CTA within the cluster
    const int rows = j.rows, col0 = rank * j.width;
    const int cols = min(j.width, max(0, j.c - col0));            // this CTA's columns, and as whole tiles
    const int tiles = (cols + 63) / 64;
    const int x_lo = slab_x_bytes(rows, j.width), a_lo = slab_a_bytes(rows);
    uint8_t* x = smem;
    uint8_t* a = smem + x_lo * (SPLIT ? 2 : 1);
    float* part = reinterpret_cast<float*>(a + a_lo * (SPLIT ? 2 : 1));
    const int pp = rows + 4;                                       // pitch of `part`

    if (tid == 0) {
        mbar_init(&bar, 1);
        fence_barrier_init();
    }
    __syncwarp();
    if (warp == 0) {
        tmem_alloc(&tmem_slot, 512);
        tmem_relinquish();
    }

    const SlabUnits units(j, col0, cols, tiles);
    float4 d[4];
    double s = 0.0;
    switch (j.mode) {
        case kWide32: s = slab_norm<kWide32>(q, j, units, d); break;
        case kWide16: s = slab_norm<kWide16>(q, j, units, d); break;
        case kAny32: s = slab_norm<kAny32>(q, j, units, d); break;
        default: s = slab_norm<kAny16>(q, j, units, d); break;
    }
    s = warp_sum_d(s);
    if (lane == 0) red[warp] = s;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    if (tid == 0) {
        double t = 0.0;
        for (int w = 0; w < kSlabThreads / 32; w++) t += red[w];
        norm = t;
    }
    cluster_sync_all();
    const double part_norm = lane < ranks ? peer_load_d(peer_addr(smem_u32(&norm), peer0 + lane)) : 0.0;
    s = 0.0;
    for (int i = 0; i < ranks; i++) s += __shfl_sync(0xffffffffu, part_norm, i);
    const Scale scale = scale_of(s, j.p);

    // X0, zero outside the matrix
    switch (j.mode) {
        case kWide32: slab_pack<kWide32, SPLIT>(q, j, units, scale, x, x_lo, d); break;
        case kWide16: slab_pack<kWide16, SPLIT>(q, j, units, scale, x, x_lo, d); break;
        case kAny32: slab_pack<kAny32, SPLIT>(q, j, units, scale, x, x_lo, d); break;
        default: slab_pack<kAny16, SPLIT>(q, j, units, scale, x, x_lo, d); break;
    }
    if (j.tall)   // columns past the matrix in the last tile
        for (int i = tid; i < (tiles * 64 - cols) * rows; i += kSlabThreads) {
            const int off = slab_offset(i % rows, cols + i / rows, rows);
            *reinterpret_cast<__half*>(x + off) = __half(0.0f);
            if (SPLIT) *reinterpret_cast<__half*>(x + x_lo + off) = __half(0.0f);
        }
    fence_proxy_async();
    __syncthreads();

    const uint32_t xs = smem_u32(x), as = smem_u32(a), ps = smem_u32(part);
    const uint64_t dx = smem_desc(xs, 0, 1024, kLayoutSw128), da = smem_desc(as, 0, 1024, kLayoutSw128);
    const uint64_t dx_mn = smem_desc(xs, rows * 128, 1024, kLayoutSw128);
    const uint64_t tile = rows * 128 / 16, dx_lo = x_lo / 16, da_lo = a_lo / 16;   // descriptor units
    const int row = (warp & 3) * 32 + lane, part_of = warp >> 2;   // accumulator row; warps share its columns
    const uint32_t trow = (uint32_t)((warp & 3) * 32) << 16, tmem_bx = tmem + slab_gram_cols(SPLIT);
    // The tensor core cuts off what an addition (of 16 products) has below the accumulator's last place, on average half a
    // place.  Sums of like sign, the diagonals of X X^T and A^2, come out low by that much per addition, which the next
    // iterations raise; raised by 2^-24 each they are right on average (five iterations, error against 64 bits: 80 x 720
    // 2.4e-6 -> 1.4e-6, positive 128 x 1024 3.8e-6 -> 1.9e-6; FP32 products 1.1e-6 and 1.6e-6).
    const float lost = SPLIT ? 0x1p-24f : 0.0f;
    const float gram_f = exp2f((float)(kGramExp - 2 * j.p)) * (1.0f + lost * ((min(j.width, j.c) + 15) / 16));
    const float back_f = exp2f((float)-kGramExp), square_f = back_f * (1.0f + lost * (rows / 16));
    const float out_f = exp2f((float)-j.p);
    uint32_t phase = 0;
    bool bad = false;
    for (int step = 0; step < q.steps; step++) {
        // X X^T over this CTA's columns
        if (tid == 0) {
            tc_fence_after();
            for (int t = 0; t < tiles; t++)
                for (int kk = 0; kk < 4; kk++) {
                    const uint64_t d = dx + t * tile + 2 * kk;
                    mma_pair<SPLIT>(tmem, d, dx_lo, d, dx_lo, idesc_f16(rows, 0), (t | kk) != 0);
                }
            mma_commit(&bar);
        }
        __syncwarp();
        mbar_wait(&bar, phase, q.status, kStatusWait);
        phase ^= 1;
        tc_fence_after();
        for (int c = part_of * 16; c < rows; c += kSlabThreads / 8) {
            float v[16];
            __syncwarp();
            load_pair16<SPLIT>(tmem + trow + c, v);
            if (ranks == 1) {
#pragma unroll
                for (int k = 0; k < 16; k++) v[k] *= gram_f;
                if (row < rows) slab_write16<SPLIT>(a, a_lo, row, c, rows, v);
            } else if (row < rows)
#pragma unroll
                for (int k = 0; k < 4; k++)
                    *reinterpret_cast<float4*>(part + row * pp + c + 4 * k) =
                        tiles ? make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3])
                              : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        tc_fence_before();
        if (ranks == 1) {
            fence_proxy_async();
            __syncthreads();
        }
        cluster_sync_all();
        // A = the sum over the cluster: this CTA's share of the rows, handed to everyone.  Each CTA begins with another
        // peer, so the order of a sum depends on the row alone.
        const int share = rows / ranks, chunks = rows / 8;
        for (int u = tid; ranks > 1 && u < share * chunks; u += kSlabThreads) {
            const int r = rank * share + u / chunks, c = u % chunks;
            float4 f[8], g[8];
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i < ranks) {
                    const uint32_t from = peer_addr(ps + (r * pp + c * 8) * 4, peer0 + ((rank + i) & (ranks - 1)));
                    f[i] = peer_load4(from), g[i] = peer_load4(from + 16);
                }
            float v[8] = {};
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i < ranks) {
                    v[0] += f[i].x, v[1] += f[i].y, v[2] += f[i].z, v[3] += f[i].w;
                    v[4] += g[i].x, v[5] += g[i].y, v[6] += g[i].z, v[7] += g[i].w;
                }
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] *= gram_f;
            uint4 hi, lo;
            pack8(v, hi, lo);
            const uint32_t to = as + slab_offset(r, c * 8, rows);
            for (int i = 0; i < ranks; i++) {
                const uint32_t peer = peer0 + ((rank + i) & (ranks - 1));
                peer_store4(peer_addr(to, peer), hi);
                if (SPLIT) peer_store4(peer_addr(to + a_lo, peer), lo);
            }
        }
        asm volatile("fence.proxy.async;" ::: "memory");
        cluster_sync_all();
        // B = b A + c A^2, over A
        if (tid == 0) {
            asm volatile("fence.proxy.async;" ::: "memory");
            tc_fence_after();
            for (int kk = 0; kk < rows / 16; kk++) {
                const uint64_t d = da + (kk >> 2) * tile + 2 * (kk & 3);
                mma_pair<SPLIT>(tmem, d, da_lo, d, da_lo, idesc_f16(rows, 0), kk != 0);
            }
            mma_commit(&bar);
        }
        __syncwarp();
        mbar_wait(&bar, phase, q.status, kStatusWait);
        phase ^= 1;
        tc_fence_after();
        for (int c = part_of * 16; c < rows; c += kSlabThreads / 8) {
            float v[16], old[16];
            __syncwarp();
            load_pair16<SPLIT>(tmem + trow + c, v);
            if (row < rows) {
                slab_read16<SPLIT>(a, a_lo, row, c, rows, old);
#pragma unroll
                for (int k = 0; k < 16; k++) v[k] = kNsB * old[k] + kNsC * (v[k] * square_f);
                slab_write16<SPLIT>(a, a_lo, row, c, rows, v);
            }
        }
        fence_proxy_async();
        tc_fence_before();
        __syncthreads();
        // X <- a X + B X
        const bool last = step + 1 == q.steps;
        for (int c0 = 0; c0 < tiles * 64; c0 += slab_round(SPLIT)) {
            const int n = min(slab_round(SPLIT), tiles * 64 - c0);
            if (tid == 0) {
                tc_fence_after();
                for (int n0 = 0; n0 < n; n0 += 256) {
                    const uint64_t b = dx_mn + (c0 + n0) / 64 * tile;
                    for (int kk = 0; kk < rows / 16; kk++)
                        mma_pair<SPLIT>(tmem_bx + n0, da + (kk >> 2) * tile + 2 * (kk & 3), da_lo, b + kk * (2048 / 16),
                                        dx_lo, idesc_f16(min(256, n - n0), 1), kk != 0);
                }
                mma_commit(&bar);
            }
            __syncwarp();
            mbar_wait(&bar, phase, q.status, kStatusWait);
            phase ^= 1;
            tc_fence_after();
            for (int c = part_of * 16; c < n; c += kSlabThreads / 8) {
                float v[16], old[16];
                __syncwarp();
                load_pair16<SPLIT>(tmem_bx + trow + c, v);
                if (row < rows) {
                    slab_read16<SPLIT>(x, x_lo, row, c0 + c, rows, old);
#pragma unroll
                    for (int k = 0; k < 16; k++) v[k] = kNsA * old[k] + v[k] * back_f;
                }
                if (last) {
#pragma unroll
                    for (int k = 0; k < 16; k++) v[k] *= out_f;
                    finish16(q, j, row & ~31, col0 + c0 + c, v, bad);
                } else if (row < rows) {
                    slab_write16<SPLIT>(x, x_lo, row, c0 + c, rows, v);
                }
            }
            fence_proxy_async();
            tc_fence_before();
            __syncthreads();
        }
    }
    if (bad && q.status) report_not_finite(q.status);
    cluster_sync_all();   // no CTA leaves while a peer may read its shared memory
    __syncwarp();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ------------------------------------------------------------------ larger matrices: tiles of a persistent kernel
//
// One cooperative launch per call.  Phases (norm, packing, and per iteration X X^T, A^2, B X) are separated by grid
// barriers.  In a product phase persistent CTAs take 128 x BN output tiles: one thread streams operand tiles (64
// along K, each one contiguous bulk copy) through a ring of stages, a warp waits for them, a warp issues the MMAs
// into one of two accumulators in TMEM, eight warps turn the other accumulator into the next operand.  The
// symmetric products compute the upper triangle of tiles and write each tile twice; where X X^T has fewer tiles than
// the GPU has SMs its K is split instead, and another phase adds the parts.
// The tensor core's FP32 accumulator truncates: each MMA shrinks a sum by half an ulp on average, which the iteration
// raises about fivefold (b A).  Pairs of fp16 therefore accumulate 128 elements along K (eight MMAs) at a time and add
// those sums in registers; with 512 the error of a 1000 x 333 matrix was 6.6e-6, three times that of FP32 arithmetic.

struct Job : Source {
    uint8_t *x[2], *a, *b;      // hi tiles; the lo tiles follow at x_bytes / a_bytes.  a null: A is kept in the X that the
                                // iteration writes, whose tiles are at least as many and written after A was last read
    long x_bytes, a_bytes;
    int rb, cb;                 // 128-row blocks of X; 64-column blocks (padded to an even number)
    int splits;                 // parts of X X^T's K
    // first unit of this matrix in: packing (128 x 64 tiles), each product, and the sum of the split X X^T (16-byte
    // pieces)
    int pack0, tile0[3], sum0;
    int part0;                  // and its first part (128 x 128 floats), splits per tile
};
__device__ __forceinline__ uint8_t* gram_of(const Job& j, int src) { return j.a ? j.a : j.x[src ^ 1]; }
template <int N>
struct Jobs : Settings {
    int count;
    int packs, sums, parts_used;                // units of packing and of the sum of split products, parts
    int tiles[3], bn[3], upper[3];              // of each product: units, tile columns, upper triangle only
    double* norms;                              // [count][gridDim]
    float* parts;
    uint32_t* barrier;
    Job job[N];
};
static_assert(sizeof(Jobs<kMaxJobs>) <= 32000, "job table exceeds the kernel parameters");

enum { kGram = 0, kSquare = 1, kApply = 2 };   // A = X X^T;  B = b A + c A A;  X <- a X + B X
constexpr int kEpilogueWarps = 8;
constexpr int kTiledThreads = 32 * (4 + kEpilogueWarps);
constexpr int kTiledBar = 1;                   // a stage is loaded: the waiting warp and the MMA warp
constexpr int kSegment = 2;                    // stages (of 64 along K) per accumulator of pairs

// A tile is 128 rows by up to kBn columns.  Pairs of fp16 keep two accumulators per tile: hi hi, and the cross products,
// whose additions would otherwise truncate the hi hi sum twice as often; with their sums in registers that leaves
// 128 columns.
template <bool SPLIT>
struct Stages {
    static constexpr int kBn = SPLIT ? 128 : 256;
    static constexpr int kAccCols = 256;                             // TMEM columns of an accumulator (set)
    static constexpr int kHalf = kTileBytes + kBn * 128;   // hi operands, then lo operands
    static constexpr int kBytes = (SPLIT ? 2 : 1) * kHalf;
    static constexpr int kCount = 196608 / kBytes;
    static constexpr int kSmem = 1024 + kCount * kBytes + (2 * kCount + 4) * 8 + 16;
};

struct TileAt {
    int job, i, j, k0, k1, split;   // 128-row block, column block of the product's width, stages along K
};

// unit t of a product: which matrix, which tile of it, which part of K
template <int N>
__device__ __forceinline__ TileAt tile_at(const Jobs<N>& q, int product, int t) {
    int n = N == 1 ? 0 : q.count - 1;
    while (N > 1 && n > 0 && t < q.job[n].tile0[product]) n--;
    const Job& j = q.job[n];
    TileAt a;
    a.job = n;
    a.split = 0;
    a.k0 = 0;
    a.k1 = ((product == kGram ? j.c : j.r) + 63) / 64;
    int u = t - j.tile0[product];
    if (q.upper[product]) {
        // the tiles that reach above the diagonal, by columns: column c holds the first w (c + 1) row blocks
        const int w = q.bn[product] >> 7;
        auto before = [&](int c) { return w * c * (c + 1) / 2; };
        int c = (int)sqrtf(2.0f * u / w);
        while (before(c) > u) c--;
        while (before(c + 1) <= u) c++;
        a.j = c;
        a.i = u - before(c);
    } else {
        if (product == kGram && j.splits > 1) {
            const int all = a.k1;
            a.split = u % j.splits;
            u /= j.splits;
            a.k0 = (int)((long)all * a.split / j.splits);
            a.k1 = (int)((long)all * (a.split + 1) / j.splits);
        }
        a.j = u / j.rb;
        a.i = u - a.j * j.rb;
    }
    return a;
}

// where piece i of lane `row` % 32 goes after transpose_pieces: byte offset from the lane's own row
__device__ __forceinline__ int piece_offset(int row, int chunk0, int i) {
    const int r = (row & ~3) + i;
    return (r - row) * 128 + (((chunk0 + (row & 3)) ^ (r & 7)) << 4);
}

// 32 columns of a row of a tile as stored: fp16 values, hi and lo; fetched in transposed pieces
template <bool SPLIT>
struct OldBits {
    uint4 hi[4], lo[SPLIT ? 4 : 1];
    __device__ __forceinline__ void load(const uint8_t* row_hi, long lo_at, int row, int chunk0) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint8_t* p = row_hi + piece_offset(row, chunk0, k);
            hi[k] = __ldcg(reinterpret_cast<const uint4*>(p));
            if (SPLIT) lo[k] = __ldcg(reinterpret_cast<const uint4*>(p + lo_at));
        }
    }
};
// v += g (hi + lo)
template <bool SPLIT>
__device__ __forceinline__ void add_old(float* v, float g, OldBits<SPLIT>& x) {
    transpose_pieces(x.hi);
    if (SPLIT) transpose_pieces(x.lo);
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const uint32_t h[4] = {x.hi[k].x, x.hi[k].y, x.hi[k].z, x.hi[k].w};
        const uint4 low = x.lo[SPLIT ? k : 0];
        const uint32_t l[4] = {low.x, low.y, low.z, low.w};
#pragma unroll
        for (int m = 0; m < 4; m++) {
            float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h[m]));
            if (SPLIT) {
                const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&l[m]));
                a.x += b.x, a.y += b.y;
            }
            v[8 * k + 2 * m] += g * a.x, v[8 * k + 2 * m + 1] += g * a.y;
        }
    }
}

// 32 columns of a row of a tile, and with `mirror` the same values as a column of the transposed tile there: lanes hold
// consecutive rows, so after an exchange with its neighbour each lane stores two rows of every other column.
template <bool SPLIT>
__device__ __forceinline__ void write32(uint8_t* hi, long lo, int row, int chunk0, const float* v, uint8_t* mirror,
                                        int mirror_row) {
    uint32_t h[16], l[16];
#pragma unroll
    for (int m = 0; m < 16; m++) {
        __half2 a, b;
        split_half(v[2 * m], a.x, b.x);
        split_half(v[2 * m + 1], a.y, b.y);
        h[m] = *reinterpret_cast<const uint32_t*>(&a);
        l[m] = *reinterpret_cast<const uint32_t*>(&b);
    }
    uint4 c[4];
#pragma unroll
    for (int k = 0; k < 4; k++) c[k] = make_uint4(h[4 * k], h[4 * k + 1], h[4 * k + 2], h[4 * k + 3]);
    transpose_pieces(c);
#pragma unroll
    for (int k = 0; k < 4; k++) *reinterpret_cast<uint4*>(hi + piece_offset(row, chunk0, k)) = c[k];
    if (SPLIT) {
#pragma unroll
        for (int k = 0; k < 4; k++) c[k] = make_uint4(l[4 * k], l[4 * k + 1], l[4 * k + 2], l[4 * k + 3]);
        transpose_pieces(c);
#pragma unroll
        for (int k = 0; k < 4; k++) *reinterpret_cast<uint4*>(hi + lo + piece_offset(row, chunk0, k)) = c[k];
    }
    if (!mirror) return;
    const bool odd = row & 1;
#pragma unroll
    for (int m = 0; m < 16; m++) {
        // word m holds columns 2 m (low half) and 2 m + 1 of this row
        const uint32_t other = __shfl_xor_sync(0xffffffffu, h[m], 1);
        const uint32_t w = odd ? __byte_perm(other, h[m], 0x7632) : __byte_perm(h[m], other, 0x5410);
        const int tr = mirror_row + 2 * m + odd, tc = (row & 63) & ~1;    // row and column in the transposed tile
        uint8_t* p = mirror + tr * 128 + (((tc >> 3) ^ (tr & 7)) << 4) + (tc & 7) * 2;
        *reinterpret_cast<uint32_t*>(p) = w;
        if (SPLIT) {
            const uint32_t other_lo = __shfl_xor_sync(0xffffffffu, l[m], 1);
            *reinterpret_cast<uint32_t*>(p + lo) =
                odd ? __byte_perm(other_lo, l[m], 0x7632) : __byte_perm(l[m], other_lo, 0x5410);
        }
    }
}

// Barrier number `turn` (from 1) of the whole grid: what every CTA wrote before it is visible to every CTA after it,
// to plain loads and to bulk copies.  Gives up after a bounded number of polls, like every wait here.
__device__ __forceinline__ bool grid_barrier(uint32_t* counter, uint32_t turn, int* status, int* s_ok) {
    asm volatile("fence.proxy.async;" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        int ok = *s_ok;
        __threadfence();
        atomicAdd(counter, 1);
        for (uint32_t polls = 0; ok; polls++) {
            uint32_t seen;
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(counter) : "memory");
            if (seen >= turn * gridDim.x) break;
            if (polls > kSpinLimit) {
                ok = 0;
                if (status) atomicExch(status, kStatusWait);
            }
        }
        *s_ok = ok;
    }
    __syncthreads();
    return *s_ok;
}

// Momentum and this thread's part of |U|^2, units of four values dealt over the whole grid.
template <int MODE>
__device__ __forceinline__ double tiled_norm(const Settings& q, const Job& j) {
    const int lines = j.tall ? j.c : j.r, length = j.tall ? j.r : j.c, per = (length + 3) / 4;
    const long units = (long)lines * per, stride = (long)gridDim.x * kTiledThreads;
    double s = 0.0;
    for (long base = (long)blockIdx.x * kTiledThreads + threadIdx.x; base < units; base += 4 * stride) {
        float4 g[4], m[4];
        long at[4];
        int n[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const long u = base + i * stride, line = u / per;
            const int k = (int)(u - line * per) * 4;
            n[i] = u < units ? length - k : 0;
            at[i] = line * j.in_pitch + k;
            g[i] = load_u4<MODE>(j.in, j.in_type, at[i], n[i]);
            if ((MODE == kWide32 || MODE == kAny32) && j.weight) m[i] = load_u4<MODE>(j.momentum, kTypeF32, at[i], n[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float v[4] = {g[i].x, g[i].y, g[i].z, g[i].w};
            if ((MODE == kWide32 || MODE == kAny32) && j.weight) update_momentum<MODE>(q, j, at[i], n[i], v, m[i]);
#pragma unroll
            for (int k = 0; k < 4; k++) s += (double)v[k] * v[k];
        }
    }
    return s;
}

// One 128 x 64 tile of X0 = U / |U| times 2^p, zero outside the matrix.
template <int MODE, bool SPLIT>
__device__ __forceinline__ void tiled_pack(const Settings& q, const Job& j, const Scale& scale, int row0, int col0,
                                           uint8_t* dst) {
    if (!j.tall) {
        // eight columns of a row per unit
        for (int u = threadIdx.x; u < 128 * 8; u += kTiledThreads) {
            const int row = u >> 3, col = (u & 7) * 8;
            float v[8];
            const int left = row0 + row < j.r ? j.c - col0 - col : 0;
            const long at = (row0 + row) * j.in_pitch + col0 + col;
            const float4 d[2] = {load_direction4<MODE>(q, j, at, left), load_direction4<MODE>(q, j, at + 4, left - 4)};
#pragma unroll
            for (int k = 0; k < 2; k++)
                v[4 * k] = scale(d[k].x), v[4 * k + 1] = scale(d[k].y), v[4 * k + 2] = scale(d[k].z),
                          v[4 * k + 3] = scale(d[k].w);
            uint4 hi, lo;
            pack8(v, hi, lo);
            uint8_t* p = dst + row * 128 + (((u & 7) ^ (row & 7)) << 4);
            *reinterpret_cast<uint4*>(p) = hi;
            if (SPLIT) *reinterpret_cast<uint4*>(p + j.x_bytes) = lo;
        }
    } else {
        // four rows of eight columns per unit: eight lines of U, lanes along them
        for (int u = threadIdx.x; u < 32 * 8; u += kTiledThreads) {
            const int row = (u & 31) * 4, chunk = u >> 5;
            float v[4][8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int line = col0 + chunk * 8 + k;
                const float4 d = load_direction4<MODE>(q, j, line * j.in_pitch + row0 + row,
                                                       line < j.c ? j.r - row0 - row : 0);
                v[0][k] = scale(d.x), v[1][k] = scale(d.y), v[2][k] = scale(d.z), v[3][k] = scale(d.w);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint4 hi, lo;
                pack8(v[i], hi, lo);
                uint8_t* p = dst + (row + i) * 128 + ((chunk ^ ((row + i) & 7)) << 4);
                *reinterpret_cast<uint4*>(p) = hi;
                if (SPLIT) *reinterpret_cast<uint4*>(p + j.x_bytes) = lo;
            }
        }
    }
}

template <bool SPLIT, int N>
__global__ void __launch_bounds__(kTiledThreads, 1) tiled_kernel(const __grid_constant__ Jobs<N> q) {
    using S = Stages<SPLIT>;
    extern __shared__ uint8_t raw[];
    __shared__ double red[kTiledThreads / 32], s_norm;
    __shared__ int s_ok;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kCount * S::kBytes);
    uint64_t *empty = full + S::kCount, *tfull = empty + S::kCount, *tempty = tfull + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int s = 0; s < S::kCount; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < 2; s++) {
            mbar_init(&tfull[s], 1);
            mbar_init(&tempty[s], 32 * kEpilogueWarps);
        }
        fence_barrier_init();
        s_ok = 1;
    }
    if (warp == 3) {
        tmem_alloc(tmem_slot, 2 * S::kAccCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    uint32_t turn = 0;

    // momentum and the partial sums of squares of U (double: no scale of the gradient overflows or loses terms)
    for (int n = 0; n < q.count; n++) {
        const Job& j = q.job[n];
        double s = 0.0;
        switch (j.mode) {
            case kWide32: s = tiled_norm<kWide32>(q, j); break;
            case kWide16: s = tiled_norm<kWide16>(q, j); break;
            case kAny32: s = tiled_norm<kAny32>(q, j); break;
            default: s = tiled_norm<kAny16>(q, j); break;
        }
        s = warp_sum_d(s);
        if (lane == 0) red[warp] = s;
        __syncthreads();
        if (tid == 0) {
            double t = 0.0;
            for (int w = 0; w < kTiledThreads / 32; w++) t += red[w];
            q.norms[(long)n * gridDim.x + blockIdx.x] = t;
        }
        __syncthreads();
    }
    bool ok = grid_barrier(q.barrier, ++turn, q.status, &s_ok);

    // X0 tiles: U / |U| times 2^p, zero outside the matrix
    for (int t = blockIdx.x, at_job = -1; ok && t < q.packs; t += gridDim.x) {
        int n = q.count - 1;
        while (n > 0 && t < q.job[n].pack0) n--;
        const Job& j = q.job[n];
        if (n != at_job) {
            __syncthreads();
            if (warp == 0) {
                double s = 0.0;
                for (int i = lane; i < (int)gridDim.x; i += 32) s += __ldcg(q.norms + (long)n * gridDim.x + i);
                s = warp_sum_d(s);
                if (lane == 0) s_norm = s;
            }
            __syncthreads();
            at_job = n;
        }
        const Scale scale = scale_of(s_norm, j.p);
        const int block = (t - j.pack0) / j.cb, row0 = block * 128, col0 = (t - j.pack0 - block * j.cb) * 64;
        uint8_t* dst = j.x[0] + (long)(t - j.pack0) * kTileBytes;
        switch (j.mode) {
            case kWide32: tiled_pack<kWide32, SPLIT>(q, j, scale, row0, col0, dst); break;
            case kWide16: tiled_pack<kWide16, SPLIT>(q, j, scale, row0, col0, dst); break;
            case kAny32: tiled_pack<kAny32, SPLIT>(q, j, scale, row0, col0, dst); break;
            default: tiled_pack<kAny16, SPLIT>(q, j, scale, row0, col0, dst); break;
        }
    }
    ok = ok && grid_barrier(q.barrier, ++turn, q.status, &s_ok);

    int n = 0, accs = 0;          // stages and accumulators that this warp's role has passed
    bool bad = false;
    for (int step = 0; ok && step < 4 * q.steps; step++) {
        const int phase = step & 3, src = (step >> 2) & 1;
        if (phase == 1) {
            // the parts of X X^T
            if (!q.sums) continue;
            for (long u = (long)blockIdx.x * kTiledThreads + tid; u < q.sums; u += (long)gridDim.x * kTiledThreads) {
                int k = q.count - 1;
                while (k > 0 && u < q.job[k].sum0) k--;
                const Job& j = q.job[k];
                const int e = (int)(u - j.sum0), tile = e >> 11, row = (e >> 4) & 127, col = (e & 15) * 8;
                const float* from = q.parts + (long)(j.part0 + tile * j.splits) * (kTile * kTile) + row * kTile + col;
                float v[8] = {};
                for (int s = 0; s < j.splits; s++) {
                    const float4 f = __ldcg(reinterpret_cast<const float4*>(from + (long)s * kTile * kTile));
                    const float4 g = __ldcg(reinterpret_cast<const float4*>(from + (long)s * kTile * kTile + 4));
                    v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
                    v[4] += g.x, v[5] += g.y, v[6] += g.z, v[7] += g.w;
                }
                const float f = exp2f((float)(kGramExp - 2 * j.p));
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] *= f;
                uint4 hi, lo;
                pack8(v, hi, lo);
                const int bj = tile / j.rb, bi = tile - bj * j.rb;
                uint8_t* p = gram_of(j, src) + tile_offset(bi * kTile + row, bj * kTile + col, 2 * j.rb);
                *reinterpret_cast<uint4*>(p) = hi;
                if (SPLIT) *reinterpret_cast<uint4*>(p + j.a_bytes) = lo;
            }
            ok = grid_barrier(q.barrier, ++turn, q.status, &s_ok);
            continue;
        }
        const int product = phase == 0 ? kGram : phase == 2 ? kSquare : kApply;
        const bool last = product == kApply && (step >> 2) + 1 == q.steps;
        const int tiles = q.tiles[product], bn = q.bn[product];
        if (warp == 0 || warp == 3) {
            // The two producers take turns.  A wait after a bulk copy holds a thread for ~1,000 cycles, whatever it waits
            // for; alternating halves that per stage.  The first stages of a phase need no wait: the phase before has
            // used up every stage.
            if (lane == 0) {
                const int first = n;
                asm volatile("fence.proxy.async;" ::: "memory");   // what the barrier made visible, to bulk copies too
                for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
                    const TileAt at = tile_at(q, product, t);
                    const Job& j = q.job[at.job];
                    const uint8_t* left = product == kGram ? j.x[src] : product == kSquare ? gram_of(j, src) : j.b;
                    const long left_lo = product == kGram ? j.x_bytes : j.a_bytes;
                    const int lcb = product == kGram ? j.cb : 2 * j.rb;
                    // the columns' operand in pieces of 64, those that exist: column blocks of X, halves of row blocks
                    constexpr int kPiece = kTileBytes / 2;
                    const int per = bn / 64, at64 = at.j * per;
                    const int pieces = min(per, (product == kApply ? j.cb : 2 * j.rb) - at64);
                    for (int k = at.k0; k < at.k1; k++, n++) {
                        if ((n & 1) != (warp == 3)) continue;
                        const int s = n % S::kCount;
                        if (n - first >= S::kCount &&
                            !(ok = mbar_wait(&empty[s], ((n / S::kCount) & 1) ^ 1, q.status, kStatusWait)))
                            break;
                        uint8_t* st = smem + s * S::kBytes;
                        mbar_arrive_expect_tx(&full[s], (kTileBytes + pieces * kPiece) * (SPLIT ? 2 : 1));
                        const uint8_t* a = left + ((long)at.i * lcb + k) * kTileBytes;
                        bulk_load(st, a, kTileBytes, &full[s]);
                        if (SPLIT) bulk_load(st + S::kHalf, a + left_lo, kTileBytes, &full[s]);
                        if (product == kApply) {
                            // 64 rows of neighbouring column blocks of X
                            const uint8_t* b = j.x[src] + ((long)(k >> 1) * j.cb + at64) * kTileBytes + (k & 1) * kPiece;
                            for (int h = 0; h < pieces; h++) {
                                bulk_load(st + kTileBytes + h * kPiece, b + h * kTileBytes, kPiece, &full[s]);
                                if (SPLIT)
                                    bulk_load(st + S::kHalf + kTileBytes + h * kPiece, b + h * kTileBytes + j.x_bytes,
                                              kPiece, &full[s]);
                            }
                        } else {
                            // neighbouring row blocks, or half of one
                            for (int h = 0; h < pieces; h += 2) {
                                const int bytes = min(2, pieces - h) * kPiece;
                                const uint8_t* b = left + ((long)((at64 + h) >> 1) * lcb + k) * kTileBytes +
                                                   ((at64 + h) & 1) * kPiece;
                                bulk_load(st + kTileBytes + h * kPiece, b, bytes, &full[s]);
                                if (SPLIT)
                                    bulk_load(st + S::kHalf + kTileBytes + h * kPiece, b + left_lo, bytes, &full[s]);
                            }
                        }
                    }
                }
                // no copy is in flight when the CTA ends, even after a wait that gave up
                for (int i = max(first, n - S::kCount); i < n; i++)
                    if ((i & 1) == (warp == 3))
                        ok &= mbar_wait(&full[i % S::kCount], (i / S::kCount) & 1, q.status, kStatusWait);
                if (!ok) s_ok = 0;
            }
        } else if (warp == 2) {
            // every wait of the MMA side; after one that gave up the hand-offs go on, so that every warp finishes
            for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
                const TileAt at = tile_at(q, product, t);
                for (int k = at.k0; k < at.k1; k++, n++) {
                    const int s = n % S::kCount, parity = (n / S::kCount) & 1;
                    if (k == at.k0 || (SPLIT && (k - at.k0) % kSegment == 0)) {
                        if (ok) ok = mbar_wait(&tempty[accs & 1], ((accs >> 1) & 1) ^ 1, q.status, kStatusWait);
                        accs++;
                    }
                    if (ok) ok = mbar_wait(&full[s], parity, q.status, kStatusWait);
                    named_bar_sync(kTiledBar, 64);
                }
            }
            if (!ok) s_ok = 0;
        } else if (warp == 1) {
            const uint32_t idesc = idesc_f16(bn, product == kApply);
            // MN-major: 64-column blocks 8 KB apart, groups of 8 K rows 1 KB apart, 16 K rows per MMA
            const uint32_t lbo = product == kApply ? kTileBytes / 2 : 0;
            const uint32_t step_b = product == kApply ? 2048 / 16 : 2;
            const uint32_t smem0 = smem_u32(smem);
            for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
                const TileAt at = tile_at(q, product, t);
                for (int k = at.k0; k < at.k1; k++, n++) {
                    const int s = n % S::kCount, in_segment = SPLIT ? (k - at.k0) % kSegment : k - at.k0;
                    const uint32_t d = tmem + (accs & 1) * S::kAccCols;
                    named_bar_sync(kTiledBar, 64);
                    tc_fence_after();
                    const uint64_t ah = smem_desc(smem0 + s * S::kBytes, 0, 1024, kLayoutSw128);
                    const uint64_t bh = smem_desc(smem0 + s * S::kBytes + kTileBytes, lbo, 1024, kLayoutSw128);
                    constexpr uint64_t kLo = S::kHalf / 16;
#pragma unroll
                    for (int kk = 0; kk < kChunk / 16; kk++) {
                        const bool more = (in_segment | kk) != 0;
                        mma_f16_elect(d, ah + 2 * kk, bh + step_b * kk, idesc, more);
                        if (SPLIT) {
                            mma_f16_elect(d + S::kBn, ah + 2 * kk, bh + kLo + step_b * kk, idesc, more);
                            mma_f16_elect(d + S::kBn, ah + kLo + 2 * kk, bh + step_b * kk, idesc, true);
                        }
                    }
                    mma_commit_elect(&empty[s]);
                    if (k + 1 == at.k1 || (SPLIT && in_segment + 1 == kSegment)) {
                        mma_commit_elect(&tfull[accs & 1]);
                        accs++;
                    }
                }
            }
        } else if (warp >= 4) {
            const int r = (warp & 3) * 32 + lane;
            // four warps share the rows, two the columns: `share` of them from c_first on, 32 at a time
            const int share = bn / 2, c_first = ((warp - 4) >> 2) * share;
            for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
                const TileAt at = tile_at(q, product, t);
                const Job& j = q.job[at.job];
                const bool part = product == kGram && j.splits > 1;
                // accumulator times: X X^T 2^2p -> A 2^14;  A A 2^28 -> 2^14;  B X 2^(14 + p) -> X 2^p
                const float f = part ? 1.0f
                                : product == kGram
                                    ? exp2f((float)(kGramExp - 2 * j.p))
                                    : exp2f((float)-kGramExp) * (product == kSquare ? kNsC : 1.0f);
                const float g = product == kSquare ? kNsB : kNsA, out_f = exp2f((float)-j.p);
                const int cb = product == kApply ? j.cb : 2 * j.rb;
                const uint8_t* old = product == kSquare ? gram_of(j, src) : j.x[src];
                const long lo = product == kApply ? j.x_bytes : j.a_bytes;
                uint8_t* dst = product == kGram ? gram_of(j, src) : product == kSquare ? j.b : j.x[src ^ 1];
                // whether the 32 columns from c on are wanted, and where they are in the tiles
                auto wanted = [&](int c) {
                    const int bj = (at.j * bn + c) >> 7;
                    return bj < cb / 2 && !(q.upper[product] && bj < at.i);
                };
                auto drained = [&] {   // this thread has read the accumulator
                    tc_fence_before();
                    mbar_arrive(&tempty[accs & 1]);
                    accs++;
                };
                auto offset = [&](int c) {
                    return ((long)at.i * cb + ((at.j * bn + c) >> 6)) * kTileBytes + r * 128;
                };
                // v: 32 columns from c on of the accumulator; x: the old operand's
                auto emit = [&](int c, float* v, OldBits<SPLIT>& x) {
#pragma unroll
                    for (int k = 0; k < 32; k++) v[k] *= f;
                    if (part) {
                        const int tile = ((at.j * bn) >> 7) * j.rb + at.i;
                        float4* to = reinterpret_cast<float4*>(
                            q.parts + ((long)(j.part0 + tile * j.splits + at.split) * kTile + r) * kTile +
                            ((at.j * bn) & 127) + c);
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            uint4 p[4];
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                const float* w = v + 16 * h + 4 * k;
                                p[k] = make_uint4(__float_as_uint(w[0]), __float_as_uint(w[1]), __float_as_uint(w[2]),
                                                  __float_as_uint(w[3]));
                            }
                            transpose_pieces(p);
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                __stcg(reinterpret_cast<uint4*>(to) + ((r & ~3) + k - r) * (kTile / 4) + 4 * h + (r & 3),
                                       p[k]);
                        }
                        return;
                    }
                    if (product != kGram) add_old<SPLIT>(v, g, x);
                    const int col = at.j * bn + c;
                    if (last) {
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            Values16 o;
#pragma unroll
                            for (int k = 0; k < 16; k++) o.v[k] = v[16 * h + k] * out_f;
                            bad |= finish16_far(q, j, at.i * kTile + (r & ~31), col + 16 * h, o);
                        }
                        return;
                    }
                    const int bj = col >> 7;
                    uint8_t* mirror = q.upper[product] && bj > at.i
                                          ? dst + ((long)bj * cb + 2 * at.i + (r >> 6)) * kTileBytes
                                          : nullptr;
                    write32<SPLIT>(dst + offset(c), lo, r, (col & 63) >> 3, v, mirror, col & 127);
                };
                // The old operand's values are fetched while the accumulator is still being filled, 32 columns ahead.
                OldBits<SPLIT> x;
                auto fetch = [&](int c) {
                    if (product != kGram && c < c_first + share && wanted(c)) x.load(old + offset(c), lo, r, (c & 63) >> 3);
                };
                fetch(c_first);
                if (SPLIT) {
                    float acc[S::kBn / 2];
                    const int segments = (at.k1 - at.k0 + kSegment - 1) / kSegment;
#pragma unroll 1
                    for (int m = 0; m < segments; m++) {
                        if (ok) ok = mbar_wait(&tfull[accs & 1], (accs >> 1) & 1, q.status, kStatusWait);
                        __syncwarp();
                        tc_fence_after();
                        const uint32_t d = tmem + (accs & 1) * S::kAccCols + c_first + ((uint32_t)((warp & 3) * 32) << 16);
#pragma unroll
                        for (int c = 0; c < S::kBn / 2; c += 16) {
                            float v[16], w[16];
                            if (c >= share) continue;
                            tmem_ld16(d + c, v);
                            tmem_ld16(d + S::kBn + c, w);
#pragma unroll
                            for (int k = 0; k < 16; k++) {
                                v[k] += w[k];
                                acc[c + k] = m ? acc[c + k] + v[k] : v[k];
                            }
                        }
                        drained();
                    }
#pragma unroll 1
                    for (int c = c_first; c < c_first + share; c += 32) {
                        if (wanted(c)) emit(c, acc, x);
                        fetch(c + 32);
#pragma unroll
                        for (int k = 0; k < S::kBn / 2 - 32; k++) acc[k] = acc[k + 32];
                    }
                } else {
                    if (ok) ok = mbar_wait(&tfull[accs & 1], (accs >> 1) & 1, q.status, kStatusWait);
                    tc_fence_after();
                    const uint32_t d = tmem + (accs & 1) * S::kAccCols + ((uint32_t)((warp & 3) * 32) << 16);
#pragma unroll 1
                    for (int c = c_first; c < c_first + share; c += 32) {
                        if (wanted(c)) {
                            float v[32];
                            __syncwarp();
                            tmem_ld32(d + c, v);
                            emit(c, v, x);
                        }
                        fetch(c + 32);
                    }
                    drained();
                }
            }
            if (!ok) s_ok = 0;
        }
        __syncwarp();
        if (last) break;
        ok = grid_barrier(q.barrier, ++turn, q.status, &s_ok);
    }
    if (bad && q.status) report_not_finite(q.status);
    tc_fence_before();
    __syncthreads();
    if (warp == 3) {
        tc_fence_after();
        tmem_dealloc(tmem, 2 * S::kAccCols);
    }
}

// ------------------------------------------------------------------ host side

struct Shape {
    int r, c, rb, cb;
    long x_bytes, a_bytes;   // of one half (hi or lo)
    Shape(int rows, int cols) {
        r = std::min(rows, cols);
        c = std::max(rows, cols);
        rb = (r + 127) / 128;
        cb = (c + 127) / 128 * 2;
        x_bytes = (long)rb * cb * kTileBytes;
        a_bytes = (long)rb * rb * 2 * kTileBytes;
    }
    // `shared`: A lies in the X that is written after it
    long bytes(bool split, bool shared) const { return (2 * x_bytes + (shared ? 1 : 2) * a_bytes) * (split ? 2 : 1); }
};

// Beside the operands: the barrier's counter, partial norms, and the parts of split X X^T (at most one per SM).
constexpr int kMaxSms = 160;
constexpr long kControlBytes = 1024, kNormBytes = (long)kMaxJobs * kMaxSms * sizeof(double),
               kPartBytes = (long)kMaxSms * kTile * kTile * sizeof(float);

long round_up(long v, long to) { return (v + to - 1) / to * to; }

int scale_exponent(const Shape& s) {
    return std::min(15, (int)std::floor(0.5 * std::log2((double)s.r * s.c)));
}

template <bool SPLIT, int N>
void launch_tiled(const Jobs<N>& q, cudaStream_t stream) {
    using S = Stages<SPLIT>;
    static PerDeviceOnce once;
    once_per_device(once, [] { set_max_dynamic_smem(tiled_kernel<SPLIT, N>, S::kSmem, "tiled_kernel"); });
    const cudaError_t e = cudaMemsetAsync(q.barrier, 0, sizeof(uint32_t), stream);
    if (e != cudaSuccess) throw std::runtime_error(std::string("cudaMemsetAsync: ") + cudaGetErrorString(e));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(std::min(device_sms(), kMaxSms));
    cfg.blockDim = dim3(kTiledThreads);
    cfg.dynamicSmemBytes = S::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeCooperative;
    attr[0].val.cooperative = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, tiled_kernel<SPLIT, N>, q);
    launch_check("tiled_kernel");
}

// Tiles of a product: all of them, or those that reach above the diagonal.
int tile_count(const Shape& s, int product, int bn, bool upper) {
    if (!upper) return s.rb * (((product == kApply ? s.cb : 2 * s.rb) * 64 + bn - 1) / bn);
    int n = 0;
    for (int c = 0; c * bn < s.rb * 128; c++) n += std::min(bn / 128 * (c + 1), s.rb);
    return n;
}

// How the products of a call are tiled, by an estimate of the cycles they take.
struct TilePlan {
    int bn[3], upper[3];
    std::vector<int> splits;
};
template <bool SPLIT>
TilePlan plan_tiles(const std::vector<Shape>& shapes, int sms) {
    TilePlan plan;
    // A stage takes the longest of its producer's turn, its copies (about 90 bytes per cycle) and its MMAs (4,096
    // multiply-adds per cycle); a tile adds its start and its epilogue.
    auto stage = [&](int bn) {
        return std::max({500.0, (SPLIT ? 2 : 1) * (kTileBytes + bn * 128) / 90.0, (SPLIT ? 3 : 1) * 2.0 * bn});
    };
    int grams = 0;
    for (const Shape& s : shapes) grams += s.rb * s.rb;
    for (const Shape& s : shapes) {
        // X X^T is split while its tiles leave SMs idle, in parts of four stages at least, where the shorter K saves
        // more cycles than writing and adding the parts takes.  Pairs, five steps, whole and split in us: 333 x 1000 (saves
        // 9,216) 170 and 172, 1000 x 2049 (12,288) 295 and 303, 768 x 1500 (13,824) 239 and 240, 333 x 1500 (15,360) 186
        // and 176, 140 x 4096 (46,080) 266 and 195; single operands, 500 x 1500 (10,000) 135 and 142, 500 x 2000 (14,000)
        // 145 and 148, 140 x 2048 (14,000) 119 and 115, 768 x 3000 (17,500) 207 and 200.
        const int stages = (s.c + 63) / 64, most = std::max(1, std::min(sms / grams, stages / 4));
        plan.splits.push_back((stages - (stages + most - 1) / most) * stage(128) > 13900 ? most : 1);
    }
    const bool any_split = *std::max_element(plan.splits.begin(), plan.splits.end()) > 1;
    for (int p = 0; p < 3; p++) {
        double least = 1e300;
        for (int upper = 0; upper < (p == kApply ? 1 : 2); upper++)
            for (int bn = upper ? 128 : 64; bn <= Stages<SPLIT>::kBn; bn *= 2) {
                if (p == kGram && any_split && (upper || bn != 128)) continue;   // the parts are whole 128 x 128 tiles
                double work = 0, longest = 0;
                for (size_t i = 0; i < shapes.size(); i++) {
                    const double stages = (p == kGram ? shapes[i].c / plan.splits[i] : shapes[i].r) / 64.0;
                    const double tile = stages * stage(bn) + 1500 + 10.0 * bn;
                    work += tile * tile_count(shapes[i], p, bn, upper) * (p == kGram ? plan.splits[i] : 1);
                    longest = std::max(longest, tile);
                }
                const double t = std::max(work / sms + longest / 2, longest);
                if (t < least) least = t, plan.bn[p] = bn, plan.upper[p] = upper;
            }
    }
    return plan;
}

template <bool SPLIT, int N>
void run_tiled(const Settings& set, const std::vector<Source>& list, bool shared, uint8_t* workspace, cudaStream_t stream) {
    Jobs<N> q{};
    static_cast<Settings&>(q) = set;
    q.barrier = reinterpret_cast<uint32_t*>(workspace);
    q.norms = reinterpret_cast<double*>(workspace + kControlBytes);
    q.parts = reinterpret_cast<float*>(workspace + kControlBytes + kNormBytes);
    uint8_t* at = workspace + kControlBytes + kNormBytes + kPartBytes;
    std::vector<Shape> shapes;
    for (const Source& source : list) shapes.emplace_back(source.r, source.c);
    const int sms = std::min(device_sms(), kMaxSms);
    const TilePlan plan = plan_tiles<SPLIT>(shapes, sms);
    for (int p = 0; p < 3; p++) q.bn[p] = plan.bn[p], q.upper[p] = plan.upper[p];
    for (size_t i = 0; i < list.size(); i++) {
        const Shape& s = shapes[i];
        Job& j = q.job[q.count++];
        static_cast<Source&>(j) = list[i];
        j.rb = s.rb, j.cb = s.cb;
        j.x_bytes = s.x_bytes, j.a_bytes = s.a_bytes;
        const int halves = SPLIT ? 2 : 1;
        j.x[0] = at;
        j.x[1] = j.x[0] + halves * s.x_bytes;
        at = j.x[1] + halves * s.x_bytes;
        if (!shared) j.a = at, at += halves * s.a_bytes;
        j.b = at;
        at += halves * s.a_bytes;
        j.splits = plan.splits[i];
        j.pack0 = q.packs, j.sum0 = q.sums;
        q.packs += s.rb * s.cb;
        for (int p = 0; p < 3; p++) {
            j.tile0[p] = q.tiles[p];
            q.tiles[p] += tile_count(s, p, q.bn[p], q.upper[p]) * (p == kGram ? j.splits : 1);
        }
        j.part0 = q.parts_used;
        if (j.splits > 1) {
            q.sums += s.rb * s.rb * kTile * kTile / 8;
            q.parts_used += s.rb * s.rb * j.splits;
        }
    }
    launch_tiled<SPLIT, N>(q, stream);
}

// Fewest CTAs (a power of two up to 8) whose shared memory holds a matrix, 0 where none does.
int slab_ranks(const Shape& s, bool split) {
    if (s.r > 128) return 0;
    const int rows = (s.r + 15) / 16 * 16;
    for (int ranks = 1; ranks <= 8; ranks *= 2) {
        const int width = (s.c + 64 * ranks - 1) / (64 * ranks) * 64;
        if ((long)rows * width * 2 > kMaxSmem) continue;   // X alone; the bytes of wider slabs may not fit an int
        if (slab_smem(rows, width, ranks, split) <= kMaxSlabSmem) return ranks;
    }
    return 0;
}

void set_ranks(SlabJob& j, int ranks) {
    j.ranks = ranks;
    j.width = (j.c + 64 * ranks - 1) / (64 * ranks) * 64;
}

// Deals CTAs to the matrices of a launch.  Narrower slabs shorten every pass over X (64 x 576 in pairs: 53 us on eight
// CTAs, 129 on one; in single operands 43 and 88), so the matrix with the most elements per CTA is given twice as many as
// long as all fit the GPU at a time, with one CTA per SM: 128 CTAs in clusters of up to four, 15 clusters of eight (of 148
// SMs; a sixteenth runs after the others: 16 of 80 x 2304 in single operands 155 us, in 15 clusters 115).
// From two CTAs on a matrix needs memory for the exchange of A: 128 x 320 pairs fit on one CTA and on four, not on two.
void deal_ranks(std::vector<SlabJob>& jobs, bool split) {
    int total = 0;
    bool eight = false;
    for (const SlabJob& j : jobs) total += j.ranks, eight |= j.ranks == 8;
    for (;;) {
        SlabJob *most = nullptr, dealt{};
        for (SlabJob& j : jobs) {
            SlabJob more = j;
            do {
                set_ranks(more, 2 * more.ranks);
            } while (more.ranks < 8 && slab_smem(more.rows, more.width, more.ranks, split) > kMaxSlabSmem);
            if (more.ranks > 8 || slab_smem(more.rows, more.width, more.ranks, split) > kMaxSlabSmem) continue;
            const int limit = eight || more.ranks == 8 ? 120 : 128;
            if (total + more.ranks - j.ranks > limit || more.width == j.width) continue;
            if (!most || (long)j.rows * j.width > (long)most->rows * most->width) most = &j, dealt = more;
        }
        if (!most) return;
        total += dealt.ranks - most->ranks, eight |= dealt.ranks == 8;
        *most = dealt;
    }
}

template <bool SPLIT, int N>
void launch_slabs(const Settings& set, const std::vector<SlabJob>& list, cudaStream_t stream) {
    SlabJobs<N> q{};
    static_cast<Settings&>(q) = set;
    // Jobs come in falling order of their ranks, all powers of two, so none straddles a cluster.
    const int size = list[0].ranks;
    // One CTA per SM: a second one would wait for the TMEM of the first, which may be waiting for it in a cluster barrier.
    int smem = kMaxSmem / 2 + 1024, ctas = 0;
    for (const SlabJob& s : list) {
        SlabJob& j = q.job[q.count++] = s;
        j.first = ctas;
        ctas += j.ranks;
        smem = std::max(smem, slab_smem(j.rows, j.width, j.ranks, SPLIT));
    }
    static PerDeviceOnce once;
    once_per_device(once, [] { set_max_dynamic_smem(slab_kernel<SPLIT, N>, kMaxSlabSmem, "slab_kernel"); });
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((ctas + size - 1) / size * size);
    cfg.blockDim = dim3(kSlabThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, slab_kernel<SPLIT, N>, q);
    launch_check("slab_kernel");
}

template <bool SPLIT>
void run_sources(const Settings& set, const std::vector<Source>& list, bool shared, void* workspace, cudaStream_t stream) {
    std::vector<SlabJob> slabs;
    std::vector<Source> tiled;
    for (const Source& s : list) {
        SlabJob j{};
        static_cast<Source&>(j) = s;
        const int ranks = slab_ranks(Shape(s.r, s.c), SPLIT);
        if (!ranks) {
            tiled.push_back(s);
            continue;
        }
        j.rows = (s.r + 15) / 16 * 16;
        set_ranks(j, ranks);
        slabs.push_back(j);
    }
    for (size_t first = 0; first < slabs.size(); first += kMaxJobs) {
        std::vector<SlabJob> part(slabs.begin() + first, slabs.begin() + std::min<size_t>(slabs.size(), first + kMaxJobs));
        deal_ranks(part, SPLIT);
        std::stable_sort(part.begin(), part.end(), [](const SlabJob& a, const SlabJob& b) {
            return a.ranks != b.ranks ? a.ranks > b.ranks : (long)a.rows * a.width > (long)b.rows * b.width;
        });
        if (part.size() == 1)
            launch_slabs<SPLIT, 1>(set, part, stream);
        else
            launch_slabs<SPLIT, kMaxJobs>(set, part, stream);
    }
    uint8_t* at = reinterpret_cast<uint8_t*>(round_up(reinterpret_cast<intptr_t>(workspace), 1024));
    for (size_t first = 0; first < tiled.size(); first += kMaxJobs) {
        const std::vector<Source> part(tiled.begin() + first,
                                       tiled.begin() + std::min<size_t>(tiled.size(), first + kMaxJobs));
        if (part.size() == 1)
            run_tiled<SPLIT, 1>(set, part, shared, at, stream);
        else
            run_tiled<SPLIT, kMaxJobs>(set, part, shared, at, stream);
    }
}

// Workspace of a call.  Matrices on the cluster path need none; whether a shape takes it does not depend on the rest of
// the list, so a call with part of a list's matrices needs no more.
size_t workspace_bytes(const std::vector<Shape>& shapes, bool split, bool shared) {
    long sum = 0;
    for (const Shape& s : shapes)
        if (!slab_ranks(s, split)) sum += s.bytes(split, shared);
    return (size_t)(1024 + (sum ? kControlBytes + kNormBytes + kPartBytes + sum : 0));
}

bool aligned(const void* p, long pitch_bytes, int bytes) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && pitch_bytes % bytes == 0;
}

}  // namespace

size_t muon_workspace_bytes(const MuonMatrix* m, int count, bool split) {
    std::vector<Shape> shapes;
    for (int i = 0; i < count; i++)
        if (m[i].rows && m[i].cols) shapes.emplace_back(m[i].rows, m[i].cols);
    return workspace_bytes(shapes, split, false);
}

void muon_update(const MuonMatrix* m, int count, const MuonRule& rule, void* workspace, int* status,
                 cudaStream_t stream) {
    const Settings set{rule.steps, rule.nesterov, rule.lr, rule.momentum, rule.decay, rule.grad_scale, status};
    std::vector<Source> list;
    for (int i = 0; i < count; i++) {
        if (m[i].rows == 0 || m[i].cols == 0) continue;
        const Shape shape(m[i].rows, m[i].cols);
        Source s{};
        s.in = m[i].grad, s.weight = m[i].weight, s.momentum = m[i].momentum;
        s.in_pitch = s.out_pitch = m[i].cols;
        s.r = shape.r, s.c = shape.c;
        s.tall = m[i].rows > m[i].cols;
        s.p = scale_exponent(shape);
        s.rate = (float)((double)rule.lr * rule.rms * std::sqrt((double)shape.c));
        s.mode = aligned(s.in, s.in_pitch * 4, 16) && aligned(s.momentum, s.in_pitch * 4, 16) ? kWide32 : kAny32;
        list.push_back(s);
    }
    if (rule.split)
        run_sources<true>(set, list, false, workspace, stream);
    else
        run_sources<false>(set, list, false, workspace, stream);
}

// An orthogonalisation runs on pairs whatever its result's type, so that a 16-bit result is the FP32 one rounded once.
// Single fp16 operands leave 1.1e-3 (relative norm) on nearly white matrices, less than bf16's own rounding of 1.7e-3, but
// the iteration raises the roundings of weak directions up to 485 times: singular values over three decades then cost
// 4e-3 to 6e-3, values falling as 1 / i^2 2e-2.  (Muon's caller chooses by sy_muon_options.precision.)
// bf16 results once ran on single operands in half the memory; their A shares memory with the X written after it, so that
// their workspace stays below that of the other types, whose size is unchanged.
static bool shares_gram(int out_type) { return out_type == kTypeBF16; }

size_t orthogonalize_workspace_bytes(int rows, int cols, int out_type) {
    if (rows == 0 || cols == 0) return 0;
    const Shape shape(rows, cols);
    return workspace_bytes({shape}, true, shares_gram(out_type));
}

void orthogonalize(const void* in, int in_type, long in_pitch, int rows, int cols, int steps, void* out, int out_type,
                   long out_pitch, void* workspace, int* status, cudaStream_t stream) {
    if (rows == 0 || cols == 0) return;
    Settings set{};
    set.steps = steps;
    set.status = status;
    const Shape shape(rows, cols);
    Source s{};
    s.in = in, s.in_type = in_type, s.in_pitch = in_pitch;
    s.out = out, s.out_type = out_type, s.out_pitch = out_pitch;
    s.r = shape.r, s.c = shape.c;
    s.tall = rows > cols;
    s.p = scale_exponent(shape);
    const int bytes = in_type == kTypeF32 ? 4 : 2;
    const bool wide = aligned(in, in_pitch * bytes, 4 * bytes) && cols % 4 == 0;
    s.mode = in_type == kTypeF32 ? (wide ? kWide32 : kAny32) : (wide ? kWide16 : kAny16);
    run_sources<true>(set, {s}, shares_gram(out_type), workspace, stream);
}

}  // namespace sy
