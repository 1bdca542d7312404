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
// Operands live in the workspace as 128 x 64 tiles of 16 KB in the swizzled form the tensor core reads
// (128-byte rows, 16-byte chunks XOR-ed with row % 8), so a stage of the pipeline is one contiguous bulk copy
// per tile, and the same X tile serves as a K-major operand of X X^T and as an MN-major operand of B X.
// All matrices of a call share the launches: one per product, tiles of all matrices in one persistent grid.
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
constexpr int kMaxNormParts = 512;
constexpr int kThreads = 256;

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
    int vec;                    // rows of every matrix start on 16 bytes (8 for 16-bit types)
};

struct Settings {
    int steps, nesterov;
    float lr, momentum, decay, grad_scale;
    int* status;
};

struct Job : Source {
    uint8_t *x[2], *a, *b;      // hi tiles; the lo tiles follow at x_bytes / a_bytes
    long x_bytes, a_bytes;
    const double* norm;         // partial sums of squares of U
    int rb, cb;                 // 128-row blocks of X; 64-column blocks (padded to a whole tile)
    int tri0, full0;            // first tile of this job in the symmetric and in the full products
};

struct Jobs : Settings {
    int count, tri_tiles, full_tiles, norm_parts;
    Job job[kMaxJobs];
};
static_assert(sizeof(Jobs) <= 32000, "job table exceeds the kernel parameters");

// element (row, col) of U: the orthogonalisation's input or Muon's direction
__device__ __forceinline__ float direction(const Settings& q, const Source& j, long row, long col) {
    const long at = row * j.in_pitch + col;
    if (j.weight) {
        const float m = j.momentum[at];
        return q.nesterov ? q.grad_scale * static_cast<const float*>(j.in)[at] + q.momentum * m : m;
    }
    if (j.in_type == kTypeF32) return static_cast<const float*>(j.in)[at];
    if (j.in_type == kTypeBF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(j.in)[at]);
    return __half2float(static_cast<const __half*>(j.in)[at]);
}

// Momentum update and the partial sums of squares of U (double: neither overflow nor lost terms for any scale
// of the gradient; block sums in a fixed order).
__global__ void __launch_bounds__(256) norm_kernel(const __grid_constant__ Jobs q, double* parts) {
    const Job& j = q.job[blockIdx.y];
    const long rows = j.tall ? j.c : j.r, cols = j.tall ? j.r : j.c;
    double s = 0.0;
    for (long i = blockIdx.x * 256L + threadIdx.x; i < rows * cols; i += gridDim.x * 256L) {
        const long row = i / cols, col = i - row * cols;
        if (j.weight)
            j.momentum[i] = q.momentum * j.momentum[i] + q.grad_scale * static_cast<const float*>(j.in)[i];
        const double u = direction(q, j, row, col);
        s += u * u;
    }
    s = warp_sum_d(s);
    __shared__ double red[8];
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int w = 0; w < 8; w++) t += red[w];
        parts[blockIdx.y * kMaxNormParts + blockIdx.x] = t;
    }
}

// byte offset of element (row, col) in a matrix of 128 x 64 tiles, `cb` tiles per row of tiles
__device__ __forceinline__ long tile_offset(int row, int col, int cb) {
    return ((long)(row >> 7) * cb + (col >> 6)) * kTileBytes + (row & 127) * 128 +
           ((((col & 63) >> 3) ^ (row & 7)) << 4) + (col & 7) * 2;
}

__device__ __forceinline__ void split_half(float v, __half& hi, __half& lo) {
    hi = __float2half_rn(v);
    lo = __float2half_rn(v - __half2float(hi));
}

// X0 tiles: U / |U| times 2^p, zero outside the matrix.  A norm of zero gives zeros; one that is not finite gives
// NaN everywhere.
template <bool SPLIT>
__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ Jobs q) {
    const Job& j = q.job[blockIdx.y];
    __shared__ double s_scale;
    if (threadIdx.x < 32) {
        double s = 0.0;
        for (int i = threadIdx.x; i < q.norm_parts; i += 32) s += j.norm[i];
        s = warp_sum_d(s);
        if (threadIdx.x == 0) s_scale = s == 0.0 ? 0.0 : s <= 1.7e308 ? exp2((double)j.p) / sqrt(s) : nan("");
    }
    __syncthreads();
    const double scale = s_scale;
    const long tiles = (long)j.rb * j.cb;
    for (long t = blockIdx.x; t < tiles; t += gridDim.x) {
        const int row0 = (int)(t / j.cb) * 128, col0 = (int)(t % j.cb) * 64;
        for (int e = threadIdx.x; e < kTile * kChunk; e += 256) {
            // lanes run along U's contiguous axis
            const int row = row0 + (j.tall ? e & 127 : e >> 6), col = col0 + (j.tall ? e >> 7 : e & 63);
            float v = 0.0f;
            if (row < j.r && col < j.c)
                v = (float)(scale * (double)(j.tall ? direction(q, j, col, row) : direction(q, j, row, col)));
            __half hi, lo;
            split_half(v, hi, lo);
            const long at = tile_offset(row, col, j.cb);
            *reinterpret_cast<__half*>(j.x[0] + at) = hi;
            if (SPLIT) *reinterpret_cast<__half*>(j.x[0] + j.x_bytes + at) = lo;
        }
    }
}

// ------------------------------------------------------------------ products

enum { kGram = 0, kSquare = 1, kApply = 2 };   // A = X X^T;  B = b A + c A A;  X <- a X + B X

template <bool SPLIT>
struct Stages {
    static constexpr int kBytes = (SPLIT ? 4 : 2) * kTileBytes;
    static constexpr int kCount = SPLIT ? 3 : 6;
    static constexpr int kSmem = 1024 + kCount * kBytes + (2 * kCount + 4) * 8 + 16;
};

struct TileAt {
    int job, i, j, kblocks;
};

// tile t of the launch: which matrix, which block of it
template <int PHASE>
__device__ __forceinline__ TileAt tile_at(const Jobs& q, int t) {
    int n = q.count - 1;
    while (n > 0 && t < (PHASE == kApply ? q.job[n].full0 : q.job[n].tri0)) n--;
    const Job& j = q.job[n];
    TileAt a;
    a.job = n;
    if (PHASE == kApply) {
        const int u = t - j.full0;
        a.j = u / j.rb;
        a.i = u - a.j * j.rb;
        a.kblocks = (j.r + 63) / 64;
    } else {   // upper triangle by columns
        const int u = t - j.tri0;
        int c = (int)((sqrtf(8.0f * u + 1.0f) - 1.0f) * 0.5f);
        while (c * (c + 1) / 2 > u) c--;
        while ((c + 1) * (c + 2) / 2 <= u) c++;
        a.j = c;
        a.i = u - c * (c + 1) / 2;
        a.kblocks = PHASE == kGram ? (j.c + 63) / 64 : (j.r + 63) / 64;
    }
    return a;
}

__device__ __forceinline__ void read32(const uint8_t* hi, const uint8_t* lo, int row, bool split, int chunk0, float* v) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const int off = ((chunk0 + k) ^ (row & 7)) << 4;
        const uint4 h = *reinterpret_cast<const uint4*>(hi + off);
        const uint32_t w[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
        for (int l = 0; l < 4; l++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[l]));
            v[8 * k + 2 * l] = f.x, v[8 * k + 2 * l + 1] = f.y;
        }
        if (split) {
            const uint4 g = *reinterpret_cast<const uint4*>(lo + off);
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
__device__ __forceinline__ void write32(uint8_t* hi, uint8_t* lo, int row, int chunk0, const float* v) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const int off = ((chunk0 + k) ^ (row & 7)) << 4;
        uint32_t h[4], l[4];
#pragma unroll
        for (int m = 0; m < 4; m++) {
            __half2 a, b;
            split_half(v[8 * k + 2 * m], a.x, b.x);
            split_half(v[8 * k + 2 * m + 1], a.y, b.y);
            h[m] = *reinterpret_cast<const uint32_t*>(&a);
            l[m] = *reinterpret_cast<const uint32_t*>(&b);
        }
        *reinterpret_cast<uint4*>(hi + off) = make_uint4(h[0], h[1], h[2], h[3]);
        if (SPLIT) *reinterpret_cast<uint4*>(lo + off) = make_uint4(l[0], l[1], l[2], l[3]);
    }
}

// N consecutive values of a row of O (X's orientation) from `col` on: the output, or the weight update.  The old
// weights are all loaded before the first is stored, so that the loads overlap.
template <int N>
__device__ __forceinline__ void finish(const Settings& q, const Source& j, int row, int col, const float* v, bool& bad) {
    if (row >= j.r || col >= j.c) return;
    const int n = min(N, j.c - col);
    const long at = j.tall ? col * j.out_pitch + row : row * j.out_pitch + col, step = j.tall ? j.out_pitch : 1;
    if (j.weight) {
        float w[N];
        const float keep = 1.0f - q.lr * q.decay;
        if (!j.tall && j.vec && n == N) {
            float4* p = reinterpret_cast<float4*>(j.weight + at);
#pragma unroll
            for (int k = 0; k < N / 4; k++) *reinterpret_cast<float4*>(w + 4 * k) = p[k];
#pragma unroll
            for (int k = 0; k < N; k++) {
                w[k] = w[k] * keep - j.rate * v[k];
                bad |= !(fabsf(w[k]) <= 3.402823466e38f);
            }
#pragma unroll
            for (int k = 0; k < N / 4; k++) p[k] = *reinterpret_cast<const float4*>(w + 4 * k);
            return;
        }
#pragma unroll
        for (int k = 0; k < N; k++) w[k] = k < n ? j.weight[at + k * step] : 0.0f;
#pragma unroll
        for (int k = 0; k < N; k++) {
            w[k] = w[k] * keep - j.rate * v[k];
            if (k < n) {
                bad |= !(fabsf(w[k]) <= 3.402823466e38f);
                j.weight[at + k * step] = w[k];
            }
        }
    } else if (j.out_type == kTypeF32) {
        float* o = static_cast<float*>(j.out) + at;
#pragma unroll
        for (int k = 0; k < N; k++)
            if (k < n) o[k * step] = v[k];
    } else {
        uint16_t* o = static_cast<uint16_t*>(j.out) + at;
#pragma unroll
        for (int k = 0; k < N; k++)
            if (k < n)
                o[k * step] = j.out_type == kTypeBF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v[k]))
                                                      : __half_as_ushort(__float2half_rn(v[k]));
    }
}

// One product of every matrix of the call.  Persistent CTAs take 128 x 128 output tiles; one thread streams
// operand tiles (64 along K) through a ring of stages, one thread issues the MMAs into one of two accumulators
// in TMEM, four warps turn the other accumulator into the next operand.  The symmetric products compute the
// upper triangle of tiles and write each tile twice.  `src` says which X buffer is current.
template <int PHASE, bool SPLIT, bool LAST>
__global__ void __launch_bounds__(kThreads, 1) ns_kernel(const __grid_constant__ Jobs q, const int src) {
    using S = Stages<SPLIT>;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kCount * S::kBytes);
    uint64_t *empty = full + S::kCount, *tfull = empty + S::kCount, *tempty = tfull + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles = PHASE == kApply ? q.full_tiles : q.tri_tiles;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kCount; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < 2; s++) {
            mbar_init(&tfull[s], 1);
            mbar_init(&tempty[s], 128);
        }
        fence_barrier_init();
    }
    if (warp == 3) {
        tmem_alloc(tmem_slot, 256);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            int n = 0;   // stages filled
            bool ok = true;
            for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
                const TileAt at = tile_at<PHASE>(q, t);
                const Job& j = q.job[at.job];
                const uint8_t* left = PHASE == kGram ? j.x[src] : PHASE == kSquare ? j.a : j.b;
                const long left_lo = PHASE == kGram ? j.x_bytes : j.a_bytes;
                const int lcb = PHASE == kGram ? j.cb : 2 * j.rb;
                for (int k = 0; k < at.kblocks; k++, n++) {
                    const int s = n % S::kCount;
                    if (!(ok = mbar_wait(&empty[s], ((n / S::kCount) & 1) ^ 1, q.status, kStatusWait))) break;
                    uint8_t* st = smem + s * S::kBytes;
                    mbar_arrive_expect_tx(&full[s], S::kBytes);
                    const uint8_t* a = left + ((long)at.i * lcb + k) * kTileBytes;
                    bulk_load(st, a, kTileBytes, &full[s]);
                    if (SPLIT) bulk_load(st + 2 * kTileBytes, a + left_lo, kTileBytes, &full[s]);
                    if (PHASE == kApply) {
                        // 64 rows of two neighbouring column blocks of X
                        const uint8_t* b =
                            j.x[src] + ((long)(k >> 1) * j.cb + 2 * at.j) * kTileBytes + (k & 1) * (kTileBytes / 2);
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            bulk_load(st + kTileBytes + h * (kTileBytes / 2), b + h * kTileBytes, kTileBytes / 2,
                                      &full[s]);
                            if (SPLIT)
                                bulk_load(st + 3 * kTileBytes + h * (kTileBytes / 2), b + h * kTileBytes + j.x_bytes,
                                          kTileBytes / 2, &full[s]);
                        }
                    } else {
                        const uint8_t* b = left + ((long)at.j * lcb + k) * kTileBytes;
                        bulk_load(st + kTileBytes, b, kTileBytes, &full[s]);
                        if (SPLIT) bulk_load(st + 3 * kTileBytes, b + left_lo, kTileBytes, &full[s]);
                    }
                }
            }
            // no copy is in flight when the CTA ends, even after a wait that gave up
            for (int i = max(0, n - S::kCount); i < n; i++)
                mbar_wait(&full[i % S::kCount], (i / S::kCount) & 1, q.status, kStatusWait);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = idesc_f16(kTile, PHASE == kApply);
            int n = 0, done = 0;
            bool ok = true;
            for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x, done++) {
                const TileAt at = tile_at<PHASE>(q, t);
                const uint32_t d = tmem + (done & 1) * kTile;
                if (!(ok = mbar_wait(&tempty[done & 1], ((done >> 1) & 1) ^ 1, q.status, kStatusWait))) break;
                tc_fence_after();
                for (int k = 0; k < at.kblocks; k++, n++) {
                    const int s = n % S::kCount;
                    if (!(ok = mbar_wait(&full[s], (n / S::kCount) & 1, q.status, kStatusWait))) break;
                    tc_fence_after();
                    const uint32_t st = smem_u32(smem + s * S::kBytes);
                    const uint64_t ah = smem_desc(st, 0, 1024, kLayoutSw128);
                    // MN-major: 64-column blocks 8 KB apart, groups of 8 K rows 1 KB apart, 16 K rows per MMA
                    const uint64_t bh = smem_desc(st + kTileBytes, PHASE == kApply ? kTileBytes / 2 : 0, 1024, kLayoutSw128);
                    constexpr int kStepB = PHASE == kApply ? 2048 / 16 : 2;
                    constexpr uint64_t kLo = 2 * kTileBytes / 16;
#pragma unroll
                    for (int kk = 0; kk < kChunk / 16; kk++) {
                        mma_f16(d, ah + 2 * kk, bh + kStepB * kk, idesc, (k | kk) != 0);
                        if (SPLIT) {
                            mma_f16(d, ah + 2 * kk, bh + kLo + kStepB * kk, idesc, 1);
                            mma_f16(d, ah + kLo + 2 * kk, bh + kStepB * kk, idesc, 1);
                        }
                    }
                    mma_commit(&empty[s]);
                }
                mma_commit(&tfull[done & 1]);
            }
        }
    } else if (warp >= 4) {
        const int w = warp & 3, r = w * 32 + lane;
        int done = 0;
        bool bad = false;
        for (int t = blockIdx.x; t < tiles; t += gridDim.x, done++) {
            const TileAt at = tile_at<PHASE>(q, t);
            const Job& j = q.job[at.job];
            if (!mbar_wait(&tfull[done & 1], (done >> 1) & 1, q.status, kStatusWait)) break;
            tc_fence_after();
            const uint32_t d = tmem + (done & 1) * kTile + ((uint32_t)(w * 32) << 16);
            const int acb = 2 * j.rb;
            // accumulator times: X X^T 2^2p -> A 2^14;  A A 2^28 -> 2^14;  B X 2^(14 + p) -> X 2^p
            const float f = PHASE == kGram ? exp2f((float)(kGramExp - 2 * j.p))
                                           : exp2f((float)-kGramExp) * (PHASE == kSquare ? kNsC : 1.0f);
            const float out_f = exp2f((float)-j.p);
#pragma unroll 1
            for (int c = 0; c < kTile; c += 32) {
                float v[32];
                tmem_ld32(d + c, v);
#pragma unroll
                for (int k = 0; k < 32; k++) v[k] *= f;
                const int cb = PHASE == kApply ? j.cb : acb;
                const long off = ((long)at.i * cb + 2 * at.j + (c >> 6)) * kTileBytes + r * 128;
                const int chunk = (c & 63) >> 3;
                if (PHASE != kGram) {
                    float x[32];
                    const uint8_t* old = (PHASE == kSquare ? j.a : j.x[src]) + off;
                    read32(old, old + (PHASE == kSquare ? j.a_bytes : j.x_bytes), r, SPLIT, chunk, x);
#pragma unroll
                    for (int k = 0; k < 32; k++) v[k] += (PHASE == kSquare ? kNsB : kNsA) * x[k];
                }
                if (LAST) {
                    const int row = at.i * kTile + r, col = at.j * kTile + c;
#pragma unroll
                    for (int k = 0; k < 32; k++) v[k] *= out_f;
                    finish<32>(q, j, row, col, v, bad);
                    continue;
                }
                uint8_t* dst = PHASE == kGram ? j.a : PHASE == kSquare ? j.b : j.x[src ^ 1];
                const long lo = PHASE == kApply ? j.x_bytes : j.a_bytes;
                write32<SPLIT>(dst + off, dst + off + lo, r, chunk, v);
                if (PHASE != kApply && at.i != at.j) {
                    // the mirrored tile: lanes hold consecutive columns of its rows
#pragma unroll
                    for (int k = 0; k < 32; k++) {
                        __half hi, l;
                        split_half(v[k], hi, l);
                        const long m = tile_offset(at.j * kTile + c + k, at.i * kTile + r, acb);
                        *reinterpret_cast<__half*>(dst + m) = hi;
                        if (SPLIT) *reinterpret_cast<__half*>(dst + m + lo) = l;
                    }
                }
            }
            tc_fence_before();
            mbar_arrive(&tempty[done & 1]);
        }
        if (LAST && bad && q.status) atomicExch(q.status, kStatusNonFinite);
    }
    __syncwarp();
    __syncthreads();
    if (warp == 3) {
        tc_fence_after();
        tmem_dealloc(tmem, 256);
    }
}

// ------------------------------------------------------------------ short matrices: one cluster each
//
// A matrix of at most 128 rows (of X) stays on chip for the whole call.  The CTAs of a cluster hold a slab of
// columns each, in shared memory as operand tiles of `rows` x 64 (rows = r rounded up to 16).  Per iteration every
// CTA forms X X^T over its columns, the cluster sums the partial products (each CTA a share of the rows, in rank
// order) and hands every CTA the whole of A; A^2, B and B X are then local.  Three products and two cluster
// barriers per iteration instead of three launches, and U is read and O written once.
// The MMA always takes 128 rows: those past `rows` read whatever follows the tile in shared memory and land in
// accumulator rows that nothing reads.

constexpr int kSlabThreads = 256;
constexpr int kSlabRound = 384;      // columns of B X in TMEM at a time, beside 128 for the products of A
constexpr int kMaxSmem = 227 * 1024;

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
int slab_smem(int rows, int width, bool split) {
    const int tiles = (slab_x_bytes(rows, width) + slab_a_bytes(rows)) * (split ? 2 : 1);
    // the last operand tile may be read for 128 rows
    return 1024 + std::max(tiles + slab_part_bytes(rows), tiles - rows * 128 + 128 * 128);
}

__device__ __forceinline__ void slab_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    return a;
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

// Four values of U from (row, col) on along its contiguous axis of `n` values; `raw` as stored (Muon: grad).
__device__ __forceinline__ float4 load_u4(const void* in, int type, long at, int n, bool vec) {
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (n <= 0) return make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (type == kTypeF32) {
        const float* p = static_cast<const float*>(in) + at;
        if (vec && n >= 4) return *reinterpret_cast<const float4*>(p);
        for (int i = 0; i < 4; i++)
            if (i < n) v[i] = p[i];
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(in) + at;
        uint16_t h[4] = {0, 0, 0, 0};
        if (vec && n >= 4) {
            const uint2 u = *reinterpret_cast<const uint2*>(p);
            h[0] = (uint16_t)u.x, h[1] = (uint16_t)(u.x >> 16), h[2] = (uint16_t)u.y, h[3] = (uint16_t)(u.y >> 16);
        } else {
            for (int i = 0; i < 4; i++)
                if (i < n) h[i] = p[i];
        }
        for (int i = 0; i < 4; i++)
            v[i] = type == kTypeBF16 ? __uint_as_float((uint32_t)h[i] << 16) : __half2float(__ushort_as_half(h[i]));
    }
    return make_float4(v[0], v[1], v[2], v[3]);
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

// D += A B over 16 K elements of operands held as hi (+ lo at byte distance `a_lo`, `b_lo`)
template <bool SPLIT>
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t a_lo, uint64_t b, uint64_t b_lo, uint32_t idesc,
                                         bool accumulate) {
    mma_f16(d, a, b, idesc, accumulate);
    if (SPLIT) {
        mma_f16(d, a, b + b_lo, idesc, 1);
        mma_f16(d, a + a_lo, b, idesc, 1);
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
        for (int i = 0; i < 2 + 2 * q.steps; i++) slab_cluster_sync();
        return;
    }
    const SlabJob& j = q.job[index];
    const int ranks = j.ranks, rank = blockIdx.x - j.first;
    uint32_t peer0;                  // the matrix's first CTA within the cluster
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(peer0));
    peer0 -= rank;
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
    if (warp == 0) {
        tmem_alloc(&tmem_slot, 512);
        tmem_relinquish();
    }

    // momentum and |U|^2: units of four values along U's contiguous axis (X's columns, or its rows when tall)
    const int across = j.tall ? cols : rows, along = j.tall ? rows : tiles * 64;
    const int live_across = j.tall ? cols : j.r, live_along = j.tall ? j.r : cols;
    const int per = along / 4, units = across * per;
    double s = 0.0;
    for (int base = tid; base < units; base += 4 * kSlabThreads) {
        float4 g[4], m[4];
        long at[4];
        int n[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int u = base + i * kSlabThreads, line = u / per, k = (u - line * per) * 4;
            n[i] = u < units && line < live_across ? live_along - k : 0;
            at[i] = (j.tall ? col0 + line : (long)line) * j.in_pitch + (j.tall ? k : col0 + k);
            g[i] = load_u4(j.in, j.in_type, at[i], n[i], j.vec);
            if (j.weight) m[i] = load_u4(j.momentum, kTypeF32, at[i], n[i], j.vec);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float v[4] = {g[i].x, g[i].y, g[i].z, g[i].w};
            if (j.weight) {
                float w[4] = {m[i].x, m[i].y, m[i].z, m[i].w};
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    w[k] = q.momentum * w[k] + q.grad_scale * v[k];
                    v[k] = q.nesterov ? q.grad_scale * v[k] + q.momentum * w[k] : w[k];
                }
                if (j.vec && n[i] >= 4) {
                    *reinterpret_cast<float4*>(j.momentum + at[i]) = make_float4(w[0], w[1], w[2], w[3]);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        if (k < n[i]) j.momentum[at[i] + k] = w[k];
                }
            }
#pragma unroll
            for (int k = 0; k < 4; k++) s += (double)v[k] * v[k];
        }
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
    slab_cluster_sync();
    s = 0.0;
    for (int i = 0; i < ranks; i++) s += peer_load_d(peer_addr(smem_u32(&norm), peer0 + i));
    // a norm of zero gives zeros; one that is not finite gives NaN everywhere
    const double scale = s == 0.0 ? 0.0 : s <= 1.7e308 ? exp2((double)j.p) / sqrt(s) : nan("");

    // X0 = U / |U| times 2^p; zero outside the matrix
    for (int base = tid; base < units; base += 4 * kSlabThreads) {
        float4 g[4], m[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int u = base + i * kSlabThreads, line = u / per, k = (u - line * per) * 4;
            const int n = u < units && line < live_across ? live_along - k : 0;
            const long at = (j.tall ? col0 + line : (long)line) * j.in_pitch + (j.tall ? k : col0 + k);
            g[i] = load_u4(j.in, j.in_type, at, n, j.vec);
            if (j.weight) m[i] = load_u4(j.momentum, kTypeF32, at, n, j.vec);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int u = base + i * kSlabThreads, line = u / per, k0 = (u - line * per) * 4;
            if (u >= units) continue;
            const float v[4] = {g[i].x, g[i].y, g[i].z, g[i].w};
            const float w[4] = {m[i].x, m[i].y, m[i].z, m[i].w};
            __half hi[4], lo[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float d = !j.weight ? v[k] : q.nesterov ? q.grad_scale * v[k] + q.momentum * w[k] : w[k];
                const bool inside = line < live_across && k0 + k < live_along;
                split_half(inside ? (float)(scale * (double)d) : 0.0f, hi[k], lo[k]);
            }
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
    const int row = (warp & 3) * 32 + lane, half = warp >> 2;      // accumulator row; warps share its columns
    const uint32_t trow = (uint32_t)((warp & 3) * 32) << 16;
    const float gram_f = exp2f((float)(kGramExp - 2 * j.p)), back_f = exp2f((float)-kGramExp), out_f = exp2f((float)-j.p);
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
        for (int c = half * 16; c < rows; c += 32) {
            float v[16];
            __syncwarp();
            tmem_ld16(tmem + trow + c, v);
            if (row < rows)
#pragma unroll
                for (int k = 0; k < 4; k++)
                    *reinterpret_cast<float4*>(part + row * pp + c + 4 * k) =
                        tiles ? make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3])
                              : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        tc_fence_before();
        slab_cluster_sync();
        // A = the sum over the cluster: this CTA's share of the rows, handed to everyone
        const int share = rows / ranks, chunks = rows / 8;
        for (int u = tid; u < share * chunks; u += kSlabThreads) {
            const int r = rank * share + u / chunks, c = u % chunks;
            float v[8] = {};
            for (int i = 0; i < ranks; i++) {
                const uint32_t from = peer_addr(ps + (r * pp + c * 8) * 4, peer0 + i);
                const float4 f = peer_load4(from), g = peer_load4(from + 16);
                v[0] += f.x, v[1] += f.y, v[2] += f.z, v[3] += f.w;
                v[4] += g.x, v[5] += g.y, v[6] += g.z, v[7] += g.w;
            }
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] *= gram_f;
            uint4 hi, lo;
            pack8(v, hi, lo);
            const uint32_t to = as + slab_offset(r, c * 8, rows);
            for (int i = 0; i < ranks; i++) {
                peer_store4(peer_addr(to, peer0 + i), hi);
                if (SPLIT) peer_store4(peer_addr(to + a_lo, peer0 + i), lo);
            }
        }
        asm volatile("fence.proxy.async;" ::: "memory");
        slab_cluster_sync();
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
        for (int c = half * 16; c < rows; c += 32) {
            float v[16], old[16];
            __syncwarp();
            tmem_ld16(tmem + trow + c, v);
            if (row < rows) {
                slab_read16<SPLIT>(a, a_lo, row, c, rows, old);
#pragma unroll
                for (int k = 0; k < 16; k++) v[k] = kNsB * old[k] + kNsC * (v[k] * back_f);
                slab_write16<SPLIT>(a, a_lo, row, c, rows, v);
            }
        }
        fence_proxy_async();
        tc_fence_before();
        __syncthreads();
        // X <- a X + B X
        const bool last = step + 1 == q.steps;
        for (int c0 = 0; c0 < tiles * 64; c0 += kSlabRound) {
            const int n = min(kSlabRound, tiles * 64 - c0);
            if (tid == 0) {
                tc_fence_after();
                for (int n0 = 0; n0 < n; n0 += 256) {
                    const uint64_t b = dx_mn + (c0 + n0) / 64 * tile;
                    for (int kk = 0; kk < rows / 16; kk++)
                        mma_pair<SPLIT>(tmem + 128 + n0, da + (kk >> 2) * tile + 2 * (kk & 3), da_lo, b + kk * (2048 / 16),
                                        dx_lo, idesc_f16(min(256, n - n0), 1), kk != 0);
                }
                mma_commit(&bar);
            }
            __syncwarp();
            mbar_wait(&bar, phase, q.status, kStatusWait);
            phase ^= 1;
            tc_fence_after();
            for (int c = half * 16; c < n; c += 32) {
                float v[16], old[16];
                __syncwarp();
                tmem_ld16(tmem + 128 + trow + c, v);
                if (row >= rows) continue;
                slab_read16<SPLIT>(x, x_lo, row, c0 + c, rows, old);
#pragma unroll
                for (int k = 0; k < 16; k++) v[k] = kNsA * old[k] + v[k] * back_f;
                if (!last) {
                    slab_write16<SPLIT>(x, x_lo, row, c0 + c, rows, v);
                } else {
#pragma unroll
                    for (int k = 0; k < 16; k++) v[k] *= out_f;
                    finish<16>(q, j, row, col0 + c0 + c, v, bad);
                }
            }
            fence_proxy_async();
            tc_fence_before();
            __syncthreads();
        }
    }
    if (bad && q.status) atomicExch(q.status, kStatusNonFinite);
    slab_cluster_sync();   // no CTA leaves while a peer may read its shared memory
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
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
    long bytes(bool split) const { return (2 * x_bytes + 2 * a_bytes) * (split ? 2 : 1); }
};

constexpr long kNormBytes = (long)kMaxJobs * kMaxNormParts * sizeof(double);

long round_up(long v, long to) { return (v + to - 1) / to * to; }

int scale_exponent(const Shape& s) {
    return std::min(15, (int)std::floor(0.5 * std::log2((double)s.r * s.c)));
}

void layout_job(Job& j, const Shape& s, bool split, uint8_t*& at, const double* norm, int index) {
    j.rb = s.rb, j.cb = s.cb;
    j.x_bytes = s.x_bytes, j.a_bytes = s.a_bytes;
    const int halves = split ? 2 : 1;
    j.x[0] = at;
    j.x[1] = j.x[0] + halves * s.x_bytes;
    j.a = j.x[1] + halves * s.x_bytes;
    j.b = j.a + halves * s.a_bytes;
    at = j.b + halves * s.a_bytes;
    j.norm = norm + (long)index * kMaxNormParts;
}

template <int PHASE, bool SPLIT, bool LAST>
void launch_ns(const Jobs& q, int src, cudaStream_t stream) {
    using S = Stages<SPLIT>;
    static PerDeviceOnce once;
    once_per_device(once, [] { set_max_dynamic_smem(ns_kernel<PHASE, SPLIT, LAST>, S::kSmem, "ns_kernel"); });
    const int tiles = PHASE == kApply ? q.full_tiles : q.tri_tiles;
    ns_kernel<PHASE, SPLIT, LAST><<<std::min(tiles, device_sms()), kThreads, S::kSmem, stream>>>(q, src);
    launch_check("ns_kernel");
}

template <bool SPLIT>
void run_jobs(Jobs& q, double* parts, cudaStream_t stream) {
    long elems = 0, xtiles = 0;
    q.tri_tiles = q.full_tiles = 0;
    for (int i = 0; i < q.count; i++) {
        Job& j = q.job[i];
        j.tri0 = q.tri_tiles;
        j.full0 = q.full_tiles;
        q.tri_tiles += j.rb * (j.rb + 1) / 2;
        q.full_tiles += j.rb * (j.cb / 2);
        elems = std::max(elems, (long)j.r * j.c);
        xtiles = std::max(xtiles, (long)j.rb * j.cb);
    }
    q.norm_parts = (int)std::min<long>(kMaxNormParts, (elems + 4095) / 4096);
    norm_kernel<<<dim3(q.norm_parts, q.count), 256, 0, stream>>>(q, parts);
    launch_check("norm_kernel");
    pack_kernel<SPLIT><<<dim3((unsigned)std::min<long>(xtiles, 2048), q.count), 256, 0, stream>>>(q);
    launch_check("pack_kernel");
    for (int s = 0; s < q.steps; s++) {
        launch_ns<kGram, SPLIT, false>(q, s & 1, stream);
        launch_ns<kSquare, SPLIT, false>(q, s & 1, stream);
        if (s + 1 < q.steps)
            launch_ns<kApply, SPLIT, false>(q, s & 1, stream);
        else
            launch_ns<kApply, SPLIT, true>(q, s & 1, stream);
    }
}

// CTAs a matrix takes on the cluster path (a power of two up to 8), 0 where it does not fit.  One per 64 columns,
// which shortens every pass over X, but no more than 128 / matrices where they fit: 128 CTAs is what clusters of eight
// with one CTA per SM can hold at a time (two in each of the GPU's eight groups of SMs).
int slab_ranks(const Shape& s, bool split, size_t matrices) {
    if (s.r > 128) return 0;
    const int rows = (s.r + 15) / 16 * 16;
    for (int ranks = 1; ranks <= 8; ranks *= 2) {
        const int width = (s.c + 64 * ranks - 1) / (64 * ranks) * 64;
        if (slab_smem(rows, width, split) > kMaxSmem - 1024) continue;
        if (ranks == 8 || width == 64 || 2 * ranks * matrices > 128) return ranks;
    }
    return 0;
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
        smem = std::max(smem, slab_smem(j.rows, j.width, SPLIT));
    }
    static PerDeviceOnce once;
    once_per_device(once, [] { set_max_dynamic_smem(slab_kernel<SPLIT, N>, kMaxSmem - 1024, "slab_kernel"); });
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
void run_sources(const Settings& set, const std::vector<Source>& list, void* workspace, cudaStream_t stream) {
    std::vector<SlabJob> slabs;
    std::vector<Source> tiled;
    for (const Source& s : list) {
        SlabJob j{};
        static_cast<Source&>(j) = s;
        j.ranks = slab_ranks(Shape(s.r, s.c), SPLIT, list.size());
        if (!j.ranks) {
            tiled.push_back(s);
            continue;
        }
        j.rows = (s.r + 15) / 16 * 16;
        j.width = (s.c + 64 * j.ranks - 1) / (64 * j.ranks) * 64;
        slabs.push_back(j);
    }
    std::stable_sort(slabs.begin(), slabs.end(), [](const SlabJob& a, const SlabJob& b) {
        return a.ranks != b.ranks ? a.ranks > b.ranks : (long)a.rows * a.width > (long)b.rows * b.width;
    });
    for (size_t first = 0; first < slabs.size(); first += kMaxJobs) {
        const std::vector<SlabJob> part(slabs.begin() + first,
                                        slabs.begin() + std::min<size_t>(slabs.size(), first + kMaxJobs));
        if (part.size() == 1)
            launch_slabs<SPLIT, 1>(set, part, stream);
        else
            launch_slabs<SPLIT, kMaxJobs>(set, part, stream);
    }
    double* parts = reinterpret_cast<double*>(round_up(reinterpret_cast<intptr_t>(workspace), 1024));
    Jobs q{};
    static_cast<Settings&>(q) = set;
    uint8_t* at = nullptr;
    for (size_t i = 0; i < tiled.size(); i++) {
        if (q.count == 0) at = reinterpret_cast<uint8_t*>(parts) + kNormBytes;
        Job& j = q.job[q.count];
        j = Job{};
        static_cast<Source&>(j) = tiled[i];
        layout_job(j, Shape(j.r, j.c), SPLIT, at, parts, q.count);
        if (++q.count == kMaxJobs || i + 1 == tiled.size()) {
            run_jobs<SPLIT>(q, parts, stream);
            q.count = 0;
        }
    }
}

// Bytes of the tiled path for these shapes; its chunks of kMaxJobs matrices run one after another in the same
// memory.  A call whose matrices all take the cluster path needs none, but the size may not depend on which
// matrices of a list are active, so every matrix counts.
size_t tiled_bytes(const std::vector<Shape>& shapes, bool split) {
    long sum = 0;
    for (const Shape& s : shapes) sum += s.bytes(split);
    return (size_t)(kNormBytes + sum + 1024);
}

bool aligned16(const void* p, long pitch_bytes, int bytes) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && pitch_bytes % bytes == 0;
}

}  // namespace

size_t muon_workspace_bytes(const MuonMatrix* m, int count, bool split) {
    std::vector<Shape> shapes;
    for (int i = 0; i < count; i++)
        if (m[i].rows && m[i].cols) shapes.emplace_back(m[i].rows, m[i].cols);
    return tiled_bytes(shapes, split);
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
        s.vec = aligned16(s.in, s.in_pitch * 4, 16) && aligned16(s.momentum, s.in_pitch * 4, 16) &&
                aligned16(s.weight, s.in_pitch * 4, 16);
        list.push_back(s);
    }
    if (rule.split)
        run_sources<true>(set, list, workspace, stream);
    else
        run_sources<false>(set, list, workspace, stream);
}

size_t orthogonalize_workspace_bytes(int rows, int cols, int out_type) {
    if (rows == 0 || cols == 0) return 0;
    return tiled_bytes({Shape(rows, cols)}, out_type == kTypeF32);
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
    s.vec = aligned16(in, in_pitch * bytes, 4 * bytes);
    if (out_type == kTypeF32)
        run_sources<true>(set, {s}, workspace, stream);
    else
        run_sources<false>(set, {s}, workspace, stream);
}

}  // namespace sy
