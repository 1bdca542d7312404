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

struct Job {
    uint8_t *x[2], *a, *b;      // hi tiles; the lo tiles follow at x_bytes / a_bytes
    long x_bytes, a_bytes;
    const double* norm;         // partial sums of squares of U
    const void* in;             // orthogonalisation: U;  Muon: grad
    float *weight, *momentum;
    void* out;
    long in_pitch, out_pitch;
    int r, c;                   // X is r x c
    int rb, cb;                 // 128-row blocks of X; 64-column blocks (padded to a whole tile)
    int tall;                   // X is U transposed
    int p;                      // X is held times 2^p
    int in_type, out_type;
    float rate;                 // Muon: factor of O in the update
    int tri0, full0;            // first tile of this job in the symmetric and in the full products
};

struct Jobs {
    int count, tri_tiles, full_tiles, norm_parts;
    int steps, nesterov;
    float lr, momentum, decay, grad_scale;
    int* status;
    Job job[kMaxJobs];
};
static_assert(sizeof(Jobs) <= 32000, "job table exceeds the kernel parameters");

// element (row, col) of U: the orthogonalisation's input or Muon's direction
__device__ __forceinline__ float direction(const Jobs& q, const Job& j, long row, long col) {
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

// value v of O at (row, col) of X's orientation: the output, or the weight update
__device__ __forceinline__ void finish(const Jobs& q, const Job& j, int row, int col, float v, bool& bad) {
    if (row >= j.r || col >= j.c) return;
    const long at = j.tall ? col * j.out_pitch + row : row * j.out_pitch + col;
    if (j.weight) {
        const float w = j.weight[at] * (1.0f - q.lr * q.decay) - j.rate * v;
        bad |= !(fabsf(w) <= 3.402823466e38f);
        j.weight[at] = w;
    } else if (j.out_type == kTypeF32) {
        static_cast<float*>(j.out)[at] = v;
    } else if (j.out_type == kTypeBF16) {
        static_cast<__nv_bfloat16*>(j.out)[at] = __float2bfloat16_rn(v);
    } else {
        static_cast<__half*>(j.out)[at] = __float2half_rn(v);
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
                    for (int k = 0; k < 32; k++) finish(q, j, row, col + k, v[k] * out_f, bad);
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

void layout_job(Job& j, const Shape& s, bool split, uint8_t*& at, const double* norm, int index) {
    j.r = s.r, j.c = s.c, j.rb = s.rb, j.cb = s.cb;
    j.x_bytes = s.x_bytes, j.a_bytes = s.a_bytes;
    const int halves = split ? 2 : 1;
    j.x[0] = at;
    j.x[1] = j.x[0] + halves * s.x_bytes;
    j.a = j.x[1] + halves * s.x_bytes;
    j.b = j.a + halves * s.a_bytes;
    at = j.b + halves * s.a_bytes;
    j.p = std::min(15, (int)std::floor(0.5 * std::log2((double)s.r * s.c)));
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

}  // namespace

size_t muon_workspace_bytes(const MuonMatrix* m, int count, bool split) {
    // chunks of kMaxJobs matrices run one after another in the same memory
    long most = 0, sum = 0;
    int n = 0;
    for (int i = 0; i < count; i++) {
        if (m[i].rows == 0 || m[i].cols == 0) continue;
        sum += Shape(m[i].rows, m[i].cols).bytes(split);
        most = std::max(most, sum);
        if (++n == kMaxJobs) n = 0, sum = 0;
    }
    return (size_t)(kNormBytes + most + 1024);
}

void muon_update(const MuonMatrix* m, int count, const MuonRule& rule, void* workspace, int* status,
                 cudaStream_t stream) {
    double* parts = reinterpret_cast<double*>(round_up(reinterpret_cast<intptr_t>(workspace), 1024));
    Jobs q{};
    q.steps = rule.steps;
    q.nesterov = rule.nesterov;
    q.lr = rule.lr, q.momentum = rule.momentum, q.decay = rule.decay, q.grad_scale = rule.grad_scale;
    q.status = status;
    uint8_t* at = nullptr;
    auto flush = [&] {
        if (!q.count) return;
        if (rule.split)
            run_jobs<true>(q, parts, stream);
        else
            run_jobs<false>(q, parts, stream);
        q.count = 0;
    };
    for (int i = 0; i < count; i++) {
        if (m[i].rows == 0 || m[i].cols == 0) continue;
        if (q.count == 0) at = reinterpret_cast<uint8_t*>(parts) + kNormBytes;
        Job& j = q.job[q.count];
        j = Job{};
        layout_job(j, Shape(m[i].rows, m[i].cols), rule.split, at, parts, q.count);
        j.tall = m[i].rows > m[i].cols;
        j.in = m[i].grad;
        j.weight = m[i].weight;
        j.momentum = m[i].momentum;
        j.in_pitch = j.out_pitch = m[i].cols;
        j.rate = (float)((double)rule.lr * rule.rms * std::sqrt((double)std::max(m[i].rows, m[i].cols)));
        if (++q.count == kMaxJobs) flush();
    }
    flush();
}

size_t orthogonalize_workspace_bytes(int rows, int cols, int out_type) {
    if (rows == 0 || cols == 0) return 0;
    return (size_t)(kNormBytes + Shape(rows, cols).bytes(out_type == kTypeF32) + 1024);
}

void orthogonalize(const void* in, int in_type, long in_pitch, int rows, int cols, int steps, void* out, int out_type,
                   long out_pitch, void* workspace, int* status, cudaStream_t stream) {
    if (rows == 0 || cols == 0) return;
    const bool split = out_type == kTypeF32;
    double* parts = reinterpret_cast<double*>(round_up(reinterpret_cast<intptr_t>(workspace), 1024));
    uint8_t* at = reinterpret_cast<uint8_t*>(parts) + kNormBytes;
    Jobs q{};
    q.count = 1;
    q.steps = steps;
    q.status = status;
    Job& j = q.job[0];
    layout_job(j, Shape(rows, cols), split, at, parts, 0);
    j.tall = rows > cols;
    j.in = in, j.in_type = in_type, j.in_pitch = in_pitch;
    j.out = out, j.out_type = out_type, j.out_pitch = out_pitch;
    if (split)
        run_jobs<true>(q, parts, stream);
    else
        run_jobs<false>(q, parts, stream);
}

}  // namespace sy
