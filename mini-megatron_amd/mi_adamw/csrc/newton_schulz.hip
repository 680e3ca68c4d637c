// newton_schulz.hip -- Newton-Schulz orthogonalisation and the Muon step built on it (gfx950).
//
// For a matrix U with m = min(rows, cols), n = max(rows, cols), seen with its smaller side as
// rows (an n x m matrix is worked on as its transpose: the iteration commutes with it):
//   X = U / max(|U|_F, eps);   then `steps` times
//   S = X X^T                  (m x m)
//   P = b S + c S^2            (m x m)
//   X = a X + P X              (m x n)
//
// The three products of a step run on the matrix cores in fp16 with fp32 sums.  Singular
// values of X stay below 2 (the host checks it for the coefficients), so every entry does, and
// powers of two known beforehand use fp16's whole range: X is held times 2^15, S times 2^14,
// P times 2^13.  Two forms:
//   half    one product of fp16 values.  What fp16's 11 bits would lose is kept where it
//           counts.  X is carried in two fp16 terms (22 bits), since a^5 = 485 multiplies the
//           rounding of small singular directions; the product reads the first term.  The
//           diagonals of S and P, their largest entries, are held apart in fp32 and enter the
//           elementwise part.  Against 64 bits, relative: 3e-4 to 7e-4 on gradients' spectra
//           and full ranks, below the 1.7e-3 of rounding the result to bf16 (1e-3 to 6e-3
//           without the two); up to 2e-3 for low ranks, dense or in few rows, and 4e-3 where a
//           handful of entries is all there is, since nothing averages their roundings.
//           (The same iteration in bf16: 1e-2 to 2e-2, and 0.1 to 1.6 for low ranks.)
//   single  every operand in two fp16 terms, hi hi + hi lo + lo hi: fp32's error (1e-6 against
//           64 bits on gradients' spectra, up to 1.4e-4 at rank one, as the same iteration in
//           fp32 has).
//
// X is stored as its transpose T [n][m] alone, padded with zeros to multiples of 64, which every
// product keeps zero.  P X reads it with its summed index contiguous; X X^T sums over T's rows and
// has LDS turn the operands round on the way into registers (ds_read_b64_tr_b16).

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>

#include <cmath>

#include "mi_adamw.h"
#include "fp32_math.h"
#include "items.h"

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4_mem __attribute__((aligned(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_mem __attribute__((aligned(2)));

#define GLOBAL __attribute__((address_space(1)))
#define CONSTANT __attribute__((address_space(4)))
#define SHARED __attribute__((address_space(3)))

constexpr float kScaleX = 32768.0f, kScaleS = 16384.0f, kScaleP = 8192.0f;
constexpr int kPad = 64;
constexpr int kBlock = 64;          // rows and columns of a block of the elementwise passes
constexpr int kMaxParts = 512;      // partial sums of squares of a matrix
constexpr int kMaxSplit = 512;      // tiles of S whose sum may be shared out
constexpr int kThreads = 256;

struct Quintic {
    float a, b, c;
};

// Where the parts of one matrix's workspace lie, in bytes from its beginning.
struct Layout {
    int32_t m, n, mp, np;
    int64_t t, s, p, ds, dp, counts, bytes;
    int64_t parts;                  // shares of the norm, then of P's trace
    int64_t t_lo, sq_lo;            // from a first term to its second
    int64_t t_turn;                 // from the transpose one step reads to the next one's
};

__host__ __device__ inline Layout layout_of(int32_t rows, int32_t cols, bool single) {
    Layout l;
    l.m = rows < cols ? rows : cols;
    l.n = rows < cols ? cols : rows;
    l.mp = (l.m + kPad - 1) / kPad * kPad;
    l.np = (l.n + kPad - 1) / kPad * kPad;
    const int64_t big = int64_t(l.mp) * l.np * 2, sq = int64_t(l.mp) * l.mp * 2;
    l.t_lo = big;
    l.t_turn = 2 * big;
    l.t = 0;
    l.sq_lo = sq;
    l.s = 4 * big;
    l.p = l.s + (single ? 2 * sq : sq);
    l.ds = l.p + (single ? 2 * sq : sq);
    l.dp = l.ds + int64_t(l.mp) * 4;
    l.parts = l.dp + int64_t(l.mp) * 4;
    l.counts = l.parts + kMaxParts * 8;
    l.bytes = l.counts + kMaxSplit * 4;     // a multiple of 256
    return l;
}

__host__ __device__ inline int32_t blocks_of(int32_t rows, int32_t cols) {
    return ((rows + kBlock - 1) / kBlock) * ((cols + kBlock - 1) / kBlock);
}
__host__ __device__ inline int32_t parts_of(int32_t rows, int32_t cols) {
    const int32_t b = blocks_of(rows, cols);
    return b < kMaxParts ? b : kMaxParts;
}

// How many workgroups share the sum of one tile of S (over n), of `want`: each for four stages or
// more, and their sums in fp32 have to fit the buffer that the iterate before last leaves free.
__host__ __device__ inline int32_t split_of(const Layout& l, int32_t tile, int32_t want) {
    const int32_t down = (l.mp + tile - 1) / tile, tiles = down * (down + 1) / 2;
    if (want <= 1 || tiles > kMaxSplit) return 1;
    const int64_t fit = l.t_turn / (int64_t(tiles) * tile * tile * 4);
    const int32_t long_enough = l.np / (4 * kPad);
    int32_t n = want < long_enough ? want : long_enough;
    if (fit < n) n = static_cast<int32_t>(fit);
    return n < 1 ? 1 : n;
}

// ---------------------------------------------------------------------------
// Work sources: which matrix a workgroup works on, and its item of that matrix.

struct Item {
    mi_adamw_matrix mat;
    int32_t row;         // of the tables
    int32_t index;
};

// Equal matrices at fixed strides (mi_adamw_newton_schulz).
struct BatchSource {
    mi_adamw_matrix mat;
    const void* x;
    void* out;
    int64_t x_batch, x_row, out_batch, out_row;
    int64_t ws_batch;
    int32_t per;         // items of a matrix, in this launch
    int32_t bf16;
    // Workgroup w runs on XCD w % 8, whose L2 its neighbours share: each XCD takes one run of
    // the items.
    static __device__ __forceinline__ uint32_t order(uint32_t w, uint32_t n) {
        const uint32_t x = w & 7, rest = n & 7;
        return x * (n >> 3) + (x < rest ? x : rest) + (w >> 3);
    }
    __device__ __forceinline__ Item get(uint32_t w) const {
        Item it;
        it.row = w / per;
        it.index = w - it.row * per;
        it.mat = mat;
        it.mat.workspace = it.row * ws_batch;
        return it;
    }
};

// The matrices of an optimizer, through tables (mi_adamw_muon_step).
struct TableSource {
    const mi_adamw_tensor* tensors;
    const mi_adamw_matrix* mats;
    const mi_adamw_chunk* items;
    // Runs of 16 items an XCD, for matrices of different lengths to be spread over all of them.
    static __device__ __forceinline__ uint32_t order(uint32_t w, uint32_t n) {
        return static_cast<uint32_t>(item_order<16>(w, n));
    }
    __device__ __forceinline__ Item get(uint32_t w) const {
        // the tables do not change while a launch runs: scalar loads
        const CONSTANT int32_t* i = (const CONSTANT int32_t*)(items + w);
        Item it;
        it.row = i[0];
        it.index = i[1];
        const CONSTANT mi_adamw_matrix* m = (const CONSTANT mi_adamw_matrix*)(mats) + it.row;
        it.mat.workspace = m->workspace;
        it.mat.rows = m->rows;
        it.mat.cols = m->cols;
        it.mat.lr_ratio = m->lr_ratio;
        it.mat.reserved = 0;
        return it;
    }
};

// ---------------------------------------------------------------------------
// Elementwise passes

__device__ __forceinline__ float lerp1(float from, float to, float w) {
    const float d = to - from;
    return __builtin_fabsf(w) < 0.5f ? __builtin_fmaf(w, d, from)
                                     : __builtin_fmaf(-d, 1.0f - w, to);
}

// Up to four elements from p (element-aligned); `count` of them are there.
__device__ __forceinline__ f32x4 ld_f32(const float* p, int count) {
    if (count >= 4) return *(const GLOBAL f32x4_mem*)(p);
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = 0; k < 3; ++k)
        if (k < count) v[k] = *(const GLOBAL float*)(p + k);
    return v;
}
__device__ __forceinline__ void st_f32(float* p, f32x4 v, int count) {
    if (count >= 4) {
        *(GLOBAL f32x4_mem*)(p) = v;
        return;
    }
    for (int k = 0; k < 3; ++k)
        if (k < count) *(GLOBAL float*)(p + k) = v[k];
}
__device__ __forceinline__ f32x4 ld_bf16(const uint16_t* p, int count) {
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (count >= 4) {
        const u32x2 w = *(const GLOBAL u32x2_mem*)(p);
        v[0] = __uint_as_float(w.x << 16);
        v[1] = __uint_as_float(w.x & 0xffff0000u);
        v[2] = __uint_as_float(w.y << 16);
        v[3] = __uint_as_float(w.y & 0xffff0000u);
        return v;
    }
    for (int k = 0; k < 3; ++k)
        if (k < count) v[k] = __uint_as_float(uint32_t(*(const GLOBAL uint16_t*)(p + k)) << 16);
    return v;
}

__device__ __forceinline__ void st_bf16(uint16_t* p, f32x4 v, int count) {
    if (count >= 4) {
        u32x2 w;
        w.x = bf16x2_bits(v[0], v[1]);
        w.y = bf16x2_bits(v[2], v[3]);
        *(GLOBAL u32x2_mem*)(p) = w;
        return;
    }
    for (int k = 0; k < 3; ++k)
        if (k < count) *(GLOBAL uint16_t*)(p + k) = static_cast<uint16_t>(bf16_bits(v[k]));
}

struct Momentum {
    float lerp_w;        // 1 - momentum
    float momentum;
    int32_t nesterov;
};

// The matrix to orthogonalise, four elements of row r from column c on.
// kFirst: the pass that also updates what it is formed from.
template <bool kFirst>
__device__ __forceinline__ f32x4 update_of(const BatchSource& src, const Item& it, int64_t r,
                                           int32_t c, int count, const Momentum&) {
    const int64_t at = it.row * src.x_batch + r * src.x_row + c;
    return src.bf16 ? ld_bf16(static_cast<const uint16_t*>(src.x) + at, count)
                    : ld_f32(static_cast<const float*>(src.x) + at, count);
}
template <bool kFirst>
__device__ __forceinline__ f32x4 update_of(const TableSource& src, const Item& it, int64_t r,
                                           int32_t c, int count, const Momentum& h) {
    const mi_adamw_tensor* t = src.tensors + it.row;
    const int64_t at = r * it.mat.cols + c;
    float* mp = static_cast<float*>(t->exp_avg) + at;
    const f32x4 g = ld_f32(t->grad + at, count);
    f32x4 m = ld_f32(mp, count);
    if (kFirst) {
        for (int k = 0; k < 4; ++k) m[k] = lerp1(m[k], g[k], h.lerp_w);
        st_f32(mp, m, count);
    }
    if (!h.nesterov) return m;
    f32x4 u;
    for (int k = 0; k < 4; ++k) u[k] = lerp1(g[k], m[k], h.momentum);
    return u;
}

__device__ __forceinline__ void split2(f32x4 v, half4& hi, half4& lo) {
    for (int e = 0; e < 4; ++e) {
        hi[e] = static_cast<_Float16>(v[e]);
        lo[e] = static_cast<_Float16>(v[e] - static_cast<float>(hi[e]));
    }
}

__device__ __forceinline__ double block_sum(double v, double* lds) {
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// Sums of squares of the matrices to orthogonalise, in 64 bits (parts_of() a matrix, in a
// fixed order), with the momentum's update.  Bound by memory: 85M parameters, 12 bytes each, 200 us
// (5.1 TB/s).
template <class Src>
__global__ __launch_bounds__(kThreads) void mi_adamw_ns_sumsq_kernel(Src src, Momentum h,
                                                                     char* ws, int32_t single) {
    __shared__ double lds[4];
    const Item it = src.get(blockIdx.x);
    const Layout l = layout_of(it.mat.rows, it.mat.cols, single);
    const int32_t across = (it.mat.cols + kBlock - 1) / kBlock;
    const int32_t blocks = blocks_of(it.mat.rows, it.mat.cols);
    const int32_t parts = parts_of(it.mat.rows, it.mat.cols);
    double sum = 0.0;
    for (int32_t b = it.index; b < blocks; b += parts) {
        const int32_t r0 = b / across * kBlock, c = b % across * kBlock + (threadIdx.x & 15) * 4;
        const int count = it.mat.cols - c;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int32_t r = r0 + k * 16 + (threadIdx.x >> 4);
            if (r < it.mat.rows && count > 0) {
                const f32x4 u = update_of<true>(src, it, r, c, count, h);
                for (int q = 0; q < 4; ++q) sum += double(u[q]) * u[q];
            }
        }
    }
    sum = block_sum(sum, lds);
    if (threadIdx.x == 0)
        reinterpret_cast<double*>(ws + it.mat.workspace + l.parts)[it.index] = sum;
}

// X^T = U^T / max(|U|, eps) in two fp16 terms; the padding is zeroed.  One 64 x 64 block of the
// padded matrix a workgroup, turned round in LDS where the matrix is wide.  Bound by memory: 85M
// parameters, 12 bytes each, 218 us (4.7 TB/s).
template <class Src>
__global__ __launch_bounds__(kThreads) void mi_adamw_ns_load_kernel(Src src, Momentum h, float eps,
                                                                    char* ws, int32_t single) {
    __shared__ double lds[4];
    __shared__ float tile[kBlock][kBlock + 1];
    const Item it = src.get(blockIdx.x);
    const int32_t rows = it.mat.rows, cols = it.mat.cols;
    const Layout l = layout_of(rows, cols, single);
    char* base = ws + it.mat.workspace;
    const double* part = reinterpret_cast<const double*>(base + l.parts);
    const int32_t parts = parts_of(rows, cols);
    double sum = 0.0;
    for (int32_t k = threadIdx.x; k < parts; k += kThreads) sum += part[k];
    const double norm = sqrt(block_sum(sum, lds));      // 64 bits: no overflow, no rounding
    const double inv = double(kScaleX) / (norm < eps ? eps : norm);
    const int32_t across = (cols + kBlock - 1) / kBlock;
    const int32_t r0 = it.index / across * kBlock, c0 = it.index % across * kBlock;
    const int32_t q = (threadIdx.x & 15) * 4, y0 = threadIdx.x >> 4;
    f32x4 u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int32_t r = r0 + k * 16 + y0, count = cols - c0 - q;
        u[k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (r < rows && count > 0) u[k] = update_of<false>(src, it, r, c0 + q, count, h);
        for (int e = 0; e < 4; ++e) u[k][e] = static_cast<float>(u[k][e] * inv);
    }
    const bool wide = rows <= cols;
    if (wide) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            for (int e = 0; e < 4; ++e) tile[k * 16 + y0][q + e] = u[k][e];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; ++k)
            for (int e = 0; e < 4; ++e) u[k][e] = tile[q + e][k * 16 + y0];
    }
    if (it.index == 0)
        for (int32_t k = threadIdx.x; k < kMaxSplit; k += kThreads)
            reinterpret_cast<uint32_t*>(base + l.counts)[k] = 0;
    // rows of X^T and columns
    const int32_t t0 = wide ? c0 : r0, i0 = wide ? r0 : c0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        half4 a, b;
        split2(u[k], a, b);
        char* at = base + l.t + (int64_t(t0 + k * 16 + y0) * l.mp + i0 + q) * 2;
        *(GLOBAL half4*)(at) = a;
        *(GLOBAL half4*)(at + l.t_lo) = b;
    }
}

// ---------------------------------------------------------------------------
// Products

enum Phase { kPhaseS, kPhaseP, kPhaseX, kPhaseLast };

struct MuonOut {
    float wd_factor;     // 1 - lr * weight_decay
    float neg_lr;
    int32_t copy;        // write param_copy
};

// Four results along a row of the matrix as stored, from column c on; `count` of them are there.
__device__ __forceinline__ void write_out(const BatchSource& src, const Item& it, int32_t r,
                                          int32_t c, f32x4 v, int count, const MuonOut&) {
    const int64_t at = it.row * src.out_batch + int64_t(r) * src.out_row + c;
    if (src.bf16) st_bf16(static_cast<uint16_t*>(src.out) + at, v, count);
    else st_f32(static_cast<float*>(src.out) + at, v, count);
}
__device__ __forceinline__ void write_out(const TableSource& src, const Item& it, int32_t r,
                                          int32_t c, f32x4 v, int count, const MuonOut& o) {
    const CONSTANT uint64_t* t = (const CONSTANT uint64_t*)(src.tensors + it.row);
    const int64_t at = int64_t(r) * it.mat.cols + c;
    float* p = reinterpret_cast<float*>(t[0]) + at;
    const float step = o.neg_lr * it.mat.lr_ratio;
    f32x4 q = ld_f32(p, count);
    for (int e = 0; e < 4; ++e) q[e] = __builtin_fmaf(step, v[e], q[e] * o.wd_factor);
    st_f32(p, q, count);
    if (o.copy) st_bf16(reinterpret_cast<uint16_t*>(t[4]) + at, q, count);
}

__device__ __forceinline__ f32x4 join2(const char* hi, int64_t lo) {
    const half4 a = *(const GLOBAL half4*)(hi), b = *(const GLOBAL half4*)(hi + lo);
    f32x4 v;
    for (int e = 0; e < 4; ++e) v[e] = static_cast<float>(a[e]) + static_cast<float>(b[e]);
    return v;
}

// An address that is the same in every lane, in scalar registers.
__device__ __forceinline__ const char* uniform(const char* p) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    const uint64_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(int(uint32_t(a))));
    const uint64_t hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(int(uint32_t(a >> 32))));
    return reinterpret_cast<const char*>(hi << 32 | lo);
}
// 16 bytes a lane from global memory (a wave-uniform base, a 32-bit offset a lane) to LDS at the
// wave-uniform byte `to` + lane * 16.  In flight until wait_stages(): the compiler does not count
// these loads, and would wait for all of them at every read of LDS if it did.
// (m0 is declared as written, for the compiler's own uses of it; it warns that it reserves m0.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_lds(uint32_t to, const char* base, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :: "s"(to), "v"(offset), "s"(base) : "m0", "memory");
}
#pragma clang diagnostic pop
// This wave's loads but the last kLeft have landed and its reads of LDS are done; then the same of
// the whole workgroup.
template <int kLeft>
__device__ __forceinline__ void wait_stages() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(kLeft) : "memory");
}

// One kT x kT tile of a product.  The left operand's index i counts columns of T, the right one's
// j rows of T (columns of S and P are the same as rows).
//   kPhaseS           sum over T's rows: both operands lie [sum][i], kBK x kT a stage
//   kPhaseP, X, Last  both lie [i][sum], kT rows of kBK a stage
// A ring of kStages stages of LDS; stages are loaded while the ones before them are multiplied, one
// barrier a stage.
//
// What bounds it: the bytes from L2 to LDS, 8 / kT of a byte for each multiply-add and term.  4096 x
// 16384, X's launch (tiles of 256): 494 to 504 us, 1.09 to 1.11 PFLOP/s beside 9.1 TB/s from L2, 24%
// of them misses; the whole call 4.63 ms, 3.66 with the products left out (11.7 TB/s) and 3.84 with
// the loads left out.  S at tiles of 192: 330 us, 830 TFLOP/s.  A fp16 library product of 8192
// reaches 1.27 PFLOP/s on this card.  With a short sum the results count as well: X of 12 x
// 768 x 3072 reads and writes 8 bytes an entry, 226 MB beside its operands in 80 us, at 540 TFLOP/s.
// Measured steps, 12 x 768 x 3072 and 4096 x 16384, us a call: a stage at a time in tiles of 128, X
// stored both ways 1453, 7350; the ring, one transposed X, tiles of 256 1173, 6214; the old
// and new iterate in whole lines 776, 5281; tiles of 192 by rounds, 128 with 4 stages and 8
// waves (2 and 4: 826) 767, 4716; the old iterate read before the last stages and tiles in
// bands per XCD 658, 4547.
// Tiles of 256 in single precision: stages of 32, so that two fit; 4 x 2048 x 8192 8.75 ms with
// tiles of 128, 6.70 with 256 alone.
template <int kT, bool kSingle>
struct Shape {
    static constexpr int kTerms = kSingle ? 2 : 1;
    // two a SIMD: one reads LDS while the other multiplies (four: 2045 x 511 fp32 173 us, 159 with
    // eight)
    static constexpr int kWaves = 8;
    static constexpr int kAcross = kWaves / 2;          // waves along j; two along i
    static constexpr int kFi = kT / 2 / 16, kFj = kT / kAcross / 16;
    static constexpr int kG = kFi % 4 == 0 ? 4 : 2, kGj = kFj % 4 == 0 ? 4 : kFj % 2 == 0 ? 2 : 1;
    static constexpr int kBK = kSingle && kT == 256 ? 32 : 64;  // summed per stage
    static constexpr int kRowBytes = kBK * 2;
    static constexpr int kStage = 2 * kTerms * kT * kRowBytes;
    static constexpr int kStages = kT == 64 ? 4 : kT == 256 || kSingle ? 2 : kT == 192 ? 3 : 4;
    static constexpr int kLoads = kStage / 1024 / kWaves;       // of a wave and stage
    static constexpr int kRow = kT * 2 + 16;            // of a tile turned round, bytes
    static constexpr int kStrip = kT / kAcross;         // columns of a wave's part
    static constexpr int kStripRow = kStrip * 4 + 16;
    static constexpr int kTurn = kT * (kRow > kStripRow ? kRow : kStripRow);
    static constexpr int kLds = kStage * kStages > kTurn ? kStage * kStages : kTurn;
};

// Rows of an operand that a fragment's 16 lanes read (and so the results a lane holds): of G
// fragments side by side, lane r of fragment f takes row (r / 4) 4 G + 4 f + r % 4, which gives a
// lane 4 G consecutive results.
template <int kG>
__device__ __forceinline__ int spread(int r, int f) {
    return f / kG * (16 * kG) + (r >> 2) * (4 * kG) + f % kG * 4 + (r & 3);
}
// The place of 16-byte piece q in a row of a [i][sum] stage is q ^ swap_row(row): the rows that
// spread() puts side by side then meet different banks.
template <int kG, int kBK>
__device__ __forceinline__ int swap_row(int row) {
    const int group = (row >> (kG == 4 ? 4 : kG == 2 ? 3 : 2)) & 3;
    return kBK == 64 ? ((row >> 1) & 1) | (group << 1) : group;
}
// The same for row k of a [sum][i] stage, in units of 32 bytes: the eight rows k % 4 + {0, 8} and
// their pairs that one read covers.
template <int kT>
__device__ __forceinline__ int swap_sum(int k) {
    return kT % 128 ? ((k >> 1) & 1) | (((k >> 3) & 1) << 1) : (k & 3) | (((k >> 3) & 1) << 2);
}

// The order of a matrix's tiles: bands of kBand rows of tiles, column by column.  The 32 tiles that
// an XCD's CUs work on at once then share 4 + 8 panels of the operands in its L2 (1 + 32 row by
// row).
constexpr int kBand = 4;
__host__ __device__ __forceinline__ void rectangle_tile(int32_t k, int32_t down, int32_t across,
                                                        int32_t& ti, int32_t& tj) {
    const int32_t band = k / (kBand * across), rest = k - band * (kBand * across);
    const int32_t high = down - band * kBand < kBand ? down - band * kBand : kBand;
    tj = rest / high;
    ti = band * kBand + rest - tj * high;
}
// The lower triangle (tj <= ti): a band's full columns, then its triangle.
__host__ __device__ __forceinline__ void triangle_tile(int32_t k, int32_t down, int32_t& ti,
                                                       int32_t& tj) {
    constexpr int kOwn = kBand * (kBand + 1) / 2;
    auto before = [](int32_t band) {
        return band * (band - 1) / 2 * kBand * kBand + band * kOwn;
    };
    int32_t band = static_cast<int32_t>(sqrtf(2.0f * k) / kBand);
    while (before(band + 1) <= k) ++band;
    while (before(band) > k) --band;
    int32_t rest = k - before(band);
    const int32_t first = band * kBand;
    const int32_t high = down - first < kBand ? down - first : kBand;
    if (rest < high * first) {
        tj = rest / high;
        ti = first + rest - tj * high;
        return;
    }
    rest -= high * first;
    int32_t y = 0;
    while ((y + 1) * (y + 2) / 2 <= rest) ++y;
    ti = first + y;
    tj = first + rest - y * (y + 1) / 2;
}

template <class Src, int kPhase, bool kSingle, int kT, int kLanes = Shape<kT, kSingle>::kWaves * 64>
__global__ __launch_bounds__(kLanes) void mi_adamw_ns_product_kernel(
    Src src, Quintic f, char* ws, int32_t turn, int32_t want, MuonOut o) {
    typedef Shape<kT, kSingle> W;
    constexpr bool kPair = kPhase == kPhaseS || kPhase == kPhaseP;
    constexpr bool kSum = kPhase == kPhaseS;
    constexpr int kTerms = W::kTerms, kFi = W::kFi, kFj = W::kFj;
    constexpr int kG = W::kG, kGj = W::kGj;
    __shared__ __attribute__((aligned(16))) char lds[W::kLds];
    const Item it = src.get(Src::order(blockIdx.x, gridDim.x));
    const Layout l = layout_of(it.mat.rows, it.mat.cols, kSingle);
    char* base = ws + it.mat.workspace;
    const int32_t down = (l.mp + kT - 1) / kT;
    int32_t ti, tj;
    const int32_t split = kPair ? split_of(l, kT, want) : 1;
    const int32_t part = kPair ? it.index % split : 0;
    if (kPhase == kPhaseP && part) return;      // P's sums are short
    if (kPair) triangle_tile(it.index / split, down, ti, tj);
    else rectangle_tile(it.index, down, (l.np + kT - 1) / kT, ti, tj);
    ti = __builtin_amdgcn_readfirstlane(ti);
    tj = __builtin_amdgcn_readfirstlane(tj);
    const char* t_now = base + l.t + turn * l.t_turn;
    const char* left = kSum ? t_now : base + (kPhase == kPhaseP ? l.s : l.p);
    const char* right = kPair ? left : t_now;
    const int64_t left_lo = kSum ? l.t_lo : l.sq_lo;
    const int64_t right_lo = kPair ? left_lo : l.t_lo;
    const int32_t left_rows = l.mp, right_rows = kPair ? l.mp : l.np;
    constexpr int kBK = W::kBK, kRowBytes = W::kRowBytes;
    const int32_t all_steps = (kSum ? l.np : l.mp) / kBK;
    const int32_t first_step = kSum ? int64_t(all_steps) * part / split : 0;
    const int32_t steps = kSum ? int64_t(all_steps) * (part + 1) / split - first_step : all_steps;
    const int64_t step_bytes = kSum ? int64_t(l.mp) * kRowBytes : kRowBytes;

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = wave / W::kAcross, wj = wave % W::kAcross;
    const int g = lane >> 4, r = lane & 15;
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((SHARED char*)lds));

    // A wave's loads of a stage: kLoads pieces of 1 KB, of [side][term][rows].
    constexpr int kPieces = W::kLoads / (2 * kTerms);   // of one side and term
    uint32_t from[2][kPieces];
#pragma unroll
    for (int side = 0; side < 2; ++side)
#pragma unroll
        for (int q = 0; q < kPieces; ++q) {
            const int piece = wave * kPieces + q;
            const int32_t first = (side ? tj : ti) * kT, rows = side ? right_rows : left_rows;
            if (kSum) {
                constexpr int kPer = kT / 8;            // 16-byte pieces of a row
                const int k = (piece * 64 + lane) / kPer, c = (piece * 64 + lane) % kPer;
                const int32_t col = first + (c ^ (swap_sum<kT>(k) << 1)) * 8;
                from[side][q] = (uint32_t(k) * l.mp + (col < rows ? col : rows - 8)) * 2;
            } else {
                constexpr int kPer = kRowBytes / 16;
                const int row = (piece * 64 + lane) / kPer;
                const int32_t at = first + row < rows ? first + row : rows - 1;
                const int c = (lane % kPer) ^
                              (side ? swap_row<kGj, kBK>(row) : swap_row<kG, kBK>(row));
                from[side][q] = (uint32_t(at - first) * l.mp + c * 8) * 2;
            }
        }
    const int64_t skip = first_step * step_bytes;
    const char* sides[2] = {uniform(left + (kSum ? skip : int64_t(ti) * kT * l.mp * 2)),
                            uniform(right + (kSum ? skip : int64_t(tj) * kT * l.mp * 2))};
    auto load_stage = [&](int32_t step) {
        const uint32_t to = lds0 + (step % W::kStages) * W::kStage;
#pragma unroll
        for (int side = 0; side < 2; ++side)
#pragma unroll
            for (int term = 0; term < kTerms; ++term)
#pragma unroll
                for (int q = 0; q < kPieces; ++q)
                    load_lds(to + (side * kTerms + term) * kT * kRowBytes +
                                 (wave * kPieces + q) * 1024,
                             uniform(sides[side] + step * step_bytes +
                                     (term ? (side ? right_lo : left_lo) : 0)),
                             from[side][q]);
    };

    // A lane's results: rows i .. i + 3 of column j for each fragment down and across.
    auto row_of = [&](int fi) {
        return ti * kT + wi * (kFi * 16) + (kSum ? fi * 16 + g * 4 : spread<kG>(g * 4, fi));
    };
    auto col_of = [&](int fj) {
        return tj * kT + wj * (kFj * 16) + (kSum ? fj * 16 + r : spread<kGj>(r, fj));
    };
    // X's values there, for X' = a X + ..: 4 kG in a row of T, the two terms.  Read while the last
    // stages are multiplied, where registers allow.
    constexpr bool kAhead = !kPair && !kSingle && kT <= 192;
    constexpr int kOld = kPair ? 1 : kG / 2;
    half8 old[kPair ? 1 : kFi / kG][kPair ? 1 : kFj][kOld][2];
    auto read_old = [&](int fb, int fj) {
        const int32_t i = row_of(fb * kG), j = col_of(fj);
        if (i >= l.mp || j >= l.np) return;
        const char* at = t_now + (int64_t(j) * l.mp + i) * 2;
#pragma unroll
        for (int q = 0; q < kOld; ++q) {
            old[fb][fj][q][0] = *(const GLOBAL half8*)(at + q * 16);
            old[fb][fj][q][1] = *(const GLOBAL half8*)(at + l.t_lo + q * 16);
        }
    };
    struct Fragments {
        half8 a[kTerms][kFi], b[kTerms][kFj];
    };
    // Fragment q of one side and term, 32 of the summed index from 32 kk on.
    auto read_one = [&](int32_t step, int kk, int side, int term, int q) {
        const char* tile = lds + (step % W::kStages) * W::kStage +
                           (side * kTerms + term) * kT * kRowBytes;
        const int first = side ? wj * (kFj * 16) : wi * (kFi * 16);
        if (kSum) {
            // lane r gives the address of four columns of row r / 4 and gets column r of four rows
            typedef __attribute__((__vector_size__(8))) short short4_;
            const int k = kk * 32 + g * 8 + (r >> 2), unit = (first + q * 16) / 16;
            const short4_ x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (SHARED short4_*)(tile + k * (kT * 2) + (unit ^ swap_sum<kT>(k)) * 32 +
                                  (r & 3) * 8));
            const short4_ y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (SHARED short4_*)(tile + (k + 4) * (kT * 2) + (unit ^ swap_sum<kT>(k + 4)) * 32 +
                                  (r & 3) * 8));
            return __builtin_shufflevector(__builtin_bit_cast(half4, x),
                                           __builtin_bit_cast(half4, y), 0, 1, 2, 3, 4, 5, 6, 7);
        }
        const int row = first + (side ? spread<kGj>(r, q) : spread<kG>(r, q));
        const int c = (kk * 4 + g) ^ (side ? swap_row<kGj, kBK>(row) : swap_row<kG, kBK>(row));
        return *(const half8*)(tile + row * kRowBytes + c * 16);
    };
    auto read = [&](int32_t step, int kk, Fragments& f) {
#pragma unroll
        for (int term = 0; term < kTerms; ++term) {
#pragma unroll
            for (int q = 0; q < kFi; ++q) f.a[term][q] = read_one(step, kk, 0, term, q);
#pragma unroll
            for (int q = 0; q < kFj; ++q) f.b[term][q] = read_one(step, kk, 1, term, q);
        }
    };
    // P's trace over m in half precision, from the shares that P's tiles on the diagonal left
    // (`want`: their side): asked for here, used after the product.
    const float* traces = reinterpret_cast<const float*>(base + l.parts);
    const int32_t n_traces = kPair || kSingle ? 0 : (l.mp + want - 1) / want;
    float trace = lane < n_traces ? *(const GLOBAL float*)(traces + lane) : 0.0f;
    f32x4 acc[kFi][kFj] = {};
    auto multiply = [&](const Fragments& f) {
#pragma unroll
        for (int i = 0; i < kFi; ++i)
#pragma unroll
            for (int j = 0; j < kFj; ++j) {
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.a[0][i], f.b[0][j], acc[i][j],
                                                                   0, 0, 0);
                if (kSingle) {
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        f.a[kTerms - 1][i], f.b[0][j], acc[i][j], 0, 0, 0);
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        f.a[0][i], f.b[kTerms - 1][j], acc[i][j], 0, 0, 0);
                }
            }
    };
    // Stage `step` has landed (the newest kStages - 2 may still be on their way) and every wave is
    // done reading the one before it, whose place the next one to load takes.
    auto arrive = [&](int32_t step) {
        if (step + W::kStages - 2 < steps) wait_stages<(W::kStages - 2) * W::kLoads>();
        else wait_stages<0>();
        if (step > 0 && step + W::kStages - 1 < steps) load_stage(step + W::kStages - 1);
    };
#pragma unroll
    for (int k = 0; k < W::kStages; ++k)
        if (k < steps) load_stage(k);
    if (W::kStages < steps) wait_stages<(W::kStages - 1) * W::kLoads>();
    else wait_stages<0>();
    if constexpr (kBK == 32) {
        // no registers to spare: term by term, the SIMD's other wave fills the gaps
        for (int32_t step = 0; step < steps; ++step) {
            if (step > 0) arrive(step);
            half8 a[kFi], b[kFj], x[kFi > kFj ? kFi : kFj];
            auto product = [&](const half8* u, const half8* v) {
#pragma unroll
                for (int i = 0; i < kFi; ++i)
#pragma unroll
                    for (int j = 0; j < kFj; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(u[i], v[j], acc[i][j], 0,
                                                                           0, 0);
            };
#pragma unroll
            for (int q = 0; q < kFi; ++q) a[q] = read_one(step, 0, 0, 0, q);
#pragma unroll
            for (int q = 0; q < kFj; ++q) b[q] = read_one(step, 0, 1, 0, q);
            product(a, b);
#pragma unroll
            for (int q = 0; q < kFj; ++q) x[q] = read_one(step, 0, 1, 1, q);
            product(a, x);
#pragma unroll
            for (int q = 0; q < kFi; ++q) x[q] = read_one(step, 0, 0, 1, q);
            product(x, b);
        }
    } else {
        // each half of a stage is read while the other one is multiplied
        Fragments even, odd;
        read(0, 0, even);
        auto both_halves = [&](int32_t step) {
            read(step, 1, odd);
            multiply(even);
            if (step + 1 < steps) {
                arrive(step + 1);
                read(step + 1, 0, even);
            }
            multiply(odd);
        };
        int32_t step = 0;
        for (; step < (kAhead ? steps - 3 : steps); ++step) both_halves(step);
        if constexpr (kAhead) {
#pragma unroll
            for (int fb = 0; fb < kFi / kG; ++fb)
#pragma unroll
                for (int fj = 0; fj < kFj; ++fj) read_old(fb, fj);
            for (; step < steps; ++step) both_halves(step);
        }
    }

    if (kSum && split > 1) {
        // The shares of this tile's sum; the workgroup that brings the last one adds them up, in
        // their order.  None waits for another.  Shares pass between XCDs, whose L2s are apart:
        // they are stored and loaded at agent scope, which goes past the L2, and a workgroup counts
        // its share only when its stores are complete.  (A release fence in that place writes back
        // all that the XCD's L2 holds: 27 us more for 2045 x 511.)
        float* shares = reinterpret_cast<float*>(base + l.t + (turn ^ 1) * l.t_turn) +
                        int64_t(it.index / split) * split * kT * kT;
        float* mine = shares + int64_t(part) * kT * kT;
        auto at = [&](int i, int j, int e) {
            return ((i * kFj + j) * 4 + e) * kLanes + int(threadIdx.x);
        };
#pragma unroll
        for (int i = 0; i < kFi; ++i)
#pragma unroll
            for (int j = 0; j < kFj; ++j)
                for (int e = 0; e < 4; ++e)
                    __hip_atomic_store(mine + at(i, j, e), acc[i][j][e], __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
        wait_stages<0>();           // every wave's stores are complete
        int* last = reinterpret_cast<int*>(lds);
        if (threadIdx.x == 0) {
            uint32_t* count = reinterpret_cast<uint32_t*>(base + l.counts) + it.index / split;
            const uint32_t before = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED,
                                                           __HIP_MEMORY_SCOPE_AGENT);
            *last = before + 1 == static_cast<uint32_t>(split);
            if (*last) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!*last) return;
#pragma unroll
        for (int i = 0; i < kFi; ++i)
#pragma unroll
            for (int j = 0; j < kFj; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int32_t p = 0; p < split; ++p)
#pragma unroll
            for (int i = 0; i < kFi; ++i)
#pragma unroll
                for (int j = 0; j < kFj; ++j)
                    for (int e = 0; e < 4; ++e)
                        acc[i][j][e] += __hip_atomic_load(
                            shares + int64_t(p) * kT * kT + at(i, j, e), __ATOMIC_RELAXED,
                            __HIP_MEMORY_SCOPE_AGENT);
    }
    const float* ds = reinterpret_cast<const float*>(base + l.ds);
    const float* dp = reinterpret_cast<const float*>(base + l.dp);
    if (kPair) {
        char* to = base + (kPhase == kPhaseS ? l.s : l.p);
        float* diag = reinterpret_cast<float*>(base + (kPhase == kPhaseS ? l.ds : l.dp));
#pragma unroll
        for (int fi = 0; fi < kFi; ++fi)
#pragma unroll
            for (int fj = 0; fj < kFj; ++fj) {
                const int32_t i = row_of(fi), j = col_of(fj);
                if (i >= l.mp || j >= l.mp) continue;
                f32x4 v = acc[fi][fj];
                const int64_t mirrored = (int64_t(j) * l.mp + i) * 2;
                if (kPhase == kPhaseS) {
                    for (int e = 0; e < 4; ++e) v[e] *= 1.0f / (kScaleX * kScaleX);
                } else {
                    // S = S' + D with S' = off the diagonal: S^2 = S'^2 + S' D + D S' + D^2
                    f32x4 s;
                    const char* sp = base + l.s + mirrored;
                    if (kSingle) {
                        s = join2(sp, l.sq_lo);
                    } else {
                        const half4 hs = *(const GLOBAL half4*)(sp);
                        for (int e = 0; e < 4; ++e) s[e] = static_cast<float>(hs[e]);
                    }
                    const float dj = ds[j];
                    const f32x4 di = *(const GLOBAL f32x4*)(ds + i);
                    for (int e = 0; e < 4; ++e) {
                        const float sv = s[e] * (1.0f / kScaleS);
                        float sq = __builtin_fmaf(sv, di[e] + dj,
                                                  v[e] * (1.0f / (kScaleS * kScaleS)));
                        if (i + e == j) sq = __builtin_fmaf(di[e], di[e], sq);
                        v[e] = __builtin_fmaf(f.c, sq, f.b * (i + e == j ? di[e] : sv));
                    }
                }
                for (int e = 0; e < 4; ++e)
                    if (i + e == j) {
                        diag[j] = v[e];
                        trace += v[e];
                        v[e] = 0.0f;
                    }
                for (int e = 0; e < 4; ++e) v[e] *= kPhase == kPhaseS ? kScaleS : kScaleP;
                acc[fi][fj] = v;
                half4 hi, lo;
                split2(v, hi, lo);
                *(GLOBAL half4*)(to + mirrored) = hi;
                if (kSingle) *(GLOBAL half4*)(to + l.sq_lo + mirrored) = lo;
            }
        if (ti == tj) {
            if (kPhase == kPhaseP && !kSingle) {
                // the tile's share of P's trace
                for (int d = 32; d > 0; d >>= 1) trace += __shfl_xor(trace, d);
                float* sums = reinterpret_cast<float*>(lds);
                __syncthreads();
                if (lane == 0) sums[wave] = trace;
                __syncthreads();
                if (threadIdx.x == 0) {
                    for (int w = 1; w < W::kWaves; ++w) trace += sums[w];
                    reinterpret_cast<float*>(base + l.parts)[ti] = trace;
                }
            }
            return;
        }
        // the other triangle: the tile turned round in LDS
#pragma unroll
        for (int term = 0; term < kTerms; ++term) {
            __syncthreads();
#pragma unroll
            for (int fi = 0; fi < kFi; ++fi)
#pragma unroll
                for (int fj = 0; fj < kFj; ++fj) {
                    half4 hi, lo;
                    split2(acc[fi][fj], hi, lo);
                    char* at = lds + (row_of(fi) - ti * kT) * W::kRow + (col_of(fj) - tj * kT) * 2;
                    for (int e = 0; e < 4; ++e)
                        *(_Float16*)(at + e * W::kRow) = term ? lo[e] : hi[e];
                }
            __syncthreads();
            for (int q = threadIdx.x; q < kT * (kT / 8); q += W::kWaves * 64) {
                const int y = q / (kT / 8), x = q % (kT / 8) * 8;
                const int32_t i = ti * kT + y, j = tj * kT + x;
                if (i < l.mp && j < l.mp)
                    *(GLOBAL half8*)(to + term * l.sq_lo + (int64_t(i) * l.mp + j) * 2) =
                        *(const half8*)(lds + y * W::kRow + x * 2);
            }
        }
        return;
    }
    // X' = (a + D) X + P' X, P' = off the diagonal.  In half precision P' reads X's first term, so D
    // takes the second one at its mean alone: what D_i - D_k of the rounding would add beyond P's own
    // product points out of the rows that X has, where the steps to come amplify it (of rank one in 2
    // of 256 rows the result was 4e-2 off with D_i there, and is 2e-3; with no D at all a full rank's
    // 7e-4 would be 1.3e-3).
    // Four of a wave's lanes write a line of 32 kG bytes; as the sides are padded to multiples of 64,
    // a lane's values are all there or none.
    float second = 0.0f;
    if (!kSingle) {
        for (int32_t k = lane + 64; k < n_traces; k += 64) trace += traces[k];
        for (int d = 32; d > 0; d >>= 1) trace += __shfl_xor(trace, d);
        second = f.a + trace / l.m;
    }
#pragma unroll
    for (int fb = 0; fb < kFi / kG; ++fb) {
        const int32_t i = row_of(fb * kG);
        if (i >= l.mp) continue;
        f32x4 d[kG];
#pragma unroll
        for (int q = 0; q < kG; ++q) {
            d[q] = *(const GLOBAL f32x4*)(dp + i + q * 4);
            for (int e = 0; e < 4; ++e) d[q][e] += f.a;
        }
#pragma unroll
        for (int fj = 0; fj < kFj; ++fj) {
            const int32_t j = col_of(fj);
            if (j >= l.np) continue;
            if (!kAhead) read_old(fb, fj);
#pragma unroll
            for (int q = 0; q < kOld; ++q) {
                half8 hi, lo;
                for (int e = 0; e < 8; ++e) {
                    const int fi = fb * kG + q * 2 + e / 4;
                    const float x0 = static_cast<float>(old[fb][fj][q][0][e]);
                    const float x1 = static_cast<float>(old[fb][fj][q][1][e]);
                    const float di = d[q * 2 + e / 4][e % 4];
                    const float px = acc[fi][fj][e % 4] * (1.0f / kScaleP);
                    const float v =
                        kSingle ? __builtin_fmaf(di, x0 + x1, px)
                                : __builtin_fmaf(di, x0, __builtin_fmaf(second, x1, px));
                    hi[e] = static_cast<_Float16>(v);
                    lo[e] = static_cast<_Float16>(v - static_cast<float>(hi[e]));
                    if (kPhase == kPhaseLast) acc[fi][fj][e % 4] = v * (1.0f / kScaleX);
                }
                if (kPhase == kPhaseX) {
                    char* at = base + l.t + (turn ^ 1) * l.t_turn +
                               (int64_t(j) * l.mp + i) * 2 + q * 16;
                    *(GLOBAL half8*)(at) = hi;
                    *(GLOBAL half8*)(at + l.t_lo) = lo;
                }
            }
        }
    }
    if (kPhase != kPhaseLast) return;
    if (it.mat.rows > it.mat.cols) {        // a tall matrix: a lane's results lie along its rows
#pragma unroll
        for (int fj = 0; fj < kFj; ++fj)
#pragma unroll
            for (int fi = 0; fi < kFi; ++fi) {
                const int32_t i = row_of(fi), j = col_of(fj);
                if (i < l.m && j < l.n) write_out(src, it, j, i, acc[fi][fj], l.m - i, o);
            }
        return;
    }
    // a wide one: turned round in LDS, the waves' columns in turn
    for (int turn_of = 0; turn_of < W::kAcross; ++turn_of) {
        __syncthreads();
        if (wj == turn_of)
#pragma unroll
            for (int fi = 0; fi < kFi; ++fi)
#pragma unroll
                for (int fj = 0; fj < kFj; ++fj) {
                    char* at = lds + (row_of(fi) - ti * kT) * W::kStripRow +
                               (col_of(fj) - tj * kT - wj * W::kStrip) * 4;
                    for (int e = 0; e < 4; ++e) *(float*)(at + e * W::kStripRow) = acc[fi][fj][e];
                }
        __syncthreads();
        for (int q = threadIdx.x; q < kT * (W::kStrip / 4); q += W::kWaves * 64) {
            const int y = q / (W::kStrip / 4), x = q % (W::kStrip / 4) * 4;
            const int32_t i = ti * kT + y, j = tj * kT + turn_of * W::kStrip + x;
            if (i < l.m && j < l.n)
                write_out(src, it, i, j, *(const f32x4*)(lds + y * W::kStripRow + x * 4), l.n - j,
                          o);
        }
    }
}

// ---------------------------------------------------------------------------
// Small matrices: everything in one workgroup's LDS and registers, one launch.

// Sides of at most kM and kN; MI_ADAMW_NS_WHOLE items, one matrix each, in single precision.
// X^T lies in LDS as [j][i] in two terms, S and then P in one square of two terms.  In the
// products' last phase a wave reads and writes rows of X^T of its own alone, so a step has four
// barriers (six at 64).  Bound by latency: LDS reads, matrix instructions and barriers in a chain,
// 5 us a step at 64 x 256.  A call of it and of the 17 launches above, fp32: 64 x 256 37 and 77 us,
// 64 x 512 65 and 85, 128 x 128 71 and 82; 512 matrices of 64 x 256 84 and 266.
constexpr int kSmallThreads = 512;

template <int kM, int kN>
struct SmallShape {
    static constexpr int kT = kM * kN * 2, kSq = kM * kM * 2;      // bytes of one term
    static constexpr int kWaves = kSmallThreads / 64;
    static constexpr int kSide = kM / 16;
    static constexpr int kSquares = kSide * kSide / kWaves;        // fragments of S a wave
    static constexpr int kBlocks = kN / 16 / kWaves;               // blocks of X^T's rows a wave
    static constexpr int kVectors = kM * kN / 4 / kSmallThreads;   // of four elements a lane
};

template <class Src, int kM, int kN>
__global__ __launch_bounds__(kSmallThreads) void mi_adamw_ns_whole_kernel(Src src, Quintic f,
                                                                          int32_t steps, float eps,
                                                                          Momentum h, MuonOut o) {
    typedef SmallShape<kM, kN> W;
    __shared__ __attribute__((aligned(16))) char t_lds[2 * W::kT];
    __shared__ __attribute__((aligned(16))) char sq_lds[2 * W::kSq];
    __shared__ float ds[kM], dp[kM];
    __shared__ double sums[W::kWaves];
    const Item it = src.get(blockIdx.x);
    const int32_t rows = it.mat.rows, cols = it.mat.cols;
    const bool wide = rows <= cols;
    const int32_t m = wide ? rows : cols, n = wide ? cols : rows;
    const int32_t np = (n + kPad - 1) / kPad * kPad;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int g = lane >> 4, r = lane & 15;
    // 16-byte piece q of row y lies at place q ^ (y & 7)
    auto place = [](int y, int x) { return y * (kM * 2) + (((x >> 3) ^ (y & 7)) << 4) + (x & 7) * 2; };

    // the matrix, padded to kM by np, four elements of a row a lane and turn
    const int32_t across = (wide ? np : kM) / 4;
    f32x4 u[W::kVectors];
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < W::kVectors; ++k) {
        const int32_t v = k * kSmallThreads + threadIdx.x, y = v / across, x = v % across * 4;
        u[k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (y < rows && x < cols) u[k] = update_of<true>(src, it, y, x, cols - x, h);
        for (int e = 0; e < 4; ++e) sum += double(u[k][e]) * u[k][e];
    }
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int k = 0; k < W::kWaves; ++k) sum += sums[k];
    const double norm = sqrt(sum);
    const double inv = double(kScaleX) / (norm < eps ? eps : norm);
#pragma unroll
    for (int k = 0; k < W::kVectors; ++k) {
        const int32_t v = k * kSmallThreads + threadIdx.x, y = v / across, x = v % across * 4;
        if (y >= (wide ? kM : np)) continue;
        for (int e = 0; e < 4; ++e) u[k][e] = static_cast<float>(u[k][e] * inv);
        half4 hi, lo;
        split2(u[k], hi, lo);
        if (!wide) {
            *(half4*)(t_lds + place(y, x)) = hi;
            *(half4*)(t_lds + W::kT + place(y, x)) = lo;
        } else {
            for (int e = 0; e < 4; ++e) {
                *(_Float16*)(t_lds + place(x + e, y)) = hi[e];
                *(_Float16*)(t_lds + W::kT + place(x + e, y)) = lo[e];
            }
        }
    }
    typedef __attribute__((__vector_size__(8))) short short4_;
    // Eight rows k0 + 8 g .. of X^T's column x0 + r, turned round.
    auto down = [&](int term, int k0, int x0) {
        const int y = k0 + g * 8 + (r >> 2), x = x0 + (r & 3) * 4;
        const char* base = t_lds + term * W::kT;
        const half4 a = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                      (SHARED short4_*)(base + place(y, x))));
        const half4 b = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                      (SHARED short4_*)(base + place(y + 4, x))));
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    auto along = [&](const char* base, int y, int x) { return *(const half8*)(base + place(y, x)); };
    auto mul3 = [](half8 ah, half8 al, half8 bh, half8 bl, f32x4 c) {
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bh, c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(al, bh, c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bl, c, 0, 0, 0);
    };
    // The wave's fragments of the square: of 4 x 4 the column 2 bj + h of the 2 x 2 block (bi, bj),
    // of 8 x 8 a block of 4 x 2.
    const int h_of = wave >> 2, bi = wave & 1, bj = kM == 64 ? (wave >> 1) & 1 : wave >> 1;
    auto row_of = [&](int q) { return (kM == 64 ? bi * 2 + q : bi * 4 + q % 4) * 16; };
    auto col_of = [&](int q) { return (kM == 64 ? bj * 2 + h_of : bj * 2 + q / 4) * 16; };
    auto put_square = [&](int q, f32x4 v, float* diag, float scale) {
        const int i = row_of(q) + g * 4, j = col_of(q) + r;
        for (int e = 0; e < 4; ++e) {
            if (i + e == j) {
                diag[j] = v[e];
                v[e] = 0.0f;
            }
            v[e] *= scale;
        }
        half4 hi, lo;
        split2(v, hi, lo);
        *(half4*)(sq_lds + place(j, i)) = hi;       // symmetric
        *(half4*)(sq_lds + W::kSq + place(j, i)) = lo;
    };
    for (int32_t step = 0; step < steps; ++step) {
        __syncthreads();                            // X^T is there, P is read
        f32x4 s[W::kSquares] = {};
        if constexpr (kM == 64) {
            // two waves share a 2 x 2 block, each sums over every other 32 rows (half the LDS reads
            // of a wave for itself), and each ends with one of its columns
            f32x4 part[2][2] = {};
#pragma unroll 2
            for (int32_t k = h_of * 32; k < np; k += 64) {
                half8 a[2][2], b[2][2];
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int term = 0; term < 2; ++term) {
                        a[q][term] = down(term, k, (bi * 2 + q) * 16);
                        b[q][term] = down(term, k, (bj * 2 + q) * 16);
                    }
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                        part[y][x] = mul3(a[x][0], a[x][1], b[y][0], b[y][1], part[y][x]);
            }
            f32x4* swap = (f32x4*)sq_lds;           // P is read
#pragma unroll
            for (int q = 0; q < 2; ++q)
                swap[(wave * 2 + q) * 64 + lane] = h_of ? part[0][q] : part[1][q];
            __syncthreads();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const f32x4 other = swap[((wave ^ 4) * 2 + q) * 64 + lane];
                const f32x4 own = h_of ? part[1][q] : part[0][q];
                for (int e = 0; e < 4; ++e) s[q][e] = own[e] + other[e];
            }
            __syncthreads();
        } else {
            for (int32_t k = 0; k < np; k += 32) {
                half8 a[4][2], b[2][2];
#pragma unroll
                for (int term = 0; term < 2; ++term) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) a[q][term] = down(term, k, row_of(q));
#pragma unroll
                    for (int q = 0; q < 2; ++q) b[q][term] = down(term, k, col_of(q * 4));
                }
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    s[q] = mul3(a[q % 4][0], a[q % 4][1], b[q / 4][0], b[q / 4][1], s[q]);
            }
        }
#pragma unroll
        for (int q = 0; q < W::kSquares; ++q) {
            for (int e = 0; e < 4; ++e) s[q][e] *= 1.0f / (kScaleX * kScaleX);
            put_square(q, s[q], ds, kScaleS);
        }
        __syncthreads();                            // S is there
        f32x4 p[W::kSquares] = {};
        // (128: a turn's operands fill the registers)
#pragma unroll(kM == 64 ? 2 : 1)
        for (int k = 0; k < kM; k += 32)
#pragma unroll
            for (int q = 0; q < W::kSquares; ++q) {
                const int i = row_of(q) + r, j = col_of(q) + r, x = k + g * 8;
                p[q] = mul3(along(sq_lds, i, x), along(sq_lds + W::kSq, i, x), along(sq_lds, j, x),
                            along(sq_lds + W::kSq, j, x), p[q]);
            }
#pragma unroll
        for (int q = 0; q < W::kSquares; ++q) {
            const int i = row_of(q) + g * 4, j = col_of(q) + r;
            const float dj = ds[j];
            for (int e = 0; e < 4; ++e) {
                // S = S' + D: S^2 = S'^2 + S' D + D S' + D^2
                const float di = ds[i + e], sv = i + e == j ? 0.0f : s[q][e];
                float sq = __builtin_fmaf(sv, di + dj, p[q][e] * (1.0f / (kScaleS * kScaleS)));
                if (i + e == j) sq = __builtin_fmaf(di, di, sq);
                p[q][e] = __builtin_fmaf(f.c, sq, f.b * (i + e == j ? di : sv));
            }
        }
        __syncthreads();                            // S is read
#pragma unroll
        for (int q = 0; q < W::kSquares; ++q) put_square(q, p[q], dp, kScaleP);
        __syncthreads();                            // P is there
        // P's fragments: 64 wide, read once for all of a wave's blocks
        constexpr bool kKeep = kM == 64;
        half8 keep[kKeep ? 2 : 1][kKeep ? 4 : 1][2];
        if constexpr (kKeep) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int term = 0; term < 2; ++term)
                        keep[k][q][term] = along(sq_lds + term * W::kSq, q * 16 + r, k * 32 + g * 8);
        }
#pragma unroll(kKeep && W::kBlocks < 4 ? W::kBlocks : 1)
        for (int b = 0; b < W::kBlocks; ++b) {
            const int j = (wave + b * W::kWaves) * 16 + r;
            if ((wave + b * W::kWaves) * 16 >= np) break;
            f32x4 x[W::kSide] = {};
#pragma unroll(kKeep ? 2 : 1)
            for (int k = 0; k < kM; k += 32) {
                const half8 bh = along(t_lds, j, k + g * 8), bl = along(t_lds + W::kT, j, k + g * 8);
#pragma unroll
                for (int q = 0; q < W::kSide; ++q) {
                    if constexpr (kKeep)
                        x[q] = mul3(keep[k / 32][q][0], keep[k / 32][q][1], bh, bl, x[q]);
                    else
                        x[q] = mul3(along(sq_lds, q * 16 + r, k + g * 8),
                                    along(sq_lds + W::kSq, q * 16 + r, k + g * 8), bh, bl, x[q]);
                }
            }
#pragma unroll
            for (int q = 0; q < W::kSide; ++q) {
                const int i = q * 16 + g * 4;
                half4* hi = (half4*)(t_lds + place(j, i));
                half4* lo = (half4*)(t_lds + W::kT + place(j, i));
                const half4 ah = *hi, al = *lo;
                f32x4 v;
                for (int e = 0; e < 4; ++e)
                    v[e] = __builtin_fmaf(f.a + dp[i + e],
                                          static_cast<float>(ah[e]) + static_cast<float>(al[e]),
                                          x[q][e] * (1.0f / kScaleP));
                if (step + 1 < steps) {
                    half4 bh, bl;
                    split2(v, bh, bl);
                    *hi = bh;
                    *lo = bl;
                } else if (j < n) {
                    for (int e = 0; e < 4; ++e) v[e] *= 1.0f / kScaleX;
                    if (!wide) {
                        if (i < m) write_out(src, it, j, i, v, m - i, o);
                    } else {
                        for (int e = 0; e < 4; ++e)
                            if (i + e < m)
                                write_out(src, it, i + e, j, f32x4{v[e], 0.0f, 0.0f, 0.0f}, 1, o);
                    }
                }
            }
        }
    }
}

// The kernels above by number, 0 for matrices that their LDS does not hold; faster wherever it does
// (the figures stand at the kernel).
int32_t whole_of(int32_t rows, int32_t cols) {
    const int32_t m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
    if (m <= 64) return n <= 256 ? 1 : n <= 512 ? 2 : 0;
    return n <= 128 ? 3 : 0;
}

template <class Src>
void launch_whole(const Src& src, unsigned grid, int32_t which, const mi_adamw_ns_options& o,
                  const Momentum& h, const MuonOut& out, hipStream_t s) {
    const Quintic f{o.a, o.b, o.c};
    if (which == 1)
        hipLaunchKernelGGL((mi_adamw_ns_whole_kernel<Src, 64, 256>), dim3(grid), dim3(kSmallThreads),
                           0, s, src, f, o.steps, o.eps, h, out);
    else if (which == 2)
        hipLaunchKernelGGL((mi_adamw_ns_whole_kernel<Src, 64, 512>), dim3(grid), dim3(kSmallThreads),
                           0, s, src, f, o.steps, o.eps, h, out);
    else
        hipLaunchKernelGGL((mi_adamw_ns_whole_kernel<Src, 128, 128>), dim3(grid),
                           dim3(kSmallThreads), 0, s, src, f, o.steps, o.eps, h, out);
}

// ---------------------------------------------------------------------------
// Host side

int status() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MI_ADAMW_OK : static_cast<int>(e);
}

// Whether singular values in [0, 1] stay where the scales above hold them, through every step:
// s (a + b s^2 + c s^4) below 1.9 (X), and b s^2 + c s^4 within 7.5 (P).  Both are largest at an
// end of the range or where the derivative by q = s^2 is 0.
bool bounded(const mi_adamw_ns_options& o) {
    const double a = o.a, b = o.b, c = o.c;
    double top = 1.0 + 1e-3;
    for (int32_t k = 0; k < o.steps; ++k) {
        const double end = top * top, root = std::sqrt(9.0 * b * b - 20.0 * a * c);
        // the end; b + 2 c q = 0; a + 3 b q + 5 c q^2 = 0, or a + 3 b q = 0 where c is 0
        const double at[5] = {end, -b / (2.0 * c), (-3.0 * b + root) / (10.0 * c),
                              (-3.0 * b - root) / (10.0 * c), -a / (3.0 * b)};
        double next = 0.0;
        for (const double q : at) {
            if (!(q >= 0.0 && q <= end)) continue;      // NaN and infinities too
            const double p = b * q + c * q * q, v = std::fabs(std::sqrt(q) * (a + p));
            if (!(std::fabs(p) < 7.5) || !(v < 1.9)) return false;
            if (v > next) next = v;
        }
        if (std::fabs(next + 1e-3 - top) < 1e-9) return true;
        top = next + 1e-3;
    }
    return true;
}

bool options_ok(const mi_adamw_ns_options* o) {
    return o && o->steps >= 1 && o->steps < 100 && o->eps >= 0.0f && std::isfinite(o->eps) &&
           (o->precision == MI_ADAMW_NS_HALF || o->precision == MI_ADAMW_NS_SINGLE) &&
           std::isfinite(o->a) && std::isfinite(o->b) && std::isfinite(o->c) && bounded(*o);
}

constexpr int32_t kMaxSide = 1 << 20;
bool sides_ok(int32_t rows, int32_t cols) {
    return rows > 0 && cols > 0 && rows <= kMaxSide && cols <= kMaxSide &&
           int64_t(rows) * cols < (int64_t(1) << 36) && (rows < cols ? rows : cols) <= 32768;
}

int64_t items_of_matrix(int32_t rows, int32_t cols, int32_t kind, int32_t tile, int32_t split) {
    const Layout l = layout_of(rows, cols, false);
    const int64_t down = (l.mp + tile - 1) / tile, across = (l.np + tile - 1) / tile;
    switch (kind) {
        case MI_ADAMW_NS_PARTS: return parts_of(rows, cols);
        case MI_ADAMW_NS_BLOCKS: return blocks_of(rows, cols);
        case MI_ADAMW_NS_PAIRS: return down * (down + 1) / 2 * split_of(l, tile, split);
        case MI_ADAMW_NS_TILES: return down * across;
        case MI_ADAMW_NS_WHOLE: return 1;
        default: return MI_ADAMW_E_INVALID;
    }
}

constexpr int64_t kCUs = 256;
constexpr int32_t kMostShares = 8;

bool tile_ok(int32_t tile, bool single) {
    return tile == 64 || tile == 128 || tile == 256 || (!single && tile == 192);
}

// What a launch's products are cut into.
struct Cut {
    int32_t pair_tile, split, tile;
};

template <class Src, int kPhase, bool kSingle, int kT>
void launch_tiles(const Src& src, unsigned grid, Quintic f, char* ws, int32_t turn, int32_t want,
                  const MuonOut& o, hipStream_t s) {
    hipLaunchKernelGGL((mi_adamw_ns_product_kernel<Src, kPhase, kSingle, kT>), dim3(grid),
                       dim3(Shape<kT, kSingle>::kWaves * 64), 0, s, src, f, ws, turn, want, o);
}

template <class Src, int kPhase, bool kSingle>
void launch_product(const Src& src, unsigned grid, const Cut& cut, Quintic f, char* ws,
                    int32_t turn, const MuonOut& o, hipStream_t s) {
    constexpr bool kPair = kPhase == kPhaseS || kPhase == kPhaseP;
    const int32_t tile = kPair ? cut.pair_tile : cut.tile;
    const int32_t want = kPair ? cut.split : cut.pair_tile;
    if (tile == 256)
        return launch_tiles<Src, kPhase, kSingle, 256>(src, grid, f, ws, turn, want, o, s);
    if constexpr (!kSingle) {
        if (tile == 192)
            return launch_tiles<Src, kPhase, kSingle, 192>(src, grid, f, ws, turn, want, o, s);
    }
    if (tile == 128) launch_tiles<Src, kPhase, kSingle, 128>(src, grid, f, ws, turn, want, o, s);
    else launch_tiles<Src, kPhase, kSingle, 64>(src, grid, f, ws, turn, want, o, s);
}

// source_of(kind): the launch's source, and its grid.
template <bool kSingle, class SourceOf>
int run_steps(const SourceOf& source_of, const mi_adamw_ns_options& o, const Cut& cut,
              const Momentum& h, const MuonOut& out, char* ws, hipStream_t s) {
    const Quintic f{o.a, o.b, o.c};
    unsigned grid = 0;
    auto src = source_of(MI_ADAMW_NS_PARTS, &grid);
    typedef decltype(src) Src;
    hipLaunchKernelGGL(mi_adamw_ns_sumsq_kernel<Src>, dim3(grid), dim3(kThreads), 0, s, src, h, ws,
                       int32_t(kSingle));
    src = source_of(MI_ADAMW_NS_BLOCKS, &grid);
    hipLaunchKernelGGL(mi_adamw_ns_load_kernel<Src>, dim3(grid), dim3(kThreads), 0, s, src, h, o.eps,
                       ws, int32_t(kSingle));
    for (int32_t k = 0; k < o.steps; ++k) {
        src = source_of(MI_ADAMW_NS_PAIRS, &grid);
        launch_product<Src, kPhaseS, kSingle>(src, grid, cut, f, ws, k & 1, out, s);
        launch_product<Src, kPhaseP, kSingle>(src, grid, cut, f, ws, 0, out, s);
        src = source_of(MI_ADAMW_NS_TILES, &grid);
        if (k + 1 < o.steps)
            launch_product<Src, kPhaseX, kSingle>(src, grid, cut, f, ws, k & 1, out, s);
        else
            launch_product<Src, kPhaseLast, kSingle>(src, grid, cut, f, ws, k & 1, out, s);
    }
    return status();
}

// Microseconds that a workgroup takes for 64 of a tile's summed index while all CUs work, by the
// tile's side; the smaller tiles load more bytes for a product.  Measured in the products of
// 768 x 768 (64), 12 x 768 x 3072 (128), 4096 x 16384 (192, 256) and their fp32 counterparts.
double stage_us(int32_t tile, bool single) {
    const double half = tile == 64 ? 0.3 : tile == 128 ? 0.7 : tile == 192 ? 1.26 : 2.05;
    return !single ? half : tile == 64 ? 0.6 : tile == 128 ? 1.7 : 5.1;
}

// The cut whose rounds over the chip's CUs take the least time: the tiles of X, and those of S and
// P with the shares of S's sums.  3 us a workgroup for its first stages and its results; shares
// are written and read again past the L2, at 1.5 TB/s.  The whole call with and without shares:
// 2045 x 511 fp32 161 and 191 us, 130 x 8000 fp32 181 and 401, 200 x 5000 bf16 145 and 200.
Cut cut_for(const mi_adamw_matrix* mats, int64_t n, int64_t times, bool single) {
    Cut best{64, 1, 64};
    double least_pairs = 0.0, least = 0.0;
    for (const int32_t tile : {64, 128, 192, 256}) {
        if (!tile_ok(tile, single)) continue;
        const double us = stage_us(tile, single);
        int64_t tiles = 0;
        double stages = 0.0;
        for (int64_t t = 0; t < n; ++t) {
            const Layout l = layout_of(mats[t].rows, mats[t].cols, single);
            const int64_t k = times * items_of_matrix(l.m, l.n, MI_ADAMW_NS_TILES, tile, 1);
            tiles += k;
            stages += double(k) * (l.mp / 64);
        }
        auto rounds = [](int64_t k) { return double((k + kCUs - 1) / kCUs); };
        const double time = rounds(tiles) * (stages / tiles * us + 3.0);
        if (tile == 64 || time < least) {
            least = time;
            best.tile = tile;
        }
        for (int32_t split = 1; split <= kMostShares; ++split) {
            int64_t squares = 0, items = 0;
            double s_stages = 0.0, p_stages = 0.0;
            for (int64_t t = 0; t < n; ++t) {
                const Layout l = layout_of(mats[t].rows, mats[t].cols, single);
                const int64_t k = times * items_of_matrix(l.m, l.n, MI_ADAMW_NS_PAIRS, tile, 1);
                squares += k;
                items += k * split_of(l, tile, split);
                s_stages += double(k) * (l.np / 64);
                p_stages += double(k) * (l.mp / 64);
            }
            if (split > 1 && items == squares) break;       // nothing to share
            const double share_us =
                items == squares ? 0.0 : 3.0 + double(items) * tile * tile * 8 / 1.5e6;
            const double pairs = rounds(items) * (s_stages / items * us + 3.0) + share_us +
                                 rounds(squares) * (p_stages / squares * us + 3.0);
            // shares only where they gain a tenth: the estimate is no better than that
            if ((tile == 64 && split == 1) || pairs < least_pairs * (split > 1 ? 0.9 : 1.0)) {
                least_pairs = pairs;
                best.pair_tile = tile;
                best.split = split;
            }
        }
    }
    return best;
}

}  // namespace

extern "C" {

int64_t mi_adamw_ns_workspace(int32_t rows, int32_t cols, int32_t precision) {
    if (!sides_ok(rows, cols) ||
        (precision != MI_ADAMW_NS_HALF && precision != MI_ADAMW_NS_SINGLE))
        return MI_ADAMW_E_INVALID;
    if (whole_of(rows, cols)) return 0;
    return layout_of(rows, cols, precision == MI_ADAMW_NS_SINGLE).bytes;
}

int32_t mi_adamw_ns_whole(int32_t rows, int32_t cols) {
    return sides_ok(rows, cols) ? whole_of(rows, cols) : MI_ADAMW_E_INVALID;
}

int mi_adamw_ns_check(const mi_adamw_ns_options* options) {
    return options_ok(options) ? MI_ADAMW_OK : MI_ADAMW_E_INVALID;
}

int mi_adamw_newton_schulz(const void* d_x, int64_t x_batch, int64_t x_row, void* d_out,
                           int64_t out_batch, int64_t out_row, int32_t batch, int32_t rows,
                           int32_t cols, int32_t dtype, const mi_adamw_ns_options* options,
                           void* d_workspace, int64_t workspace_bytes, void* stream) {
    if (!d_x || !d_out || batch <= 0 || !sides_ok(rows, cols) ||
        !options_ok(options) || x_row < cols || out_row < cols ||
        (dtype != MI_ADAMW_DTYPE_F32 && dtype != MI_ADAMW_DTYPE_BF16))
        return MI_ADAMW_E_INVALID;
    const bool single = options->precision == MI_ADAMW_NS_SINGLE;
    const Layout l = layout_of(rows, cols, single);
    const int32_t whole = whole_of(rows, cols);
    if (!whole) {
        if (!d_workspace) return MI_ADAMW_E_INVALID;
        if (reinterpret_cast<uintptr_t>(d_workspace) % 16) return MI_ADAMW_E_ALIGN;
        if (workspace_bytes / l.bytes < batch) return MI_ADAMW_E_SCRATCH;
    }
    mi_adamw_matrix one{};
    one.rows = rows;
    one.cols = cols;
    const Cut cut = whole ? Cut{64, 1, 64} : cut_for(&one, 1, batch, single);
    if ((whole ? 1 : items_of_matrix(rows, cols, MI_ADAMW_NS_TILES, 64, 1)) * batch > 0x7fffff)
        return MI_ADAMW_E_INVALID;
    BatchSource src;
    memset(&src, 0, sizeof(src));
    src.mat.rows = rows;
    src.mat.cols = cols;
    src.x = d_x;
    src.out = d_out;
    src.x_batch = x_batch;
    src.x_row = x_row;
    src.out_batch = out_batch;
    src.out_row = out_row;
    src.ws_batch = l.bytes;
    src.bf16 = dtype == MI_ADAMW_DTYPE_BF16;
    auto source_of = [&](int32_t kind, unsigned* grid) {
        BatchSource s = src;
        s.per = static_cast<int32_t>(items_of_matrix(
            rows, cols, kind, kind == MI_ADAMW_NS_PAIRS ? cut.pair_tile : cut.tile, cut.split));
        *grid = static_cast<unsigned>(s.per) * batch;
        return s;
    };
    const Momentum h{};
    const MuonOut out{};
    char* ws = static_cast<char*>(d_workspace);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (whole) {
        src.per = 1;
        launch_whole(src, static_cast<unsigned>(batch), whole, *options, h, out, s);
        return status();
    }
    return single ? run_steps<true>(source_of, *options, cut, h, out, ws, s)
                  : run_steps<false>(source_of, *options, cut, h, out, ws, s);
}

int mi_adamw_muon_cut(const mi_adamw_matrix* mats, int32_t n, int32_t precision,
                      mi_adamw_muon_tables* out) {
    if (!mats || n <= 0 || !out ||
        (precision != MI_ADAMW_NS_HALF && precision != MI_ADAMW_NS_SINGLE))
        return MI_ADAMW_E_INVALID;
    for (int32_t t = 0; t < n; ++t)
        if (!sides_ok(mats[t].rows, mats[t].cols)) return MI_ADAMW_E_INVALID;
    const Cut cut = cut_for(mats, n, 1, precision == MI_ADAMW_NS_SINGLE);
    out->pair_tile = cut.pair_tile;
    out->split = cut.split;
    out->tile = cut.tile;
    return MI_ADAMW_OK;
}

int64_t mi_adamw_muon_items(const mi_adamw_matrix* mats, int32_t n, int32_t kind, int32_t tile,
                            int32_t split, mi_adamw_chunk* out, int64_t cap) {
    if (!mats || n < 0 || !tile_ok(tile, false) || split < 1 || split > kMostShares ||
        kind < MI_ADAMW_NS_PARTS || kind > MI_ADAMW_NS_WHOLE)
        return MI_ADAMW_E_INVALID;
    int64_t total = 0;
    for (int32_t t = 0; t < n; ++t) {
        if (!sides_ok(mats[t].rows, mats[t].cols)) return MI_ADAMW_E_INVALID;
        const int64_t k = items_of_matrix(mats[t].rows, mats[t].cols, kind, tile, split);
        for (int64_t i = 0; i < k; ++i, ++total) {
            if (!out) continue;
            if (total >= cap) return MI_ADAMW_E_INVALID;
            out[total].tensor = t;
            out[total].index = static_cast<int32_t>(i);
        }
    }
    return total;
}

int mi_adamw_muon_step(const mi_adamw_tensor* d_tensors, const mi_adamw_matrix* d_matrices,
                       const mi_adamw_muon_tables* tables, const mi_adamw_muon_hyper* hyper,
                       const mi_adamw_ns_options* options, int32_t flags, void* d_workspace,
                       void* stream) {
    if (!d_tensors || !d_matrices || !tables || !hyper || !options_ok(options) ||
        (flags & ~MI_ADAMW_F_BF16_COPY) || tables->whole < 0 || tables->whole > 3)
        return MI_ADAMW_E_INVALID;
    for (int k = tables->whole ? MI_ADAMW_NS_WHOLE : 0; k < (tables->whole ? 5 : 4); ++k)
        if (!tables->items[k] || tables->n_items[k] <= 0 || tables->n_items[k] > 0x7fffff)
            return MI_ADAMW_E_INVALID;
    const bool single = options->precision == MI_ADAMW_NS_SINGLE;
    if (!tables->whole) {
        if (!d_workspace || !tile_ok(tables->pair_tile, single) || !tile_ok(tables->tile, single) ||
            tables->split < 1 || tables->split > kMostShares)
            return MI_ADAMW_E_INVALID;
        if (reinterpret_cast<uintptr_t>(d_workspace) % 16) return MI_ADAMW_E_ALIGN;
    }
    auto source_of = [&](int32_t kind, unsigned* grid) {
        *grid = static_cast<unsigned>(tables->n_items[kind]);
        return TableSource{d_tensors, d_matrices, tables->items[kind]};
    };
    const Momentum h{hyper->lerp_w, hyper->momentum, hyper->nesterov};
    const MuonOut out{hyper->wd_factor, hyper->neg_lr, flags & MI_ADAMW_F_BF16_COPY ? 1 : 0};
    char* ws = static_cast<char*>(d_workspace);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (tables->whole) {
        unsigned grid = 0;
        const TableSource src = source_of(MI_ADAMW_NS_WHOLE, &grid);
        launch_whole(src, grid, tables->whole, *options, h, out, s);
        return status();
    }
    const Cut cut{tables->pair_tile, tables->split, tables->tile};
    return single ? run_steps<true>(source_of, *options, cut, h, out, ws, s)
                  : run_steps<false>(source_of, *options, cut, h, out, ws, s);
}

}  // extern "C"
