// layer_norm.hip -- layer norm over the last dimension, with an optional residual addition in
// front of it, and its gradient (gfx950).
//
// Forward, a row of H values s = x (+ residual, rounded to the sum's type, which is an output):
//   mean = sum(s) / H,  var = sum((s - mean)^2) / H,  rstd = 1 / sqrt(var + eps)
//   y = (s - mean) rstd w + b
// Backward, with h = (s - mean) rstd and g = dy w:
//   dx = rstd (g - sum(g) / H - h sum(g h) / H) (+ dsum),  dw = sum over rows of dy h,
//   db = sum over rows of dy
//
// Both are bound by memory: a row is read once into registers, its sums are formed there in
// fp32 (the variance from the centred values), and the results leave from there.  A row takes
// one wave up to 1024 values, and one workgroup of 256 or 1024 lanes above that (bf16 rows then in
// 16-byte loads).  The
// backward's workgroups walk many rows each and keep their columns' share of dw and db in
// registers; the shares are added up in a fixed order by a second launch, so that results
// never depend on timing.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <cmath>

#include "mi_adamw.h"
#include "fp32_math.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// Element-aligned groups in memory: rows of an odd width begin anywhere.
typedef f32x4 f32x4_mem __attribute__((aligned(4)));
typedef u32x2 u32x2_mem __attribute__((aligned(2)));
typedef u32x4 u32x4_mem __attribute__((aligned(2)));

#define GLOBAL __attribute__((address_space(1)))

constexpr int kLongThreads = 1024;
constexpr int kStrip = 256;         // columns of a workgroup of the long rows' weight pass
constexpr int kF32 = MI_ADAMW_DTYPE_F32, kBf16 = MI_ADAMW_DTYPE_BF16, kNone = -1;

typedef mi_adamw_layer_norm_args Fwd;
typedef mi_adamw_layer_norm_grad_args Bwd;

template <int kN>
struct Vec {
    float v[kN];
    __device__ __forceinline__ float& operator[](int i) { return v[i]; }
    __device__ __forceinline__ float operator[](int i) const { return v[i]; }
};

// kN elements as they lie in memory: a row's loads are all under way before the first value is
// used.
template <int kType, int kN>
struct Raw {
    alignas(kType == kBf16 && kN == 4 ? 8 : 16) uint32_t w[kType == kF32 ? kN : kN / 2];
};

// Elements i .. i + kN - 1; `count` of them are there, the rest 0.
template <int kType, int kN>
__device__ __forceinline__ Raw<kType, kN> ld_raw(const void* p, int64_t i, int count) {
    Raw<kType, kN> r;
    constexpr int kWords = sizeof(r.w) / 4;
    if (count >= kN) {
        if (kType == kF32) {
            const float* q = static_cast<const float*>(p) + i;
#pragma unroll
            for (int k = 0; k < kN; k += 4)
                *(f32x4*)(r.w + k) = *(const GLOBAL f32x4_mem*)(q + k);
        } else {
            const uint16_t* q = static_cast<const uint16_t*>(p) + i;
            if (kN == 4) *(u32x2*)(r.w) = *(const GLOBAL u32x2_mem*)(q);
            else *(u32x4*)(r.w) = *(const GLOBAL u32x4_mem*)(q);
        }
        return r;
    }
#pragma unroll
    for (int k = 0; k < kWords; ++k) r.w[k] = 0;
#pragma unroll
    for (int k = 0; k < kN - 1; ++k)
        if (k < count) {
            if (kType == kF32) {
                r.w[k] = *(const GLOBAL uint32_t*)(static_cast<const uint32_t*>(p) + i + k);
            } else {
                const uint32_t h = *(const GLOBAL uint16_t*)(static_cast<const uint16_t*>(p) + i + k);
                r.w[k / 2] |= h << (k % 2 * 16);
            }
        }
    return r;
}

template <int kType, int kN>
__device__ __forceinline__ Vec<kN> values(const Raw<kType, kN>& r) {
    Vec<kN> v;
#pragma unroll
    for (int k = 0; k < kN; ++k) {
        if (kType == kF32) v[k] = __uint_as_float(r.w[k]);
        else v[k] = __uint_as_float(k % 2 ? r.w[k / 2] & 0xffff0000u : r.w[k / 2] << 16);
    }
    return v;
}

template <int kType, int kN>
__device__ __forceinline__ Vec<kN> ld(const void* p, int64_t i, int count) {
    return values<kType, kN>(ld_raw<kType, kN>(p, i, count));
}
// The same of a type that is known only at run time.
template <int kN>
__device__ __forceinline__ Vec<kN> ld_any(const void* p, int32_t dtype, int64_t i, int count) {
    return dtype == kF32 ? ld<kF32, kN>(p, i, count) : ld<kBf16, kN>(p, i, count);
}

// kPast: without displacing what the caches hold.  Outputs: 16384 x 4096 bf16, forward 46 us so and
// 63 with ordinary stores, backward 88 and 93; a reader right behind takes the same time either
// way at 16 to 256 MB.
template <bool kPast, int kN>
__device__ __forceinline__ void st(void* p, int32_t dtype, int64_t i, const Vec<kN>& v, int count) {
    if (dtype == kF32) {
        float* q = static_cast<float*>(p) + i;
        if (count >= kN) {
#pragma unroll
            for (int k = 0; k < kN; k += 4) {
                const f32x4 w = {v[k], v[k + 1], v[k + 2], v[k + 3]};
                if (kPast) __builtin_nontemporal_store(w, (GLOBAL f32x4_mem*)(q + k));
                else *(GLOBAL f32x4_mem*)(q + k) = w;
            }
            return;
        }
#pragma unroll
        for (int k = 0; k < kN - 1; ++k)
            if (k < count) *(GLOBAL float*)(q + k) = v[k];
    } else {
        uint16_t* q = static_cast<uint16_t*>(p) + i;
        if (count >= kN) {
            alignas(kN == 4 ? 8 : 16) uint32_t w[kN / 2];
#pragma unroll
            for (int k = 0; k < kN / 2; ++k) w[k] = bf16x2_bits(v[2 * k], v[2 * k + 1]);
            if (kN == 4) {
                if (kPast) __builtin_nontemporal_store(*(const u32x2*)(w), (GLOBAL u32x2_mem*)(q));
                else *(GLOBAL u32x2_mem*)(q) = *(const u32x2*)(w);
            } else {
                if (kPast) __builtin_nontemporal_store(*(const u32x4*)(w), (GLOBAL u32x4_mem*)(q));
                else *(GLOBAL u32x4_mem*)(q) = *(const u32x4*)(w);
            }
            return;
        }
#pragma unroll
        for (int k = 0; k < kN - 1; ++k)
            if (k < count)
                *(GLOBAL uint16_t*)(q + k) = static_cast<uint16_t>(bf16_bits(v[k]));
    }
}

// v as it reads back from a tensor of the dtype.
template <int kN>
__device__ __forceinline__ void round_to(Vec<kN>& v, int32_t dtype) {
    if (dtype == kF32) return;
#pragma unroll
    for (int k = 0; k < kN; ++k) v[k] = __uint_as_float(bf16_bits(v[k]) << 16);
}

// The weight (or bias) of columns c .. c + kN - 1, or `other` where there is none.
template <int kN>
__device__ __forceinline__ Vec<kN> affine(const float* p, int64_t c, int count, float other) {
    if (p) return ld<kF32, kN>(p, c, count);
    Vec<kN> v;
#pragma unroll
    for (int k = 0; k < kN; ++k) v[k] = other;
    return v;
}

// The sums over the kLanes lanes of a row, in every one of them; the same bits in each.  Calls of
// one kernel alternate between the two halves of lds, so that one barrier does.
template <int kLanes, int kSums>
__device__ __forceinline__ void row_sums(float (&v)[kSums], float* lds) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1)
#pragma unroll
        for (int k = 0; k < kSums; ++k) v[k] += __shfl_xor(v[k], d);
    if (kLanes == 64) return;
    constexpr int kWaves = kLanes / 64;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int k = 0; k < kSums; ++k) lds[k * kWaves + (threadIdx.x >> 6)] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSums; ++k) {
        v[k] = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) v[k] += lds[k * kWaves + w];
    }
}

// kLanes lanes a row, kIter groups of kN elements a lane.  16384 x 4096 bf16: 46 us, 5.8 TB/s;
// 2048 x 768 fp32 with a bf16 branch 6.2 us, most of it a launch's and two memory latencies.
template <int kLanes, int kIter, int kN, int kX, int kRes>
__global__ __launch_bounds__(kLanes > 256 ? kLanes : 256) void mi_adamw_layer_norm_kernel(Fwd f) {
    constexpr int kRows = kLanes > 256 ? 1 : 256 / kLanes;
    __shared__ float lds[2][16];
    const int lane = threadIdx.x % kLanes;
    const int64_t row = int64_t(blockIdx.x) * kRows + threadIdx.x / kLanes;
    if (row >= f.rows) return;              // whole rows: a wave's, or a workgroup's
    const int32_t h = static_cast<int32_t>(f.hidden);
    Raw<kX, kN> raw[kIter];
    Raw<kRes == kNone ? kF32 : kRes, kN> raw2[kRes == kNone ? 1 : kIter];
#pragma unroll
    for (int k = 0; k < kIter; ++k) {
        const int32_t c = (k * kLanes + lane) * kN;
        raw[k] = ld_raw<kX, kN>(f.x, row * f.x_row + c, h - c);
        if (kRes != kNone)
            raw2[k] = ld_raw<kRes == kNone ? kF32 : kRes, kN>(f.residual, row * f.residual_row + c,
                                                              h - c);
    }
    Vec<kN> v[kIter];
    float sum[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < kIter; ++k) {
        v[k] = values<kX, kN>(raw[k]);
        if (kRes != kNone) {
            constexpr int kSum = kX == kBf16 && kRes == kBf16 ? kBf16 : kF32;
            const int32_t c = (k * kLanes + lane) * kN;
            const Vec<kN> r = values<kRes == kNone ? kF32 : kRes, kN>(raw2[k]);
            for (int e = 0; e < kN; ++e) v[k][e] += r[e];
            round_to(v[k], kSum);
            st<true>(f.sum, kSum, row * h + c, v[k], h - c);
        }
        float part = 0.0f;
        for (int e = 0; e < kN; e += 4) part += (v[k][e] + v[k][e + 1]) + (v[k][e + 2] + v[k][e + 3]);
        sum[0] += part;
    }
    row_sums<kLanes>(sum, lds[0]);
    const float mean = sum[0] / h;
    float sq[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < kIter; ++k) {
        const int32_t c = (k * kLanes + lane) * kN;
        for (int e = 0; e < kN; ++e) {
            v[k][e] = c + e < h ? v[k][e] - mean : 0.0f;
            sq[0] = __builtin_fmaf(v[k][e], v[k][e], sq[0]);
        }
    }
    row_sums<kLanes>(sq, lds[1]);
    const float rstd = 1.0f / sqrtf(sq[0] / h + f.eps);
#pragma unroll
    for (int k = 0; k < kIter; ++k) {
        const int32_t c = (k * kLanes + lane) * kN;
        const Vec<kN> w = affine<kN>(f.weight, c, h - c, 1.0f);
        const Vec<kN> b = affine<kN>(f.bias, c, h - c, 0.0f);
        for (int e = 0; e < kN; ++e) v[k][e] = __builtin_fmaf(v[k][e] * rstd, w[e], b[e]);
        st<true>(f.y, f.y_dtype, row * h + c, v[k], h - c);
    }
    if (f.mean && lane == 0) {
        f.mean[row] = mean;
        f.rstd[row] = rstd;
    }
}

__device__ __forceinline__ int32_t sum_dtype(const Fwd& f) {
    return f.x_dtype == kBf16 && f.residual_dtype == kBf16 ? kBf16 : kF32;
}

// Rows of any length, read again for each sum, from the caches while a row fits them: 2048 x 32769
// bf16 87 us (3.1 TB/s of what has to move), fp32 159 (3.4); 64 x 1048576 bf16 409 (0.66), a quarter
// of the CUs at work.  Widths past 32768 are no model's here; that there is an answer is the point.
__global__ __launch_bounds__(kLongThreads) void mi_adamw_layer_norm_long_kernel(Fwd f) {
    __shared__ float lds[2][16];
    const int64_t row = blockIdx.x;
    const int64_t h = f.hidden;
    const int32_t dtype = sum_dtype(f);
    const void* from = f.residual ? f.sum : f.x;
    const int32_t from_dtype = f.residual ? dtype : f.x_dtype;
    const int64_t base = f.residual ? row * h : row * f.x_row;
    float sum[1] = {0.0f};
    for (int64_t c = threadIdx.x * 4; c < h; c += kLongThreads * 4) {
        const int count = static_cast<int>(h - c < 4 ? h - c : 4);
        Vec<4> v = ld_any<4>(f.x, f.x_dtype, row * f.x_row + c, count);
        if (f.residual) {
            const Vec<4> r =
                ld_any<4>(f.residual, f.residual_dtype, row * f.residual_row + c, count);
            for (int e = 0; e < 4; ++e) v[e] += r[e];
            round_to(v, dtype);
            st<false>(f.sum, dtype, base + c, v, count);   // read back by the lane that wrote it
        }
        sum[0] += (v[0] + v[1]) + (v[2] + v[3]);
    }
    row_sums<kLongThreads>(sum, lds[0]);
    const float mean = sum[0] / h;
    float sq[1] = {0.0f};
    for (int64_t c = threadIdx.x * 4; c < h; c += kLongThreads * 4) {
        const int count = static_cast<int>(h - c < 4 ? h - c : 4);
        const Vec<4> v = ld_any<4>(from, from_dtype, base + c, count);
        for (int e = 0; e < 4; ++e) {
            const float d = e < count ? v[e] - mean : 0.0f;
            sq[0] = __builtin_fmaf(d, d, sq[0]);
        }
    }
    row_sums<kLongThreads>(sq, lds[1]);
    const float rstd = 1.0f / sqrtf(sq[0] / h + f.eps);
    for (int64_t c = threadIdx.x * 4; c < h; c += kLongThreads * 4) {
        const int count = static_cast<int>(h - c < 4 ? h - c : 4);
        Vec<4> v = ld_any<4>(from, from_dtype, base + c, count);
        const Vec<4> w = affine<4>(f.weight, c, count, 1.0f);
        const Vec<4> b = affine<4>(f.bias, c, count, 0.0f);
        for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf((v[e] - mean) * rstd, w[e], b[e]);
        st<false>(f.y, f.y_dtype, row * h + c, v, count);
    }
    if (f.mean && threadIdx.x == 0) {
        f.mean[row] = mean;
        f.rstd[row] = rstd;
    }
}

// The gradient's rows w, w + groups, ...: dx, and the group's share of dw and db.  The next row is
// on its way while one is worked on: 16384 x 4096 bf16 88 us, 4.6 TB/s, where a row at a time
// took 223.
template <int kLanes, int kIter, int kN, int kX, int kDy>
__global__ __launch_bounds__(kLanes > 256 ? kLanes : 256) void mi_adamw_layer_norm_grad_kernel(
    Bwd f) {
    constexpr int kRows = kLanes > 256 ? 1 : 256 / kLanes;
    __shared__ float lds[2][32];
    __shared__ float fold[kLanes == 64 ? kIter * 64 * kN : 1];
    const int lane = threadIdx.x % kLanes;
    const int group = threadIdx.x / kLanes;
    const int32_t h = static_cast<int32_t>(f.hidden);
    const float inv_h = 1.0f / h;
    Vec<kN> w[kIter], dw[kIter], db[kIter];
#pragma unroll
    for (int k = 0; k < kIter; ++k) {
        const int32_t c = (k * kLanes + lane) * kN;
        w[k] = affine<kN>(f.weight, c, h - c, 1.0f);
        for (int e = 0; e < kN; ++e) dw[k][e] = db[k][e] = 0.0f;
    }
    struct Row {
        Raw<kX, kN> x[kIter];
        Raw<kDy, kN> g[kIter];
        float mean, rstd;
    };
    auto fetch = [&](int64_t row, Row& r) {
#pragma unroll
        for (int k = 0; k < kIter; ++k) {
            const int32_t c = (k * kLanes + lane) * kN;
            r.x[k] = ld_raw<kX, kN>(f.x, row * f.x_row + c, h - c);
            r.g[k] = ld_raw<kDy, kN>(f.dy, row * f.dy_row + c, h - c);
        }
        r.mean = f.mean[row];
        r.rstd = f.rstd[row];
    };
    const int64_t step = int64_t(gridDim.x) * kRows;
    int64_t row = int64_t(blockIdx.x) * kRows + group;
    // (1024 lanes have 128 registers each, none to spare for that)
    constexpr bool kAhead = kLanes <= 256;
    Row now;
    if (kAhead && row < f.rows) fetch(row, now);
    for (int turn = 0; row < f.rows; row += step, turn ^= 1) {
        Row next;
        if (!kAhead) fetch(row, now);
        else if (row + step < f.rows) fetch(row + step, next);
        Raw<kX, kN> old[kIter];
        if (f.dsum)
#pragma unroll
            for (int k = 0; k < kIter; ++k) {
                const int32_t c = (k * kLanes + lane) * kN;
                old[k] = ld_raw<kX, kN>(f.dsum, row * f.dsum_row + c, h - c);
            }
        Vec<kN> x[kIter], g[kIter];
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < kIter; ++k) {
            const int32_t c = (k * kLanes + lane) * kN;
            x[k] = values<kX, kN>(now.x[k]);
            g[k] = values<kDy, kN>(now.g[k]);
            for (int e = 0; e < kN; ++e) {
                const float hat = c + e < h ? (x[k][e] - now.mean) * now.rstd : 0.0f;
                x[k][e] = hat;
                dw[k][e] = __builtin_fmaf(g[k][e], hat, dw[k][e]);
                db[k][e] += g[k][e];
                g[k][e] *= w[k][e];
                s[0] += g[k][e];
                s[1] = __builtin_fmaf(g[k][e], hat, s[1]);
            }
        }
        if (f.dx) {
            row_sums<kLanes>(s, lds[turn]);
            s[0] *= inv_h;
            s[1] *= inv_h;
#pragma unroll
            for (int k = 0; k < kIter; ++k) {
                const int32_t c = (k * kLanes + lane) * kN;
                Vec<kN> d;
                for (int e = 0; e < kN; ++e)
                    d[e] = now.rstd * (g[k][e] - __builtin_fmaf(x[k][e], s[1], s[0]));
                if (f.dsum) {
                    const Vec<kN> ds = values<kX, kN>(old[k]);
                    for (int e = 0; e < kN; ++e) d[e] += ds[e];
                }
                st<true>(f.dx, f.dx_dtype, row * h + c, d, h - c);
                if (f.dresidual) st<true>(f.dresidual, f.dresidual_dtype, row * h + c, d, h - c);
            }
        }
        if (kAhead) now = next;
    }
    if (!f.partials) return;
    // shares: [workgroup][dw, db][h]
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float* out = f.partials + (int64_t(blockIdx.x) * 2 + which) * h;
        if (kLanes == 64) {
            // the workgroup's four waves, one after the other
            for (int turn = 0; turn < kRows; ++turn) {
                __syncthreads();
                if (group == turn)
#pragma unroll
                    for (int k = 0; k < kIter; ++k) {
                        const int at = (k * kLanes + lane) * kN;
                        for (int e = 0; e < kN; ++e) {
                            const float v = which ? db[k][e] : dw[k][e];
                            fold[at + e] = turn ? fold[at + e] + v : v;
                        }
                    }
            }
            __syncthreads();
            for (int c = threadIdx.x; c < h; c += 256) out[c] = fold[c];
        } else {
#pragma unroll
            for (int k = 0; k < kIter; ++k) {
                const int32_t c = (k * kLanes + lane) * kN;
                st<false>(out, kF32, c, which ? db[k] : dw[k], h - c);
            }
        }
    }
}

// dx of rows of any length, read twice: 2048 x 32769 bf16 215 us, fp32 221, with the weights'
// gradient 361 and 341 (four bytes at a time a lane, two for bf16: 1.1 and 2.4 TB/s of what has to
// move).
__global__ __launch_bounds__(kLongThreads) void mi_adamw_layer_norm_long_grad_kernel(Bwd f) {
    __shared__ float lds[32];
    const int64_t row = blockIdx.x, h = f.hidden;
    const float mean = f.mean[row], rstd = f.rstd[row], inv_h = 1.0f / h;
    float s[2] = {0.0f, 0.0f};
    for (int turn = 0; turn < 2; ++turn) {
        for (int64_t c = threadIdx.x * 4; c < h; c += kLongThreads * 4) {
            const int count = static_cast<int>(h - c < 4 ? h - c : 4);
            const Vec<4> x = ld_any<4>(f.x, f.x_dtype, row * f.x_row + c, count);
            Vec<4> g = ld_any<4>(f.dy, f.dy_dtype, row * f.dy_row + c, count), d;
            const Vec<4> w = affine<4>(f.weight, c, count, 1.0f);
            for (int e = 0; e < 4; ++e) {
                const float hat = e < count ? (x[e] - mean) * rstd : 0.0f;
                g[e] *= w[e];
                if (turn == 0) {
                    s[0] += g[e];
                    s[1] = __builtin_fmaf(g[e], hat, s[1]);
                } else {
                    d[e] = rstd * (g[e] - __builtin_fmaf(hat, s[1], s[0]));
                }
            }
            if (turn == 0) continue;
            if (f.dsum) {
                const Vec<4> ds = ld_any<4>(f.dsum, f.x_dtype, row * f.dsum_row + c, count);
                for (int e = 0; e < 4; ++e) d[e] += ds[e];
            }
            st<false>(f.dx, f.dx_dtype, row * h + c, d, count);
            if (f.dresidual) st<false>(f.dresidual, f.dresidual_dtype, row * h + c, d, count);
        }
        if (turn == 0) {
            row_sums<kLongThreads>(s, lds);
            s[0] *= inv_h;
            s[1] *= inv_h;
        }
    }
}

// Shares of dw and db of long rows: a strip of columns and every gridDim.y-th row, an element a lane.
__global__ __launch_bounds__(kStrip) void mi_adamw_layer_norm_long_weight_kernel(Bwd f) {
    const int64_t c = int64_t(blockIdx.x) * kStrip + threadIdx.x, h = f.hidden;
    if (c >= h) return;
    float dw = 0.0f, db = 0.0f;
    for (int64_t row = blockIdx.y; row < f.rows; row += gridDim.y) {
        const float x = ld_any<4>(f.x, f.x_dtype, row * f.x_row + c, 1)[0];
        const float g = ld_any<4>(f.dy, f.dy_dtype, row * f.dy_row + c, 1)[0];
        dw = __builtin_fmaf(g, (x - f.mean[row]) * f.rstd[row], dw);
        db += g;
    }
    float* out = f.partials + int64_t(blockIdx.y) * 2 * h + c;
    out[0] = dw;
    out[h] = db;
}

// dw and db from the shares: 16 columns a workgroup, its 16 rows of lanes every sixteenth share
// each, added up in 64 bits.  512 shares of 2 x 4096: 6.9 us (2.4 TB/s); of 2 x 768 4.0 us (11.6
// with 64 columns a workgroup).
__global__ __launch_bounds__(256) void mi_adamw_layer_norm_fold_kernel(Bwd f, int32_t parts) {
    __shared__ double lds[16][17];
    const int64_t h = f.hidden;
    const int x = threadIdx.x & 15, y = threadIdx.x >> 4;
    const int64_t c = int64_t(blockIdx.x) * 16 + x;
    float* out = blockIdx.y ? f.dbias : f.dweight;
    if (!out) return;
    double sum = 0.0;
    if (c < h) {
        const float* from = f.partials + blockIdx.y * h + c;
        int32_t p = y;
        for (; p + 7 * 16 < parts; p += 8 * 16) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = from[int64_t(p + k * 16) * 2 * h];
#pragma unroll
            for (int k = 0; k < 8; ++k) sum += v[k];
        }
        for (; p < parts; p += 16) sum += from[int64_t(p) * 2 * h];
    }
    lds[y][x] = sum;
    __syncthreads();
    if (y == 0 && c < h) {
        for (int k = 1; k < 16; ++k) sum += lds[k][x];
        out[c] = static_cast<float>(sum);
    }
}

// ---------------------------------------------------------------------------
// Host side

int status() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MI_ADAMW_OK : static_cast<int>(e);
}

bool dtype_ok(int32_t d) { return d == MI_ADAMW_DTYPE_F32 || d == MI_ADAMW_DTYPE_BF16; }

constexpr int64_t kMaxHidden = int64_t(1) << 24;
constexpr int64_t kMaxRows = 0x7fffff;
constexpr int64_t kLongForward = 32768, kLongBackward = 16384;

bool sizes_ok(int64_t rows, int64_t hidden) {
    return rows > 0 && hidden > 0 && rows <= kMaxRows && hidden <= kMaxHidden;
}

// Shares of dw and db: the workgroups that the rows are dealt to, two for each CU at most (16384 x
// 4096 bf16: 93 us and 7 for the fold, with 1024 of them 95 and 12).  Few rows get a workgroup or
// wave each (2048 x 768: 7.7 us and 4.0 for the fold, with two rows each 9.5 and 3.4).
int32_t parts_of(int64_t rows, int64_t hidden) {
    const int64_t per = hidden <= 1024 ? 4 : 1;
    const int64_t most = hidden > kLongBackward ? 64 : 512;
    const int64_t groups = (rows + per - 1) / per;
    return static_cast<int32_t>(groups < most ? groups : most);
}

template <int kLanes, int kIter, int kN, int kX>
void launch_forward(const Fwd& a, hipStream_t s) {
    constexpr int kRows = kLanes > 256 ? 1 : 256 / kLanes;
    const dim3 grid(static_cast<unsigned>((a.rows + kRows - 1) / kRows));
    const dim3 lanes(kLanes > 256 ? kLanes : 256);
    if (!a.residual)
        hipLaunchKernelGGL((mi_adamw_layer_norm_kernel<kLanes, kIter, kN, kX, kNone>), grid, lanes, 0,
                           s, a);
    else if (a.residual_dtype == kF32)
        hipLaunchKernelGGL((mi_adamw_layer_norm_kernel<kLanes, kIter, kN, kX, kF32>), grid, lanes, 0,
                           s, a);
    else
        hipLaunchKernelGGL((mi_adamw_layer_norm_kernel<kLanes, kIter, kN, kX, kBf16>), grid, lanes,
                           0, s, a);
}

template <int kLanes, int kIter, int kN>
void launch(const Fwd& a, hipStream_t s) {
    if (a.x_dtype == kF32) launch_forward<kLanes, kIter, kN, kF32>(a, s);
    else launch_forward<kLanes, kIter, kN, kBf16>(a, s);
}

template <int kLanes, int kIter, int kN>
void launch(const Bwd& a, int32_t parts, hipStream_t s) {
    const dim3 grid(parts), lanes(kLanes > 256 ? kLanes : 256);
    if (a.x_dtype == kF32 && a.dy_dtype == kF32)
        hipLaunchKernelGGL((mi_adamw_layer_norm_grad_kernel<kLanes, kIter, kN, kF32, kF32>), grid,
                           lanes, 0, s, a);
    else if (a.x_dtype == kF32)
        hipLaunchKernelGGL((mi_adamw_layer_norm_grad_kernel<kLanes, kIter, kN, kF32, kBf16>), grid,
                           lanes, 0, s, a);
    else if (a.dy_dtype == kF32)
        hipLaunchKernelGGL((mi_adamw_layer_norm_grad_kernel<kLanes, kIter, kN, kBf16, kF32>), grid,
                           lanes, 0, s, a);
    else
        hipLaunchKernelGGL((mi_adamw_layer_norm_grad_kernel<kLanes, kIter, kN, kBf16, kBf16>), grid,
                           lanes, 0, s, a);
}

}  // namespace

extern "C" {

int mi_adamw_layer_norm(const mi_adamw_layer_norm_args* a, void* stream) {
    if (!a || !a->x || !a->y || !sizes_ok(a->rows, a->hidden) || !dtype_ok(a->x_dtype) ||
        !dtype_ok(a->y_dtype) || a->x_row < 0 || !a->mean != !a->rstd || !(a->eps >= 0.0f) ||
        !std::isfinite(a->eps) || !a->residual != !a->sum ||
        (a->residual && (!dtype_ok(a->residual_dtype) || a->residual_row < 0)))
        return MI_ADAMW_E_INVALID;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t h = a->hidden;
    if (h <= 256) launch<64, 1, 4>(*a, s);
    else if (h <= 512) launch<64, 2, 4>(*a, s);
    else if (h <= 768) launch<64, 3, 4>(*a, s);
    else if (h <= 1024) launch<64, 4, 4>(*a, s);
    else if (h <= 2048) launch<256, 1, 8>(*a, s);
    else if (h <= 4096) launch<256, 2, 8>(*a, s);
    else if (h <= 8192) launch<256, 4, 8>(*a, s);
    else if (h <= 16384) launch<1024, 2, 8>(*a, s);
    else if (h <= kLongForward) launch<1024, 4, 8>(*a, s);
    else
        hipLaunchKernelGGL(mi_adamw_layer_norm_long_kernel, dim3(static_cast<unsigned>(a->rows)),
                           dim3(kLongThreads), 0, s, *a);
    return status();
}

int64_t mi_adamw_layer_norm_grad_workspace(int64_t rows, int64_t hidden) {
    if (!sizes_ok(rows, hidden)) return MI_ADAMW_E_INVALID;
    return int64_t(parts_of(rows, hidden)) * 2 * hidden * 4;
}

int mi_adamw_layer_norm_grad(const mi_adamw_layer_norm_grad_args* a, void* stream) {
    if (!a || !a->x || !a->dy || !a->mean || !a->rstd || !sizes_ok(a->rows, a->hidden) ||
        !dtype_ok(a->x_dtype) || !dtype_ok(a->dy_dtype) || a->x_row < 0 || a->dy_row < 0 ||
        (a->dx && !dtype_ok(a->dx_dtype)) || (a->dsum && a->dsum_row < 0) ||
        (a->dresidual && (!a->dx || !dtype_ok(a->dresidual_dtype))) ||
        ((a->dweight || a->dbias) && !a->partials) || (!a->dx && !a->dweight && !a->dbias))
        return MI_ADAMW_E_INVALID;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t h = a->hidden;
    mi_adamw_layer_norm_grad_args b = *a;
    if (!a->dweight && !a->dbias) b.partials = nullptr;
    const int32_t parts = parts_of(a->rows, h);
    if (h <= 256) launch<64, 1, 4>(b, parts, s);
    else if (h <= 512) launch<64, 2, 4>(b, parts, s);
    else if (h <= 768) launch<64, 3, 4>(b, parts, s);
    else if (h <= 1024) launch<64, 4, 4>(b, parts, s);
    else if (h <= 2048) launch<256, 1, 8>(b, parts, s);
    else if (h <= 4096) launch<256, 2, 8>(b, parts, s);
    else if (h <= 8192) launch<256, 4, 8>(b, parts, s);
    else if (h <= kLongBackward) launch<1024, 2, 8>(b, parts, s);
    else {
        if (b.dx)
            hipLaunchKernelGGL(mi_adamw_layer_norm_long_grad_kernel,
                               dim3(static_cast<unsigned>(a->rows)), dim3(kLongThreads), 0, s, b);
        if (b.partials)
            hipLaunchKernelGGL(mi_adamw_layer_norm_long_weight_kernel,
                               dim3(static_cast<unsigned>((h + kStrip - 1) / kStrip), parts),
                               dim3(kStrip), 0, s, b);
    }
    if (b.partials)
        hipLaunchKernelGGL(mi_adamw_layer_norm_fold_kernel,
                           dim3(static_cast<unsigned>((h + 15) / 16), 2), dim3(256), 0, s, b,
                           parts);
    return status();
}

}  // extern "C"
