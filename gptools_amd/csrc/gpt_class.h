// What the kernels of the categorical log density share (gpt_class.hip, gpt_class_narrow.hip).
#pragma once
#include "gpt_types.h"
#include <type_traits>

namespace gptt {

template <typename A> __device__ __forceinline__ A neg_inf() { return -(A)__builtin_inf(); }

// In fp32 logits, maxima and lse are kept times log2(e): an exponential is one instruction then
constexpr float LOG2E = 1.44269504088896340736f;
__device__ __forceinline__ float times_log2e(float v) { return v * LOG2E; }
__device__ __forceinline__ float from_log2e(float v) { return v * 0.69314718055994530942f; }
__device__ __forceinline__ float exp_log2e(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ double times_log2e(double v) { return v; }
__device__ __forceinline__ double from_log2e(double v) { return v; }
__device__ __forceinline__ double exp_log2e(double v) { return exp(v); }
__device__ __forceinline__ float log_(float x) { return logf(x); }
__device__ __forceinline__ double log_(double x) { return log(x); }
__device__ __forceinline__ float log1p_(float x) { return log1pf(x); }
__device__ __forceinline__ double log1p_(double x) { return log1p(x); }
// alpha: a finite one stays finite (the type's lowest value is no exclusion)
__device__ __forceinline__ float level_log2e(float v) {
    return v == neg_inf<float>() ? v : fmaxf(times_log2e(v), -3.40282346638528859812e38f);
}
__device__ __forceinline__ double level_log2e(double v) { return v; }

// the value that exponentials are taken about: the maximum, or zero where no class is possible (their sum is then zero)
template <typename A> __device__ __forceinline__ A about(A mx) { return mx == neg_inf<A>() ? (A)0 : mx; }
// (mx, s) <- maximum and sum of exponentials about it of two sets of classes. A NaN among the logits is a NaN in s
template <typename A> __device__ __forceinline__ void join(A& mx, A& s, A mo, A so) {
    const A mm = fmax(mx, mo), ref = about(mm);
    s = s * exp_log2e(mx - ref) + so * exp_log2e(mo - ref);
    mx = mm;
}
// What a row's probabilities come from: exp(eta - top) * share, share = 1 / (the sum of the exponentials about top). (exp(eta - lse)
// is one operation less, but lse's own rounding is relative to its size: a level common to all classes, which cancels, would cost
// them digits.) top infinite, share zero: none, where no class is possible; NaN where the row's class is none
template <typename A> struct RowSum {
    A top, share;
};
template <typename A> __device__ __forceinline__ RowSum<A> row_sum_of(int64_t y, int64_t classes, A mx, A s) {
    if (mx == neg_inf<A>() && s == 0) return {(A)__builtin_inf(), (A)0};
    return {about(mx), y >= classes ? (A)__builtin_nan("") : (A)1 / s};
}
// a row's log probability from all classes' maximum (or a reference below it) and sum. eta_y is the logit that the sum holds, to the
// bit: where it takes more than half of the sum, the rest comes from the same values, and the log probability is never above zero
template <typename A> __device__ __forceinline__ A row_lp(int64_t y, int64_t classes, A mx, A s, A eta_y) {
    const A p = exp_log2e(eta_y - about(mx));
    if (y < 0) return 0;
    if (y >= classes) return (A)__builtin_nan("");
    if (mx == neg_inf<A>() && s == 0) return neg_inf<A>();
    return p > (A)0.5 * s ? -log1p_(fmax(s - p, (A)0) / p) : from_log2e(eta_y - about(mx)) - log_(s);
}

// sum over the 16 lanes of a row of lanes, in each of them
__device__ __forceinline__ float sum16(float v) {
#define GPT_ADD_DPP(ctrl) v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, 0xf, 0xf, true))
    GPT_ADD_DPP(0xb1);  // lane ^ 1
    GPT_ADD_DPP(0x4e);  // lane ^ 2
    GPT_ADD_DPP(0x141); // the other four of eight
    GPT_ADD_DPP(0x140); // the other eight
#undef GPT_ADD_DPP
    return v;
}
__device__ __forceinline__ double sum16(double v) {
#pragma unroll
    for (int k = 8; k >= 1; k >>= 1) v += __shfl_xor(v, k, 64);
    return v;
}


template <typename T> __host__ __device__ constexpr float stored_scale() { return std::is_same<T, half_t>::value ? 16384.f : 1.f; }

constexpr int SCALE_PARTS = 64;
// largest |lpbar| of the observed rows from class_scale's parts (null: no lpbar, 1), for a whole wave; 1 where it is no scale
template <typename A> struct Largest {
    const A* parts;
    __device__ __forceinline__ A get() const {
        if (!parts) return 1;
        A m = parts[threadIdx.x & 63];
#pragma unroll
        for (int k = 32; k >= 1; k >>= 1) m = fmax(m, __shfl_xor(m, k, 64));
        return m > 0 && m < (A)__builtin_inf() ? m : (A)1;
    }
};

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    typedef T V2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, V2{(T)a, (T)b});
}

namespace { // (a kernel of its own in each of the two)

// Numbers the observed rows: row[number], y[number] (or null; any y that is no class as `classes`), their count; behind them row lists the
// others, whose lp is 0. place (or null): the rows' numbers, -1 where there is no observation. parts (or null): the largest |lpbar| of
// the observed rows of a workgroup, as class_scale leaves it. A workgroup takes INDEX_ROWS rows; runs: the observed ones of every
// INDEX_ROWS (class_count), or null, and it counts those before its own for itself.
constexpr int INDEX_ROWS = 4096;
constexpr int64_t INDEX_ALONE = 4 * INDEX_ROWS; // rows up to which counting the ones before is shorter than another launch
__global__ __launch_bounds__(1024) void class_count(const int64_t* y, int64_t rows, int* runs) {
    __shared__ int red[16];
    const int64_t mine = (int64_t)blockIdx.x * INDEX_ROWS + 4 * threadIdx.x;
    int n = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) n += mine + k < rows && y[mine + k] >= 0;
    n = wave_sum(n);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x) return;
#pragma unroll
    for (int k = 1; k < 16; ++k) n += red[k];
    runs[blockIdx.x] = n;
}
template <typename A> __global__ __launch_bounds__(1024) void class_index(const int64_t* y, int64_t rows, int64_t classes, int* place, int* row,
                                                                         int* y_of, int* count, A* lp, const A* lpbar, A* parts,
                                                                         const int* runs) {
    __shared__ int red[2][16];
    __shared__ A most[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t first = (int64_t)blockIdx.x * INDEX_ROWS, mine = first + 4 * threadIdx.x;
    int before = 0, n = 0;
    if (runs) {
        for (int i = threadIdx.x; i < (int)blockIdx.x; i += 1024) before += runs[i];
    } else {
        for (int64_t i = threadIdx.x; i < first; i += INDEX_ROWS) { // (whole runs)
            int64_t u[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) u[k] = y[i + 1024 * k];
#pragma unroll
            for (int k = 0; k < 4; ++k) before += u[k] >= 0;
        }
    }
    int64_t v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        v[k] = mine + k < rows ? y[mine + k] : -1;
        n += v[k] >= 0;
    }
    if (parts) {
        A m = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (v[k] >= 0) m = fmax(m, fabs(lpbar[mine + k]));
#pragma unroll
        for (int k = 32; k >= 1; k >>= 1) m = fmax(m, __shfl_xor(m, k, 64));
        if (lane == 0) most[wave] = m;
    }
    int upto = n; // of this wave's lanes up to this one
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
        const int o = __shfl_up(upto, k, 64);
        if (lane >= k) upto += o;
    }
    before = wave_sum(before);
    if (lane == 63) {
        red[0][wave] = before;
        red[1][wave] = upto;
    }
    __syncthreads();
    int at = upto - n, all = 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        at += red[0][k] + (k < wave ? red[1][k] : 0);
        all += red[0][k] + red[1][k];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t i = mine + k;
        if (i >= rows) continue;
        const bool seen = v[k] >= 0;
        if (place) place[i] = seen ? at : -1;
        if (seen) {
            row[at] = (int)i;
            if (y_of) y_of[at] = (int)(v[k] < classes ? v[k] : classes);
            ++at;
        } else {
            row[rows - 1 - (i - at)] = (int)i; // (i - at rows before this one have no observation)
            lp[i] = 0;
        }
    }
    if (threadIdx.x == 0 && blockIdx.x == gridDim.x - 1) *count = all;
    if (parts && threadIdx.x == 0) {
        A m = most[0];
#pragma unroll
        for (int k = 1; k < 16; ++k) m = fmax(m, most[k]);
        parts[blockIdx.x] = m;
        if (blockIdx.x == 0)
            for (int k = gridDim.x; k < SCALE_PARTS; ++k) parts[k] = 0;
    }
}

// parts[b] = the largest |lpbar| of the observed rows that workgroup b of SCALE_PARTS takes
template <typename A> __global__ __launch_bounds__(256) void class_scale(const A* lpbar, const int64_t* y, int64_t rows, A* parts) {
    __shared__ A red[4];
    A m = 0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows; i += 256 * SCALE_PARTS)
        if (y[i] >= 0) m = fmax(m, fabs(lpbar[i]));
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) m = fmax(m, __shfl_xor(m, k, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) parts[blockIdx.x] = fmax(fmax(red[0], red[1]), fmax(red[2], red[3]));
}

// runs: room for a count of every INDEX_ROWS rows
template <typename A> void number_rows(const int64_t* y, int64_t rows, int64_t classes, int* place, int* row, int* y_of, int* count, A* lp,
                                       const A* lpbar, A* parts, int* runs, hipStream_t st) {
    const dim3 grid((unsigned)((rows + INDEX_ROWS - 1) / INDEX_ROWS));
    const bool alone = rows <= INDEX_ALONE;
    if (!alone) class_count<<<grid, dim3(1024), 0, st>>>(y, rows, runs);
    class_index<A><<<grid, dim3(1024), 0, st>>>(y, rows, classes, place, row, y_of, count, lp, lpbar, parts, alone ? nullptr : runs);
}

} // namespace
} // namespace gptt
