// Matrix-core tiles of the read-out (gpt_class.hip): C[m][n] = sum_k A[m][k] B[n][k], both operands with k contiguous.
//
// A workgroup of WM x WN waves takes BM x BN of C and walks k in steps of 128 bytes a row. The step's rows stand in LDS in
// 16-byte chunks, chunk c of row r in slot c ^ (r & 7), so that the 16 rows that a wave reads at once spread over all banks.
// One 16-byte chunk a lane feeds one 16x16x32 instruction in 16 bits, four 16x16x4 in fp32 and two 16x16x4 in fp64: which k
// a lane's j-th value stands for does not matter as long as both operands agree.
#pragma once
#include "gpt_types.h"

namespace gptt {

template <typename T> struct Mma; // C fragment, product of two 16-byte chunks, row of C that register r of lane group q holds
template <> struct Mma<bf16_t> {
    typedef float C __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ C mul(Vec16<bf16_t>::V a, Vec16<bf16_t>::V b, C c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ int row(int q, int r) { return 4 * q + r; }
};
template <> struct Mma<half_t> {
    typedef float C __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ C mul(Vec16<half_t>::V a, Vec16<half_t>::V b, C c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ int row(int q, int r) { return 4 * q + r; }
};
template <> struct Mma<float> {
    typedef float C __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ C mul(Vec16<float>::V a, Vec16<float>::V b, C c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ int row(int q, int r) { return 4 * q + r; }
};
template <> struct Mma<double> {
    typedef double C __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ C mul(Vec16<double>::V a, Vec16<double>::V b, C c) {
#pragma unroll
        for (int j = 0; j < 2; ++j) c = __builtin_amdgcn_mfma_f64_16x16x4f64(a[j], b[j], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ int row(int q, int r) { return q + 4 * r; }
};

constexpr int TILE_CHUNKS = 8; // 16-byte chunks of a row in one k step
template <typename T> constexpr int tile_k() { return TILE_CHUNKS * Vec16<T>::N; }

template <typename T> struct Operand {
    const T* p; // [rows][ld]
    int64_t ld, rows;
};

// One 16-byte chunk, zeros where it lies outside rows x [0, k1)
template <typename T> __device__ __forceinline__ typename Vec16<T>::V tile_chunk(const Operand<T>& o, int64_t row, int64_t k, int64_t k1) {
    constexpr int N = Vec16<T>::N;
    typename Vec16<T>::V v = {};
    if (row < o.rows) {
        const T* p = o.p + row * o.ld + k;
        if (k + N <= k1) v = load16(p);
        else {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (k + e < k1) v[e] = p[e];
        }
    }
    return v;
}

template <typename T, int BM, int BN, int WM, int WN> struct Tile {
    typedef typename Vec16<T>::V Vec;
    typedef typename Mma<T>::C C;
    static constexpr int THREADS = 64 * WM * WN;
    static constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
    static constexpr int LOADS = (BM + BN) * TILE_CHUNKS / THREADS;
    static constexpr int LDS_BYTES = 2 * (BM + BN) * TILE_CHUNKS * 16;
    C acc[TM][TN];

    // acc <- the product over k in [k0, k1) of rows m0.. of A and n0.. of B; lds: LDS_BYTES, free again after the next barrier
    __device__ __forceinline__ void run(const Operand<T>& A, int64_t m0, const Operand<T>& B, int64_t n0, int64_t k0, int64_t k1,
                                        Vec* lds) {
        const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
        const int fm = (wave / WN) * (BM / WM) + (lane & 15), fn = BM + (wave % WN) * (BN / WN) + (lane & 15), q = lane >> 4;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = C{0, 0, 0, 0};
        Vec next[LOADS];
        auto fetch = [&](int64_t k) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int id = i * THREADS + t, row = id / TILE_CHUNKS, c = id % TILE_CHUNKS;
                const int64_t kk = k + c * Vec16<T>::N;
                next[i] = row < BM ? tile_chunk(A, m0 + row, kk, k1) : tile_chunk(B, n0 + (row - BM), kk, k1);
            }
        };
        auto put = [&](Vec* to) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int id = i * THREADS + t, row = id / TILE_CHUNKS, c = id % TILE_CHUNKS;
                to[row * TILE_CHUNKS + (c ^ (row & 7))] = next[i];
            }
        };
        if (k0 >= k1) return;
        fetch(k0);
        put(lds);
        __syncthreads();
        int side = 0;
        for (int64_t k = k0; k < k1; k += tile_k<T>()) {
            const bool more = k + tile_k<T>() < k1;
            if (more) fetch(k + tile_k<T>());
            const Vec* at = lds + side * (BM + BN) * TILE_CHUNKS;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                Vec a[TM], b[TN];
#pragma unroll
                for (int i = 0; i < TM; ++i) a[i] = at[(fm + 16 * i) * TILE_CHUNKS + ((4 * g + q) ^ (fm & 7))];
#pragma unroll
                for (int j = 0; j < TN; ++j) b[j] = at[(fn + 16 * j) * TILE_CHUNKS + ((4 * g + q) ^ (fn & 7))];
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j) acc[i][j] = Mma<T>::mul(a[i], b[j], acc[i][j]);
            }
            if (more) {
                put(lds + (side ^ 1) * (BM + BN) * TILE_CHUNKS);
                side ^= 1;
            }
            __syncthreads();
        }
    }
    // row of C (within the tile) of register r of fragment i; column of fragment j
    static __device__ __forceinline__ int row(int i, int r) {
        return ((int)(threadIdx.x >> 6) / WN) * (BM / WM) + 16 * i + Mma<T>::row((threadIdx.x & 63) >> 4, r);
    }
    static __device__ __forceinline__ int col(int j) {
        return ((int)(threadIdx.x >> 6) % WN) * (BN / WN) + 16 * j + (threadIdx.x & 15);
    }
};

} // namespace gptt
