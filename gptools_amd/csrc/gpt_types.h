// Element types of the read-out operators (gpt_norm.hip, gpt_class.hip): fp64, fp32, fp16, bf16. Sums, statistics and
// accumulators are held in Acc (fp32, or fp64 for fp64 data); a value is rounded to the element type once, on its way out.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gptt {

typedef _Float16 half_t;
typedef __bf16 bf16_t;

template <typename T> struct Elem {
    typedef float Acc;
};
template <> struct Elem<double> {
    typedef double Acc;
};
template <typename T> using acc_t = typename Elem<T>::Acc;

// 16 bytes of elements at an address that is aligned to the element only (gfx950 reads and writes such vectors in one
// instruction): rows of odd length keep wide accesses
template <typename T> struct Vec16 {
    static constexpr int N = 16 / (int)sizeof(T);
    typedef T V __attribute__((ext_vector_type(16 / sizeof(T))));
    typedef T U __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};
template <typename T> __device__ __forceinline__ typename Vec16<T>::V load16(const T* p) {
    return *reinterpret_cast<const typename Vec16<T>::U*>(p);
}
// The same for 16-bit elements that may start in the middle of a word, where lanes read rows of their own (such reads take twice the
// time): whole words, and one more (which the last element lies in), moved by half a word
template <typename T> __device__ __forceinline__ typename Vec16<T>::V load16_words(const T* p) {
    static_assert(sizeof(T) == 2, "two elements a word");
    typedef uint32_t W __attribute__((ext_vector_type(4), aligned(4)));
    const uint32_t odd = (uint32_t)(uintptr_t)p & 2;
    const uint32_t* q = reinterpret_cast<const uint32_t*>(reinterpret_cast<const char*>(p) - odd);
    const W w = *reinterpret_cast<const W*>(q);
    const uint32_t e = q[odd ? 4 : 3];
    const uint4 u = make_uint4(__builtin_amdgcn_alignbyte(w[1], w[0], odd), __builtin_amdgcn_alignbyte(w[2], w[1], odd),
                               __builtin_amdgcn_alignbyte(w[3], w[2], odd), __builtin_amdgcn_alignbyte(e, w[3], odd));
    return __builtin_bit_cast(typename Vec16<T>::V, u);
}
template <typename T> __device__ __forceinline__ void store16(T* p, typename Vec16<T>::V v) {
    *reinterpret_cast<typename Vec16<T>::U*>(p) = v;
}

template <typename T> __device__ __forceinline__ void store4(T* p, const T (&v)[4]) {
    typedef T V __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    *reinterpret_cast<V*>(p) = V{v[0], v[1], v[2], v[3]};
}

// A grid of many workgroups, in two dimensions (one counts its threads in 32 bits); workgroups behind the last of them may be there
inline dim3 wide_grid(int64_t blocks) {
    constexpr int64_t ROW = (int64_t)1 << 20;
    return blocks <= ROW ? dim3((unsigned)blocks) : dim3((unsigned)ROW, (unsigned)((blocks + ROW - 1) / ROW));
}
__device__ __forceinline__ int64_t wide_block() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

// sum over the 64 lanes of a wave, in every lane
template <typename A> __device__ __forceinline__ A wave_sum(A v) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
    return v;
}

// K sums over the THREADS consecutive threads that share a row (THREADS is 64, or the whole workgroup), in every one of
// them. red: THREADS / 64 * K values of LDS; two calls that use the same red need a barrier between them (`last` false
// leaves one behind).
template <int THREADS, int K, typename A> __device__ __forceinline__ void row_sum(A (&v)[K], A* red, bool last) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = wave_sum(v[k]);
    if (THREADS > 64) {
        constexpr int NW = THREADS / 64;
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) red[w * K + k] = v[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            A s = red[k];
#pragma unroll
            for (int i = 1; i < NW; ++i) s += red[i * K + k];
            v[k] = s;
        }
        if (!last) __syncthreads();
    }
}

} // namespace gptt
