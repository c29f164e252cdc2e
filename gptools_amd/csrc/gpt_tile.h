// Matrix-core tiles of the read-out (gpt_class.hip): C[m][n] = sum_k A[m][k] B[n][k], both operands with k contiguous.
//
// A workgroup of WM x WN waves takes BM x BN of C and walks k in steps of 128 bytes a row. The step's rows stand in LDS in
// 16-byte chunks, chunk c of row r in slot c ^ (r & 7), so that the 16 rows that a wave reads at once spread over all banks.
// One 16-byte chunk a lane feeds one 16x16x32 instruction in 16 bits, four 16x16x4 in fp32 and two 16x16x4 in fp64: which k
// a lane's j-th value stands for does not matter as long as both operands agree.
#pragma once
#include "gpt_types.h"
#include <type_traits>

namespace gptt {

template <typename T> struct Mma; // C fragment, product of two 16-byte chunks, row of C that register r of lane group q holds;
                                 // mul1: of one value a lane, that of lane group q standing for k = q; mul4: of four, k = 4 q + r
template <> struct Mma<bf16_t> {
    typedef float C __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ C mul(Vec16<bf16_t>::V a, Vec16<bf16_t>::V b, C c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    typedef short V4 __attribute__((ext_vector_type(4))); // bf16 bits
    static __device__ __forceinline__ C mul4(V4 a, V4 b, C c) { return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ int row(int q, int r) { return 4 * q + r; }
};
template <> struct Mma<half_t> {
    typedef float C __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ C mul(Vec16<half_t>::V a, Vec16<half_t>::V b, C c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    typedef half_t V4 __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ C mul4(V4 a, V4 b, C c) { return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ int row(int q, int r) { return 4 * q + r; }
};
template <> struct Mma<float> {
    typedef float C __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ C mul(Vec16<float>::V a, Vec16<float>::V b, C c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = mul1(a[j], b[j], c);
        return c;
    }
    static __device__ __forceinline__ C mul1(float a, float b, C c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ int row(int q, int r) { return 4 * q + r; }
};
template <> struct Mma<double> {
    typedef double C __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ C mul(Vec16<double>::V a, Vec16<double>::V b, C c) {
#pragma unroll
        for (int j = 0; j < 2; ++j) c = mul1(a[j], b[j], c);
        return c;
    }
    static __device__ __forceinline__ C mul1(double a, double b, C c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ int row(int q, int r) { return q + 4 * r; }
};

constexpr int TILE_CHUNKS = 8; // 16-byte chunks of a row in one k step
template <typename T> constexpr int tile_k() { return TILE_CHUNKS * Vec16<T>::N; }

template <typename T> struct Operand {
    const T* p; // [rows][ld], or several planes of that
    int64_t ld, rows;
    int64_t plane; // elements from one plane to the next
};

// fp32 as a sum of three bf16 values, by cutting off bits: each holds the eight leading bits of what is left. Six of the nine products
// of two such sums are taken; those left out are at most 2^-21 of the whole (the second value is below 2^-7 of the first, the third
// below 2^-15; two of them are second times third), 2^-24.5 on average for normal data, and have the product's sign. Here as fp32
// values whose low halves are zero.
// An infinity is the largest bf16 number twice and an infinity in the third place, which meets the other operand's first value alone:
// with a finite value other than zero all six products have one sign and one of them is infinite, as the product is. (In the first
// place it would meet the zeros that the second and third values of a short number are.) A NaN stands in the third place too.
__device__ __forceinline__ float split_high(float v) {
    constexpr float MOST = 3.38953138925153547590e38f; // (bf16's largest)
    return __builtin_amdgcn_fmed3f(__builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & 0xffff0000u), -MOST, MOST);
}
__device__ __forceinline__ void split3(float v, uint32_t& a, uint32_t& b, uint32_t& c) {
    const float fa = split_high(v), r = v - fa, fb = split_high(r);
    a = __builtin_bit_cast(uint32_t, fa);
    b = __builtin_bit_cast(uint32_t, fb);
    c = __builtin_bit_cast(uint32_t, r - fb);
}
// ... of two values, two bf16 in a word each
__device__ __forceinline__ void split3(float v, float w, uint32_t (&u)[3]) {
    uint32_t x[3], y[3];
    split3(v, x[0], x[1], x[2]);
    split3(w, y[0], y[1], y[2]);
#pragma unroll
    for (int p = 0; p < 3; ++p) u[p] = __builtin_amdgcn_perm(y[p], x[p], 0x07060302u);
}

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

template <typename T> struct SmallTile {
    typedef T Element;
    static constexpr int BM = 128, BN = 128, WM = 2, WN = 2;
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
        // rows behind the last repeat it: their products are not used
        const T* from[LOADS];
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int id = i * THREADS + t, row = id / TILE_CHUNKS, c = id % TILE_CHUNKS;
            const bool a = row < BM;
            const int64_t r = a ? m0 + row : n0 + (row - BM), last = (a ? A.rows : B.rows) - 1;
            from[i] = (a ? A.p : B.p) + (r < last ? r : last) * (a ? A.ld : B.ld) + c * Vec16<T>::N;
        }
        auto fetch = [&](int64_t k) {
            if (k + tile_k<T>() <= k1) {
#pragma unroll
                for (int i = 0; i < LOADS; ++i) next[i] = load16(from[i] + k);
                return;
            }
#pragma unroll
            for (int i = 0; i < LOADS; ++i) { // the rest of k: zeros behind it
                const int64_t left = k1 - k - (i * THREADS + t) % TILE_CHUNKS * Vec16<T>::N;
                next[i] = Vec{};
                if (left >= Vec16<T>::N) next[i] = load16(from[i] + k);
                else {
#pragma unroll
                    for (int e = 0; e < Vec16<T>::N; ++e)
                        if (e < left) next[i][e] = from[i][k + e];
                }
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
    // does this lane hold row m of C (within the tile)?
    static __device__ __forceinline__ bool holds(int m) {
        const int q = (threadIdx.x & 63) >> 4;
        return m / (BM / WM) == (int)(threadIdx.x >> 6) / WN && (Mma<T>::row(1, 0) == 1 ? (m & 3) : (m >> 2 & 3)) == q;
    }
    // row of C (within the tile) of register r of fragment i; column of fragment j
    static __device__ __forceinline__ int row(int i, int r) {
        return ((int)(threadIdx.x >> 6) / WN) * (BM / WM) + 16 * i + Mma<T>::row((threadIdx.x & 63) >> 4, r);
    }
    static __device__ __forceinline__ int col(int j) {
        return ((int)(threadIdx.x >> 6) % WN) * (BN / WN) + 16 * j + (threadIdx.x & 15);
    }
};

// May a LineTile read it? (its rows start on 16 bytes, a tile of them spans less than 4 GB)
template <typename T> bool tile_fits(const Operand<T>& o) {
    return ((uintptr_t)o.p & 15) == 0 && (o.ld * (int64_t)sizeof(T)) % 16 == 0 && o.ld < ((int64_t)1 << 22);
}

// The same product for operands whose rows start on 16 bytes (in 16 bits): 256 x 256 of C for 8 waves (or 256 x 128) or 128 x 128 for 4
// (WideTile, MidTile), each step's rows (64 KB, 32) taken from memory straight into LDS, two steps deep. Registers hold the fragments of the half step that is being multiplied
// and receive those of the next half from LDS meanwhile; one barrier a step. The stay of a step:
//   loads are issued in the middle of step s for step s + 2 (its buffer is free then: every wave holds the second half of
//   step s in registers), and must have landed in the middle of step s + 1.
// A rest of k behind the last whole step goes through registers at the end.
//
// Which rows of the operands stand in a fragment is free, and chosen so that the results leave in whole lines: lane group q
// holds rows 16 q .. 16 q + 15 of C in registers r of fragments 4 i' .. 4 i' + 3 (and four neighbouring lanes 16 columns), so
// that 16 neighbouring values of a column are one lane's, and the four groups' fill 128 bytes in 16 bits. The chunks of a row
// are swizzled by the row bits that differ within such a fragment.
//
// PLANES == 3: the operands are fp32 values split in three (split3), and k runs through six pairs of planes.
// TURN: A stands the other way, [k][m] (A.rows: its columns). Its step is 64 rows of BM values; the LDS read that transposes takes 4 rows of
// 4 times 4 columns for 16 lanes, which a swizzle of the chunks by the row spreads over half of the banks. (Over all of them, for 32 lanes at
// once, takes one more addition for every other fragment: no conflicts, and 1 % more time.) Fragment i holds rows 16 i .. of C then.
template <typename T, int PLANES, int BM_, int BN_, bool TURN = false> struct LineTile {
    typedef T Element;
    typedef typename Vec16<T>::V Vec;
    typedef typename Mma<T>::C C;
    static constexpr int BM = BM_, BN = BN_, WM = BN == 256 ? 2 : BM / 64, WN = BN / 64;
    static constexpr int THREADS = 64 * WM * WN, TM = BM / WM / 16, TN = 4;
    static constexpr int LOADS = (BM + BN) * TILE_CHUNKS / THREADS; // of a step
    static_assert(BM * TILE_CHUNKS == 4 * THREADS && (LOADS == 8 || LOADS == 6), "four loads of A a step, four of B or two");
    static constexpr int STEP = (BM + BN) * TILE_CHUNKS; // chunks
    static __device__ __forceinline__ int key(int row) { return (row & 3) | (row >> 2 & 4); }
    static __device__ __forceinline__ int fragment(int i) { return 64 * (i >> 2) + 4 * (i & 3); } // first row of fragment i
    static constexpr int LDS_BYTES = 2 * STEP * 16;
    C acc[TM][TN];

    // bytes of row's chunk from the tile's first row on (rows behind the last repeat it: their products are not used)
    static __device__ __forceinline__ uint32_t source(const Operand<T>& o, int64_t r0, int row, int slot) {
        const int64_t last = o.rows - 1 - r0;
        const int64_t r = row < last ? row : last;
        return (uint32_t)(r * o.ld * (int64_t)sizeof(T)) + (uint32_t)(slot ^ key(row)) * 16;
    }
    static constexpr int ACROSS = BM / 8; // TURN: chunks of a row of A
    // byte of A's chunk in row k, slot `slot` of the step (columns behind the last whole chunk repeat it)
    static __device__ __forceinline__ uint32_t source_turned(const Operand<T>& o, int64_t m0, int k, int slot) {
        const int64_t last = (o.rows + 7) / 8 - 1 - m0 / 8;
        const int c = slot ^ (k & 3) << 1;
        return (uint32_t)(k * o.ld * (int64_t)sizeof(T)) + (uint32_t)(c < last ? c : last) * 16;
    }
    // this lane's part of a fragment's address: see read_turned
    static __device__ __forceinline__ uint32_t turned(int i, int wm) {
        const int lane = threadIdx.x & 63, kk = lane >> 2 & 3;
        return (8 * (lane >> 4) + kk) * (BM * 2) + (wm / 8 + 2 * (i ^ kk) + (lane >> 1 & 1)) * 16 + (lane & 1) * 8;
    }
    // fragment i, k = 32 g + 8 (lane group) + 0 .. 7
    static __device__ __forceinline__ Vec read_turned(const Vec* at, const uint32_t (&from)[4], int i, int g) {
        typedef short V4 __attribute__((ext_vector_type(4)));
        typedef short V8 __attribute__((ext_vector_type(8)));
        typedef __attribute__((address_space(3))) V4 L;
        auto* p = (__attribute__((address_space(3))) char*)at + from[i & 3] + (i >> 2) * 128 + 32 * g * (BM * 2);
        const V4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L*)p), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L*)(p + 4 * (BM * 2)));
        return __builtin_bit_cast(Vec, (V8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    // LOADS loads of 16 bytes a lane into LDS (a wave's 64 lanes side by side). The LDS address goes through m0; the waits that
    // the hardware does not make by itself: a scalar register that a vector instruction wrote, m0 before its use
    static __device__ __forceinline__ void take(const T* a, const T* b, const uint32_t (&from)[LOADS], uint32_t to) {
        asm volatile("s_nop 4\n\t"
                     "s_mov_b32 m0, %5\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %0\n\t"
                     "s_add_u32 m0, %5, %6\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %0\n\t"
                     "s_add_u32 m0, %5, %7\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %0\n\t"
                     "s_add_u32 m0, %5, %8\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %4, %0"
                     :
                     : "s"(a), "v"(from[0]), "v"(from[1]), "v"(from[2]), "v"(from[3]), "s"(to), "i"(16 * THREADS),
                       "i"(32 * THREADS), "i"(48 * THREADS)
                     : "memory", "scc"); // (m0 is the compiler's scratch: it sets it before each use of its own)
        asm volatile("s_nop 4\n\t"
                     "s_add_u32 m0, %3, %4\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %0\n\t"
                     "s_add_u32 m0, %3, %5\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %0"
                     :
                     : "s"(b), "v"(from[4]), "v"(from[5]), "s"(to), "i"(64 * THREADS), "i"(80 * THREADS)
                     : "memory", "scc");
        if constexpr (LOADS == 8)
            asm volatile("s_nop 4\n\t"
                         "s_add_u32 m0, %3, %4\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %0\n\t"
                         "s_add_u32 m0, %3, %5\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %0"
                         :
                         : "s"(b), "v"(from[6]), "v"(from[7]), "s"(to), "i"(96 * THREADS), "i"(112 * THREADS)
                         : "memory", "scc");
    }
    static __device__ __forceinline__ void arrive() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

    __device__ __forceinline__ void run(const Operand<T>& A, int64_t m0, const Operand<T>& B, int64_t n0, int64_t k0, int64_t k1,
                                        Vec* lds) {
        const int t = threadIdx.x, lane = t & 63, wave = t >> 6, q = lane >> 4;
        const int at16 = 16 * (lane >> 2 & 3) + (lane & 3); // this lane's row within a fragment
        const int fm = (wave / WN) * (BM / WM) + at16, fn = BM + (wave % WN) * (BN / WN) + at16;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = C{0, 0, 0, 0};
        constexpr int PAIRS = PLANES == 3 ? 6 : 1;
        const int64_t each = (k1 - k0) / tile_k<T>(), steps = PAIRS * each; // (with planes k1 - k0 is a whole number of steps)
        uint32_t turn[4];
        if constexpr (TURN) {
#pragma unroll
            for (int i = 0; i < 4; ++i) turn[i] = turned(i, (wave / WN) * (BM / WM));
        }
        auto fragment_a = [&](const Vec* at, int i, int g, int cm) {
            if constexpr (TURN) return read_turned(at, turn, i, g);
            else return at[(fm + fragment(i)) * TILE_CHUNKS + cm];
        };
        // one half step: acc += a b, while a and bn take the fragments of half g of the step at `at`
        Vec a[TM + 1];
        // A ninth slot lets every fragment of the next half leave LDS one group of instructions early, so that the barrier behind a half
        // does not wait for the last (bf16 4096 x 4096 x 32000: 819 us against 849). Fragments stand in slots 0 .. TM - 1 before FORTH, and
        // one on (0 in TM) after it; BACK takes them back
        auto half = [&](auto forth, const Vec(&b)[TN], Vec(&bn)[TN], const Vec* at, int g) {
            constexpr bool FORTH = decltype(forth)::value;
            const int cm = (4 * g + q) ^ key(fm), cn = (4 * g + q) ^ key(fn);
            if (FORTH) a[TM] = fragment_a(at, 0, g, cm);
            else a[TM - 1] = fragment_a(at, TM - 1, g, cm);
#pragma unroll
            for (int s = 0; s < TM; ++s) {
                const int i = FORTH ? s : TM - 1 - s, slot = FORTH ? i : (i + TM) % (TM + 1); // FORTH: i in i; BACK: i in i - 1, 0 in TM
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = Mma<T>::mul(a[slot], b[j], acc[i][j]);
                if (FORTH && i + 1 < TM) a[i] = fragment_a(at, i + 1, g, cm);
                if (!FORTH && i > 0) a[i - 1] = fragment_a(at, i - 1, g, cm);
                if (s < TN) bn[s] = at[(fn + fragment(s)) * TILE_CHUNKS + cn];
            }
            __builtin_amdgcn_sched_group_barrier(0x100, TURN ? 2 : 1, 0);
#pragma unroll
            for (int s = 0; s < TM; ++s) { // matrix instructions, reads of LDS
                __builtin_amdgcn_sched_group_barrier(0x008, TN, 0);
                if (s < TN) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                if (s + 1 < TM) __builtin_amdgcn_sched_group_barrier(0x100, TURN ? 2 : 1, 0);
            }
        };
        auto first = [&](Vec(&b)[TN], const Vec* at) {
#pragma unroll
            for (int j = 0; j < TN; ++j) b[j] = at[(fn + fragment(j)) * TILE_CHUNKS + (q ^ key(fn))];
#pragma unroll
            for (int i = 0; i < TM; ++i) a[i] = fragment_a(at, i, 0, q ^ key(fm));
        };
        auto mul = [&](const Vec(&b)[TN]) {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = Mma<T>::mul(a[i], b[j], acc[i][j]);
        };
        auto mul_on = [&](const Vec(&b)[TN]) {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = Mma<T>::mul(a[(i + TM) % (TM + 1)], b[j], acc[i][j]);
        };
        auto second = [&](Vec(&b)[TN], const Vec* at) {
#pragma unroll
            for (int j = 0; j < TN; ++j) b[j] = at[(fn + fragment(j)) * TILE_CHUNKS + ((4 + q) ^ key(fn))];
#pragma unroll
            for (int i = 0; i < TM; ++i) a[i] = fragment_a(at, i, 1, (4 + q) ^ key(fm));
        };
        Vec b0[TN], b1[TN];
        if (steps > 0) {
            uint32_t from[LOADS];
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int id = (i & 3) * THREADS + t;
                from[i] = TURN && i < 4 ? source_turned(A, m0, id / ACROSS, id % ACROSS)
                                        : source(i < 4 ? A : B, i < 4 ? m0 : n0, id / TILE_CHUNKS, id % TILE_CHUNKS);
            }
            const T *const a0 = TURN ? A.p + k0 * A.ld + m0 : A.p + m0 * A.ld + k0, *const b0_ = B.p + n0 * B.ld + k0, *pa = a0, *pb = b0_;
            int64_t left = each;
            int pair = 0;
            auto onward = [&]() {
                pa += TURN ? tile_k<T>() * A.ld : tile_k<T>(), pb += tile_k<T>();
                if (PLANES == 3 && --left == 0) { // pairs of planes (0,0) (0,1) (1,0) (1,1) (0,2) (2,0)
                    left = each;
                    ++pair;
                    pa = a0 + (0x001102 >> 4 * (pair > 5 ? 0 : 5 - pair) & 15) * A.plane;
                    pb = b0_ + (0x010120 >> 4 * (pair > 5 ? 0 : 5 - pair) & 15) * B.plane;
                }
            };
            const uint32_t to = __builtin_amdgcn_readfirstlane(
                (uint32_t)(uintptr_t)(__attribute__((address_space(3))) Vec*)lds + (uint32_t)wave * 1024);
            take(pa, pb, from, to);
            onward();
            arrive();
            if (steps > 1) take(pa, pb, from, to + STEP * 16);
            onward();
            first(b0, lds);
            int side = 0;
            for (int64_t s = 0; s + 1 < steps; ++s) {
                half(std::true_type(), b0, b1, lds + side * STEP, 1);
                arrive(); // step s + 1 is there, and step s is in registers to its end
                if (s + 2 < steps) take(pa, pb, from, to + side * STEP * 16);
                onward();
                side ^= 1;
                half(std::false_type(), b1, b0, lds + side * STEP, 0);
            }
            half(std::true_type(), b0, b1, lds + side * STEP, 1);
            mul_on(b1);
        }
        const int64_t k = k0 + each * tile_k<T>();
        if (PLANES == 1 && k < k1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int id = (i & 3) * THREADS + t, row = id / TILE_CHUNKS, c = id % TILE_CHUNKS;
                if (TURN && i < 4) {
                    const int r = id / ACROSS, slot = id % ACROSS;
                    lds[id] = k + r < k1 ? load16(A.p + (k + r) * A.ld + m0 + source_turned(A, m0, 0, slot ^ (r & 3) << 1) / sizeof(T)) : Vec{};
                } else lds[(i < 4 ? 0 : BM * TILE_CHUNKS) + row * TILE_CHUNKS + (c ^ key(row))] =
                    tile_chunk(i < 4 ? A : B, (i < 4 ? m0 : n0) + row, k + c * Vec16<T>::N, k1);
            }
            __syncthreads();
            first(b0, lds);
            mul(b0);
            second(b0, lds);
            mul(b0);
        }
        __syncthreads();
    }
    static __device__ __forceinline__ bool holds(int m) {
        return m / (BM / WM) == (int)(threadIdx.x >> 6) / WN && (m >> 4 & 3) == (int)(threadIdx.x & 63) >> 4;
    }
    static __device__ __forceinline__ int row(int i, int r) {
        const int q = (threadIdx.x & 63) >> 4;
        return ((int)(threadIdx.x >> 6) / WN) * (BM / WM) + (TURN ? 16 * i + 4 * q : fragment(i) + 16 * q) + r;
    }
    static __device__ __forceinline__ int col(int j) {
        return ((int)(threadIdx.x >> 6) % WN) * (BN / WN) + fragment(j) + 16 * (threadIdx.x >> 2 & 3) + (threadIdx.x & 3);
    }
};

template <typename T, int PLANES = 1> using WideTile = LineTile<T, PLANES, 256, 256>;
template <typename T, int PLANES = 1> using MidTile = LineTile<T, PLANES, 128, 128>;
// What the last columns are taken with where they fill no more than half of a tile (void: the same). 600 rows x 4096 x 128000 classes
// in bf16: 615 us against 655, 1375 x 2048 x 50001 in fp16 268 against 284. (Half a tile takes four fifths of a whole one's time)
template <typename Tl> struct HalfOf {
    typedef void Tile;
};
template <typename T, int PLANES, bool TURN> struct HalfOf<LineTile<T, PLANES, 256, 256, TURN>> {
    typedef LineTile<T, PLANES, 256, 128, TURN> Tile;
};
// The tile with A the other way, where there is one
template <typename Tl> struct TurnedOf {
    typedef Tl Tile;
};
template <typename T, int PLANES, int BM, int BN> struct TurnedOf<LineTile<T, PLANES, BM, BN>> {
    typedef LineTile<T, PLANES, BM, BN, true> Tile;
};

// Which tile a workgroup takes: workgroups go round the 8 XCDs, each of which has an L2 of its own, so each XCD takes a
// contiguous run of tiles, and a run goes through 8 columns of tiles row by row (32 tiles at work share 4 + 8 panels).
// false: none (the grid is rounded up to the XCDs)
__device__ __forceinline__ bool tile_place(int64_t id, int64_t tiles_m, int64_t tiles_n, int64_t& m, int64_t& n) {
    const int64_t total = tiles_m * tiles_n, run = (total + 7) / 8;
    const int64_t at = (id & 7) * run + (id >> 3);
    if (id >> 3 >= run || at >= total) return false;
    const int64_t band = at / (8 * tiles_m), in = at - band * 8 * tiles_m;
    const int64_t wide = tiles_n - 8 * band < 8 ? tiles_n - 8 * band : 8;
    m = __builtin_amdgcn_readfirstlane((int)(in / wide)); // (the same in all lanes, which division does not show)
    n = __builtin_amdgcn_readfirstlane((int)(8 * band + in % wide));
    return true;
}
// ... of Tl's size, for `cols` columns. Whole tiles before halves, so that the halves fill the card's last round, but in stretches of
// BAND rows of tiles at most: the halves find them in the last-level cache (128 MB of rows of 8 KB)
constexpr int64_t BAND = 64;
__host__ __device__ __forceinline__ int64_t tile_band(int64_t tiles_m) {
    const int64_t bands = (tiles_m + BAND - 1) / BAND;
    return (tiles_m + bands - 1) / bands;
}
template <typename Tl> __device__ __forceinline__ bool tile_place(int64_t id, int64_t tiles_m, int64_t cols, int64_t& m, int64_t& n, bool& half) {
    typedef typename HalfOf<Tl>::Tile Half;
    const int64_t rest = cols % Tl::BN, whole = cols / Tl::BN;
    half = false;
    if constexpr (!std::is_void<Half>::value) half = rest > 0 && rest <= Half::BN;
    if (!half) return tile_place(id, tiles_m, whole + (rest > 0), m, n);
    const int64_t band = tile_band(tiles_m), first = (band * whole + 7) / 8 * 8, each = first + (band + 7) / 8 * 8, m0 = id / each * band;
    const int64_t here = tiles_m - m0 < band ? tiles_m - m0 : band;
    if (here <= 0) return false;
    id %= each;
    half = id >= first;
    if (half) id -= first;
    if (!tile_place(id, here, half ? 1 : whole, m, n)) return false;
    m += m0;
    if (half) n = whole;
    return true;
}
// The number of workgroup `in` of split `split`: the splits of fewer tiles than there are XCDs start on different ones (fp32 100 rows x
// 300 x 30000 with the reverse mode: 130 us against 172)
__device__ __forceinline__ int64_t split_place(int64_t in, int64_t split, int64_t tiles) {
    return (in & ~(int64_t)7) | ((in + split * tiles) & 7);
}
template <typename Tl> int64_t tile_grid(int64_t tiles_m, int64_t cols) {
    const int64_t tiles_n = (cols + Tl::BN - 1) / Tl::BN;
    if (std::is_void<typename HalfOf<Tl>::Tile>::value) return (tiles_m * tiles_n + 7) / 8 * 8;
    const int64_t band = tile_band(tiles_m);
    return (tiles_m + band - 1) / band * ((band * tiles_n + 7) / 8 * 8 + 8);
}

} // namespace gptt
