// The categorical log density for few rows (up to 64; gpt_class.hip includes this): a token or a batch of tokens of a generating
// model. Bound by reading beta (and writing betabar): the products have few columns, so beta's rows go from memory straight
// into the registers that the matrix instruction reads, no LDS between.
//
//   class_few_logits  16 classes a workgroup or 64 (32 in fp64), whose waves share the features; their logits' maximum and sum for every row,
//                     and for the reverse mode the logits themselves, or, where the classes are too many to hold these and r
//                     at once, those of a piece of the classes at a time when all sums are known
//   class_few_r       r in both orders, alphabar
//   class_few_back    xbar = r beta, and betabar = r^T x, which is bound by writing it. For xbar beta's rows lie along the
//                     features, the sum runs over the classes: a lane reads 16 bytes of eight classes and turns the block over in
//                     its registers (in 16 bits one byte permutation for two values)
#pragma once
#include "gpt_class.h"
#include "gpt_tile.h"

namespace gptt {

constexpr int FEW = 64; // rows

template <typename T> struct FewArgs {
    Operand<T> x, beta;
    const T* alpha;
    const int64_t* y;
    const acc_t<T>* lpbar;
    int64_t features, v0; // v0: class of beta's first row
    acc_t<T>*part_max, *part_sum; // [rows][tiles]
    acc_t<T>* eta_y;              // [rows]: logits of the rows' classes, as the sums have them
    int64_t tiles;
    acc_t<T>* eta; // [rows][ldv], times log2(e) in fp32
    int64_t ldv;
    RowSum<acc_t<T>>* of;  // [rows]; null: no reverse mode
    acc_t<T>*lp, *largest; // largest: |lpbar| of each observed row, zero to FEW
    T *r, *rt;                   // [rows][ldv], [classes][ldrt]
    int64_t ldrt;
    T* alphabar;
    acc_t<T>* xpart; // [splits][rows][features]; null: one split, the result itself
    bool add;        // xpart holds earlier pieces' sums
    T* xbar;
    int64_t share;   // classes of a split
};

// NT tiles of 16 rows, CT of 16 classes, WK waves that share the features. HALF: rows may start in the middle of a word (bf16 12 rows x
// 1959 x 34026 54 us against 80)
template <typename T, int NT, int CT, int WK, bool HALF> __global__ __launch_bounds__(64 * WK) void class_few_logits(FewArgs<T> a) {
    typedef acc_t<T> A;
    typedef typename Vec16<T>::V Vec;
    typedef typename Mma<T>::C C;
    constexpr int N = Vec16<T>::N, STEP = 4 * N; // a wave's step: 64 bytes of a row
    __shared__ A sum[WK][CT * 16][NT * 16 + 1];
    __shared__ int own[NT * 16]; // the rows' classes where they are among the workgroup's, counted from its first
    const int64_t y = threadIdx.x < NT * 16 && threadIdx.x < a.x.rows ? a.y[threadIdx.x] : -1; // (on its way while the product runs)
    const int lane = threadIdx.x & 63, q = lane >> 4, wave = threadIdx.x >> 6;
    const int64_t v0 = (int64_t)blockIdx.x * CT * 16, V = a.beta.rows, D = a.features;
    C c[CT][NT];
#pragma unroll
    for (int i = 0; i < CT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) c[i][t] = C{0, 0, 0, 0};
    const T *pb[CT], *px[NT];
#pragma unroll
    for (int i = 0; i < CT; ++i) { // (rows behind the last repeat it: their results are not used)
        const int64_t v = v0 + 16 * i + (lane & 15);
        pb[i] = a.beta.p + (v < V ? v : V - 1) * a.beta.ld + q * N;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int64_t n = 16 * t + (lane & 15);
        px[t] = a.x.p + (n < a.x.rows ? n : a.x.rows - 1) * a.x.ld + q * N;
    }
    auto load = [](const T* p) {
        if constexpr (HALF) return load16_words(p);
        else return load16(p);
    };
    const int64_t whole = D / STEP;
    // Runs of AHEAD steps a wave. Few steps on their way, and many waves, read beta faster than the other way round; and four
    // class tiles share each read of x, which comes from the caches at the same rate: bf16, 64 rows x 128000 classes x 4096
    // features 262 us with CT = 4, AHEAD = 2 (284 with 4; CT = 2 421, 8 370); 16 x 69974 x 3584 106 us (CT = 1 142); one row x
    // 32000 x 4096 39 us (45)
    constexpr int AHEAD = CT >= 4 ? 2 : 4;
    const int64_t runs = whole / AHEAD;
    for (int64_t g = wave; g < runs; g += WK) {
        Vec b[AHEAD][CT], x[AHEAD][NT];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
#pragma unroll
            for (int i = 0; i < CT; ++i) b[u][i] = load(pb[i] + (g * AHEAD + u) * STEP);
#pragma unroll
            for (int t = 0; t < NT; ++t) x[u][t] = load(px[t] + (g * AHEAD + u) * STEP);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int i = 0; i < CT; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t) c[i][t] = Mma<T>::mul(b[u][i], x[u][t], c[i][t]);
    }
    for (int64_t s = runs * AHEAD + wave; s < whole; s += WK) {
#pragma unroll
        for (int i = 0; i < CT; ++i) {
            const Vec b = load(pb[i] + s * STEP);
#pragma unroll
            for (int t = 0; t < NT; ++t) c[i][t] = Mma<T>::mul(b, load(px[t] + s * STEP), c[i][t]);
        }
    }
    if (whole * STEP < D && wave == (int)(whole % WK)) {
        const int64_t k = whole * STEP + q * N;
#pragma unroll
        for (int i = 0; i < CT; ++i) {
            const int64_t v = v0 + 16 * i + (lane & 15);
            const Vec b = tile_chunk(a.beta, v, k, D);
#pragma unroll
            for (int t = 0; t < NT; ++t) c[i][t] = Mma<T>::mul(b, tile_chunk(a.x, (int64_t)16 * t + (lane & 15), k, D), c[i][t]);
        }
    }
#pragma unroll
    for (int i = 0; i < CT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) sum[wave][16 * i + Mma<T>::row(q, r)][16 * t + (lane & 15)] = c[i][t][r];
    if (threadIdx.x < NT * 16) {
        const int64_t at = y - a.v0 - v0;
        own[threadIdx.x] = at >= 0 && at < V - v0 && at < 16 * CT ? (int)at : -1;
    }
    __syncthreads();
    // 16 threads a row (NT * 16 rows; the workgroup may take them in several goes), CT classes each
    const int k = threadIdx.x & 15;
    for (int n = threadIdx.x >> 4; n < NT * 16; n += 4 * WK) {
        A e[CT], mx = neg_inf<A>(), s = 0;
#pragma unroll
        for (int i = 0; i < CT; ++i) {
            const int64_t v = v0 + 16 * i + k;
            A u = 0;
#pragma unroll
            for (int w = 0; w < WK; ++w) u += sum[w][16 * i + k][n];
            e[i] = times_log2e(u) + (v < V ? (a.alpha ? level_log2e((A)a.alpha[v]) : (A)0) : neg_inf<A>());
            mx = fmax(mx, e[i]);
            if (a.eta && n < a.x.rows && v < a.ldv) a.eta[n * a.ldv + v] = e[i];
        }
#pragma unroll
        for (int m = 8; m >= 1; m >>= 1) mx = fmax(mx, __shfl_xor(mx, m, 64));
#pragma unroll
        for (int i = 0; i < CT; ++i) s += exp_log2e(e[i] - about(mx));
        s = sum16(s);
        if (own[n] >= 0) { // (few workgroups hold a row's class)
#pragma unroll
            for (int i = 0; i < CT; ++i)
                if (own[n] == 16 * i + k) a.eta_y[n] = e[i];
        }
        if (k == 0 && n < a.x.rows) {
            a.part_max[n * a.tiles + blockIdx.x] = mx;
            a.part_sum[n * a.tiles + blockIdx.x] = s;
        }
    }
}

// xt[d][n] = x[n][d] (zero without an observation, and behind the last row): 64 features
template <typename T> __device__ __forceinline__ void few_turn(const FewArgs<T>& a, int64_t d0, T* xt) {
    __shared__ T tile[FEW][66];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (int n = w; n < (int)a.ldrt; n += 4)
        tile[n][lane] = n < a.x.rows && d0 + lane < a.features && a.y[n] >= 0 ? a.x.p[n * a.x.ld + d0 + lane] : (T)0;
    __syncthreads();
    for (int k = w; k < 64; k += 4)
        if (lane < a.ldrt && d0 + k < a.features) xt[(d0 + k) * a.ldrt + lane] = tile[lane][k];
}
// One workgroup a row: its sum and lp. The workgroups behind the last row turn x over
template <typename T> __global__ __launch_bounds__(256) void class_few_join(FewArgs<T> a, T* xt) {
    typedef acc_t<T> A;
    __shared__ A red[2][4];
    if (blockIdx.x >= a.x.rows) {
        few_turn(a, (blockIdx.x - a.x.rows) * 64, xt);
        return;
    }
    const int64_t n = blockIdx.x, y = a.y[n], V = a.beta.rows;
    const bool known = y >= 0 && y < V;
    A mx = neg_inf<A>(), s = 0;
    const A eta = known ? a.eta_y[n] : (A)0;
    for (int64_t i = threadIdx.x; i < a.tiles; i += 256) join(mx, s, a.part_max[n * a.tiles + i], a.part_sum[n * a.tiles + i]);
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) join(mx, s, __shfl_xor(mx, m, 64), __shfl_xor(s, m, 64));
    if ((threadIdx.x & 63) == 0) {
        red[0][threadIdx.x >> 6] = mx;
        red[1][threadIdx.x >> 6] = s;
    }
    __syncthreads();
    if (a.largest && n == 0) // (rows behind the last)
        for (int64_t i = a.x.rows + threadIdx.x; i < FEW; i += 256) a.largest[i] = 0;
    if (threadIdx.x) return;
    for (int w = 1; w < 4; ++w) join(mx, s, red[0][w], red[1][w]);
    a.lp[n] = row_lp(y, V, mx, s, eta);
    if (a.of) a.of[n] = row_sum_of(y, V, mx, s);
    if (a.largest) a.largest[n] = y < 0 || !a.lpbar ? (A)0 : fabs(a.lpbar[n]);
}

// r of 64 classes: a wave takes a quarter of the rows, a lane a class -- rt's entries side by side, r's column, alphabar
template <typename T> __global__ __launch_bounds__(256) void class_few_r(FewArgs<T> a, Largest<acc_t<T>> largest_of) {
    typedef acc_t<T> A;
    constexpr int N = Vec16<T>::N;
    __shared__ A top[FEW], share_of[FEW], w[FEW], sum[4][64];
    __shared__ int64_t y[FEW];
    const A largest = largest_of.get();
    constexpr A up = stored_scale<T>();
    const int64_t V = a.beta.rows;
    const int rows = (int)a.x.rows, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (threadIdx.x < FEW) {
        const int n = threadIdx.x;
        const int64_t yn = n < rows ? a.y[n] : -1;
        const RowSum<A> of = yn >= 0 ? a.of[n] : RowSum<A>{(A)__builtin_inf(), (A)0};
        const bool none = of.share == 0;
        y[n] = none ? -1 : yn;
        top[n] = of.top;
        share_of[n] = up * of.share;
        w[n] = none ? (A)0 : a.lpbar ? a.lpbar[n] / largest : (A)1;
    }
    __syncthreads();
    const int64_t v = (int64_t)blockIdx.x * 64 + lane; // (below ldv, a multiple of 64)
    A total = 0;
    const int share = (int)a.ldrt / 4;
    for (int n0 = wave * share; n0 < (wave + 1) * share; n0 += N) {
        typename Vec16<T>::V u;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const int n = n0 + e;
            A g = 0;
            if (n < rows) {
                g = y[n] < 0 || v >= V ? (A)0 : (y[n] == a.v0 + v ? up : (A)0) - share_of[n] * exp_log2e(a.eta[n * a.ldv + v] - top[n]);
                a.r[n * a.ldv + v] = (T)g;
                g *= w[n];
            }
            total += g;
            u[e] = (T)g;
        }
        if (v < V) *reinterpret_cast<typename Vec16<T>::V*>(a.rt + v * a.ldrt + n0) = u;
    }
    if (!a.alphabar) return;
    sum[wave][lane] = total;
    __syncthreads();
    if (wave == 0 && v < V) a.alphabar[v] = (T)(((sum[0][lane] + sum[1][lane]) + (sum[2][lane] + sum[3][lane])) * (largest / up));
}

// Fragment j (feature 16-byte chunk's element j) of eight classes' chunks
template <typename T> struct Turn;
template <> struct Turn<float> {
    static __device__ __forceinline__ void mul(const Vec16<float>::V (&b)[8], int j, const float (&r)[8], Mma<float>::C& c) {
#pragma unroll
        for (int u = 0; u < 8; ++u) c = Mma<float>::mul1(b[u][j], r[u], c);
    }
};
template <> struct Turn<double> {
    static __device__ __forceinline__ void mul(const Vec16<double>::V (&b)[8], int j, const double (&r)[8], Mma<double>::C& c) {
#pragma unroll
        for (int u = 0; u < 8; ++u) c = Mma<double>::mul1(b[u][j], r[u], c);
    }
};
template <typename T> struct Turn { // 16 bits
    static __device__ __forceinline__ void mul(const typename Vec16<T>::V (&b)[8], int j, const T (&r)[8], typename Mma<T>::C& c) {
        typename Vec16<T>::V f, g;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            f[u] = b[u][j];
            g[u] = r[u];
        }
        c = Mma<T>::mul(f, g, c);
    }
};

// an entry of xbar from its sum: times the row's cotangent
template <typename T> __device__ __forceinline__ T few_cotangent(const FewArgs<T>& a, int64_t n, acc_t<T> s) {
    return (T)(a.y[n] < 0 ? (acc_t<T>)0 : s * ((a.lpbar ? a.lpbar[n] : (acc_t<T>)1) / (acc_t<T>)stored_scale<T>()));
}

// xbar's sums over a share of the classes for 16 chunks of features: four waves with a quarter of the share each
template <typename T, int NT, bool HALF> __device__ __forceinline__ void few_xbar(const FewArgs<T>& a, int64_t slab, int64_t split) {
    typedef acc_t<T> A;
    typedef typename Vec16<T>::V Vec;
    typedef typename Mma<T>::C C;
    constexpr int N = Vec16<T>::N;
    __shared__ A sum[4][16][16 * N + 1];
    const int lane = threadIdx.x & 63, q = lane >> 4, wave = threadIdx.x >> 6;
    // a chunk that lies behind the last whole one is taken as the last N features (some of which the one before has too): no guard
    // holds a load back (bf16 12 rows x 1958 x 34026 with the reverse mode 126 us against 157)
    const int64_t d0 = slab * 16 * N, D = a.features, V = a.beta.rows;
    const auto start = [=](int chunk) { return D < N || d0 + (chunk + 1) * N <= D ? d0 + chunk * N : D - N; };
    const int64_t d = start(lane & 15);
    const int64_t s0 = split * a.share, s1 = s0 + a.share < V ? s0 + a.share : V;
    C c[NT][N];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < N; ++j) c[t][j] = C{0, 0, 0, 0};
    // lane group q: classes v + 8 q .. + 7 (r is zero behind the last class, up to ldv, a multiple of 32)
    for (int64_t v = s0 + 32 * wave; v < s1; v += 128) {
        Vec b[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int64_t at = v + 8 * q + u, row = at < V ? at : V - 1;
            if (D < N) b[u] = tile_chunk(a.beta, row, d, D);
            else if constexpr (HALF) b[u] = load16_words(a.beta.p + row * a.beta.ld + d);
            else b[u] = load16(a.beta.p + row * a.beta.ld + d);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int64_t n = 16 * t + (lane & 15);
            T r[8];
#pragma unroll
            for (int k = 0; k < 8; k += N) {
                const Vec u = *reinterpret_cast<const Vec*>(a.r + (n < a.x.rows ? n : a.x.rows - 1) * a.ldv + v + 8 * q + k);
#pragma unroll
                for (int e = 0; e < N && k + e < 8; ++e) r[k + e] = u[e];
            }
#pragma unroll
            for (int j = 0; j < N; ++j) Turn<T>::mul(b, j, r, c[t][j]);
        }
    }
    // c[t][j] register r: row of x 16 t + (lane & 15), feature (row(q, r)) N + j
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) sum[wave][lane & 15][Mma<T>::row(q, r) * N + j] = c[t][j][r];
        __syncthreads();
        for (int id = threadIdx.x; id < 16 * 16 * N; id += 256) {
            const int n = id / (16 * N), k = id % (16 * N);
            const int64_t to = start(k / N) + k % N;
            if (16 * t + n >= a.x.rows || to < d0 + k / N * N || to >= D) continue; // (each feature by the chunk that it lies in)
            const A s = (sum[0][n][k] + sum[1][n][k]) + (sum[2][n][k] + sum[3][n][k]);
            if (a.xpart) {
                A* part = a.xpart + (split * a.x.rows + 16 * t + n) * D + to;
                *part = a.add ? *part + s : s;
            } else a.xbar[(16 * t + n) * D + to] = few_cotangent(a, 16 * t + n, s);
        }
        __syncthreads();
    }
}
// xbar <- the splits' sums times the rows' cotangents
template <typename T> __global__ __launch_bounds__(256) void class_few_xbar_join(FewArgs<T> a, int splits) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, count = a.x.rows * a.features;
    if (i >= count) return;
    acc_t<T> s = 0;
#pragma unroll 4
    for (int k = 0; k < splits; ++k) s += a.xpart[k * count + i];
    a.xbar[i] = few_cotangent(a, i / a.features, s);
}

// betabar[v][d] = sum_n rt[v][n] x[n][d] for a slab of features and a share of the classes: the slab's x stays in registers (xt, its
// transpose: [features][ldrt]), 16 classes at a time pass by. NG: steps of k, ldrt = NG * 4 chunks. As in WideTile the features of a
// fragment's rows are chosen so that a lane's results lie side by side (16 bytes of them, four lanes 64).
template <typename T> struct Slab {
    static constexpr int FRAGS = 64 / (4 * (int)sizeof(T)) < 2 ? 2 : 64 / (4 * (int)sizeof(T)), WIDTH = 16 * FRAGS;
    static constexpr int RUN = sizeof(T) == 2 ? 8 : 4; // results side by side
    static __device__ __forceinline__ int feature(int j, int row) {
        if (sizeof(T) == 2) return 32 * (j >> 1) + 8 * (row >> 2) + 4 * (j & 1) + (row & 3);
        if (sizeof(T) == 4) return 16 * j + row;
        return 16 * j + 4 * (row & 3) + (row >> 2);
    }
};
template <typename T, int NG> __device__ __forceinline__ void few_beta(const FewArgs<T>& a, const T* xt, T* betabar, Largest<acc_t<T>> largest,
                                                                     int64_t slab, int64_t share, int64_t shares) {
    typedef acc_t<T> A;
    typedef typename Vec16<T>::V Vec;
    typedef typename Mma<T>::C C;
    typedef Slab<T> S;
    constexpr int N = Vec16<T>::N, AHEAD = NG <= 2 ? 4 : 2;
    const int lane = threadIdx.x & 63, q = lane >> 4, wave = threadIdx.x >> 6;
    const int64_t d0 = slab * S::WIDTH, D = a.features, V = a.beta.rows, ldrt = a.ldrt;
    const A back = largest.get() / (A)stored_scale<T>();
    Vec x[S::FRAGS][NG];
#pragma unroll
    for (int j = 0; j < S::FRAGS; ++j) {
        const int64_t d = d0 + S::feature(j, lane & 15);
#pragma unroll
        for (int g = 0; g < NG; ++g) x[j][g] = d < D ? *reinterpret_cast<const Vec*>(xt + d * ldrt + (4 * g + q) * N) : Vec{};
    }
    const bool full = d0 + S::WIDTH <= D;
    const int64_t step = shares * 4 * 16 * AHEAD;
    for (int64_t v0 = (share * 4 + wave) * 16 * AHEAD; v0 < V; v0 += step) {
        Vec b[AHEAD][NG];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int64_t v = v0 + 16 * u + (lane & 15), at = v < V ? v : V - 1;
#pragma unroll
            for (int g = 0; g < NG; ++g) b[u][g] = *reinterpret_cast<const Vec*>(a.rt + at * ldrt + (4 * g + q) * N);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int64_t v = v0 + 16 * u + (lane & 15);
            A out[S::FRAGS * 4];
#pragma unroll
            for (int j = 0; j < S::FRAGS; ++j) {
                C c = {0, 0, 0, 0};
#pragma unroll
                for (int g = 0; g < NG; ++g) c = Mma<T>::mul(x[j][g], b[u][g], c);
#pragma unroll
                for (int r = 0; r < 4; ++r) out[4 * j + r] = c[r] * back;
            }
            if (v >= V) continue;
#pragma unroll
            for (int i = 0; i < S::FRAGS * 4 / S::RUN; ++i) {
                const int64_t d = d0 + i * 4 * S::RUN + q * S::RUN;
                T* to = betabar + v * D + d;
#pragma unroll
                for (int k = 0; k < S::RUN; k += N) {
                    if (full) {
                        Vec w;
#pragma unroll
                        for (int e = 0; e < N; ++e) w[e] = (T)out[i * S::RUN + k + e];
                        store16(to + k, w);
                    } else {
#pragma unroll
                        for (int e = 0; e < N; ++e)
                            if (d + k + e < D) to[k + e] = (T)out[i * S::RUN + k + e];
                    }
                }
            }
        }
    }
}

// xbar's sums by the first xslabs x splits workgroups, betabar by the others
template <typename T, int NT, int NG, bool HALF> __global__ __launch_bounds__(256) void class_few_back(FewArgs<T> a, const T* xt, T* betabar,
                                                                                           Largest<acc_t<T>> largest, int xslabs, int splits,
                                                                                           int bslabs, int shares) {
    const int id = blockIdx.x;
    if (id < xslabs * splits) few_xbar<T, NT, HALF>(a, id % xslabs, id / xslabs);
    else few_beta<T, NG>(a, xt, betabar, largest, (id - xslabs * splits) % bslabs, (id - xslabs * splits) / bslabs, shares);
}

} // namespace gptt
