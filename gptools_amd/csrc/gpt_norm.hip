// Layer norm and its reverse mode (gpt_layer_norm, gpt_layer_norm_vjp): rows of n values, standardised one by one.
//
//   mean = sum x / n, var = sum (x - mean)^2 / n, rstd = 1 / sqrt(var + eps), h = (x - mean) rstd, y = h w + b
//   g = ybar w, xbar = rstd (g - <g> - h <g h>), wbar = sum_rows ybar h, bbar = sum_rows ybar
//
// Both are bound by HBM: forward reads x and writes y, reverse reads x and ybar and writes xbar. A row of up to ROW_BYTES
// stays in the registers of the threads that read it (norm_row, norm_row_vjp): every value is read once, and the variance is
// a sum of squares about the mean, not a difference of two sums. A longer row (a whole lattice) is cut into pieces that
// many workgroups take (norm_long_*): statistics of the pieces, then a second sweep.
#include "gpt_readout.h"
#include "gpt_types.h"

using namespace gptt;

namespace {

// ---- rows that fit the registers of one workgroup ---------------------------------------------------------------------
// THREADS consecutive threads take a row, ITER 16-byte vectors each, THREADS apart. load() only issues loads, whole vectors without a
// branch, so that none waits for another: those behind the row's end read its last N values, and so does the one that the end cuts.
// settle() puts them right when they have come: the cut one moved to its place, zeros behind the end. (8191 rows of 1001 fp32 values,
// reverse mode: 19 us against 22 with a branch at every vector.) Where every value is taken by itself, nothing need move: mine()
// says which values of a vector are the row's and no other vector's. FULL: n is THREADS * ITER * N.
template <typename T, int THREADS, int ITER> struct RowRaw {
    static constexpr int N = Vec16<T>::N;
    typename Vec16<T>::V v[ITER];
    template <bool FULL = false> __device__ __forceinline__ void load(const T* p, int64_t n, int t) {
        if (!FULL && n < N) {
#pragma unroll
            for (int i = 0; i < ITER; ++i)
#pragma unroll
                for (int e = 0; e < N; ++e) v[i][e] = e < n ? p[e] : (T)0;
            return;
        }
        const int last = (int)n - N;
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int k = (i * THREADS + t) * N;
            v[i] = load16(p + (FULL || k < last ? k : last));
        }
    }
    template <bool FULL = false> __device__ __forceinline__ void settle(int64_t n, int t) {
        if (FULL) return;
        const int whole = (int)n / N, rest = (int)n % N, by = rest && n > N ? (N - rest) * (int)sizeof(T) : 0; // bytes
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int at = i * THREADS + t;
            uint4 u = __builtin_bit_cast(uint4, v[i]);
            if (by) { // (the same for all threads)
                uint4 s = u;
                if (by & 8) s = make_uint4(s.z, s.w, 0, 0);
                if (by & 4) s = make_uint4(s.y, s.z, s.w, 0);
                if (by & 2)
                    s = make_uint4(__builtin_amdgcn_alignbyte(s.y, s.x, 2), __builtin_amdgcn_alignbyte(s.z, s.y, 2),
                                   __builtin_amdgcn_alignbyte(s.w, s.z, 2), s.w >> 16);
                const bool cut = at == whole;
                u = make_uint4(cut ? s.x : u.x, cut ? s.y : u.y, cut ? s.z : u.z, cut ? s.w : u.w);
            }
            const bool in = at < whole + (rest > 0);
            u = make_uint4(in ? u.x : 0, in ? u.y : 0, in ? u.z : 0, in ? u.w : 0);
            v[i] = __builtin_bit_cast(typename Vec16<T>::V, u);
        }
    }
    static __device__ __forceinline__ bool mine(int j, int64_t n, int t) {
        const int whole = (int)n / N, rest = (int)n % N, at = j / N * THREADS + t, e = j % N;
        return at < whole || (at == whole && (n < N ? e < rest : e >= N - rest));
    }
    __device__ __forceinline__ acc_t<T> at(int j) const { return (acc_t<T>)v[j / N][j % N]; }
};
template <typename T, int THREADS, int ITER> struct RowRegs {
    static constexpr int N = Vec16<T>::N;
    acc_t<T> v[ITER * N];
    template <bool FULL = false> __device__ __forceinline__ void load(const T* p, int64_t n, int t) {
        RowRaw<T, THREADS, ITER> u;
        u.template load<FULL>(p, n, t);
        u.template settle<FULL>(n, t);
#pragma unroll
        for (int j = 0; j < ITER * N; ++j) v[j] = u.at(j);
    }
    __device__ __forceinline__ void store(T* p, int64_t n, int t) const {
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int64_t k = (int64_t)(i * THREADS + t) * N;
            if (k + N <= n) {
                typename Vec16<T>::V u;
#pragma unroll
                for (int e = 0; e < N; ++e) u[e] = (T)v[i * N + e];
                store16(p + k, u);
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (k + e < n) p[k + e] = (T)v[i * N + e];
            }
        }
    }
    // in the first n values of the row? (index of register j)
    static __device__ __forceinline__ bool inside(int j, int64_t n, int t) {
        return (int64_t)((j / N) * THREADS + t) * N + j % N < n;
    }
};

template <typename T, int THREADS, int ITER>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void norm_row(NormArgs a) {
    typedef acc_t<T> A;
    constexpr int BLOCK = THREADS < 256 ? 256 : THREADS, K = ITER * Vec16<T>::N;
    __shared__ A red[THREADS / 64];
    const int t = threadIdx.x % THREADS;
    const int64_t row = wide_block() * (BLOCK / THREADS) + threadIdx.x / THREADS;
    if (row >= a.rows) return; // (whole waves; a workgroup with barriers has one row)
    const int64_t n = a.width;
    typedef RowRaw<T, THREADS, ITER> Raw;
    constexpr int N = Vec16<T>::N;
    Raw u;
    u.load((const T*)a.x + row * n, n, t);
    A x[K], s[1] = {0};
#pragma unroll
    for (int j = 0; j < K; ++j) {
        x[j] = u.at(j);
        if (Raw::mine(j, n, t)) s[0] += x[j];
    }
    row_sum<THREADS>(s, red, false);
    const A mean = s[0] / (A)n;
    s[0] = 0;
#pragma unroll
    for (int j = 0; j < K; ++j) {
        x[j] -= mean;
        if (Raw::mine(j, n, t)) s[0] += x[j] * x[j];
    }
    row_sum<THREADS>(s, red, true);
    const A rstd = (A)1 / sqrt(s[0] / (A)n + (A)a.eps);
    if (t == 0) {
        ((A*)a.mean)[row] = mean;
        ((A*)a.rstd)[row] = rstd;
    }
#pragma unroll
    for (int j = 0; j < K; ++j) x[j] *= rstd;
    if (a.weight) {
        u.load((const T*)a.weight, n, t);
#pragma unroll
        for (int j = 0; j < K; ++j) x[j] *= u.at(j);
    }
    if (a.bias) {
        u.load((const T*)a.bias, n, t);
#pragma unroll
        for (int j = 0; j < K; ++j) x[j] += u.at(j);
    }
    T* y = (T*)a.y + row * n;
    if (n < N) {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (Raw::mine(e, n, t)) y[e] = (T)x[e];
        return;
    }
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int k = (i * THREADS + t) * N, last = (int)n - N;
        typename Vec16<T>::V v;
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = (T)x[i * N + e];
        if (k < n) store16(y + (k < last ? k : last), v); // (values that two vectors hold are the same in both)
    }
}

// Rows go round the workgroups' groups of THREADS threads; the next row's vectors are on their way while this one is
// reduced. The sums for the parameters' gradients stay in registers, and go to partial[2][gridDim.x][n] at the end
// (norm_param_sum adds them up in a fixed order).
// A workgroup alone (few rows) writes the results themselves.
// COLUMNS: little data. The first column_blocks workgroups sum the columns of x and ybar by themselves (column_sums), which
// takes no launch after this one: fp64 64 rows of 2100 values 13.5 us against 18.
enum { NO_PARAMS, PARTS, COLUMNS };
constexpr int SLICES = 16; // of the rows, in column_sums
template <typename T, int BLOCK> __device__ __forceinline__ void column_sums(const NormArgs& a, int64_t block) {
    typedef acc_t<T> A;
    constexpr int COLS = BLOCK / SLICES;
    __shared__ A red[2][SLICES][COLS];
    const int c = threadIdx.x % COLS, w = threadIdx.x / COLS;
    const int64_t k = block * COLS + c, n = a.width;
    A wbar = 0, bbar = 0;
    if (k < n) {
#pragma unroll 4
        for (int64_t row = w; row < a.rows; row += SLICES) {
            const A g = (A)((const T*)a.ybar)[row * n + k];
            wbar += g * (((A)((const T*)a.x)[row * n + k] - ((const A*)a.mean)[row]) * ((const A*)a.rstd)[row]);
            bbar += g;
        }
    }
    red[0][w][c] = wbar;
    red[1][w][c] = bbar;
    __syncthreads();
    if (w > 1 || k >= n) return;
    A s = red[w][0][c];
#pragma unroll
    for (int i = 1; i < SLICES; ++i) s += red[w][i][c];
    ((T*)(w ? a.bbar : a.wbar))[k] = (T)s;
}
template <typename T, int THREADS, int ITER, int HOW, int GROUPS>
__global__ __launch_bounds__(THREADS * GROUPS) void norm_row_vjp(NormArgs a) {
    constexpr bool PARAMS = HOW == PARTS;
    if constexpr (HOW == COLUMNS) {
        if (blockIdx.x < a.column_blocks) {
            column_sums<T, THREADS * GROUPS>(a, blockIdx.x);
            return;
        }
    }
    typedef acc_t<T> A;
    constexpr int N = Vec16<T>::N, K = ITER * N;
    __shared__ A red[2][THREADS / 64 * 2];
    __shared__ A joined[PARAMS && GROUPS > 1 ? GROUPS - 1 : 1][PARAMS && GROUPS > 1 ? 2 * K * THREADS : 1];
    const int t = threadIdx.x % THREADS, group = threadIdx.x / THREADS;
    const int64_t n = a.width, first = HOW == COLUMNS ? a.column_blocks : 0, step = (gridDim.x - first) * GROUPS;
    A wbar[PARAMS ? K : 1], bbar[PARAMS ? K : 1];
    if (PARAMS) {
#pragma unroll
        for (int j = 0; j < K; ++j) wbar[j] = bbar[j] = 0;
    }
    RowRaw<T, THREADS, ITER> w, xn, gn;
    if (a.weight) {
        w.load((const T*)a.weight, n, t);
        w.settle(n, t);
    }
    int64_t row = (blockIdx.x - first) * GROUPS + group;
    A mean = 0, rstd = 0;
    auto fetch = [&](int64_t r) {
        xn.load((const T*)a.x + r * n, n, t);
        gn.load((const T*)a.ybar + r * n, n, t);
        mean = ((const A*)a.mean)[r], rstd = ((const A*)a.rstd)[r];
    };
    constexpr bool AHEAD = sizeof(T) > 2 || ITER < 4; // (else the registers do not suffice)
    if (AHEAD && row < a.rows) fetch(row);
    int side = 0;
    for (; row < a.rows; row += step) { // (a group of several waves is the whole workgroup: its barriers are met by all)
        RowRegs<T, THREADS, ITER> x, g;
        if (!AHEAD) fetch(row);
        const A mu = mean, rs = rstd;
        A s[2] = {0, 0};
        xn.settle(n, t);
        gn.settle(n, t);
#pragma unroll
        for (int j = 0; j < K; ++j) {
            x.v[j] = (xn.at(j) - mu) * rs;
            g.v[j] = gn.at(j);
        }
        if (AHEAD && row + step < a.rows) fetch(row + step);
#pragma unroll
        for (int j = 0; j < K; ++j) {
            if (PARAMS) {
                wbar[j] += g.v[j] * x.v[j];
                bbar[j] += g.v[j];
            }
            if (a.weight) g.v[j] *= w.at(j);
            s[0] += g.v[j]; // (zero behind the row's end: g is)
            s[1] += g.v[j] * x.v[j];
        }
        row_sum<THREADS>(s, red[side], true); // (the other half is next: one barrier a row)
        side ^= 1;
        const A c0 = s[0] / (A)n, c1 = s[1] / (A)n;
#pragma unroll
        for (int j = 0; j < K; ++j) x.v[j] = rs * (g.v[j] - c0 - x.v[j] * c1);
        x.store((T*)a.xbar + row * n, n, t);
    }
    if (PARAMS) {
        if (GROUPS > 1) {
            if (group) {
#pragma unroll
                for (int j = 0; j < K; ++j) {
                    joined[group - 1][j * THREADS + t] = wbar[j];
                    joined[group - 1][(K + j) * THREADS + t] = bbar[j];
                }
            }
            __syncthreads();
            if (group) return;
#pragma unroll
            for (int k = 0; k < GROUPS - 1; ++k)
#pragma unroll
                for (int j = 0; j < K; ++j) {
                    wbar[j] += joined[k][j * THREADS + t];
                    bbar[j] += joined[k][(K + j) * THREADS + t];
                }
        }
        if (gridDim.x == 1) {
            RowRegs<T, THREADS, ITER> u;
#pragma unroll
            for (int j = 0; j < K; ++j) u.v[j] = wbar[j];
            u.store((T*)a.wbar, n, t);
#pragma unroll
            for (int j = 0; j < K; ++j) u.v[j] = bbar[j];
            u.store((T*)a.bbar, n, t);
            return;
        }
        A* p = (A*)a.partial + (int64_t)blockIdx.x * n;
        const int64_t other = (int64_t)gridDim.x * n;
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            const int64_t k = (int64_t)(i * THREADS + t) * N;
            if (k + N <= n) {
#pragma unroll
                for (int e = 0; e < N; e += Vec16<A>::N) {
                    typename Vec16<A>::V u, v;
#pragma unroll
                    for (int f = 0; f < Vec16<A>::N; ++f) {
                        u[f] = wbar[i * N + e + f];
                        v[f] = bbar[i * N + e + f];
                    }
                    store16(p + k + e, u);
                    store16(p + other + k + e, v);
                }
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (k + e < n) {
                        p[k + e] = wbar[i * N + e];
                        p[other + k + e] = bbar[i * N + e];
                    }
            }
        }
    }
}

// wbar, bbar <- the sums over the `parts` rows of partial[2][parts][n]: COLS columns a workgroup, whose threads share the parts
template <typename T, int COLS> __global__ __launch_bounds__(1024) void norm_param_sum(const acc_t<T>* partial, int64_t parts, int64_t n,
                                                                                      T* wbar, T* bbar) {
    typedef acc_t<T> A;
    constexpr int SLICES = 1024 / COLS;
    __shared__ A red[SLICES][COLS];
    const int c = threadIdx.x % COLS, w = threadIdx.x / COLS;
    const int64_t k = (int64_t)blockIdx.x * COLS + c;
    const A* p = partial + (int64_t)blockIdx.y * parts * n + k;
    A s[4] = {0, 0, 0, 0};
    if (k < n) {
        int64_t i = w;
        for (; i + 7 * SLICES < parts; i += 8 * SLICES) {
            A v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = p[(i + u * SLICES) * n];
#pragma unroll
            for (int u = 0; u < 8; ++u) s[u & 3] += v[u];
        }
        for (; i < parts; i += SLICES) s[0] += p[i * n];
    }
    red[w][c] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (w || k >= n) return;
    A t = red[0][c];
#pragma unroll
    for (int i = 1; i < SLICES; ++i) t += red[i][c];
    (blockIdx.y ? bbar : wbar)[k] = (T)t;
}

// ---- rows cut into pieces ---------------------------------------------------------------------------------------------
constexpr int LONG_THREADS = 256;
constexpr int LONG_ITER = 8; // a sweep of a workgroup: 256 threads x 8 vectors = 32 KB, in registers
template <typename T> constexpr int64_t long_sweep() { return (int64_t)LONG_THREADS * LONG_ITER * Vec16<T>::N; }
constexpr int LONGB_ITER = 4; // 16 KB where more than x is held
template <typename T> constexpr int64_t longb_sweep() { return (int64_t)LONG_THREADS * LONGB_ITER * Vec16<T>::N; }

// Statistics of piece blockIdx.x of row blockIdx.y: partial[row][piece] = (c, sum (x - c), sum (x - c)^2) with c the mean of
// the piece's first values, as rounded. Sums about a value near the piece's mean keep what a level far from zero would take
// from them, and they join without the error of a rounded piece's mean: about any other m,
// sum (x - m)^2 = sum (x - c)^2 + 2 (c - m) sum (x - c) + n (c - m)^2.
template <typename T> __global__ __launch_bounds__(LONG_THREADS) void norm_long_stats(NormArgs a) {
    typedef acc_t<T> A;
    constexpr int N = Vec16<T>::N, K = LONG_ITER * N;
    __shared__ A red[LONG_THREADS / 64 * 2];
    const int t = threadIdx.x;
    const T* x = (const T*)a.x + (int64_t)blockIdx.y * a.width;
    const int64_t k0 = (int64_t)blockIdx.x * a.piece, k1 = k0 + a.piece < a.width ? k0 + a.piece : a.width;
    // each wave sums the first 64 vectors (or what there is of them) for itself
    const int64_t lead = k1 - k0 < 64 * N ? k1 - k0 : 64 * N;
    RowRegs<T, 64, 1> r0;
    r0.load(x + k0, lead, t & 63);
    A c = 0, s[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < N; ++j) c += r0.v[j];
    c = wave_sum(c) / (A)lead;
    int64_t k = k0;
    for (; k + long_sweep<T>() <= k1; k += long_sweep<T>()) {
        RowRegs<T, LONG_THREADS, LONG_ITER> r;
        r.template load<true>(x + k, long_sweep<T>(), t);
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const A d = r.v[j] - c;
            s[0] += d;
            s[1] += d * d;
        }
    }
    if (k < k1) {
        RowRegs<T, LONG_THREADS, LONG_ITER> r;
        r.load(x + k, k1 - k, t);
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const A d = RowRegs<T, LONG_THREADS, LONG_ITER>::inside(j, k1 - k, t) ? r.v[j] - c : (A)0;
            s[0] += d;
            s[1] += d * d;
        }
    }
    row_sum<LONG_THREADS>(s, red, true);
    if (t == 0) {
        A* p = (A*)a.partial + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 3;
        p[0] = c;
        p[1] = s[0];
        p[2] = s[1];
    }
}

// mean and rstd of a row from its pieces', for a whole workgroup
template <typename T> __device__ __forceinline__ void long_moments(const NormArgs& a, int64_t row, int pieces, acc_t<T>& mean, acc_t<T>& rstd) {
    typedef acc_t<T> A;
    __shared__ A red[2][LONG_THREADS / 64]; // (in turn: one barrier a sum, also from row to row)
    const int t = threadIdx.x;
    const A* p = (const A*)a.partial + row * pieces * 3;
    const A whole = (A)a.piece, tail = (A)(a.width - (int64_t)(pieces - 1) * a.piece); // values of a piece, of the last
    A s[1] = {0};
    for (int i = t; i < pieces; i += LONG_THREADS) s[0] += (i + 1 < pieces ? whole : tail) * p[3 * i] + p[3 * i + 1];
    row_sum<LONG_THREADS>(s, red[0], true);
    mean = s[0] / (A)a.width;
    s[0] = 0;
    for (int i = t; i < pieces; i += LONG_THREADS) {
        const A d = p[3 * i] - mean;
        s[0] += p[3 * i + 2] + d * ((A)2 * p[3 * i + 1] + (i + 1 < pieces ? whole : tail) * d);
    }
    row_sum<LONG_THREADS>(s, red[1], true);
    rstd = (A)1 / sqrt(s[0] / (A)a.width + (A)a.eps);
}
// ... one workgroup a row
template <typename T> __global__ __launch_bounds__(LONG_THREADS) void norm_long_join(NormArgs a, int pieces) {
    acc_t<T> mean, rstd;
    long_moments<T>(a, blockIdx.x, pieces, mean, rstd);
    if (threadIdx.x == 0) {
        ((acc_t<T>*)a.mean)[blockIdx.x] = mean;
        ((acc_t<T>*)a.rstd)[blockIdx.x] = rstd;
    }
}

// The second sweep, 16 KB of a row at a time. join > 0: the row's moments from that many pieces, by each workgroup for itself.
// Bound by HBM: 16 lattices of 4096 x 4096 in fp64 765 us, 5.6 TB/s, after 380 us for their statistics. (Taking the rows one
// lattice at a time, so that it finds them in the last-level cache, costs more in short launches than it saves: 1350 us
// against 1170 for both sweeps.)
template <typename T, bool FULL> __device__ __forceinline__ void long_apply(NormArgs a, int join) {
    typedef acc_t<T> A;
    constexpr int K = LONGB_ITER * Vec16<T>::N;
    const int t = threadIdx.x;
    const int64_t k = (int64_t)blockIdx.x * longb_sweep<T>();
    const int64_t n = a.width - k < longb_sweep<T>() ? a.width - k : longb_sweep<T>();
    RowRaw<T, LONG_THREADS, LONGB_ITER> w, b;
    if (a.weight) w.template load<FULL>((const T*)a.weight + k, n, t);
    if (a.bias) b.template load<FULL>((const T*)a.bias + k, n, t);
    if (a.weight) w.template settle<FULL>(n, t);
    if (a.bias) b.template settle<FULL>(n, t);
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        RowRegs<T, LONG_THREADS, LONGB_ITER> r;
        r.template load<FULL>((const T*)a.x + row * a.width + k, n, t);
        A mean, rstd;
        if (join) {
            long_moments<T>(a, row, join, mean, rstd);
            if (t == 0 && blockIdx.x == 0) {
                ((A*)a.mean)[row] = mean;
                ((A*)a.rstd)[row] = rstd;
            }
        } else mean = ((const A*)a.mean)[row], rstd = ((const A*)a.rstd)[row];
#pragma unroll
        for (int j = 0; j < K; ++j) {
            r.v[j] = (r.v[j] - mean) * rstd;
            if (a.weight) r.v[j] *= w.at(j);
            if (a.bias) r.v[j] += b.at(j);
        }
        r.store((T*)a.y + row * a.width + k, n, t);
    }
}
template <typename T> __global__ __launch_bounds__(LONG_THREADS) void norm_long_apply(NormArgs a, int join) {
    if (((int64_t)blockIdx.x + 1) * longb_sweep<T>() <= a.width) long_apply<T, true>(a, join);
    else long_apply<T, false>(a, join);
}

// Reverse mode, first sweep: columns [blockIdx.x * sweep, + sweep) of the rows of group blockIdx.y: the columns' gradient
// sums over these rows (partial2[2][groups][n], or the outputs themselves where there is one group) and this piece's part of
// the rows' two sums, partial[row][piece] = (sum g, sum g h).
template <typename T, bool FULL> __device__ __forceinline__ void long_vjp_sums(NormArgs a) {
    typedef acc_t<T> A;
    constexpr int K = LONGB_ITER * Vec16<T>::N;
    __shared__ A red[2][LONG_THREADS / 64 * 2];
    const int t = threadIdx.x;
    const int64_t k0 = (int64_t)blockIdx.x * longb_sweep<T>();
    const int64_t n = a.width - k0 < longb_sweep<T>() ? a.width - k0 : longb_sweep<T>();
    RowRaw<T, LONG_THREADS, LONGB_ITER> w, xn, gn;
    if (a.weight) {
        w.template load<FULL>((const T*)a.weight + k0, n, t);
        w.template settle<FULL>(n, t);
    }
    A wbar[K], bbar[K], mean = 0, rstd = 0;
#pragma unroll
    for (int j = 0; j < K; ++j) wbar[j] = bbar[j] = 0;
    auto fetch = [&](int64_t row) {
        xn.template load<FULL>((const T*)a.x + row * a.width + k0, n, t);
        gn.template load<FULL>((const T*)a.ybar + row * a.width + k0, n, t);
        mean = ((const A*)a.mean)[row], rstd = ((const A*)a.rstd)[row];
    };
    if (blockIdx.y < a.rows) fetch(blockIdx.y);
    int side = 0;
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        A h[K], g[K], s[2] = {0, 0};
        xn.template settle<FULL>(n, t);
        gn.template settle<FULL>(n, t);
#pragma unroll
        for (int j = 0; j < K; ++j) {
            h[j] = (xn.at(j) - mean) * rstd;
            g[j] = gn.at(j);
        }
        if (row + gridDim.y < a.rows) fetch(row + gridDim.y);
#pragma unroll
        for (int j = 0; j < K; ++j) {
            wbar[j] += g[j] * h[j];
            bbar[j] += g[j];
            const A gw = a.weight ? g[j] * w.at(j) : g[j];
            s[0] += gw;
            s[1] += gw * h[j];
        }
        row_sum<LONG_THREADS>(s, red[side], true); // (the other half is next: one barrier a row)
        side ^= 1;
        if (t == 0) {
            A* p = (A*)a.partial + (row * gridDim.x + blockIdx.x) * 2;
            p[0] = s[0];
            p[1] = s[1];
        }
    }
    if (!a.wbar) return;
    const bool direct = gridDim.y == 1;
    A* q = (A*)a.partial2 + (int64_t)blockIdx.y * a.width + k0;
    const int64_t other = (int64_t)gridDim.y * a.width;
#pragma unroll
    for (int j = 0; j < K; ++j) {
        const int64_t k = (int64_t)((j / Vec16<T>::N) * LONG_THREADS + t) * Vec16<T>::N + j % Vec16<T>::N;
        if (k >= n) continue;
        if (direct) {
            ((T*)a.wbar)[k0 + k] = (T)wbar[j];
            ((T*)a.bbar)[k0 + k] = (T)bbar[j];
        } else {
            q[k] = wbar[j];
            q[k + other] = bbar[j];
        }
    }
}
template <typename T> __global__ __launch_bounds__(LONG_THREADS) void norm_long_vjp_sums(NormArgs a) {
    if (((int64_t)blockIdx.x + 1) * longb_sweep<T>() <= a.width) long_vjp_sums<T, true>(a);
    else long_vjp_sums<T, false>(a);
}

// (<g>, <g h>) of a row from its pieces', for a whole workgroup
template <typename T> __device__ __forceinline__ void long_means(const NormArgs& a, int64_t row, int64_t pieces, int side, acc_t<T> (&s)[2]) {
    typedef acc_t<T> A;
    __shared__ A red[2][LONG_THREADS / 64 * 2]; // (side: in turn from row to row)
    const A* p = (const A*)a.partial + row * pieces * 2;
    s[0] = s[1] = 0;
    for (int64_t i = threadIdx.x; i < pieces; i += LONG_THREADS) {
        s[0] += p[2 * i];
        s[1] += p[2 * i + 1];
    }
    row_sum<LONG_THREADS>(s, red[side], true);
    s[0] /= (A)a.width;
    s[1] /= (A)a.width;
}
// ... one workgroup a row, into sums
template <typename T> __global__ __launch_bounds__(LONG_THREADS) void norm_long_vjp_rows(NormArgs a, int64_t pieces) {
    acc_t<T> s[2];
    long_means<T>(a, blockIdx.x, pieces, 0, s);
    if (threadIdx.x == 0) {
        ((acc_t<T>*)a.sums)[2 * (int64_t)blockIdx.x] = s[0];
        ((acc_t<T>*)a.sums)[2 * (int64_t)blockIdx.x + 1] = s[1];
    }
}

// second sweep: xbar. join > 0: the row's means from that many pieces, by each workgroup for itself
template <typename T, bool FULL> __device__ __forceinline__ void long_vjp_apply(NormArgs a, int64_t join) {
    typedef acc_t<T> A;
    constexpr int K = LONGB_ITER * Vec16<T>::N;
    const int t = threadIdx.x;
    const int64_t k0 = (int64_t)blockIdx.x * longb_sweep<T>();
    const int64_t n = a.width - k0 < longb_sweep<T>() ? a.width - k0 : longb_sweep<T>();
    RowRaw<T, LONG_THREADS, LONGB_ITER> w;
    if (a.weight) {
        w.template load<FULL>((const T*)a.weight + k0, n, t);
        w.template settle<FULL>(n, t);
    }
    int side = 0;
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y, side ^= 1) {
        const A mean = ((const A*)a.mean)[row], rstd = ((const A*)a.rstd)[row];
        RowRegs<T, LONG_THREADS, LONGB_ITER> x, g;
        x.template load<FULL>((const T*)a.x + row * a.width + k0, n, t);
        g.template load<FULL>((const T*)a.ybar + row * a.width + k0, n, t);
        A c[2];
        if (join) long_means<T>(a, row, join, side, c);
        else c[0] = ((const A*)a.sums)[2 * row], c[1] = ((const A*)a.sums)[2 * row + 1];
#pragma unroll
        for (int j = 0; j < K; ++j) {
            if (a.weight) g.v[j] *= w.at(j);
            x.v[j] = rstd * (g.v[j] - c[0] - (x.v[j] - mean) * rstd * c[1]);
        }
        x.store((T*)a.xbar + row * a.width + k0, n, t);
    }
}
template <typename T> __global__ __launch_bounds__(LONG_THREADS) void norm_long_vjp_apply(NormArgs a, int64_t join) {
    if (((int64_t)blockIdx.x + 1) * longb_sweep<T>() <= a.width) long_vjp_apply<T, true>(a, join);
    else long_vjp_apply<T, false>(a, join);
}

// ---- plans ------------------------------------------------------------------------------------------------------------
constexpr int64_t ROW_BYTES = 65536;   // longest row that one workgroup keeps in registers (1024 threads x 4 vectors)
constexpr int64_t VJP_ROW_BYTES = 32768; // ... with its cotangent and its gradient sums (512 threads x 4 vectors)
constexpr int64_t COLUMN_BYTES = (int64_t)8 << 20;
constexpr int64_t MAX_GRID_Y = 65535;
// Pieces of a row that the second sweep's workgroups add up for themselves rather than in a launch before (four fp64 lattices of 1024 x
// 1024, 512 pieces each, reverse mode: 34 us against 37)
constexpr int64_t FEW_PIECES = 512;

struct LongPlan {
    int64_t piece, pieces;   // forward: elements of a piece (a multiple of the sweep), pieces of a row
    int64_t vpieces, groups; // reverse: pieces of a row, row groups
};
template <typename T> LongPlan long_plan(int64_t rows, int64_t n) {
    LongPlan p;
    const int64_t sweeps = (n + long_sweep<T>() - 1) / long_sweep<T>();
    // pieces of all rows enough to fill the card, and at most 2048 of one: its join stays short
    const int64_t fill = sweeps * rows / 4096, per = fill > (sweeps + 2047) / 2048 ? fill : (sweeps + 2047) / 2048;
    p.piece = per * long_sweep<T>();
    p.pieces = (n + p.piece - 1) / p.piece;
    p.vpieces = (n + longb_sweep<T>() - 1) / longb_sweep<T>();
    p.groups = 1;
    while (p.groups < rows && p.groups < 256 && p.vpieces * p.groups < 512) p.groups *= 2;
    if (p.groups > rows) p.groups = rows;
    return p;
}
template <typename T> bool small_row(int64_t n) { return n <= 128 * Vec16<T>::N; }
// Workgroups of the reverse mode on whole rows: one where the rows are few (its rounds are shorter than another launch), else
// enough to fill the card, and at least 8 rows each where there are as many (each leaves 2 n partial sums), at most those that stay on it at
// once: a CU holds one of 512 threads or more, three of 256 with sums of 16 values, four others (bf16, 16384 rows of 8192: 163 us
// against 180 with 1024). Short rows: a wave takes a row, a workgroup 4 at a time, or 16 if it is alone
template <typename T> int64_t row_blocks(int64_t rows, int64_t n) {
    const bool small = small_row<T>(n);
    if (rows <= (small ? 32 : 2)) return 1;
    const int64_t groups = small ? (rows + 3) / 4 : rows, vecs = (n + Vec16<T>::N - 1) / Vec16<T>::N;
    const int64_t most = vecs > 512 ? 256 : vecs > 256 && sizeof(T) == 2 ? 768 : 1024;
    if (groups < 256) return groups;
    return groups / 8 < 256 ? 256 : groups / 8 < most ? groups / 8 : most;
}

// Rows and values few enough for their columns to be summed apart (fp32 512 rows of 4000 14 us against 19, but 2000 of 2000 21 against 18)
template <typename T> bool columns(int64_t rows, int64_t n) { return rows <= 2048 && rows * n * (int64_t)sizeof(T) <= COLUMN_BYTES; }

// Row groups of a second sweep: a workgroup that has weights takes several rows with them, if enough workgroups are left to fill the
// card (32 lattices of 1024 x 1500 in fp64: 142 us against 214 with one row each). Not so in the reverse mode, with three streams
// for the one of weights: 64 lattices of 300 x 1500 128 us against 111
unsigned apply_groups(int64_t rows, int64_t pieces, bool weights) {
    int64_t g = weights ? (2048 + pieces - 1) / pieces : rows;
    if (g > rows) g = rows;
    return (unsigned)(g < MAX_GRID_Y ? g : MAX_GRID_Y);
}
template <typename T> size_t workspace(int64_t rows, int64_t n, bool vjp) {
    const size_t A = sizeof(acc_t<T>);
    if (n * (int64_t)sizeof(T) <= (vjp ? VJP_ROW_BYTES : ROW_BYTES)) {
        const int64_t blocks = vjp ? row_blocks<T>(rows, n) : 1;
        return blocks > 1 && !(vjp && columns<T>(rows, n)) ? A * 2 * (size_t)(blocks * n) : 0;
    }
    const LongPlan p = long_plan<T>(rows, n);
    if (!vjp) return A * 3 * (size_t)(rows * p.pieces);
    return A * (2 * (size_t)(rows * p.vpieces) + 2 * (size_t)rows + (p.groups > 1 ? 2 * (size_t)(p.groups * n) : 0));
}

template <typename T, int THREADS, int ITER> void launch_row(const NormArgs& a, hipStream_t st) {
    constexpr int BLOCK = THREADS < 256 ? 256 : THREADS, RPB = BLOCK / THREADS;
    norm_row<T, THREADS, ITER><<<wide_grid((a.rows + RPB - 1) / RPB), dim3(BLOCK), 0, st>>>(a);
}
template <typename T> hipError_t forward(NormArgs a, hipStream_t st) {
    const int64_t vecs = (a.width + Vec16<T>::N - 1) / Vec16<T>::N;
    if (a.width * (int64_t)sizeof(T) <= ROW_BYTES) {
        // a wave a row where that is at most two vectors a lane; then 256 threads, then 1024
        if (vecs <= 64) launch_row<T, 64, 1>(a, st);
        else if (vecs <= 128) launch_row<T, 64, 2>(a, st);
        else if (vecs <= 256) launch_row<T, 256, 1>(a, st);
        else if (vecs <= 512) launch_row<T, 256, 2>(a, st);
        else if (vecs <= 1024) launch_row<T, 512, 2>(a, st);
        else if (vecs <= 2048) launch_row<T, 512, 4>(a, st);
        else launch_row<T, 1024, 4>(a, st);
        return hipGetLastError();
    }
    const LongPlan p = long_plan<T>(a.rows, a.width);
    const size_t es = sizeof(T), as = sizeof(acc_t<T>);
    a.piece = p.piece;
    for (int64_t r0 = 0; r0 < a.rows; r0 += MAX_GRID_Y) {
        NormArgs s = a;
        s.rows = a.rows - r0 < MAX_GRID_Y ? a.rows - r0 : MAX_GRID_Y;
        s.x = (const char*)a.x + es * (size_t)(r0 * a.width);
        s.y = (char*)a.y + es * (size_t)(r0 * a.width);
        s.mean = (char*)a.mean + as * (size_t)r0;
        s.rstd = (char*)a.rstd + as * (size_t)r0;
        s.partial = (char*)a.partial + as * 3 * (size_t)(r0 * p.pieces);
        norm_long_stats<T><<<dim3((unsigned)p.pieces, (unsigned)s.rows), dim3(LONG_THREADS), 0, st>>>(s);
        const bool small = p.pieces <= FEW_PIECES;
        if (!small) norm_long_join<T><<<dim3((unsigned)s.rows), dim3(LONG_THREADS), 0, st>>>(s, (int)p.pieces);
        const int64_t sweeps = (a.width + longb_sweep<T>() - 1) / longb_sweep<T>();
        norm_long_apply<T><<<dim3((unsigned)sweeps, apply_groups(s.rows, sweeps, a.weight || a.bias)), dim3(LONG_THREADS), 0, st>>>(
            s, small ? (int)p.pieces : 0);
    }
    return hipGetLastError();
}

template <typename T, int THREADS, int ITER, int GROUPS> void launch_groups(NormArgs a, unsigned blocks, hipStream_t st) {
    if (!a.wbar) norm_row_vjp<T, THREADS, ITER, NO_PARAMS, GROUPS><<<dim3(blocks), dim3(THREADS * GROUPS), 0, st>>>(a);
    else if (blocks > 1 && columns<T>(a.rows, a.width)) {
        constexpr int COLS = THREADS * GROUPS / SLICES;
        a.column_blocks = (unsigned)((a.width + COLS - 1) / COLS);
        norm_row_vjp<T, THREADS, ITER, COLUMNS, GROUPS>
            <<<dim3(a.column_blocks + (unsigned)((a.rows + GROUPS - 1) / GROUPS)), dim3(THREADS * GROUPS), 0, st>>>(a);
    } else norm_row_vjp<T, THREADS, ITER, PARTS, GROUPS><<<dim3(blocks), dim3(THREADS * GROUPS), 0, st>>>(a);
}
template <typename T, int THREADS, int ITER> void launch_row_vjp(const NormArgs& a, unsigned blocks, hipStream_t st) {
    if constexpr (THREADS > 64) launch_groups<T, THREADS, ITER, 1>(a, blocks, st);
    else if (blocks == 1) launch_groups<T, THREADS, ITER, 16>(a, blocks, st);
    else launch_groups<T, THREADS, ITER, 4>(a, blocks, st);
}
template <typename T> hipError_t reverse(NormArgs a, hipStream_t st) {
    typedef acc_t<T> A;
    const int64_t n = a.width, vecs = (n + Vec16<T>::N - 1) / Vec16<T>::N;
    int64_t parts = 0;
    A* parted = (A*)a.partial;
    if (n * (int64_t)sizeof(T) <= VJP_ROW_BYTES) {
        parts = row_blocks<T>(a.rows, n);
        const unsigned b = (unsigned)parts;
        if (parts == 1 || columns<T>(a.rows, n)) parts = 0; // (nothing left to add up)
        if (vecs <= 64) launch_row_vjp<T, 64, 1>(a, b, st);
        else if (vecs <= 128) launch_row_vjp<T, 64, 2>(a, b, st);
        else if (vecs <= 256) launch_row_vjp<T, 256, 1>(a, b, st);
        else if (vecs <= 512) launch_row_vjp<T, 256, 2>(a, b, st);
        else if (vecs <= 1024) launch_row_vjp<T, 512, 2>(a, b, st);
        else launch_row_vjp<T, 512, 4>(a, b, st);
    } else {
        const LongPlan p = long_plan<T>(a.rows, n);
        a.sums = (A*)a.partial + 2 * a.rows * p.vpieces;
        a.partial2 = (A*)a.sums + 2 * a.rows;
        norm_long_vjp_sums<T><<<dim3((unsigned)p.vpieces, (unsigned)p.groups), dim3(LONG_THREADS), 0, st>>>(a);
        const bool small = p.vpieces <= FEW_PIECES;
        if (!small) norm_long_vjp_rows<T><<<dim3((unsigned)a.rows), dim3(LONG_THREADS), 0, st>>>(a, p.vpieces);
        norm_long_vjp_apply<T><<<dim3((unsigned)p.vpieces, apply_groups(a.rows, p.vpieces, false)), dim3(LONG_THREADS), 0, st>>>(
            a, small ? p.vpieces : 0);
        parts = p.groups > 1 ? p.groups : 0;
        parted = (A*)a.partial2;
    }
    if (a.wbar && parts > 16)
        norm_param_sum<T, 64><<<dim3((unsigned)((n + 63) / 64), 2), dim3(1024), 0, st>>>(parted, parts, n, (T*)a.wbar, (T*)a.bbar);
    else if (a.wbar && parts > 0)
        norm_param_sum<T, 512><<<dim3((unsigned)((n + 511) / 512), 2), dim3(1024), 0, st>>>(parted, parts, n, (T*)a.wbar, (T*)a.bbar);
    return hipGetLastError();
}

} // namespace

size_t gpt_norm_workspace(int dtype, int64_t rows, int64_t width, bool vjp) {
    switch (dtype) {
    case GPT_F64: return workspace<double>(rows, width, vjp);
    case GPT_F32: return workspace<float>(rows, width, vjp);
    case GPT_F16: return workspace<half_t>(rows, width, vjp);
    default: return workspace<bf16_t>(rows, width, vjp);
    }
}
hipError_t gpt_launch_norm(int dtype, const NormArgs& a, hipStream_t st) {
    switch (dtype) {
    case GPT_F64: return forward<double>(a, st);
    case GPT_F32: return forward<float>(a, st);
    case GPT_F16: return forward<half_t>(a, st);
    default: return forward<bf16_t>(a, st);
    }
}
hipError_t gpt_launch_norm_vjp(int dtype, const NormArgs& a, hipStream_t st) {
    switch (dtype) {
    case GPT_F64: return reverse<double>(a, st);
    case GPT_F32: return reverse<float>(a, st);
    case GPT_F16: return reverse<half_t>(a, st);
    default: return reverse<bf16_t>(a, st);
    }
}
