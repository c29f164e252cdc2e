// Log probability of observed classes under a linear read-out, and its reverse mode (gpt_categorical_logit_glm_lpmf, _vjp):
//
//   eta[n][v] = alpha[v] + beta[v] . x[n],  lse[n] = log sum_v exp eta[n][v],  lp[n] = eta[n][y[n]] - lse[n]
//   r[n][v] = lpbar[n] ([v = y[n]] - exp(eta[n][v] - lse[n])),  xbar = r beta,  alphabar = sum_n r,  betabar = r^T x
//
// The logits eta are never kept: one pass over the classes leaves a maximum and a sum for every row and tile of classes; the
// reverse mode computes eta once more, a piece of the classes at a time, and turns it into the piece's r in a workspace of
// bounded size, from which two more matrix products take xbar and betabar. Everything that a product sums over stands
// contiguously for both operands: r is written in both orders, x and the piece of beta are transposed once.
//
// Sums, statistics and accumulators are Acc (fp32; fp64 for fp64 data). One intermediate is rounded to 16 bits where the data
// have 16 bits: r, because the matrix instructions take both operands in one type. Its error (half a step, 2^-9 of each
// entry in bf16) is independent from entry to entry, and no larger than that of rounding the result. fp16 has too few exponents
// for the small probabilities of a large vocabulary: there r is stored times a power of two that brings max |lpbar| to 2^14
// and taken back from the products' Acc results.
#include "gpt_readout.h"
#include "gpt_tile.h"
#include <type_traits>

using namespace gptt;

namespace {

template <typename A> __device__ __forceinline__ A neg_inf() { return -(A)__builtin_inf(); }
__device__ __forceinline__ float exp_(float x) { return expf(x); }
__device__ __forceinline__ double exp_(double x) { return exp(x); }
__device__ __forceinline__ float log_(float x) { return logf(x); }
__device__ __forceinline__ double log_(double x) { return log(x); }

struct Scale { // of the stored r: host value, or (device) [scale, 1 / scale]
    const float* dev;
    float host, inverse;
    __device__ __forceinline__ float times() const { return dev ? dev[0] : host; }
    __device__ __forceinline__ float back() const { return dev ? dev[1] : inverse; }
};

template <typename T> struct LogitArgs {
    Operand<T> beta, x; // beta: the classes from v0 on
    const T* alpha;     // from v0 on, or null
    int64_t features, v0, classes; // classes: all of them
    const int64_t* y;
    int64_t tiles_v, tiles_n;
    // statistics
    acc_t<T>*part_max, *part_sum, *eta_y; // [tiles_v][rows], [tiles_v][rows], [rows]
    // r
    const acc_t<T>*lse, *lpbar;
    T *r, *rt; // [rows][ldr] and [classes of the piece][ldrt], zero up to ldr and ldrt
    int64_t ldr, ldrt;
    acc_t<T>* part_alpha; // [tiles_n][ldr] or null
    Scale scale;
};

constexpr int BM = 128, BN = 128, WM = 2, WN = 2;

// Tiles of eta, classes x rows. STATS: each tile's maximum and sum of exponentials for every row. else: r.
template <typename T, bool STATS> __global__ __launch_bounds__(64 * WM * WN) void class_logits(LogitArgs<T> a) {
    typedef acc_t<T> A;
    typedef Tile<T, BM, BN, WM, WN> Tl;
    __shared__ typename Tl::Vec lds[Tl::LDS_BYTES / 16];
    __shared__ A red[2][WM > WN ? WM : WN][BM > BN ? BM : BN];
    const int64_t m0 = (int64_t)(blockIdx.x / a.tiles_n) * BM, n0 = (int64_t)(blockIdx.x % a.tiles_n) * BN;
    Tl tl;
    tl.run(a.beta, m0, a.x, n0, 0, a.features, lds);
    const int lane = threadIdx.x & 63, wm = (threadIdx.x >> 6) / WN, wn = (threadIdx.x >> 6) % WN;
    const int64_t nv = a.beta.rows; // classes of this launch
#pragma unroll
    for (int i = 0; i < Tl::TM; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int64_t m = m0 + Tl::row(i, r);
            const A al = m < nv ? (a.alpha ? (A)a.alpha[m] : (A)0) : neg_inf<A>();
#pragma unroll
            for (int j = 0; j < Tl::TN; ++j) tl.acc[i][j][r] += al;
        }
    if (STATS) {
#pragma unroll
        for (int j = 0; j < Tl::TN; ++j) {
            const int64_t n = n0 + Tl::col(j);
            const int64_t y = n < a.x.rows ? a.y[n] : -1;
            A mx = neg_inf<A>();
            bool nan = false;
#pragma unroll
            for (int i = 0; i < Tl::TM; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    mx = fmax(mx, tl.acc[i][j][r]);
                    nan |= tl.acc[i][j][r] != tl.acc[i][j][r];
                    if (m0 + Tl::row(i, r) == y) a.eta_y[n] = tl.acc[i][j][r];
                }
            A s = 0;
#pragma unroll
            for (int i = 0; i < Tl::TM; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) s += mx == neg_inf<A>() ? (A)0 : exp_(tl.acc[i][j][r] - mx);
            if (nan) s = mx = (A)__builtin_nan("");
            // the four lane groups hold other classes of the same rows
#pragma unroll
            for (int k = 16; k <= 32; k <<= 1) {
                const A mo = __shfl_xor(mx, k, 64), so = __shfl_xor(s, k, 64);
                const A mm = (mx != mx || mo != mo) ? (A)__builtin_nan("") : fmax(mx, mo);
                s = mm == neg_inf<A>() ? (A)0 : s * exp_(mx - mm) + so * exp_(mo - mm);
                mx = mm;
            }
            if (lane < 16) {
                red[0][wm][Tl::col(j)] = mx;
                red[1][wm][Tl::col(j)] = s;
            }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < BN; c += Tl::THREADS) {
            A mx = red[0][0][c], s = red[1][0][c];
#pragma unroll
            for (int w = 1; w < WM; ++w) {
                const A mo = red[0][w][c], so = red[1][w][c];
                const A mm = (mx != mx || mo != mo) ? (A)__builtin_nan("") : fmax(mx, mo);
                s = mm == neg_inf<A>() ? (A)0 : s * exp_(mx - mm) + so * exp_(mo - mm);
                mx = mm;
            }
            if (n0 + c < a.x.rows) {
                a.part_max[(m0 / BM) * a.x.rows + n0 + c] = mx;
                a.part_sum[(m0 / BM) * a.x.rows + n0 + c] = s;
            }
        }
        return;
    }
    A lse[Tl::TN], w[Tl::TN];
    int64_t at[Tl::TN];
    const A up = (A)a.scale.times();
#pragma unroll
    for (int j = 0; j < Tl::TN; ++j) {
        const int64_t n = n0 + Tl::col(j), y = n < a.x.rows ? a.y[n] : -1;
        lse[j] = y >= 0 ? a.lse[n] : neg_inf<A>();
        w[j] = y < 0 ? (A)0 : y >= a.classes ? (A)__builtin_nan("") : a.lpbar ? a.lpbar[n] * up : up;
        at[j] = y - a.v0;
    }
#pragma unroll
    for (int i = 0; i < Tl::TM; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int64_t m = m0 + Tl::row(i, r);
            A total = 0;
#pragma unroll
            for (int j = 0; j < Tl::TN; ++j) {
                const int64_t n = n0 + Tl::col(j);
                // a row without an observation, a class behind the last, a row without any possible class: nothing
                const bool none = (lse[j] == neg_inf<A>() && w[j] == w[j]) || m >= nv;
                const A p = exp_(tl.acc[i][j][r] - lse[j]);
                const A v = none ? (A)0 : w[j] * ((m == at[j] ? (A)1 : (A)0) - p);
                total += v;
                if (m < a.ldr && n < a.x.rows) a.r[n * a.ldr + m] = (T)v;
                if (m < nv && n < a.ldrt) a.rt[m * a.ldrt + n] = (T)v;
            }
            if (a.part_alpha) {
#pragma unroll
                for (int k = 8; k >= 1; k >>= 1) total += __shfl_xor(total, k, 64);
                if ((lane & 15) == 0) red[0][wn][Tl::row(i, r)] = total;
            }
        }
    if (!a.part_alpha) return;
    __syncthreads();
    for (int c = threadIdx.x; c < BM; c += Tl::THREADS) {
        A s = red[0][0][c];
#pragma unroll
        for (int k = 1; k < WN; ++k) s += red[0][k][c];
        if (m0 + c < nv) a.part_alpha[(n0 / BN) * a.ldr + m0 + c] = s * (A)a.scale.back();
    }
}

// lse and lp of 16 rows from their tiles' statistics, 16 slices of the tiles in parallel
template <typename T> __global__ __launch_bounds__(256) void class_join(const acc_t<T>* part_max, const acc_t<T>* part_sum,
                                                                       const acc_t<T>* eta_y, const int64_t* y, int64_t tiles,
                                                                       int64_t rows, int64_t classes, acc_t<T>* lse, acc_t<T>* lp) {
    typedef acc_t<T> A;
    __shared__ A red[2][16][17];
    const int c = threadIdx.x & 15, k = threadIdx.x >> 4;
    const int64_t n = (int64_t)blockIdx.x * 16 + c;
    A mx = neg_inf<A>(), s = 0;
    bool nan = false;
    if (n < rows)
        for (int64_t i = k; i < tiles; i += 16) {
            const A mo = part_max[i * rows + n], so = part_sum[i * rows + n];
            nan |= mo != mo;
            const A mm = fmax(mx, mo);
            if (mm != neg_inf<A>()) s = s * exp_(mx - mm) + so * exp_(mo - mm);
            mx = mm;
        }
    red[0][k][c] = nan ? (A)__builtin_nan("") : mx;
    red[1][k][c] = s;
    __syncthreads();
    if (k || n >= rows) return;
    A top = neg_inf<A>();
    for (int i = 0; i < 16; ++i) {
        nan |= red[0][i][c] != red[0][i][c];
        top = fmax(top, red[0][i][c]);
    }
    A sum = 0;
    for (int i = 0; i < 16; ++i)
        if (red[0][i][c] != neg_inf<A>()) sum += red[1][i][c] * exp_(red[0][i][c] - top);
    const A l = nan ? (A)__builtin_nan("") : top == neg_inf<A>() ? top : top + log_(sum);
    if (lse) lse[n] = l;
    const int64_t yn = y[n];
    lp[n] = yn < 0 ? (A)0 : yn >= classes ? (A)__builtin_nan("") : l == neg_inf<A>() ? l : eta_y[n] - l;
}

// out[c][r] = in[r][c], rows behind the last, and (y given) those without an observation, zero. 64 x 64 through LDS
template <typename T> __global__ __launch_bounds__(256) void class_transpose(const T* in, int64_t ld, int64_t rows, int64_t cols,
                                                                            const int64_t* y, T* out, int64_t ldo) {
    __shared__ T tile[64][65];
    const int64_t r0 = (int64_t)blockIdx.x * 64, c0 = (int64_t)blockIdx.y * 64;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (int i = w; i < 64; i += 4) {
        const int64_t r = r0 + i, c = c0 + lane;
        tile[i][lane] = r < rows && c < cols && !(y && y[r] < 0) ? in[r * ld + c] : (T)0;
    }
    __syncthreads();
    for (int i = w; i < 64; i += 4) {
        const int64_t c = c0 + i, r = r0 + lane;
        if (c < cols && r < ldo) out[c * ldo + r] = tile[lane][i];
    }
}

// The products with r: out[n][m] = sum_k A[m][k] B[n][k] over this launch's share of k.
template <typename T> struct ProductArgs {
    Operand<T> A, B;
    int64_t K, share; // k of one split (a multiple of the tile's step)
    int64_t tiles_n;
    acc_t<T>* acc; // [splits][B.rows][A.rows]: sums so far
    int64_t plane; // elements from one split's sums to the next
    T* out;        // the result, where this launch completes it; else null
    int64_t ldo;
    bool add;        // acc holds earlier launches' sums
    const int64_t* y; // of B's rows, where those without an observation give zero; or null
    Scale scale;
};
template <typename T> __global__ __launch_bounds__(64 * WM * WN) void class_product(ProductArgs<T> a) {
    typedef acc_t<T> A;
    typedef Tile<T, BM, BN, WM, WN> Tl;
    __shared__ typename Tl::Vec lds[Tl::LDS_BYTES / 16];
    const int64_t m0 = (int64_t)(blockIdx.x / a.tiles_n) * BM, n0 = (int64_t)(blockIdx.x % a.tiles_n) * BN;
    const int64_t k0 = (int64_t)blockIdx.y * a.share, k1 = k0 + a.share < a.K ? k0 + a.share : a.K;
    Tl tl;
    tl.run(a.A, m0, a.B, n0, k0, k1, lds);
    const A back = (A)a.scale.back();
    A* acc = a.acc + (int64_t)blockIdx.y * a.plane;
#pragma unroll
    for (int j = 0; j < Tl::TN; ++j) {
        const int64_t n = n0 + Tl::col(j);
        if (n >= a.B.rows) continue;
        const bool none = a.y && a.y[n] < 0;
#pragma unroll
        for (int i = 0; i < Tl::TM; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int64_t m = m0 + Tl::row(i, r);
                if (m >= a.A.rows) continue;
                A v = none ? (A)0 : tl.acc[i][j][r] * back;
                if (a.add) v += acc[n * a.A.rows + m];
                if (a.out) a.out[n * a.ldo + m] = (T)v;
                else acc[n * a.A.rows + m] = v;
            }
    }
}
// out[i] <- sum over the splits
template <typename T> __global__ __launch_bounds__(256) void class_join_splits(const acc_t<T>* acc, int splits, int64_t plane,
                                                                              int64_t count, T* out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= count) return;
    acc_t<T> s = acc[i];
    for (int k = 1; k < splits; ++k) s += acc[k * plane + i];
    out[i] = (T)s;
}
// alphabar of a piece from the tiles' sums: 64 classes a workgroup, 4 waves share the tiles. acc: sums over row blocks
template <typename T> __global__ __launch_bounds__(256) void class_alpha(const acc_t<T>* part, int64_t tiles, int64_t ld, int64_t nv,
                                                                        acc_t<T>* acc, bool add, T* out) {
    typedef acc_t<T> A;
    __shared__ A red[4][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t v = (int64_t)blockIdx.x * 64 + lane;
    A s = 0;
    if (v < nv)
        for (int64_t i = w; i < tiles; i += 4) s += part[i * ld + v];
    red[w][lane] = s;
    __syncthreads();
    if (w || v >= nv) return;
    s = red[0][lane] + red[1][lane] + red[2][lane] + red[3][lane];
    if (add) s += acc[v];
    if (out) out[v] = (T)s;
    else acc[v] = s;
}
// fp16: scale = the power of two that brings max |lpbar| to [2^13, 2^14], and its inverse
__global__ __launch_bounds__(1024) void class_scale(const float* lpbar, const int64_t* y, int64_t rows, float* scale) {
    __shared__ float red[16];
    float m = 0.f;
    for (int64_t i = threadIdx.x; i < rows; i += 1024)
        if (y[i] >= 0) m = fmaxf(m, fabsf(lpbar[i]));
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) m = fmaxf(m, __shfl_xor(m, k, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x) return;
    for (int i = 1; i < 16; ++i) m = fmaxf(m, red[i]);
    int e = 0;
    if (m > 0.f && m < __builtin_inff()) (void)frexpf(m, &e); // m < 2^e
    e = e < -100 ? -100 : e > 100 ? 100 : e;
    scale[0] = ldexpf(1.f, 14 - e);
    scale[1] = ldexpf(1.f, e - 14);
}

// ---- plan -------------------------------------------------------------------------------------------------------------
int64_t up_to(int64_t n, int64_t m) { return (n + m - 1) / m * m; }
int64_t tiles_of(int64_t n, int64_t b) { return (n + b - 1) / b; }

constexpr int64_t ROW_BLOCK = 1 << 18;             // rows taken at a time
constexpr int64_t PIECE_BYTES = (int64_t)512 << 20; // r in both orders, of a piece of the classes and a block of the rows
constexpr int64_t FILL = 512;                       // workgroups that fill the card

// Splits of a product's k: enough workgroups to fill the card, at least 4 steps of k each
int64_t splits_of(int64_t tiles, int64_t K, int64_t step) {
    int64_t s = FILL / tiles;
    const int64_t most = K / (4 * step);
    if (s > most) s = most;
    return s < 1 ? 1 : s > 64 ? 64 : s;
}

template <typename T> struct Plan {
    int64_t block, blocks, piece, pieces, tiles_v, tiles_n, ldr, ldrt;
    int64_t xsplits, bsplits;
    // offsets in bytes
    size_t part_max, part_sum, eta_y, lse, scale, r, rt, xt, bt, part_alpha, alpha_acc, xacc, bacc, bytes;
    Plan(int64_t rows, int64_t features, int64_t classes, bool vjp) {
        const size_t A = sizeof(acc_t<T>), E = sizeof(T);
        block = rows < ROW_BLOCK ? rows : ROW_BLOCK;
        blocks = tiles_of(rows, block);
        tiles_v = tiles_of(classes, BM);
        tiles_n = tiles_of(block, BN);
        size_t at = 0;
        auto take = [&](size_t n) {
            const size_t p = at;
            at += (n + 255) / 256 * 256;
            return p;
        };
        part_max = take(A * (size_t)(tiles_v * block));
        part_sum = take(A * (size_t)(tiles_v * block));
        eta_y = take(A * (size_t)block);
        if (vjp) {
            piece = PIECE_BYTES / (int64_t)(2 * E) / up_to(block, BN) / BM * BM;
            if (piece < BM) piece = BM;
            if (piece > up_to(classes, BM)) piece = up_to(classes, BM);
            pieces = tiles_of(classes, piece);
            piece = up_to(tiles_of(classes, pieces), BM); // of about the same size
            pieces = tiles_of(classes, piece);
            ldr = piece;
            ldrt = up_to(block, BN);
            lse = take(A * (size_t)block);
            scale = take(8);
            r = take(E * (size_t)(block * ldr));
            rt = take(E * (size_t)(piece * ldrt));
            xt = take(E * (size_t)(features * ldrt));
            bt = take(E * (size_t)(features * ldr));
            part_alpha = take(A * (size_t)(tiles_n * ldr));
            alpha_acc = blocks > 1 ? take(A * (size_t)classes) : 0;
            xsplits = splits_of(tiles_of(features, BM) * tiles_n, piece, tile_k<T>());
            bsplits = splits_of(tiles_of(features, BM) * tiles_of(piece, BN), block, tile_k<T>());
            xacc = xsplits > 1 || pieces > 1 ? take(A * (size_t)(xsplits * block * features)) : 0;
            bacc = blocks > 1 ? take(A * (size_t)(bsplits * classes * features))
                              : bsplits > 1 ? take(A * (size_t)(bsplits * piece * features)) : 0;
        }
        bytes = at;
    }
};

template <typename T> hipError_t product(const Operand<T>& A, const Operand<T>& B, int64_t K, int64_t splits, acc_t<T>* acc,
                                         int64_t plane, bool add, bool last, T* out, const int64_t* y, Scale scale, hipStream_t st) {
    ProductArgs<T> p;
    p.A = A;
    p.B = B;
    p.K = K;
    p.share = up_to(tiles_of(K, splits), tile_k<T>());
    p.tiles_n = tiles_of(B.rows, BN);
    p.acc = acc;
    p.plane = plane;
    p.out = last && splits == 1 ? out : nullptr;
    p.ldo = A.rows;
    p.add = add;
    p.y = y;
    p.scale = scale;
    class_product<T><<<dim3((unsigned)(tiles_of(A.rows, BM) * p.tiles_n), (unsigned)splits), dim3(64 * WM * WN), 0, st>>>(p);
    if (last && splits > 1) {
        const int64_t count = A.rows * B.rows;
        class_join_splits<T><<<dim3((unsigned)tiles_of(count, 256)), dim3(256), 0, st>>>(acc, (int)splits, plane, count, out);
    }
    return hipGetLastError();
}

template <typename T> hipError_t launch(const ClassArgs& c, bool vjp, hipStream_t st) {
    typedef acc_t<T> A;
    const Plan<T> p(c.rows, c.features, c.classes, vjp);
    char* ws = (char*)c.ws;
    const int64_t D = c.features, V = c.classes;
    hipError_t e;
    Scale scale = {nullptr, 1.f, 1.f};
    if (vjp && std::is_same<T, half_t>::value) {
        if (c.lpbar) {
            scale.dev = (const float*)(ws + p.scale);
            class_scale<<<1, 1024, 0, st>>>((const float*)c.lpbar, c.y, c.rows, (float*)(ws + p.scale));
        } else {
            scale.host = 16384.f;
            scale.inverse = 1.f / 16384.f;
        }
    }
    for (int64_t n0 = 0; n0 < c.rows; n0 += p.block) {
        const int64_t N = c.rows - n0 < p.block ? c.rows - n0 : p.block;
        const bool first_block = n0 == 0, last_block = n0 + N == c.rows;
        LogitArgs<T> l;
        l.beta = {(const T*)c.beta, c.ldbeta, V};
        l.x = {(const T*)c.x + n0 * c.ldx, c.ldx, N};
        l.alpha = (const T*)c.alpha;
        l.features = D;
        l.v0 = 0;
        l.classes = V;
        l.y = c.y + n0;
        l.tiles_v = p.tiles_v;
        l.tiles_n = tiles_of(N, BN);
        l.part_max = (A*)(ws + p.part_max);
        l.part_sum = (A*)(ws + p.part_sum);
        l.eta_y = (A*)(ws + p.eta_y);
        l.scale = scale;
        class_logits<T, true><<<dim3((unsigned)(l.tiles_v * l.tiles_n)), dim3(64 * WM * WN), 0, st>>>(l);
        A* lse = vjp ? (A*)(ws + p.lse) : nullptr;
        class_join<T><<<dim3((unsigned)tiles_of(N, 16)), dim3(256), 0, st>>>(l.part_max, l.part_sum, l.eta_y, l.y, p.tiles_v, N, V,
                                                                             lse, (A*)c.lp + n0);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        if (!vjp) continue;
        const int64_t ldrt = up_to(N, BN);
        T *r = (T*)(ws + p.r), *rt = (T*)(ws + p.rt), *xt = (T*)(ws + p.xt), *bt = (T*)(ws + p.bt);
        class_transpose<T><<<dim3((unsigned)tiles_of(ldrt, 64), (unsigned)tiles_of(D, 64)), dim3(256), 0, st>>>(
            l.x.p, c.ldx, N, D, l.y, xt, ldrt);
        l.lse = lse;
        l.lpbar = c.lpbar ? (const A*)c.lpbar + n0 : nullptr;
        l.r = r;
        l.rt = rt;
        l.ldrt = ldrt;
        l.part_alpha = c.alphabar ? (A*)(ws + p.part_alpha) : nullptr;
        for (int64_t v0 = 0; v0 < V; v0 += p.piece) {
            const int64_t nv = V - v0 < p.piece ? V - v0 : p.piece;
            const bool first = v0 == 0, last = v0 + nv == V;
            l.beta = {(const T*)c.beta + v0 * c.ldbeta, c.ldbeta, nv};
            l.alpha = c.alpha ? (const T*)c.alpha + v0 : nullptr;
            l.v0 = v0;
            l.tiles_v = tiles_of(nv, BM);
            l.ldr = up_to(nv, BM);
            class_logits<T, false><<<dim3((unsigned)(l.tiles_v * l.tiles_n)), dim3(64 * WM * WN), 0, st>>>(l);
            class_transpose<T><<<dim3((unsigned)tiles_of(l.ldr, 64), (unsigned)tiles_of(D, 64)), dim3(256), 0, st>>>(
                l.beta.p, c.ldbeta, nv, D, nullptr, bt, l.ldr);
            if (c.alphabar)
                class_alpha<T><<<dim3((unsigned)tiles_of(nv, 64)), dim3(256), 0, st>>>(
                    l.part_alpha, l.tiles_n, l.ldr, nv, (A*)(ws + p.alpha_acc) + v0, !first_block,
                    last_block ? (T*)c.alphabar + v0 : nullptr);
            if ((e = hipGetLastError()) != hipSuccess) return e;
            if ((e = product<T>({bt, l.ldr, D}, {r, l.ldr, N}, l.ldr, p.xsplits, (A*)(ws + p.xacc), p.block * D, !first, last,
                                (T*)c.xbar + n0 * D, l.y, scale, st)) != hipSuccess)
                return e;
            A* bacc = (A*)(ws + p.bacc) + (p.blocks > 1 ? v0 * D : 0);
            if ((e = product<T>({xt, ldrt, D}, {rt, ldrt, nv}, ldrt, p.bsplits, bacc, (p.blocks > 1 ? V : p.piece) * D, !first_block,
                                last_block, (T*)c.betabar + v0 * D, nullptr, scale, st)) != hipSuccess)
                return e;
        }
    }
    return hipSuccess;
}

} // namespace

size_t gpt_class_workspace(int dtype, int64_t rows, int64_t features, int64_t classes, bool vjp) {
    switch (dtype) {
    case GPT_F64: return Plan<double>(rows, features, classes, vjp).bytes;
    case GPT_F32: return Plan<float>(rows, features, classes, vjp).bytes;
    case GPT_F16: return Plan<half_t>(rows, features, classes, vjp).bytes;
    default: return Plan<bf16_t>(rows, features, classes, vjp).bytes;
    }
}
hipError_t gpt_launch_class(int dtype, const ClassArgs& a, bool vjp, hipStream_t st) {
    switch (dtype) {
    case GPT_F64: return launch<double>(a, vjp, st);
    case GPT_F32: return launch<float>(a, vjp, st);
    case GPT_F16: return launch<half_t>(a, vjp, st);
    default: return launch<bf16_t>(a, vjp, st);
    }
}
