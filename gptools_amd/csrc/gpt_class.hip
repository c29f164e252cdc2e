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
// have 16 bits: r, because the matrix instructions take both operands in one type. Its error (half a step of each entry) is
// independent from entry to entry, and no larger than that of rounding the result. The rows' cotangents stay out of that
// rounding where they can: for xbar they multiply the product's Acc rows, for betabar (whose sum runs over the rows) r
// holds them divided by the largest of them, so that cotangents that are all alike (a sum's, a mean's) leave [v = y] exact. fp16
// has too few exponents for the small probabilities of a large vocabulary: there r is stored times 2^14.
#include "gpt_class_few.h"
#include "gpt_readout.h"
#include "gpt_tile.h"
#include <type_traits>

using namespace gptt;

namespace {

// The 4 x 4 transpose within every four neighbouring lanes: lane b gives value r in place r, and takes lane k's value b in
// place k. 16-bit values, two a word.
__device__ __forceinline__ void transpose4(uint32_t& lo, uint32_t& hi) {
    const int b = threadIdx.x & 3;
    const uint32_t give = b & 2 ? lo : hi;
    const uint32_t got = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)give, 0x4e, 0xf, 0xf, true); // lane ^ 2
    const uint32_t p = b & 2 ? got : lo, q = b & 2 ? hi : got; // values 2 (b / 2), + 1 of lanes b & 1 and (b & 1) + 2
    const uint32_t po = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)p, 0xb1, 0xf, 0xf, true); // lane ^ 1
    const uint32_t qo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)q, 0xb1, 0xf, 0xf, true);
    const uint32_t sel = b & 1 ? 0x03020706u : 0x05040100u;
    lo = __builtin_amdgcn_perm(po, p, sel);
    hi = __builtin_amdgcn_perm(qo, q, sel);
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    typedef T V2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, V2{(T)a, (T)b});
}

template <typename T> struct LogitArgs {
    Operand<T> beta, x; // beta: the classes from v0 on
    const T* alpha;     // from v0 on, or null
    int64_t features, v0, classes; // classes: all of them
    const int64_t* y;
    int64_t tiles_v, tiles_n;
    // statistics
    acc_t<T>*part_max, *part_sum, *eta_y; // [tiles_v][rows], [tiles_v][rows], [rows]
    // r, and r with the rows' cotangents in the other order: [rows][ldr] and [classes of the piece][ldrt], in whole tiles
    const acc_t<T>*lse, *lpbar;
    T *r, *rt;
    int64_t ldr, ldrt;
    acc_t<T>* part_alpha; // [tiles_n][ldr] or null
    Largest<acc_t<T>> largest;
};

// Tiles of eta, classes x rows. STATS: each tile's maximum and sum of exponentials for every row. else: r.
template <typename T, typename Tl, bool STATS> __global__ __launch_bounds__(Tl::THREADS) void class_logits(LogitArgs<T> a) {
    typedef acc_t<T> A;
    __shared__ typename Tl::Vec lds[Tl::LDS_BYTES / 16];
    __shared__ A red[2][Tl::WM > Tl::WN ? Tl::WM : Tl::WN][Tl::BM > Tl::BN ? Tl::BM : Tl::BN];
    int64_t tm, tn;
    if (!tile_place(blockIdx.x, a.tiles_v, a.tiles_n, tm, tn)) return;
    const int64_t m0 = tm * Tl::BM, n0 = tn * Tl::BN;
    Tl tl;
    tl.run(a.beta, m0, a.x, n0, 0, a.features, lds);
    const int lane = threadIdx.x & 63, wm = (threadIdx.x >> 6) / Tl::WN, wn = (threadIdx.x >> 6) % Tl::WN;
    const int nv = (int)(a.beta.rows - m0 < Tl::BM ? a.beta.rows - m0 : Tl::BM); // classes of this tile
#pragma unroll
    for (int i = 0; i < Tl::TM; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int m = Tl::row(i, r);
            const A al = m < nv ? (a.alpha ? level_log2e((A)a.alpha[m0 + m]) : (A)0) : neg_inf<A>();
#pragma unroll
            for (int j = 0; j < Tl::TN; ++j) tl.acc[i][j][r] = times_log2e(tl.acc[i][j][r]) + al;
        }
    if (STATS) {
#pragma unroll
        for (int j = 0; j < Tl::TN; ++j) {
            const int64_t n = n0 + Tl::col(j);
            const int64_t y = n < a.x.rows ? a.y[n] - m0 : -1;
            const int at = y >= 0 && y < Tl::BM ? (int)y : -1;
            A mx = neg_inf<A>(), here = 0;
            bool mine = false; // (one lane group of one wave holds the row's class)
#pragma unroll
            for (int i = 0; i < Tl::TM; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    mx = fmax(mx, tl.acc[i][j][r]);
                    const bool is = Tl::row(i, r) == at;
                    mine |= is;
                    here = is ? tl.acc[i][j][r] : here;
                }
            if (mine && at < nv) a.eta_y[n] = here;
            A s = 0;
            const A ref = about(mx);
#pragma unroll
            for (int i = 0; i < Tl::TM; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) s += exp_log2e(tl.acc[i][j][r] - ref);
            // the four lane groups hold other classes of the same rows
#pragma unroll
            for (int k = 16; k <= 32; k <<= 1) join(mx, s, __shfl_xor(mx, k, 64), __shfl_xor(s, k, 64));
            if (lane < 16) {
                red[0][wm][Tl::col(j)] = mx;
                red[1][wm][Tl::col(j)] = s;
            }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < Tl::BN; c += Tl::THREADS) {
            A mx = red[0][0][c], s = red[1][0][c];
#pragma unroll
            for (int w = 1; w < Tl::WM; ++w) join(mx, s, red[0][w][c], red[1][w][c]);
            if (n0 + c < a.x.rows) {
                a.part_max[tm * a.x.rows + n0 + c] = mx;
                a.part_sum[tm * a.x.rows + n0 + c] = s;
            }
        }
        return;
    }
    A lse[Tl::TN], w[Tl::TN];
    bool none[Tl::TN];
    int at[Tl::TN];
    const A largest = a.largest.get();
#pragma unroll
    for (int j = 0; j < Tl::TN; ++j) {
        const int64_t n = n0 + Tl::col(j), y = n < a.x.rows ? a.y[n] : -1;
        lse[j] = y < 0 ? (A)0 : y >= a.classes ? (A)__builtin_nan("") : a.lse[n];
        none[j] = y < 0 || lse[j] == neg_inf<A>(); // no observation, or no possible class
        w[j] = none[j] ? (A)0 : a.lpbar ? a.lpbar[n] / largest : (A)1;
        const int64_t from = y - a.v0 - m0;
        at[j] = y >= 0 && from >= 0 && from < Tl::BM ? (int)from : -1;
    }
    constexpr A up = stored_scale<T>();
    A total[Tl::TM][4];
#pragma unroll
    for (int i = 0; i < Tl::TM; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            total[i][r] = 0;
#pragma unroll
            for (int j = 0; j < Tl::TN; ++j) {
                const A p = exp_log2e(tl.acc[i][j][r] - lse[j]);
                const A v = none[j] ? (A)0 : (Tl::row(i, r) == at[j] ? up : (A)0) - up * p;
                tl.acc[i][j][r] = v;
                total[i][r] += v * w[j];
            }
        }
    if constexpr (Tl::TM == 8 && sizeof(T) == 2) {
        // r: 16 neighbouring classes of one row a lane; rt: after the transpose, 16 neighbouring rows of one class a lane
        const int64_t mq = m0 + Tl::row(0, 0), nq = n0 + Tl::col(0);
#pragma unroll
        for (int j = 0; j < Tl::TN; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint4* to = reinterpret_cast<uint4*>(a.r + (nq + Tl::fragment(j)) * a.ldr + mq + 64 * h);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const auto &c = tl.acc[4 * h + 2 * k][j], &d = tl.acc[4 * h + 2 * k + 1][j];
                    to[k] = make_uint4(pack2<T>(c[0], c[1]), pack2<T>(c[2], c[3]), pack2<T>(d[0], d[1]), pack2<T>(d[2], d[3]));
                }
            }
        const int64_t nb = nq - (lane & 3), mb = mq + (lane & 3);
#pragma unroll
        for (int i = 0; i < Tl::TM; ++i) {
            uint32_t u[Tl::TN][2];
#pragma unroll
            for (int j = 0; j < Tl::TN; ++j) {
                const auto& c = tl.acc[i][j];
                u[j][0] = pack2<T>(c[0] * w[j], c[1] * w[j]);
                u[j][1] = pack2<T>(c[2] * w[j], c[3] * w[j]);
                transpose4(u[j][0], u[j][1]);
            }
            uint4* to = reinterpret_cast<uint4*>(a.rt + (mb + Tl::fragment(i)) * a.ldrt + nb);
            to[0] = make_uint4(u[0][0], u[0][1], u[1][0], u[1][1]);
            to[1] = make_uint4(u[2][0], u[2][1], u[3][0], u[3][1]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < Tl::TM; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < Tl::TN; ++j) {
                    const int64_t m = m0 + Tl::row(i, r), n = n0 + Tl::col(j);
                    a.r[n * a.ldr + m] = (T)tl.acc[i][j][r];
                    a.rt[m * a.ldrt + n] = (T)(tl.acc[i][j][r] * w[j]);
                }
    }
    if (!a.part_alpha) return;
#pragma unroll
    for (int i = 0; i < Tl::TM; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const A s = sum16(total[i][r]);
            if ((lane & 15) == 0) red[0][wn][Tl::row(i, r)] = s;
        }
    __syncthreads();
    for (int c = threadIdx.x; c < nv; c += Tl::THREADS) {
        A s = red[0][0][c];
#pragma unroll
        for (int k = 1; k < Tl::WN; ++k) s += red[0][k][c];
        a.part_alpha[tn * a.ldr + m0 + c] = s * (largest / up);
    }
}

// lse (times log2(e) in fp32) and lp of 16 rows from their tiles' statistics, 16 slices of the tiles in parallel
template <typename T> __global__ __launch_bounds__(256) void class_join(const acc_t<T>* part_max, const acc_t<T>* part_sum,
                                                                       const acc_t<T>* eta_y, const int64_t* y, int64_t tiles,
                                                                       int64_t rows, int64_t classes, acc_t<T>* lse, acc_t<T>* lp) {
    typedef acc_t<T> A;
    __shared__ A red[2][16][17];
    const int c = threadIdx.x & 15, k = threadIdx.x >> 4;
    const int64_t n = (int64_t)blockIdx.x * 16 + c;
    A mx = neg_inf<A>(), s = 0;
    if (n < rows)
        for (int64_t i = k; i < tiles; i += 16) join(mx, s, part_max[i * rows + n], part_sum[i * rows + n]);
    red[0][k][c] = mx;
    red[1][k][c] = s;
    __syncthreads();
    if (k || n >= rows) return;
    for (int i = 1; i < 16; ++i) join(mx, s, red[0][i][c], red[1][i][c]);
    const int64_t yn = y[n];
    A l;
    lp[n] = row_lp(yn, classes, mx, s, yn >= 0 && yn < classes ? eta_y[n] : (A)0, l);
    if (lse) lse[n] = l;
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

// out[r][0..ldo) = in[r][0..cols), zeros behind: rows that start on 16 bytes and end with a step of k
template <typename T> __global__ __launch_bounds__(256) void class_align(const T* in, int64_t ld, int64_t rows, int64_t cols, T* out,
                                                                        int64_t ldo) {
    constexpr int N = Vec16<T>::N;
    const int64_t per = ldo / N, count = rows * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / per, k = (i - r * per) * N;
        *reinterpret_cast<typename Vec16<T>::V*>(out + r * ldo + k) = tile_chunk<T>({in, ld, rows}, r, k, cols);
    }
}

// The products with r: out[n][m] = sum_k A[m][k] B[n][k] over this launch's share of k.
template <typename T> struct ProductArgs {
    Operand<T> A, B;
    int64_t K, share; // k of one split (a multiple of the tile's step)
    int64_t tiles_m, tiles_n;
    acc_t<T>* acc; // [splits][B.rows][A.rows]: sums so far
    int64_t plane; // elements from one split's sums to the next
    T* out;        // the result, where this launch completes it; else null
    int64_t ldo;
    bool add; // acc holds earlier launches' sums
    // xbar: B's rows are the rows of x, each times its cotangent (zero without an observation). betabar: y null
    const int64_t* y;
    const acc_t<T>* lpbar;
    Largest<acc_t<T>> largest;
};
template <typename T, typename Tl> __global__ __launch_bounds__(Tl::THREADS) void class_product(ProductArgs<T> a) {
    typedef acc_t<T> A;
    __shared__ typename Tl::Vec lds[Tl::LDS_BYTES / 16];
    int64_t tm, tn;
    if (!tile_place(blockIdx.x, a.tiles_m, a.tiles_n, tm, tn)) return;
    const int64_t m0 = tm * Tl::BM, n0 = tn * Tl::BN;
    const int64_t k0 = (int64_t)blockIdx.y * a.share, k1 = k0 + a.share < a.K ? k0 + a.share : a.K;
    Tl tl;
    tl.run(a.A, m0, a.B, n0, k0, k1, lds);
    A* acc = a.acc + (int64_t)blockIdx.y * a.plane;
    const A largest = a.y ? (A)1 : a.largest.get();
#pragma unroll
    for (int j = 0; j < Tl::TN; ++j) {
        const int64_t n = n0 + Tl::col(j);
        if (n >= a.B.rows) continue;
        A back = largest;
        bool none = false;
        if (a.y) {
            none = a.y[n] < 0;
            if (a.lpbar && !none) back = a.lpbar[n];
        }
        back /= (A)stored_scale<T>();
        if constexpr (Tl::TM == 8) {
            // 16 neighbouring values a lane: whole vectors where the rows of the result allow them
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int64_t m = m0 + Tl::row(4 * h, 0);
                A v[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) v[k] = none ? (A)0 : tl.acc[4 * h + k / 4][j][k % 4] * back;
                A* s = acc + n * a.A.rows + m;
                T* o = a.out + n * a.ldo + m;
                if (m + 16 <= a.A.rows) {
                    if (a.add) {
#pragma unroll
                        for (int k = 0; k < 16; k += Vec16<A>::N) {
                            const auto u = load16(s + k);
#pragma unroll
                            for (int e = 0; e < Vec16<A>::N; ++e) v[k + e] += u[e];
                        }
                    }
                    if (a.out) {
#pragma unroll
                        for (int k = 0; k < 16; k += Vec16<T>::N) {
                            typename Vec16<T>::V u;
#pragma unroll
                            for (int e = 0; e < Vec16<T>::N; ++e) u[e] = (T)v[k + e];
                            store16(o + k, u);
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < 16; k += Vec16<A>::N) {
                            typename Vec16<A>::V u;
#pragma unroll
                            for (int e = 0; e < Vec16<A>::N; ++e) u[e] = v[k + e];
                            store16(s + k, u);
                        }
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        if (m + k >= a.A.rows) continue;
                        if (a.add) v[k] += s[k];
                        if (a.out) o[k] = (T)v[k];
                        else s[k] = v[k];
                    }
                }
            }
        } else {
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

// ---- plan -------------------------------------------------------------------------------------------------------------
int64_t up_to(int64_t n, int64_t m) { return (n + m - 1) / m * m; }
int64_t tiles_of(int64_t n, int64_t b) { return (n + b - 1) / b; }

constexpr int64_t ROW_BLOCK = 1 << 18;              // rows taken at a time
constexpr int64_t PIECE_BYTES = (int64_t)512 << 20; // r in both orders, of a piece of the classes and a block of the rows
constexpr int64_t FILL = 512;                       // workgroups that fill the card
constexpr int64_t EDGE = 256;                       // the largest tile's edge
constexpr int64_t WIDE_TILES = 96;                  // wide tiles from this many on

// Splits of a product's k: enough workgroups to fill the card, at least 4 steps of k each
int64_t splits_of(int64_t tiles, int64_t K, int64_t step) {
    int64_t s = FILL / tiles;
    const int64_t most = K / (4 * step);
    if (s > most) s = most;
    return s < 1 ? 1 : s > 64 ? 64 : s;
}
// 256 x 256 tiles for a product of m x n results?
template <typename T> bool wide(int64_t m, int64_t n) {
    return sizeof(T) == 2 && tiles_of(m, WideTile<T>::BM) * tiles_of(n, WideTile<T>::BN) >= WIDE_TILES;
}

template <typename T> struct Plan {
    int64_t block, blocks, piece, pieces, tiles_v, tiles_n, ldr, ldrt, ldk;
    int64_t xsplits, bsplits;
    // offsets in bytes
    size_t part_max, part_sum, eta_y, lse, scale, r, rt, xt, bt, part_alpha, alpha_acc, xacc, bacc, xa, ba, bytes;
    Plan(int64_t rows, int64_t features, int64_t classes, bool vjp) {
        const size_t A = sizeof(acc_t<T>), E = sizeof(T);
        block = rows < ROW_BLOCK ? rows : ROW_BLOCK;
        blocks = tiles_of(rows, block);
        tiles_v = tiles_of(classes, SmallTile<T>::BM);
        tiles_n = tiles_of(block, SmallTile<T>::BN);
        size_t at = 0;
        auto take = [&](size_t n) {
            const size_t p = at;
            at += (n + 255) / 256 * 256;
            return p;
        };
        part_max = take(A * (size_t)(tiles_v * block));
        part_sum = take(A * (size_t)(tiles_v * block));
        eta_y = take(A * (size_t)block);
        ldk = 0;
        if (wide<T>(classes, block) && features * E % 16) { // copies whose rows start on 16 bytes
            ldk = up_to(features, tile_k<T>());
            xa = take(E * (size_t)(block * ldk));
            ba = take(E * (size_t)(classes * ldk));
        }
        if (vjp) {
            piece = PIECE_BYTES / (int64_t)(2 * E) / up_to(block, EDGE) / EDGE * EDGE;
            if (piece < EDGE) piece = EDGE;
            if (piece > up_to(classes, EDGE)) piece = up_to(classes, EDGE);
            pieces = tiles_of(classes, piece);
            piece = up_to(tiles_of(classes, pieces), EDGE); // of about the same size
            pieces = tiles_of(classes, piece);
            ldr = piece;
            ldrt = up_to(block, EDGE);
            lse = take(A * (size_t)block);
            scale = take(A * SCALE_PARTS);
            r = take(E * (size_t)(ldrt * ldr));
            rt = take(E * (size_t)(ldr * ldrt));
            xt = take(E * (size_t)(features * ldrt));
            bt = take(E * (size_t)(features * ldr));
            part_alpha = take(A * (size_t)(tiles_n * ldr));
            alpha_acc = blocks > 1 ? take(A * (size_t)classes) : 0;
            xsplits = product_splits(features, block, piece);
            bsplits = product_splits(features, piece, block);
            xacc = xsplits > 1 || pieces > 1 ? take(A * (size_t)(xsplits * block * features)) : 0;
            bacc = blocks > 1 ? take(A * (size_t)(bsplits * classes * features))
                              : bsplits > 1 ? take(A * (size_t)(bsplits * piece * features)) : 0;
        }
        bytes = at;
    }
    static int64_t product_splits(int64_t m, int64_t n, int64_t K) {
        const int64_t edge = wide<T>(m, n) ? WideTile<T>::BM : SmallTile<T>::BM;
        return splits_of(tiles_of(m, edge) * tiles_of(n, edge) * (wide<T>(m, n) ? 2 : 1), K, tile_k<T>());
    }
};

template <typename T, typename Tl> void logits(LogitArgs<T> l, bool stats, hipStream_t st) {
    l.tiles_v = tiles_of(l.beta.rows, Tl::BM);
    l.tiles_n = tiles_of(l.x.rows, Tl::BN);
    const dim3 grid(tile_grid(l.tiles_v, l.tiles_n));
    if (stats) class_logits<T, Tl, true><<<grid, dim3(Tl::THREADS), 0, st>>>(l);
    else class_logits<T, Tl, false><<<grid, dim3(Tl::THREADS), 0, st>>>(l);
}
// -> edge of the tiles taken
template <typename T> int64_t logits_any(const LogitArgs<T>& l, bool use_wide, bool stats, hipStream_t st) {
    if constexpr (sizeof(T) == 2) {
        if (use_wide) {
            logits<T, WideTile<T>>(l, stats, st);
            return WideTile<T>::BM;
        }
    }
    logits<T, SmallTile<T>>(l, stats, st);
    return SmallTile<T>::BM;
}

template <typename T> hipError_t product(ProductArgs<T> p, int64_t splits, bool last, T* out, hipStream_t st) {
    p.share = up_to(tiles_of(p.K, splits), tile_k<T>());
    p.out = last && splits == 1 ? out : nullptr;
    p.ldo = p.A.rows;
    bool done = false;
    if constexpr (sizeof(T) == 2) {
        typedef WideTile<T> Tl;
        if (wide<T>(p.A.rows, p.B.rows)) {
            p.tiles_m = tiles_of(p.A.rows, Tl::BM);
            p.tiles_n = tiles_of(p.B.rows, Tl::BN);
            class_product<T, Tl><<<dim3(tile_grid(p.tiles_m, p.tiles_n), (unsigned)splits), dim3(Tl::THREADS), 0, st>>>(p);
            done = true;
        }
    }
    if (!done) {
        typedef SmallTile<T> Tl;
        p.tiles_m = tiles_of(p.A.rows, Tl::BM);
        p.tiles_n = tiles_of(p.B.rows, Tl::BN);
        class_product<T, Tl><<<dim3(tile_grid(p.tiles_m, p.tiles_n), (unsigned)splits), dim3(Tl::THREADS), 0, st>>>(p);
    }
    if (last && splits > 1) {
        const int64_t count = p.A.rows * p.B.rows;
        class_join_splits<T><<<dim3((unsigned)tiles_of(count, 256)), dim3(256), 0, st>>>(p.acc, (int)splits, p.plane, count, out);
    }
    return hipGetLastError();
}

// ---- few rows
template <typename T> struct FewPlan {
    // class tiles of a workgroup where the classes are enough to fill the card that way (fp64 has not the LDS for more)
    static constexpr int CT = sizeof(T) == 8 ? 2 : 4;
    bool large;
    int64_t tiles, ldv, ldrt, share, splits;
    size_t part_max, part_sum, eta, lse, largest, r, rt, xt, xpart, bytes;
    FewPlan(int64_t rows, int64_t D, int64_t V, bool vjp) {
        const size_t A = sizeof(acc_t<T>), E = sizeof(T);
        size_t at = 0;
        auto take = [&](size_t n) {
            const size_t p = at;
            at += (n + 255) / 256 * 256;
            return p;
        };
        large = V >= 16 * CT * FILL / 2;
        tiles = tiles_of(V, large ? 16 * CT : 16);
        part_max = take(A * (size_t)(rows * tiles));
        part_sum = take(A * (size_t)(rows * tiles));
        if (vjp) {
            ldv = up_to(V, 64);
            ldrt = rows <= 32 ? 32 : 64;
            const int64_t slabs = tiles_of(D, 16 * Vec16<T>::N);
            splits = tiles_of(2 * FILL, slabs);
            if (splits > tiles_of(V, 128)) splits = tiles_of(V, 128);
            share = up_to(tiles_of(V, splits), 128);
            splits = tiles_of(V, share);
            eta = take(A * (size_t)(rows * ldv));
            lse = take(A * (size_t)rows);
            largest = take(A * FEW);
            r = take(E * (size_t)(rows * ldv));
            rt = take(E * (size_t)(V * ldrt));
            xt = take(E * (size_t)(D * ldrt));
            xpart = take(A * (size_t)(splits * rows * D));
        }
        bytes = at;
    }
};
template <typename T, int NT> hipError_t launch_few(const ClassArgs& c, bool vjp, hipStream_t st) {
    typedef acc_t<T> A;
    const int64_t D = c.features, V = c.classes;
    const FewPlan<T> p(c.rows, D, V, vjp);
    char* ws = (char*)c.ws;
    FewArgs<T> a = {};
    a.x = {(const T*)c.x, c.ldx, c.rows};
    a.beta = {(const T*)c.beta, c.ldbeta, V};
    a.alpha = (const T*)c.alpha;
    a.y = c.y;
    a.lpbar = (const A*)c.lpbar;
    a.features = D;
    a.part_max = (A*)(ws + p.part_max);
    a.part_sum = (A*)(ws + p.part_sum);
    a.tiles = p.tiles;
    a.lp = (A*)c.lp;
    if (vjp) {
        a.eta = (A*)(ws + p.eta);
        a.ldv = p.ldv;
        a.lse = (A*)(ws + p.lse);
        a.largest = (A*)(ws + p.largest);
        a.r = (T*)(ws + p.r);
        a.rt = (T*)(ws + p.rt);
        a.ldrt = p.ldrt;
        a.alphabar = (T*)c.alphabar;
        a.xpart = (A*)(ws + p.xpart);
        a.share = p.share;
    }
    const dim3 grid((unsigned)p.tiles);
    if (p.large) class_few_logits<T, NT, FewPlan<T>::CT, 4><<<grid, dim3(256), 0, st>>>(a);
    else class_few_logits<T, NT, 1, 8><<<grid, dim3(512), 0, st>>>(a);
    class_few_join<T><<<dim3((unsigned)c.rows), dim3(256), 0, st>>>(a);
    if (!vjp) return hipGetLastError();
    const Largest<A> largest = {c.lpbar ? a.largest : nullptr};
    class_few_r<T><<<dim3((unsigned)(p.ldv / 64)), dim3(256), 0, st>>>(a, largest);
    class_few_xbar<T, NT><<<dim3((unsigned)tiles_of(D, 16 * Vec16<T>::N), (unsigned)p.splits), dim3(256), 0, st>>>(a);
    class_few_xbar_join<T><<<dim3((unsigned)tiles_of(c.rows * D, 256)), dim3(256), 0, st>>>(a, (int)p.splits, (T*)c.xbar);
    T* xt = (T*)(ws + p.xt);
    class_transpose<T><<<dim3((unsigned)tiles_of(p.ldrt, 64), (unsigned)tiles_of(D, 64)), dim3(256), 0, st>>>(a.x.p, c.ldx, c.rows, D,
                                                                                                            c.y, xt, p.ldrt);
    constexpr int NG = (NT <= 2 ? 32 : 64) / (4 * Vec16<T>::N);
    const int64_t slabs = tiles_of(D, Slab<T>::WIDTH);
    int64_t shares = tiles_of(4 * FILL, slabs);
    if (shares > tiles_of(V, 128)) shares = tiles_of(V, 128);
    class_few_beta<T, NG><<<dim3((unsigned)slabs, (unsigned)shares), dim3(256), 0, st>>>(a, xt, (T*)c.betabar, largest);
    return hipGetLastError();
}
template <typename T> size_t space(int64_t rows, int64_t features, int64_t classes, bool vjp) {
    return rows <= FEW ? FewPlan<T>(rows, features, classes, vjp).bytes : Plan<T>(rows, features, classes, vjp).bytes;
}
template <typename T> hipError_t launch_few(const ClassArgs& c, bool vjp, hipStream_t st) {
    if (c.rows <= 16) return launch_few<T, 1>(c, vjp, st);
    if (c.rows <= 32) return launch_few<T, 2>(c, vjp, st);
    return launch_few<T, 4>(c, vjp, st);
}

template <typename T> hipError_t launch(const ClassArgs& c, bool vjp, hipStream_t st) {
    typedef acc_t<T> A;
    if (c.rows <= FEW) return launch_few<T>(c, vjp, st);
    const Plan<T> p(c.rows, c.features, c.classes, vjp);
    char* ws = (char*)c.ws;
    const int64_t D = c.features, V = c.classes;
    hipError_t e;
    Operand<T> beta = {(const T*)c.beta, c.ldbeta, V};
    int64_t K = D;
    if (p.ldk) {
        T* to = (T*)(ws + p.ba);
        class_align<T><<<dim3(2048), dim3(256), 0, st>>>(beta.p, beta.ld, V, D, to, p.ldk);
        beta = {to, p.ldk, V};
        K = p.ldk;
    }
    Largest<A> largest = {nullptr};
    if (vjp && c.lpbar) {
        largest.parts = (A*)(ws + p.scale);
        class_scale<A><<<dim3(SCALE_PARTS), dim3(256), 0, st>>>((const A*)c.lpbar, c.y, c.rows, (A*)(ws + p.scale));
    }
    for (int64_t n0 = 0; n0 < c.rows; n0 += p.block) {
        const int64_t N = c.rows - n0 < p.block ? c.rows - n0 : p.block;
        const bool first_block = n0 == 0, last_block = n0 + N == c.rows;
        const T* x = (const T*)c.x + n0 * c.ldx;
        LogitArgs<T> l = {};
        l.beta = beta;
        l.x = {x, c.ldx, N};
        if (p.ldk) {
            T* to = (T*)(ws + p.xa);
            class_align<T><<<dim3(1024), dim3(256), 0, st>>>(x, c.ldx, N, D, to, p.ldk);
            l.x = {to, p.ldk, N};
        }
        bool use_wide = false;
        if constexpr (sizeof(T) == 2) use_wide = wide<T>(V, N) && WideTile<T>::fits(l.beta) && WideTile<T>::fits(l.x);
        l.alpha = (const T*)c.alpha;
        l.features = K;
        l.classes = V;
        l.y = c.y + n0;
        l.part_max = (A*)(ws + p.part_max);
        l.part_sum = (A*)(ws + p.part_sum);
        l.eta_y = (A*)(ws + p.eta_y);
        l.largest = largest;
        const int64_t edge = logits_any<T>(l, use_wide, true, st);
        A* lse = vjp ? (A*)(ws + p.lse) : nullptr;
        class_join<T><<<dim3((unsigned)tiles_of(N, 16)), dim3(256), 0, st>>>(l.part_max, l.part_sum, l.eta_y, l.y, tiles_of(V, edge), N,
                                                                             V, lse, (A*)c.lp + n0);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        if (!vjp) continue;
        const int64_t ldrt = up_to(N, edge); // (r is written in whole tiles)
        T *r = (T*)(ws + p.r), *rt = (T*)(ws + p.rt), *xt = (T*)(ws + p.xt), *bt = (T*)(ws + p.bt);
        class_transpose<T><<<dim3((unsigned)tiles_of(ldrt, 64), (unsigned)tiles_of(D, 64)), dim3(256), 0, st>>>(x, c.ldx, N, D, l.y, xt,
                                                                                                              ldrt);
        l.lse = lse;
        l.lpbar = c.lpbar ? (const A*)c.lpbar + n0 : nullptr;
        l.r = r;
        l.rt = rt;
        l.ldrt = ldrt;
        l.part_alpha = c.alphabar ? (A*)(ws + p.part_alpha) : nullptr;
        for (int64_t v0 = 0; v0 < V; v0 += p.piece) {
            const int64_t nv = V - v0 < p.piece ? V - v0 : p.piece;
            const bool first = v0 == 0, last = v0 + nv == V;
            l.beta = {beta.p + v0 * beta.ld, beta.ld, nv};
            l.alpha = c.alpha ? (const T*)c.alpha + v0 : nullptr;
            l.v0 = v0;
            l.ldr = up_to(nv, edge);
            logits_any<T>(l, use_wide, false, st);
            class_transpose<T><<<dim3((unsigned)tiles_of(l.ldr, 64), (unsigned)tiles_of(D, 64)), dim3(256), 0, st>>>(
                (const T*)c.beta + v0 * c.ldbeta, c.ldbeta, nv, D, nullptr, bt, l.ldr);
            if (c.alphabar)
                class_alpha<T><<<dim3((unsigned)tiles_of(nv, 64)), dim3(256), 0, st>>>(
                    l.part_alpha, tiles_of(N, edge), l.ldr, nv, (A*)(ws + p.alpha_acc) + v0, !first_block,
                    last_block ? (T*)c.alphabar + v0 : nullptr);
            if ((e = hipGetLastError()) != hipSuccess) return e;
            ProductArgs<T> x_ = {}, b_ = {};
            x_.A = {bt, l.ldr, D};
            x_.B = {r, l.ldr, N};
            x_.K = l.ldr;
            x_.acc = (A*)(ws + p.xacc);
            x_.plane = p.block * D;
            x_.add = !first;
            x_.y = l.y;
            x_.lpbar = l.lpbar;
            if ((e = product<T>(x_, p.xsplits, last, (T*)c.xbar + n0 * D, st)) != hipSuccess) return e;
            b_.A = {xt, ldrt, D};
            b_.B = {rt, ldrt, nv};
            b_.K = ldrt;
            b_.acc = (A*)(ws + p.bacc) + (p.blocks > 1 ? v0 * D : 0);
            b_.plane = (p.blocks > 1 ? V : p.piece) * D;
            b_.add = !first_block;
            b_.largest = largest;
            if ((e = product<T>(b_, p.bsplits, last_block, (T*)c.betabar + v0 * D, st)) != hipSuccess) return e;
        }
    }
    return hipSuccess;
}

} // namespace

size_t gpt_class_workspace(int dtype, int64_t rows, int64_t features, int64_t classes, bool vjp) {
    if (gpt_class_narrow(dtype, rows, features, classes)) return gpt_class_narrow_workspace(dtype, rows, features, classes, vjp);
    switch (dtype) {
    case GPT_F64: return space<double>(rows, features, classes, vjp);
    case GPT_F32: return space<float>(rows, features, classes, vjp);
    case GPT_F16: return space<half_t>(rows, features, classes, vjp);
    default: return space<bf16_t>(rows, features, classes, vjp);
    }
}
hipError_t gpt_launch_class(int dtype, const ClassArgs& a, bool vjp, hipStream_t st) {
    if (gpt_class_narrow(dtype, a.rows, a.features, a.classes)) return gpt_launch_class_narrow(dtype, a, vjp, st);
    switch (dtype) {
    case GPT_F64: return launch<double>(a, vjp, st);
    case GPT_F32: return launch<float>(a, vjp, st);
    case GPT_F16: return launch<half_t>(a, vjp, st);
    default: return launch<bf16_t>(a, vjp, st);
    }
}
