// Log probability of observed classes under a linear read-out, and its reverse mode (gpt_categorical_logit_glm_lpmf, _vjp):
//
//   eta[n][v] = alpha[v] + beta[v] . x[n],  lse[n] = log sum_v exp eta[n][v],  lp[n] = eta[n][y[n]] - lse[n]
//   r[n][v] = lpbar[n] ([v = y[n]] - exp(eta[n][v] - lse[n])),  xbar = r beta,  alphabar = sum_n r,  betabar = r^T x
//
// Two passes over the classes. The first leaves a maximum and a sum for every row and tile of classes; the second takes a piece of
// the classes at a time and turns its logits into the piece's r in a workspace of bounded size, from which two more matrix
// products take xbar and betabar. Of the logits a bounded part is kept from the first pass (the tiles' registers as they are, up to
// KEPT_BYTES), the rest is computed again. r is written in both orders, so that what a product sums over stands contiguously in it; of beta
// and x, whose sums run down their columns there, the large tiles take transposed reads from LDS (for 65 rows x 4096 x 32000 in bf16 a
// transposed copy of beta cost 400 us against 301), the small one transposed copies.
//
// What bounds it are the matrix cores: 4096 rows (3892 observed) x 4096 features x 128000 classes in bf16 take 12.1 to 12.5 ms, 1.14
// PFLOP/s in the first sweep's logits and 1.19 in the products, at the 1.85-1.9 GHz that the power leaves (matrix cores 63 % busy).
//
// Sums, statistics and accumulators are Acc (fp32; fp64 for fp64 data). One intermediate is rounded to 16 bits where the data
// have 16 bits: r, because the matrix instructions take both operands in one type. Its error (half a step of each entry) is
// independent from entry to entry, and no larger than that of rounding the result. The rows' cotangents stay out of that
// rounding where they can: for xbar they multiply the product's Acc rows, for betabar (whose sum runs over the rows) r
// holds them divided by the largest of them, so that cotangents that are all alike (a sum's, a mean's) leave [v = y] exact. fp16
// has too few exponents for the small probabilities of a large vocabulary: there r is stored times 2^14. Large products of fp32 data
// run on the bf16 matrix cores, each value split in three (gpt_tile.h): six bf16 products, which take a little over half the time
// of the fp32 instructions' one, at fp32's precision.
//
// Rows without an observation cost nothing: the others are numbered first (class_index), and their x copied side by side; all
// that follows counts in those numbers, up to a count that only the device knows.
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
template <typename T> struct LogitArgs {
    typedef typename T::Element E;
    typedef typename T::Acc A;
    Operand<E> beta, x; // beta: the classes from v0 on; x: the observed rows (x.rows: the most there can be)
    const int* count;   // observed rows
    const typename T::Data* alpha; // from v0 on, or null
    int64_t features, v0, classes; // features: k of the operands; classes: all of them
    const int* y;                  // class of an observed row; `classes` or more: none such
    const int* row;                // its row
    int64_t tiles_v;
    // statistics
    A *part_max, *part_sum, *eta_y; // [tiles_v][rows], [tiles_v][rows], [rows]
    // r, and r with the rows' cotangents in the other order: [rows][ldr] and [classes of the piece][ldrt], in whole tiles
    const RowSum<A>* of;
    const A* lpbar; // of all rows
    E *r, *rt;
    int64_t ldr, ldrt, r_plane, rt_plane;
    A* part_alpha; // [tiles_n][ldr] or null
    Largest<A> largest;
    // logits of the first kept_classes classes, as the first sweep leaves them for the second: tile by tile, a lane's fragments
    typename T::Tl::C* kept;
    int64_t kept_classes;
    // ... or, if the first sweep's tiles are few, shares of k that are added up then: [splits] of those, `plane` apart
    int64_t splits, plane, grid; // grid: workgroups of one share
};

// One way to run the products: data type, tile, type and number of planes of its operands
template <typename T, typename Tl_, int PLANES_> struct Way {
    typedef T Data;
    typedef acc_t<T> Acc;
    typedef Tl_ Tl;
    typedef typename TurnedOf<Tl>::Tile Product; // of the products with r
    typedef typename Tl::Element Element;
    static constexpr int PLANES = PLANES_;
    static constexpr bool LINES = Tl::TN == 4 && !std::is_same<Tl, SmallTile<T>>::value; // a LineTile
};

// Two values in one word (plane p of them)
template <typename W> __device__ __forceinline__ void words(float a, float b, uint32_t (&u)[W::PLANES]) {
    if constexpr (W::PLANES == 3) {
        split3(a, b, u);
    } else u[0] = pack2<typename W::Element>(a, b);
}

// Tiles of eta, classes x rows. STATS: each tile's maximum and sum of exponentials for every row. else: r. KEPT: eta was kept (STATS: the
// shares of class_partial).
template <typename W> struct LogitRoom { // LDS
    typedef typename W::Acc A;
    typedef typename W::Tl Tl;
    A red[2][Tl::WM > Tl::WN ? Tl::WM : Tl::WN][Tl::BM > Tl::BN ? Tl::BM : Tl::BN];
    A al[Tl::BM], top[Tl::BN], share[Tl::BN], w[Tl::BN];
    int at[Tl::BN];
};
template <typename W, typename Tl, bool STATS, bool KEPT>
__device__ __forceinline__ void logits_tile(LogitArgs<W> a, int64_t rows, int64_t tm, int64_t tn, LogitRoom<W>& room, typename Tl::Vec* lds) {
    typedef typename W::Acc A;
    const int64_t ld = a.x.rows, m0 = tm * W::Tl::BM, n0 = tn * W::Tl::BN;
    const int nv = (int)(a.beta.rows - m0 < Tl::BM ? a.beta.rows - m0 : Tl::BM); // classes of this tile
    // what the tile's classes and rows need besides, on its way into LDS while the product runs (which ends with a barrier)
    A largest = 1;
    if (!STATS) largest = a.largest.get();
    for (int c = threadIdx.x; (STATS || !KEPT) && c < Tl::BM; c += Tl::THREADS)
        room.al[c] = c < nv ? (a.alpha ? level_log2e((A)a.alpha[m0 + c]) : (A)0) : neg_inf<A>();
    for (int c = threadIdx.x; c < Tl::BN; c += Tl::THREADS) {
        const int64_t n = n0 + c, y = n < rows ? a.y[n] : -1, from = y - (a.v0 + m0);
        room.at[c] = y >= 0 && from >= 0 && from < nv ? (int)from : -1; // the row's class within the tile
        if (!STATS) {
            const RowSum<A> of = y < 0 ? RowSum<A>{(A)__builtin_inf(), (A)0} : a.of[n]; // (behind the last row: none)
            const bool none = of.share == 0;
            room.top[c] = of.top;
            room.share[c] = stored_scale<typename W::Data>() * of.share;
            room.w[c] = none ? (A)0 : a.lpbar ? a.lpbar[a.row[n]] / largest : (A)1;
        }
    }
    a.x.rows = rows;
    const int lane = threadIdx.x & 63, wm = (threadIdx.x >> 6) / Tl::WN, wn = (threadIdx.x >> 6) % Tl::WN;
    const int64_t kept_tile = (a.v0 + m0) / Tl::BM * ((ld + W::Tl::BN - 1) / W::Tl::BN) + tn;
    auto* kept = a.kept + kept_tile * (W::Tl::TM * W::Tl::TN * W::Tl::THREADS) + threadIdx.x;
    Tl tl;
    if constexpr (KEPT) {
#pragma unroll
        for (int i = 0; i < Tl::TM; ++i)
#pragma unroll
            for (int j = 0; j < Tl::TN; ++j) tl.acc[i][j] = kept[(i * Tl::TN + j) * Tl::THREADS];
#pragma unroll 2
        for (int64_t k = 1; STATS && k < a.splits; ++k)
#pragma unroll
            for (int i = 0; i < Tl::TM; ++i)
#pragma unroll
                for (int j = 0; j < Tl::TN; ++j) tl.acc[i][j] += kept[k * a.plane + (i * Tl::TN + j) * Tl::THREADS];
        __syncthreads();
    } else tl.run(a.beta, m0, a.x, n0, 0, a.features, lds);
    if (STATS || !KEPT) {
#pragma unroll
        for (int i = 0; i < Tl::TM; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const A v = room.al[Tl::row(i, r)];
#pragma unroll
                for (int j = 0; j < Tl::TN; ++j) tl.acc[i][j][r] = times_log2e(tl.acc[i][j][r]) + v;
            }
    }
    if (STATS && m0 < a.kept_classes) {
#pragma unroll
        for (int i = 0; i < Tl::TM; ++i)
#pragma unroll
            for (int j = 0; j < Tl::TN; ++j) kept[(i * Tl::TN + j) * Tl::THREADS] = tl.acc[i][j];
    }
    if (STATS) {
#pragma unroll
        for (int j = 0; j < Tl::TN; ++j) {
            const int at = room.at[Tl::col(j)];
            A mx = neg_inf<A>();
#pragma unroll
            for (int i = 0; i < Tl::TM; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmax(mx, tl.acc[i][j][r]);
            if (at >= 0 && Tl::holds(at)) { // (few tiles hold a row's class)
                A here = 0;
#pragma unroll
                for (int i = 0; i < Tl::TM; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) here = Tl::row(i, r) == at ? tl.acc[i][j][r] : here;
                a.eta_y[n0 + Tl::col(j)] = here;
            }
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
                room.red[0][wm][Tl::col(j)] = mx;
                room.red[1][wm][Tl::col(j)] = s;
            }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < Tl::BN; c += Tl::THREADS) {
            A mx = room.red[0][0][c], s = room.red[1][0][c];
#pragma unroll
            for (int w = 1; w < Tl::WM; ++w) join(mx, s, room.red[0][w][c], room.red[1][w][c]);
            if (n0 + c < rows) {
                a.part_max[tm * ld + n0 + c] = mx;
                a.part_sum[tm * ld + n0 + c] = s;
            }
        }
        return;
    }
    A top[Tl::TN], share[Tl::TN], w[Tl::TN];
    int at[Tl::TN];
#pragma unroll
    for (int j = 0; j < Tl::TN; ++j) {
        top[j] = room.top[Tl::col(j)];
        share[j] = room.share[Tl::col(j)];
        w[j] = room.w[Tl::col(j)];
        at[j] = share[j] == 0 ? -1 : room.at[Tl::col(j)];
    }
    constexpr A up = stored_scale<typename W::Data>();
    A total[Tl::TM][4];
#pragma unroll
    for (int i = 0; i < Tl::TM; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            total[i][r] = 0;
#pragma unroll
            for (int j = 0; j < Tl::TN; ++j) {
                const A v = (Tl::row(i, r) == at[j] ? up : (A)0) - share[j] * exp_log2e(tl.acc[i][j][r] - top[j]);
                tl.acc[i][j][r] = v;
                total[i][r] += v * w[j];
            }
        }
    if constexpr (W::LINES) {
        // r: 16 neighbouring classes of one row a lane; rt: after the transpose, 16 neighbouring rows of one class a lane
        const int64_t mq = m0 + Tl::row(0, 0), nq = n0 + Tl::col(0);
#pragma unroll
        for (int j = 0; j < Tl::TN; ++j)
#pragma unroll
            for (int h = 0; h < Tl::TM / 4; ++h)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    uint32_t u[4][W::PLANES];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const auto& c = tl.acc[4 * h + 2 * k + e / 2][j];
                        words<W>(c[2 * (e & 1)], c[2 * (e & 1) + 1], u[e]);
                    }
#pragma unroll
                    for (int p = 0; p < W::PLANES; ++p)
                        *reinterpret_cast<uint4*>(a.r + p * a.r_plane + (nq + Tl::fragment(j)) * a.ldr + mq + 64 * h + 8 * k) =
                            make_uint4(u[0][p], u[1][p], u[2][p], u[3][p]);
                }
        const int64_t nb = nq - (lane & 3), mb = mq + (lane & 3);
#pragma unroll
        for (int i = 0; i < Tl::TM; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t lo[2][W::PLANES], hi[2][W::PLANES];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int j = 2 * h + e;
                    const auto& c = tl.acc[i][j];
                    words<W>(c[0] * w[j], c[1] * w[j], lo[e]);
                    words<W>(c[2] * w[j], c[3] * w[j], hi[e]);
                }
#pragma unroll
                for (int p = 0; p < W::PLANES; ++p) {
                    transpose4(lo[0][p], hi[0][p]);
                    transpose4(lo[1][p], hi[1][p]);
                    *reinterpret_cast<uint4*>(a.rt + p * a.rt_plane + (mb + Tl::fragment(i)) * a.ldrt + nb + 8 * h) =
                        make_uint4(lo[0][p], hi[0][p], lo[1][p], hi[1][p]);
                }
            }
    } else {
#pragma unroll
        for (int i = 0; i < Tl::TM; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < Tl::TN; ++j) {
                    const int64_t m = m0 + Tl::row(i, r), n = n0 + Tl::col(j);
                    a.r[n * a.ldr + m] = (typename W::Element)tl.acc[i][j][r];
                    a.rt[m * a.ldrt + n] = (typename W::Element)(tl.acc[i][j][r] * w[j]);
                }
    }
    if (!a.part_alpha) return;
#pragma unroll
    for (int i = 0; i < Tl::TM; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const A s = sum16(total[i][r]);
            if ((lane & 15) == 0) room.red[0][wn][Tl::row(i, r)] = s;
        }
    __syncthreads();
    for (int c = threadIdx.x; c < nv; c += Tl::THREADS) {
        A s = room.red[0][0][c];
#pragma unroll
        for (int k = 1; k < Tl::WN; ++k) s += room.red[0][k][c];
        a.part_alpha[tn * a.ldr + m0 + c] = s * (largest / up);
    }
}
template <typename W, bool STATS, bool KEPT> __global__ __launch_bounds__(W::Tl::THREADS, 2) void class_logits(LogitArgs<W> a) {
    typedef typename W::Tl Tl;
    typedef typename HalfOf<Tl>::Tile Half;
    __shared__ typename Tl::Vec lds[KEPT ? 1 : Tl::LDS_BYTES / 16];
    __shared__ LogitRoom<W> room;
    const int64_t rows = *a.count;
    int64_t tm, tn;
    bool half;
    if (!tile_place<Tl>(wide_block(), a.tiles_v, rows, tm, tn, half)) return;
    if constexpr (!std::is_void<Half>::value) {
        if (half) {
            logits_tile<W, Half, STATS, KEPT>(a, rows, tm, tn, room, lds);
            return;
        }
    }
    logits_tile<W, Tl, STATS, KEPT>(a, rows, tm, tn, room, lds);
}

// A share of k's part of eta's tiles, as they are
template <typename W> __global__ __launch_bounds__(W::Tl::THREADS, 2) void class_partial(LogitArgs<W> a) {
    typedef typename W::Tl Tl;
    __shared__ typename Tl::Vec lds[Tl::LDS_BYTES / 16];
    const int64_t ld = a.x.rows, split = blockIdx.x / a.grid, step = tile_k<typename W::Element>();
    a.x.rows = *a.count;
    int64_t tm, tn;
    bool half;
    const int64_t in = split_place(blockIdx.x - split * a.grid, split, a.tiles_v * ((a.x.rows + Tl::BN - 1) / Tl::BN));
    if (!tile_place<Tl>(in, a.tiles_v, a.x.rows, tm, tn, half)) return;
    const int64_t share = ((a.features + a.splits - 1) / a.splits + step - 1) / step * step;
    const int64_t k0 = split * share, k1 = k0 + share < a.features ? k0 + share : a.features;
    Tl tl;
    tl.run(a.beta, tm * Tl::BM, a.x, tn * Tl::BN, k0, k1, lds);
    auto* to = a.kept + split * a.plane + (tm * ((ld + Tl::BN - 1) / Tl::BN) + tn) * (Tl::TM * Tl::TN * Tl::THREADS) + threadIdx.x;
#pragma unroll
    for (int i = 0; i < Tl::TM; ++i)
#pragma unroll
        for (int j = 0; j < Tl::TN; ++j) to[(i * Tl::TN + j) * Tl::THREADS] = tl.acc[i][j];
}

__host__ __device__ __forceinline__ int64_t tiles_up(int64_t n, int64_t b) { return (n + b - 1) / b; }

// The observed rows of x side by side, as operands (zeros behind their features); zeros into xbar's other rows
template <typename W> struct GatherArgs {
    const typename W::Data* x;
    int64_t ld, rows, cols;
    const int* place; // null: all rows
    typename W::Element* out;
    int64_t ldo, plane;
    typename W::Data* xbar;
    const int* count; // rows of out (null: rows), which zeros fill up to a multiple of 64 where a product runs along them
};
template <typename W> __device__ __forceinline__ void gather(const GatherArgs<W>& a, int64_t block, int64_t blocks) {
    typedef typename W::Data T;
    constexpr int N = 8;
    const T* x = a.x;
    const int64_t ld = a.ld, rows = a.rows, cols = a.cols, ldo = a.ldo, plane = a.plane, per = ldo / N, total = rows * per;
    const int* place = a.place;
    T* xbar = a.xbar;
    if (W::LINES) {
        const int64_t from = a.count ? *a.count : rows, more = (tiles_up(from, 64) * 64 - from) * per;
        for (int64_t i = block * 256 + threadIdx.x; i < more; i += blocks * 256)
#pragma unroll
            for (int p = 0; p < W::PLANES; ++p) *reinterpret_cast<uint4*>(a.out + p * plane + from * ldo + i * N) = make_uint4(0, 0, 0, 0);
    }
    for (int64_t i = block * 256 + threadIdx.x; i < total; i += blocks * 256) {
        const int64_t r = i / per, k = (i - r * per) * N;
        const int at = place ? place[r] : (int)r;
        if (at < 0) {
            if (xbar)
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (k + e < cols) xbar[r * cols + k + e] = (T)0;
            continue;
        }
        T v[N];
#pragma unroll
        for (int h = 0; h < N; h += Vec16<T>::N) {
            const auto u = tile_chunk<T>({x, ld, rows}, r, k + h, cols);
#pragma unroll
            for (int e = 0; e < Vec16<T>::N; ++e) v[h + e] = u[e];
        }
        typename W::Element* to = a.out + at * ldo + k;
        if constexpr (W::PLANES == 3) {
            uint32_t u[N / 2][3];
#pragma unroll
            for (int e = 0; e < N / 2; ++e) split3(v[2 * e], v[2 * e + 1], u[e]);
#pragma unroll
            for (int p = 0; p < 3; ++p) *reinterpret_cast<uint4*>(to + p * plane) = make_uint4(u[0][p], u[1][p], u[2][p], u[3][p]);
        } else {
#pragma unroll
            for (int h = 0; h < N; h += Vec16<T>::N) {
                typename Vec16<T>::V u;
#pragma unroll
                for (int e = 0; e < Vec16<T>::N; ++e) u[e] = v[h + e];
                *reinterpret_cast<typename Vec16<T>::V*>(to + h) = u;
            }
        }
    }
}

// The sums and lp of 8 observed rows from their tiles' statistics, 32 slices of the tiles in parallel
template <typename A> __global__ __launch_bounds__(256) void class_join(const A* part_max, const A* part_sum, const A* eta_y, const int* y,
                                                                       const int* row, const int* count, int64_t tiles, int64_t ld,
                                                                       int64_t classes, RowSum<A>* of, A* lp) {
    __shared__ A red[2][32][9];
    const int c = threadIdx.x & 7, k = threadIdx.x >> 3;
    const int64_t n = (int64_t)blockIdx.x * 8 + c, rows = *count;
    if ((int64_t)blockIdx.x * 8 >= rows) return;
    A mx = neg_inf<A>(), s = 0;
    if (n < rows) {
        int64_t i = k;
        for (; i + 96 < tiles; i += 128) {
            A m[4], t[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                m[u] = part_max[(i + 32 * u) * ld + n];
                t[u] = part_sum[(i + 32 * u) * ld + n];
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) join(mx, s, m[u], t[u]);
        }
        for (; i < tiles; i += 32) join(mx, s, part_max[i * ld + n], part_sum[i * ld + n]);
    }
    red[0][k][c] = mx;
    red[1][k][c] = s;
    __syncthreads();
    if (k || n >= rows) return;
    for (int i = 1; i < 32; ++i) join(mx, s, red[0][i][c], red[1][i][c]);
    const int64_t yn = y[n];
    lp[row[n]] = row_lp(yn, classes, mx, s, yn < classes ? eta_y[n] : (A)0);
    if (of) of[n] = row_sum_of(yn, classes, mx, s);
}

// out[c][r] = in[row[r]][c] as operands (row null: r itself), zeros behind the last row up to ldo. 64 x 64 through LDS; each side in
// vectors of eight
template <typename W> struct TransposeArgs {
    const typename W::Data* in;
    int64_t ld, rows;
    const int* count; // null: rows
    int64_t cols;
    const int* row; // null: as they come
    typename W::Element* out;
    int64_t ldo, plane;
};
template <typename W> __device__ __forceinline__ void transpose(const TransposeArgs<W>& t, int64_t block) {
    typedef typename W::Data T;
    __shared__ T tile[64][66];
    const int64_t across = (t.ldo + 63) / 64, r0 = block % across * 64, c0 = block / across * 64;
    const T* in = t.in;
    const int64_t ld = t.ld, rows = t.count ? *t.count : t.rows, cols = t.cols, ldo = t.ldo, plane = t.plane;
    const int* row = t.row;
    typename W::Element* out = t.out;
    const int a = threadIdx.x >> 3, b = 8 * (threadIdx.x & 7);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int64_t r = r0 + a + 32 * h;
        const T* from = r < rows ? in + (row ? row[r] : r) * ld : nullptr;
#pragma unroll
        for (int k = 0; k < 8; k += Vec16<T>::N) {
            typename Vec16<T>::V v = {};
            if (from) v = tile_chunk<T>({from, ld, 1}, 0, c0 + b + k, cols);
#pragma unroll
            for (int e = 0; e < Vec16<T>::N; ++e) tile[a + 32 * h][b + k + e] = v[e];
        }
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int64_t c = c0 + a + 32 * h, r = r0 + b;
        if (c >= cols || r >= ldo) continue;
        typename W::Element* to = out + c * ldo + r;
        if constexpr (W::PLANES == 3) {
            uint32_t u[4][3];
#pragma unroll
            for (int e = 0; e < 4; ++e) split3(tile[b + 2 * e][a + 32 * h], tile[b + 2 * e + 1][a + 32 * h], u[e]);
#pragma unroll
            for (int p = 0; p < 3; ++p) *reinterpret_cast<uint4*>(to + p * plane) = make_uint4(u[0][p], u[1][p], u[2][p], u[3][p]);
        } else {
#pragma unroll
            for (int k = 0; k < 8; k += Vec16<T>::N) {
                typename Vec16<T>::V u;
#pragma unroll
                for (int e = 0; e < Vec16<T>::N; ++e) u[e] = tile[b + k + e][a + 32 * h];
                *reinterpret_cast<typename Vec16<T>::V*>(to + k) = u;
            }
        }
    }
}

// All that is copied before the logits, in one launch: the workgroups up to end[k] do part k. end[0], end[1]: x side by side, and beta
// with rows that start on 16 bytes (gather); end[2], end[3]: the transposes of x and of beta's first piece for the small tile
template <typename W> struct PrepareArgs {
    GatherArgs<W> g[2];
    TransposeArgs<W> t[2];
    int end[4];
};
template <typename W> __global__ __launch_bounds__(256) void class_prepare(PrepareArgs<W> a) {
    const int id = blockIdx.x;
    if (id < a.end[0]) gather<W>(a.g[0], id, a.end[0]);
    else if (id < a.end[1]) gather<W>(a.g[1], id - a.end[0], a.end[1] - a.end[0]);
    else if (id < a.end[2]) transpose<W>(a.t[0], id - a.end[1]);
    else transpose<W>(a.t[1], id - a.end[2]);
}

// The products with r: out[n][m] = sum_k A[m][k] B[n][k] over this launch's share of k.
template <typename T, typename E> struct ProductArgs {
    typedef acc_t<T> Acc;
    Operand<E> A, B;
    int64_t K;        // (betabar: the observed rows', rounded up to k_edge)
    int64_t k_edge;
    const int* count; // observed rows: B's rows (xbar), or k (betabar)
    int64_t tiles_m, splits, grid; // grid: workgroups of one split
    Acc* acc;      // [splits][B.rows][A.rows]: sums so far
    int64_t plane; // elements from one split's sums to the next
    T* out;        // the result, where this launch completes it; else null
    int64_t ldo;
    bool add; // acc holds earlier launches' sums
    // xbar: B's rows are the observed rows, each times its cotangent, and go where row says. betabar: row null
    const int* row;
    const Acc* lpbar;
    Largest<Acc> largest;
};
template <typename W, typename Tl>
__device__ __forceinline__ void product_at(const ProductArgs<typename W::Data, typename W::Element>& a, int64_t split, int64_t tm, int64_t tn,
                                           typename Tl::Vec* lds) {
    typedef typename W::Acc A;
    typedef typename W::Data T;
    const int64_t m0 = tm * W::Tl::BM, n0 = tn * W::Tl::BN, step = tile_k<typename W::Element>();
    const int64_t share = ((a.K + a.splits - 1) / a.splits + step - 1) / step * step;
    const int64_t k0 = split * share, k1 = k0 + share < a.K ? k0 + share : a.K;
    Tl tl;
    tl.run(a.A, m0, a.B, n0, k0, k1, lds);
    A* acc = a.acc + split * a.plane;
    const A largest = a.row ? (A)1 : a.largest.get();
#pragma unroll
    for (int j = 0; j < Tl::TN; ++j) {
        const int64_t n = n0 + Tl::col(j);
        if (n >= a.B.rows) continue;
        const int64_t to = a.row ? a.row[n] : n;
        const A back = (a.row && a.lpbar ? a.lpbar[to] : largest) / (A)stored_scale<T>();
        if constexpr (W::LINES) { // four neighbouring values a lane
#pragma unroll
            for (int i = 0; i < Tl::TM; ++i) {
                const int64_t m = m0 + Tl::row(i, 0);
                A v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = tl.acc[i][j][r] * back;
                A* s = acc + n * a.A.rows + m;
                T* o = a.out + to * a.ldo + m;
                if (m + 4 <= a.A.rows) {
                    if (a.add) {
                        const auto u = load16(s);
#pragma unroll
                        for (int r = 0; r < 4; ++r) v[r] += u[r];
                    }
                    if (a.out) {
                        const T u[4] = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
                        store4(o, u);
                    } else store4(s, v);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        if (m + r >= a.A.rows) continue;
                        if (a.add) v[r] += s[r];
                        if (a.out) o[r] = (T)v[r];
                        else s[r] = v[r];
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
                    A v = tl.acc[i][j][r] * back;
                    if (a.add) v += acc[n * a.A.rows + m];
                    if (a.out) a.out[to * a.ldo + m] = (T)v;
                    else acc[n * a.A.rows + m] = v;
                }
        }
    }
}
template <typename W> __device__ __forceinline__ void product_tile(ProductArgs<typename W::Data, typename W::Element> a, int64_t id,
                                                                   typename W::Tl::Vec* lds) {
    typedef typename W::Product Tl;
    typedef typename HalfOf<Tl>::Tile Half;
    const int64_t split = id / a.grid;
    if (a.row) a.B.rows = *a.count;
    else a.K = (*a.count + a.k_edge - 1) / a.k_edge * a.k_edge;
    int64_t tm, tn;
    bool half;
    const int64_t in = split_place(id - split * a.grid, split, a.tiles_m * ((a.B.rows + Tl::BN - 1) / Tl::BN));
    if (!tile_place<Tl>(in, a.tiles_m, a.B.rows, tm, tn, half)) return;
    if constexpr (!std::is_void<Half>::value) {
        if (half) {
            product_at<W, Half>(a, split, tm, tn, lds);
            return;
        }
    }
    product_at<W, Tl>(a, split, tm, tn, lds);
}
// alphabar of a piece from the tiles' sums, 64 classes a wave, or a workgroup whose waves share the tiles where these are many.
// acc: sums over row blocks
template <typename T> struct AlphaArgs {
    const acc_t<T>* part;
    const int* count;
    int64_t edge, ld, nv;
    bool shared;
    acc_t<T>* acc;
    bool add;
    T* out;
};
template <typename T, int WAVES> __device__ __forceinline__ void alpha_sums(const AlphaArgs<T>& a, int64_t block, acc_t<T>* red) {
    typedef acc_t<T> A;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t v = (a.shared ? block : block * WAVES + w) * 64 + lane, tiles = (*a.count + a.edge - 1) / a.edge;
    A s = 0;
    if (v < a.nv) {
#pragma unroll 4
        for (int64_t i = a.shared ? w : 0; i < tiles; i += a.shared ? WAVES : 1) s += a.part[i * a.ld + v];
    }
    if (a.shared) {
        red[w * 64 + lane] = s;
        __syncthreads();
        if (w) return;
#pragma unroll
        for (int k = 1; k < WAVES; ++k) s += red[k * 64 + lane];
    }
    if (v >= a.nv) return;
    if (a.add) s += a.acc[v];
    if (a.out) a.out[v] = (T)s;
    else a.acc[v] = s;
}
// Both products with r, and alphabar, in one launch where they run the same way: the workgroups up to end[0] take xbar, those up to
// end[1] betabar, the others alphabar
template <typename W> struct ProductsArgs {
    ProductArgs<typename W::Data, typename W::Element> x, b;
    AlphaArgs<typename W::Data> alpha;
    int end[2];
};
template <typename W> __global__ __launch_bounds__(W::Tl::THREADS, 2) void class_products(ProductsArgs<W> a) {
    typedef typename W::Product Tl;
    __shared__ typename Tl::Vec lds[Tl::LDS_BYTES / 16];
    const int id = blockIdx.x;
    if (id < a.end[1]) { // (one call: the tile's code stands once)
        const bool x = id < a.end[0];
        product_tile<W>(x ? a.x : a.b, x ? id : id - a.end[0], lds);
    } else alpha_sums<typename W::Data, Tl::THREADS / 64>(a.alpha, id - a.end[1], reinterpret_cast<typename W::Acc*>(lds));
}

// out[row[n]][0..cols) <- sum over the splits (row null: all `rows` rows, else the observed ones)
template <typename T> struct SplitsArgs {
    const acc_t<T>* acc;
    int splits;
    int64_t plane, rows, cols;
    const int *count, *row;
    T* out;
};
template <typename T> __device__ __forceinline__ void join_splits(const SplitsArgs<T>& a, int64_t block) {
    const int64_t i = block * 256 + threadIdx.x;
    if (i >= (a.row ? *a.count : a.rows) * a.cols) return;
    acc_t<T> s = 0;
#pragma unroll 4
    for (int k = 0; k < a.splits; ++k) s += a.acc[k * a.plane + i];
    const int64_t n = i / a.cols;
    a.out[a.row ? a.row[n] * a.cols + (i - n * a.cols) : i] = (T)s;
}
template <typename T> __global__ __launch_bounds__(256) void class_join_splits(SplitsArgs<T> x, SplitsArgs<T> b, int64_t end) {
    if (blockIdx.x < end) join_splits<T>(x, blockIdx.x);
    else join_splits<T>(b, blockIdx.x - end);
}

// ---- plan -------------------------------------------------------------------------------------------------------------
int64_t up_to(int64_t n, int64_t m) { return (n + m - 1) / m * m; }
int64_t tiles_of(int64_t n, int64_t b) { return (n + b - 1) / b; }

constexpr int64_t ROW_BLOCK = 1 << 18;              // rows taken at a time
constexpr int64_t PIECE_BYTES = (int64_t)512 << 20; // r in both orders, of a piece of the classes and a block of the rows
constexpr int64_t KEPT_BYTES = (int64_t)1 << 30;    // logits kept from the first sweep for the second
constexpr int64_t FILL = 512;                       // workgroups that fill the card
constexpr int64_t WIDE_TILES = 192;                 // 256 x 256 tiles from this many on

// Splits of a product's k: enough workgroups to fill the card, at least 4 steps of k each
int64_t splits_of(int64_t tiles, int64_t K, int64_t step) {
    int64_t s = FILL / tiles;
    const int64_t most = K / (4 * step);
    if (s > most) s = most;
    return s < 1 ? 1 : s > 64 ? 64 : s;
}
// Shares of k of the first sweep's tiles where these are few: at least 24 steps of k each, 16 of the fp32 instructions', 8 of fp64's (fp32 65 rows x 4000 x 8000 170 us
// against 308, fp64 500 x 500 x 2000 71 against 100; but fp32 1000 x 500 x 1500 in five shares 53 against 48)
template <typename E> int64_t logit_splits(int64_t tiles, int64_t K) {
    return tiles < FILL / 2 ? splits_of(tiles, K, (sizeof(E) == 8 ? 2 : sizeof(E) == 4 ? 4 : 6) * tile_k<E>()) : 1;
}
// 256 x 256 tiles for a product of m x n results?
bool wide(int64_t m, int64_t n) { return tiles_of(m, 256) * tiles_of(n, 256) >= WIDE_TILES; }

// Features from which writing a logit and reading it again takes less time than computing it again. With and without, in us: bf16 4096 x
// 32000, 512 features 763 / 724, 1024 features 1125 / 1188; fp32 100 features (2000 x 8000) 205 / 194, 270 (275 x 13636) 192 / 215; fp64
// 100 (2000 x 2000) 194 / 211
template <typename T> constexpr int64_t keep_features() { return sizeof(T) == 2 ? 768 : sizeof(T) == 4 ? 160 : 64; }

// W: the way of the logits. The products with r take the larger tile or the smaller by themselves
template <typename W> struct Plan {
    typedef typename W::Data T;
    typedef typename W::Element E;
    static constexpr int64_t EDGE = W::Tl::BM;
    int64_t block, blocks, piece, pieces, tiles_v, tiles_n, ldr, ldrt, ldk, xrows, brows;
    int64_t lsplits, xsplits, bsplits, kept_pieces;
    bool wide_products; // wide tiles for xbar and betabar
    bool copy;         // beta as operands of its own
    // offsets in bytes
    size_t kept, place, row, y, count, runs, part_max, part_sum, eta_y, of, scale, r, rt, xt, bt, part_alpha, alpha_acc, xacc, bacc, xa, ba, bytes;
    // (a product's splits of k count too: 16 large tiles with a sixteenth of a long k each fill the card as well. Fewer than nine would need
    // too many of them: bf16 200 rows x 1000 x 100000 472 us against 372 with small ones, fp32 500 x 500 x 60000 1061 against 831, but
    // 700 x 700 x 60000 1445 against 1617)
    static bool product_wide(int64_t m, int64_t n, int64_t K) {
        const int64_t tiles = tiles_of(m, 256) * tiles_of(n, 256);
        return W::LINES && tiles > 8 && tiles * splits_of(2 * tiles, K, 4 * tile_k<E>()) >= WIDE_TILES;
    }
    Plan(int64_t rows, int64_t features, int64_t classes, bool vjp) {
        const size_t A = sizeof(acc_t<T>), S = sizeof(E) * W::PLANES;
        block = rows < ROW_BLOCK ? rows : ROW_BLOCK;
        blocks = tiles_of(rows, block);
        tiles_v = tiles_of(classes, EDGE);
        tiles_n = tiles_of(block, EDGE);
        size_t at = 0;
        auto take = [&](size_t n) {
            const size_t p = at;
            at += (n + 255) / 256 * 256;
            return p;
        };
        place = take(4 * (size_t)block);
        row = take(4 * (size_t)block);
        y = take(4 * (size_t)block);
        count = take(4);
        runs = take(4 * (size_t)tiles_of(block, INDEX_ROWS));
        part_max = take(A * (size_t)(tiles_v * block));
        part_sum = take(A * (size_t)(tiles_v * block));
        eta_y = take(A * (size_t)block);
        ldk = up_to(features, tile_k<E>());
        xrows = up_to(block, 64);
        brows = up_to(classes, 64);
        xa = take(S * (size_t)(xrows * ldk));
        copy = W::PLANES == 3 || (W::LINES && features * sizeof(T) % 16);
        if (copy) ba = take(S * (size_t)(brows * ldk));
        const int64_t tiles = tiles_v * tiles_n;
        lsplits = std::is_void<typename HalfOf<typename W::Tl>::Tile>::value ? logit_splits<E>(tiles, (W::PLANES == 3 ? 6 : 1) * features) : 1;
        kept_pieces = 0;
        if (lsplits > 1) kept = take((size_t)(lsplits * tiles * EDGE * EDGE) * A);
        if (vjp) {
            piece = PIECE_BYTES / (int64_t)(2 * S) / up_to(block, EDGE) / EDGE * EDGE;
            if (piece < EDGE) piece = EDGE;
            if (piece > up_to(classes, EDGE)) piece = up_to(classes, EDGE);
            pieces = tiles_of(classes, piece);
            piece = up_to(tiles_of(classes, pieces), EDGE); // of about the same size
            pieces = tiles_of(classes, piece);
            ldr = piece;
            ldrt = up_to(block, EDGE);
            const int64_t logits = (int64_t)A * piece * ldrt;
            kept_pieces = lsplits > 1 || features >= keep_features<T>() ? KEPT_BYTES / logits : 0;
            if (kept_pieces > pieces) kept_pieces = pieces;
            if (lsplits == 1) kept = take((size_t)(kept_pieces * logits)); // (else in the first share's place)
            of = take(2 * A * (size_t)block);
            scale = take(A * SCALE_PARTS);
            r = take(S * (size_t)(ldrt * ldr));
            rt = take(S * (size_t)(ldr * ldrt));
            xt = bt = 0;
            if (!W::LINES) {
                xt = take(S * (size_t)(features * ldrt));
                bt = take(S * (size_t)(features * ldr));
            }
            part_alpha = take(A * (size_t)(tiles_n * ldr));
            alpha_acc = blocks > 1 ? take(A * (size_t)classes) : 0;
            wide_products = product_wide(features, block, piece) && product_wide(features, piece, block);
            xsplits = product_splits(features, block, piece);
            bsplits = product_splits(features, piece, block);
            xacc = xsplits > 1 || pieces > 1 ? take(A * (size_t)(xsplits * block * features)) : 0;
            bacc = blocks > 1 ? take(A * (size_t)(bsplits * classes * features))
                              : bsplits > 1 ? take(A * (size_t)(bsplits * piece * features)) : 0;
        }
        bytes = at;
    }
    int64_t product_splits(int64_t m, int64_t n, int64_t K) const {
        const int64_t large = wide_products ? 2 : 1, edge = 128 * large;
        return splits_of(tiles_of(m, edge) * tiles_of(n, edge) * large, K, 2 * large * tile_k<E>());
    }
};

template <typename W, bool STATS, bool KEPT> void logits(LogitArgs<W> l, hipStream_t st) {
    typedef typename W::Tl Tl;
    l.tiles_v = tiles_of(l.beta.rows, Tl::BM);
    class_logits<W, STATS, KEPT><<<wide_grid(tile_grid<Tl>(l.tiles_v, l.x.rows)), dim3(Tl::THREADS), 0, st>>>(l);
}

// xbar and betabar of a piece (each complete if its `last`), alphabar (of alpha.nv classes)
template <typename W> hipError_t products(ProductsArgs<W> p, const Plan<W>& plan, bool xlast, typename W::Data* xbar, bool blast,
                                          typename W::Data* betabar, hipStream_t st) {
    typedef typename W::Data T;
    typedef typename W::Element E;
    auto ready = [](auto& q, int64_t splits, bool last, T* out) {
        q.splits = splits;
        q.out = last && splits == 1 ? out : nullptr;
        q.ldo = q.A.rows;
    };
    ready(p.x, plan.xsplits, xlast, xbar);
    ready(p.b, plan.bsplits, blast, betabar);
    auto run = [&](auto way) {
        typedef decltype(way) U;
        typedef typename U::Tl Tl;
        ProductsArgs<U> u = {p.x, p.b, p.alpha, {0, 0}};
        auto size = [](auto& q) {
            q.tiles_m = tiles_of(q.A.rows, Tl::BM);
            q.grid = tile_grid<typename U::Product>(q.tiles_m, q.B.rows);
            return (int)(q.grid * q.splits);
        };
        const int64_t alpha = p.alpha.shared ? 64 : Tl::THREADS;
        u.end[0] = size(u.x);
        u.end[1] = u.end[0] + size(u.b);
        class_products<U><<<dim3((unsigned)(u.end[1] + tiles_of(p.alpha.nv, alpha))), dim3(Tl::THREADS), 0, st>>>(u);
    };
    if constexpr (W::LINES) {
        typedef Way<T, WideTile<E, W::PLANES>, W::PLANES> Wide;
        typedef Way<T, MidTile<E, W::PLANES>, W::PLANES> Mid;
        if (plan.wide_products) run(Wide());
        else run(Mid());
    } else run(W());
    const bool xjoin = xlast && plan.xsplits > 1, bjoin = blast && plan.bsplits > 1;
    if (xjoin || bjoin) {
        auto args = [](const auto& q, T* out) {
            return SplitsArgs<T>{q.acc, (int)q.splits, q.plane, q.B.rows, q.A.rows, q.count, q.row, out};
        };
        const int64_t nx = xjoin ? tiles_of(p.x.A.rows * p.x.B.rows, 256) : 0, nb = bjoin ? tiles_of(p.b.A.rows * p.b.B.rows, 256) : 0;
        class_join_splits<T><<<dim3((unsigned)(nx + nb)), dim3(256), 0, st>>>(args(p.x, xbar), args(p.b, betabar), nx);
    }
    return hipGetLastError();
}

// (REVERSE: that mode is asked of it at all)
template <typename W, bool REVERSE = true> hipError_t launch_rows(const ClassArgs& c, bool vjp, hipStream_t st) {
    typedef typename W::Data T;
    typedef typename W::Element E;
    typedef acc_t<T> A;
    constexpr int64_t EDGE = W::Tl::BM;
    constexpr bool PARTED = std::is_void<typename HalfOf<typename W::Tl>::Tile>::value;
    const Plan<W> p(c.rows, c.features, c.classes, vjp);
    char* ws = (char*)c.ws;
    const int64_t D = c.features, V = c.classes;
    hipError_t e;
    int *place = (int*)(ws + p.place), *row = (int*)(ws + p.row), *count = (int*)(ws + p.count);
    E *xa = (E*)(ws + p.xa), *ba = (E*)(ws + p.ba);
    E *r = (E*)(ws + p.r), *rt = (E*)(ws + p.rt), *xt = (E*)(ws + p.xt), *bt = (E*)(ws + p.bt);
    const Operand<E> beta = p.copy ? Operand<E>{ba, p.ldk, V, p.brows * p.ldk} : Operand<E>{(const E*)c.beta, c.ldbeta, V, 0};
    Largest<A> largest = {nullptr};
    if (vjp && c.lpbar) {
        largest.parts = (A*)(ws + p.scale);
        if (p.blocks > 1)
            class_scale<A><<<dim3(SCALE_PARTS), dim3(256), 0, st>>>((const A*)c.lpbar, c.y, c.rows, (A*)(ws + p.scale));
    }
    auto turn = [&](int64_t v0) { // a piece of beta
        const int64_t nv = V - v0 < p.piece ? V - v0 : p.piece, ldr = up_to(nv, EDGE);
        return TransposeArgs<W>{(const T*)c.beta + v0 * c.ldbeta, c.ldbeta, nv, nullptr, D, nullptr, bt, ldr, D * ldr};
    };
    auto blocks_of = [&](const TransposeArgs<W>& t) { return tiles_of(t.ldo, 64) * tiles_of(t.cols, 64); };
    for (int64_t n0 = 0; n0 < c.rows; n0 += p.block) {
        const int64_t N = c.rows - n0 < p.block ? c.rows - n0 : p.block;
        const bool first_block = n0 == 0, last_block = n0 + N == c.rows;
        const T* x = (const T*)c.x + n0 * c.ldx;
        const int64_t ldrt = up_to(N, EDGE); // (r is written in whole tiles)
        const bool scale_here = largest.parts && p.blocks == 1;
        number_rows<A>(c.y + n0, N, V, place, row, (int*)(ws + p.y), count, (A*)c.lp + n0, (const A*)c.lpbar,
                       scale_here ? (A*)(ws + p.scale) : nullptr, (int*)(ws + p.runs), st);
        PrepareArgs<W> q = {};
        q.g[0] = {x, c.ldx, N, D, place, xa, p.ldk, p.xrows * p.ldk, vjp ? (T*)c.xbar + n0 * D : nullptr, count};
        q.end[0] = (int)(tiles_of(N * (p.ldk / 8), 256) < 1024 ? tiles_of(N * (p.ldk / 8), 256) : 1024);
        q.end[1] = q.end[0];
        if (p.copy && first_block) {
            q.g[1] = {(const T*)c.beta, c.ldbeta, V, D, nullptr, ba, p.ldk, p.brows * p.ldk, nullptr, nullptr};
            q.end[1] += (int)(tiles_of(V * (p.ldk / 8), 256) < 2048 ? tiles_of(V * (p.ldk / 8), 256) : 2048);
        }
        q.end[2] = q.end[3] = q.end[1];
        if (vjp && !W::LINES) {
            q.t[0] = {x, c.ldx, N, count, D, row, xt, ldrt, D * ldrt};
            q.t[1] = turn(0);
            q.end[2] += (int)blocks_of(q.t[0]);
            q.end[3] = q.end[2] + (first_block || p.pieces > 1 ? (int)blocks_of(q.t[1]) : 0);
        }
        class_prepare<W><<<dim3((unsigned)q.end[3]), dim3(256), 0, st>>>(q);
        LogitArgs<W> l = {};
        l.beta = beta;
        l.x = {xa, p.ldk, N, p.xrows * p.ldk};
        l.count = count;
        l.alpha = (const T*)c.alpha;
        l.features = p.copy ? p.ldk : D;
        l.classes = V;
        l.y = (const int*)(ws + p.y);
        l.row = row;
        l.part_max = (A*)(ws + p.part_max);
        l.part_sum = (A*)(ws + p.part_sum);
        l.eta_y = (A*)(ws + p.eta_y);
        l.largest = largest;
        l.kept = (typename W::Tl::C*)(ws + p.kept);
        l.kept_classes = vjp ? p.kept_pieces * p.piece : 0;
        l.splits = p.lsplits;
        if constexpr (!PARTED) logits<W, true, false>(l, st);
        else if (p.lsplits == 1) logits<W, true, false>(l, st);
        else {
            typedef typename W::Tl Tl;
            l.tiles_v = p.tiles_v;
            l.grid = tile_grid<Tl>(l.tiles_v, N);
            l.plane = p.tiles_v * p.tiles_n * (Tl::TM * Tl::TN * Tl::THREADS);
            class_partial<W><<<dim3((unsigned)(l.grid * l.splits)), dim3(Tl::THREADS), 0, st>>>(l);
            logits<W, true, true>(l, st);
        }
        RowSum<A>* of = vjp ? (RowSum<A>*)(ws + p.of) : nullptr;
        class_join<A><<<dim3((unsigned)tiles_of(N, 8)), dim3(256), 0, st>>>(l.part_max, l.part_sum, l.eta_y, l.y, row, count,
                                                                            tiles_of(V, EDGE), N, V, of, (A*)c.lp + n0);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        if (!vjp) continue;
        if constexpr (REVERSE) {
            l.of = of;
            l.lpbar = c.lpbar ? (const A*)c.lpbar + n0 : nullptr;
            l.r = r;
            l.rt = rt;
            l.ldrt = ldrt;
            l.part_alpha = c.alphabar ? (A*)(ws + p.part_alpha) : nullptr;
            for (int64_t v0 = 0; v0 < V; v0 += p.piece) {
                const int64_t nv = V - v0 < p.piece ? V - v0 : p.piece;
                const bool first = v0 == 0, last = v0 + nv == V;
                if (!first && !W::LINES) {
                    PrepareArgs<W> t = {};
                    t.t[1] = turn(v0);
                    class_prepare<W><<<dim3((unsigned)blocks_of(t.t[1])), dim3(256), 0, st>>>(t);
                }
                l.beta = {beta.p + v0 * beta.ld, beta.ld, nv, beta.plane};
                l.alpha = c.alpha ? (const T*)c.alpha + v0 : nullptr;
                l.v0 = v0;
                l.ldr = up_to(nv, EDGE);
                l.r_plane = ldrt * l.ldr;
                l.rt_plane = l.ldr * ldrt;
                if (v0 < l.kept_classes) logits<W, false, true>(l, st);
                else logits<W, false, false>(l, st);
                ProductsArgs<W> m = {};
                if (W::LINES) m.x.A = {l.beta.p, l.beta.ld, D, l.beta.plane};
                else m.x.A = {bt, l.ldr, D, D * l.ldr};
                m.x.B = {r, l.ldr, N, l.r_plane};
                m.x.K = !W::LINES ? l.ldr : W::PLANES == 3 ? up_to(nv, 64) : nv; // (r is zero from nv on)
                m.x.count = count;
                m.x.acc = (A*)(ws + p.xacc);
                m.x.plane = p.block * D;
                m.x.add = !first;
                m.x.row = row;
                m.x.lpbar = l.lpbar;
                if (W::LINES) m.b.A = {xa, p.ldk, D, p.xrows * p.ldk};
                else m.b.A = {xt, ldrt, D, D * ldrt};
                m.b.B = {rt, ldrt, nv, l.rt_plane};
                m.b.k_edge = tile_k<E>(); // (rt and x are zero from the last row to there)
                m.b.count = count;
                m.b.acc = (A*)(ws + p.bacc) + (p.blocks > 1 ? v0 * D : 0);
                m.b.plane = (p.blocks > 1 ? V : p.piece) * D;
                m.b.add = !first_block;
                m.b.largest = largest;
                if (c.alphabar)
                    m.alpha = {l.part_alpha, count, EDGE, l.ldr, nv, tiles_of(N, EDGE) > 32, (A*)(ws + p.alpha_acc) + v0, !first_block,
                               last_block ? (T*)c.alphabar + v0 : nullptr};
                e = products<W>(m, p, last, (T*)c.xbar + n0 * D, last_block, (T*)c.betabar + v0 * D, st);
                if (e != hipSuccess) return e;
            }
        }
    }
    return hipSuccess;
}

// ---- few rows
template <typename T> struct FewPlan {
    // class tiles of a workgroup where the classes are enough to fill the card that way (fp64 has not the LDS for more)
    static constexpr int CT = sizeof(T) == 8 ? 2 : 4;
    bool large;
    int64_t tiles, piece, pieces, ldv, ldrt, share, splits; // (splits: of a piece)
    size_t part_max, part_sum, eta_y, eta, of, largest, r, rt, xt, xpart, bytes;
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
        eta_y = take(A * (size_t)rows);
        if (vjp) {
            ldrt = rows <= 32 ? 32 : 64;
            // logits, r and its transpose: as much as the other way's pieces and kept logits may take. (Beyond it logits are computed twice:
            // one row x 128 x 24 M classes in bf16 6.6 ms against 5.7, 64 x 512 x 1.1 M in fp64 9.3 against 7.2; the other way 14.8 and 12.6)
            const int64_t held = (int64_t)(rows * (A + E) + ldrt * E), most = (PIECE_BYTES + KEPT_BYTES) / held / 128 * 128;
            pieces = tiles_of(V, most);
            piece = pieces > 1 ? up_to(tiles_of(V, pieces), 128) : V;
            pieces = tiles_of(V, piece);
            ldv = up_to(piece, 64);
            const int64_t slabs = tiles_of(D, 16 * Vec16<T>::N);
            splits = tiles_of(2 * FILL, slabs);
            if (splits > tiles_of(piece, 128)) splits = tiles_of(piece, 128);
            if (V <= 1024) splits = 1; // (eight rounds of one workgroup are shorter than another launch)
            share = up_to(tiles_of(piece, splits), 128);
            splits = tiles_of(piece, share);
            eta = take(A * (size_t)(rows * ldv));
            of = take(2 * A * (size_t)rows);
            largest = take(A * FEW);
            r = take(E * (size_t)(rows * ldv));
            rt = take(E * (size_t)(piece * ldrt));
            xt = take(E * (size_t)(D * ldrt));
            xpart = pieces * splits > 1 ? take(A * (size_t)(splits * rows * D)) : 0;
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
    a.eta_y = (A*)(ws + p.eta_y);
    a.tiles = p.tiles;
    a.lp = (A*)c.lp;
    if (vjp) {
        a.eta = p.pieces == 1 ? (A*)(ws + p.eta) : nullptr;
        a.ldv = p.ldv;
        a.of = (RowSum<A>*)(ws + p.of);
        a.largest = (A*)(ws + p.largest);
        a.r = (T*)(ws + p.r);
        a.rt = (T*)(ws + p.rt);
        a.ldrt = p.ldrt;
        a.alphabar = (T*)c.alphabar;
        a.xpart = p.pieces * p.splits > 1 ? (A*)(ws + p.xpart) : nullptr;
        a.xbar = (T*)c.xbar;
        a.share = p.share;
    }
    bool odd = false; // rows that start in the middle of a word
    if (sizeof(T) == 2) odd = (((uintptr_t)c.beta | (uintptr_t)c.x) & 2) || ((c.ldbeta | c.ldx) & 1);
    auto with = [&](auto run) {
        if constexpr (sizeof(T) == 2) {
            if (odd) {
                run(std::true_type());
                return;
            }
        }
        run(std::false_type());
    };
    auto logits = [&](const FewArgs<T>& a) {
        with([&](auto half) {
            constexpr bool HALF = decltype(half)::value;
            const unsigned large = (unsigned)tiles_of(a.beta.rows, 16 * FewPlan<T>::CT), small = (unsigned)tiles_of(a.beta.rows, 16);
            if (p.large) class_few_logits<T, NT, FewPlan<T>::CT, 4, HALF><<<dim3(large), dim3(256), 0, st>>>(a);
            else class_few_logits<T, NT, 1, 8, HALF><<<dim3(small), dim3(512), 0, st>>>(a);
        });
    };
    logits(a);
    T* xt = vjp ? (T*)(ws + p.xt) : nullptr;
    class_few_join<T><<<dim3((unsigned)(c.rows + (vjp ? tiles_of(D, 64) : 0))), dim3(256), 0, st>>>(a, xt);
    if (!vjp) return hipGetLastError();
    const Largest<A> largest = {c.lpbar ? a.largest : nullptr};
    constexpr int NG = (NT <= 2 ? 32 : 64) / (4 * Vec16<T>::N);
    const int64_t xslabs = tiles_of(D, 16 * Vec16<T>::N), bslabs = tiles_of(D, Slab<T>::WIDTH);
    for (int64_t v0 = 0; v0 < V; v0 += p.piece) {
        const int64_t nv = V - v0 < p.piece ? V - v0 : p.piece, splits = tiles_of(nv, p.share);
        FewArgs<T> b = a;
        b.beta = {(const T*)c.beta + v0 * c.ldbeta, c.ldbeta, nv};
        b.v0 = v0;
        if (c.alpha) b.alpha = (const T*)c.alpha + v0;
        if (c.alphabar) b.alphabar = (T*)c.alphabar + v0;
        if (p.pieces > 1) {
            b.eta = (A*)(ws + p.eta);
            b.add = v0 > 0;
            logits(b);
        }
        class_few_r<T><<<dim3((unsigned)tiles_of(nv, 64)), dim3(256), 0, st>>>(b, largest);
        int64_t shares = tiles_of(4 * FILL, bslabs);
        if (shares > tiles_of(nv, 128)) shares = tiles_of(nv, 128);
        with([&](auto half) {
            class_few_back<T, NT, NG, decltype(half)::value><<<dim3((unsigned)(xslabs * splits + bslabs * shares)), dim3(256), 0, st>>>(
                b, xt, (T*)c.betabar + v0 * D, largest, (int)xslabs, (int)splits, (int)bslabs, (int)shares);
        });
    }
    if (a.xpart) class_few_xbar_join<T><<<dim3((unsigned)tiles_of(c.rows * D, 256)), dim3(256), 0, st>>>(a, (int)p.splits);
    return hipGetLastError();
}
template <typename T> hipError_t launch_few(const ClassArgs& c, bool vjp, hipStream_t st) {
    if (c.rows <= 16) return launch_few<T, 1>(c, vjp, st);
    if (c.rows <= 32) return launch_few<T, 2>(c, vjp, st);
    return launch_few<T, 4>(c, vjp, st);
}

// The fp32 log density of few rows and many classes stays with the fp32 instructions: splitting beta takes longer than they do. With and
// without splitting, in us: 100 rows x 1024 x 32000 146 / 88, 200 rows 166 / 151; but where the tiles do not fill the card (130 x 2000 x 5000)
// 132 / 160, and with the reverse mode (100 x 4000 x 8000) 311 / 395
bool whole(int64_t rows, int64_t features, int64_t classes) {
    const int64_t tiles = tiles_of(classes, 128) * tiles_of(rows, 128);
    return rows <= 256 && tiles * logit_splits<float>(tiles, features) >= WIDE_TILES;
}

// fp32 runs in three planes of bf16; fp64 has neither the instructions nor the registers for line tiles
template <typename T> struct Ways {
    typedef Way<T, WideTile<T>, 1> Wide;
    typedef Way<T, MidTile<T>, 1> Mid;
    typedef Way<T, SmallTile<T>, 1> Other; // operands that do not start on 16 bytes
};
template <> struct Ways<float> {
    typedef Way<float, WideTile<bf16_t, 3>, 3> Wide;
    typedef Way<float, MidTile<bf16_t, 3>, 3> Mid;
    typedef Way<float, SmallTile<float>, 1> Other; // the log density of few rows
};
template <> struct Ways<double> {
    typedef Way<double, SmallTile<double>, 1> Other;
};
template <typename T> size_t space(int64_t rows, int64_t features, int64_t classes, bool vjp) {
    if (rows <= FEW) return FewPlan<T>(rows, features, classes, vjp).bytes;
    typedef Ways<T> Y;
    if constexpr (sizeof(T) == 8) return Plan<typename Y::Other>(rows, features, classes, vjp).bytes;
    else {
        const bool large = wide(classes, rows < ROW_BLOCK ? rows : ROW_BLOCK);
        const size_t n = large ? Plan<typename Y::Wide>(rows, features, classes, vjp).bytes : Plan<typename Y::Mid>(rows, features, classes, vjp).bytes;
        if (sizeof(T) == 4 && !vjp && whole(rows, features, classes)) return Plan<typename Y::Other>(rows, features, classes, vjp).bytes;
        if constexpr (sizeof(T) == 2) { // (whether beta starts on 16 bytes shows only in the call)
            const size_t other = Plan<typename Y::Other>(rows, features, classes, vjp).bytes;
            return n > other ? n : other;
        }
        return n;
    }
}
template <typename T> hipError_t launch(const ClassArgs& c, bool vjp, hipStream_t st) {
    if (c.rows <= FEW) return launch_few<T>(c, vjp, st);
    typedef Ways<T> Y;
    if constexpr (sizeof(T) == 8) return launch_rows<typename Y::Other>(c, vjp, st);
    else {
        if constexpr (sizeof(T) == 4) {
            if (!vjp && whole(c.rows, c.features, c.classes)) return launch_rows<typename Y::Other, false>(c, false, st);
        }
        if constexpr (sizeof(T) == 2) {
            // (rows of an odd length are copied, whole ones need to start on 16 bytes where they are)
            if (c.features * sizeof(T) % 16 == 0 && !tile_fits(Operand<T>{(const T*)c.beta, c.ldbeta, c.classes, 0}))
                return launch_rows<typename Y::Other>(c, vjp, st);
        }
        return wide(c.classes, c.rows < ROW_BLOCK ? c.rows : ROW_BLOCK) ? launch_rows<typename Y::Wide>(c, vjp, st)
                                                                         : launch_rows<typename Y::Mid>(c, vjp, st);
    }
}

} // namespace

size_t gpt_class_workspace(int dtype, int64_t rows, int64_t features, int64_t classes, bool vjp) {
    if (gpt_class_narrow(dtype, rows, features, classes, vjp)) return gpt_class_narrow_workspace(dtype, rows, features, classes, vjp);
    switch (dtype) {
    case GPT_F64: return space<double>(rows, features, classes, vjp);
    case GPT_F32: return space<float>(rows, features, classes, vjp);
    case GPT_F16: return space<half_t>(rows, features, classes, vjp);
    default: return space<bf16_t>(rows, features, classes, vjp);
    }
}
hipError_t gpt_launch_class(int dtype, const ClassArgs& a, bool vjp, hipStream_t st) {
    if (gpt_class_narrow(dtype, a.rows, a.features, a.classes, vjp)) return gpt_launch_class_narrow(dtype, a, vjp, st);
    switch (dtype) {
    case GPT_F64: return launch<double>(a, vjp, st);
    case GPT_F32: return launch<float>(a, vjp, st);
    case GPT_F16: return launch<half_t>(a, vjp, st);
    default: return launch<bf16_t>(a, vjp, st);
    }
}
