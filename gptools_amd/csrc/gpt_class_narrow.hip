// The categorical log density for few features (up to 64): fields at the sites of a lattice, some hundreds of
// classes. What bounds it there is not the products but what passes between them, so neither the logits nor r leave the
// registers:
//
//   class_narrow_rows    a wave holds 16 rows of x (or 32) and walks the classes 32 at a time: logits of 16 classes x 16 rows on the
//                        matrix cores, their exponentials about a running reference, and sum_v p beta_v from the same registers.
//                        Leaves lp, the sums, and xbar = lpbar (beta_y - sum_v p beta_v).
//   class_narrow_classes a wave holds 16 classes (or 32) and walks the rows, logits again, r, betabar and alphabar.
//
// That the second product needs no shuffle is the matrix instruction's doing: it leaves value (v, n) of C in register r of lane
// group q with v = row(q, r), n = lane & 15, which is where an operand of the next product has k = v: in fp32 and fp64 the four
// registers are four steps of k, whichever classes they stand for; in 16 bits, rounded, they are the four k of one 16x16x16
// instruction. The other operand is read from LDS row by row (rows padded by 16 bytes: 16 rows of the first product's reads and 4
// of the second's fall on different banks), in 16 bits from a transposed copy.
//
// In 16 bits p and r are rounded for the second products, as their operands are of one type. p is at most 2^8 of the row's
// running reference; in fp16, which has too few exponents for the small probabilities, it is held times 2^13 and at most 2^2 of the
// reference. r is taken relative to the largest cotangent, in fp16 times 2^14, as in gpt_class.hip.
// p of the row's own class meets beta_y's other coefficient, 1, there: where it is nearly 1 xbar is small against both, and half a
// step of p_y would be as large as xbar. That one rounding is therefore known and taken back: the class's logit is computed once more
// after the walk, in the same order of operations and so to the same bit, and p_y with the reference that it met. What is left
// are roundings of entries of r, and of Acc.
#include "gpt_class.h"
#include "gpt_readout.h"
#include "gpt_tile.h"

using namespace gptt;

namespace {

template <typename T> struct NarrowArgs {
    typedef acc_t<T> A;
    Operand<T> x, beta;
    const T* alpha;
    const int64_t* y;
    const A* lpbar;
    int64_t features;
    // rows in the order they are taken, the observed ones first, and how many those are (null: as they come, all)
    const int *order, *count;
    // in that order: w: the row's cotangent over the largest, 0 without an observation; top: what its exponentials are taken about,
    // infinite there; share: w over their sum (16 bits: top is the lse and share is not there)
    A *lp, *top, *share_of, *w;
    int* at; // ... and the row's class
    Largest<A> largest;
    T* xbar;       // [rows][features]
    A* part;       // [shares][classes][features + 1]: betabar, alphabar; null: one share, the results themselves
    T *betabar, *alphabar;
    int64_t share; // rows of one share
};

// Tiles of 16 that a wave takes at a time of what it walks along. (fp64 and fp32 with many features, and the prefetch spread over four
// waves' shares, have not the registers and the LDS for two)
template <typename T, int DT, int SHARES> constexpr int VT_ = sizeof(T) >= 4 && DT == 4 && SHARES == 4 ? 1 : 2;

// Waves of a SIMD that the registers have to leave room for (bf16 5000 rows x 64 x 1000, fp32 5000 x 32 x 1000, whose waves share the rows:
// 39 and 41 us with two, 43 and 46 with four, which spill)
template <typename T, int DT, int SHARES>
constexpr int WAVES_ = sizeof(T) == 8 || (sizeof(T) == 4 && DT == 4) || (SHARES == 4 && DT * (int)sizeof(T) == 8) ? 2 : 4;

template <typename T, int DT> struct Narrow {
    typedef acc_t<T> A;
    typedef typename Vec16<T>::V Vec;
    typedef typename Mma<T>::C C;
    static constexpr int N = Vec16<T>::N, DP = 16 * DT; // features, padded
    static constexpr int G = DP / (4 * N);              // 16-byte chunks of a row that a lane holds
    static constexpr int LD = DP + N;                   // a row in LDS
    static constexpr bool TURN = sizeof(T) == 2;        // a transposed copy stands in LDS too
    // fp32: logits on the bf16 matrix cores, each value split in three (six products of 32 features take 96 cycles, the fp32
    // instructions of their one 256); three planes of the rows stand in LDS
    static constexpr bool SPLIT = std::is_same<T, float>::value && DT >= 2;
    static constexpr int SLD = DP + 8, SG = DP / 32;
    typedef Vec16<bf16_t>::V SVec;
    // rows of a step in LDS, and what they take: the rows, their transpose [DP][STEP + 4] or planes [3][STEP][SLD]
    template <int STEP> static constexpr int stage() { return STEP * LD + (TURN ? DP * (STEP + 4) : SPLIT ? 3 * STEP * SLD / 2 : 0); }
    // fp32: what stands in registers is times log2(e) already, so that logits come in that unit
    static constexpr bool UNIT = sizeof(T) >= 4;
    // the second kernel's probabilities as RowSum has them; in 16 bits about the lse, whose rounding (2^-24 of its size) is nothing
    // beside r's, and which takes fewer registers (fp16 65536 x 64 x 1000 124 us against 160)
    static constexpr bool SHARE = UNIT;
    // fp16: p is 2^HEAD where the logit is the reference's own, and at most 2^15: a probability is off by 2^-38 at most besides its
    // relative rounding, as r is, which holds 2^14 for one. The reference then follows the maximum more closely (65536 rows x 64 x 1000
    // 124 us, with a HEAD of 7 121)
    static constexpr int HEAD = std::is_same<T, half_t>::value ? 13 : 0;
    // a lane's part of one row (its column of the logits): chunks 4 g + q
    struct Part {
        Vec v[SPLIT ? 1 : G];
        SVec s[SPLIT ? 3 : 1][SPLIT ? SG : 1];
        __device__ __forceinline__ void load(const Operand<T>& o, int64_t row, int64_t D) {
            const int q = (threadIdx.x & 63) >> 4;
            if constexpr (SPLIT) {
#pragma unroll
                for (int g = 0; g < SG; ++g)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const Vec u = tile_chunk(o, row, (int64_t)((4 * g + q) * 8 + 4 * h), D);
                        uint32_t w[2][3];
                        split3(times_log2e(u[0]), times_log2e(u[1]), w[0]);
                        split3(times_log2e(u[2]), times_log2e(u[3]), w[1]);
#pragma unroll
                        for (int p = 0; p < 3; ++p) {
                            uint4 k = __builtin_bit_cast(uint4, s[p][g]);
                            if (h) k.z = w[0][p], k.w = w[1][p];
                            else k.x = w[0][p], k.y = w[1][p];
                            s[p][g] = __builtin_bit_cast(SVec, k);
                        }
                    }
            } else {
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    v[g] = tile_chunk(o, row, (int64_t)(4 * g + q) * N, D);
                    if constexpr (UNIT) {
#pragma unroll
                        for (int e = 0; e < N; ++e) v[g][e] = times_log2e(v[g][e]);
                    }
                }
            }
        }
        __device__ __forceinline__ void clear() {
            if constexpr (SPLIT) {
#pragma unroll
                for (int g = 0; g < SG; ++g) s[0][g] = s[1][g] = s[2][g] = SVec{};
            } else {
#pragma unroll
                for (int g = 0; g < G; ++g) v[g] = Vec{};
            }
        }
    };
    template <int STEP> static constexpr int loads() { return STEP * (DP / N) / 256 > 0 ? STEP * (DP / N) / 256 : 1; }

    // Rows r0.. of an operand (order given: order[r0..], rows of which y says that they are observed) into registers, and from
    // there into LDS. Rows behind the last repeat it (nothing counts them); no branch keeps a load from leaving before the one ahead of it
    // is back, unless a row ends within 16 bytes
    template <int STEP> struct Rows {
        Vec v[loads<STEP>()];
        bool seen[loads<STEP>()];
        __device__ __forceinline__ void fetch(const Operand<T>& o, int64_t r0, int64_t D, const int* order, const int64_t* y) {
            const int last = (int)(o.rows - r0 < STEP ? o.rows - r0 : STEP) - 1, d = (int)D;
#pragma unroll
            for (int i = 0; i < loads<STEP>(); ++i) {
                const int id = i * 256 + threadIdx.x, k = id % (DP / N) * N;
                int64_t row = r0 + (id / (DP / N) < last ? id / (DP / N) : last);
                if (order) row = order[row];
                seen[i] = k < d && (!y || y[row] >= 0);
                const T* from = o.p + row * o.ld;
                if (d % N == 0) v[i] = load16(from + (k < d ? k : 0));
                else {
                    v[i] = Vec{};
                    if (k + N <= d) v[i] = load16(from + k);
                    else {
#pragma unroll
                        for (int e = 0; e < N; ++e)
                            if (k + e < d) v[i][e] = from[k + e];
                    }
                }
            }
        }
        __device__ __forceinline__ void put(T* lds) const {
#pragma unroll
            for (int i = 0; i < loads<STEP>(); ++i) {
                const int id = i * 256 + threadIdx.x, r = id / (DP / N), c = id % (DP / N);
                if (r >= STEP) continue;
                uint4 word = __builtin_bit_cast(uint4, v[i]);
                if (!seen[i]) word = make_uint4(0, 0, 0, 0);
                const Vec w = __builtin_bit_cast(Vec, word);
                *reinterpret_cast<Vec*>(lds + r * LD + c * N) = w;
                if constexpr (TURN) {
                    T* t = lds + STEP * LD + c * N * (STEP + 4) + r;
#pragma unroll
                    for (int e = 0; e < N; ++e) t[e * (STEP + 4)] = w[e];
                }
                if constexpr (SPLIT) {
                    bf16_t* t = reinterpret_cast<bf16_t*>(lds + STEP * LD) + r * SLD + c * N;
                    uint32_t u[2][3];
                    split3(w[0], w[1], u[0]);
                    split3(w[2], w[3], u[1]);
#pragma unroll
                    for (int p = 0; p < 3; ++p) *reinterpret_cast<uint2*>(t + p * STEP * SLD) = make_uint2(u[0][p], u[1][p]);
                }
            }
        }
    };
    static __device__ __forceinline__ C split_mul(const SVec (&a)[3], const Part& f, int g, C c) {
        c = Mma<bf16_t>::mul(a[2], f.s[0][g], c); // (the smallest first)
        c = Mma<bf16_t>::mul(a[0], f.s[2][g], c);
        c = Mma<bf16_t>::mul(a[1], f.s[1][g], c);
        c = Mma<bf16_t>::mul(a[1], f.s[0][g], c);
        c = Mma<bf16_t>::mul(a[0], f.s[1][g], c);
        return Mma<bf16_t>::mul(a[0], f.s[0][g], c);
    }
    // a logit (times log2(e) in fp32) from the product with its level, or without it
    static __device__ __forceinline__ A eta(A p, A level) {
        if constexpr (UNIT) return p;
        else return __builtin_fmaf(p, LOG2E, level);
    }
    // the logit of row `row` of o (at least 0) for this lane's column, to the bit as logits() and eta() have it: the columns' rows
    // make a tile, whose diagonal it is
    static __device__ __forceinline__ A eta_at(const Operand<T>& o, int64_t row, int64_t D, const Part& f, A level) {
        const int lane = threadIdx.x & 63, q = lane >> 4;
        const A l = UNIT ? level : (A)0;
        C c = {l, l, l, l};
        if constexpr (SPLIT) {
#pragma unroll
            for (int g = 0; g < SG; ++g) {
                uint32_t w[4][3];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const Vec u = tile_chunk(o, row, (int64_t)((4 * g + q) * 8 + 4 * h), D);
                    split3(u[0], u[1], w[2 * h]);
                    split3(u[2], u[3], w[2 * h + 1]);
                }
                SVec a[3];
#pragma unroll
                for (int p = 0; p < 3; ++p) a[p] = __builtin_bit_cast(SVec, make_uint4(w[0][p], w[1][p], w[2][p], w[3][p]));
                c = split_mul(a, f, g, c);
            }
        } else {
#pragma unroll
            for (int g = 0; g < G; ++g) c = Mma<T>::mul(tile_chunk(o, row, (int64_t)(4 * g + q) * N, D), f.v[g], c);
        }
        A e = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) e = Mma<T>::row(q, r) == (lane & 15) ? c[r] : e;
        e += __shfl_xor(e, 16, 64); // (one of the four lane groups has it, the others zero)
        e += __shfl_xor(e, 32, 64);
        return eta(e, level);
    }
    // C[row base + .. of lds][column held in f] plus c in UNIT, and its use as an operand
    template <int STEP> static __device__ __forceinline__ C logits(const T* lds, int base, const Part& f, C c) {
        const int lane = threadIdx.x & 63, q = lane >> 4;
        if constexpr (SPLIT) {
            const bf16_t* t = reinterpret_cast<const bf16_t*>(lds + STEP * LD) + (base + (lane & 15)) * SLD;
#pragma unroll
            for (int g = 0; g < SG; ++g) {
                SVec a[3];
#pragma unroll
                for (int p = 0; p < 3; ++p) a[p] = *reinterpret_cast<const SVec*>(t + p * STEP * SLD + (4 * g + q) * 8);
                c = split_mul(a, f, g, c);
            }
        } else {
#pragma unroll
            for (int g = 0; g < G; ++g)
                c = Mma<T>::mul(*reinterpret_cast<const Vec*>(lds + (base + (lane & 15)) * LD + (4 * g + q) * N), f.v[g], c);
        }
        return c;
    }
    template <int STEP> static __device__ __forceinline__ void gather(const T* lds, int base, const C& p, C (&o)[DT]) {
        const int lane = threadIdx.x & 63, q = lane >> 4;
        if constexpr (TURN) {
            typedef typename Mma<T>::V4 V4;
            const uint2 u = make_uint2(pack2<T>(p[0], p[1]), pack2<T>(p[2], p[3]));
            const V4 b = __builtin_bit_cast(V4, u);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const V4 a = *reinterpret_cast<const V4*>(lds + STEP * LD + (16 * d + (lane & 15)) * (STEP + 4) + base + 4 * q);
                o[d] = Mma<T>::mul4(a, b, o[d]);
            }
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    o[d] = Mma<T>::mul1(lds[(base + Mma<T>::row(q, r)) * LD + 16 * d + (lane & 15)], p[r], o[d]);
        }
    }
    // o (a wave's: column = lane & 15, feature = 16 d + row(q, r)) into out[column][OLD]
    static constexpr int OLD = DP + 1;
    static __device__ __forceinline__ void spill(const C (&o)[DT], A* out) {
        const int lane = threadIdx.x & 63, q = lane >> 4;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) out[(lane & 15) * OLD + 16 * d + Mma<T>::row(q, r)] = o[d][r];
    }
};
constexpr int larger(int a, int b) { return a > b ? a : b; }

// WR groups of 16 NT rows x WV shares of the classes a workgroup
template <typename T, int DT, int WR, int WV, int NT, bool VJP> __global__ __launch_bounds__(256, (WAVES_<T, DT, WV>)) void class_narrow_rows(NarrowArgs<T> a) {
    typedef Narrow<T, DT> W;
    typedef typename W::A A;
    typedef typename W::C C;
    constexpr int VT = VT_<T, DT, WV>, STEP = 16 * VT * WV, ROWS = 16 * NT * WR;
    constexpr int STAGE = W::template stage<STEP>() * (int)sizeof(T), SPILL = VJP ? WV * ROWS * W::OLD * (int)sizeof(A) : 0;
    __shared__ uint4 room[(larger(STAGE, SPILL) + 15) / 16];
    __shared__ __attribute__((aligned(16))) A al[STEP];
    __shared__ A red[2][WV][ROWS];
    constexpr bool BACK = VJP && W::TURN; // p is rounded
    constexpr int HEAD = BACK ? W::HEAD : 0, LAG = HEAD ? 15 - HEAD : 8;
    __shared__ A met[BACK ? ROWS : 1], own[VJP ? ROWS : 1]; // the reference that a row's class met; beta_y's coefficient in xbar
    T* lds = reinterpret_cast<T*>(room);
    const int lane = threadIdx.x & 63, q = lane >> 4, wave = threadIdx.x >> 6, wr = wave / WV, wv = wave % WV;
    const int64_t n0 = wide_block() * ROWS, V = a.beta.rows, D = a.features;
    if (n0 >= a.x.rows) return;
    if (a.count && n0 >= *a.count) { // nothing observed here: zeros (lp has them)
        if (VJP)
            for (int id = threadIdx.x; id < ROWS * (int)D; id += 256) {
                const int r = id / (int)D;
                if (n0 + r < a.x.rows) a.xbar[a.order[n0 + r] * D + (id - r * (int)D)] = (T)0;
            }
        return;
    }
    typename W::Part x[NT];
    int y[NT], row[NT]; // y: -1 without an observation, V where it is no class
    A ref[NT], sum[NT], ref_y[BACK ? NT : 1];
    C o[NT][DT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int64_t n = n0 + (wr * NT + t) * 16 + (lane & 15);
        row[t] = n < a.x.rows ? (a.order ? a.order[n] : (int)n) : -1;
        const int64_t yn = row[t] >= 0 ? a.y[row[t]] : -1;
        y[t] = yn < 0 ? -1 : yn < V ? (int)yn : (int)V;
        if (y[t] >= 0) x[t].load(a.x, row[t], D);
        else x[t].clear();
        ref[t] = neg_inf<A>();
        if (BACK) ref_y[t] = neg_inf<A>();
        sum[t] = 0;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[t][d] = C{0, 0, 0, 0};
    }
    typename W::template Rows<STEP> next;
    A next_al = 0;
    auto fetch = [&](int64_t v0) {
        next.fetch(a.beta, v0, D, nullptr, nullptr);
        if (threadIdx.x < STEP) {
            const int64_t v = v0 + threadIdx.x;
            next_al = v < V ? (a.alpha ? level_log2e((A)a.alpha[v]) : (A)0) : neg_inf<A>();
        }
    };
    fetch(0);
    for (int64_t v0 = 0; v0 < V; v0 += STEP) {
        __syncthreads();
        next.put(lds);
        if (threadIdx.x < STEP) al[threadIdx.x] = next_al;
        __syncthreads();
        if (v0 + STEP < V) fetch(v0 + STEP);
        C p[NT][VT];
        A mx[NT];
        bool far = false;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            mx[t] = neg_inf<A>();
#pragma unroll
            for (int v = 0; v < VT; ++v) {
                const int base = (wv * VT + v) * 16;
                C level;
#pragma unroll
                for (int r = 0; r < 4; ++r) level[r] = al[base + Mma<T>::row(q, r)];
                p[t][v] = W::template logits<STEP>(lds, base, x[t], W::UNIT ? level : C{0, 0, 0, 0});
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    p[t][v][r] = W::eta(p[t][v][r], level[r]);
                    mx[t] = fmax(mx[t], p[t][v][r]);
                }
            }
            // the reference follows the maximum only where it falls behind by more than LAG (exponentials up to 2^LAG, or e^LAG, over
            // that of HEAD); whether it does shows without joining the four lane groups' maxima
            far |= mx[t] > ref[t] + (A)(LAG + HEAD);
        }
        if (__any(far)) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                mx[t] = fmax(mx[t], __shfl_xor(mx[t], 16, 64));
                mx[t] = fmax(mx[t], __shfl_xor(mx[t], 32, 64));
                const A to = fmax(ref[t], mx[t] - (A)HEAD);
                const A f = exp_log2e(ref[t] - about(to));
                ref[t] = to;
                sum[t] *= f;
                if (VJP) {
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[t][d][r] *= f;
                }
            }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const A m = about(ref[t]);
            if (BACK) ref_y[t] = (int)v0 <= y[t] ? ref[t] : ref_y[t]; // (the step that holds y is the last such)
#pragma unroll
            for (int v = 0; v < VT; ++v) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    p[t][v][r] = exp_log2e(p[t][v][r] - m);
                    sum[t] += p[t][v][r];
                }
                if (VJP) W::template gather<STEP>(lds, (wv * VT + v) * 16, p[t][v], o[t]);
            }
        }
    }
    // the waves' shares of the classes
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        sum[t] += __shfl_xor(sum[t], 16, 64);
        sum[t] += __shfl_xor(sum[t], 32, 64);
        if (q == 0) {
            red[0][wv][(wr * NT + t) * 16 + lane] = ref[t];
            red[1][wv][(wr * NT + t) * 16 + lane] = sum[t];
            // (of the waves that share the rows the one whose classes y is among)
            if (BACK && y[t] >= 0 && y[t] / (16 * VT) % WV == wv) met[(wr * NT + t) * 16 + lane] = ref_y[t];
        }
    }
    __syncthreads(); // (and the last step's rows have been read)
    A largest = 1;
    if (VJP) largest = a.largest.get();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int at = (wr * NT + t) * 16 + (lane & 15);
        const int64_t n = n0 + at;
        A mx = neg_inf<A>(), s = 0;
#pragma unroll
        for (int k = 0; k < WV; ++k) join(mx, s, red[0][k][at], red[1][k][at]);
        const bool known = y[t] >= 0 && y[t] < V;
        A eta = 0; // of the row's class
        if (wv == 0) eta = W::eta_at(a.beta, known ? y[t] : 0, D, x[t], known && a.alpha ? level_log2e((A)a.alpha[y[t]]) : (A)0);
        const A lp = row_lp(y[t], V, mx, s, eta);
        const RowSum<A> of = row_sum_of((int64_t)y[t], V, mx, s);
        const bool none = y[t] < 0 || of.share == 0;
        A w = 0;
        if (VJP) w = none ? (A)0 : known ? (a.lpbar ? a.lpbar[row[t]] : (A)1) : (A)__builtin_nan("");
        if (wv == 0 && q == 0 && n < a.x.rows) {
            a.lp[row[t]] = lp;
            if (VJP) {
                a.top[n] = none ? -neg_inf<A>() : W::SHARE ? of.top : of.top + times_log2e(log_(s));
                a.w[n] = w / largest;
                if (W::SHARE) a.share_of[n] = none ? (A)0 : w * of.share;
                a.at[n] = known ? y[t] : -1;
            }
        }
        if (VJP && wv == 0 && q == 0) {
            A more = 0; // what the rounding took from p_y, of the sum
            if constexpr (BACK) {
                if (known && !none) {
                    const A p = exp_log2e(eta - about(met[at]));
                    more = (p - (A)(T)p) * (exp_log2e(about(met[at]) - about(mx)) / s);
                }
            }
            own[at] = w * ((A)1 - more);
        }
        if (VJP) {
            const A f = none ? (A)0 : w * (exp_log2e(ref[t] - about(mx)) / s);
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[t][d][r] = none ? (A)0 : o[t][d][r] * f;
            W::spill(o[t], reinterpret_cast<A*>(room) + (wv * ROWS + (wr * NT + t) * 16) * W::OLD);
        }
    }
    if (!VJP) return;
    __syncthreads();
    const A* spilt = reinterpret_cast<const A*>(room);
    for (int id = threadIdx.x; id < ROWS * W::DP; id += 256) {
        const int r = id / W::DP, d = id % W::DP;
        const int64_t n = n0 + r;
        if (d >= D || n >= a.x.rows) continue;
        const int64_t to = a.order ? a.order[n] : n, yn = a.at[n];
        const A w = own[r];
        A s = 0;
#pragma unroll
        for (int k = 0; k < WV; ++k) s += spilt[(k * ROWS + r) * W::OLD + d];
        const A b = yn >= 0 ? (A)a.beta.p[yn * a.beta.ld + d] : (A)0;
        a.xbar[to * D + d] = w == 0 ? (T)0 : (T)(w * b - s);
    }
}

// WV groups of 16 NT classes x WR shares of the rows of this workgroup's share
template <typename T, int DT, int WR, int WV, int NT> __global__ __launch_bounds__(256, (WAVES_<T, DT, WR>)) void class_narrow_classes(NarrowArgs<T> a) {
    typedef Narrow<T, DT> W;
    typedef typename W::A A;
    typedef typename W::C C;
    constexpr int VT = VT_<T, DT, WR>, STEP = 16 * VT * WR, CLASSES = 16 * NT * WV;
    constexpr int STAGE = W::template stage<STEP>() * (int)sizeof(T), SPILL = WR * CLASSES * W::OLD * (int)sizeof(A);
    __shared__ uint4 room[(larger(STAGE, SPILL) + 15) / 16];
    __shared__ __attribute__((aligned(16))) A top[STEP], part_of[W::SHARE ? STEP : 4], wt[STEP];
    __shared__ __attribute__((aligned(16))) int yt[STEP];
    T* lds = reinterpret_cast<T*>(room);
    const int lane = threadIdx.x & 63, q = lane >> 4, wave = threadIdx.x >> 6, wv = wave / WR, wr = wave % WR;
    const int64_t v0 = (int64_t)blockIdx.x * CLASSES, V = a.beta.rows, D = a.features;
    constexpr A up = stored_scale<T>();
    typename W::Part b[NT];
    A al[NT], abar[NT];
    C o[NT][DT];
    int me[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int64_t v = v0 + (wv * NT + t) * 16 + (lane & 15);
        me[t] = (int)v;
        b[t].load(a.beta, v, D);
        al[t] = v < V ? (a.alpha ? level_log2e((A)a.alpha[v]) : (A)0) : neg_inf<A>();
        abar[t] = 0;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[t][d] = C{0, 0, 0, 0};
    }
    int64_t rows = a.x.rows, share = a.share;
    if (a.count) {
        rows = *a.count;
        share = ((rows + gridDim.y - 1) / gridDim.y + STEP - 1) / STEP * STEP;
    }
    const int64_t r0 = (int64_t)blockIdx.y * share, r1 = r0 + share < rows ? r0 + share : rows;
    const Operand<T> x = {a.x.p, a.x.ld, r1, 0};
    typename W::template Rows<STEP> next;
    A next_top = 0, next_part = 0, next_w = 0;
    int next_y = -1;
    auto fetch = [&](int64_t n0) {
        next.fetch(x, n0, D, a.order, a.order ? nullptr : a.y);
        if (threadIdx.x < STEP) {
            const int64_t n = n0 + threadIdx.x;
            next_top = n < r1 ? a.top[n] : -neg_inf<A>();
            if (W::SHARE) next_part = n < r1 ? a.share_of[n] : (A)0;
            next_w = n < r1 ? a.w[n] * up : (A)0;
            next_y = n < r1 ? a.at[n] : -1;
        }
    };
    if (r0 < r1) fetch(r0);
    for (int64_t n0 = r0; n0 < r1; n0 += STEP) {
        __syncthreads();
        next.put(lds);
        if (threadIdx.x < STEP) {
            top[threadIdx.x] = next_top;
            if (W::SHARE) part_of[threadIdx.x] = next_part;
            wt[threadIdx.x] = next_w;
            yt[threadIdx.x] = next_y;
        }
        __syncthreads();
        if (n0 + STEP < r1) fetch(n0 + STEP);
#pragma unroll
        for (int u = 0; u < VT; ++u) {
            const int base = (wr * VT + u) * 16;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                C p = {0, 0, 0, 0};
                // fp32: the product starts from the level less the row's top, which is in no register afterwards. (fp64 65536 x 32 x 1000
                // 459 us that way, 446 with the top taken off behind it)
                constexpr bool BEFORE = sizeof(T) == 4;
                if constexpr (W::SHARE) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) p[r] = BEFORE ? al[t] - top[base + Mma<T>::row(q, r)] : al[t];
                }
                p = W::template logits<STEP>(lds, base, b[t], p);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int n = base + Mma<T>::row(q, r);
                    const bool own = yt[n] == me[t];
                    if constexpr (W::SHARE) p[r] = (own ? wt[n] : (A)0) - part_of[n] * exp_log2e(BEFORE ? p[r] : p[r] - top[n]);
                    else p[r] = wt[n] * ((own ? (A)1 : (A)0) - exp_log2e(W::eta(p[r], al[t]) - top[n]));
                    abar[t] += p[r];
                }
                W::template gather<STEP>(lds, base, p, o[t]);
            }
        }
    }
    __syncthreads();
    A* spilt = reinterpret_cast<A*>(room);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        abar[t] += __shfl_xor(abar[t], 16, 64);
        abar[t] += __shfl_xor(abar[t], 32, 64);
        A* to = spilt + (wr * CLASSES + (wv * NT + t) * 16) * W::OLD;
        W::spill(o[t], to);
        if (q == 0) to[lane * W::OLD + W::DP] = abar[t];
    }
    __syncthreads();
    A* part = a.part + (int64_t)blockIdx.y * V * (D + 1);
    const A back = a.largest.get() / up;
    for (int id = threadIdx.x; id < CLASSES * W::OLD; id += 256) {
        const int c = id / W::OLD, d = id % W::OLD;
        if (v0 + c >= V || (d >= D && d != W::DP)) continue;
        A s = 0;
#pragma unroll
        for (int k = 0; k < WR; ++k) s += spilt[(k * CLASSES + c) * W::OLD + d];
        if (a.part) part[(v0 + c) * (D + 1) + (d == W::DP ? D : d)] = s;
        else if (d < D) a.betabar[(v0 + c) * D + d] = (T)(s * back);
        else if (a.alphabar) a.alphabar[v0 + c] = (T)(s * back);
    }
}

// betabar, alphabar <- sums over the shares. (The last share to arrive could add them up without this launch, but making its values
// visible across the XCDs costs more: fp64 2100 rows x 8 x 300 49 us against 23)
template <typename T> __global__ __launch_bounds__(256) void class_narrow_join(const acc_t<T>* part, int shares, int64_t V, int64_t D,
                                                                              Largest<acc_t<T>> largest, T* betabar, T* alphabar) {
    typedef acc_t<T> A;
    const A back = largest.get() / (A)stored_scale<T>();
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, count = V * (D + 1);
    if (i >= count) return;
    A s[4] = {0, 0, 0, 0};
    int k = 0;
    for (; k + 16 <= shares; k += 16) {
        A u[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) u[e] = part[(k + e) * count + i];
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e & 3] += u[e];
    }
    for (; k + 4 <= shares; k += 4)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += part[(k + e) * count + i];
    for (; k < shares; ++k) s[0] += part[k * count + i];
    const A t = ((s[0] + s[1]) + (s[2] + s[3])) * back;
    const int64_t v = i / (D + 1), d = i - v * (D + 1);
    if (d < D) betabar[v * D + d] = (T)t;
    else if (alphabar) alphabar[v] = (T)t;
}

int64_t tiles_of(int64_t n, int64_t b) { return (n + b - 1) / b; }

constexpr int64_t INDEXED = 16384; // rows from which the observed ones are numbered (one launch more)

// Shapes of the two kernels. Many rows: four waves share the classes' rows in LDS, each with its own rows (and, but for fp64, two
// tiles of them: that has not the registers). Few: the four waves share the rows, each with a quarter of the classes.
template <typename T> struct NarrowPlan {
    static constexpr int NT = sizeof(T) == 8 ? 1 : 2;
    bool many_rows, many_classes, indexed;
    int64_t share, shares;
    size_t top, share_of, w, at, scale, order, count, runs, part, bytes;
    NarrowPlan(int64_t rows, int64_t D, int64_t V, bool vjp) {
        const size_t A = sizeof(acc_t<T>);
        many_rows = tiles_of(rows, 64 * NT) >= 512;
        const int64_t groups = tiles_of(V, 64 * NT);
        many_classes = groups * tiles_of(rows, 32 * 8) >= 512;
        const int64_t blocks = many_classes ? groups : tiles_of(V, 16 * NT), step = many_classes ? 32 : 128;
        int64_t s = tiles_of(1024, blocks);
        const int64_t most = tiles_of(rows, step);
        if (s > most) s = most;
        if (s > 1024) s = 1024;
        if (rows <= 256) s = 1; // (two steps of one workgroup are shorter than another launch)
        share = tiles_of(tiles_of(rows, s), step) * step;
        shares = tiles_of(rows, share);
        indexed = rows >= INDEXED;
        size_t to = 0;
        auto take = [&](size_t n) {
            const size_t p = to;
            to += (n + 255) / 256 * 256;
            return p;
        };
        order = count = runs = 0;
        if (indexed) {
            order = take(4 * (size_t)rows);
            count = take(4);
            runs = take(4 * (size_t)tiles_of(rows, INDEX_ROWS));
        }
        if (vjp) {
            top = take(A * (size_t)rows);
            share_of = take(sizeof(T) >= 4 ? A * (size_t)rows : 0);
            w = take(A * (size_t)rows);
            at = take(4 * (size_t)rows);
            scale = take(A * SCALE_PARTS);
            part = shares > 1 ? take(A * (size_t)(shares * V * (D + 1))) : 0;
        }
        bytes = to;
    }
};

template <typename T, int DT, bool VJP> void rows_kernel(const NarrowArgs<T>& a, const NarrowPlan<T>& p, hipStream_t st) {
    constexpr int NT = NarrowPlan<T>::NT;
    if (p.many_rows)
        class_narrow_rows<T, DT, 2, 2, NT, VJP><<<wide_grid(tiles_of(a.x.rows, 32 * NT)), dim3(256), 0, st>>>(a);
    else class_narrow_rows<T, DT, 1, 4, 1, VJP><<<dim3((unsigned)tiles_of(a.x.rows, 16)), dim3(256), 0, st>>>(a);
}
template <typename T, int DT> void run(const NarrowArgs<T>& a, const NarrowPlan<T>& p, bool vjp, hipStream_t st) {
    constexpr int NT = NarrowPlan<T>::NT;
    if (!vjp) {
        rows_kernel<T, DT, false>(a, p, st);
        return;
    }
    rows_kernel<T, DT, true>(a, p, st);
    if (p.many_classes)
        class_narrow_classes<T, DT, 1, 4, NT>
            <<<dim3((unsigned)tiles_of(a.beta.rows, 64 * NT), (unsigned)p.shares), dim3(256), 0, st>>>(a);
    else class_narrow_classes<T, DT, 4, 1, NT><<<dim3((unsigned)tiles_of(a.beta.rows, 16 * NT), (unsigned)p.shares), dim3(256), 0, st>>>(a);
}
template <typename T> hipError_t launch(const ClassArgs& c, bool vjp, hipStream_t st) {
    typedef acc_t<T> A;
    const NarrowPlan<T> p(c.rows, c.features, c.classes, vjp);
    char* ws = (char*)c.ws;
    NarrowArgs<T> a = {};
    a.x = {(const T*)c.x, c.ldx, c.rows, 0};
    a.beta = {(const T*)c.beta, c.ldbeta, c.classes, 0};
    a.alpha = (const T*)c.alpha;
    a.y = c.y;
    a.lpbar = (const A*)c.lpbar;
    a.features = c.features;
    a.lp = (A*)c.lp;
    if (p.indexed) {
        number_rows<A>(c.y, c.rows, c.classes, nullptr, (int*)(ws + p.order), nullptr, (int*)(ws + p.count), a.lp, nullptr,
                       nullptr, (int*)(ws + p.runs), st);
        a.order = (const int*)(ws + p.order);
        a.count = (const int*)(ws + p.count);
    }
    if (vjp) {
        a.top = (A*)(ws + p.top);
        a.share_of = (A*)(ws + p.share_of);
        a.w = (A*)(ws + p.w);
        a.at = (int*)(ws + p.at);
        a.xbar = (T*)c.xbar;
        a.part = p.shares > 1 ? (A*)(ws + p.part) : nullptr;
        a.betabar = (T*)c.betabar;
        a.alphabar = (T*)c.alphabar;
        a.share = p.share;
        if (sizeof(T) == 2 && c.lpbar) { // (r is not rounded otherwise)
            a.largest.parts = (const A*)(ws + p.scale);
            class_scale<A><<<dim3(SCALE_PARTS), dim3(256), 0, st>>>(a.lpbar, c.y, c.rows, (A*)(ws + p.scale));
        }
    }
    if constexpr (sizeof(T) == 2) {
        if (c.features <= 32) run<T, 2>(a, p, vjp, st);
        else run<T, 4>(a, p, vjp, st);
    } else {
        if (c.features <= 16) run<T, 1>(a, p, vjp, st);
        else if (c.features <= 32) run<T, 2>(a, p, vjp, st);
        else run<T, 4>(a, p, vjp, st);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !vjp || p.shares == 1) return e;
    class_narrow_join<T><<<dim3((unsigned)tiles_of(c.classes * (c.features + 1), 256)), dim3(256), 0, st>>>(
        a.part, (int)p.shares, c.classes, c.features, a.largest, (T*)c.betabar, (T*)c.alphabar);
    return hipGetLastError();
}

} // namespace

// Few features, and classes few enough for the workgroups of a call's rows to walk them all: some hundreds, or not many more
// than the rows. In 16 bits large tiles are better for lp alone (8192 rows x 8000 classes x 64 features in bf16: 47 us against 116;
// with the reverse mode 238 against 213, 65536 x 1000 x 64 316 against 165)
bool gpt_class_narrow(int dtype, int64_t rows, int64_t features, int64_t classes, bool vjp) {
    if (features > 64) return false;
    return classes <= 1024 || (classes / 4 <= rows && (vjp || dtype == GPT_F64 || dtype == GPT_F32));
}
size_t gpt_class_narrow_workspace(int dtype, int64_t rows, int64_t features, int64_t classes, bool vjp) {
    switch (dtype) {
    case GPT_F64: return NarrowPlan<double>(rows, features, classes, vjp).bytes;
    case GPT_F32: return NarrowPlan<float>(rows, features, classes, vjp).bytes;
    case GPT_F16: return NarrowPlan<half_t>(rows, features, classes, vjp).bytes;
    default: return NarrowPlan<bf16_t>(rows, features, classes, vjp).bytes;
    }
}
hipError_t gpt_launch_class_narrow(int dtype, const ClassArgs& a, bool vjp, hipStream_t st) {
    switch (dtype) {
    case GPT_F64: return launch<double>(a, vjp, st);
    case GPT_F32: return launch<float>(a, vjp, st);
    case GPT_F16: return launch<half_t>(a, vjp, st);
    default: return launch<bf16_t>(a, vjp, st);
    }
}
