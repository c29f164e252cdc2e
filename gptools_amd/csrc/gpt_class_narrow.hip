// The categorical log density for few features (up to 64, fp64 and fp32): fields at the sites of a lattice, some hundreds of
// classes. What bounds it there is not the products but what passes between them, so neither the logits nor r leave the
// registers:
//
//   class_narrow_rows    a wave holds 16 rows of x (or 32) and walks the classes 32 at a time: logits of 16 classes x 16 rows on the
//                        matrix cores, their exponentials about a running reference, and sum_v p beta_v from the same registers.
//                        Leaves lp, lse, and xbar = lpbar (beta_y - sum_v p beta_v).
//   class_narrow_classes a wave holds 16 classes (or 32) and walks the rows, logits again, r, betabar and alphabar.
//
// That the second product needs no shuffle is the matrix instruction's doing: it leaves value (v, n) of C in register r of lane
// group q with v = row(q, r), n = lane & 15, which is where an operand of the next product has k = v: the four registers are four
// steps of k, whichever classes they stand for. The other operand is read from LDS row by row (rows padded by 16 bytes: 16 rows
// of the first product's reads and 4 of the second's fall on different banks).
#include "gpt_class.h"
#include "gpt_readout.h"
#include "gpt_tile.h"

using namespace gptt;

namespace {

template <typename T> struct NarrowArgs {
    Operand<T> x, beta;
    const T* alpha;
    const int64_t* y;
    const T* lpbar; // (Acc is T here)
    int64_t features;
    T *lp, *lse, *w; // w: the row's cotangent, 0 without an observation; lse: infinite there
    T* xbar;         // [rows][features]
    T* part;         // [shares][classes][features + 1]: betabar, alphabar
    int64_t share;   // rows of one share
};

constexpr int VT = 2; // tiles of 16 that a wave takes at a time of what it walks along

template <typename T, int DT> struct Narrow {
    typedef typename Vec16<T>::V Vec;
    typedef typename Mma<T>::C C;
    static constexpr int N = Vec16<T>::N, DP = 16 * DT; // features, padded
    static constexpr int G = DP / (4 * N);              // 16-byte chunks of a row that a lane holds
    static constexpr int LD = DP + N;                   // a row in LDS
    // Rows r0.. of an operand into registers (LOADS chunks of 256 threads), and from there into LDS
    template <int LOADS> static __device__ __forceinline__ void fetch(Vec (&v)[LOADS], const Operand<T>& o, int64_t r0, int64_t D,
                                                                      const int64_t* y) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int id = i * 256 + threadIdx.x, r = id / (DP / N), c = id % (DP / N);
            const bool seen = !y || (r0 + r < o.rows && y[r0 + r] >= 0);
            v[i] = seen ? tile_chunk(o, r0 + r, (int64_t)c * N, D) : Vec{};
        }
    }
    template <int LOADS> static __device__ __forceinline__ void put(const Vec (&v)[LOADS], T* lds) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int id = i * 256 + threadIdx.x, r = id / (DP / N), c = id % (DP / N);
            *reinterpret_cast<Vec*>(lds + r * LD + c * N) = v[i];
        }
    }
    // C[row of lds][column held in f] and its use as an operand
    static __device__ __forceinline__ C logits(const T* rows, const Vec (&f)[G]) {
        const int lane = threadIdx.x & 63, q = lane >> 4;
        C c = {0, 0, 0, 0};
#pragma unroll
        for (int g = 0; g < G; ++g)
            c = Mma<T>::mul(*reinterpret_cast<const Vec*>(rows + (lane & 15) * LD + (4 * g + q) * N), f[g], c);
        return c;
    }
    static __device__ __forceinline__ void gather(const T* rows, const C& p, C (&o)[DT]) {
        const int lane = threadIdx.x & 63, q = lane >> 4;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] = Mma<T>::mul1(rows[Mma<T>::row(q, r) * LD + 16 * d + (lane & 15)], p[r], o[d]);
    }
    // o (a wave's: column = lane & 15, feature = 16 d + row(q, r)) into out[column][OLD]
    static constexpr int OLD = DP + 1;
    static __device__ __forceinline__ void spill(const C (&o)[DT], T* out) {
        const int lane = threadIdx.x & 63, q = lane >> 4;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) out[(lane & 15) * OLD + 16 * d + Mma<T>::row(q, r)] = o[d][r];
    }
};

// WR groups of 16 NT rows x WV shares of the classes a workgroup
template <typename T, int DT, int WR, int WV, int NT, bool VJP> __global__ __launch_bounds__(256) void class_narrow_rows(NarrowArgs<T> a) {
    typedef Narrow<T, DT> W;
    typedef typename W::C C;
    typedef typename W::Vec Vec;
    constexpr int STEP = 16 * VT * WV, ROWS = 16 * NT * WR, N = W::N;
    constexpr int STAGE = STEP * W::LD, SPILL = VJP ? WV * ROWS * W::OLD : 0;
    __shared__ __attribute__((aligned(16))) T lds[STAGE > SPILL ? STAGE : SPILL];
    __shared__ T al[STEP], red[2][WV][ROWS];
    const int lane = threadIdx.x & 63, q = lane >> 4, wave = threadIdx.x >> 6, wr = wave / WV, wv = wave % WV;
    const int64_t n0 = (int64_t)blockIdx.x * ROWS, V = a.beta.rows;
    Vec x[NT][W::G];
    int64_t y[NT];
    T ref[NT], sum[NT];
    C o[NT][DT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int64_t n = n0 + (wr * NT + t) * 16 + (lane & 15);
        y[t] = n < a.x.rows ? a.y[n] : -1;
#pragma unroll
        for (int g = 0; g < W::G; ++g) x[t][g] = y[t] >= 0 ? tile_chunk(a.x, n, (int64_t)(4 * g + q) * N, a.features) : Vec{};
        ref[t] = neg_inf<T>();
        sum[t] = 0;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[t][d] = C{0, 0, 0, 0};
    }
    constexpr int CHUNKS = STEP * (W::DP / N), LOADS = CHUNKS / 256 > 0 ? CHUNKS / 256 : 1;
    static_assert(CHUNKS % 256 == 0 || CHUNKS < 256, "whole loads");
    const bool loads = CHUNKS >= 256 || threadIdx.x < CHUNKS;
    Vec next[LOADS];
    T next_al = 0;
    auto fetch = [&](int64_t v0) {
        if (loads) W::fetch(next, a.beta, v0, a.features, nullptr);
        if (threadIdx.x < STEP) {
            const int64_t v = v0 + threadIdx.x;
            next_al = v < V ? (a.alpha ? level_log2e(a.alpha[v]) : (T)0) : neg_inf<T>();
        }
    };
    fetch(0);
    for (int64_t v0 = 0; v0 < V; v0 += STEP) {
        __syncthreads();
        if (loads) W::put(next, lds);
        if (threadIdx.x < STEP) al[threadIdx.x] = next_al;
        __syncthreads();
        if (v0 + STEP < V) fetch(v0 + STEP);
        const T* rows = lds + wv * 16 * VT * W::LD;
        C p[NT][VT];
        T mx[NT];
        bool far = false;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            mx[t] = neg_inf<T>();
#pragma unroll
            for (int v = 0; v < VT; ++v) {
                p[t][v] = W::logits(rows + v * 16 * W::LD, x[t]);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    p[t][v][r] = times_log2e(p[t][v][r]) + al[(wv * VT + v) * 16 + Mma<T>::row(q, r)];
                    mx[t] = fmax(mx[t], p[t][v][r]);
                }
            }
            mx[t] = fmax(mx[t], __shfl_xor(mx[t], 16, 64));
            mx[t] = fmax(mx[t], __shfl_xor(mx[t], 32, 64));
            // the reference follows the maximum only where it falls behind by more than 8 (exponentials up to 2^8, or e^8)
            far |= mx[t] > ref[t] + (T)8 || (ref[t] == neg_inf<T>() && mx[t] > ref[t]);
        }
        if (__any(far)) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const T to = fmax(ref[t], mx[t]);
                const T f = exp_log2e(ref[t] - about(to));
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
            const T m = about(ref[t]);
#pragma unroll
            for (int v = 0; v < VT; ++v) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    p[t][v][r] = exp_log2e(p[t][v][r] - m);
                    sum[t] += p[t][v][r];
                }
                if (VJP) W::gather(rows + v * 16 * W::LD, p[t][v], o[t]);
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
        }
    }
    __syncthreads(); // (and the last step's rows have been read)
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int at = (wr * NT + t) * 16 + (lane & 15);
        const int64_t n = n0 + at;
        T mx = neg_inf<T>(), s = 0;
#pragma unroll
        for (int k = 0; k < WV; ++k) join(mx, s, red[0][k][at], red[1][k][at]);
        const bool known = y[t] >= 0 && y[t] < V;
        T eta = 0; // of the row's class, as the matrix cores have it up to rounding
        if (wv == 0 && known) {
#pragma unroll
            for (int g = 0; g < W::G; ++g) {
                const Vec b = tile_chunk(a.beta, y[t], (int64_t)(4 * g + q) * N, a.features);
#pragma unroll
                for (int e = 0; e < N; ++e) eta += x[t][g][e] * b[e];
            }
        }
        eta += __shfl_xor(eta, 16, 64);
        eta += __shfl_xor(eta, 32, 64);
        eta = times_log2e(eta);
        if (known && a.alpha) eta += level_log2e(a.alpha[y[t]]);
        T lse;
        const T lp = row_lp(y[t], V, mx, s, eta, lse);
        const bool none = y[t] < 0 || lse == neg_inf<T>();
        T w = 0;
        if (VJP) w = none ? (T)0 : known ? (a.lpbar ? a.lpbar[n] : (T)1) : (T)__builtin_nan("");
        if (wv == 0 && q == 0 && n < a.x.rows) {
            a.lp[n] = lp;
            if (VJP) {
                a.lse[n] = none ? -neg_inf<T>() : lse;
                a.w[n] = w;
            }
        }
        if (VJP) {
            const T f = none ? (T)0 : w * (exp_log2e(ref[t] - about(mx)) / s);
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[t][d][r] = none ? (T)0 : o[t][d][r] * f;
            W::spill(o[t], lds + (wv * ROWS + (wr * NT + t) * 16) * W::OLD);
        }
    }
    if (!VJP) return;
    __syncthreads();
    for (int id = threadIdx.x; id < ROWS * W::DP; id += 256) {
        const int r = id / W::DP, d = id % W::DP;
        const int64_t n = n0 + r;
        if (d >= a.features || n >= a.x.rows) continue;
        const int64_t yn = a.y[n];
        const T w = a.w[n];
        T s = 0;
#pragma unroll
        for (int k = 0; k < WV; ++k) s += lds[(k * ROWS + r) * W::OLD + d];
        const T b = yn >= 0 && yn < V ? a.beta.p[yn * a.beta.ld + d] : (T)0;
        a.xbar[n * a.features + d] = yn < 0 || w == 0 ? (T)0 : w * b - s;
    }
}

// WV groups of 16 NT classes x WR shares of the rows of this workgroup's share
template <typename T, int DT, int WR, int WV, int NT> __global__ __launch_bounds__(256) void class_narrow_classes(NarrowArgs<T> a) {
    typedef Narrow<T, DT> W;
    typedef typename W::C C;
    typedef typename W::Vec Vec;
    constexpr int STEP = 16 * VT * WR, CLASSES = 16 * NT * WV, N = W::N;
    constexpr int STAGE = STEP * W::LD, SPILL = WR * CLASSES * W::OLD;
    __shared__ __attribute__((aligned(16))) T lds[STAGE > SPILL ? STAGE : SPILL];
    __shared__ T lse[STEP], wt[STEP];
    __shared__ int yt[STEP];
    const int lane = threadIdx.x & 63, q = lane >> 4, wave = threadIdx.x >> 6, wv = wave / WR, wr = wave % WR;
    const int64_t v0 = (int64_t)blockIdx.x * CLASSES, V = a.beta.rows, D = a.features;
    Vec b[NT][W::G];
    T al[NT], abar[NT];
    C o[NT][DT];
    int me[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int64_t v = v0 + (wv * NT + t) * 16 + (lane & 15);
        me[t] = (int)v;
#pragma unroll
        for (int g = 0; g < W::G; ++g) b[t][g] = tile_chunk(a.beta, v, (int64_t)(4 * g + q) * N, D);
        al[t] = v < V ? (a.alpha ? level_log2e(a.alpha[v]) : (T)0) : neg_inf<T>();
        abar[t] = 0;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[t][d] = C{0, 0, 0, 0};
    }
    const int64_t r0 = (int64_t)blockIdx.y * a.share, r1 = r0 + a.share < a.x.rows ? r0 + a.share : a.x.rows;
    constexpr int CHUNKS = STEP * (W::DP / N), LOADS = CHUNKS / 256 > 0 ? CHUNKS / 256 : 1;
    static_assert(CHUNKS % 256 == 0 || CHUNKS < 256, "whole loads");
    const bool loads = CHUNKS >= 256 || threadIdx.x < CHUNKS;
    const Operand<T> x = {a.x.p, a.x.ld, r1};
    Vec next[LOADS];
    T next_lse = 0, next_w = 0;
    int next_y = -1;
    auto fetch = [&](int64_t n0) {
        if (loads) W::fetch(next, x, n0, D, a.y);
        if (threadIdx.x < STEP) {
            const int64_t n = n0 + threadIdx.x;
            next_lse = n < r1 ? a.lse[n] : -neg_inf<T>();
            next_w = n < r1 ? a.w[n] : (T)0;
            next_y = n < r1 ? (int)a.y[n] : -1; // (a class fits; anything else matches none)
        }
    };
    if (r0 < r1) fetch(r0);
    for (int64_t n0 = r0; n0 < r1; n0 += STEP) {
        __syncthreads();
        if (loads) W::put(next, lds);
        if (threadIdx.x < STEP) {
            lse[threadIdx.x] = next_lse;
            wt[threadIdx.x] = next_w;
            yt[threadIdx.x] = next_y;
        }
        __syncthreads();
        if (n0 + STEP < r1) fetch(n0 + STEP);
#pragma unroll
        for (int u = 0; u < VT; ++u) {
            const int base = (wr * VT + u) * 16;
            const T* rows = lds + base * W::LD;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                C p = W::logits(rows, b[t]);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int n = base + Mma<T>::row(q, r);
                    const T e = exp_log2e(times_log2e(p[r]) + al[t] - lse[n]);
                    p[r] = wt[n] * ((yt[n] == me[t] ? (T)1 : (T)0) - e);
                    abar[t] += p[r];
                }
                W::gather(rows, p, o[t]);
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        abar[t] += __shfl_xor(abar[t], 16, 64);
        abar[t] += __shfl_xor(abar[t], 32, 64);
        T* to = lds + (wr * CLASSES + (wv * NT + t) * 16) * W::OLD;
        W::spill(o[t], to);
        if (q == 0) to[lane * W::OLD + W::DP] = abar[t];
    }
    __syncthreads();
    T* part = a.part + (int64_t)blockIdx.y * V * (D + 1);
    for (int id = threadIdx.x; id < CLASSES * W::OLD; id += 256) {
        const int c = id / W::OLD, d = id % W::OLD;
        if (v0 + c >= V || (d >= D && d != W::DP)) continue;
        T s = 0;
#pragma unroll
        for (int k = 0; k < WR; ++k) s += lds[(k * CLASSES + c) * W::OLD + d];
        part[(v0 + c) * (D + 1) + (d == W::DP ? D : d)] = s;
    }
}

// betabar, alphabar <- sums over the shares
template <typename T> __global__ __launch_bounds__(256) void class_narrow_join(const T* part, int shares, int64_t V, int64_t D, T* betabar,
                                                                              T* alphabar) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, count = V * (D + 1);
    if (i >= count) return;
    T s[4] = {0, 0, 0, 0};
    int k = 0;
    for (; k + 4 <= shares; k += 4)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += part[(k + e) * count + i];
    for (; k < shares; ++k) s[0] += part[k * count + i];
    const T t = (s[0] + s[1]) + (s[2] + s[3]);
    const int64_t v = i / (D + 1), d = i - v * (D + 1);
    if (d < D) betabar[v * D + d] = t;
    else if (alphabar) alphabar[v] = t;
}

int64_t tiles_of(int64_t n, int64_t b) { return (n + b - 1) / b; }

// Shapes of the two kernels. Many rows: four waves share the classes' rows in LDS, each with its own rows (and, in fp32, two tiles of
// them: fp64 has not the registers). Few: the four waves share the rows, each with a quarter of the classes.
template <typename T> struct NarrowPlan {
    static constexpr int NT = sizeof(T) == 4 ? 2 : 1;
    bool many_rows, many_classes;
    int64_t share, shares;
    size_t lse, w, part, bytes;
    NarrowPlan(int64_t rows, int64_t D, int64_t V, bool vjp) {
        many_rows = tiles_of(rows, 64 * NT) >= 512;
        const int64_t groups = tiles_of(V, 64 * NT);
        many_classes = groups * tiles_of(rows, 32 * 8) >= 512;
        const int64_t blocks = many_classes ? groups : tiles_of(V, 16 * NT), step = many_classes ? 32 : 128;
        int64_t s = tiles_of(768, blocks);
        const int64_t most = tiles_of(rows, step);
        if (s > most) s = most;
        if (s > 1024) s = 1024;
        share = tiles_of(tiles_of(rows, s), step) * step;
        shares = tiles_of(rows, share);
        lse = 0;
        w = (sizeof(T) * (size_t)rows + 255) / 256 * 256;
        part = 2 * w;
        bytes = vjp ? part + sizeof(T) * (size_t)(shares * V * (D + 1)) : 0;
    }
};

template <typename T, int DT, bool VJP> void rows_kernel(const NarrowArgs<T>& a, const NarrowPlan<T>& p, hipStream_t st) {
    constexpr int NT = NarrowPlan<T>::NT;
    if (p.many_rows)
        class_narrow_rows<T, DT, 4, 1, NT, VJP><<<dim3((unsigned)tiles_of(a.x.rows, 64 * NT)), dim3(256), 0, st>>>(a);
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
    const NarrowPlan<T> p(c.rows, c.features, c.classes, vjp);
    char* ws = (char*)c.ws;
    NarrowArgs<T> a = {};
    a.x = {(const T*)c.x, c.ldx, c.rows};
    a.beta = {(const T*)c.beta, c.ldbeta, c.classes};
    a.alpha = (const T*)c.alpha;
    a.y = c.y;
    a.lpbar = (const T*)c.lpbar;
    a.features = c.features;
    a.lp = (T*)c.lp;
    a.lse = (T*)(ws + p.lse);
    a.w = (T*)(ws + p.w);
    a.xbar = (T*)c.xbar;
    a.part = (T*)(ws + p.part);
    a.share = p.share;
    if (c.features <= 16) run<T, 1>(a, p, vjp, st);
    else if (c.features <= 32) run<T, 2>(a, p, vjp, st);
    else run<T, 4>(a, p, vjp, st);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !vjp) return e;
    class_narrow_join<T><<<dim3((unsigned)tiles_of(c.classes * (c.features + 1), 256)), dim3(256), 0, st>>>(
        a.part, (int)p.shares, c.classes, c.features, (T*)c.betabar, (T*)c.alphabar);
    return hipGetLastError();
}

} // namespace

// Few features in fp32 or fp64, and classes few enough for the workgroups of a call's rows to walk them all: some
// hundreds, or not many more than the rows
bool gpt_class_narrow(int dtype, int64_t rows, int64_t features, int64_t classes) {
    return (dtype == GPT_F64 || dtype == GPT_F32) && features <= 64 && (classes <= 1024 || classes / 4 <= rows);
}
size_t gpt_class_narrow_workspace(int dtype, int64_t rows, int64_t features, int64_t classes, bool vjp) {
    return dtype == GPT_F64 ? NarrowPlan<double>(rows, features, classes, vjp).bytes : NarrowPlan<float>(rows, features, classes, vjp).bytes;
}
hipError_t gpt_launch_class_narrow(int dtype, const ClassArgs& a, bool vjp, hipStream_t st) {
    return dtype == GPT_F64 ? launch<double>(a, vjp, st) : launch<float>(a, vjp, st);
}
