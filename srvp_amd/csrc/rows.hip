// Row operators of the temporal networks: rotary positions, and the root-mean-square norm with the residual's addition (forward, backward, and with an
// output in 8 bits).  All of them read every element once and write it once: HBM bandwidth is the bound, the rows stay in registers in between.
#include "common.h"
#include "../../include/srvp_hip.h"

namespace {

// ---------------------------------------------------------------------------------------------------------------------- rotary
// Pair p of a head is turned by positions[t][b] * freq[p] radians.  The angle is formed as a number of whole turns in pairs of 64-bit values, of which only the
// fraction matters; its sine and cosine are computed once a (row, pair) for all heads of q and k, in LDS.
struct Div {                               // n / d for n < 2^31 as one high product: m = ceil(2^(32 + s) / d), s = ceil(log2 d) - 1
    unsigned d, m, s;
    __device__ __forceinline__ unsigned of(unsigned n) const { return d == 1 ? n : __umulhi(n, m) >> s; }
};
Div divide(unsigned d) {
    Div r{d, 0, 0};
    if (d > 1) {
        while ((2ull << r.s) < d) ++r.s;
        r.m = (unsigned)(((1ull << (32 + r.s)) + d - 1) / d);
    }
    return r;
}
// pos * freq / (2 pi) without its whole turns, to 2^-52 of a turn for |pos| up to 2^53: every product with its rounding (the fma's) beside it, 1 / (2 pi) in two
// values.  In one value each, the angle would be off by 2.5 * 2^-53 of itself: by more than the sine's own rounding from 10^8 radians on.
__device__ __forceinline__ double fraction_of_turns(double pos, double freq) {
#pragma clang fp contract(off)
    constexpr double c = 0x1.45f306dc9c883p-3, c_rest = -0x1.6b01ec5417056p-57;
    const double w = freq * c, w_rest = fma(freq, c, -w) + freq * c_rest;
    const double t = pos * w, t_rest = fma(pos, w, -t) + pos * w_rest;
    const double r = (t - rint(t)) + t_rest;
    return r - rint(r);
}
struct RotArgs {
    const void *x[2];
    void *o[2];
    long long xs[2][3], os[2][3];
    const long long* pos;
    long long pt, pb;
    const double* freq;
    int T, B, H0, H1, D, n, inter, R;      // n pairs; R rows a workgroup
    Div dB, dn, dH, ditems;
    float sign, mult;
};
constexpr int ROT_TAB = 2048;
enum { SINGLE, HALVES, PAIRS };            // single pairs and elements; 16-byte vectors of the halves layout; 16-byte vectors of adjacent pairs

// (written out, so that a pair has the same bits wherever in a vector it lies)
__device__ __forceinline__ void turn(float& v, float& z, float c, float s) {
    const float a = __builtin_fmaf(v, c, -(z * s)), b = __builtin_fmaf(v, s, z * c);
    v = a;
    z = b;
}
// A head is `first` items that turn (HALVES: two vectors each) and the rest of the head, copied.  A thread has U items' loads in flight.  Vectors are read and
// written at any address; the last one that turns and the last one copied end with their part of the head and share features with the one in front, which both
// write alike (2048 x 4, 16 + 16 heads of 126 bfloat16, us: 27.4; pair by pair 53.4; of 84 18, 38.9; 1024 x 4 heads of 65 float32, 32 of them turned 16.8, 37.9).
template <class E, int VE, int MODE>
__global__ __launch_bounds__(256) void rotary_kernel(const RotArgs g) {
    __shared__ __align__(16) float tc[ROT_TAB], ts[ROT_TAB];
    const int tid = threadIdx.x;
    const long long rows = (long long)g.T * g.B, row0 = (long long)blockIdx.x * g.R;
    const int R = (int)min((long long)g.R, rows - row0);
    for (int i = tid; i < R * g.n; i += 256) {
        const unsigned r = g.dn.of(i), p = i - r * g.n, row = (unsigned)row0 + r, t = g.dB.of(row), b = row - t * g.B;
        const double turns = fraction_of_turns((double)g.pos[t * g.pt + b * g.pb], g.freq[p]);
        float s, c;
        const float near = (float)turns, rest = (float)(turns - (double)near) * 6.28318531f;      // (to the first order: what the fp32 fraction leaves, up to 10^-7 radians)
        sincospif(2.f * near, &s, &c);
        tc[i] = __builtin_fmaf(-s, rest, c) * g.mult;
        ts[i] = __builtin_fmaf(c, rest, s) * g.mult * g.sign;
    }
    __syncthreads();
    const int H = g.H0 + g.H1, items = g.ditems.d, total = R * H * items;
    const int first = MODE == SINGLE ? g.n : ((MODE == HALVES ? g.n : 2 * g.n) + VE - 1) / VE;
    constexpr int U = MODE == SINGLE ? 1 : 4;
    for (int i0 = tid; i0 < total; i0 += 256 * U) {
        const E* x[U];
        E* o[U];
        int it[U], tab[U], at[U];
        u32x4_t e[U], f[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const unsigned i = min(i0 + u * 256, total - 1), rh = g.ditems.of(i), r = g.dH.of(rh), hh = rh - r * H;      // (repeated items write the same)
            it[u] = i - rh * items;
            tab[u] = r * g.n;
            const int w = (int)hh >= g.H0, h = w ? hh - g.H0 : hh;
            const unsigned row = (unsigned)row0 + r, t = g.dB.of(row), b = row - t * g.B;
            x[u] = (const E*)g.x[w] + (long long)t * g.xs[w][0] + (long long)b * g.xs[w][1] + h * g.xs[w][2];
            o[u] = (E*)g.o[w] + (long long)t * g.os[w][0] + (long long)b * g.os[w][1] + h * g.os[w][2];
            if constexpr (MODE != SINGLE) {
                at[u] = it[u] < first ? min(it[u] * VE, (MODE == HALVES ? g.n : 2 * g.n) - VE) : min(2 * g.n + (it[u] - first) * VE, g.D - VE);
                __builtin_memcpy(&e[u], x[u] + at[u], 16);
                if (MODE == HALVES) __builtin_memcpy(&f[u], x[u] + at[u] + (it[u] < first ? g.n : 0), 16);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if constexpr (MODE == SINGLE) {
                if (it[u] >= first) {
                    o[u][2 * g.n + it[u] - first] = x[u][2 * g.n + it[u] - first];
                } else {
                    const int a0 = g.inter ? 2 * it[u] : it[u], a1 = g.inter ? 2 * it[u] + 1 : g.n + it[u];
                    float v = El<E>::ld(x[u] + a0), z = El<E>::ld(x[u] + a1);
                    turn(v, z, tc[tab[u] + it[u]], ts[tab[u] + it[u]]);
                    El<E>::st(o[u] + a0, v);
                    El<E>::st(o[u] + a1, z);
                }
            } else if (it[u] >= first) {
                const int rest = g.D - 2 * g.n;
                if (rest >= VE) {
                    __builtin_memcpy(o[u] + at[u], &e[u], 16);
                } else {                                   // (what turns is not copied over)
                    E a[VE];
                    __builtin_memcpy(a, &e[u], 16);
#pragma unroll
                    for (int j = 1; j < VE; ++j)
                        if (j >= VE - rest) o[u][at[u] + j] = a[j];
                }
            } else if constexpr (MODE == HALVES) {
                const int p = at[u];
                E a[VE], b[VE];
                __builtin_memcpy(a, &e[u], 16);
                __builtin_memcpy(b, &f[u], 16);
#pragma unroll
                for (int j = 0; j < VE; ++j) {
                    float v = El<E>::ld(a + j), z = El<E>::ld(b + j);
                    turn(v, z, tc[tab[u] + p + j], ts[tab[u] + p + j]);
                    El<E>::st(a + j, v);
                    El<E>::st(b + j, z);
                }
                __builtin_memcpy(o[u] + p, a, 16);
                __builtin_memcpy(o[u] + g.n + p, b, 16);
            } else {
                const int p = at[u] / 2;
                E a[VE];
                __builtin_memcpy(a, &e[u], 16);
#pragma unroll
                for (int j = 0; j < VE / 2; ++j) {
                    float v = El<E>::ld(a + 2 * j), z = El<E>::ld(a + 2 * j + 1);
                    turn(v, z, tc[tab[u] + p + j], ts[tab[u] + p + j]);
                    El<E>::st(a + 2 * j, v);
                    El<E>::st(a + 2 * j + 1, z);
                }
                __builtin_memcpy(o[u] + 2 * p, a, 16);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------------ norm
//     h = x + residual,  y = h * w / sqrt(mean(h^2) + eps)          sum_out = h
// (Squares are summed in 32 bits, with 8-bit output in 64: a float32 row above 1.8e19 has an infinite norm in the former.)
// backward (n = h * rstd):  dh = rstd * (dy w - n mean(dy w n)) + d_sum,   dw = sum over rows of dy n
// of the unrounded sum, which is formed again from x and residual (from a bfloat16 sum the fp32 dw would be off by its rounding, 2e-3), as is its row norm,
// beside the other sum of the row: nothing is kept between the passes but the inputs.
// 8-bit output: row scale s = max|y| / 127, q = round-half-even(h w * (127 / max|h w|)), i.e. y / s: the row's root mean square cancels.  Products and the
// quotient are formed in 64 bits, so q does not depend on the order of any sum.  A row of zeros has scale 0; a row of y with an infinity or NaN (its own, or the
// weight's) has scale NaN and q = 0, i.e. stands for NaN.
// TPR threads hold one row in registers: V vectors of VE elements each.
// Measured (us): 16384 x 4096 bfloat16 with a residual forward 84 to 89 = 6.0 TB/s, backward 143 + 5 for dw = 4.7 TB/s; 2304 x 256 float32 3.8, 5.5 + 3.6 (launches);
// 8-bit output 7 x 4096 5.  Rows that are not whole vectors at borders of 16 bytes take the same vectors from any address (one element a load, a value's
// neighbours in the next threads: 16384 x 4095 forward 177, backward 436, 8-bit 246 us, now 125, 172, 134; 16384 x 4096 100, 130, 91).
struct NormArgs {
    const void *x, *res;
    const float* w;
    void *y, *sum;
    signed char* q;
    float* scale;
    long long xs, rs, ys, ss, qs;      // row strides
    long long M;
    int N;
    float eps;
};

// Value i of thread t of a row is column (i / VE * TPR + t) * VE + i % VE.
template <int VE, int TPR> __device__ __forceinline__ int column(int i, int t) { return (i / VE * TPR + t) * VE + i % VE; }

// A row as it lies in memory: the next row's loads are in flight while this one is reduced and written.  VEC: all vectors are whole, at borders of 16 bytes.
// Otherwise they are read from any address and the last one ends with the row, to be put right when it has `arrived`.
template <class E, int VE, int V, int TPR, bool VEC> struct Raw {
    u32x4_t v[V];
    __device__ __forceinline__ void load(const E* p, int N, int t) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = (i * TPR + t) * VE;
            if (VEC || N < VE) v[i] = u32x4_t{0, 0, 0, 0};
            if constexpr (VEC) {
                if (c < N) v[i] = *reinterpret_cast<const u32x4_t*>(p + c);
            } else if (N >= VE) {
                __builtin_memcpy(&v[i], p + min(c, N - VE), 16);
            } else if (c == 0) {
                E e[VE];
#pragma unroll
                for (int j = 0; j < VE; ++j) e[j] = j < N ? p[j] : E(0);
                __builtin_memcpy(&v[i], e, 16);
            }
        }
    }
    __device__ __forceinline__ void arrived(int N, int t) {
        if (VEC || N < VE) return;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = (i * TPR + t) * VE;
            v[i] = without_low(v[i], max(0, c - (N - VE)) * (int)sizeof(E) * 8);
        }
    }
    __device__ __forceinline__ float get(int i) const {      // (unrolled loops only: i is a constant)
        E e[VE];
        __builtin_memcpy(e, &v[i / VE], 16);
        return El<E>::ld(e + i % VE);
    }
};
template <int VE, int V, int TPR> __device__ __forceinline__ void load_weight(const float* w, int N, int t, float* f) {
#pragma unroll
    for (int i = 0; i < V * VE; i += 4) {
        const int c = column<VE, TPR>(i, t);
        if (c + 4 <= N) {
            __builtin_memcpy(f + i, w + c, 16);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) f[i + j] = c + j < N ? w[c + j] : 0.f;
        }
    }
}
template <class E, int VE, int V, int TPR, bool VEC>
__device__ __forceinline__ void row_store(E* p, int N, int t, const float* f) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
        E e[VE];
#pragma unroll
        for (int j = 0; j < VE; ++j) El<E>::st(e + j, f[v * VE + j]);
        const int c = (v * TPR + t) * VE;
        if constexpr (VEC) {
            u32x4_t x;
            __builtin_memcpy(&x, e, 16);
            if (c < N) *reinterpret_cast<u32x4_t*>(p + c) = x;
        } else if (c + VE <= N) {
            __builtin_memcpy(p + c, e, 16);
        } else {
#pragma unroll
            for (int j = 0; j < VE; ++j)
                if (c + j < N) p[c + j] = e[j];
        }
    }
}
// two sums over the threads of one row, the same values in all of them; `red`: 2 TPR / 64 floats
template <int TPR> __device__ __forceinline__ void row_sum(float& u, float& v, float* red, int tid) {
    u = wave_sum(u);
    v = wave_sum(v);
    if constexpr (TPR > 64) {
        constexpr int NW = TPR / 64;
        __syncthreads();
        if ((tid & 63) == 0) { red[tid >> 6] = u; red[NW + (tid >> 6)] = v; }
        __syncthreads();
        u = v = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) { u += red[i]; v += red[NW + i]; }
    }
}
template <int TPR, class F> __device__ __forceinline__ F row_sum(F u, F* red, int tid) {
    if constexpr (sizeof(F) == 8) u = wave_sum_d(u);
    else u = wave_sum(u);
    if constexpr (TPR > 64) {
        __syncthreads();
        if ((tid & 63) == 0) red[tid >> 6] = u;
        __syncthreads();
        u = 0;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) u += red[i];
    }
    return u;
}
template <int TPR> __device__ __forceinline__ double row_max(double v, double* red, int tid) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmax(v, __shfl_xor(v, o));
    if constexpr (TPR > 64) {
        __syncthreads();
        if ((tid & 63) == 0) red[tid >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int i = 1; i < TPR / 64; ++i) v = fmax(v, red[i]);
    }
    return v;
}

template <class E, int V, int TPR, bool Q8, bool NORM, bool VEC>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_fwd_kernel(const NormArgs g) {
    constexpr int VE = 16 / sizeof(E), NT = TPR > 256 ? TPR : 256, RPW = NT / TPR;
    __shared__ double redd[NT / 64];
    float* red = reinterpret_cast<float*>(redd);
    const int tid = threadIdx.x, t = tid % TPR;
    float wv[V * VE];
    if (NORM) load_weight<VE, V, TPR>(g.w, g.N, t, wv);
    Raw<E, VE, V, TPR, VEC> x, r;
    const long long step = (long long)gridDim.x * RPW;
    long long row = (long long)blockIdx.x * RPW + tid / TPR;
    auto fetch = [&](long long at) {
        x.load((const E*)g.x + at * g.xs, g.N, t);
        if (g.res) r.load((const E*)g.res + at * g.rs, g.N, t);
    };
    if (row < g.M) fetch(row);
    // the exponent of NaN if a weight of this wave's is NaN or infinite, which leaves no row finite (fmax passes over a NaN): put over the row's sum of squares
    unsigned wild = 0;
    if constexpr (Q8 && NORM) {
        float x = 0.f;
#pragma unroll
        for (int i = 0; i < V * VE; ++i) x += 0.f * wv[i];
        wild = __builtin_amdgcn_readfirstlane(__any(!(x == 0.f)) ? 0x7ff80000u : 0u);
    }
    for (; row < g.M; row += step) {                       // (the same for all threads of a row, and of a workgroup whose waves meet)
        x.arrived(g.N, t);
        if (g.res) r.arrived(g.N, t);
        float h[V * VE];
        double hd[Q8 ? V * VE : 1];
#pragma unroll
        for (int i = 0; i < V * VE; ++i) {
            const float u = x.get(i), v = g.res ? r.get(i) : 0.f;
            h[i] = u + v;
            if (Q8) hd[i] = (double)u + (double)v;
        }
        if (row + step < g.M) fetch(row + step);
        if (g.sum) row_store<E, VE, V, TPR, VEC>((E*)g.sum + row * g.ss, g.N, t, h);
        if constexpr (!Q8) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < V * VE; ++i) ss += h[i] * h[i];
            const float rstd = 1.f / sqrtf(row_sum<TPR>(ss, red, tid) / (float)g.N + g.eps);
#pragma unroll
            for (int i = 0; i < V * VE; ++i) h[i] *= rstd * wv[i];
            row_store<E, VE, V, TPR, VEC>((E*)g.y + row * g.ys, g.N, t, h);
        } else {
            double most = 0, ss = 0;                       // (the squares in 64 bits too: a row of 1e20s is not an infinite one)
#pragma unroll
            for (int i = 0; i < V * VE; ++i) {
                ss += hd[i] * hd[i];
                if (NORM) hd[i] *= (double)wv[i];
                most = fmax(most, fabs(hd[i]));
            }
            if (NORM) ss = __hiloint2double(__double2hiint(ss) | wild, __double2loint(ss));
            ss = row_sum<TPR>(ss, redd, tid);
            most = row_max<TPR>(most, redd, tid);
            const bool fine = ss < (double)INFINITY && most < (double)INFINITY;      // (false for NaN)
            const double to = fine && most > 0 ? 127.0 / most : 0.0;
            if (t == 0) g.scale[row] = fine ? (float)(most * (NORM ? 1.0 / sqrt(ss / g.N + (double)g.eps) : 1.0) / 127.0) : NAN;
            signed char* q = g.q + row * g.qs;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                signed char e[VE];
#pragma unroll
                for (int j = 0; j < VE; ++j) e[j] = fine ? (signed char)(int)rint(hd[v * VE + j] * to) : 0;
                const int c = (v * TPR + t) * VE;
                if (c + VE <= g.N) {
                    __builtin_memcpy(q + c, e, VE);
                } else {
#pragma unroll
                    for (int j = 0; j < VE; ++j)
                        if (c + j < g.N) q[c + j] = e[j];
                }
            }
        }
    }
}

struct NormBwdArgs {
    const void *x, *res, *dy, *dsum;
    const float* w;
    void* dx;
    float* part;                      // [workgroup][N] sums of dy * n over the workgroup's rows
    long long xs, rs, dys, dss, dxs;
    long long M;
    int N;
    float eps;
};
template <class E, int V, int TPR, bool VEC>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_bwd_kernel(const NormBwdArgs g) {
    constexpr int VE = 16 / sizeof(E), NT = TPR > 256 ? TPR : 256, RPW = NT / TPR;
    __shared__ float red[NT / 32];
    __shared__ float cols[RPW > 1 ? NT * V * VE : 1];
    const int tid = threadIdx.x, t = tid % TPR;
    float wv[V * VE], dw[V * VE];
    load_weight<VE, V, TPR>(g.w, g.N, t, wv);
#pragma unroll
    for (int i = 0; i < V * VE; ++i) dw[i] = 0.f;
    Raw<E, VE, V, TPR, VEC> x, r, dy, ds;
    const long long step = (long long)gridDim.x * RPW;
    long long row = (long long)blockIdx.x * RPW + tid / TPR;
    auto fetch = [&](long long at) {
        x.load((const E*)g.x + at * g.xs, g.N, t);
        if (g.res) r.load((const E*)g.res + at * g.rs, g.N, t);
        dy.load((const E*)g.dy + at * g.dys, g.N, t);
        if (g.dsum) ds.load((const E*)g.dsum + at * g.dss, g.N, t);
    };
    if (row < g.M) fetch(row);
    for (; row < g.M; row += step) {
        x.arrived(g.N, t);
        if (g.res) r.arrived(g.N, t);
        dy.arrived(g.N, t);
        if (g.dsum) ds.arrived(g.N, t);
        float n[V * VE], d[V * VE], f[V * VE];
        float ss = 0.f, dot = 0.f;
#pragma unroll
        for (int i = 0; i < V * VE; ++i) {
            n[i] = x.get(i) + (g.res ? r.get(i) : 0.f);
            d[i] = dy.get(i);
            f[i] = g.dsum ? ds.get(i) : 0.f;
            ss += n[i] * n[i];
            dot += d[i] * wv[i] * n[i];
        }
        if (row + step < g.M) fetch(row + step);
        row_sum<TPR>(ss, dot, red, tid);
        const float rstd = 1.f / sqrtf(ss / (float)g.N + g.eps);
        dot *= rstd / (float)g.N;
#pragma unroll
        for (int i = 0; i < V * VE; ++i) {
            n[i] *= rstd;
            dw[i] += d[i] * n[i];
            d[i] = rstd * (d[i] * wv[i] - n[i] * dot) + f[i];
        }
        row_store<E, VE, V, TPR, VEC>((E*)g.dx + row * g.dxs, g.N, t, d);
    }
    float* part = g.part + (long long)blockIdx.x * g.N;
    if constexpr (RPW > 1) {
#pragma unroll
        for (int i = 0; i < V * VE; ++i) cols[(tid / TPR) * V * TPR * VE + column<VE, TPR>(i, t)] = dw[i];
        __syncthreads();
        for (int c = tid; c < g.N; c += NT) {
            float s = 0.f;
#pragma unroll
            for (int k = 0; k < RPW; ++k) s += cols[k * V * TPR * VE + c];
            part[c] = s;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V * VE; i += 4) {
            const int c = column<VE, TPR>(i, t);
            if (c + 4 <= g.N) {
                __builtin_memcpy(part + c, dw + i, 16);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c + j < g.N) part[c + j] = dw[i + j];
            }
        }
    }
}
// column sums of the workgroups' partial rows, in a fixed order: 16 columns (64 bytes) a workgroup, so that a narrow weight still fills some of the chip
__global__ __launch_bounds__(1024) void norm_dw_kernel(const float* __restrict__ part, int n, int N, float* __restrict__ dw) {
    __shared__ float red[64][17];
    const int x = threadIdx.x & 15, c = blockIdx.x * 16 + x, y = threadIdx.x >> 4;
    float s = 0.f;
    if (c < N) {
        float a[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        for (int i = y; i < n; i += 512) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (i + k * 64 < n) a[k] += part[(long long)(i + k * 64) * N + c];
        }
        s = ((a[0] + a[1]) + (a[2] + a[3])) + ((a[4] + a[5]) + (a[6] + a[7]));
    }
    red[y][x] = s;
    __syncthreads();
    if (y == 0 && c < N) {
        float a[8];                                        // (in eights and pairs: one behind the other, 64 sums would put a quarter more on dw than its terms)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float b[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) b[i] = red[i * 8 + k][x];
            a[k] = ((b[0] + b[1]) + (b[2] + b[3])) + ((b[4] + b[5]) + (b[6] + b[7]));
        }
        dw[c] = ((a[0] + a[1]) + (a[2] + a[3])) + ((a[4] + a[5]) + (a[6] + a[7]));
    }
}

bool al(const void* p, long long stride, int bytes, int e) { return (uintptr_t)p % bytes == 0 && (stride * e) % bytes == 0; }

// Threads of a row, so that its values stay in registers: a wave up to 128 vectors of 16 bytes (1024 bfloat16 / 512 float32 features), a workgroup of 256
// up to 512, 512 up to 2048 (with four vectors a thread), 1024 for the widest.  Workgroups walk rows: the next row is in flight and the weight stays.  16384 x
// 4096 bfloat16 with a residual: forward 88 us at 1024 workgroups, 93 at 2048, 156 with one a row; backward (512; 768: 149, 1024: 142 + 15 for dw) 144 us.
#define NORM_ROWS(GO)                              \
    do {                                           \
        if (N <= 64 * VE) GO(1, 64);               \
        else if (N <= 128 * VE) GO(2, 64);         \
        else if (N <= 256 * VE) GO(1, 256);        \
        else if (N <= 512 * VE) GO(2, 256);        \
        else if (N <= 1024 * VE) GO(2, 512);       \
        else if (N <= 2048 * VE) GO(4, 512);       \
        else if constexpr (VE == 4) GO(4, 1024);   \
    } while (0)

template <class E, bool Q8, bool NORM, bool VEC>
void fwd_go(const NormArgs& g, hipStream_t st) {
    constexpr int VE = 16 / sizeof(E);
    const int N = g.N;
    const long long rows = N <= 128 * VE ? (g.M + 3) / 4 : g.M;
    const dim3 grid((unsigned)(rows < 1024 ? rows : 1024));
#define GO(V, T) hipLaunchKernelGGL((norm_fwd_kernel<E, V, T, Q8, NORM, VEC>), grid, dim3(T > 256 ? T : 256), 0, st, g)
    NORM_ROWS(GO);
#undef GO
}
template <class E, bool Q8, bool NORM>
void fwd_launch(const NormArgs& g, bool vec, hipStream_t st) { vec ? fwd_go<E, Q8, NORM, true>(g, st) : fwd_go<E, Q8, NORM, false>(g, st); }
int bwd_groups(long long M, int N, int VE) {
    const long long rows = N <= 128 * VE ? (M + 3) / 4 : M;
    const int most = N <= 128 * VE ? 256 : 512;
    return (int)(rows < most ? rows : most);
}
template <class E, bool VEC>
void bwd_go(const NormBwdArgs& g, hipStream_t st) {
    constexpr int VE = 16 / sizeof(E);
    const int N = g.N, n = bwd_groups(g.M, N, VE);
#define GO(V, T) hipLaunchKernelGGL((norm_bwd_kernel<E, V, T, VEC>), dim3(n), dim3(T > 256 ? T : 256), 0, st, g)
    NORM_ROWS(GO);
#undef GO
}
template <class E>
void bwd_launch(const NormBwdArgs& g, bool vec, hipStream_t st) { vec ? bwd_go<E, true>(g, st) : bwd_go<E, false>(g, st); }
constexpr int NORM_MAX = 16384;

}  // namespace

extern "C" int srvp_rotary(const srvp_rotary_desc* d, void* stream) {
    SRVP_REQUIRE(d, "srvp_rotary: null descriptor");
    SRVP_REQUIRE(d->T >= 0 && d->B >= 0 && d->Hq >= 0 && d->Hk >= 0 && d->Hq < (1 << 20) && d->Hk < (1 << 20) && d->D >= 1 && d->pairs >= 0 && 2 * d->pairs <= d->D && d->D <= 4096,
                 "srvp_rotary: bad sizes (fewer than 2^20 heads of 1 to 4096 features, at most half as many pairs)");
    const long long rows = (long long)d->T * d->B;
    if (rows == 0 || d->Hq + d->Hk == 0) return SRVP_OK;
    SRVP_REQUIRE((d->Hq == 0 || (d->q && d->oq)) && (d->Hk == 0 || (d->k && d->ok)) && d->positions && (d->freq || d->pairs == 0), "srvp_rotary: null pointer");
    RotArgs g;
    memset(&g, 0, sizeof(g));
    const int e = d->elem_f32 ? 4 : 2, ve = 16 / e;
    g.x[0] = d->q; g.x[1] = d->k; g.o[0] = d->oq; g.o[1] = d->ok;
    // vectors where what turns holds at least one (nothing turns: the head)
    const int half = d->interleaved ? 2 * d->pairs : d->pairs, rest = d->D - 2 * d->pairs;
    const bool vec = half > 0 ? half >= ve : d->D >= ve;
    for (int i = 0; i < 3; ++i) { g.xs[0][i] = d->qs[i]; g.xs[1][i] = d->ks[i]; g.os[0][i] = d->oqs[i]; g.os[1][i] = d->oks[i]; }
    g.pos = (const long long*)d->positions; g.pt = d->pos_t; g.pb = d->pos_b; g.freq = d->freq;
    g.T = d->T; g.B = d->B; g.H0 = d->Hq; g.H1 = d->Hk; g.D = d->D; g.n = d->pairs; g.inter = d->interleaved;
    g.sign = d->back ? -1.f : 1.f; g.mult = d->magnitude;
    // rows a workgroup: one sine and cosine a thread, at most 64 KB (16 items a thread).  2048 x 4, 16 + 16 heads of 128, bfloat16, us, half and all of it turned: 22.8 and 21.1
    // (5.9, 6.4 TB/s; tensors of 34 MB, partly from cache: half of it turned from memory 26); 16 KB 25.7, 21.7; one row 33.6, 38.7; two sines a thread 25.3, 22.2; four 25.3, 24.5 (but 4096 x 3, 2 + 2
    // heads of 256, where the sines are the cost: 22, two 20, four 15)
    const int n = d->pairs > 0 ? d->pairs : 1, H = d->Hq + d->Hk;
    long long R = (256 + n - 1) / n, most = 65536LL / ((long long)H * d->D * e) + 1;
    if (R > most) R = most;
    if (R < (rows >> 23) + 1) R = (rows >> 23) + 1;       // (a grid is fewer than 2^24 workgroups)
    if (R * n > ROT_TAB) R = ROT_TAB / n;
    if (R < 1) R = 1;
    g.R = (int)R;
    const int items = vec ? (half + ve - 1) / ve + (rest + ve - 1) / ve : d->pairs + rest;
    const long long grid = (rows + R - 1) / R;
    SRVP_REQUIRE(rows < (1LL << 31) && grid < (1 << 24) && R * H * items < (1LL << 30), "srvp_rotary: too many rows or heads");
    SRVP_REQUIRE((d->Hq == 0 || d->q != d->oq) && (d->Hk == 0 || d->k != d->ok), "srvp_rotary: an output in the place of its input");
    g.dB = divide(d->B); g.dn = divide(n); g.dH = divide(H); g.ditems = divide(items);
    hipStream_t st = (hipStream_t)stream;
#define ROTARY(E, VE, MODE) hipLaunchKernelGGL((rotary_kernel<E, VE, MODE>), dim3((unsigned)grid), dim3(256), 0, st, g)
    if (d->elem_f32) { if (!vec) ROTARY(float, 4, SINGLE); else if (d->interleaved) ROTARY(float, 4, PAIRS); else ROTARY(float, 4, HALVES); }
    else { if (!vec) ROTARY(bf16_t, 8, SINGLE); else if (d->interleaved) ROTARY(bf16_t, 8, PAIRS); else ROTARY(bf16_t, 8, HALVES); }
#undef ROTARY
    SRVP_CHECK_LAUNCH("srvp_rotary");
    return SRVP_OK;
}

static int norm_check(const srvp_rms_norm_desc* d, const char* who) {
    SRVP_REQUIRE(d, "%s: null descriptor", who);
    SRVP_REQUIRE(d->M >= 0 && d->M < (1LL << 31) && d->N >= 1 && d->N <= NORM_MAX, "%s: rows of 1 to %d features (got %d), fewer than 2^31 rows", who, NORM_MAX, d->N);
    return SRVP_OK;
}

extern "C" int srvp_rms_norm(const srvp_rms_norm_desc* d, void* stream) {
    if (int rc = norm_check(d, "srvp_rms_norm")) return rc;
    if (d->M == 0) return SRVP_OK;
    SRVP_REQUIRE(d->x && (d->q8 ? d->scale != nullptr : (d->w && d->y)), "srvp_rms_norm: null pointer");
    NormArgs g;
    g.x = d->x; g.res = d->residual; g.w = d->w; g.y = d->y; g.sum = d->sum; g.q = (signed char*)d->q8; g.scale = d->scale;
    g.xs = d->xs; g.rs = d->rs; g.ys = d->ys; g.ss = d->ss; g.qs = d->qs; g.M = d->M; g.N = d->N; g.eps = d->eps;
    const int e = d->elem_f32 ? 4 : 2, ve = 16 / e;
    const bool vec = d->N % ve == 0 && al(d->x, d->xs, 16, e) && (!d->residual || al(d->residual, d->rs, 16, e)) && (!d->sum || al(d->sum, d->ss, 16, e))
            && (d->q8 ? al(d->q8, d->qs, ve, 1) : al(d->y, d->ys, 16, e));
    hipStream_t st = (hipStream_t)stream;
    if (d->q8) {
        if (d->elem_f32) { if (d->w) fwd_launch<float, true, true>(g, vec, st); else fwd_launch<float, true, false>(g, vec, st); }
        else { if (d->w) fwd_launch<bf16_t, true, true>(g, vec, st); else fwd_launch<bf16_t, true, false>(g, vec, st); }
    } else {
        if (d->elem_f32) fwd_launch<float, false, true>(g, vec, st); else fwd_launch<bf16_t, false, true>(g, vec, st);
    }
    SRVP_CHECK_LAUNCH("srvp_rms_norm");
    return SRVP_OK;
}

extern "C" int64_t srvp_rms_norm_bwd_ws_bytes(int64_t M, int32_t N, int32_t elem_f32) {
    return M <= 0 ? 0 : (int64_t)bwd_groups(M, N, elem_f32 ? 4 : 8) * N * 4;
}

extern "C" int srvp_rms_norm_bwd(const srvp_rms_norm_bwd_desc* d, void* stream) {
    SRVP_REQUIRE(d, "srvp_rms_norm_bwd: null descriptor");
    SRVP_REQUIRE(d->M >= 1 && d->M < (1LL << 31) && d->N >= 1 && d->N <= NORM_MAX, "srvp_rms_norm_bwd: rows of 1 to %d features (got %d), 1 to 2^31 - 1 rows", NORM_MAX, d->N);
    SRVP_REQUIRE(d->x && d->d_y && d->w && d->dx && d->dw && d->ws, "srvp_rms_norm_bwd: null pointer");
    SRVP_REQUIRE(d->ws_bytes >= srvp_rms_norm_bwd_ws_bytes(d->M, d->N, d->elem_f32), "srvp_rms_norm_bwd: workspace too small");
    NormBwdArgs g;
    g.x = d->x; g.res = d->residual; g.dy = d->d_y; g.dsum = d->d_sum; g.w = d->w; g.dx = d->dx; g.part = (float*)d->ws;
    g.xs = d->xs; g.rs = d->rs; g.dys = d->dys; g.dss = d->dss; g.dxs = d->dxs; g.M = d->M; g.N = d->N; g.eps = d->eps;
    const int e = d->elem_f32 ? 4 : 2, ve = 16 / e;
    const bool vec = d->N % ve == 0 && al(d->x, d->xs, 16, e) && (!d->residual || al(d->residual, d->rs, 16, e)) && al(d->d_y, d->dys, 16, e) && (!d->d_sum || al(d->d_sum, d->dss, 16, e)) && al(d->dx, d->dxs, 16, e);
    hipStream_t st = (hipStream_t)stream;
    if (d->elem_f32) bwd_launch<float>(g, vec, st); else bwd_launch<bf16_t>(g, vec, st);
    SRVP_CHECK_LAUNCH("srvp_rms_norm_bwd");
    hipLaunchKernelGGL(norm_dw_kernel, dim3((d->N + 15) / 16), dim3(1024), 0, st, (const float*)d->ws, bwd_groups(d->M, d->N, ve), d->N, d->dw);
    SRVP_CHECK_LAUNCH("srvp_rms_norm_bwd(weight)");
    return SRVP_OK;
}
