// Row operators of the temporal networks: rotary positions, and the root-mean-square norm with the residual's addition (forward, backward, and with an
// output in 8 bits).  All of them read every element once and write it once: HBM bandwidth is the bound, the rows stay in registers in between.
#include "common.h"
#include "../../include/srvp_hip.h"

namespace {

// ---------------------------------------------------------------------------------------------------------------------- rotary
// Pair p of a head is turned by positions[t][b] * freq[p] radians.  The angle is formed in 64 bits as a number of whole turns, of which only the
// fraction matters; its sine and cosine are computed once a (row, pair) for all heads of q and k, in LDS.
struct RotArgs {
    const void *x[2];
    void *o[2];
    long long xs[2][3], os[2][3];
    const long long* pos;
    long long pt, pb;
    const double* freq;
    int T, B, H0, H1, D, n, inter, R;      // n pairs; R rows a workgroup
    float sign, mult;
};
constexpr int ROT_TAB = 2048;

template <class E, int VE, bool VEC>
__global__ __launch_bounds__(256) void rotary_kernel(const RotArgs g) {
    __shared__ float tc[ROT_TAB], ts[ROT_TAB];
    const int tid = threadIdx.x;
    const long long rows = (long long)g.T * g.B, row0 = (long long)blockIdx.x * g.R;
    const int R = (int)min((long long)g.R, rows - row0);
    for (int i = tid; i < R * g.n; i += 256) {
        const int r = i / g.n, p = i - r * g.n;
        const long long row = row0 + r, t = row / g.B, b = row - t * g.B;
        double turns = (double)g.pos[t * g.pt + b * g.pb] * (g.freq[p] * 0.15915494309189535);
        turns -= rint(turns);
        float s, c;
        sincospif(2.f * (float)turns, &s, &c);
        tc[i] = c * g.mult;
        ts[i] = s * g.mult * g.sign;
    }
    __syncthreads();
    const int H = g.H0 + g.H1;
    // items of a head: VEC, halves layout: n / VE pairs of vectors, then the rest of the head in vectors; VEC, adjacent pairs: D / VE vectors;
    // otherwise single pairs, then single elements
    const int first = VEC ? (g.inter ? 2 * g.n / VE : g.n / VE) : g.n, items = first + (g.D - 2 * g.n) / (VEC ? VE : 1);
    const int total = R * H * items;
    for (int i = tid; i < total; i += 256) {
        const int it = i % items, rh = i / items, hh = rh % H, r = rh / H;
        const int w = hh >= g.H0, h = w ? hh - g.H0 : hh;
        const long long row = row0 + r, t = row / g.B, b = row - t * g.B;
        const E* x = (const E*)g.x[w] + t * g.xs[w][0] + b * g.xs[w][1] + h * g.xs[w][2];
        E* o = (E*)g.o[w] + t * g.os[w][0] + b * g.os[w][1] + h * g.os[w][2];
        const float *c = tc + r * g.n, *s = ts + r * g.n;
        if constexpr (VEC) {
            typedef u32x4_t vec;
            if (it >= first) {
                const int at = 2 * g.n + (it - first) * VE;
                *reinterpret_cast<vec*>(o + at) = *reinterpret_cast<const vec*>(x + at);
            } else if (g.inter) {
                float u[VE];
                const int at = it * VE, p = at / 2;
                E e[VE];
                *reinterpret_cast<vec*>(e) = *reinterpret_cast<const vec*>(x + at);
#pragma unroll
                for (int j = 0; j < VE; ++j) u[j] = El<E>::ld(e + j);
#pragma unroll
                for (int j = 0; j < VE / 2; ++j) {
                    El<E>::st(e + 2 * j, u[2 * j] * c[p + j] - u[2 * j + 1] * s[p + j]);
                    El<E>::st(e + 2 * j + 1, u[2 * j] * s[p + j] + u[2 * j + 1] * c[p + j]);
                }
                *reinterpret_cast<vec*>(o + at) = *reinterpret_cast<vec*>(e);
            } else {
                const int p = it * VE;
                E e[VE], f[VE];
                *reinterpret_cast<vec*>(e) = *reinterpret_cast<const vec*>(x + p);
                *reinterpret_cast<vec*>(f) = *reinterpret_cast<const vec*>(x + g.n + p);
#pragma unroll
                for (int j = 0; j < VE; ++j) {
                    const float u = El<E>::ld(e + j), v = El<E>::ld(f + j);
                    El<E>::st(e + j, u * c[p + j] - v * s[p + j]);
                    El<E>::st(f + j, u * s[p + j] + v * c[p + j]);
                }
                *reinterpret_cast<vec*>(o + p) = *reinterpret_cast<vec*>(e);
                *reinterpret_cast<vec*>(o + g.n + p) = *reinterpret_cast<vec*>(f);
            }
        } else {
            if (it >= first) {
                o[2 * g.n + it - first] = x[2 * g.n + it - first];
            } else {
                const int a0 = g.inter ? 2 * it : it, a1 = g.inter ? 2 * it + 1 : g.n + it;
                const float u = El<E>::ld(x + a0), v = El<E>::ld(x + a1);
                El<E>::st(o + a0, u * c[it] - v * s[it]);
                El<E>::st(o + a1, u * s[it] + v * c[it]);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------------ norm
//     h = x + residual,  y = h * w / sqrt(mean(h^2) + eps)          sum_out = h
// backward (n = h * rstd):  dh = rstd * (dy w - n mean(dy w n)) + d_sum,   dw = sum over rows of dy n
// of the unrounded sum, which is formed again from x and residual (from a bfloat16 sum the fp32 dw would be off by its rounding, 2e-3), as is its row norm,
// beside the other sum of the row: nothing is kept between the passes but the inputs.
// 8-bit output: row scale s = max|y| / 127, q = round-half-even(h w * (127 / max|h w|)), i.e. y / s: the row's root mean square cancels.  Products and the
// quotient are formed in 64 bits, so q does not depend on the order of any sum.  A row of zeros has scale 0; a row with an infinity or NaN has scale NaN
// and q = 0, i.e. stands for NaN.
// TPR threads (a wave, or a workgroup of 256) hold one row in registers: V vectors of VE elements each.
struct NormArgs {
    const void *x, *res;
    const float* w;
    void *y, *sum;
    signed char* q;
    float* scale;
    long long xs, rs, ys, ss, qs;      // row strides
    long long M;
    int N, vec;
    float eps;
};

template <class E, int VE, int V, int TPR>
__device__ __forceinline__ void row_load(const E* p, int N, int vec, int t, float* f) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = (v * TPR + t) * VE;
        E e[VE];
        if (vec) {
            u32x4_t x = {0, 0, 0, 0};
            if (c < N) x = *reinterpret_cast<const u32x4_t*>(p + c);
            __builtin_memcpy(e, &x, 16);
        } else {
#pragma unroll
            for (int j = 0; j < VE; ++j) e[j] = c + j < N ? p[c + j] : E(0);
        }
#pragma unroll
        for (int j = 0; j < VE; ++j) f[v * VE + j] = El<E>::ld(e + j);
    }
}
template <class E, int VE, int V, int TPR>
__device__ __forceinline__ void row_store(E* p, int N, int vec, int t, const float* f) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = (v * TPR + t) * VE;
        E e[VE];
#pragma unroll
        for (int j = 0; j < VE; ++j) El<E>::st(e + j, f[v * VE + j]);
        if (vec) {
            u32x4_t x;
            __builtin_memcpy(&x, e, 16);
            if (c < N) *reinterpret_cast<u32x4_t*>(p + c) = x;
        } else {
#pragma unroll
            for (int j = 0; j < VE; ++j)
                if (c + j < N) p[c + j] = e[j];
        }
    }
}
// sum over the threads of one row, the same value in all of them
template <int TPR> __device__ __forceinline__ float row_sum(float v, float* red, int tid) {
    v = wave_sum(v);
    if constexpr (TPR == 256) {
        __syncthreads();
        if ((tid & 63) == 0) red[tid >> 6] = v;
        __syncthreads();
        v = (red[0] + red[1]) + (red[2] + red[3]);
    }
    return v;
}
template <int TPR> __device__ __forceinline__ void row_sum2(float& u, float& v, float* red, int tid) {
    u = wave_sum(u);
    v = wave_sum(v);
    if constexpr (TPR == 256) {
        __syncthreads();
        if ((tid & 63) == 0) { red[tid >> 6] = u; red[4 + (tid >> 6)] = v; }
        __syncthreads();
        u = (red[0] + red[1]) + (red[2] + red[3]);
        v = (red[4] + red[5]) + (red[6] + red[7]);
    }
}
template <int TPR> __device__ __forceinline__ double row_max(double v, double* red, int tid) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmax(v, __shfl_xor(v, o));
    if constexpr (TPR == 256) {
        __syncthreads();
        if ((tid & 63) == 0) red[tid >> 6] = v;
        __syncthreads();
        v = fmax(fmax(red[0], red[1]), fmax(red[2], red[3]));
    }
    return v;
}

template <class E, int V, int TPR, bool Q8, bool NORM>
__global__ __launch_bounds__(256) void norm_fwd_kernel(const NormArgs g) {
    constexpr int VE = 16 / sizeof(E);
    __shared__ double redd[4];
    float* red = reinterpret_cast<float*>(redd);
    const int tid = threadIdx.x, t = tid % TPR;
    const long long row = (long long)blockIdx.x * (256 / TPR) + tid / TPR;
    if (row >= g.M) return;                               // (whole waves; with TPR = 256 there is no such workgroup)
    float h[V * VE], r[V * VE];
    row_load<E, VE, V, TPR>((const E*)g.x + row * g.xs, g.N, g.vec, t, h);
    if (g.res) row_load<E, VE, V, TPR>((const E*)g.res + row * g.rs, g.N, g.vec, t, r);
    else {
#pragma unroll
        for (int i = 0; i < V * VE; ++i) r[i] = 0.f;
    }
    float ss = 0.f;
    if constexpr (!Q8) {
#pragma unroll
        for (int i = 0; i < V * VE; ++i) { h[i] += r[i]; ss += h[i] * h[i]; }
        if (g.sum) row_store<E, VE, V, TPR>((E*)g.sum + row * g.ss, g.N, g.vec, t, h);
        const float rstd = 1.f / sqrtf(row_sum<TPR>(ss, red, tid) / (float)g.N + g.eps);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (v * TPR + t) * VE;
#pragma unroll
            for (int j = 0; j < VE; ++j) h[v * VE + j] *= rstd * (c + j < g.N ? g.w[c + j] : 0.f);
        }
        row_store<E, VE, V, TPR>((E*)g.y + row * g.ys, g.N, g.vec, t, h);
    } else {
        double most = 0;
        float wv[V * VE];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (v * TPR + t) * VE;
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                const int i = v * VE + j;
                wv[i] = NORM ? (c + j < g.N ? g.w[c + j] : 0.f) : 1.f;
                const double d = (double)h[i] + (double)r[i];
                ss += (float)d * (float)d;
                most = fmax(most, fabs(d * (double)wv[i]));
            }
        }
        if (g.sum) {
            float s[V * VE];
#pragma unroll
            for (int i = 0; i < V * VE; ++i) s[i] = h[i] + r[i];
            row_store<E, VE, V, TPR>((E*)g.sum + row * g.ss, g.N, g.vec, t, s);
        }
        ss = row_sum<TPR>(ss, red, tid);
        most = row_max<TPR>(most, redd, tid);
        const bool fine = ss < INFINITY && most < (double)INFINITY;      // (false for NaN)
        const double to = fine && most > 0 ? 127.0 / most : 0.0;
        if (t == 0) g.scale[row] = fine ? (float)(most * (NORM ? 1.0 / sqrt((double)ss / g.N + (double)g.eps) : 1.0) / 127.0) : NAN;
        signed char* q = g.q + row * g.qs;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (v * TPR + t) * VE;
            signed char e[VE];
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                const int i = v * VE + j;
                e[j] = fine ? (signed char)(int)rint(((double)h[i] + (double)r[i]) * (double)wv[i] * to) : 0;
            }
            if (g.vec) {
                if (c < g.N) __builtin_memcpy(q + c, e, VE);
            } else {
#pragma unroll
                for (int j = 0; j < VE; ++j)
                    if (c + j < g.N) q[c + j] = e[j];
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
    int N, vec;
    float eps;
};
template <class E, int V, int TPR>
__global__ __launch_bounds__(256) void norm_bwd_kernel(const NormBwdArgs g) {
    constexpr int VE = 16 / sizeof(E), RPW = 256 / TPR;
    __shared__ float red[8];
    __shared__ float cols[RPW > 1 ? RPW * V * TPR * VE : 1];
    const int tid = threadIdx.x, t = tid % TPR;
    float wv[V * VE], dw[V * VE];
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            const int c = (v * TPR + t) * VE + j;
            wv[v * VE + j] = c < g.N ? g.w[c] : 0.f;
            dw[v * VE + j] = 0.f;
        }
    const long long per = (long long)gridDim.x * RPW;
    for (long long row0 = (long long)blockIdx.x * RPW; row0 < g.M; row0 += per) {
        const long long row = row0 + tid / TPR;
        if (row < g.M) {                                  // (whole waves; TPR = 256: always)
            float n[V * VE], d[V * VE], f[V * VE];
            row_load<E, VE, V, TPR>((const E*)g.x + row * g.xs, g.N, g.vec, t, n);
            if (g.res) row_load<E, VE, V, TPR>((const E*)g.res + row * g.rs, g.N, g.vec, t, f);
            row_load<E, VE, V, TPR>((const E*)g.dy + row * g.dys, g.N, g.vec, t, d);
            if (g.res) {
#pragma unroll
                for (int i = 0; i < V * VE; ++i) n[i] += f[i];
            }
            if (g.dsum) row_load<E, VE, V, TPR>((const E*)g.dsum + row * g.dss, g.N, g.vec, t, f);
            float ss = 0.f, dot = 0.f;
#pragma unroll
            for (int i = 0; i < V * VE; ++i) {
                ss += n[i] * n[i];
                dot += d[i] * wv[i] * n[i];
            }
            row_sum2<TPR>(ss, dot, red, tid);
            const float rstd = 1.f / sqrtf(ss / (float)g.N + g.eps);
            dot *= rstd / (float)g.N;
#pragma unroll
            for (int i = 0; i < V * VE; ++i) {
                n[i] *= rstd;
                dw[i] += d[i] * n[i];
                d[i] *= wv[i];
            }
#pragma unroll
            for (int i = 0; i < V * VE; ++i) d[i] = rstd * (d[i] - n[i] * dot) + (g.dsum ? f[i] : 0.f);
            row_store<E, VE, V, TPR>((E*)g.dx + row * g.dxs, g.N, g.vec, t, d);
        }
    }
    if constexpr (RPW > 1) {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int j = 0; j < VE; ++j) cols[(tid / TPR) * V * TPR * VE + (v * TPR + t) * VE + j] = dw[v * VE + j];
        __syncthreads();
        for (int c = tid; c < g.N; c += 256) {
            float s = 0.f;
#pragma unroll
            for (int r = 0; r < RPW; ++r) s += cols[r * V * TPR * VE + c];
            g.part[(long long)blockIdx.x * g.N + c] = s;
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                const int c = (v * TPR + t) * VE + j;
                if (c < g.N) g.part[(long long)blockIdx.x * g.N + c] = dw[v * VE + j];
            }
    }
}
// column sums of the workgroups' partial rows, in a fixed order
__global__ __launch_bounds__(1024) void norm_dw_kernel(const float* __restrict__ part, int n, int N, float* __restrict__ dw) {
    __shared__ float red[16][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), y = threadIdx.x >> 6;
    float s = 0.f;
    if (c < N)
        for (int i = y; i < n; i += 16) s += part[(long long)i * N + c];
    red[y][threadIdx.x & 63] = s;
    __syncthreads();
    if (y == 0 && c < N) {
        s = 0.f;
        for (int i = 0; i < 16; ++i) s += red[i][threadIdx.x];
        dw[c] = s;
    }
}

bool al(const void* p, long long stride, int bytes, int e) { return (uintptr_t)p % bytes == 0 && (stride * e) % bytes == 0; }

template <class E, bool Q8, bool NORM>
void fwd_launch(const NormArgs& g, hipStream_t st) {
    constexpr int VE = 16 / sizeof(E);
    const int N = g.N;
#define ROWS64(V) hipLaunchKernelGGL((norm_fwd_kernel<E, V, 64, Q8, NORM>), dim3((unsigned)((g.M + 3) / 4)), dim3(256), 0, st, g)
#define ROWS256(V) hipLaunchKernelGGL((norm_fwd_kernel<E, V, 256, Q8, NORM>), dim3((unsigned)g.M), dim3(256), 0, st, g)
    if (N <= 64 * VE) ROWS64(1);
    else if (N <= 128 * VE) ROWS64(2);
    else if (N <= 512 * VE) ROWS256(2);
    else if (N <= 1024 * VE) ROWS256(4);
    else if (N <= 2048 * VE) ROWS256(8);
    else ROWS256(16);
#undef ROWS64
#undef ROWS256
}
int bwd_groups(long long M, int N, int VE) {
    const long long rows = N <= 128 * VE ? (M + 3) / 4 : M;
    return (int)(rows < 512 ? rows : 512);
}
template <class E>
void bwd_launch(const NormBwdArgs& g, hipStream_t st) {
    constexpr int VE = 16 / sizeof(E);
    const int N = g.N, n = bwd_groups(g.M, N, VE);
#define GO(V, T) hipLaunchKernelGGL((norm_bwd_kernel<E, V, T>), dim3(n), dim3(256), 0, st, g)
    if (N <= 64 * VE) GO(1, 64);
    else if (N <= 128 * VE) GO(2, 64);
    else if (N <= 512 * VE) GO(2, 256);
    else if (N <= 1024 * VE) GO(4, 256);
    else if (N <= 2048 * VE) GO(8, 256);
    else GO(16, 256);
#undef GO
}
constexpr int NORM_MAX = 16384;

}  // namespace

extern "C" int srvp_rotary(const srvp_rotary_desc* d, void* stream) {
    SRVP_REQUIRE(d, "srvp_rotary: null descriptor");
    SRVP_REQUIRE(d->T >= 0 && d->B >= 0 && d->Hq >= 0 && d->Hk >= 0 && d->D >= 1 && d->pairs >= 0 && 2 * d->pairs <= d->D && d->D <= 4096,
                 "srvp_rotary: bad sizes (heads of 1 to 4096 features, at most half as many pairs)");
    const long long rows = (long long)d->T * d->B;
    if (rows == 0 || d->Hq + d->Hk == 0) return SRVP_OK;
    SRVP_REQUIRE((d->Hq == 0 || (d->q && d->oq)) && (d->Hk == 0 || (d->k && d->ok)) && d->positions && (d->freq || d->pairs == 0), "srvp_rotary: null pointer");
    RotArgs g;
    memset(&g, 0, sizeof(g));
    const int e = d->elem_f32 ? 4 : 2, ve = 16 / e;
    g.x[0] = d->q; g.x[1] = d->k; g.o[0] = d->oq; g.o[1] = d->ok;
    bool vec = d->D % ve == 0 && (d->interleaved ? 2 * d->pairs % ve == 0 : d->pairs % ve == 0);
    for (int i = 0; i < 3; ++i) {
        g.xs[0][i] = d->qs[i]; g.xs[1][i] = d->ks[i]; g.os[0][i] = d->oqs[i]; g.os[1][i] = d->oks[i];
        for (int w = 0; w < 2; ++w)
            if ((w ? d->Hk : d->Hq) > 0) vec = vec && al(g.x[w], g.xs[w][i], 16, e) && al(g.o[w], g.os[w][i], 16, e);
    }
    g.pos = (const long long*)d->positions; g.pt = d->pos_t; g.pb = d->pos_b; g.freq = d->freq;
    g.T = d->T; g.B = d->B; g.H0 = d->Hq; g.H1 = d->Hk; g.D = d->D; g.n = d->pairs; g.inter = d->interleaved;
    g.sign = d->back ? -1.f : 1.f; g.mult = d->magnitude;
    const int n = d->pairs > 0 ? d->pairs : 1;
    int R = 256 / n;                                      // one sine and cosine a thread, ..
    if (R > 16) R = 16;
    if (R < 1) R = 1;
    g.R = R;
    const long long grid = (rows + R - 1) / R;
    SRVP_REQUIRE(grid < (1LL << 31) && (long long)R * (d->Hq + d->Hk) * d->D < (1LL << 31), "srvp_rotary: too many rows or heads");
    hipStream_t st = (hipStream_t)stream;
    if (d->elem_f32) {
        if (vec) hipLaunchKernelGGL((rotary_kernel<float, 4, true>), dim3((unsigned)grid), dim3(256), 0, st, g);
        else hipLaunchKernelGGL((rotary_kernel<float, 4, false>), dim3((unsigned)grid), dim3(256), 0, st, g);
    } else {
        if (vec) hipLaunchKernelGGL((rotary_kernel<bf16_t, 8, true>), dim3((unsigned)grid), dim3(256), 0, st, g);
        else hipLaunchKernelGGL((rotary_kernel<bf16_t, 8, false>), dim3((unsigned)grid), dim3(256), 0, st, g);
    }
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
    g.vec = d->N % ve == 0 && al(d->x, d->xs, 16, e) && (!d->residual || al(d->residual, d->rs, 16, e)) && (!d->sum || al(d->sum, d->ss, 16, e))
            && (d->q8 ? al(d->q8, d->qs, ve, 1) : al(d->y, d->ys, 16, e));
    hipStream_t st = (hipStream_t)stream;
    if (d->q8) {
        if (d->elem_f32) { if (d->w) fwd_launch<float, true, true>(g, st); else fwd_launch<float, true, false>(g, st); }
        else { if (d->w) fwd_launch<bf16_t, true, true>(g, st); else fwd_launch<bf16_t, true, false>(g, st); }
    } else {
        if (d->elem_f32) fwd_launch<float, false, true>(g, st); else fwd_launch<bf16_t, false, true>(g, st);
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
    g.vec = d->N % ve == 0 && al(d->x, d->xs, 16, e) && (!d->residual || al(d->residual, d->rs, 16, e)) && al(d->d_y, d->dys, 16, e) && (!d->d_sum || al(d->d_sum, d->dss, 16, e)) && al(d->dx, d->dxs, 16, e);
    hipStream_t st = (hipStream_t)stream;
    if (d->elem_f32) bwd_launch<float>(g, st); else bwd_launch<bf16_t>(g, st);
    SRVP_CHECK_LAUNCH("srvp_rms_norm_bwd");
    hipLaunchKernelGGL(norm_dw_kernel, dim3((d->N + 63) / 64), dim3(1024), 0, st, (const float*)d->ws, bwd_groups(d->M, d->N, ve), d->N, d->dw);
    SRVP_CHECK_LAUNCH("srvp_rms_norm_bwd(weight)");
    return SRVP_OK;
}
