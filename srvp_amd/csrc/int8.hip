// y[m][n] = (sum_k x[m][k] w[n][k]) * x_scale[m] * w_scale[n] + bias[n] on 8-bit integers, the sum exact in 32 bits.
#include "common.h"
#include "../../include/srvp_hip.h"

namespace {

typedef int i32x4_t __attribute__((ext_vector_type(4)));

struct Int8Args {
    const signed char *x, *w;
    const float *xs, *ws, *bias;
    void* y;
    long long ldx, ldw, ldy;
    int M, N, K, vecy, vecy16;      // 4 outputs / 16 bytes of them may be stored together
};

// 16 bytes of row `p` from byte k on, zero behind K (rows may start at any byte; K >= 16: the row's last 16 bytes, moved, are one load)
__device__ __forceinline__ u32x4_t bytes16(const signed char* p, int k, int K) {
    u32x4_t v = {0, 0, 0, 0};
    if (K >= 16) {
        const int at = min(k, K - 16);
        __builtin_memcpy(&v, p + at, 16);
        v = without_low(v, (k - at) * 8);
    } else if (k < K) {
        signed char e[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) e[i] = k + i < K ? p[k + i] : 0;
        __builtin_memcpy(&v, e, 16);
    }
    return v;
}
// the first n bytes of v zero
__device__ __forceinline__ u32x4_t without_first(u32x4_t v, int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int m = n - 4 * i;
        v[i] = m >= 4 ? 0 : m > 0 ? v[i] >> 8 * m << 8 * m : v[i];
    }
    return v;
}
__device__ __forceinline__ void put(bf16_t* p, float v) { *p = f2bf(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put4(bf16_t* p, const f32x4_t& v) { *reinterpret_cast<uint2*>(p) = make_uint2(pack2bf(v[0], v[1]), pack2bf(v[2], v[3])); }
__device__ __forceinline__ void put4(float* p, const f32x4_t& v) { *reinterpret_cast<f32x4_t*>(p) = v; }

// W is the left operand of every product, so that a lane holds 4 neighbouring columns of one row of y.
struct Cols { f32x4_t ws, bias; };
__device__ __forceinline__ Cols cols_of(const Int8Args& g, int n) {
    Cols c;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int at = min(n + r, g.N - 1);
        c.ws[r] = g.ws[at];
        c.bias[r] = g.bias ? g.bias[at] : 0.f;
    }
    return c;
}
template <class E> __device__ __forceinline__ void finish(const Int8Args& g, int m, int n, float xs, const Cols& c, const int* acc) {
    if (m >= g.M) return;
    E* y = (E*)g.y + (long long)m * g.ldy + n;
    f32x4_t o;
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = (float)acc[r] * xs * c.ws[r] + c.bias[r];
    if (g.vecy) {
        if (n < g.N) put4(y, o);
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (n + r < g.N) put(y + r, o[r]);
    }
}

// workgroup -> tile: every XCD owns a contiguous range of tiles (xcd_remap), which walks bands of 8 row tiles down the columns: the 32 tiles in flight on an
// XCD are 8 x 4, and share their operands' rows in its L2
__device__ __forceinline__ void tile_of(unsigned id, unsigned tm, unsigned tn, unsigned& im, unsigned& in) {
    id = xcd_remap(id, tm * tn);
    const unsigned band = id / (8 * tn), rows = min(8u, tm - band * 8), in_band = id - band * 8 * tn;
    im = band * 8 + in_band % rows;
    in = in_band / rows;
}

__device__ __align__(16) signed char zero16[16];

// BM x BN outputs a workgroup of WM x WN waves; rows 16-byte aligned, K a multiple of 16.  Four LDS stages of 64 bytes of k are filled by LDS-DMA three ahead
// of the products; 16-byte chunks are exchanged (chunk ^= (row >> 2) & 3, on the global side: the LDS side of a DMA is linear) so that 16 rows of one chunk lie
// on all 64 banks.  One barrier a stage: behind it every wave has both stage i (its own loads waited for) and left the buffer of stage i + 3.
template <class E, int BM, int BN, int WM, int WN, int STAGES>
__global__ __launch_bounds__(WM * WN * 64, 2) void int8_dma_kernel(const Int8Args g) {
    constexpr int NT = WM * WN * 64, BK = 64, MT = BM / WM / 32, NTL = BN / WN / 32, LA = BM * 4 / NT, LW = BN * 4 / NT;
    typedef int i32x16_t __attribute__((ext_vector_type(16)));
    typedef __attribute__((address_space(1))) const void* gptr_t;
    typedef __attribute__((address_space(3))) void* lptr_t;
    extern __shared__ __align__(16) signed char lds[];       // [stage][BM + BN rows][BK]
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, l32 = lane & 31;
    const int wm = (wid % WM) * (BM / WM), wn = (wid / WM) * (BN / WN);
    unsigned im, in;
    tile_of(blockIdx.x, (g.M + BM - 1) / BM, (g.N + BN - 1) / BN, im, in);
    const int m0 = im * BM, n0 = in * BN;
    // this thread's rows and chunk (the same in every stage)
    const signed char *px[LA], *pw[LW];
    const int chunk = tid & 3;
    int kx[LA], kw[LW];
#pragma unroll
    for (int i = 0; i < LA; ++i) {
        const int row = (i * NT + tid) >> 2;
        kx[i] = (chunk ^ ((row >> 2) & 3)) * 16;
        px[i] = g.x + (long long)min(m0 + row, g.M - 1) * g.ldx + kx[i];
    }
#pragma unroll
    for (int i = 0; i < LW; ++i) {
        const int row = (i * NT + tid) >> 2;
        kw[i] = (chunk ^ ((row >> 2) & 3)) * 16;
        pw[i] = g.w + (long long)min(n0 + row, g.N - 1) * g.ldw + kw[i];
    }
    const int steps = (g.K + BK - 1) / BK;
    auto issue = [&](int s) {
        const int k0 = s * BK;
        signed char* lx = lds + (s % STAGES) * (BM + BN) * BK;
        signed char* lw = lx + BM * BK;
#pragma unroll
        for (int i = 0; i < LA; ++i)
            __builtin_amdgcn_global_load_lds((gptr_t)(k0 + kx[i] < g.K ? px[i] + k0 : zero16), (lptr_t)(lx + (i * NT + wid * 64) * 16), 16, 0, 0);
#pragma unroll
        for (int i = 0; i < LW; ++i)
            __builtin_amdgcn_global_load_lds((gptr_t)(k0 + kw[i] < g.K ? pw[i] + k0 : zero16), (lptr_t)(lw + (i * NT + wid * 64) * 16), 16, 0, 0);
    };
    i32x16_t acc[MT][NTL];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NTL; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
    // byte offset of the lane's chunk of k step ks in row l32 (+ 32 t: the same exchange)
    const int sw = (l32 >> 2) & 3;
    const int off[2] = {l32 * BK + ((half ^ sw) << 4), l32 * BK + (((2 + half) ^ sw) << 4)};
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s)
        if (s < steps) issue(s);
    for (int s = 0; s < steps; ++s) {
        // stage s has landed: all but the loads of the stages behind it; and this wave's reads of the stage before it are back, so its buffer may be filled again
        if (steps - 1 - s >= STAGES - 2) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((STAGES - 2) * (LA + LW)) : "memory");
        else if (STAGES == 4 && steps - 1 - s == 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LA + LW) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (s + STAGES - 1 < steps) issue(s + STAGES - 1);
        const signed char* lx = lds + (s % STAGES) * (BM + BN) * BK;
        const signed char* lw = lx + BM * BK;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            i32x4_t fx[MT], fw[NTL];
#pragma unroll
            for (int i = 0; i < MT; ++i) fx[i] = *reinterpret_cast<const i32x4_t*>(lx + (wm + i * 32) * BK + off[ks]);
#pragma unroll
            for (int j = 0; j < NTL; ++j) fw[j] = *reinterpret_cast<const i32x4_t*>(lw + (wn + j * 32) * BK + off[ks]);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NTL; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[j], fx[i], acc[i][j], 0, 0, 0);
        }
    }
    float xs[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) xs[i] = g.xs[min(m0 + wm + i * 32 + l32, g.M - 1)];
    if (g.vecy16) {
        // whole lines: a wave passes 32 rows at a time through its own part of LDS and stores 16 bytes a lane along the rows (4 columns a lane straight from
        // the registers write a quarter of 32 lines at a time)
        constexpr int CW = NTL * 32, LDE = CW + 16 / sizeof(E), VE = 16 / sizeof(E), PER = CW / VE;
        static_assert(WM * WN * 32 * LDE * (int)sizeof(E) <= STAGES * (BM + BN) * BK, "the rows fit the stages' memory");
        __syncthreads();
        E* my = reinterpret_cast<E*>(lds) + wid * 32 * LDE;
        Cols c[NTL][4];
#pragma unroll
        for (int j = 0; j < NTL; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) c[j][q] = cols_of(g, n0 + wn + j * 32 + 8 * q + 4 * half);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
#pragma unroll
            for (int j = 0; j < NTL; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    f32x4_t o;
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[r] = (float)acc[i][j][4 * q + r] * xs[i] * c[j][q].ws[r] + c[j][q].bias[r];
                    put4(my + l32 * LDE + j * 32 + 8 * q + 4 * half, o);
                }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int k = 0; k < 32 * PER / 64; ++k) {
                const int at = k * 64 + lane, row = at / PER, n = n0 + wn + (at % PER) * VE, m = m0 + wm + i * 32 + row;
                const u32x4_t v = *reinterpret_cast<const u32x4_t*>(my + row * LDE + (at % PER) * VE);
                if (m < g.M && n < g.N) *reinterpret_cast<u32x4_t*>((E*)g.y + (long long)m * g.ldy + n) = v;
            }
            __builtin_amdgcn_wave_barrier();
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < NTL; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int n = n0 + wn + j * 32 + 8 * q + 4 * half;
            const Cols c = cols_of(g, n);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int a[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                finish<E>(g, m0 + wm + i * 32 + l32, n, xs[i], c, a);
            }
        }
}

// BM x BN outputs a workgroup, rows at any byte: 64 bytes of k pass through registers, the next ones under the products (2305 x 1001 x 771: 13 us, 16 steps
// of a latency each; two to four steps in flight: 14).  KG groups of 2 x 2 waves take the
// steps of k in turn, each with its own stages, and their sums (whole numbers: any order) meet in LDS: where there are fewer tiles than the chip takes, the
// steps one behind the other are the time, a latency each.
template <class E, int BM, int BN, int KG>
__global__ __launch_bounds__(256 * KG, KG > 2 ? 1 : 2) void int8_tile_kernel(const Int8Args g) {
    constexpr int BK = 64, LD = BK + 16, MT = BM / 32, NTL = BN / 32, LA = BM * 4 / 256, LW = BN * 4 / 256;
    __shared__ __align__(16) signed char lds[KG][(BM + BN) * LD];
    static_assert(KG / 2 * BM * BN * 4 <= KG * (BM + BN) * LD, "half the groups' sums fit the stages' memory");
    const int tid = threadIdx.x & 255, lane = tid & 63, wv = tid >> 6, lg = lane >> 4, ls = lane & 15, kg = threadIdx.x >> 8;
    signed char *lx = lds[kg], *lw = lx + BM * LD;
    unsigned im, in;
    tile_of(blockIdx.x, (g.M + BM - 1) / BM, (g.N + BN - 1) / BN, im, in);
    const int m0 = im * BM, n0 = in * BN, wm = (wv & 1) * (BM / 2), wn = (wv >> 1) * (BN / 2);
    i32x4_t acc[MT][NTL];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NTL; ++j) acc[i][j] = i32x4_t{0, 0, 0, 0};
    u32x4_t vx[LA], vw[LW];
    const signed char *px[LA], *pw[LW];
    const int kc = (tid & 3) * 16;
#pragma unroll
    for (int i = 0; i < LA; ++i) px[i] = g.x + (long long)min(m0 + ((i * 256 + tid) >> 2), g.M - 1) * g.ldx;      // (rows behind the last: not written)
#pragma unroll
    for (int i = 0; i < LW; ++i) pw[i] = g.w + (long long)min(n0 + ((i * 256 + tid) >> 2), g.N - 1) * g.ldw;
    auto fetch = [&](int k0) {
        if (k0 + BK <= g.K) {
#pragma unroll
            for (int i = 0; i < LA; ++i) __builtin_memcpy(&vx[i], px[i] + k0 + kc, 16);
#pragma unroll
            for (int i = 0; i < LW; ++i) __builtin_memcpy(&vw[i], pw[i] + k0 + kc, 16);
        } else {                                          // (a group's step may lie behind the end: zeros)
#pragma unroll
            for (int i = 0; i < LA; ++i) vx[i] = bytes16(px[i], k0 + kc, g.K);
#pragma unroll
            for (int i = 0; i < LW; ++i) vw[i] = bytes16(pw[i], k0 + kc, g.K);
        }
    };
    fetch(kg * BK);
    for (int k0 = 0; k0 < g.K; k0 += KG * BK) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < LA; ++i) *reinterpret_cast<u32x4_t*>(lx + ((i * 256 + tid) >> 2) * LD + kc) = vx[i];
#pragma unroll
        for (int i = 0; i < LW; ++i) *reinterpret_cast<u32x4_t*>(lw + ((i * 256 + tid) >> 2) * LD + kc) = vw[i];
        __syncthreads();
        if (k0 + KG * BK < g.K) fetch(k0 + (KG + kg) * BK);
        i32x4_t fx[MT], fw[NTL];
#pragma unroll
        for (int i = 0; i < MT; ++i) fx[i] = *reinterpret_cast<const i32x4_t*>(lx + (wm + i * 16 + ls) * LD + lg * 16);
#pragma unroll
        for (int j = 0; j < NTL; ++j) fw[j] = *reinterpret_cast<const i32x4_t*>(lw + (wn + j * 16 + ls) * LD + lg * 16);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NTL; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[j], fx[i], acc[i][j], 0, 0, 0);
    }
    // the upper half of the groups hands its sums to the lower, until one is left
    i32x4_t* sums = reinterpret_cast<i32x4_t*>(lds[0]);
#pragma unroll
    for (int half = KG / 2; half > 0; half /= 2) {
        __syncthreads();
        if (kg >= half && kg < 2 * half)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NTL; ++j) sums[((kg - half) * MT * NTL + i * NTL + j) * 256 + tid] = acc[i][j];
        __syncthreads();
        if (kg < half)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NTL; ++j) acc[i][j] += sums[(kg * MT * NTL + i * NTL + j) * 256 + tid];
    }
    if (kg > 0) return;
    float xs[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) xs[i] = g.xs[min(m0 + wm + i * 16 + ls, g.M - 1)];
#pragma unroll
    for (int j = 0; j < NTL; ++j) {
        const int n = n0 + wn + j * 16 + lg * 4;
        const Cols c = cols_of(g, n);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int a[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
            finish<E>(g, m0 + wm + i * 16 + ls, n, xs[i], c, a);
        }
    }
}

// Few rows (M <= 16 MT): the weight's bytes are the cost (7 x 4096 x 4096: 5.3 us = 3.2 TB/s, the launch included).  A workgroup owns 16 rows of w and all rows of x; its 8 waves deal the steps of 64 bytes of k among
// them, w straight from memory into the fragments, UNROLL steps in flight; the partial sums (whole numbers: any order) meet in LDS.  Other rows than whole vectors
// at borders of 16 bytes: behind the last whole ones the last 16 bytes of a row are read, of both operands, and the bytes already taken are zero in w.  Rows at
// borders of 4 bytes cost little (7 x 4092 x 4096: 6.0), at odd bytes the memory system splits the loads (7 x 4095: 13.3, 64 x 4095 x 4095 37).
template <class E, int MT, bool ALIGNED>
__global__ __launch_bounds__(512) void int8_rows_kernel(const Int8Args g) {
    constexpr int UNROLL = MT == 1 ? 8 : 4;
    __shared__ int red[8][MT * 4 * 64];
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), lg = lane >> 4, ls = lane & 15;
    const int n0 = blockIdx.x * 16;
    const Cols c = cols_of(g, n0 + lg * 4);                  // (early: behind the sums they would be one more memory latency)
    const float xs = wid < MT ? g.xs[min(wid * 16 + ls, g.M - 1)] : 0.f;
    const signed char* w = g.w + (long long)min(n0 + ls, g.N - 1) * g.ldw;
    const signed char* x[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) x[i] = g.x + (long long)min(i * 16 + ls, g.M - 1) * g.ldx;
    i32x4_t acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = i32x4_t{0, 0, 0, 0};
    const int steps = (g.K + 63) / 64;
    for (int s0 = wid; s0 < steps; s0 += 8 * UNROLL) {
        u32x4_t fw[UNROLL], fx[UNROLL][MT];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int k = (s0 + u * 8) * 64 + lg * 16;
            if (ALIGNED) {
                const bool in = k < g.K;
                const int at = in ? k : 0;
                fw[u] = *reinterpret_cast<const u32x4_t*>(w + at);
#pragma unroll
                for (int i = 0; i < MT; ++i) fx[u][i] = *reinterpret_cast<const u32x4_t*>(x[i] + at);
                if (!in) fw[u] = u32x4_t{0, 0, 0, 0};
            } else if (g.K >= 16) {
                const int at = min(k, g.K - 16);
                __builtin_memcpy(&fw[u], w + at, 16);
#pragma unroll
                for (int i = 0; i < MT; ++i) __builtin_memcpy(&fx[u][i], x[i] + at, 16);
                fw[u] = without_first(fw[u], k - at);
            } else {
                fw[u] = bytes16(w, k, g.K);
#pragma unroll
                for (int i = 0; i < MT; ++i) fx[u][i] = bytes16(x[i], k, g.K);
            }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i)
                acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, fw[u]), __builtin_bit_cast(i32x4_t, fx[u][i]), acc[i], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) red[wid][(i * 4 + r) * 64 + lane] = acc[i][r];
    __syncthreads();
    if (wid < MT) {
        const int i = wid;
        int a[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            a[r] = 0;
#pragma unroll
            for (int v = 0; v < 8; ++v) a[r] += red[v][(i * 4 + r) * 64 + lane];
        }
        finish<E>(g, i * 16 + ls, n0 + lg * 4, xs, c, a);
    }
}

template <class E, int BM, int BN, int WM, int WN, int STAGES>
hipError_t dma_launch(const Int8Args& g, hipStream_t st) {
    constexpr int bytes = STAGES * (BM + BN) * 64;
    const auto kern = int8_dma_kernel<E, BM, BN, WM, WN, STAGES>;
    const hipError_t e = hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kern, dim3(((g.M + BM - 1) / BM) * ((g.N + BN - 1) / BN)), dim3(WM * WN * 64), bytes, st, g);
    return hipSuccess;
}
// Which kernel (K = N = 4096, bfloat16 out, us; x the chosen side):
//   rows    7: x 5, 64 x 64 tiles 13    rows   64: x 12, 64 x 64 tiles 14    (up to 64 rows)
//   rows   65: x 14 (64 x 64 tiles, four groups of k), 15 (two), 20 (one); 94 x 6976 x 4544: x 26, 31, 50; 1024 x 1001 x 771: x 10, 10, 11; 192 x 256 x 256: 4.5, 4.0, x 4.0
//              (four groups up to 256 tiles, from 16 steps of 64 on; two up to 512, from 32 steps on: rows 512: x 24, one group 26; 2304 x 256 x 768: 5.2, x 4.9)
//   rows  512: x 24 (64 x 64 tiles), 28 (128 x 128 by DMA)     rows 1024: x 30 (128 x 128 by DMA), 41 (64 x 64)     (by DMA from 192 tiles of 128 x 128 on)
//   rows 3000: x 66 (256 x 256 by DMA), 84 (128 x 128)         rows 2048: x 49 (128 x 128), 61 (256 x 256)          (256 x 256 from 192 such tiles on)
// 8192 x 4096 x 4096: 143 us = 1.92 P operations/s, 8192 x 8192 x 8192: 2.01 P/s; the dense peak is 5, and the large bfloat16 product of the vendor's library
// reaches 56 % of its own here (the package's power limit).
template <class E>
hipError_t launch(const Int8Args& g, bool aligned, hipStream_t st) {
    const long long t256 = (long long)((g.M + 255) / 256) * ((g.N + 255) / 256), t128 = (long long)((g.M + 127) / 128) * ((g.N + 127) / 128);
    if (g.M <= 64) {
        const dim3 grid((g.N + 15) / 16);
#define ROWS(MT)                                                                                                   \
    do {                                                                                                           \
        if (aligned) hipLaunchKernelGGL((int8_rows_kernel<E, MT, true>), grid, dim3(512), 0, st, g);               \
        else hipLaunchKernelGGL((int8_rows_kernel<E, MT, false>), grid, dim3(512), 0, st, g);                      \
    } while (0)
        if (g.M <= 16) ROWS(1);
        else if (g.M <= 32) ROWS(2);
        else ROWS(4);
#undef ROWS
        return hipSuccess;
    }
    if (aligned && t256 >= 192) return dma_launch<E, 256, 256, 2, 4, 4>(g, st);
    if (aligned && t128 >= 192) return dma_launch<E, 128, 128, 2, 2, 4>(g, st);
    if (!aligned && t128 >= 512) {
        hipLaunchKernelGGL((int8_tile_kernel<E, 128, 128, 1>), dim3((unsigned)t128), dim3(256), 0, st, g);
        return hipSuccess;
    }
    const unsigned t64 = (unsigned)(((g.M + 63) / 64) * ((g.N + 63) / 64));
    const int steps = (g.K + 63) / 64, kg = steps >= 16 && t64 <= 256 ? 4 : steps >= 32 && t64 <= 512 ? 2 : 1;
    if (kg == 4) hipLaunchKernelGGL((int8_tile_kernel<E, 64, 64, 4>), dim3(t64), dim3(1024), 0, st, g);
    else if (kg == 2) hipLaunchKernelGGL((int8_tile_kernel<E, 64, 64, 2>), dim3(t64), dim3(512), 0, st, g);
    else hipLaunchKernelGGL((int8_tile_kernel<E, 64, 64, 1>), dim3(t64), dim3(256), 0, st, g);
    return hipSuccess;
}

}  // namespace

extern "C" int srvp_linear_int8(const srvp_linear_int8_desc* d, void* stream) {
    SRVP_REQUIRE(d, "srvp_linear_int8: null descriptor");
    SRVP_REQUIRE(d->M >= 0 && d->N >= 0 && d->K >= 0, "srvp_linear_int8: negative size");
    SRVP_REQUIRE(d->K <= 131071, "srvp_linear_int8: more than 131071 products could pass 32 bits (K = %d)", d->K);
    if (d->M == 0 || d->N == 0) return SRVP_OK;
    SRVP_REQUIRE(d->K > 0, "srvp_linear_int8: K must be positive");
    SRVP_REQUIRE(d->x && d->w && d->x_scale && d->w_scale && d->y, "srvp_linear_int8: null pointer");
    const int e = d->out_f32 ? 4 : 2;
    Int8Args g;
    g.x = (const signed char*)d->x; g.w = (const signed char*)d->w; g.xs = d->x_scale; g.ws = d->w_scale; g.bias = d->bias; g.y = d->y;
    g.ldx = d->ldx; g.ldw = d->ldw; g.ldy = d->ldy; g.M = d->M; g.N = d->N; g.K = d->K;
    g.vecy = (uintptr_t)d->y % (4 * e) == 0 && d->ldy % 4 == 0 && d->N % 4 == 0;
    g.vecy16 = (uintptr_t)d->y % 16 == 0 && d->ldy * e % 16 == 0 && d->N * e % 16 == 0;
    // (a grid is fewer than 2^32 threads: tiles of 128 x 128 for 256 of them, 16 columns for 512)
    SRVP_REQUIRE(((long long)d->M + 63) / 64 * (((long long)d->N + 63) / 64) < (1LL << 25) && d->N <= (1 << 26) && d->M <= (1 << 30), "srvp_linear_int8: too many outputs (%d x %d)", d->M, d->N);
    const bool aligned = d->K % 16 == 0 && d->ldx % 16 == 0 && d->ldw % 16 == 0 && (uintptr_t)d->x % 16 == 0 && (uintptr_t)d->w % 16 == 0;
    const hipError_t err = d->out_f32 ? launch<float>(g, aligned, (hipStream_t)stream) : launch<bf16_t>(g, aligned, (hipStream_t)stream);
    if (err != hipSuccess) {
        srvp_set_error("srvp_linear_int8: %s", hipGetErrorString(err));
        return SRVP_ERR_LAUNCH;
    }
    SRVP_CHECK_LAUNCH("srvp_linear_int8");
    return SRVP_OK;
}
