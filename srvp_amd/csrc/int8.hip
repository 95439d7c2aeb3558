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
    int M, N, K, vecy;
};

// 16 bytes of row `p` from byte k on, zero behind K (rows may start at any byte)
__device__ __forceinline__ u32x4_t bytes16(const signed char* p, int k, int K) {
    u32x4_t v = {0, 0, 0, 0};
    if (k + 16 <= K) __builtin_memcpy(&v, p + k, 16);
    else if (k < K) {
        signed char e[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) e[i] = k + i < K ? p[k + i] : 0;
        __builtin_memcpy(&v, e, 16);
    }
    return v;
}
__device__ __forceinline__ void put(bf16_t* p, float v) { *p = f2bf(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put4(bf16_t* p, const f32x4_t& v) { *reinterpret_cast<uint2*>(p) = make_uint2(pack2bf(v[0], v[1]), pack2bf(v[2], v[3])); }
__device__ __forceinline__ void put4(float* p, const f32x4_t& v) { *reinterpret_cast<f32x4_t*>(p) = v; }

// 128 x 128 outputs a workgroup, 4 waves of 64 x 64; W is the left operand, so that a lane holds 4 neighbouring columns of one row of y.
template <class E>
__global__ __launch_bounds__(256) void int8_tile_kernel(const Int8Args g) {
    constexpr int BK = 64, LD = BK + 16;
    __shared__ __align__(16) signed char lx[128 * LD], lw[128 * LD];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, lg = lane >> 4, ls = lane & 15;
    const int m0 = blockIdx.y * 128, n0 = blockIdx.x * 128, wm = (wv & 1) * 64, wn = (wv >> 1) * 64;
    i32x4_t acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = i32x4_t{0, 0, 0, 0};
    for (int k0 = 0; k0 < g.K; k0 += BK) {
        u32x4_t vx[2], vw[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int idx = i * 256 + tid, row = idx >> 2, k = k0 + (idx & 3) * 16;
            vx[i] = m0 + row < g.M ? bytes16(g.x + (long long)(m0 + row) * g.ldx, k, g.K) : u32x4_t{0, 0, 0, 0};
            vw[i] = n0 + row < g.N ? bytes16(g.w + (long long)(n0 + row) * g.ldw, k, g.K) : u32x4_t{0, 0, 0, 0};
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int idx = i * 256 + tid, row = idx >> 2, k = (idx & 3) * 16;
            *reinterpret_cast<u32x4_t*>(lx + row * LD + k) = vx[i];
            *reinterpret_cast<u32x4_t*>(lw + row * LD + k) = vw[i];
        }
        __syncthreads();
        i32x4_t fx[4], fw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            fx[i] = *reinterpret_cast<const i32x4_t*>(lx + (wm + i * 16 + ls) * LD + lg * 16);
            fw[i] = *reinterpret_cast<const i32x4_t*>(lw + (wn + i * 16 + ls) * LD + lg * 16);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[j], fx[i], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int m = m0 + wm + i * 16 + ls;
        if (m < g.M) {
            const float xs = g.xs[m];
            E* y = (E*)g.y + (long long)m * g.ldy;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int n = n0 + wn + j * 16 + lg * 4;
                f32x4_t o;
#pragma unroll
                for (int r = 0; r < 4; ++r) o[r] = n + r < g.N ? (float)acc[i][j][r] * xs * g.ws[n + r] + (g.bias ? g.bias[n + r] : 0.f) : 0.f;
                if (g.vecy) {
                    if (n < g.N) put4(y + n, o);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n + r < g.N) put(y + n + r, o[r]);
                }
            }
        }
    }
}

}  // namespace

extern "C" int srvp_linear_int8(const srvp_linear_int8_desc* d, void* stream) {
    SRVP_REQUIRE(d, "srvp_linear_int8: null descriptor");
    SRVP_REQUIRE(d->M >= 0 && d->N >= 0 && d->K >= 0, "srvp_linear_int8: negative size");
    SRVP_REQUIRE(d->K <= 131071, "srvp_linear_int8: more than 131071 products could pass 32 bits (K = %d)", d->K);
    if (d->M == 0 || d->N == 0) return SRVP_OK;
    SRVP_REQUIRE((d->K == 0 || (d->x && d->w)) && d->x_scale && d->w_scale && d->y, "srvp_linear_int8: null pointer");
    const int e = d->out_f32 ? 4 : 2;
    Int8Args g;
    g.x = (const signed char*)d->x; g.w = (const signed char*)d->w; g.xs = d->x_scale; g.ws = d->w_scale; g.bias = d->bias; g.y = d->y;
    g.ldx = d->ldx; g.ldw = d->ldw; g.ldy = d->ldy; g.M = d->M; g.N = d->N; g.K = d->K;
    g.vecy = (uintptr_t)d->y % (4 * e) == 0 && d->ldy % 4 == 0 && d->N % 4 == 0;
    SRVP_REQUIRE((d->M + 127) / 128 < 65536, "srvp_linear_int8: too many rows (M = %d)", d->M);
    const dim3 grid((d->N + 127) / 128, (d->M + 127) / 128);
    if (d->out_f32) hipLaunchKernelGGL(int8_tile_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, g);
    else hipLaunchKernelGGL(int8_tile_kernel<bf16_t>, grid, dim3(256), 0, (hipStream_t)stream, g);
    SRVP_CHECK_LAUNCH("srvp_linear_int8");
    return SRVP_OK;
}
