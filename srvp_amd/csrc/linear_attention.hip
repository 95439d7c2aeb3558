// Linear attention with a decay for each head, over time-major tensors (T, B, H, D):
//
//     S_t = a_h S_{t-1} + k_t v_t^T          (Dk x Dv, fp32)          o_t = scale * q_t S_t
//
// Chunked form.  Within a chunk of C tokens (index i, decay a, state S in front of it)
//
//     o_i = scale * ( sum_{j <= i} a^(i-j) (q_i . k_j) v_j  +  a^(i+1) q_i S ),        S' = a^C S + sum_j a^(C-1-j) k_j v_j^T
//
// so a chunk is four matrix products on the matrix cores and the recurrence advances once a chunk.  The gradients are the same sum with its
// operands exchanged and, for two of them, time reversed:
//
//     dq_i = scale * sum_{j <= i} a^(i-j) (do_i . v_j) k_j  +  scale a^(i+1) do_i S_0^T
//     dv_j = scale * sum_{i >= j} a^(i-j) (k_j . q_i) do_i  +  a^(n-1-j) k_j dS_n          dk_j: (v, do, q) and dS_n^T
//     dS_0 = scale * sum_i a^(i+1) q_i do_i^T + a^n dS_n
//
// One kernel (scan_kernel) therefore serves forward and backward: a "role" names its operands a, b, c, the output, the direction and where the
// carried state comes from and goes to.  In reversed time the carry is taken after its decay (X_t = a R_t), which moves the two exponents by one
// (`e` below) and leaves no division by a.  No power of a is ever formed with a negative exponent: a = 0 (log_decay = -inf) is an ordinary value.
#include "common.h"
#include "../../include/srvp_hip.h"

namespace {

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));
// what is written in front stays in front (arithmetic may pass): keeps reads of LDS ahead of the products that hide them
#define PIN __builtin_amdgcn_sched_barrier(0x6)
typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));

struct Operand {
    const void* p;
    long long st, sb, sh;      // elements between tokens, sequences, heads
    int d;                     // features
    int vec;                   // 16-byte loads allowed
};

struct Role {
    Operand a, b, c;
    void* o;
    long long ot, ob, oh;
    int ovec;
    int rev;                   // time runs backwards
    const float* init;         // carry in front of the first token [b][h][...], or null
    const float* prefix;       // carry in front of every segment [b][h][seg][...], or null (one segment)
    float* fin;                // carry behind the last token, or null
    int init_a, init_c;        // strides of all three (elements of a, of c)
    float init_mul, fin_mul;
};

struct ScanArgs {
    Role r[3];
    int nroles;
    const float* log_decay;
    const long long* lengths;
    int T, B, H, nseg, seg_len, ncb;
    float scale;
    float* part;               // state-only launch: segment sums [role][b][h][seg][da][dc]
};

__device__ __forceinline__ float dpow(float l2, int n) { return n <= 0 ? 1.f : exp2f(l2 * (float)n); }      // decay^n, n >= 0 (0^0 = 1)

// ---- the two element types.  KS = contraction elements of one step; lane (g = lane >> 4, s = lane & 15) holds KS/4 of them, of row / column s.
//
// Over features (scores, a S): bf16 8g .. 8g+7 of every 32, 16 bytes of a row.  The state's tiles lie so that they are the next product's operand without
// leaving the registers: a 16x16 accumulator has rows 4g .. 4g+3 in lane group g, so tiles 2d and 2d+1 are given the features 32d + 8g + {0..3} and {4..7}
// (`feature`).  Columns likewise where a wave owns 32 of them (`col_of`): a lane's two tiles are 8 neighbouring columns of the output, 16 bytes.
// Over tokens: 4g .. 4g+3 and 16 + 4g .. of every 32, what a transposing read gives; the scores are laid down in that order.
// fp32: 4g .. 4g+3 of every 16, everything in its natural place.
//
// View<E, W>: a tile of W features a row in LDS, read as fragments along its rows (contraction over features) and across them (over tokens).
// bf16: 16-byte units, exchanged within every 256 bytes (128 for W = 64) by unit ^= swz(row).  16 lanes read one unit of 16 rows, write whole rows, or
// (ds_read_b64_tr_b16) read half of 4 units of 4 rows: all of them touch every bank at most once.  fp32: rows padded by 16 bytes.
template <class E> struct Ty;
template <class E, int W> struct View;

template <> struct Ty<bf16_t> {
    static constexpr int KS = 32, TPK = 2, C = 64, VE = 8;
    typedef s16x8_t frag;
    static __device__ __forceinline__ int feature(int tile, int g) { return (tile >> 1) * 32 + g * 8 + (tile & 1) * 4; }      // of row 4g of a tile
    template <int NCT> static __device__ __forceinline__ int col_of(int w, int ct, int i) { return NCT == 2 ? w * 32 + (i >> 2) * 8 + ct * 4 + (i & 3) : w * 16 + i; }
    static __device__ __forceinline__ float value(bf16_t x) { return bf2f(x); }
    // whether an element is NaN or infinite (the exponent's bits and one more carry into the sign's)
    static __device__ __forceinline__ unsigned wild(const frag& x) {
        const u32x4_t v = __builtin_bit_cast(u32x4_t, x), y = (v & 0x7fff7fffu) + 0x00800080u;
        return (y.x | y.y | y.z | y.w) & 0x80008000u;
    }
    static __device__ __forceinline__ frag tame(frag x) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (x[i] & 0x7f80) == 0x7f80 ? 0 : x[i];
        return x;
    }
    static __device__ __forceinline__ frag pack(const f32x4_t* t) {
        u32x4_t v;
        v.x = pack2bf(t[0][0], t[0][1]); v.y = pack2bf(t[0][2], t[0][3]);
        v.z = pack2bf(t[1][0], t[1][1]); v.w = pack2bf(t[1][2], t[1][3]);
        return __builtin_bit_cast(frag, v);
    }
    // 8 values as the sum of two bf16 terms (to 2^-17 of each)
    static __device__ __forceinline__ void terms(const f32x4_t* t, frag* out) {
        out[0] = pack(t);
        float h[8];
        unpack8(__builtin_bit_cast(u32x4_t, out[0]), h);
        f32x4_t rest[2];
#pragma unroll
        for (int i = 0; i < 8; ++i) rest[i >> 2][i & 3] = t[i >> 2][i & 3] - h[i];
        out[1] = pack(rest);
    }
    static __device__ __forceinline__ f32x4_t mfma(const frag& x, const frag& y, const f32x4_t& c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, x), __builtin_bit_cast(bf16x8_t, y), c, 0, 0, 0);
    }
    // x * w as a sum of SPLIT bf16 values of 8 significant bits each.  Three are the fp32 product to its last bit, so the state and its gradient (results of their
    // own) have fp32's accuracy.  Two (2^-17) serve the other gradients' sums, which only pass into bfloat16 values (10 % of the backward pass).  Neither depends on
    // what else the caller asks for: the forward pass takes three with the new state wanted or not, the state's gradient has a pass of its own.
    template <int SPLIT> static __device__ __forceinline__ void weigh(const frag& x, const float* w, frag* out) {
        float f[8];
        unpack8(__builtin_bit_cast(u32x4_t, x), f);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] *= w[i];
#pragma unroll
        for (int s = 0; s < SPLIT; ++s) {
            const u32x4_t v = pack8(f);
            out[s] = __builtin_bit_cast(frag, v);
            float h[8];
            unpack8(v, h);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] -= h[i];
        }
    }
};
template <int W> struct View<bf16_t, W> {
    typedef __attribute__((address_space(3))) s16x4_t lds_t;
    typedef s16x8_t frag;
    static constexpr int RB = W * 2;                       // bytes of a row
    static constexpr int elems(int rows) { return rows * W; }
    static __device__ __forceinline__ int swz(int row) { return W == 64 ? ((row & 2) << 1) | ((row >> 2) & 3) : ((row & 3) << 2) | ((row >> 2) & 3); }
    static __device__ __forceinline__ int at(int row, int col) { return row * W + ((((col >> 3) ^ swz(row)) << 3) | (col & 7)); }
    int r[4], t[4];                                        // byte offsets of the lane's units 4x + ..: row s, unit g; row 4g + (s >> 2), unit s & 3
    __device__ __forceinline__ explicit View(int lane) {
        const int g = lane >> 4, s = lane & 15, q = 4 * g + (s >> 2);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            r[x] = s * RB + (((4 * x + g) ^ swz(s)) << 4);
            t[x] = q * RB + (((4 * x + (s & 3)) ^ swz(q)) << 4);
        }
    }
    // rows row0 + s, step d of the features
    __device__ __forceinline__ frag rows(const bf16_t* base, int row0, int d) const {
        return *reinterpret_cast<const s16x8_t*>((const char*)base + row0 * RB + (d >> 2) * 256 + r[d & 3]);
    }
    // tile c of the features, tokens row0 .. row0 + 31.  ds_read_b64_tr_b16: lane s of a 16-lane group receives column s of the 4 x 16 block whose row j the
    // lanes 4j .. 4j+3 address
    __device__ __forceinline__ frag cols(const bf16_t* base, int row0, int c) const { return at_column(base, row0, (c >> 3) * 256 + t[(c >> 1) & 3] + (c & 1) * 8); }
    // the same for tile ct of wave w's columns: the byte offset, and the read
    template <int NCT> static __device__ __forceinline__ int column(int lane, int w, int ct) {
        const int s = lane & 15, q = 4 * (lane >> 4) + (s >> 2), col = Ty<bf16_t>::col_of<NCT>(w, ct, 4 * (s & 3));
        return at(q, col) * 2;
    }
    static __device__ __forceinline__ frag at_column(const bf16_t* base, int row0, int off) {
        const char* p = (const char*)base + row0 * RB + off;
        const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)p);
        const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)(p + 16 * RB));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    static __device__ __forceinline__ void put16(bf16_t* base, int row, int col, const u32x4_t& v) { *reinterpret_cast<u32x4_t*>(base + at(row, col)) = v; }
    // where the scores of row `row` with tokens 16 tile + 4g .. lie
    static __device__ __forceinline__ int score(int row, int tile, int g) { return at(row, (tile >> 1) * 32 + g * 8 + (tile & 1) * 4); }
};

template <> struct Ty<float> {
    static constexpr int KS = 16, TPK = 1, C = 32, VE = 4;
    typedef f32x4_t frag;
    static __device__ __forceinline__ int feature(int tile, int g) { return tile * 16 + g * 4; }
    template <int NCT> static __device__ __forceinline__ int col_of(int w, int ct, int i) { return (w * NCT + ct) * 16 + i; }
    static __device__ __forceinline__ float value(float x) { return x; }
    static __device__ __forceinline__ unsigned wild(const frag& x) {
        const u32x4_t v = __builtin_bit_cast(u32x4_t, x), y = (v & 0x7fffffffu) + 0x00800000u;
        return (y.x | y.y | y.z | y.w) & 0x80000000u;
    }
    static __device__ __forceinline__ frag tame(frag x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = x[i] - x[i] == 0.f ? x[i] : 0.f;
        return x;
    }
    static __device__ __forceinline__ void terms(const f32x4_t* t, frag* out) { out[0] = t[0]; }
    static __device__ __forceinline__ f32x4_t mfma(const frag& x, const frag& y, f32x4_t c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], c, 0, 0, 0);
        return c;
    }
    template <int SPLIT> static __device__ __forceinline__ void weigh(const frag& x, const float* w, frag* out) { out[0] = frag{x[0] * w[0], x[1] * w[1], x[2] * w[2], x[3] * w[3]}; }
};
template <int W> struct View<float, W> {
    typedef f32x4_t frag;
    static constexpr int LD = W + 4;
    static constexpr int elems(int rows) { return rows * LD; }
    static __device__ __forceinline__ int at(int row, int col) { return row * LD + col; }
    int r, t;
    __device__ __forceinline__ explicit View(int lane) : r((lane & 15) * LD + (lane >> 4) * 4), t((lane >> 4) * 4 * LD + (lane & 15)) {}
    __device__ __forceinline__ frag rows(const float* base, int row0, int d) const { return *reinterpret_cast<const f32x4_t*>(base + row0 * LD + d * 16 + r); }
    template <int NCT> static __device__ __forceinline__ int column(int lane, int w, int ct) { return (lane >> 4) * 4 * LD + (lane & 15) + (w * NCT + ct) * 16; }
    __device__ __forceinline__ frag cols(const float* base, int row0, int c) const { return at_column(base, row0, t + c * 16); }
    static __device__ __forceinline__ frag at_column(const float* base, int row0, int off) {
        const float* p = base + row0 * LD + off;
        return frag{p[0], p[LD], p[2 * LD], p[3 * LD]};
    }
    static __device__ __forceinline__ void put16(float* base, int row, int col, const u32x4_t& v) { *reinterpret_cast<u32x4_t*>(base + at(row, col)) = v; }
    static __device__ __forceinline__ int score(int row, int tile, int g) { return at(row, tile * 16 + g * 4); }
};

__device__ __forceinline__ void put(bf16_t* p, float v) { *p = f2bf(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put4(bf16_t* p, const f32x4_t& v) { *reinterpret_cast<uint2*>(p) = make_uint2(pack2bf(v[0], v[1]), pack2bf(v[2], v[3])); }
__device__ __forceinline__ void put4(float* p, const f32x4_t& v) { *reinterpret_cast<f32x4_t*>(p) = v; }

// ---- global -> registers -> LDS: C rows x W columns of one operand, zero outside the chunk's tokens and the operand's features.  Row i of the tile is
// token c0 + i, or c0 + mm - 1 - i in reversed time: everything behind the loader sees time running forwards.
// VEC: 16 bytes at a time, by buffer loads whose bound is the chunk's last row: what lies behind it and behind the operand's features comes as zero, with no
// condition (a load under a branch makes the compiler wait for every load in flight where the paths meet, three memory latencies a chunk) and one address
// register.  Otherwise (rows at other borders than 16 bytes, features not in eights) 16 bytes from any address: rows behind the last are the last again, the
// last vector of a row ends with the row, and both are put right on the way into LDS.  Fewer features than a vector: one by one, in `store`.
// 512 x 32, 16 heads of 127 x 127, forward / backward: 95 / 266 us (element by element 333 / 1160); of 128 x 128 through the same code's VEC form 66 / 165.
constexpr unsigned OUTSIDE = 0x80000000u;      // an offset behind every bound: a chunk is at most 2^30 bytes (see operand())
template <class E, int W, bool VEC> struct Tile {
    using V = View<E, W>;
    static constexpr int C = Ty<E>::C, VE = Ty<E>::VE, NV = C * W / VE / 256, ROWS = 256 / (W / VE);
    u32x4_t v[NV];
    // chunk: its first token; step: bytes of a token; col: this thread's columns, in bytes (column())
    static __device__ __forceinline__ unsigned column(int d, int col0, int tid) {
        const int c = col0 + tid % (W / VE) * VE;
        return c < d ? c * (unsigned)sizeof(E) : OUTSIDE;
    }
    __device__ __forceinline__ void load(const char* chunk, unsigned step, unsigned col, int mm, int rev, int tid, const Operand& s, int col0) {
        if constexpr (!VEC) {
            if (s.d < VE) return;
            const int row = tid / (W / VE), at = min(col0 + tid % (W / VE) * VE, s.d - VE);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int r = min(row + i * ROWS, mm - 1);
                __builtin_memcpy(&v[i], reinterpret_cast<const E*>(chunk) + (long long)(rev ? mm - 1 - r : r) * s.st + at, 16);
            }
        } else {
            const int row = tid / (W / VE);
            const auto from = __builtin_amdgcn_make_buffer_rsrc((void*)chunk, 0, mm * step, 0x00027000);
            const unsigned next = rev ? 0u - ROWS * step : ROWS * step;
            unsigned at = (unsigned)(rev ? mm - 1 - row : row) * step + col;      // (rows behind the last, reversed: below zero)
#pragma unroll
            for (int i = 0; i < NV; ++i, at += next) v[i] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(from, at, 0, 0));
        }
    }
    __device__ __forceinline__ void store(E* lds, const Operand& s, const E* base, int c0, int mm, int rev, int col0, int tid) const {
        if constexpr (VEC) {
            const int row = tid / (W / VE), col = (tid % (W / VE)) * VE;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if constexpr (ROWS % 16 == 0) V::put16(lds + i * V::elems(ROWS), row, col, v[i]);      // (the exchange of chunks repeats every 16 rows)
                else V::put16(lds, row + i * ROWS, col, v[i]);
            }
        } else if (s.d >= VE) {
            const int row = tid / (W / VE), col = (tid % (W / VE)) * VE;
            const int behind = (col0 + col - min(col0 + col, s.d - VE)) * (int)sizeof(E) * 8;      // bits of the vector in front of its column
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                V::put16(lds, row + i * ROWS, col, row + i * ROWS < mm ? without_low(v[i], behind) : u32x4_t{0, 0, 0, 0});
            }
        } else {
#pragma unroll 1
            for (int i = tid; i < C * W; i += 256) {
                const int row = i / W, col = i % W;
                lds[V::at(row, col)] = row < mm && col0 + col < s.d ? base[(long long)(c0 + (rev ? mm - 1 - row : row)) * s.st + col0 + col] : E(0);
            }
        }
    }
};

// One workgroup (4 waves) walks one segment of one (sequence, head) in scan order; wave w owns 16 * NCT columns of c, hence of the state (registers,
// fp32) and of the output.  OUT = false: only the segment's own sum  sum_j a^(..) b_j c_j^T  is formed (segments are joined by join_kernel), or, of a sequence in
// one piece, the carry behind it (fin).
// A chunk: the three tiles go to LDS (the next chunk's loads are in flight meanwhile); the lower-triangular 16 x 16 tiles of the scores are dealt to the
// waves and exchanged through LDS; then every wave forms its columns of the output and of the state.
//
// Bound: HBM and the matrix cores, where two workgroups share a CU.  A chunk of bfloat16, 128 features, moves 64 KB: 7400 cycles at the CU's part of 5.3 TB/s; it
// costs 196 matrix instructions (3100 cycles a wave, two waves a matrix core), 800 others and 2700 cycles of LDS, in turn within a wave, under each other between
// the waves.  Measured (16 heads of 128, bfloat16): 512 x 32 forward 67 us = 4.0 TB/s, backward (three roles, each reads three operands) 168; 2048 x 16 (one
// workgroup a CU: the latency of a chunk's steps) 161 and 359.  With the state rounded once these were 61, 153, 147 and 330: the second term is a sixth of the matrix
// instructions.  fp32 (12 x 192, 4 heads of 64, one chunk a workgroup) 8 and 17 us; 1024 x 16 210 and 521: fp32 products at a sixteenth of the rate.
// Four waves of 32 columns: eight of 16 read every tile of a and b twice as often; one chunk of 64 tokens: 32 halve the products between barriers.  The limit
// is the registers: 243 of 256 (the state 64, the loads in flight 48, sums of past tokens 32).  64 features of a and 32 columns a wave would spill at three
// workgroups a CU: 512 x 32, 16 heads of 64 -> 128: 52 us against 47.
//
// The products run over whole tiles, tokens behind the row's own weighted with zero, which a NaN or infinity in c would pass through: it enters them as zero,
// and its column of the output (from its row on) and of the state are made NaN behind them.
template <class E, int DA, int NCT, bool OUT, bool VEC, int SPLIT>
__global__ __launch_bounds__(256, DA > 128 ? 1 : DA > 64 || (sizeof(E) == 2 && OUT && NCT == 2) ? 2 : 3) void scan_kernel(const ScanArgs g) {
    using Y = Ty<E>;
    typedef typename Y::frag frag;
    constexpr int C = Y::C, KS = Y::KS, TPK = Y::TPK, CB = 64 * NCT, ND = DA / KS, NJ = C / KS, NTA = DA / 16, NTI = C / 16;
    using VA = View<E, DA>;
    using VC = View<E, CB>;
    using VP = View<E, C>;
    constexpr int TG = sizeof(E) == 2 ? NTI : 1;            // tiles of 16 tokens whose product with the state is formed at a time
    constexpr int PT = sizeof(E) == 2 ? 2 : 1;              // bf16: scores, and the state that multiplies a, are sums of two terms, as the products that formed them are fp32
    __shared__ __align__(16) E lb[VA::elems(C)], lc[VC::elems(C)], la[OUT ? VA::elems(C) : 1], lp[OUT ? PT * VP::elems(C) : 1];      // lp: scores [term][i][j]
    __shared__ float power[2][2 * C + 4];                    // a^n and scale a^n, n = -C .. C: zero in front of n = 0
    const float *pw = power[0] + C, *spw = power[1] + C;

    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), lg = lane >> 4, ls = lane & 15;
    // what reads the same tokens (roles, column blocks) follows one another on one XCD, whose L2 (or the memory-side cache, for the role that walks the other
    // way) then holds them: workgroups go round the 8 XCDs (backward, 512 x 32 x 16 x 128, an earlier kernel: 179 us; one role behind the other: 184)
    int id = blockIdx.x / 8;
    const int cb = id % g.ncb; id /= g.ncb;
    const int ro = id % g.nroles;
    id = id / g.nroles * 8 + blockIdx.x % 8;
    const int h = id % g.H; id /= g.H;
    const int seg = id % g.nseg, b = id / g.nseg;
    if (b >= g.B) return;
    const Role& r = g.r[ro];
    const long long bh = (long long)b * g.H + h;
    const int da = r.a.d, dc = r.c.d, col0 = cb * CB, rev = r.rev, e = rev ? 0 : 1;
    const float l2 = (float)((double)g.log_decay[h] * 1.4426950408889634);

    int n = g.T;
    if (g.lengths) { const long long x = g.lengths[b]; n = x < 0 ? 0 : x < g.T ? (int)x : g.T; }
    const int t0 = seg * g.seg_len, te = min(t0 + g.seg_len, g.T), t1 = min(te, n);
    const int m = max(0, t1 - t0), nch = (m + C - 1) / C;

    const E* pa = (const E*)r.a.p + b * r.a.sb + h * r.a.sh;
    const E* pb = (const E*)r.b.p + b * r.b.sb + h * r.b.sh;
    const E* pc = (const E*)r.c.p + b * r.c.sb + h * r.c.sh;
    E* po = (E*)r.o + b * r.ob + h * r.oh;

    Tile<E, DA, VEC> ra, rb;
    Tile<E, CB, VEC> rc;
    const unsigned stepa = (unsigned)r.a.st * sizeof(E), stepb = (unsigned)r.b.st * sizeof(E), stepc = (unsigned)r.c.st * sizeof(E);
    const unsigned colb = Tile<E, DA, VEC>::column(da, 0, tid), colc = Tile<E, CB, VEC>::column(dc, col0, tid);
    auto fetch = [&](int cc) {
        const int c0 = t0 + (rev ? nch - 1 - cc : cc) * C, mm = min(C, t1 - c0);
        // (steps in 32 bits are those of the bounded loads)
        const auto from = [&](const E* p, const Operand& s, unsigned step) { return (const char*)p + (VEC ? (long long)c0 * step : (long long)c0 * s.st * (long long)sizeof(E)); };
        if (OUT) ra.load(from(pa, r.a, stepa), stepa, colb, mm, rev, tid, r.a, 0);
        rb.load(from(pb, r.b, stepb), stepb, colb, mm, rev, tid, r.b, 0);
        rc.load(from(pc, r.c, stepc), stepc, colc, mm, rev, tid, r.c, col0);
    };

    if (tid <= 2 * C) {
        power[0][tid] = tid < C ? 0.f : dpow(l2, tid - C);
        power[1][tid] = power[0][tid] * g.scale;
    }
    if (OUT) {
        // rows behind the sequence's last token: zero
        const int cw = min(CB, dc - col0), first = max(t0, n);
        if (VEC) {
            constexpr int PER = CB / 4;                    // (4 elements: what the output's alignment allows)
            for (int i = tid; i < (te - first) * PER; i += 256) {
                const int c = i % PER * 4;
                if (c < cw) put4(po + (long long)(first + i / PER) * r.ot + col0 + c, f32x4_t{0, 0, 0, 0});
            }
        } else {
            for (int t = first; t < te; ++t)
                for (int c = tid; c < cw; c += 256) put(po + t * r.ot + col0 + c, 0.f);
        }
        // scores above the diagonal tiles: zero, once
        for (int i = tid; i < PT * VP::elems(C); i += 256) lp[i] = E(0);
    }

    // state: tile (ta, ct) holds rows feature(ta, lg) + {0..3}, column col_of(w, ct, ls).  Read and written through a bound too, the four rows of a lane together
    // where they are neighbours (with a branch an element: 24 us more for 512 states of 128 x 128 read, 14 written).
    const unsigned state_bytes = (unsigned)(da * dc) * 4u, bya = (unsigned)r.init_a * 4u, byc = (unsigned)r.init_c * 4u;
    auto place = [&](int ta, int ct, int g4, int i) {
        const int a = Y::feature(ta, g4) + i, c = col0 + Y::template col_of<NCT>(w, ct, ls);
        return a < da && c < dc ? (unsigned)a * bya + (unsigned)c * byc : OUTSIDE;
    };
    auto in_fours = [&](const float* p) { return r.init_a == 1 && da % 4 == 0 && (uintptr_t)p % 16 == 0; };
    f32x4_t S[NCT][NTA];
    {
        const float* src = nullptr;
        float mul = 1.f;
        if (OUT || r.fin) {
            if (r.prefix) src = r.prefix + (bh * g.nseg + seg) * (long long)da * dc;
            else if (r.init) { src = r.init + bh * (long long)da * dc; mul = r.init_mul; }
        }
        const auto from = __builtin_amdgcn_make_buffer_rsrc((void*)src, 0, state_bytes, 0x00027000);
        if (!src) {
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
                for (int ta = 0; ta < NTA; ++ta) S[ct][ta] = f32x4_t{0, 0, 0, 0};
        } else if (in_fours(src)) {
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
                for (int ta = 0; ta < NTA; ++ta) S[ct][ta] = __builtin_bit_cast(f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(from, place(ta, ct, lg, 0), 0, 0)) * mul;
        } else {
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
                for (int ta = 0; ta < NTA; ++ta)
#pragma unroll
                    for (int i = 0; i < 4; ++i) S[ct][ta][i] = mul * __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(from, place(ta, ct, lg, i), 0, 0));
        }
    }
    if (nch > 0) fetch(0);
    const VA va(lane);
    int vcol[NCT];
#pragma unroll
    for (int ct = 0; ct < NCT; ++ct) vcol[ct] = VC::template column<NCT>(lane, w, ct);
    const VP vp(lane);

    auto chunk = [&](int c0, int mm) {
        if (OUT) {
            // Tiles (ti, tj <= ti).  bf16: wave w has (w, w) and one more, waves 0 and 1 a third: (2, 0), (3, 0); (2, 1), (3, 1); (3, 2); (1, 0).
            // fp32: (0, 0), (1, 1), (1, 0).  Those on the diagonal come first: they alone have scores to be left out.
            auto score = [&](int ti, int tj, bool diagonal) {
                f32x4_t P = {0, 0, 0, 0};
#pragma unroll
                for (int d = 0; d < ND; ++d) P = Y::mfma(va.rows(lb, tj * 16, d), va.rows(la, ti * 16, d), P);
                const float* f = spw + (ti - tj) * 16 + ls - lg * 4;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    P[x] *= f[-x];
                    if (diagonal) P[x] = ls < lg * 4 + x ? 0.f : P[x];
                }
                E* at = lp + VP::score(ti * 16 + ls, tj, lg);
                put4(at, P);
                if constexpr (PT == 2) {
                    // (one term alone: a short sequence's few scores carry their rounding into whole rows of the output, 1.7 times its own rounding)
#pragma unroll
                    for (int x = 0; x < 4; ++x) P[x] -= Y::value(f2bf(P[x]));
                    put4(at + VP::elems(C), P);
                }
            };
            if constexpr (NTI == 4) {
                score(w, w, true);
                score(w < 2 ? 2 : w == 2 ? 3 : 1, w < 3 ? w : 0, false);
                if (w < 2) score(3, w, false);
            } else {
                if (w < 2) score(w, w, true);
                else if (w == 2) score(1, 0, false);
            }
        }
        bool spoilt = false;
        frag vf[NJ][NCT];
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct) vf[j][ct] = VC::at_column(lc, j * KS, vcol[ct]);

        if (OUT) {
            // a S, for TG tiles of 16 tokens at a time, a step of the features after the other.  bf16: the state as two terms, as the scores (rounded once it
            // alone would add two thirds of the output's own rounding, 0.0022 of the output against 0.0017, and be the larger part of short sums that cancel).
            f32x4_t old[TG][NCT];
            auto past_products = [&](int t0) {
#pragma unroll
                for (int t = 0; t < TG; ++t)
#pragma unroll
                    for (int ct = 0; ct < NCT; ++ct) old[t][ct] = f32x4_t{0, 0, 0, 0};
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    frag sf[NCT][PT];
#pragma unroll
                    for (int ct = 0; ct < NCT; ++ct) Y::terms(S[ct] + d * TPK, sf[ct]);
#pragma unroll
                    for (int t = 0; t < TG; ++t) {
                        const frag af = va.rows(la, (t0 + t) * 16, d);
#pragma unroll
                        for (int x = 0; x < PT; ++x)
#pragma unroll
                            for (int ct = 0; ct < NCT; ++ct) old[t][ct] = Y::mfma(sf[ct][x], af, old[t][ct]);
                    }
                }
            };
            past_products(0);
            __syncthreads();                              // the scores are complete
            unsigned x = 0;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int ct = 0; ct < NCT; ++ct) x |= Y::wild(vf[j][ct]);
            spoilt = __any(x != 0);
            if (spoilt) {
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int ct = 0; ct < NCT; ++ct) vf[j][ct] = Y::tame(vf[j][ct]);
            }
            // output^T tiles: rows = columns of c (4 lg + ..), column = token ti * 16 + ls
            frag pf[PT][NJ];
            // stores by offsets whose bound is the chunk's last row, as the loads
            const unsigned step = (unsigned)r.ot * sizeof(E), next = rev ? 0u - 16 * step : 16 * step;
            const auto out = __builtin_amdgcn_make_buffer_rsrc(po + (long long)c0 * r.ot, 0, mm * step, 0x00027000);
            unsigned at[NCT];
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct) {
                const int c = col0 + Y::template col_of<NCT>(w, ct, lg * 4);
                at[ct] = c < dc ? (unsigned)(rev ? mm - 1 - ls : ls) * step + c * (unsigned)sizeof(E) : OUTSIDE;
            }
#pragma unroll
            for (int ti = 0; ti < NTI; ++ti) {
                // bf16: all four tiles of 16 tokens in one run of code (with a branch a tile the waits of one tile do not overlap the next's products)
                if (VEC && sizeof(E) == 2 || ti * 16 < mm) {
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
                        if (j * KS <= ti * 16 + 15)
#pragma unroll
                            for (int x = 0; x < PT; ++x) pf[x][j] = vp.rows(lp + x * VP::elems(C), ti * 16, j);
                    if (ti > 0 && ti % TG == 0) past_products(ti);
                    f32x4_t* acc = old[ti % TG];
                    const float past = spw[ti * 16 + ls + e];
#pragma unroll
                    for (int ct = 0; ct < NCT; ++ct) acc[ct] *= past;
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
                        if (j * KS <= ti * 16 + 15)
#pragma unroll
                            for (int x = 0; x < PT; ++x)
#pragma unroll
                                for (int ct = 0; ct < NCT; ++ct) acc[ct] = Y::mfma(vf[j][ct], pf[x][j], acc[ct]);
                    if constexpr (VEC && sizeof(E) == 2 && NCT == 2) {
                        const u32x4_t v = {pack2bf(acc[0][0], acc[0][1]), pack2bf(acc[0][2], acc[0][3]), pack2bf(acc[1][0], acc[1][1]), pack2bf(acc[1][2], acc[1][3])};
                        __builtin_amdgcn_raw_buffer_store_b128(v, out, at[0], 0, 0);
                        at[0] += next;
                    } else if constexpr (VEC) {
#pragma unroll
                        for (int ct = 0; ct < NCT; ++ct) {
                            if constexpr (sizeof(E) == 2) __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{pack2bf(acc[ct][0], acc[ct][1]), pack2bf(acc[ct][2], acc[ct][3])}, out, at[ct], 0, 0);
                            else __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, acc[ct]), out, at[ct], 0, 0);
                            at[ct] += next;
                        }
                    } else {
                        // (a lane's columns are neighbours over all its tiles for bfloat16)
                        constexpr int RUN = sizeof(E) == 2 ? NCT * 4 : 4;
                        const int i = ti * 16 + ls;
                        unsigned e[NCT * sizeof(E)];      // (the lane's columns as they lie in memory)
#pragma unroll
                        for (int x = 0; x < NCT; ++x) {
                            if constexpr (sizeof(E) == 2) { e[2 * x] = pack2bf(acc[x][0], acc[x][1]); e[2 * x + 1] = pack2bf(acc[x][2], acc[x][3]); }
                            else __builtin_memcpy(e + 4 * x, &acc[x], 16);
                        }
#pragma unroll
                        for (int x = 0; x < NCT * 4; x += RUN) {
                            const int c = col0 + Y::template col_of<NCT>(w, x / 4, lg * 4);
                            E* q = po + (long long)(c0 + (rev ? mm - 1 - i : i)) * r.ot + c;
                            if (i < mm && c + RUN <= dc) {
                                __builtin_memcpy(q, (const char*)e + x * sizeof(E), RUN * sizeof(E));
                            } else if (i < mm) {
#pragma unroll
                                for (int y = 0; y < RUN; ++y)
                                    if (c + y < dc) put(q + y, acc[(x + y) / 4][(x + y) % 4]);
                            }
                        }
                    }
                }
            }
        }
        // state update
        const float all = pw[mm];
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
            for (int ta = 0; ta < NTA; ++ta) S[ct][ta] *= all;
        constexpr int AHEAD = 2;                          // tiles of b in flight under the products
        frag kf[AHEAD + 1];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            if (sizeof(E) == 2 || j * KS < mm) {
#pragma unroll
                for (int n = 0; n < AHEAD; ++n) kf[n] = va.cols(lb, j * KS, n);
                const float* f = pw + mm - e - j * KS - lg * 4;      // (rows behind mm: zero by zero)
                float wt[KS / 4];
#pragma unroll
                for (int x = 0; x < KS / 4; ++x) wt[x] = f[-((x >> 2) * 16 + (x & 3))];
                frag wv[NCT][SPLIT];
#pragma unroll
                for (int ct = 0; ct < NCT; ++ct) Y::template weigh<SPLIT>(vf[j][ct], wt, wv[ct]);
#pragma unroll
                for (int ta = 0; ta < NTA; ++ta) {
                    if (ta + AHEAD < NTA) { kf[(ta + AHEAD) % (AHEAD + 1)] = va.cols(lb, j * KS, ta + AHEAD); PIN; }
#pragma unroll
                    for (int x = 0; x < SPLIT; ++x)
#pragma unroll
                        for (int ct = 0; ct < NCT; ++ct) S[ct][ta] = Y::mfma(kf[ta % (AHEAD + 1)], wv[ct][x], S[ct][ta]);
                }
            }
        }
        if (spoilt) {
            auto first = [&](int c) {                     // the first row whose value of column c is not finite
                int j = 0;
                while (j < mm && Y::value(lc[VC::at(j, c)]) - Y::value(lc[VC::at(j, c)]) == 0.f) ++j;
                return j;
            };
#pragma unroll 1
            for (int x = 0; x < NCT * 4; ++x) {           // (this lane's own outputs, overwritten)
                const int c = Y::template col_of<NCT>(w, x / 4, lg * 4 + x % 4), from = first(c);
#pragma unroll 1
                for (int i = ls; i < mm; i += 16)
                    if (i >= from && col0 + c < dc) put(po + (long long)(c0 + (rev ? mm - 1 - i : i)) * r.ot + col0 + c, NAN);
            }
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct) {
                const float add = first(Y::template col_of<NCT>(w, ct, ls)) < mm ? NAN : 0.f;
#pragma unroll
                for (int ta = 0; ta < NTA; ++ta) S[ct][ta] += add;
            }
        }
    };

    for (int cc = 0; cc < nch; ++cc) {
        const int c0 = t0 + (rev ? nch - 1 - cc : cc) * C, mm = min(C, t1 - c0);
        __syncthreads();                                  // (the previous chunk's tiles have been read)
        if (OUT) ra.store(la, r.a, pa, c0, mm, rev, 0, tid);
        rb.store(lb, r.b, pb, c0, mm, rev, 0, tid);
        rc.store(lc, r.c, pc, c0, mm, rev, col0, tid);
        __syncthreads();
        if (cc + 1 < nch) fetch(cc + 1);                  // in flight under this chunk's products
        chunk(c0, mm);
    }

    float* dst = nullptr;
    float mul = 1.f;
    if (!OUT && !r.fin) {
        dst = g.part + (((long long)ro * g.B * g.H + bh) * g.nseg + seg) * (long long)da * dc;
    } else if (r.fin) {
        const int last = rev ? 0 : n > 0 ? (n - 1) / g.seg_len : 0;
        if (seg == last) { dst = r.fin + bh * (long long)da * dc; mul = r.fin_mul; }
    }
    if (dst) {
        const auto to = __builtin_amdgcn_make_buffer_rsrc(dst, 0, state_bytes, 0x00027000);
        int g4 = lg;
        asm volatile("" : "+v"(g4));                      // (or the offsets of the state's read would be kept, in memory, for its write)
        if (in_fours(dst)) {
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
                for (int ta = 0; ta < NTA; ++ta) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, S[ct][ta] * mul), to, place(ta, ct, g4, 0), 0, 0);
        } else {
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
                for (int ta = 0; ta < NTA; ++ta)
#pragma unroll
                    for (int i = 0; i < 4; ++i) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, mul * S[ct][ta][i]), to, place(ta, ct, g4, i), 0, 0);
        }
    }
}

// Segment sums -> the carry in front of every segment, in place, and (fin) behind the last.  One thread owns one element
// of the state and walks the segments in scan order.  512 states of 128 x 128 (67 MB in and out): 12.5 us = 5.4 TB/s.
struct JoinArgs {
    float *part, *fin;
    const float* init[2];
    float init_mul[2], fin_mul;
    int rev[2];
    const float* log_decay;
    const long long* lengths;
    int T, B, H, nseg, seg_len, n;      // n = elements of a state
};
__global__ __launch_bounds__(256) void join_kernel(const JoinArgs g) {
    const int el = blockIdx.x * 256 + threadIdx.x, bh = blockIdx.y, set = blockIdx.z;
    if (el >= g.n) return;
    const int b = bh / g.H;
    const float l2 = (float)((double)g.log_decay[bh % g.H] * 1.4426950408889634);
    int n = g.T;
    if (g.lengths) { const long long x = g.lengths[b]; n = x < 0 ? 0 : x < g.T ? (int)x : g.T; }
    float* p = g.part + ((long long)set * g.B * g.H + bh) * g.nseg * (long long)g.n + el;
    float carry = g.init[set] ? g.init_mul[set] * g.init[set][(long long)bh * g.n + el] : 0.f;
    for (int i0 = 0; i0 < g.nseg; i0 += 8) {
        float x[8];                                       // (eight loads in flight; the stores go to the same places)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int i = min(i0 + k, g.nseg - 1);
            x[k] = p[(long long)(g.rev[set] ? g.nseg - 1 - i : i) * g.n];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int i = i0 + k, s = g.rev[set] ? g.nseg - 1 - i : i;
            if (i < g.nseg) {
                const int m = min(max(n - s * g.seg_len, 0), g.seg_len);
                p[(long long)s * g.n] = carry;
                carry = m > 0 ? dpow(l2, m) * carry + x[k] : carry;
            }
        }
    }
    if (g.fin) g.fin[(long long)bh * g.n + el] = g.fin_mul * carry;
}

// ---- recurrent form: one token a row, states updated in place.  A workgroup owns BLOCK columns of one (row, head): the state passes through the registers
// once (read + written: 8 Dk Dv bytes are the whole cost), columns across the lanes, rows of the state across the rest of the workgroup, eight in flight.
// Rows that name the same slot are successive tokens of that sequence, in row order: the first of them does the others' work as well.
// 128 columns (us; 64, 256 columns): 512 rows x 16 heads of 128 x 128 209 = 5.1 TB/s (220, 208); 64 x 8 of 256 x 255 52 (59, 49); 1 x 2 of 256 x 256 8.0 (5.4, 12.7);
// 2 x 3 of 202 x 122 11 (10, 11); 1 x 4 of 64 x 64 4, the launch's.  One width for all, so that a row's result does not depend on how many there are.
constexpr int BLOCK = 128;                                 // columns of a workgroup
struct StepArgs {
    const void *q, *k, *v;
    void* o;
    long long qs[2], ks[2], vs[2], os[2];
    const float* log_decay;
    float* state;
    const long long* slots;
    int B, H, Dk, Dv, nslots;
    float scale;
};
template <class E> __device__ __forceinline__ float get(const E* p);
template <> __device__ __forceinline__ float get<bf16_t>(const bf16_t* p) { return bf2f(*p); }
template <> __device__ __forceinline__ float get<float>(const float* p) { return *p; }

template <class E>
__global__ __launch_bounds__(256) void step_kernel(const StepArgs g) {
    __shared__ float sq[256], sk[256], red[4][BLOCK / 4][4];
    __shared__ int first, next;
    const int tid = threadIdx.x, h = blockIdx.x % g.H;
    int b = blockIdx.x / g.H;
    long long slot = b;
    if (g.slots) {
        slot = g.slots[b];
        if (slot < 0 || slot >= g.nslots) {               // a padded row: no state, output zero
            E* o = (E*)g.o + b * g.os[0] + h * g.os[1];
            for (int c = blockIdx.y * BLOCK + tid; c < min(g.Dv, (int)(blockIdx.y + 1) * BLOCK); c += 256) put(o + c, 0.f);
            return;
        }
        if (tid == 0) { first = 1; next = g.B; }
        __syncthreads();
        int mine = g.B;
        for (int x = tid; x < g.B; x += 256)
            if (x != b && g.slots[x] == slot) {
                if (x < b) first = 0;
                else mine = min(mine, x);
            }
        if (mine < g.B) atomicMin(&next, mine);
        __syncthreads();
        if (!first) return;
    }
    const float a = expf(g.log_decay[h]);
    float* st = g.state + (slot * g.H + h) * (long long)g.Dk * g.Dv;
    const int nc = min((g.Dv + 3) / 4, BLOCK / 4);        // columns in fours; 256 / nct rows of the state at a time
    int nct = 1;
    while (nct < nc) nct <<= 1;
    const int rows = 256 / nct, c4 = tid % nct, r0 = tid / nct, col0 = blockIdx.y * BLOCK;
    while (true) {
        const E* q = (const E*)g.q + b * g.qs[0] + h * g.qs[1];
        const E* k = (const E*)g.k + b * g.ks[0] + h * g.ks[1];
        const E* v = (const E*)g.v + b * g.vs[0] + h * g.vs[1];
        E* o = (E*)g.o + b * g.os[0] + h * g.os[1];
        for (int i = tid; i < g.Dk; i += 256) { sq[i] = g.scale * get(q + i); sk[i] = get(k + i); }
        __syncthreads();
        const int c = col0 + c4 * 4;
        float vv[4], acc[4] = {0, 0, 0, 0};
#pragma unroll
        for (int x = 0; x < 4; ++x) vv[x] = c + x < g.Dv ? get(v + c + x) : 0.f;
        // U rows in flight (the compiler does not move a load in front of a store that it cannot tell apart)
        constexpr int U = 8;
        const bool four = c + 4 <= g.Dv;                  // (rows of a state need not start at 16-byte borders; the last columns may be fewer than four)
        for (int i0 = r0; i0 < g.Dk; i0 += rows * U) {
            f32x4_t s[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float* p = st + (long long)min(i0 + u * rows, g.Dk - 1) * g.Dv;
                if (four) __builtin_memcpy(&s[u], p + c, 16);
                else s[u] = f32x4_t{p[min(c, g.Dv - 1)], p[min(c + 1, g.Dv - 1)], p[min(c + 2, g.Dv - 1)], 0.f};
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u * rows;
                if (i < g.Dk) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) { s[u][x] = a * s[u][x] + sk[i] * vv[x]; acc[x] += sq[i] * s[u][x]; }
                    float* p = st + (long long)i * g.Dv + c;
                    if (four) __builtin_memcpy(p, &s[u], 16);
                    else {
#pragma unroll
                        for (int x = 0; x < 3; ++x)
                            if (c + x < g.Dv) p[x] = s[u][x];
                    }
                }
            }
        }
        // sum over the row groups, in a fixed order: within the wave, then the four waves
        for (int o = nct; o < 64; o <<= 1)
#pragma unroll
            for (int x = 0; x < 4; ++x) acc[x] += __shfl_xor(acc[x], o);
        if ((tid & 63) < nct)
#pragma unroll
            for (int x = 0; x < 4; ++x) red[tid >> 6][c4][x] = acc[x];
        __syncthreads();
        if (tid < nct)
#pragma unroll
            for (int x = 0; x < 4; ++x)
                if (c + x < g.Dv) put(o + c + x, (red[0][c4][x] + red[1][c4][x]) + (red[2][c4][x] + red[3][c4][x]));
        __syncthreads();
        if (!g.slots) return;
        b = next;
        if (b >= g.B) return;
        __syncthreads();
        if (tid == 0) next = g.B;
        __syncthreads();
        int mine = g.B;
        for (int x = b + 1 + tid; x < g.B; x += 256)
            if (g.slots[x] == slot) mine = min(mine, x);
        if (mine < g.B) atomicMin(&next, mine);
        __syncthreads();
    }
}

bool aligned(const void* p, long long s0, long long s1, long long s2, int d, int e, int bytes) {
    const int n = bytes / e;
    return ((uintptr_t)p % bytes) == 0 && s0 % n == 0 && s1 % n == 0 && s2 % n == 0 && d % n == 0;
}
Operand operand(const void* p, const int64_t* s, int d, int f32) {
    return Operand{p, s[0], s[1], s[2], d, aligned(p, s[0], s[1], s[2], d, f32 ? 4 : 2, 16) && s[0] >= d && s[0] < (1 << 22) ? 1 : 0};      // (rows apart; 64 of them under 2^30 bytes)
}
void output(Role& r, void* p, const int64_t* s, int d, int f32) {
    r.o = p; r.ot = s[0]; r.ob = s[1]; r.oh = s[2];
    r.ovec = aligned(p, s[0], s[1], s[2], d, f32 ? 4 : 2, 16) && s[0] >= d && s[0] < (1 << 22);
}

template <class E, int DA, int NCT, int SPLIT>
void launch_split(const ScanArgs& g, bool out, bool vec, hipStream_t st) {
    const dim3 grid((unsigned)g.nroles * g.ncb * ((g.B * g.nseg * g.H + 7) / 8) * 8), wg(256);
    if (out) {
        if (vec) hipLaunchKernelGGL((scan_kernel<E, DA, NCT, true, true, SPLIT>), grid, wg, 0, st, g);
        else hipLaunchKernelGGL((scan_kernel<E, DA, NCT, true, false, SPLIT>), grid, wg, 0, st, g);
    } else {
        if (vec) hipLaunchKernelGGL((scan_kernel<E, DA, NCT, false, true, SPLIT>), grid, wg, 0, st, g);
        else hipLaunchKernelGGL((scan_kernel<E, DA, NCT, false, false, SPLIT>), grid, wg, 0, st, g);
    }
}
template <class E, int DA, int NCT>
void launch_one(const ScanArgs& g, bool out, bool vec, bool exact, hipStream_t st) {
    if constexpr (sizeof(E) == 4) launch_split<E, DA, NCT, 1>(g, out, vec, st);
    else if (exact) launch_split<E, DA, NCT, 3>(g, out, vec, st);
    else launch_split<E, DA, NCT, 2>(g, out, vec, st);
}
int da_class(int da) { return da <= 64 ? 64 : da <= 128 ? 128 : 256; }
int nct_of(int da, int dc) { return da <= 128 && dc > 64 ? 2 : 1; }       // (256 features of a: 64 columns a workgroup, or the state would not fit its registers)

// Launches `n` roles; those that take the same kernel share a launch.
template <class E>
void launch(const ScanArgs& base, const Role* roles, int n, bool out, bool exact, float* part, hipStream_t st) {
    bool done[3] = {false, false, false};
    for (int i = 0; i < n; ++i) {
        if (done[i]) continue;
        ScanArgs g = base;
        g.nroles = 0;
        const int da = da_class(roles[i].a.d), nct = nct_of(roles[i].a.d, roles[i].c.d), ncb = (roles[i].c.d + 64 * nct - 1) / (64 * nct);
        for (int j = i; j < n; ++j)
            if (!done[j] && da_class(roles[j].a.d) == da && nct_of(roles[j].a.d, roles[j].c.d) == nct && (roles[j].c.d + 64 * nct - 1) / (64 * nct) == ncb
                && (out || roles[j].a.d == roles[i].a.d)) {
                g.r[g.nroles++] = roles[j];
                done[j] = true;
            }
        g.ncb = ncb;
        bool vec = true;                                  // 16-byte rows in and out
        for (int j = 0; j < g.nroles; ++j) vec = vec && g.r[j].b.vec && g.r[j].c.vec && (!out || (g.r[j].a.vec && g.r[j].ovec));
        g.part = part + (out ? 0 : (long long)i * g.B * g.H * g.nseg * roles[i].a.d * roles[i].c.d);
        if (da == 64) { if (nct == 2) launch_one<E, 64, 2>(g, out, vec, exact, st); else launch_one<E, 64, 1>(g, out, vec, exact, st); }
        else if (da == 128) { if (nct == 2) launch_one<E, 128, 2>(g, out, vec, exact, st); else launch_one<E, 128, 1>(g, out, vec, exact, st); }
        else launch_one<E, 256, 1>(g, out, vec, exact, st);
    }
}

// Segments: with fewer (sequence, head) pairs than the chip has room for (two workgroups on each of 256 CUs), a sequence is cut into as many segments as fill
// it, of four chunks or more, walked side by side.  That costs the segments' own sums first and a pass over them, so three segments are the least.  bfloat16, us,
// whole and cut (pairs x roles; forward unless said; both sides of an earlier kernel, now 5 to 10 % longer):
//   192, 1024 tokens: 65 and 110 (2 segments)      210, 4096 tokens, backward: 224 and 283 (2)      256, 2048 tokens: 160 and 271 (2)
//   128, 2048 tokens: 122 and 129 (4); 8192 tokens: 481 and 416; float32, 64 features: 145 and 96      144, 4096 tokens, backward: 220 and 202 (3)
// Twice as many segments: 8192 x 2 x 16 x 128 115 -> 144, 4096 x 3 x 12 x 128 77 -> 94; half as many: 141 -> 147 (an earlier kernel).
void segments(const srvp_linear_attention_desc* d, int roles, int* nseg, int* seg_len) {
    const int C = d->elem_f32 ? 32 : 64;
    const long long ncb = (d->Dv + 127) / 128, base = (long long)d->B * d->H * ncb * roles;
    const long long chunks = (d->T + C - 1) / C;
    long long n = base == 0 ? 1 : 512 / base;
    if (n > (chunks + 3) / 4) n = (chunks + 3) / 4;
    if (n < 3) n = 1;
    const long long per = chunks > n ? (chunks + n - 1) / n : 1;
    *seg_len = (int)(per * C);
    *nseg = (int)((chunks + per - 1) / per);
    if (*nseg < 1) *nseg = 1;
}

int check(const srvp_linear_attention_desc* d, const char* who) {
    SRVP_REQUIRE(d, "%s: null descriptor", who);
    SRVP_REQUIRE(d->T >= 0 && d->B >= 0 && d->H >= 0, "%s: negative size", who);
    SRVP_REQUIRE(d->Dk >= 1 && d->Dk <= 256 && d->Dv >= 1 && d->Dv <= 256, "%s: heads of 1 to 256 features (got %d, %d)", who, d->Dk, d->Dv);
    SRVP_REQUIRE(d->T < (1 << 30) && (long long)d->B * d->H < (1 << 20), "%s: more than 2^30 tokens or 2^20 (sequence, head) pairs", who);
    const float size = fabsf(d->scale);                     // (the gradients of the state pass through 1 / scale)
    SRVP_REQUIRE(size >= 1e-30f && size <= 1e30f, "%s: scale of 1e-30 to 1e30", who);
    return SRVP_OK;
}

}  // namespace

extern "C" int64_t srvp_linear_attention_ws_bytes(const srvp_linear_attention_desc* d, int32_t backward) {
    if (check(d, "srvp_linear_attention_ws_bytes")) return -1;
    int nseg, len;
    segments(d, backward ? 3 : 1, &nseg, &len);
    return nseg <= 1 ? 0 : (int64_t)(backward ? 2 : 1) * d->B * d->H * nseg * d->Dk * d->Dv * 4;
}

static int run_join(const ScanArgs& base, const srvp_linear_attention_desc* d, int sets, const float* const* init, const float* mul, const int* rev, float* part, float* fin, float fin_mul, hipStream_t st) {
    JoinArgs j;
    memset(&j, 0, sizeof(j));
    j.part = part; j.fin = fin; j.fin_mul = fin_mul; j.log_decay = d->log_decay; j.lengths = base.lengths;
    for (int i = 0; i < sets; ++i) { j.init[i] = init[i]; j.init_mul[i] = mul[i]; j.rev[i] = rev[i]; }
    j.T = d->T; j.B = d->B; j.H = d->H; j.nseg = base.nseg; j.seg_len = base.seg_len; j.n = d->Dk * d->Dv;
    // (grid.y: a sequence is cut where there are fewer than 256 pairs)
    hipLaunchKernelGGL(join_kernel, dim3((j.n + 255) / 256, d->B * d->H, sets), dim3(256), 0, st, j);
    SRVP_CHECK_LAUNCH("srvp_linear_attention(join)");
    return SRVP_OK;
}

static void base_args(ScanArgs& g, const srvp_linear_attention_desc* d, int roles) {
    memset(&g, 0, sizeof(g));
    g.log_decay = d->log_decay; g.lengths = (const long long*)d->lengths;
    g.T = d->T; g.B = d->B; g.H = d->H; g.scale = d->scale;
    segments(d, roles, &g.nseg, &g.seg_len);
}

extern "C" int srvp_linear_attention_fwd(const srvp_linear_attention_desc* d, void* stream) {
    if (int rc = check(d, "srvp_linear_attention_fwd")) return rc;
    if (d->B == 0 || d->H == 0) return SRVP_OK;
    SRVP_REQUIRE(d->log_decay && (d->T == 0 || (d->q && d->k && d->v && d->o)), "srvp_linear_attention_fwd: null pointer");
    hipStream_t st = (hipStream_t)stream;
    ScanArgs g;
    base_args(g, d, 1);
    const int64_t need = srvp_linear_attention_ws_bytes(d, 0);
    SRVP_REQUIRE(need == 0 || (d->ws && d->ws_bytes >= need), "srvp_linear_attention_fwd: workspace of %lld bytes needed", (long long)need);
    Role r;
    memset(&r, 0, sizeof(r));
    r.a = operand(d->q, d->qs, d->Dk, d->elem_f32);
    r.b = operand(d->k, d->ks, d->Dk, d->elem_f32);
    r.c = operand(d->v, d->vs, d->Dv, d->elem_f32);
    output(r, d->o, d->os, d->Dv, d->elem_f32);
    r.init = d->state_in; r.init_mul = 1.f; r.fin = d->state_out; r.fin_mul = 1.f;
    r.init_a = d->Dv; r.init_c = 1;
    if (g.nseg > 1) {
        float* part = (float*)d->ws;
        Role sums = r;
        sums.fin = nullptr;
        if (d->elem_f32) launch<float>(g, &sums, 1, false, true, part, st); else launch<bf16_t>(g, &sums, 1, false, true, part, st);
        SRVP_CHECK_LAUNCH("srvp_linear_attention_fwd(segments)");
        const float* init[1] = {d->state_in};
        const float mul[1] = {1.f};
        const int rev[1] = {0};
        if (int rc = run_join(g, d, 1, init, mul, rev, part, nullptr, 0.f, st)) return rc;
        r.prefix = part;
    }
    if (d->elem_f32) launch<float>(g, &r, 1, true, true, nullptr, st); else launch<bf16_t>(g, &r, 1, true, true, nullptr, st);
    SRVP_CHECK_LAUNCH("srvp_linear_attention_fwd");
    return SRVP_OK;
}

extern "C" int srvp_linear_attention_bwd(const srvp_linear_attention_bwd_desc* bd, void* stream) {
    SRVP_REQUIRE(bd, "srvp_linear_attention_bwd: null descriptor");
    const srvp_linear_attention_desc* d = &bd->f;
    if (int rc = check(d, "srvp_linear_attention_bwd")) return rc;
    if (d->B == 0 || d->H == 0) return SRVP_OK;
    SRVP_REQUIRE(d->log_decay && (d->T == 0 || (d->q && d->k && d->v && bd->d_o && bd->dq && bd->dk && bd->dv)), "srvp_linear_attention_bwd: null pointer");
    hipStream_t st = (hipStream_t)stream;
    ScanArgs g;
    base_args(g, d, 3);
    const int64_t need = srvp_linear_attention_ws_bytes(d, 1);
    SRVP_REQUIRE(need == 0 || (d->ws && d->ws_bytes >= need), "srvp_linear_attention_bwd: workspace of %lld bytes needed", (long long)need);
    const int f32 = d->elem_f32, Dk = d->Dk, Dv = d->Dv;
    const Operand q = operand(d->q, d->qs, Dk, f32), k = operand(d->k, d->ks, Dk, f32), v = operand(d->v, d->vs, Dv, f32), go = operand(bd->d_o, bd->d_os, Dv, f32);
    Role r[3];
    memset(r, 0, sizeof(r));
    // dv: (k, q, do), reversed, carry X (Dk x Dv)
    r[0].a = k; r[0].b = q; r[0].c = go; output(r[0], bd->dv, bd->dvs, Dv, f32);
    r[0].rev = 1; r[0].init = bd->d_state_out; r[0].init_mul = 1.f / d->scale;
    if (f32) { r[0].fin = bd->d_state_in; r[0].fin_mul = d->scale; }
    r[0].init_a = Dv; r[0].init_c = 1;
    // dk: (v, do, q), reversed, carry X^T
    r[1].a = v; r[1].b = go; r[1].c = q; output(r[1], bd->dk, bd->dks, Dk, f32);
    r[1].rev = 1; r[1].init = bd->d_state_out; r[1].init_mul = 1.f / d->scale; r[1].init_a = 1; r[1].init_c = Dv;
    // dq: (do, v, k), forwards, carry S^T
    r[2].a = go; r[2].b = v; r[2].c = k; output(r[2], bd->dq, bd->dqs, Dk, f32);
    r[2].init = d->state_in; r[2].init_mul = 1.f; r[2].init_a = 1; r[2].init_c = Dv;
    Role p[2];                                            // segment sums of S (k, v) and of X (q, do)
    memset(p, 0, sizeof(p));
    p[0].a = k; p[0].b = k; p[0].c = v; p[0].init_a = Dv; p[0].init_c = 1;
    p[1].a = q; p[1].b = q; p[1].c = go; p[1].init_a = Dv; p[1].init_c = 1; p[1].rev = 1;
    const float* init[2] = {d->state_in, bd->d_state_out};
    const float mul[2] = {1.f, 1.f / d->scale};
    const int rev[2] = {0, 1};
    if (bd->d_state_in && !f32) {
        // dS_0 of bfloat16 tensors: X once more, in fp32's accuracy.  (One of the roles with three terms instead of two takes the others' time too where all are in
        // flight at once, also for callers without a state: 8192 x 2, 16 heads of 128: 288 -> 322 us.  With this pass only those with one pay: 512 x 32, 16 heads of
        // 128 -> 64: 138, with a state 167; three terms for all roles 156.)
        Role x = p[1];
        if (g.nseg == 1) { x.init = init[1]; x.init_mul = mul[1]; x.fin = bd->d_state_in; x.fin_mul = d->scale; }
        launch<bf16_t>(g, &x, 1, false, true, (float*)d->ws, st);
        SRVP_CHECK_LAUNCH("srvp_linear_attention_bwd(state)");
        if (g.nseg > 1)
            if (int rc = run_join(g, d, 1, init + 1, mul + 1, rev + 1, (float*)d->ws, bd->d_state_in, d->scale, st)) return rc;
    }
    if (g.nseg > 1) {
        float* part = (float*)d->ws;
        const long long set = (long long)d->B * d->H * g.nseg * Dk * Dv;
        if (f32) launch<float>(g, p, 2, false, false, part, st); else launch<bf16_t>(g, p, 2, false, false, part, st);
        SRVP_CHECK_LAUNCH("srvp_linear_attention_bwd(segments)");
        if (int rc = run_join(g, d, 2, init, mul, rev, part, nullptr, 0.f, st)) return rc;
        r[0].prefix = r[1].prefix = part + set;
        r[2].prefix = part;
    }
    if (f32) launch<float>(g, r, 3, true, false, nullptr, st); else launch<bf16_t>(g, r, 3, true, false, nullptr, st);
    SRVP_CHECK_LAUNCH("srvp_linear_attention_bwd");
    return SRVP_OK;
}

extern "C" int srvp_linear_attention_step(const srvp_linear_attention_step_desc* d, void* stream) {
    SRVP_REQUIRE(d, "srvp_linear_attention_step: null descriptor");
    SRVP_REQUIRE(d->B >= 0 && d->H >= 0 && d->nslots >= 0 && (long long)d->B * d->H < (1 << 24), "srvp_linear_attention_step: fewer than 2^24 (row, head) pairs");
    SRVP_REQUIRE(d->Dk >= 1 && d->Dk <= 256 && d->Dv >= 1 && d->Dv <= 256, "srvp_linear_attention_step: heads of 1 to 256 features (got %d, %d)", d->Dk, d->Dv);
    if (d->B == 0 || d->H == 0) return SRVP_OK;
    SRVP_REQUIRE(d->q && d->k && d->v && d->o && d->log_decay && (d->state || d->nslots == 0), "srvp_linear_attention_step: null pointer");
    // (every workgroup looks through all slots: the search grows with the square of the rows, 65536 of them read 34 GB of slots a head)
    SRVP_REQUIRE(!d->slots || d->B <= 65536, "srvp_linear_attention_step: at most 65536 rows with slots, got %d", d->B);
    SRVP_REQUIRE(d->slots || d->B <= d->nslots, "srvp_linear_attention_step: %d rows for %d states", d->B, d->nslots);
    SRVP_REQUIRE((uintptr_t)d->state % 16 == 0, "srvp_linear_attention_step: state must be 16-byte aligned");
    StepArgs g;
    g.q = d->q; g.k = d->k; g.v = d->v; g.o = d->o;
    for (int i = 0; i < 2; ++i) { g.qs[i] = d->qs[i]; g.ks[i] = d->ks[i]; g.vs[i] = d->vs[i]; g.os[i] = d->os[i]; }
    g.log_decay = d->log_decay; g.state = d->state; g.slots = (const long long*)d->slots;
    g.B = d->B; g.H = d->H; g.Dk = d->Dk; g.Dv = d->Dv; g.nslots = d->nslots; g.scale = d->scale;
    if (d->elem_f32) hipLaunchKernelGGL(step_kernel<float>, dim3(d->B * d->H, (d->Dv + BLOCK - 1) / BLOCK), dim3(256), 0, (hipStream_t)stream, g);
    else hipLaunchKernelGGL(step_kernel<bf16_t>, dim3(d->B * d->H, (d->Dv + BLOCK - 1) / BLOCK), dim3(256), 0, (hipStream_t)stream, g);
    SRVP_CHECK_LAUNCH("srvp_linear_attention_step");
    return SRVP_OK;
}
