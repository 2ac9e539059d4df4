// Orthogonalised updates: the quintic Newton-Schulz iteration
//     X <- X / max(|X|_F, eps);   steps times:  A = X X^T,  X <- a X + (b A + c A A) X
// on the short side of each matrix, and the optimiser step that uses it (momentum, iteration, update of the weights).
//
// Matrices of up to 64 x 128 run in one workgroup, in fp32 out of LDS.  Larger ones that fit into the LDS of a compute unit as
// fp16 factors run in one workgroup as well (one launch instead of 17 that wait for each other: 128 x 128 fp32 64 us
// instead of 102).  The others take three tiled products a step (gemm_nt.h).  The factors of both are fp16, scaled by powers of
// two so that the range is used: the iterates' singular values, and with them the entries, stay below 3.9, so X is held times
// S = 2^14 and A, B = b A + c A A (below 15.3) times 2^12.  One fp16 term has a relative rounding of 2^-11, an eighth of that of
// bf16 inputs.  Two terms (the split form of gemm_nt.h) hold 22 bits of every entry of X above 2^-28 of the matrix's norm and an
// absolute 2^-50 of the norm below, so that rows and columns far smaller than the others come out as accurate as an fp32
// evaluation has them (1000 x 1000, half of the rows times 1e-2, 1e-4, 1e-6: the worst row 3.6e-6, 3.8e-6, 3.1e-6 off, nearly all
// of it from the sums; times 1e-8: 4.3e-5).  Sums are fp32 in the matrix cores, the norm is a sum of fp64.
#include <cmath>
#include <utility>
#include "gemm_nt.h"

namespace {

constexpr float S_SCALE = 16384.f, T_SCALE = 4096.f;
constexpr int MAX_STEPS = 32, NORM_BLOCKS = 512;

struct Coef {
    float v[3 * MAX_STEPS];
};

// ---- what is orthogonalised, and where the result goes ------------------------------------------
template <class T>
struct FromTensor {                                   // a matrix of a batch
    const T *x;
    int64_t batch;
    bool whole;                                       // matrices and rows of whole 16-byte pieces
    bool is_wide;
    DEV bool wide(int) const { return is_wide; }
    DEV void first8(int z, int64_t i, float *v, int valid) const { load8(x + z * batch + i, v, valid, whole); }
    DEV void again8(int z, int64_t i, float *v, int valid) const { load8(x + z * batch + i, v, valid, whole); }
    DEV float first(int z, int64_t i) const { return to_f32(x[z * batch + i]); }
    DEV float again(int z, int64_t i) const { return to_f32(x[z * batch + i]); }
};
template <class T>
struct FromMomentum {                                 // g and the momentum, which the first pass updates
    const T *g;
    float *m;
    float mu;
    int nesterov;
    DEV float first(int, int64_t i) const {
        const float w = mu * m[i] + to_f32(g[i]);
        m[i] = w;
        return nesterov ? to_f32(g[i]) + mu * w : w;
    }
    DEV float again(int, int64_t i) const { return nesterov ? to_f32(g[i]) + mu * m[i] : m[i]; }
};
constexpr int TOGETHER = 8;                           // large matrices of one size that go through the products together
template <class T>
struct FromMomenta {                                  // the same for several matrices, with pieces of 8
    const T *g[TOGETHER];
    float *m[TOGETHER];
    float mu;
    int nesterov;
    unsigned whole_bits, wide_bits;
    DEV bool wide(int z) const { return wide_bits >> z & 1; }
    DEV void first8(int z, int64_t i, float *v, int valid) const {
        const bool whole = whole_bits >> z & 1;
        float w[8];
        load8((const float *)m[z] + i, w, valid, whole);
        load8(g[z] + i, v, valid, whole);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            w[k] = mu * w[k] + v[k];
            v[k] = nesterov ? v[k] + mu * w[k] : w[k];
        }
        store8(m[z] + i, w, valid, whole);
    }
    DEV void again8(int z, int64_t i, float *v, int valid) const {
        const bool whole = whole_bits >> z & 1;
        float w[8];
        load8((const float *)m[z] + i, w, valid, whole);
        if (nesterov) load8(g[z] + i, v, valid, whole);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = nesterov ? v[k] + mu * w[k] : w[k];
    }
};
template <class T>
struct ToTensor {
    T *out;
    int64_t batch;
    bool whole;                                       // rows of whole 16-byte pieces
    DEV void put(int z, int64_t i, float v) const { out[z * batch + i] = from_f32<T>(v); }
    DEV void put8(int z, int64_t i, const float *v, int valid) const { store8(out + z * batch + i, v, valid, whole); }
};
template <class T>
struct ToWeights {
    T *p;
    float keep, factor;                               // 1 - lr wd, lr sqrt(max(1, rows / cols))
    DEV void put(int, int64_t i, float v) const { p[i] = from_f32<T>(to_f32(p[i]) * keep - factor * v); }
};
template <class T>
struct ToManyWeights {
    T *p[TOGETHER];
    float keep, factor;
    unsigned whole_bits;
    DEV void put8(int z, int64_t i, float *v, int valid) const {
        const bool whole = whole_bits >> z & 1;
        float w[8];
        load8((const T *)p[z] + i, w, valid, whole);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = w[k] * keep - factor * v[k];
        store8(p[z] + i, v, valid, whole);
    }
};

DEV double block_sum_d(double v, double *red) {       // over the 256 threads of a workgroup, the same value in all
    v = wave_sum_d(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

// ---- small matrices --------------------------------------------------------------------------
// One workgroup, one matrix, in fp32: r <= c after the transposition, X [r][c], A and B [r][r] in LDS, padded with zeros
// to whole 16 x 16 blocks.  A wave forms a block with v_mfma_f32_16x16x4_f32 (32 cycles for 4 of the sum's terms: these, the
// LDS reads in front of them and four barriers a step are the time): 16 terms from one 16-byte read of each factor, lane
// q of a row taking terms 4 q .. 4 q + 3 of them, which for both factors is the same order.
// Row strides are 4 modulo 64 words: 16 rows of 16 bytes touch every bank as often.  32 x 30, 5 steps: 10.4 us.
constexpr int SMALL_R = 64, SMALL_C = 128, XS = SMALL_C + 4, AS = SMALL_R + 4;
constexpr int SMALL_LDS = SMALL_R * XS + 2 * SMALL_R * AS;

DEV f32x4_t mfma_f32(float a, float b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

template <int WAVES>
DEV double group_sum_d(double v, double *red) {       // over the workgroup, the same value in all threads
    v = wave_sum_d(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) s += red[i];
    return s;
}

template <int WAVES, class From, class To>
DEV void small_iterate(const From &from, const To &to, int z, int rows, int cols, const Coef &coef, int steps, double eps, float *lds) {
    __shared__ double red[WAVES];
    constexpr int THREADS = 64 * WAVES, MAX_BLOCKS = (SMALL_R / 16) * (SMALL_C / 16) / WAVES;      // of X, a wave
    float *X = lds, *A = X + SMALL_R * XS, *B = A + SMALL_R * AS;
    const bool wide = rows <= cols;
    const int r = wide ? rows : cols, c = wide ? cols : rows, n = rows * cols, t = threadIdx.x;
    const int rb = (r + 15) >> 4, cb = (c + 15) >> 4, lane = t & 63, wave = t >> 6, i16 = lane & 15, q = lane >> 4;
    for (int e = t; e < SMALL_R * XS; e += THREADS) X[e] = 0.f;
    __syncthreads();
    double s = 0.0;
    for (int e = t; e < n; e += THREADS) {
        const int i = e / cols, j = e - i * cols;
        const float v = from.first(z, e);
        X[wide ? i * XS + j : j * XS + i] = v;
        s += (double)v * (double)v;
    }
    const double norm = sqrt(group_sum_d<WAVES>(s, red)), inv = 1.0 / (norm > eps ? norm : (norm == norm ? eps : norm));
    for (int e = t; e < r * c; e += THREADS) {
        const int i = e / c, at = i * XS + e - i * c;
        X[at] = (float)((double)X[at] * inv);
    }
    __syncthreads();
    // sum over `blocks` groups of 16 terms of rows u (of U) and v (of V), both contiguous along the sum
    auto dot = [&](const float *U, const float *V, int blocks, f32x4_t acc) {
        for (int k = 0; k < blocks; ++k) {
            const f32x4_t u = *(const f32x4_t *)(U + k * 16 + q * 4), v = *(const f32x4_t *)(V + k * 16 + q * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc = mfma_f32(u[e], v[e], acc);
        }
        return acc;
    };
    for (int k = 0; k < steps; ++k) {
        const float ca = coef.v[3 * k], cb3 = coef.v[3 * k + 1], cc = coef.v[3 * k + 2];
        for (int b = wave; b < rb * rb; b += WAVES) {          // A = X X^T
            const int bi = b / rb, bj = b - bi * rb;
            const f32x4_t acc = dot(X + (bi * 16 + i16) * XS, X + (bj * 16 + i16) * XS, cb, f32x4_t{0, 0, 0, 0});
#pragma unroll
            for (int e = 0; e < 4; ++e) A[(bi * 16 + q * 4 + e) * AS + bj * 16 + i16] = acc[e];
        }
        __syncthreads();
        for (int b = wave; b < rb * rb; b += WAVES) {          // B = b A + c A A (the second factor by its rows: A is symmetric)
            const int bi = b / rb, bj = b - bi * rb;
            const f32x4_t acc = dot(A + (bi * 16 + i16) * AS, A + (bj * 16 + i16) * AS, rb, f32x4_t{0, 0, 0, 0});
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int at = (bi * 16 + q * 4 + e) * AS + bj * 16 + i16;
                B[at] = __builtin_fmaf(cc, acc[e], cb3 * A[at]);
            }
        }
        __syncthreads();
        f32x4_t next[MAX_BLOCKS];                              // X <- a X + B X, written once every wave has read X
#pragma unroll
        for (int h = 0; h < MAX_BLOCKS; ++h) {
            const int b = wave + h * WAVES;
            if (b >= rb * cb) break;
            const int bi = b / cb, bj = b - bi * cb;
            f32x4_t acc;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = ca * X[(bi * 16 + q * 4 + e) * XS + bj * 16 + i16];
            for (int m = 0; m < rb; ++m) {
                const f32x4_t u = *(const f32x4_t *)(B + (bi * 16 + i16) * AS + m * 16 + q * 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc = mfma_f32(u[e], X[(m * 16 + q * 4 + e) * XS + bj * 16 + i16], acc);
            }
            next[h] = acc;
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < MAX_BLOCKS; ++h) {
            const int b = wave + h * WAVES;
            if (b >= rb * cb) break;
            const int bi = b / cb, bj = b - bi * cb;
#pragma unroll
            for (int e = 0; e < 4; ++e) X[(bi * 16 + q * 4 + e) * XS + bj * 16 + i16] = next[h][e];
        }
        __syncthreads();
    }
    for (int e = t; e < n; e += THREADS) {
        const int i = e / cols, j = e - i * cols;
        to.put(z, e, X[wide ? i * XS + j : j * XS + i]);
    }
}

// Waves of a workgroup: 4 hold up to 32 x 32, 16 everything up to 64 x 128.
inline bool needs_16_waves(int64_t rows, int64_t cols) { return rows > 32 || cols > 32; }

template <int WAVES, class T>
__global__ __launch_bounds__(64 * WAVES) void k_small(FromTensor<T> from, ToTensor<T> to, int rows, int cols, Coef coef, int steps, double eps) {
    __shared__ __attribute__((aligned(16))) float lds[SMALL_LDS];
    small_iterate<WAVES>(from, to, blockIdx.x, rows, cols, coef, steps, eps, lds);
}

constexpr int TABLE = 24;              // matrices of one launch: the table travels with the kernel's arguments
struct SmallTable {
    void *p[TABLE];
    const void *g[TABLE];
    float *m[TABLE];
    int rows[TABLE], cols[TABLE];
    float factor[TABLE];
};

// ---- matrices that fit into one compute unit as fp16 factors --------------------------------------
// One workgroup of 16 waves, one matrix: X [r][c] and A, overwritten by B, [r][r] in LDS as fp16, scaled as the images of
// the large path are (one term, or two planes in the split form), padded with zeros to whole 32 x 32 blocks.  A wave forms
// such blocks on v_mfma_f32_16x16x32_f16 (four 16 x 16 tiles from two fragments of each factor; a tile's lane holds four
// successive columns of one row).  The sums of A and A A run along rows of LDS; that of B X runs down the columns of X,
// which the transposing read ds_read_b64_tr_b16 gives (4 rows of 16 columns each).  Rows are 16 bytes longer than their
// padded length, so that 16 of them spread over the banks.  Five barriers a step instead of three launches.  Bound by the one
// compute unit's LDS reads and by latency: 65 x 65 with one term 22 us (75 with tiled products), 38 with two;
// 128 x 128 40 and 64, 64 x 512 52 and 78.
constexpr int FIT_LDS = 150 * 1024, FIT_WAVES = 16, FIT_BLOCKS = 3;     // blocks of X that a wave holds

__host__ DEV int64_t fit_bytes(int64_t r, int64_t c, bool split) {
    const int64_t r32 = (r + 31) & ~31, c32 = (c + 31) & ~31;
    return r32 * (c32 + 8 + r32 + 8) * (split ? 4 : 2);
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) char lds_byte;

DEV nt::f16x8 read_down(const _Float16 *p, int pitch) {        // 8 rows of one column, out of what 16 lanes point at
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)p), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p + 4 * pitch));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    return __builtin_bit_cast(nt::f16x8, (s16x8)__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

template <bool SPLIT>
struct Plane {                          // a factor in LDS
    _Float16 *h, *l;
    int pitch;
    DEV f32x4_t get4(int row, int col) const {
        const nt::f16x4 a = *(const nt::f16x4 *)(h + row * pitch + col);
        f32x4_t v = {(float)a[0], (float)a[1], (float)a[2], (float)a[3]};
        if (SPLIT) {
            const nt::f16x4 b = *(const nt::f16x4 *)(l + row * pitch + col);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += (float)b[e] * (1.f / nt::REST);
        }
        return v;
    }
    DEV void put4(int row, int col, f32x4_t v) const {
        nt::f16x4 a, b;
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = (_Float16)v[e], b[e] = (_Float16)((v[e] - (float)a[e]) * nt::REST);
        *(nt::f16x4 *)(h + row * pitch + col) = a;
        if (SPLIT) *(nt::f16x4 *)(l + row * pitch + col) = b;
    }
    DEV void put(int row, int col, float v) const {
        const _Float16 a = (_Float16)v;
        h[row * pitch + col] = a;
        if (SPLIT) l[row * pitch + col] = (_Float16)((v - (float)a) * nt::REST);
    }
};

template <int N>
struct Block {                          // N x N tiles of a product: tile (ti, tj), row ti * 16 + (lane & 15), columns tj * 16 + 4 (lane >> 4) + 0..3
    f32x4_t t[N][N];
};

// sum over n terms of rows u0.. of U and rows v0.. of V (DOWN: of columns v0.. of V, whose rows the sum runs along)
template <bool SPLIT, bool DOWN, int N>
DEV Block<N> block_product(const Plane<SPLIT> &U, int u0, const Plane<SPLIT> &V, int v0, int n, int lane) {
    const int r = lane & 15, q = lane >> 4;
    Block<N> b, cross;                  // cross: the products with remainders
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) b.t[i][j] = cross.t[i][j] = f32x4_t{0, 0, 0, 0};
    const int u_at = (u0 + r) * U.pitch + q * 8, v_at = DOWN ? (q * 8 + (r >> 2)) * V.pitch + v0 + (r & 3) * 4 : (v0 + r) * V.pitch + q * 8;
#pragma unroll 2
    for (int k = 0; k < n; k += 32) {
        nt::f16x8 uh[N], ul[N], vh[N], vl[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = u_at + i * 16 * U.pitch + k;
            uh[i] = *(const nt::f16x8 *)(U.h + at);
            if (SPLIT) ul[i] = *(const nt::f16x8 *)(U.l + at);
            if (DOWN) {
                const int to = v_at + k * V.pitch + i * 16;
                vh[i] = read_down(V.h + to, V.pitch);
                if (SPLIT) vl[i] = read_down(V.l + to, V.pitch);
            } else {
                const int to = v_at + i * 16 * V.pitch + k;
                vh[i] = *(const nt::f16x8 *)(V.h + to);
                if (SPLIT) vl[i] = *(const nt::f16x8 *)(V.l + to);
            }
        }
        auto add = [&](const nt::f16x8 *v, const nt::f16x8 *u, Block<N> &to) {
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int j = 0; j < N; ++j) to.t[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[j], u[i], to.t[i][j], 0, 0, 0);
        };
        if (SPLIT) add(vl, uh, cross), add(vh, ul, cross);
        add(vh, uh, b);
    }
    if (SPLIT) {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) b.t[i][j] += cross.t[i][j] * (1.f / nt::REST);
    }
    return b;
}

// A = X X^T (times T_SCALE), then B = b A + c A A in its place, by blocks of N x N tiles: at most one a wave.
template <bool SPLIT, int N>
DEV void fit_poly(const Plane<SPLIT> &X, const Plane<SPLIT> &A, int r32, int c32, float cb3, float cc, int wave, int lane) {
    const int i16 = lane & 15, q = lane >> 4, side = r32 / (16 * N), ba = wave / side, bj = wave - ba * side;
    const bool has = wave < side * side;
    auto each = [&](auto f) {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) f(i, j, (ba * N + i) * 16 + i16, (bj * N + j) * 16 + q * 4);
    };
    Block<N> b;
    if (has) {
        b = block_product<SPLIT, false, N>(X, ba * N * 16, X, bj * N * 16, c32, lane);
        each([&](int i, int j, int row, int col) {
            f32x4_t v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = b.t[i][j][e] * (T_SCALE / (S_SCALE * S_SCALE));
            A.put4(row, col, v);
        });
    }
    __syncthreads();
    if (has) {                                         // the second factor by its rows: A is symmetric
        b = block_product<SPLIT, false, N>(A, ba * N * 16, A, bj * N * 16, r32, lane);
        each([&](int i, int j, int row, int col) {
            const f32x4_t a = A.get4(row, col);
#pragma unroll
            for (int e = 0; e < 4; ++e) b.t[i][j][e] = __builtin_fmaf(cc, b.t[i][j][e] * (1.f / T_SCALE), cb3 * a[e]);
        });
    }
    __syncthreads();
    if (has) each([&](int i, int j, int row, int col) { A.put4(row, col, b.t[i][j]); });
    __syncthreads();
}

template <bool SPLIT, class From, class To>
DEV void fit_iterate(const From &from, const To &to, int z, int rows, int cols, const Coef &coef, int steps, double eps, _Float16 *lds) {
    __shared__ double red[FIT_WAVES];
    const bool wide = rows <= cols;
    const int r = wide ? rows : cols, c = wide ? cols : rows, n = rows * cols, t = threadIdx.x;
    const int r32 = (r + 31) & ~31, c32 = (c + 31) & ~31, rb = r32 >> 5, cb = c32 >> 5;
    const int wave0 = __builtin_amdgcn_readfirstlane(t >> 6);
    Plane<SPLIT> X{lds, lds + r32 * (c32 + 8), c32 + 8}, A;
    A.h = lds + r32 * (c32 + 8) * (SPLIT ? 2 : 1), A.l = A.h + r32 * (r32 + 8), A.pitch = r32 + 8;
    for (int e = t; e < r32 * (c32 + 8) * (SPLIT ? 2 : 1) / 8; e += 64 * FIT_WAVES) ((f32x4_t *)lds)[e] = f32x4_t{0, 0, 0, 0};
    double s = 0.0;
    for (int e = t; e < n; e += 64 * FIT_WAVES) {
        const float v = from.first(z, e);
        s += (double)v * (double)v;
    }
    const double norm = sqrt(group_sum_d<FIT_WAVES>(s, red)), inv = (double)S_SCALE / (norm > eps ? norm : (norm == norm ? eps : norm));
    for (int e = t; e < n; e += 64 * FIT_WAVES) {      // the same thread saw the same elements: no barrier for the momentum
        const int i = e / cols, j = e - i * cols;
        const float v = (float)((double)from.again(z, e) * inv);
        X.put(wide ? i : j, wide ? j : i, v);
    }
    __syncthreads();
    for (int k = 0; k < steps; ++k) {
        // the compiler would keep every address of a step in registers through the loop: they are formed anew instead
        int wave = wave0, lane = t & 63;
        asm volatile("" : "+s"(wave), "+v"(lane));
        const int i16 = lane & 15, q = lane >> 4;
        const float ca = coef.v[3 * k], cb3 = coef.v[3 * k + 1], cc = coef.v[3 * k + 2];
        if (r32 <= 64) fit_poly<SPLIT, 1>(X, A, r32, c32, cb3, cc, wave, lane);       // 16 tiles for 16 waves
        else fit_poly<SPLIT, 2>(X, A, r32, c32, cb3, cc, wave, lane);
        const bool last = k + 1 == steps;
        Block<2> x[FIT_BLOCKS];                           // X <- a X + B X, written once every wave has read X
#pragma unroll
        for (int h = 0; h < FIT_BLOCKS; ++h) {
            const int id = wave + h * FIT_WAVES, bi = id / cb, bc = id - bi * cb;
            if (id < rb * cb) {
                x[h] = block_product<SPLIT, true, 2>(A, bi * 32, X, bc * 32, r32, lane);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const f32x4_t old = X.get4(bi * 32 + i * 16 + i16, bc * 32 + j * 16 + q * 4);
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[h].t[i][j][e] = __builtin_fmaf(ca, old[e], x[h].t[i][j][e] * (1.f / T_SCALE));
                    }
            }
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < FIT_BLOCKS; ++h) {
            const int id = wave + h * FIT_WAVES, bi = id / cb, bc = id - bi * cb;
            if (id < rb * cb) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int row = bi * 32 + i * 16 + i16, col = bc * 32 + j * 16 + q * 4;
                        if (!last) {
                            X.put4(row, col, x[h].t[i][j]);
                        } else if (row < r) {          // in fp32, where it belongs
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (col + e < c) to.put(z, wide ? (int64_t)row * cols + col + e : (int64_t)(col + e) * cols + row, x[h].t[i][j][e] * (1.f / S_SCALE));
                        }
                    }
            }
        }
        __syncthreads();
    }
}

template <bool SPLIT, class T>
__global__ __launch_bounds__(64 * FIT_WAVES) void k_fit(FromTensor<T> from, ToTensor<T> to, int rows, int cols, Coef coef, int steps, double eps) {
    __shared__ __attribute__((aligned(16))) _Float16 lds[FIT_LDS / 2];
    fit_iterate<SPLIT>(from, to, blockIdx.x, rows, cols, coef, steps, eps, lds);
}

template <class T>
__global__ __launch_bounds__(1024) void k_small_muon(SmallTable tab, float mu, int nesterov, float keep, Coef coef, int steps, double eps) {
    __shared__ __attribute__((aligned(16))) float lds[SMALL_LDS];
    const int z = blockIdx.x;
    small_iterate<16>(FromMomentum<T>{(const T *)tab.g[z], tab.m[z], mu, nesterov}, ToWeights<T>{(T *)tab.p[z], keep, tab.factor[z]}, 0, tab.rows[z],
                  tab.cols[z], coef, steps, eps, lds);
}

template <bool SPLIT, class T>
__global__ __launch_bounds__(64 * FIT_WAVES) void k_fit_muon(SmallTable tab, float mu, int nesterov, float keep, Coef coef, int steps, double eps) {
    __shared__ __attribute__((aligned(16))) _Float16 lds[FIT_LDS / 2];
    const int z = blockIdx.x;
    fit_iterate<SPLIT>(FromMomentum<T>{(const T *)tab.g[z], tab.m[z], mu, nesterov}, ToWeights<T>{(T *)tab.p[z], keep, tab.factor[z]}, 0, tab.rows[z],
                       tab.cols[z], coef, steps, eps, lds);
}

// ---- large matrices ----------------------------------------------------------------------------
// A factor in the workspace: rows of fp16, or of blocks of 32 leading halves and 32 remainders (SPLIT).
struct Image {
    char *base;
    int64_t ld, batch;                 // bytes
};
DEV int64_t img_row(const Image &im, int z, int64_t row) { return z * im.batch + row * im.ld; }
template <bool SPLIT>
DEV int64_t img_col(int col) { return SPLIT ? (int64_t)(col >> 5) * 128 + (col & 31) * 2 : (int64_t)col * 2; }

template <bool SPLIT>
struct Eight {                         // eight values of an image as they lie there
    nt::f16x8 h[SPLIT ? 2 : 1];
    DEV float operator[](int i) const { return SPLIT ? (float)h[0][i] + (float)h[SPLIT ? 1 : 0][i] * (1.f / nt::REST) : (float)h[0][i]; }
};
template <bool SPLIT>
DEV Eight<SPLIT> img_load8(const Image &im, int z, int64_t row, int col) {
    const char *p = im.base + img_row(im, z, row) + img_col<SPLIT>(col);
    Eight<SPLIT> v;
    v.h[0] = *(const nt::f16x8 *)p;
    if (SPLIT) v.h[SPLIT ? 1 : 0] = *(const nt::f16x8 *)(p + 64);
    return v;
}
template <bool SPLIT>
DEV void img_store8(const Image &im, int z, int64_t row, int col, const float *v) {
    char *p = im.base + img_row(im, z, row) + img_col<SPLIT>(col);
    nt::f16x8 h, l;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (_Float16)v[i], l[i] = (_Float16)((v[i] - (float)h[i]) * nt::REST);
    *(nt::f16x8 *)p = h;
    if (SPLIT) *(nt::f16x8 *)(p + 64) = l;
}

// Sum of squares of each matrix (and, for the optimiser, the new momentum): NORM_BLOCKS fp64 partial sums each.  Bound by
// memory: 4096 x 4096 bf16 9.8 us (3.4 TB/s).
template <class From>
__global__ __launch_bounds__(256) void k_norm(From from, int64_t n, double *__restrict__ part) {
    __shared__ double red[4];
    const int z = blockIdx.z;
    double s = 0.0;
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; i < n; i += (int64_t)gridDim.x * 2048) {
        float v[8];
        from.first8(z, i, v, (int)(n - i < 8 ? n - i : 8));
#pragma unroll
        for (int k = 0; k < 8; ++k) s += (double)v[k] * (double)v[k];
    }
    s = block_sum_d(s, red);
    if (threadIdx.x == 0) part[z * NORM_BLOCKS + blockIdx.x] = s;
}

// 64 rows of an image from `row`: zeros from column `from` to the end of the row (16-byte pieces; `from` rounded down to 8,
// the columns in front of it are written later, by the products).
template <bool SPLIT>
DEV void zero_pads(const Image &im, int z, int row, int rows, int from) {
    const int end = (int)(SPLIT ? im.ld / 4 : im.ld / 2), first = from & ~7, pieces = (end - first) / 8;
    const float zero[8] = {};
    for (int e = threadIdx.x; e < 64 * pieces; e += 256) {
        const int i = row + e / pieces, j = first + e % pieces * 8;
        if (i < rows) img_store8<SPLIT>(im, z, i, j, zero);
    }
}

// X0 = x S_SCALE / max(norm, eps) into both images, P [r, c] and Q = P^T [c, r], zeros behind the rows.  64 x 64 tiles.  The images
// that the products fill first get the zeros behind their rows here too.  Bound by memory: 4096 x 4096 bf16 18 us (5.5 TB/s,
// x out of the last-level cache).
template <class From, bool SPLIT>
__global__ __launch_bounds__(256) void k_prepare(From from, int r, int c, const double *__restrict__ part, int blocks, double eps, double scale,
                                                 Image P, Image Q, Image Q2, Image A, Image B) {
    __shared__ double red[4];
    __shared__ float tile[64][65];
    const int z = blockIdx.z, t = threadIdx.x;
    double s = 0.0;
    for (int i = t; i < blocks; i += 256) s += part[z * NORM_BLOCKS + i];
    const double norm = sqrt(block_sum_d(s, red)), inv = scale / (norm > eps ? norm : (norm == norm ? eps : norm));
    if (blockIdx.y == 0) zero_pads<SPLIT>(Q2, z, blockIdx.x * 64, c, r);
    if (blockIdx.x == 0) zero_pads<SPLIT>(A, z, blockIdx.y * 64, r, r), zero_pads<SPLIT>(B, z, blockIdx.y * 64, r, r);
    const bool wide = from.wide(z);
    const int rows = wide ? r : c, cols = wide ? c : r;            // of x, and the tile's place in it
    const int r0 = (wide ? blockIdx.y : blockIdx.x) * 64, c0 = (wide ? blockIdx.x : blockIdx.y) * 64;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int e = t + h * 256, i = e >> 3, j = (e & 7) * 8;
        float v[8] = {};
        if (r0 + i < rows && c0 + j < cols) from.again8(z, (int64_t)(r0 + i) * cols + c0 + j, v, cols - c0 - j);
#pragma unroll
        for (int k = 0; k < 8; ++k) tile[i][j + k] = (float)((double)v[k] * inv);
    }
    __syncthreads();
    const Image &same = wide ? P : Q, &flip = wide ? Q : P;        // the image in x's orientation, and the other one
    const int64_t end_c = SPLIT ? same.ld / 4 : same.ld / 2, end_r = SPLIT ? flip.ld / 4 : flip.ld / 2;
    for (int e = t; e < 512; e += 256) {
        const int i = e >> 3, j = (e & 7) * 8;
        float v[8];
        if (r0 + i < rows && c0 + j < end_c) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = tile[i][j + k];
            img_store8<SPLIT>(same, z, r0 + i, c0 + j, v);
        }
        if (c0 + i < cols && r0 + j < end_r) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = tile[j + k][i];
            img_store8<SPLIT>(flip, z, c0 + i, r0 + j, v);
        }
    }
}

struct NoFactors {
    static constexpr bool TURNED = false;
    typedef None Row, Col, Pre;
    DEV Pre pre(int, int, int) const { return {}; }
    DEV Row row(int, int) const { return {}; }
    DEV Col col(int, int) const { return {}; }
};
template <bool SPLIT>
DEV void img_store_half(const Image &im, int z, int64_t row, int col, int half, nt::f16x8 v) {
    *(nt::f16x8 *)(im.base + img_row(im, z, row) + img_col<SPLIT>(col) + half * 64) = v;
}
// The two symmetric products compute their tiles on and below the diagonal; a tile below it is stored turned as well.
// 4096 x 4096, one term: Gram and polynomial 71 to 76 us each (253 tiles of 192 x 192, 0.95 PFLOP/s of what is computed),
// the update 113 to 120 us (1.2 PFLOP/s); 1024 x 4096: 14.7, 7.2 and 16.6 us.  Split form: 245, 255 and 348 us (528 tiles of
// 128 x 128, 16 of them in a third round; 1.2 PFLOP/s in the update's three products); 33.7, 12.8 and 35.7 us; 3 of 777 x 1000
// 16.9, 15.9 and 28.0 us.
template <bool SPLIT>
struct GramOut : NoFactors {           // A = X X^T (times T_SCALE); zeros behind the rows
    static constexpr bool TURNED = true;
    Image A;
    float scale;
    int N;
    DEV void put_turned(int z, int row, int col, int half, nt::f16x8 v) const { img_store_half<SPLIT>(A, z, row, col, half, v); }
    DEV void put(int z, int m, int n, float *v, Row, Col, Pre) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = n + i < N ? v[i] * scale : 0.f;
        img_store8<SPLIT>(A, z, m, n, v);
    }
};
template <bool SPLIT>
struct PolyOut : NoFactors {           // B = b A + c A A (times T_SCALE)
    static constexpr bool TURNED = true;
    Image A, B;
    float b, c;
    int N;
    DEV void put_turned(int z, int row, int col, int half, nt::f16x8 v) const { img_store_half<SPLIT>(B, z, row, col, half, v); }
    typedef Eight<SPLIT> Pre;
    DEV Pre pre(int z, int m, int n) const { return img_load8<SPLIT>(A, z, m, n); }
    DEV void put(int z, int m, int n, float *v, Row, Col, const Pre &a) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = n + i < N ? __builtin_fmaf(c, v[i] * (1.f / T_SCALE), b * a[i]) : 0.f;
        img_store8<SPLIT>(B, z, m, n, v);
    }
};
template <bool SPLIT>
struct NextOut : NoFactors {           // X <- a X + B X into P (in place: a tile reads its own entries only) and the other Q
    static constexpr bool TURNED = true;
    Image P, Q;
    float a;
    int N;
    DEV void put_turned(int z, int row, int col, int half, nt::f16x8 v) const { img_store_half<SPLIT>(Q, z, row, col, half, v); }
    typedef Eight<SPLIT> Pre;
    DEV Pre pre(int z, int m, int n) const { return img_load8<SPLIT>(P, z, m, n); }
    DEV void put(int z, int m, int n, float *v, Row, Col, const Pre &x) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = n + i < N ? __builtin_fmaf(a, x[i], v[i] * (1.f / T_SCALE)) : 0.f;
        img_store8<SPLIT>(P, z, m, n, v);
    }
};
template <bool SPLIT, class To>
struct LastOut : NoFactors {           // the last step: X in the orientation of the result (P, or Q for tall matrices)
    Image X;
    float a, scale;                    // scale = 1 / S_SCALE
    To to;
    int N;
    typedef Eight<SPLIT> Pre;
    DEV Pre pre(int z, int m, int n) const { return img_load8<SPLIT>(X, z, m, n); }
    DEV void put(int z, int m, int n, float *v, Row, Col, const Pre &x) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __builtin_fmaf(a, x[i], v[i] * (1.f / T_SCALE)) * scale;
        to.put8(z, (int64_t)m * N + n, v, N - n);
    }
};

struct Plan {
    int64_t r, c, part, p, q0, q1, a, b, total;
    int64_t ld_r, ld_c;                // bytes of a row along the short and the long side
    Plan(int64_t batch, int64_t rows, int64_t cols, bool split) {
        r = rows < cols ? rows : cols, c = rows < cols ? cols : rows;
        ld_r = split ? nt::pad_to(r, 32) * 4 : nt::pad_to(r, 64) * 2;
        ld_c = split ? nt::pad_to(c, 32) * 4 : nt::pad_to(c, 64) * 2;
        int64_t at = 0;
        auto take = [&](int64_t bytes) {
            const int64_t here = at;
            at += nt::pad_to(bytes, 256);
            return here;
        };
        part = take(batch * NORM_BLOCKS * 8);
        p = take(batch * r * ld_c);
        q0 = take(batch * c * ld_r);
        q1 = take(batch * c * ld_r);
        a = take(batch * r * ld_r);
        b = take(batch * r * ld_r);
        total = at;
    }
};

bool is_small(int64_t rows, int64_t cols) {
    const int64_t r = rows < cols ? rows : cols, c = rows < cols ? cols : rows;
    return r <= SMALL_R && c <= SMALL_C;
}

// One compute unit holds the matrix (it needs no workspace then, like a small one).
bool fits(int64_t rows, int64_t cols, bool split) {
    const int64_t r = rows < cols ? rows : cols, c = rows < cols ? cols : rows;
    return r <= 128 && c <= 65536 && fit_bytes(r, c, split) <= FIT_LDS && ((r + 31) / 32) * ((c + 31) / 32) <= FIT_WAVES * FIT_BLOCKS;
}

// `batch` matrices of short side r and long side c, the first `wides` of them with rows <= cols.  `to_wide`, `to_tall`: where
// the two kinds go, counted from the first of each.
template <bool SPLIT, class From, class To>
int large(const From &from, const To &to_wide, const To &to_tall, int batch, int wides, int64_t r64, int64_t c64, int steps, const float *coef, double eps,
          char *ws, hipStream_t st) {
    constexpr int KIND = SPLIT ? nt::F16_SPLIT : nt::F16;
    const Plan pl(batch, r64, c64, SPLIT);
    const int r = (int)pl.r, c = (int)pl.c;
    double *part = (double *)(ws + pl.part);
    const Image P{ws + pl.p, pl.ld_c, r * pl.ld_c}, A{ws + pl.a, pl.ld_r, r * pl.ld_r}, B{ws + pl.b, pl.ld_r, r * pl.ld_r};
    Image Q{ws + pl.q0, pl.ld_r, c * pl.ld_r}, Q2{ws + pl.q1, pl.ld_r, c * pl.ld_r};
    const int64_t n = (int64_t)r * c;
    const int blocks = grid_for(n, 256 * 8, NORM_BLOCKS);
    hipLaunchKernelGGL((k_norm<From>), dim3(blocks, 1, batch), dim3(256), 0, st, from, n, part);
    DPD_LAUNCH_CHECK();
    hipLaunchKernelGGL((k_prepare<From, SPLIT>), dim3((unsigned)((c + 63) / 64), (unsigned)((r + 63) / 64), batch), dim3(256), 0, st, from, r, c, part, blocks,
                       eps, (double)S_SCALE, P, Q, Q2, A, B);
    DPD_LAUNCH_CHECK();
    auto product = [&](const Image &x, int M, const Image &y, int N, bool symmetric, int many, const auto &epi) {
        nt::Args g{};
        g.a = x.base, g.lda = x.ld, g.a_batch = x.batch, g.b = y.base, g.ldb = y.ld, g.b_batch = y.batch, g.M = M, g.N = N;
        g.steps = g.wrap = (int)(x.ld / nt::STEP), g.tail = nt::STEP, g.lower = symmetric;
        return nt::product<KIND>(g, many, epi, st);
    };
    auto from_z = [](Image im, int z) {
        im.base += z * im.batch;
        return im;
    };
    for (int k = 0; k < steps; ++k) {
        const float *f = coef + 3 * k;
        int rc = product(P, r, P, r, true, batch, GramOut<SPLIT>{{}, A, T_SCALE / (S_SCALE * S_SCALE), r});
        if (!rc) rc = product(A, r, A, r, true, batch, PolyOut<SPLIT>{{}, A, B, f[1], f[2], r});
        if (!rc && k + 1 < steps) {
            rc = product(B, r, Q, c, false, batch, NextOut<SPLIT>{{}, P, Q2, f[0], c});
            std::swap(Q, Q2);
        } else if (!rc) {
            if (wides) rc = product(B, r, Q, c, false, wides, LastOut<SPLIT, To>{{}, P, f[0], 1.f / S_SCALE, to_wide, c});
            if (!rc && batch > wides) {
                const Image q = from_z(Q, wides);
                rc = product(q, c, from_z(B, wides), r, false, batch - wides, LastOut<SPLIT, To>{{}, q, f[0], 1.f / S_SCALE, to_tall, r});
            }
        }
        if (rc) return rc;
    }
    return DPD_OK;
}

// The largest singular value that `steps` steps can reach from 1, and the largest |b s^2 + c s^4| on the way, must stay
// inside the range of the scaled fp16 factors.
int check_iteration(const char *who, int steps, const float *coef, double eps) {
    DPD_REQUIRE(steps >= 1 && steps <= MAX_STEPS && coef, DPD_ERR_SHAPE, "%s: %d steps not in 1..%d", who, steps, MAX_STEPS);
    DPD_REQUIRE(eps > 0.0 && eps < 1e300, DPD_ERR_SHAPE, "%s: eps must be positive and finite", who);
    double top = 1.0;
    for (int k = 0; k < steps; ++k) {
        const double a = coef[3 * k], b = coef[3 * k + 1], c = coef[3 * k + 2];
        double next = 0.0, poly = 0.0;
        for (int i = 1; i <= 64; ++i) {
            const double s = top * i / 64, s2 = s * s, p = b * s2 + c * s2 * s2;
            next = fmax(next, fabs(s * (a + p)));
            poly = fmax(poly, fabs(p));
        }
        next *= 1.02;
        DPD_REQUIRE(std::isfinite(a) && std::isfinite(b) && std::isfinite(c) && next <= 3.9 && poly <= 15.0, DPD_ERR_SHAPE, "%s: step %d with coefficients (%g, %g, %g) can take singular values out of range", who,
                    k, a, b, c);
        top = fmax(next, 1e-3);
    }
    return DPD_OK;
}

int check_matrix(const char *who, int64_t rows, int64_t cols) {
    DPD_REQUIRE(rows >= 0 && cols >= 0, DPD_ERR_INVALID_ARG, "%s: negative size", who);
    DPD_REQUIRE((rows < cols ? cols : rows) * 4 <= nt::MAX_ROW_BYTES - 512, DPD_ERR_SHAPE, "%s: a side of %lld is too long", who,
                (long long)(rows < cols ? cols : rows));
    return DPD_OK;
}

}  // namespace

extern "C" size_t dpd_orthogonalize_workspace_bytes(int64_t batch, int64_t rows, int64_t cols, int accurate) {
    if (batch <= 0 || rows <= 0 || cols <= 0 || is_small(rows, cols) || fits(rows, cols, accurate != 0)) return 256;
    return (size_t)Plan(batch, rows, cols, accurate != 0).total + 256;
}

extern "C" int dpd_orthogonalize(const void *x, int type, int64_t batch, int64_t rows, int64_t cols, int steps, const float *h_coef, double eps,
                                 int accurate, void *out, void *ws, size_t ws_bytes, void *stream) {
    DPD_REQUIRE(type == DPD_F32 || type == DPD_BF16 || type == DPD_F16, DPD_ERR_INVALID_ARG, "orthogonalize: element type %d", type);
    DPD_REQUIRE(batch >= 0 && batch <= INT32_MAX, DPD_ERR_INVALID_ARG, "orthogonalize: batch");
    if (const int rc = check_matrix("orthogonalize", rows, cols)) return rc;
    if (const int rc = check_iteration("orthogonalize", steps, h_coef, eps)) return rc;
    if (batch == 0 || rows == 0 || cols == 0) return DPD_OK;
    DPD_REQUIRE(x && out, DPD_ERR_INVALID_ARG, "orthogonalize: null pointer");
    hipStream_t st = as_stream(stream);
    Coef coef{};
    for (int i = 0; i < 3 * steps; ++i) coef.v[i] = h_coef[i];
    const bool small = is_small(rows, cols);
    if (small || fits(rows, cols, accurate != 0))
        return with_type(type, [&](auto t) {
            using T = decltype(t);
            constexpr int64_t MOST = 1 << 20;          // matrices a launch: a grid has fewer than 2^32 threads
            for (int64_t z = 0; z < batch; z += MOST) {
                const FromTensor<T> from{(const T *)x + z * rows * cols, rows * cols, false, rows <= cols};
                const ToTensor<T> to{(T *)out + z * rows * cols, rows * cols, false};
                const dim3 many((unsigned)(batch - z < MOST ? batch - z : MOST));
                auto go = [&](auto kernel, int threads) { hipLaunchKernelGGL(kernel, many, dim3(threads), 0, st, from, to, (int)rows, (int)cols, coef, steps, eps); };
                if (small && needs_16_waves(rows, cols)) go(k_small<16, T>, 1024);
                else if (small) go(k_small<4, T>, 256);
                else if (accurate) go(k_fit<true, T>, 64 * FIT_WAVES);
                else go(k_fit<false, T>, 64 * FIT_WAVES);
                DPD_LAUNCH_CHECK();
            }
            return DPD_OK;
        });
    DPD_REQUIRE(batch <= 65535, DPD_ERR_SHAPE, "orthogonalize: %lld matrices of this size in one call (at most 65535)", (long long)batch);
    DPD_REQUIRE(ws && ws_bytes >= dpd_orthogonalize_workspace_bytes(batch, rows, cols, accurate), DPD_ERR_WORKSPACE, "orthogonalize: workspace");
    char *w = (char *)(((uintptr_t)ws + 255) & ~(uintptr_t)255);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        const FromTensor<T> from{(const T *)x, rows * cols, ((uintptr_t)x & 15) == 0 && cols % 8 == 0, rows <= cols};
        const ToTensor<T> to{(T *)out, rows * cols, ((uintptr_t)out & 15) == 0 && cols % 8 == 0};
        const int wides = rows <= cols ? (int)batch : 0;
        return accurate ? large<true>(from, to, to, (int)batch, wides, rows, cols, steps, coef.v, eps, w, st)
                        : large<false>(from, to, to, (int)batch, wides, rows, cols, steps, coef.v, eps, w, st);
    });
}

// Large matrices with the same two sides share the launches of the products: up to TOGETHER of them, and no more than a
// gigabyte of workspace (a matrix that takes more goes alone).  The first of such a set finds its members.
struct Set {
    int index[TOGETHER], n, wides;
    int64_t r, c;
};
static int set_limit(int64_t r, int64_t c, int accurate) {
    const int64_t one = Plan(1, r, c, accurate != 0).total, fit = ((int64_t)1 << 30) / one;
    return fit < 1 ? 1 : fit > TOGETHER ? TOGETHER : (int)fit;
}
static bool leads_set(int i, int n, const int64_t *rows, const int64_t *cols, int accurate, Set *out) {
    auto lo = [&](int k) { return rows[k] < cols[k] ? rows[k] : cols[k]; };
    auto hi = [&](int k) { return rows[k] < cols[k] ? cols[k] : rows[k]; };
    const int64_t r = lo(i), c = hi(i);
    if (r <= 0 || is_small(r, c) || fits(r, c, accurate != 0)) return false;
    const int limit = set_limit(r, c, accurate);
    int before = 0;
    for (int k = 0; k < i; ++k) before += lo(k) == r && hi(k) == c;
    if (before % limit) return false;
    *out = Set{{}, 0, 0, r, c};
    int found[TOGETHER], m = 0;
    for (int k = i; k < n && m < limit; ++k)
        if (lo(k) == r && hi(k) == c) found[m++] = k;
    for (int tall = 0; tall < 2; ++tall)               // those with rows <= cols first
        for (int k = 0; k < m; ++k)
            if ((rows[found[k]] > cols[found[k]]) == (tall == 1)) out->index[out->n++] = found[k], out->wides += !tall;
    return true;
}

extern "C" size_t dpd_muon_workspace_bytes(int n, const int64_t *h_rows, const int64_t *h_cols, int accurate) {
    size_t most = 256;
    if (!h_rows || !h_cols) return most;
    for (int i = 0; i < n; ++i) {
        Set s;
        if (!leads_set(i, n, h_rows, h_cols, accurate, &s)) continue;
        const size_t b = (size_t)Plan(s.n, s.r, s.c, accurate != 0).total + 256;
        most = b > most ? b : most;
    }
    return most;
}

extern "C" int dpd_muon_step(int n, void *const *h_p, const void *const *h_g, float *const *h_m, const int64_t *h_rows, const int64_t *h_cols, int p_type,
                             double lr, double momentum, int nesterov, double weight_decay, int steps, const float *h_coef, double eps, int accurate, void *ws,
                             size_t ws_bytes, void *stream) {
    DPD_REQUIRE(n >= 0 && (n == 0 || (h_p && h_g && h_m && h_rows && h_cols)), DPD_ERR_INVALID_ARG, "muon_step: null pointer");
    DPD_REQUIRE(p_type == DPD_F32 || p_type == DPD_BF16 || p_type == DPD_F16, DPD_ERR_INVALID_ARG, "muon_step: element type %d", p_type);
    if (const int rc = check_iteration("muon_step", steps, h_coef, eps)) return rc;
    bool any_large = false;
    for (int i = 0; i < n; ++i) {                  // every matrix is looked at before the first one changes
        if (const int rc = check_matrix("muon_step", h_rows[i], h_cols[i])) return rc;
        const bool empty = h_rows[i] == 0 || h_cols[i] == 0;
        DPD_REQUIRE(empty || (h_p[i] && h_g[i] && h_m[i]), DPD_ERR_INVALID_ARG, "muon_step: null pointer (matrix %d)", i);
        any_large = any_large || (!empty && !is_small(h_rows[i], h_cols[i]) && !fits(h_rows[i], h_cols[i], accurate != 0));
    }
    DPD_REQUIRE(!any_large || (ws && ws_bytes >= dpd_muon_workspace_bytes(n, h_rows, h_cols, accurate)), DPD_ERR_WORKSPACE, "muon_step: workspace");
    char *w = (char *)(((uintptr_t)ws + 255) & ~(uintptr_t)255);
    hipStream_t st = as_stream(stream);
    Coef coef{};
    for (int i = 0; i < 3 * steps; ++i) coef.v[i] = h_coef[i];
    const float keep = (float)(1.0 - lr * weight_decay), mu = (float)momentum;
    return with_type(p_type, [&](auto t) {
        using T = decltype(t);
        SmallTable tabs[2]{};                      // small ones, and those that fit into a compute unit
        int used[2] = {0, 0};
        auto flush = [&](int kind) {
            const int many = used[kind];
            used[kind] = 0;
            if (!many) return DPD_OK;
            if (kind == 0) hipLaunchKernelGGL((k_small_muon<T>), dim3(many), dim3(1024), 0, st, tabs[0], mu, nesterov, keep, coef, steps, eps);
            else if (accurate) hipLaunchKernelGGL((k_fit_muon<true, T>), dim3(many), dim3(64 * FIT_WAVES), 0, st, tabs[1], mu, nesterov, keep, coef, steps, eps);
            else hipLaunchKernelGGL((k_fit_muon<false, T>), dim3(many), dim3(64 * FIT_WAVES), 0, st, tabs[1], mu, nesterov, keep, coef, steps, eps);
            DPD_LAUNCH_CHECK();
            return DPD_OK;
        };
        for (int i = 0; i < n; ++i) {
            const int64_t rows = h_rows[i], cols = h_cols[i];
            if (rows == 0 || cols == 0) continue;
            auto factor_of = [&](int k) { return (float)(lr * sqrt(h_rows[k] > h_cols[k] ? (double)h_rows[k] / (double)h_cols[k] : 1.0)); };
            const float factor = factor_of(i);
            const int kind = is_small(rows, cols) ? 0 : fits(rows, cols, accurate != 0) ? 1 : 2;
            if (kind == 2) {
                Set s;
                if (!leads_set(i, n, h_rows, h_cols, accurate, &s)) continue;          // went with an earlier one
                FromMomenta<T> from{{}, {}, mu, nesterov, 0, 0};
                ToManyWeights<T> to[2] = {{{}, keep, 0.f, 0}, {{}, keep, 0.f, 0}};
                for (int k = 0; k < s.n; ++k) {
                    const int j = s.index[k], tall = k >= s.wides, at = tall ? k - s.wides : k;
                    from.g[k] = (const T *)h_g[j], from.m[k] = h_m[j];
                    from.whole_bits |= (unsigned)((((uintptr_t)h_g[j] | (uintptr_t)h_m[j]) & 15) == 0 && h_cols[j] % 8 == 0) << k;
                    from.wide_bits |= (unsigned)!tall << k;
                    to[tall].p[at] = (T *)h_p[j], to[tall].factor = factor_of(j);
                    to[tall].whole_bits |= (unsigned)(((uintptr_t)h_p[j] & 15) == 0 && h_cols[j] % 8 == 0) << at;
                }
                const int rc = accurate ? large<true>(from, to[0], to[1], s.n, s.wides, s.r, s.c, steps, coef.v, eps, w, st)
                                        : large<false>(from, to[0], to[1], s.n, s.wides, s.r, s.c, steps, coef.v, eps, w, st);
                if (rc) return rc;
                continue;
            }
            SmallTable &tab = tabs[kind];
            const int at = used[kind]++;
            tab.p[at] = h_p[i], tab.g[at] = h_g[i], tab.m[at] = h_m[i], tab.rows[at] = (int)rows, tab.cols[at] = (int)cols, tab.factor[at] = factor;
            if (at + 1 == TABLE)
                if (const int rc = flush(kind)) return rc;
        }
        const int rc = flush(0);
        return rc ? rc : flush(1);
    });
}
