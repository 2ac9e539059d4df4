// The 8-bit linear layer: rows quantised with one scale each, the int8 product of two sets of such rows, and the
// straight-through gradients.
//
//   quantiser   s = fl32(max(max|x|, 2^-100) fl32(1 / 127)),  q = round-half-even(x / s) of the exact quotient
//   product     y[m, n] = ((sum_k qa[m, k] qb[n, k]) * sa[m]) * sb[n] + bias[n]     (the sum exactly, in int32)
//   gradients   gx = g (qw sw),  gw = g^T (qx sx),  gb = column sums of g
#include <type_traits>
#include "gemm_nt.h"

int g_product_tile = -1;

namespace {

constexpr float SCALE_FLOOR = 0x1p-100f;      // rows below it share its scale: a row of zeros has a finite one
constexpr int64_t MAX_K = 131071;             // 128^2 * 131071 < 2^31: the int32 sum cannot overflow

DEV unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }   // ordered like |v|, NaN above infinity

DEV unsigned wave_umax(unsigned v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, o));
    return v;
}

// The scale of a row from the largest |x| (as bits); NaN if the row holds a NaN or an infinity.
DEV float row_scale(unsigned top) {
    return top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : fmaxf(__uint_as_float(top), SCALE_FLOOR) * (1.0f / 127.0f);
}

// round-half-even(x / s) of the exact quotient.  x * inv is off by less than 2^-15, so rint gives the integer or its
// neighbour across the half-way point b; the sign of x - b s (one rounding, exact in sign) says which, and zero is a tie.
DEV int quantise(float x, float s, float inv) {
    const float n = rintf(x * inv), d = x * inv - n;
    if (fabsf(d) < 0.4998f) return (int)n;
    const float b = n + copysignf(0.5f, d);
    const float t = __builtin_fmaf(-b, s, x);
    const float r = t > 0.f ? b + 0.5f : (t < 0.f ? b - 0.5f : rintf(b));
    return (int)fminf(fmaxf(r, -127.f), 127.f);
}

// A row in the hands of TEAM threads, VEC elements a piece: a thread keeps its first HELD pieces in registers between the
// search for the largest value and the quantisation, and reads the others again.
template <class T, int TEAM, int VEC, int HELD>
struct HeldRow {
    typedef T TV __attribute__((ext_vector_type(VEC)));
    typedef int8_t QV __attribute__((ext_vector_type(VEC)));
    TV held[HELD];
    DEV void load(const T *x, int pieces, int t) {
#pragma unroll
        for (int h = 0; h < HELD; ++h) held[h] = ((const TV *)x)[min(t + h * TEAM, pieces - 1)];       // behind the row its last piece again
    }
    DEV unsigned top(const T *x, int pieces, int t) const {            // of this thread's pieces
        unsigned top = 0;
#pragma unroll
        for (int h = 0; h < HELD; ++h)
#pragma unroll
            for (int e = 0; e < VEC; ++e) top = max(top, abs_bits(to_f32(held[h][e])));
        for (int i = t + HELD * TEAM; i < pieces; i += TEAM) {
            const TV v = ((const TV *)x)[i];
#pragma unroll
            for (int e = 0; e < VEC; ++e) top = max(top, abs_bits(to_f32(v[e])));
        }
        return top;
    }
    DEV float put(const T *x, int pieces, int t, unsigned top, int8_t *q, int all) const {     // `all` pieces with the zeros behind the row
        const float s = row_scale(top), inv = 1.0f / s;
        const bool fine = top < 0x7f800000u;
        auto one = [&](int i, TV v) {
            QV o;
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] = fine ? (int8_t)quantise(to_f32(v[e]), s, inv) : (int8_t)0;
            ((QV *)q)[i] = o;
        };
#pragma unroll
        for (int h = 0; h < HELD; ++h)
            if (t + h * TEAM < all) one(t + h * TEAM, t + h * TEAM < pieces ? held[h] : TV{});
        for (int i = t + HELD * TEAM; i < all; i += TEAM) one(i, i < pieces ? ((const TV *)x)[i] : TV{});
        return s;
    }
};

// One row per TEAM threads (a wave, or the whole workgroup): 16 bytes a piece where the rows allow it, single elements where
// not; the rows of two matrices where both factors of a layer are quantised.  Bound by memory: 2 + 1 bytes an element (bf16);
// 8192 x 8192 bf16 takes 44 us (4.6 TB/s).
template <class T>
struct Rows {
    const T *x;
    int64_t rows, ldx;
    int8_t *q;
    int64_t ldq;
    float *scale;
};

template <class T, int TEAM, int VEC>
__global__ __launch_bounds__(256) void k_quantize_rows(Rows<T> a, Rows<T> b, int cols) {
    __shared__ unsigned top4[4];
    const int t = threadIdx.x % TEAM;
    int64_t row = (int64_t)blockIdx.x * (256 / TEAM) + threadIdx.x / TEAM;
    if (TEAM == 64 && row >= a.rows + b.rows) return;
    const bool second = row >= a.rows;
    if (second) row -= a.rows;
    const Rows<T> &m = second ? b : a;
    const T *xr = m.x + row * m.ldx;
    const int pieces = cols / VEC;
    HeldRow<T, TEAM, VEC, VEC == 1 ? 8 : 4> r;
    r.load(xr, pieces, t);
    unsigned top = wave_umax(r.top(xr, pieces, t));
    if (TEAM == 256) {
        if ((threadIdx.x & 63) == 0) top4[threadIdx.x >> 6] = top;
        __syncthreads();
        top = max(max(top4[0], top4[1]), max(top4[2], top4[3]));
    }
    const float s = r.put(xr, pieces, t, top, m.q + row * m.ldq, (int)(m.ldq / VEC));
    if (t == 0) m.scale[row] = s;
}

template <class T>
bool in_pieces(const Rows<T> &m, int cols) {
    constexpr int V = 16 / sizeof(T);
    return ((uintptr_t)m.x & 15) == 0 && m.ldx % V == 0 && cols % V == 0 && ((uintptr_t)m.q & 15) == 0 && m.ldq % V == 0;
}

template <class T>
int quantize_rows(const Rows<T> &a, const Rows<T> &b, int cols, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    constexpr int64_t MOST = 1 << 22;                  // rows a launch: a grid has fewer than 2^32 threads
    auto go = [&](auto kernel, int rows_per_block) {
        for (Rows<T> c = a, d = b; c.rows + d.rows > 0;) {
            Rows<T> now = c, then = d;
            now.rows = c.rows < MOST ? c.rows : MOST;
            then.rows = d.rows < MOST - now.rows ? d.rows : MOST - now.rows;
            hipLaunchKernelGGL(kernel, dim3((unsigned)((now.rows + then.rows + rows_per_block - 1) / rows_per_block)), dim3(256), 0, st, now, then, cols);
            DPD_LAUNCH_CHECK();
            c = Rows<T>{c.x + now.rows * c.ldx, c.rows - now.rows, c.ldx, c.q + now.rows * c.ldq, c.ldq, c.scale + now.rows};
            d = Rows<T>{d.x + then.rows * d.ldx, d.rows - then.rows, d.ldx, d.q + then.rows * d.ldq, d.ldq, d.scale + then.rows};
        }
        return DPD_OK;
    };
    if (in_pieces(a, cols) && (b.rows == 0 || in_pieces(b, cols))) return cols <= 1024 ? go(k_quantize_rows<T, 64, V>, 4) : go(k_quantize_rows<T, 256, V>, 1);
    return cols <= 1024 ? go(k_quantize_rows<T, 64, 1>, 4) : go(k_quantize_rows<T, 256, 1>, 1);
}
template <class T>
int quantize_rows(const T *x, int64_t rows, int cols, int64_t ldx, int8_t *q, int64_t ldq, float *scale, hipStream_t st) {
    return quantize_rows(Rows<T>{x, rows, ldx, q, ldq, scale}, Rows<T>{}, cols, st);
}

template <class T>
struct ScaleOut {
    const float *sa, *sb;
    const void *bias;
    int bias_type;
    T *out;
    int64_t ldo;
    int N;
    bool whole;
    static constexpr bool TURNED = false;
    typedef float Row;
    typedef None Pre;
    DEV Pre pre(int, int, int) const { return {}; }
    struct Col {
        float s[8], b[8];
    };
    DEV Row row(int, int m) const { return sa[m]; }
    DEV Col col(int, int n) const {
        Col c;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int k = min(n + i, N - 1);
            c.s[i] = sb[k];
            c.b[i] = bias ? load_any(bias, bias_type, k) : 0.f;
        }
        return c;
    }
    DEV void put(int, int m, int n, float *v, const Row &r, const Col &c, Pre) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] * r * c.s[i] + c.b[i];
        store8(out + (int64_t)m * ldo + n, v, N - n, whole);
    }
};

template <class T>
struct PlainOut {
    T *out;
    int64_t ldo;
    int N;
    bool whole;
    static constexpr bool TURNED = false;
    typedef None Row, Col, Pre;
    DEV Pre pre(int, int, int) const { return {}; }
    DEV Row row(int, int) const { return {}; }
    DEV Col col(int, int) const { return {}; }
    DEV void put(int, int m, int n, float *v, Row, Col, Pre) const { store8(out + (int64_t)m * ldo + n, v, N - n, whole); }
};

// Few tokens (at most 16): a workgroup owns 16 output channels, quantises the tokens for itself, VEC elements a piece,
// while its first weights are on their way, and reads those weights once, straight into the fragments of the matrix
// instruction (64 bytes of 16 rows a load; the waves take the 64-byte steps of the rows in turn and are joined in LDS: integer
// sums, so the order does not matter).  A token row beyond the last one repeats it.  One launch, bound by the read of the
// weights and by latency: 1 token of 4096 x 4096 bf16 7.9 us (2.1 TB/s), of 16384 x 4096 17.0 us (3.9 TB/s).
constexpr int FEW_HELD = 8;                             // pieces of the tokens that a thread quantises

template <class T, int WAVES, int VEC>
__global__ __launch_bounds__(64 * WAVES) void k_few_tokens(const T *__restrict__ x, int64_t ldx, int cols, int64_t ld, int M, const int8_t *__restrict__ qw,
                                                           ScaleOut<T> epi) {
    constexpr int U = 8;                                // steps of a wave in flight
    typedef T TV __attribute__((ext_vector_type(VEC)));
    typedef int8_t QV __attribute__((ext_vector_type(VEC)));
    extern __shared__ __attribute__((aligned(16))) char few_lds[];
    nt::i32x4 *part = (nt::i32x4 *)few_lds;             // [WAVES][64]
    unsigned *tops = (unsigned *)(few_lds + WAVES * 1024);              // [16]
    int8_t *mine = (int8_t *)(tops + 16);                               // [M][ld]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * 16, steps = (int)(ld / 64);
    const int8_t *wr = qw + (int64_t)min(n0 + r, epi.N - 1) * ld + q * 16;
    nt::i32x4 w[U];
    auto fetch = [&](int i) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = (i + u) * WAVES + wave;
            w[u] = s < steps ? *(const nt::i32x4 *)(wr + (int64_t)s * 64) : nt::i32x4{0, 0, 0, 0};
        }
    };
    fetch(0);
    const int pieces = cols / VEC, total = M * pieces;
    if (threadIdx.x < 16) tops[threadIdx.x] = 0;
    for (int i = threadIdx.x; i < M * (int)(ld - cols); i += 64 * WAVES) {          // zeros behind the rows
        const int m = i / (int)(ld - cols);
        mine[m * ld + cols + i - m * (int)(ld - cols)] = 0;
    }
    TV v[FEW_HELD];
    int row[FEW_HELD];
#pragma unroll
    for (int h = 0; h < FEW_HELD; ++h) {
        const int e = min((int)threadIdx.x + h * 64 * WAVES, total - 1);            // behind the last piece: again, harmless
        row[h] = e / pieces;
        v[h] = *(const TV *)(x + row[h] * ldx + (int64_t)(e - row[h] * pieces) * VEC);
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < FEW_HELD; ++h) {
        if (h * 64 * WAVES >= total) break;
        unsigned top = 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) top = max(top, abs_bits(to_f32(v[h][e])));
        const int first = __builtin_amdgcn_readfirstlane(row[h]);
        if (__all(row[h] == first)) {
            top = wave_umax(top);
            if (lane == 0) atomicMax(tops + first, top);
        } else {
            atomicMax(tops + row[h], top);
        }
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < FEW_HELD; ++h) {
        const int e = (int)threadIdx.x + h * 64 * WAVES;
        if (e >= total) break;
        const unsigned top = tops[row[h]];
        const float s = row_scale(top), inv = 1.0f / s;
        QV o;
#pragma unroll
        for (int k = 0; k < VEC; ++k) o[k] = top < 0x7f800000u ? (int8_t)quantise(to_f32(v[h][k]), s, inv) : (int8_t)0;
        *(QV *)(mine + row[h] * ld + (e - row[h] * pieces) * VEC) = o;
    }
    __syncthreads();
    const int8_t *tok = mine + min(r, M - 1) * ld + q * 16;
    nt::i32x4 acc = {0, 0, 0, 0};
    for (int i = 0; i * WAVES < steps; i += U) {
        nt::i32x4 now[U];
#pragma unroll
        for (int u = 0; u < U; ++u) now[u] = w[u];
        if ((i + U) * WAVES < steps) fetch(i + U);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = min((i + u) * WAVES + wave, steps - 1);                   // behind the last step the weights are zeros
            acc = nt::mfma<nt::I8>(now[u], *(const nt::i32x4 *)(tok + (int64_t)s * 64), acc);
        }
    }
    part[wave * 64 + lane] = acc;
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int k = 1; k < WAVES; ++k) acc += part[k * 64 + lane];
    const int n = n0 + q * 4;
    if (r >= M || n >= epi.N) return;
    const float s = row_scale(tops[r]);
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (n + e < epi.N) {
            float y = (float)acc[e] * s * epi.sb[n + e];
            if (epi.bias) y += load_any(epi.bias, epi.bias_type, n + e);
            epi.out[(int64_t)r * epi.ldo + n + e] = from_f32<T>(y);
        }
}

// Whether the tokens go through k_few_tokens, with how many waves and in what pieces.  Measured with 2 and more tokens, us,
// one launch against the quantiser and a tiled product: 4096 x 4096, 2 tokens 8.2 against 9.6 and 4 tokens 9.7 against 9.7
// (16 waves; 4 waves 10.4 and 13.6); 16384 x 4096, 2 tokens 16.7 against 17.5 and 4 tokens 21.3 against 16.9; 1024 x 8192,
// 1 token 8.8 (16 waves) against 11.1.  4 waves are better for short rows: 2048 x 2048, 1 token 4.5 against 6.1 with 16.
struct FewPlan {
    int waves, vec;                                     // 0: no
};
template <class T>
FewPlan few_plan(const T *x, int64_t M, int64_t N, int64_t K, int64_t ldx, int64_t ld) {
    constexpr int V = 16 / sizeof(T);
    const int waves = ld >= 4096 && N <= 8192 ? 16 : 4;
    if (M > 16 || M * ld > (waves == 16 ? 8192 : 4096)) return {0, 0};
    if ((N + 15) / 16 * 64 * waves > UINT32_MAX) return {0, 0};                // a grid has fewer than 2^32 threads
    const int vec = ((uintptr_t)x & 15) == 0 && ldx % V == 0 && K % V == 0 ? V : 1;
    return M * (K / vec) <= (int64_t)FEW_HELD * 64 * waves ? FewPlan{waves, vec} : FewPlan{0, 0};
}

template <class T, int WAVES, int VEC>
int few_tokens(const T *x, int64_t M, int64_t K, int64_t ldx, int64_t ld, const int8_t *qw, const ScaleOut<T> &epi, hipStream_t st) {
    hipLaunchKernelGGL((k_few_tokens<T, WAVES, VEC>), dim3((unsigned)((epi.N + 15) / 16)), dim3(64 * WAVES), (size_t)(WAVES * 1024 + 64 + M * ld), st, x, ldx,
                       (int)K, ld, (int)M, qw, epi);
    DPD_LAUNCH_CHECK();
    return DPD_OK;
}

// More tokens, up to MB blocks of 16: as above, but a wave quantises whole rows (the next one is on its way meanwhile), and each
// weight fragment meets MB blocks of 16 tokens.  Rows of LDS are 16 bytes longer than the image's, so that 16 of them spread
// over the banks; the waves' sums take their place at the end.  Bound by latency: 8 tokens of 1024 x 1024 bf16 5.4 us.
constexpr int SOME_BYTES = 32 * 1024;                   // quantised tokens

template <class T, int VEC, int MB>
__global__ __launch_bounds__(1024) void k_some_tokens(const T *__restrict__ x, int64_t ldx, int cols, int ld, int M, const int8_t *__restrict__ qw,
                                                      ScaleOut<T> epi) {
    constexpr int WAVES = 16, U = 4;
    __shared__ __attribute__((aligned(16))) char lds[SOME_BYTES + 16 * 16 * MB];
    __shared__ float scale[16 * MB];
    nt::i32x4 *part = (nt::i32x4 *)lds;                 // [WAVES][MB][64], once the tokens [M][ld + 16] have been read
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * 16, steps = ld / 64, pitch = ld + 16;
    const int8_t *wr = qw + (int64_t)min(n0 + r, epi.N - 1) * ld + q * 16;
    nt::i32x4 w[U];
    auto fetch = [&](int i) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = (i + u) * WAVES + wave;
            w[u] = s < steps ? *(const nt::i32x4 *)(wr + (int64_t)s * 64) : nt::i32x4{0, 0, 0, 0};
        }
    };
    fetch(0);
    const int pieces = cols / VEC;
    HeldRow<T, 64, VEC, VEC == 1 ? 16 : 4> row, next;
    if (wave < M) next.load(x + (int64_t)wave * ldx, pieces, lane);
    for (int m = wave; m < M; m += WAVES) {
        const T *xr = x + (int64_t)m * ldx;
        row = next;
        if (m + WAVES < M) next.load(xr + WAVES * ldx, pieces, lane);
        const unsigned top = wave_umax(row.top(xr, pieces, lane));
        const float s = row.put(xr, pieces, lane, top, (int8_t *)lds + m * pitch, ld / VEC);
        if (lane == 0) scale[m] = s;
    }
    __syncthreads();
    nt::i32x4 acc[MB] = {};
    const int8_t *tok[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) tok[b] = (const int8_t *)lds + min(b * 16 + r, M - 1) * pitch + q * 16;
    for (int i = 0; i * WAVES < steps; i += U) {
        nt::i32x4 now[U];
#pragma unroll
        for (int u = 0; u < U; ++u) now[u] = w[u];
        if ((i + U) * WAVES < steps) fetch(i + U);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = min((i + u) * WAVES + wave, steps - 1);                   // behind the last step the weights are zeros
#pragma unroll
            for (int b = 0; b < MB; ++b) acc[b] = nt::mfma<nt::I8>(now[u], *(const nt::i32x4 *)(tok[b] + s * 64), acc[b]);
        }
    }
    __syncthreads();
#pragma unroll
    for (int b = 0; b < MB; ++b) part[(wave * MB + b) * 64 + lane] = acc[b];
    __syncthreads();
    if (wave >= MB) return;
    nt::i32x4 sum = part[wave * 64 + lane];
#pragma unroll
    for (int k = 1; k < WAVES; ++k) sum += part[(k * MB + wave) * 64 + lane];
    const int m = wave * 16 + r, n = n0 + q * 4;
    if (m >= M) return;
    const float s = scale[m];
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (n + e < epi.N) {
            float y = (float)sum[e] * s * epi.sb[n + e];
            if (epi.bias) y += load_any(epi.bias, epi.bias_type, n + e);
            epi.out[(int64_t)m * epi.ldo + n + e] = from_f32<T>(y);
        }
}

template <class T, int VEC>
int some_tokens(const T *x, int64_t M, int64_t K, int64_t ldx, int64_t ld, const int8_t *qw, const ScaleOut<T> &epi, hipStream_t st) {
    const dim3 grid((unsigned)((epi.N + 15) / 16));
    if (M <= 16) hipLaunchKernelGGL((k_some_tokens<T, VEC, 1>), grid, dim3(1024), 0, st, x, ldx, (int)K, (int)ld, (int)M, qw, epi);
    else hipLaunchKernelGGL((k_some_tokens<T, VEC, 2>), grid, dim3(1024), 0, st, x, ldx, (int)K, (int)ld, (int)M, qw, epi);
    DPD_LAUNCH_CHECK();
    return DPD_OK;
}

// Whether the tokens go through k_some_tokens.  On the device, one launch against the quantiser and a tiled product, bf16, us:
// 1024 x 1024 with 4, 8, 16, 17, 32 tokens 5.2, 5.4, 6.1, 7.0, 8.7 against 6.9, 7.3, 7.3, 7.6, 7.8; 4096 x 2048 with 16 tokens
// 8.4 against 7.6.  On the host the second launch and its workspace cost 4 us, which is more than any of these loses.  Not
// for 64 tokens (1024 x 1024: 13.9 against 7.9), longer rows (2048 x 4096, 8 tokens: 10 against 8.9) or more than one
// round of workgroups (16384 x 1024, 8 tokens: 14 against 8.0).  One and two tokens are faster in k_few_tokens (1024 x 1024,
// 2 tokens: 4.7 against 5.1), where it takes them.
bool takes_some(int64_t M, int64_t N, int64_t ld) { return M <= 32 && N <= 4096 && ld <= 2048 && M * ld <= SOME_BYTES; }

// rows of an int8 matrix at a stride that the product can read (a multiple of 128 bytes, zeros behind the row)
__global__ __launch_bounds__(256) void k_pad_rows(const int8_t *__restrict__ q, int64_t rows, int cols, int64_t ld,
                                                  int8_t *__restrict__ out, int64_t ldo) {
    const int64_t total = rows * ldo;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / ldo;
        const int c = (int)(i - r * ldo);
        out[i] = c < cols ? q[r * ld + c] : (int8_t)0;
    }
}

bool readable(const int8_t *q, int64_t ld, int64_t K) { return ((uintptr_t)q & 15) == 0 && ld % 16 == 0 && K % 16 == 0; }

template <class T>
bool whole8(const T *p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0; }

template <class T>
int int8_product(const int8_t *a, int64_t lda, const float *sa, const int8_t *b, int64_t ldb, const float *sb, const void *bias,
                 int bias_type, int64_t M, int64_t N, int64_t K, T *out, int64_t ldo, hipStream_t st) {
    nt::Args g{};
    g.a = (const char *)a, g.b = (const char *)b, g.lda = lda, g.ldb = ldb, g.M = (int)M, g.N = (int)N;
    g.steps = g.wrap = (int)((K + 127) / 128);
    g.tail = (int)(K - (int64_t)(g.steps - 1) * 128);
    return nt::product<nt::I8>(g, 1, ScaleOut<T>{sa, sb, bias, bias_type, out, ldo, (int)N, whole8(out, ldo)}, st);
}

// ---- gradients ---------------------------------------------------------------------------
// bf16 planes of a gradient times a scale: 2 for bf16 and fp16 gradients (2^-16, so that the rounding of the result is
// the only one that shows), 3 for fp32 (the whole value): the planes of a row lie one behind the other along k, the smallest
// first.  One plane for bf16 would halve the two products (4096 tokens of 4096 x 4096: 364 instead of 517 to 574 us for the
// training pass), but every term would be rounded by 2^-8 and the gradients be 2.3e-3 off in place of 1.7e-3.
template <class T>
constexpr int planes_of() { return std::is_same<T, float>::value ? 3 : 2; }

template <int P>
DEV void put_planes8(__bf16 *p, int64_t plane, const float *v) {
    typedef __bf16 b8 __attribute__((ext_vector_type(8)));
    float rest[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) rest[e] = v[e];
#pragma unroll
    for (int i = P - 1; i >= 0; --i) {
        b8 o;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            o[e] = (__bf16)rest[e];
            rest[e] = fabsf((float)o[e]) < INFINITY ? rest[e] - (float)o[e] : 0.f;      // an infinity stays one: nothing is left of it
        }
        *(b8 *)(p + i * plane) = o;
    }
}

// One 64 x 64 tile of g [M, N]: gs[m, n] = g sw[n] (row-major, for gx), gt[n, m] = g sx[m] (transposed, for gw), each as
// bf16 planes with zeros behind the rows, and this tile's column sums for gb.  Pieces of 8 elements on every access; bound
// by memory (2 + 8 bytes an element in bf16).
template <class T>
DEV void grad_images(int bx, int by, float (*t)[65], const T *__restrict__ g, int64_t M, int N, int64_t ldg, bool whole, const float *__restrict__ sw,
                     const float *__restrict__ sx, __bf16 *__restrict__ gs, int64_t n_pad, __bf16 *__restrict__ gt, int64_t m_pad,
                     float *__restrict__ gb_part) {
    constexpr int P = planes_of<T>();
    const int64_t m0 = (int64_t)bx * 64;
    const int n0 = by * 64;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int e = threadIdx.x + h * 256, i = e >> 3, j = (e & 7) * 8;
        float v[8] = {};
        if (m0 + i < M && n0 + j < N) load8(g + (m0 + i) * ldg + n0 + j, v, N - n0 - j, whole);
#pragma unroll
        for (int k = 0; k < 8; ++k) t[i][j + k] = v[k];
        if (gs && m0 + i < M) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = n0 + j + k < N ? v[k] * sw[n0 + j + k] : 0.f;
            put_planes8<P>(gs + (m0 + i) * (P * n_pad) + n0 + j, n_pad, v);
        }
    }
    __syncthreads();
    if (gt) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int e = threadIdx.x + h * 256, j = e >> 3, i = (e & 7) * 8;
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = m0 + i + k < M ? t[i + k][j] * sx[m0 + i + k] : 0.f;
            if (n0 + j < N) put_planes8<P>(gt + (int64_t)(n0 + j) * (P * m_pad) + m0 + i, m_pad, v);
        }
    }
    if (gb_part && threadIdx.x < 64 && n0 + threadIdx.x < N) {
        float s = 0.f;
        for (int i = 0; i < 64; ++i) s += t[i][threadIdx.x];
        gb_part[(int64_t)bx * N + n0 + threadIdx.x] = s;
    }
}

// Sums the tiles' column sums in fp64: 32 columns a workgroup, 8 threads a column.  Latency: 4096 x 4096 5 us.
template <class T>
__global__ __launch_bounds__(256) void k_bias_grad(const float *__restrict__ part, int64_t blocks, int N, T *__restrict__ gb) {
    __shared__ double red[8][32];
    const int c = threadIdx.x & 31, k = threadIdx.x >> 5, n = blockIdx.x * 32 + c;
    double s = 0.0;
    if (n < N)
#pragma unroll 4
        for (int64_t b = k; b < blocks; b += 8) s += (double)part[b * N + n];
    red[k][c] = s;
    __syncthreads();
    if (k == 0 && n < N) {
        for (int i = 1; i < 8; ++i) s += red[i][c];
        gb[n] = from_f32<T>((float)s);
    }
}

// q [rows, cols] int8 -> out [cols, rows_pad] bf16, zeros behind the rows: the integers themselves, which are exact.  A wave
// takes 64 x 64, a thread 4 rows of 16 columns, whose bytes it turns in registers; the words meet in LDS (4 rows of a column a word) and leave as 16 bytes of 8 rows.  Bound by memory.
struct Turn {
    const int8_t *q;
    int64_t rows, ld;
    int cols;
    bool whole;
    __bf16 *out;
    int64_t rows_pad;
    int bx, by;                                       // workgroups along the rows and the columns; none: 0
};

DEV void transpose_i8(int bx, int by, unsigned (*t)[66], const Turn &a) {
    const int8_t *__restrict__ q = a.q;
    const int64_t rows = a.rows, ld = a.ld, rows_pad = a.rows_pad;
    const int cols = a.cols;
    const bool whole = a.whole;
    __bf16 *__restrict__ out = a.out;
    typedef __bf16 b8 __attribute__((ext_vector_type(8)));
    typedef unsigned u4 __attribute__((ext_vector_type(4)));
    const int64_t r0 = (int64_t)bx * 256;             // t: [column][4 rows], 256 rows
    const int c0 = by * 64;
    {
        const int i = (threadIdx.x >> 2) * 4, j = (threadIdx.x & 3) * 16;
        u4 v[4];
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            v[a] = u4{0, 0, 0, 0};
            if (r0 + i + a < rows && c0 + j < cols) {
                const int8_t *p = q + (r0 + i + a) * ld + c0 + j;
                if (whole && (c0 + j + 16 <= cols || r0 + i + a + 1 < rows)) {      // the row's memory goes on to a multiple of 16
                    v[a] = *(const u4 *)p;
                } else {
                    for (int k = 0; k < 16 && c0 + j + k < cols; ++k) v[a][k >> 2] |= (unsigned)(uint8_t)p[k] << (8 * (k & 3));
                }
            }
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {                 // 4 rows x 4 columns of bytes
            const unsigned lo01 = __builtin_amdgcn_perm(v[1][w], v[0][w], 0x05010400), hi01 = __builtin_amdgcn_perm(v[1][w], v[0][w], 0x07030602);
            const unsigned lo23 = __builtin_amdgcn_perm(v[3][w], v[2][w], 0x05010400), hi23 = __builtin_amdgcn_perm(v[3][w], v[2][w], 0x07030602);
            t[j + w * 4 + 0][i >> 2] = __builtin_amdgcn_perm(lo23, lo01, 0x05040100);
            t[j + w * 4 + 1][i >> 2] = __builtin_amdgcn_perm(lo23, lo01, 0x07060302);
            t[j + w * 4 + 2][i >> 2] = __builtin_amdgcn_perm(hi23, hi01, 0x05040100);
            t[j + w * 4 + 3][i >> 2] = __builtin_amdgcn_perm(hi23, hi01, 0x07060302);
        }
    }
    const int i = (threadIdx.x & 31) * 8;             // this thread's rows
    __syncthreads();
    if (r0 + i >= rows_pad) return;
#pragma unroll
    for (int h = 0; h < 8; ++h) {
        const int j = (threadIdx.x >> 5) + h * 8;
        if (c0 + j >= cols) return;
        b8 o;
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = (__bf16)(float)(int8_t)(t[j][(i + k) >> 2] >> (8 * (k & 3)));
        *(b8 *)(out + (int64_t)(c0 + j) * rows_pad + r0 + i) = o;
    }
}

// Everything that the two products of the backward read, in one launch: the images of g, and both 8-bit factors turned.  Bound
// by memory: 4096 tokens of 4096 x 4096 bf16 move 269 MB in 63 to 78 us (3.5 to 4.3 TB/s).
template <class T>
__global__ __launch_bounds__(256) void k_backward_images(const T *__restrict__ g, int64_t M, int N, int64_t ldg, bool whole, const float *__restrict__ sw,
                                                         const float *__restrict__ sx, __bf16 *__restrict__ gs, int64_t n_pad, __bf16 *__restrict__ gt,
                                                         int64_t m_pad, float *__restrict__ gb_part, int gx, int gy, Turn w, Turn x) {
    __shared__ union {
        float f[64][65];
        unsigned u[64][66];
    } lds;
    int id = blockIdx.x;
    if (id < gx * gy) {
        grad_images(id % gx, id / gx, lds.f, g, M, N, ldg, whole, sw, sx, gs, n_pad, gt, m_pad, gb_part);
        return;
    }
    id -= gx * gy;
    if (id < w.bx * w.by) {
        transpose_i8(id % w.bx, id / w.bx, lds.u, w);
        return;
    }
    id -= w.bx * w.by;
    transpose_i8(id % x.bx, id / x.bx, lds.u, x);
}

int planes_for(int type) { return type == DPD_F32 ? 3 : 2; }

struct BackwardPlan {
    int64_t m_pad, n_pad, gs, gt, wt, xt, part, total;      // element counts and byte offsets into the workspace
    BackwardPlan(int64_t M, int64_t N, int64_t K, int p, bool gx, bool gw, bool gb) {
        m_pad = nt::pad_to(M, 64), n_pad = nt::pad_to(N, 64);
        int64_t at = 0;
        auto take = [&](bool want, int64_t bytes) {
            const int64_t here = at;
            if (want) at += nt::pad_to(bytes, 256);
            return here;
        };
        gs = take(gx, M * p * n_pad * 2);
        wt = take(gx, K * n_pad * 2);
        gt = take(gw, N * p * m_pad * 2);
        xt = take(gw, K * m_pad * 2);
        part = take(gb, m_pad / 64 * N * 4);
        total = at;
    }
};

bool whole16(const int8_t *q, int64_t ld, int64_t cols) { return ((uintptr_t)q & 15) == 0 && ld % 16 == 0 && ld >= nt::pad_to(cols, 16); }

template <class T>
int gradients(const T *g, int64_t ldg, int64_t M, int64_t N, int64_t K, const int8_t *qx, int64_t ldqx, const float *sx,
              const int8_t *qw, int64_t ldqw, const float *sw, T *gx, void *gw, int gw_type, void *gb, int gb_type, char *ws, hipStream_t st) {
    constexpr int P = planes_of<T>();
    const BackwardPlan p(M, N, K, P, gx, gw, gb);
    __bf16 *gs = gx ? (__bf16 *)(ws + p.gs) : nullptr, *wt = (__bf16 *)(ws + p.wt), *gt = gw ? (__bf16 *)(ws + p.gt) : nullptr,
           *xt = (__bf16 *)(ws + p.xt);
    float *part = gb ? (float *)(ws + p.part) : nullptr;
    auto turn = [&](bool want, const int8_t *q, int64_t rows, int64_t ld, __bf16 *out, int64_t rows_pad) {
        Turn a{q, rows, ld, (int)K, whole16(q, ld, K), out, rows_pad, 0, 0};
        if (want) a.bx = (int)((rows_pad + 255) / 256), a.by = (int)((K + 63) / 64);
        return a;
    };
    const Turn tw = turn(gx, qw, N, ldqw, wt, p.n_pad), tx = turn(gw, qx, M, ldqx, xt, p.m_pad);
    const int bx = gs || gt || part ? (int)(p.m_pad / 64) : 0, by = (int)(p.n_pad / 64);
    const int64_t blocks = (int64_t)bx * by + (int64_t)tw.bx * tw.by + (int64_t)tx.bx * tx.by;
    DPD_REQUIRE(blocks * 256 <= UINT32_MAX, DPD_ERR_SHAPE, "int8_linear_backward: %lld x %lld gradients are too many for one call", (long long)M, (long long)N);
    hipLaunchKernelGGL((k_backward_images<T>), dim3((unsigned)blocks), dim3(256), 0, st, g, M, (int)N, ldg, whole8(g, ldg), sw, sx, gs, p.n_pad, gt,
                       p.m_pad, part, bx, by, tw, tx);
    DPD_LAUNCH_CHECK();
    if (gb) {
        const int rc = with_type(gb_type, [&](auto t) {
            using B = decltype(t);
            hipLaunchKernelGGL((k_bias_grad<B>), dim3((unsigned)((N + 31) / 32)), dim3(256), 0, st, part, p.m_pad / 64, (int)N, (B *)gb);
            DPD_LAUNCH_CHECK();
            return DPD_OK;
        });
        if (rc) return rc;
    }
    if (gx) {
        nt::Args a{};
        a.a = (const char *)gs, a.lda = P * p.n_pad * 2, a.b = (const char *)wt, a.ldb = p.n_pad * 2, a.M = (int)M, a.N = (int)K;
        a.wrap = (int)(p.n_pad / 64), a.steps = P * a.wrap, a.tail = 128;
        const int rc = nt::product<nt::BF16>(a, 1, PlainOut<T>{gx, K, (int)K, whole8(gx, K)}, st);
        if (rc) return rc;
    }
    if (gw) {
        nt::Args a{};
        a.a = (const char *)gt, a.lda = P * p.m_pad * 2, a.b = (const char *)xt, a.ldb = p.m_pad * 2, a.M = (int)N, a.N = (int)K;
        a.wrap = (int)(p.m_pad / 64), a.steps = P * a.wrap, a.tail = 128;
        const int rc = with_type(gw_type, [&](auto t) {
            using W = decltype(t);
            return nt::product<nt::BF16>(a, 1, PlainOut<W>{(W *)gw, K, (int)K, whole8((W *)gw, K)}, st);
        });
        if (rc) return rc;
    }
    return DPD_OK;
}

bool is_type(int t) { return t == DPD_F32 || t == DPD_BF16 || t == DPD_F16; }

template <class T>
__global__ __launch_bounds__(256) void k_fill_zero(T *__restrict__ p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = from_f32<T>(0.f);
}

int zero_any(void *p, int type, int64_t n, hipStream_t st) {
    if (!p || n == 0) return DPD_OK;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((k_fill_zero<T>), dim3(grid_for(n, 256)), dim3(256), 0, st, (T *)p, n);
        DPD_LAUNCH_CHECK();
        return DPD_OK;
    });
}

// What every entry point with a product asks of its sizes.
int check_sizes(const char *who, int64_t M, int64_t N, int64_t K) {
    DPD_REQUIRE(M >= 0 && N >= 0 && K >= 0, DPD_ERR_INVALID_ARG, "%s: negative size", who);
    DPD_REQUIRE(K >= 1 && K <= MAX_K, DPD_ERR_SHAPE, "%s: %lld input features; 1 to %lld keep the 32-bit sum exact", who, (long long)K,
                (long long)MAX_K);
    DPD_REQUIRE(M <= INT32_MAX - 256 && N <= INT32_MAX - 256, DPD_ERR_SHAPE, "%s: %lld tokens or %lld output features are too many", who,
                (long long)M, (long long)N);
    return DPD_OK;
}

}  // namespace

extern "C" int dpd_quantize_rows_int8(const void *x, int type, int64_t rows, int64_t cols, int64_t ldx, int8_t *q, int64_t ldq,
                                      float *scale, void *stream) {
    DPD_REQUIRE(is_type(type), DPD_ERR_INVALID_ARG, "quantize_rows_int8: element type %d", type);
    DPD_REQUIRE(rows >= 0 && cols >= 0, DPD_ERR_INVALID_ARG, "quantize_rows_int8: negative size");
    DPD_REQUIRE(cols >= 1 && cols <= INT32_MAX / 2 && rows <= INT32_MAX - 256, DPD_ERR_SHAPE, "quantize_rows_int8: bad shape [%lld, %lld]",
                (long long)rows, (long long)cols);
    DPD_REQUIRE(rows == 0 || (x && q && scale), DPD_ERR_INVALID_ARG, "quantize_rows_int8: null pointer");
    DPD_REQUIRE(ldx >= cols && ldq >= cols && ldq <= INT32_MAX, DPD_ERR_INVALID_ARG, "quantize_rows_int8: row stride below the row length");
    if (rows == 0) return DPD_OK;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        return quantize_rows((const T *)x, rows, (int)cols, ldx, q, ldq, scale, as_stream(stream));
    });
}

extern "C" size_t dpd_int8_matmul_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    return M < 0 || N < 0 || K < 0 ? 0 : (size_t)((M + N) * nt::pad_to(K, 128) + 512);
}

extern "C" int dpd_int8_matmul(const int8_t *a, int64_t lda, const float *a_scale, const int8_t *b, int64_t ldb, const float *b_scale,
                               const void *bias, int bias_type, int64_t M, int64_t N, int64_t K, void *out, int out_type, int64_t ldo,
                               void *ws, size_t ws_bytes, void *stream) {
    DPD_REQUIRE(is_type(out_type) && (!bias || is_type(bias_type)), DPD_ERR_INVALID_ARG, "int8_matmul: element type");
    if (const int rc = check_sizes("int8_matmul", M, N, K)) return rc;
    if (M == 0 || N == 0) return DPD_OK;
    DPD_REQUIRE(a && b && a_scale && b_scale && out, DPD_ERR_INVALID_ARG, "int8_matmul: null pointer");
    DPD_REQUIRE(lda >= K && ldb >= K && ldo >= N && lda <= nt::MAX_ROW_BYTES && ldb <= nt::MAX_ROW_BYTES, DPD_ERR_INVALID_ARG, "int8_matmul: row stride");
    hipStream_t st = as_stream(stream);
    const int64_t ld = nt::pad_to(K, 128);
    const bool copy_a = !readable(a, lda, K), copy_b = !readable(b, ldb, K);
    if (copy_a || copy_b) {
        char *w = (char *)(((uintptr_t)ws + 255) & ~(uintptr_t)255);
        DPD_REQUIRE(ws && (size_t)((copy_a ? M * ld : 0) + (copy_b ? N * ld : 0)) + (size_t)(w - (char *)ws) <= ws_bytes, DPD_ERR_WORKSPACE,
                    "int8_matmul: rows that are not 16-byte aligned need a workspace of dpd_int8_matmul_workspace_bytes()");
        if (copy_a) {
            hipLaunchKernelGGL(k_pad_rows, dim3(grid_for(M * ld, 256)), dim3(256), 0, st, a, M, (int)K, lda, (int8_t *)w, ld);
            DPD_LAUNCH_CHECK();
            a = (const int8_t *)w, lda = ld, w += M * ld;
        }
        if (copy_b) {
            hipLaunchKernelGGL(k_pad_rows, dim3(grid_for(N * ld, 256)), dim3(256), 0, st, b, N, (int)K, ldb, (int8_t *)w, ld);
            DPD_LAUNCH_CHECK();
            b = (const int8_t *)w, ldb = ld;
        }
        if (copy_a && copy_b) K = ld;      // both carry zeros behind the row
    }
    return with_type(out_type, [&](auto t) {
        using T = decltype(t);
        return int8_product(a, lda, a_scale, b, ldb, b_scale, bias, bias_type, M, N, K, (T *)out, ldo, st);
    });
}

// ---- tokens against weights that are quantised once -----------------------------------------
extern "C" int64_t dpd_int8_row_bytes(int64_t K) { return K < 0 ? 0 : nt::pad_to(K, 128); }

extern "C" size_t dpd_int8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    return M < 0 || N < 0 || K < 0 ? 0 : (size_t)(M * nt::pad_to(K, 128) + nt::pad_to(M * 4, 256) + 256);
}

extern "C" int dpd_int8_linear(const void *x, int type, int64_t M, int64_t K, int64_t ldx, const int8_t *qw, const float *w_scale,
                               const void *bias, int bias_type, int64_t N, void *out, int64_t ldo, void *ws, size_t ws_bytes, void *stream) {
    DPD_REQUIRE(is_type(type) && (!bias || is_type(bias_type)), DPD_ERR_INVALID_ARG, "int8_linear: element type");
    if (const int rc = check_sizes("int8_linear", M, N, K)) return rc;
    if (M == 0 || N == 0) return DPD_OK;
    DPD_REQUIRE(x && qw && w_scale && out, DPD_ERR_INVALID_ARG, "int8_linear: null pointer");
    DPD_REQUIRE(ldx >= K && ldo >= N, DPD_ERR_INVALID_ARG, "int8_linear: row stride");
    DPD_REQUIRE(((uintptr_t)qw & 15) == 0, DPD_ERR_INVALID_ARG, "int8_linear: the weight image is 16-byte aligned");
    const int64_t ld = nt::pad_to(K, 128);
    hipStream_t st = as_stream(stream);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        const T *xt = (const T *)x;
        constexpr int V = 16 / sizeof(T);
        const FewPlan few = few_plan(xt, M, N, K, ldx, ld);
        if (takes_some(M, N, ld) && (M >= 3 || !few.waves)) {
            const ScaleOut<T> epi{nullptr, w_scale, bias, bias_type, (T *)out, ldo, (int)N, false};
            return in_pieces(Rows<T>{xt, M, ldx, nullptr, ld, nullptr}, (int)K) ? some_tokens<T, V>(xt, M, K, ldx, ld, qw, epi, st)
                                                                              : some_tokens<T, 1>(xt, M, K, ldx, ld, qw, epi, st);
        }
        if (few.waves) {
            const ScaleOut<T> epi{nullptr, w_scale, bias, bias_type, (T *)out, ldo, (int)N, false};
            if (few.waves == 16) return few.vec == V ? few_tokens<T, 16, V>(xt, M, K, ldx, ld, qw, epi, st) : few_tokens<T, 16, 1>(xt, M, K, ldx, ld, qw, epi, st);
            return few.vec == V ? few_tokens<T, 4, V>(xt, M, K, ldx, ld, qw, epi, st) : few_tokens<T, 4, 1>(xt, M, K, ldx, ld, qw, epi, st);
        }
        DPD_REQUIRE(ws && ws_bytes >= dpd_int8_linear_workspace_bytes(M, N, K), DPD_ERR_WORKSPACE, "int8_linear: workspace");
        float *sx = (float *)(((uintptr_t)ws + 255) & ~(uintptr_t)255);
        int8_t *qx = (int8_t *)sx + nt::pad_to(M * 4, 256);
        const int rc = quantize_rows(xt, M, (int)K, ldx, qx, ld, sx, st);
        return rc ? rc : int8_product(qx, ld, sx, qw, ld, w_scale, bias, bias_type, M, N, ld, (T *)out, ldo, st);
    });
}

extern "C" int dpd_int8_linear_forward(const void *x, int type, int64_t M, int64_t K, int64_t ldx, const void *w, int w_type, int64_t N, int64_t ldw,
                                       const void *bias, int bias_type, void *out, int64_t ldo, int8_t *qx, float *x_scale, int8_t *qw, float *w_scale,
                                       void *stream) {
    DPD_REQUIRE(is_type(type) && is_type(w_type) && (!bias || is_type(bias_type)), DPD_ERR_INVALID_ARG, "int8_linear_forward: element type");
    if (const int rc = check_sizes("int8_linear_forward", M, N, K)) return rc;
    DPD_REQUIRE((M == 0 || (x && qx && x_scale)) && (N == 0 || (w && qw && w_scale)) && (M == 0 || N == 0 || out), DPD_ERR_INVALID_ARG,
                "int8_linear_forward: null pointer");
    DPD_REQUIRE(ldx >= K && ldw >= K && ldo >= N, DPD_ERR_INVALID_ARG, "int8_linear_forward: row stride");
    DPD_REQUIRE((((uintptr_t)qx | (uintptr_t)qw) & 15) == 0, DPD_ERR_INVALID_ARG, "int8_linear_forward: the images are 16-byte aligned");
    const int64_t ld = nt::pad_to(K, 128);
    hipStream_t st = as_stream(stream);
    auto quantize = [&](int t, bool tokens, bool weight) {
        return with_type(t, [&](auto e) {
            using T = decltype(e);
            const Rows<T> a{(const T *)x, tokens ? M : 0, ldx, qx, ld, x_scale}, b{(const T *)w, weight ? N : 0, ldw, qw, ld, w_scale};
            // one launch for both, unless one of them can be read in wide pieces and the other cannot
            if (a.rows && b.rows && in_pieces(a, (int)K) != in_pieces(b, (int)K)) {
                const int rc = quantize_rows(a, Rows<T>{}, (int)K, st);
                return rc ? rc : quantize_rows(b, Rows<T>{}, (int)K, st);
            }
            return a.rows ? quantize_rows(a, b, (int)K, st) : quantize_rows(b, a, (int)K, st);
        });
    };
    int rc = quantize(type, true, type == w_type);
    if (!rc && type != w_type) rc = quantize(w_type, false, true);
    if (rc || M == 0 || N == 0) return rc;
    return with_type(type, [&](auto e) {
        using T = decltype(e);
        return int8_product(qx, ld, x_scale, qw, ld, w_scale, bias, bias_type, M, N, ld, (T *)out, ldo, st);
    });
}

extern "C" size_t dpd_int8_linear_backward_workspace_bytes(int64_t M, int64_t N, int64_t K, int type, int need_gx, int need_gw, int need_gb) {
    if (M < 0 || N < 0 || K < 0 || !is_type(type)) return 0;
    return (size_t)BackwardPlan(M, N, K, planes_for(type), need_gx, need_gw, need_gb).total + 256;
}

extern "C" int dpd_int8_linear_backward(const void *g, int type, int64_t M, int64_t N, int64_t K, int64_t ldg, const int8_t *qx, int64_t ldqx,
                                        const float *x_scale, const int8_t *qw, int64_t ldqw, const float *w_scale, void *gx, void *gw,
                                        int gw_type, void *gb, int gb_type, void *ws, size_t ws_bytes, void *stream) {
    DPD_REQUIRE(is_type(type) && (!gw || is_type(gw_type)) && (!gb || is_type(gb_type)), DPD_ERR_INVALID_ARG, "int8_linear_backward: element type");
    if (const int rc = check_sizes("int8_linear_backward", M, N, K)) return rc;
    hipStream_t st = as_stream(stream);
    if (M == 0 || N == 0) {                        // sums over nothing
        if (const int rc = zero_any(gx, type, M * K, st)) return rc;
        if (const int rc = zero_any(gw, gw_type, N * K, st)) return rc;
        return zero_any(gb, gb_type, N, st);
    }
    if (!gx && !gw && !gb) return DPD_OK;
    DPD_REQUIRE(g && (!gx || (qw && w_scale)) && (!gw || (qx && x_scale)), DPD_ERR_INVALID_ARG, "int8_linear_backward: null pointer");
    DPD_REQUIRE(ldg >= N && (!gw || ldqx >= K) && (!gx || ldqw >= K), DPD_ERR_INVALID_ARG, "int8_linear_backward: row stride");
    // gx sums along the output features, gw along the tokens: so long are the rows of g's images
    const int64_t row_x = gx ? planes_for(type) * 2 * nt::pad_to(N, 64) : 0, row_w = gw ? planes_for(type) * 2 * nt::pad_to(M, 64) : 0;
    DPD_REQUIRE(row_x <= nt::MAX_ROW_BYTES, DPD_ERR_SHAPE, "int8_linear_backward: %lld output features are too many for the gradient of x", (long long)N);
    DPD_REQUIRE(row_w <= nt::MAX_ROW_BYTES, DPD_ERR_SHAPE, "int8_linear_backward: %lld tokens are too many for the weight's gradient in one call",
                (long long)M);
    DPD_REQUIRE(ws && ws_bytes >= dpd_int8_linear_backward_workspace_bytes(M, N, K, type, gx != nullptr, gw != nullptr, gb != nullptr),
                DPD_ERR_WORKSPACE, "int8_linear_backward: workspace");
    char *w = (char *)(((uintptr_t)ws + 255) & ~(uintptr_t)255);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        return gradients((const T *)g, ldg, M, N, K, qx, ldqx, x_scale, qw, ldqw, w_scale, (T *)gx, gw, gw_type, gb, gb_type, w, st);
    });
}
