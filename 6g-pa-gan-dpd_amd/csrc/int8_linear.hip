// The 8-bit linear layer: rows quantised with one scale each, the int8 product of two sets of such rows, and the
// straight-through gradients.
//
//   quantiser   s = fl32(max(max|x|, 2^-100) / 127),  q = round-half-even(x / s) of the exact quotient
//   product     y[m, n] = ((sum_k qa[m, k] qb[n, k]) * sa[m]) * sb[n] + bias[n]     (the sum exactly, in int32)
//   gradients   gx = g (qw sw),  gw = g^T (qx sx),  gb = column sums of g
#include <type_traits>
#include "gemm_nt.h"

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
    return top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : fmaxf(__uint_as_float(top), SCALE_FLOOR) / 127.0f;
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

// One row per TEAM threads (a wave, or the whole workgroup).  The row is read twice: the second time from the cache.
template <class T, int TEAM>
__global__ __launch_bounds__(256) void k_quantize_rows(const T *__restrict__ x, int64_t rows, int cols, int64_t ldx,
                                                       int8_t *__restrict__ q, int64_t ldq, float *__restrict__ scale) {
    __shared__ unsigned top4[4];
    const int t = threadIdx.x % TEAM;
    const int64_t row = (int64_t)blockIdx.x * (256 / TEAM) + threadIdx.x / TEAM;
    if (TEAM == 64 && row >= rows) return;
    const T *xr = x + row * ldx;
    unsigned top = 0;
    for (int i = t; i < cols; i += TEAM) top = max(top, abs_bits(to_f32(xr[i])));
    top = wave_umax(top);
    if (TEAM == 256) {
        if ((threadIdx.x & 63) == 0) top4[threadIdx.x >> 6] = top;
        __syncthreads();
        top = max(max(top4[0], top4[1]), max(top4[2], top4[3]));
    }
    const float s = row_scale(top);
    const bool fine = top < 0x7f800000u;
    const float inv = 1.0f / s;
    int8_t *qr = q + row * ldq;
    for (int i = t; i < ldq; i += TEAM) qr[i] = (fine && i < cols) ? (int8_t)quantise(to_f32(xr[i]), s, inv) : (int8_t)0;
    if (t == 0) scale[row] = s;
}

template <class T>
int quantize_rows(const T *x, int64_t rows, int cols, int64_t ldx, int8_t *q, int64_t ldq, float *scale, hipStream_t st) {
    if (cols <= 1024)
        hipLaunchKernelGGL((k_quantize_rows<T, 64>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, x, rows, cols, ldx, q, ldq, scale);
    else
        hipLaunchKernelGGL((k_quantize_rows<T, 256>), dim3((unsigned)rows), dim3(256), 0, st, x, rows, cols, ldx, q, ldq, scale);
    DPD_LAUNCH_CHECK();
    return DPD_OK;
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
    DEV void put(int, int m, int n, float *v, const Row &r, const Col &c) const {
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
    typedef None Row, Col;
    DEV Row row(int, int) const { return {}; }
    DEV Col col(int, int) const { return {}; }
    DEV void put(int, int m, int n, float *v, Row, Col) const { store8(out + (int64_t)m * ldo + n, v, N - n, whole); }
};

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
// bf16 planes of a value: 1 for bf16 gradients (one rounding of 2^-8, the type's own), 2 for fp16 (2^-16),
// 3 for fp32 (the whole value): the planes of a row lie one behind the other along k, the smallest first.
template <class T>
constexpr int planes_of() { return std::is_same<T, float>::value ? 3 : std::is_same<T, __bf16>::value ? 1 : 2; }

template <int P>
DEV void put_planes(__bf16 *p, int64_t plane, float v) {
#pragma unroll
    for (int i = P - 1; i >= 0; --i) {
        const __bf16 h = (__bf16)v;
        p[i * plane] = h;
        v = fabsf((float)h) < INFINITY ? v - (float)h : 0.f;      // an infinity stays one: nothing is left of it
    }
}

// One 64 x 64 tile of g [M, N]: gs[m, n] = g sw[n] (row-major, for gx), gt[n, m] = g sx[m] (transposed, for gw), each as
// bf16 planes with zeros behind the rows, and this tile's column sums for gb.
template <class T>
__global__ __launch_bounds__(256) void k_grad_images(const T *__restrict__ g, int64_t M, int N, int64_t ldg, const float *__restrict__ sw,
                                                     const float *__restrict__ sx, __bf16 *__restrict__ gs, int64_t n_pad,
                                                     __bf16 *__restrict__ gt, int64_t m_pad, float *__restrict__ gb_part) {
    constexpr int P = planes_of<T>();
    __shared__ float t[64][65];
    const int64_t m0 = (int64_t)blockIdx.x * 64;
    const int n0 = blockIdx.y * 64;
    for (int e = threadIdx.x; e < 4096; e += 256) {
        const int i = e >> 6, j = e & 63;
        const float v = (m0 + i < M && n0 + j < N) ? to_f32(g[(m0 + i) * ldg + n0 + j]) : 0.f;
        t[i][j] = v;
        if (gs && m0 + i < M) put_planes<P>(gs + (m0 + i) * (P * n_pad) + n0 + j, n_pad, n0 + j < N ? v * sw[n0 + j] : 0.f);
    }
    __syncthreads();
    if (gt)
        for (int e = threadIdx.x; e < 4096; e += 256) {
            const int j = e >> 6, i = e & 63;
            if (n0 + j < N) put_planes<P>(gt + (int64_t)(n0 + j) * (P * m_pad) + m0 + i, m_pad, m0 + i < M ? t[i][j] * sx[m0 + i] : 0.f);
        }
    if (gb_part && threadIdx.x < 64 && n0 + threadIdx.x < N) {
        float s = 0.f;
        for (int i = 0; i < 64; ++i) s += t[i][threadIdx.x];
        gb_part[(int64_t)blockIdx.x * N + n0 + threadIdx.x] = s;
    }
}

template <class T>
__global__ __launch_bounds__(256) void k_bias_grad(const float *__restrict__ part, int64_t blocks, int N, T *__restrict__ gb) {
    const int n = blockIdx.x * 256 + threadIdx.x;
    if (n >= N) return;
    double s = 0.0;
    for (int64_t b = 0; b < blocks; ++b) s += (double)part[b * N + n];
    gb[n] = from_f32<T>((float)s);
}

// q [rows, cols] int8 -> out [cols, rows_pad] bf16 (exact), zeros behind the rows
__global__ __launch_bounds__(256) void k_transpose_i8(const int8_t *__restrict__ q, int64_t rows, int cols, int64_t ld,
                                                      __bf16 *__restrict__ out, int64_t rows_pad) {
    __shared__ int8_t t[64][68];
    const int64_t r0 = (int64_t)blockIdx.x * 64;
    const int c0 = blockIdx.y * 64;
    for (int e = threadIdx.x; e < 4096; e += 256) {
        const int i = e >> 6, j = e & 63;
        t[i][j] = (r0 + i < rows && c0 + j < cols) ? q[(r0 + i) * ld + c0 + j] : (int8_t)0;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 4096; e += 256) {
        const int j = e >> 6, i = e & 63;
        if (c0 + j < cols) out[(int64_t)(c0 + j) * rows_pad + r0 + i] = (__bf16)(float)t[i][j];
    }
}

int planes_for(int type) { return type == DPD_F32 ? 3 : type == DPD_BF16 ? 1 : 2; }

struct BackwardPlan {
    int64_t m_pad, n_pad, gs, gt, wt, xt, part, total;      // element counts and byte offsets into the workspace
    BackwardPlan(int64_t M, int64_t N, int64_t K, int type, bool gx, bool gw, bool gb) {
        const int p = planes_for(type);
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

template <class T>
int gradients(const T *g, int64_t ldg, int64_t M, int64_t N, int64_t K, const int8_t *qx, int64_t ldqx, const float *sx,
              const int8_t *qw, int64_t ldqw, const float *sw, T *gx, void *gw, int gw_type, void *gb, int gb_type, char *ws, hipStream_t st) {
    constexpr int P = planes_of<T>();
    const BackwardPlan p(M, N, K, std::is_same<T, float>::value ? DPD_F32 : P == 1 ? DPD_BF16 : DPD_F16, gx, gw, gb);
    __bf16 *gs = gx ? (__bf16 *)(ws + p.gs) : nullptr, *wt = (__bf16 *)(ws + p.wt), *gt = gw ? (__bf16 *)(ws + p.gt) : nullptr,
           *xt = (__bf16 *)(ws + p.xt);
    float *part = gb ? (float *)(ws + p.part) : nullptr;
    hipLaunchKernelGGL((k_grad_images<T>), dim3((unsigned)(p.m_pad / 64), (unsigned)(p.n_pad / 64)), dim3(256), 0, st, g, M, (int)N, ldg, sw,
                       sx, gs, p.n_pad, gt, p.m_pad, part);
    DPD_LAUNCH_CHECK();
    if (gb) {
        const int rc = with_type(gb_type, [&](auto t) {
            using B = decltype(t);
            hipLaunchKernelGGL((k_bias_grad<B>), dim3((unsigned)((N + 255) / 256)), dim3(256), 0, st, part, p.m_pad / 64, (int)N, (B *)gb);
            DPD_LAUNCH_CHECK();
            return DPD_OK;
        });
        if (rc) return rc;
    }
    if (gx) {
        hipLaunchKernelGGL(k_transpose_i8, dim3((unsigned)(p.n_pad / 64), (unsigned)((K + 63) / 64)), dim3(256), 0, st, qw, N, (int)K, ldqw, wt, p.n_pad);
        DPD_LAUNCH_CHECK();
        nt::Args a{};
        a.a = (const char *)gs, a.lda = P * p.n_pad * 2, a.b = (const char *)wt, a.ldb = p.n_pad * 2, a.M = (int)M, a.N = (int)K;
        a.wrap = (int)(p.n_pad / 64), a.steps = P * a.wrap, a.tail = 128;
        const int rc = nt::product<nt::BF16>(a, 1, PlainOut<T>{gx, K, (int)K, whole8(gx, K)}, st);
        if (rc) return rc;
    }
    if (gw) {
        hipLaunchKernelGGL(k_transpose_i8, dim3((unsigned)(p.m_pad / 64), (unsigned)((K + 63) / 64)), dim3(256), 0, st, qx, M, (int)K, ldqx, xt, p.m_pad);
        DPD_LAUNCH_CHECK();
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
    DPD_REQUIRE(ws && ws_bytes >= dpd_int8_linear_workspace_bytes(M, N, K), DPD_ERR_WORKSPACE, "int8_linear: workspace");
    const int64_t ld = nt::pad_to(K, 128);
    float *sx = (float *)(((uintptr_t)ws + 255) & ~(uintptr_t)255);
    int8_t *qx = (int8_t *)sx + nt::pad_to(M * 4, 256);
    hipStream_t st = as_stream(stream);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        const int rc = quantize_rows((const T *)x, M, (int)K, ldx, qx, ld, sx, st);
        return rc ? rc : int8_product(qx, ld, sx, qw, ld, w_scale, bias, bias_type, M, N, ld, (T *)out, ldo, st);
    });
}

extern "C" size_t dpd_int8_linear_backward_workspace_bytes(int64_t M, int64_t N, int64_t K, int type, int need_gx, int need_gw, int need_gb) {
    if (M < 0 || N < 0 || K < 0 || !is_type(type)) return 0;
    return (size_t)BackwardPlan(M, N, K, type, need_gx, need_gw, need_gb).total + 256;
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
    const int64_t row = planes_for(type) * 2 * nt::pad_to(M > N ? M : N, 64);
    DPD_REQUIRE(row <= nt::MAX_ROW_BYTES, DPD_ERR_SHAPE, "int8_linear_backward: %lld tokens or %lld output features are too many for one call",
                (long long)M, (long long)N);
    DPD_REQUIRE(ws && ws_bytes >= dpd_int8_linear_backward_workspace_bytes(M, N, K, type, gx != nullptr, gw != nullptr, gb != nullptr),
                DPD_ERR_WORKSPACE, "int8_linear_backward: workspace");
    char *w = (char *)(((uintptr_t)ws + 255) & ~(uintptr_t)255);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        return gradients((const T *)g, ldg, M, N, K, qx, ldqx, x_scale, qw, ldqw, w_scale, (T *)gx, gw, gw_type, gb, gb_type, w, st);
    });
}
