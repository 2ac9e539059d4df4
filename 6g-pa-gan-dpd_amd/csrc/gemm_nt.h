// Tiled matrix-core product of two row-major operands, C[m, n] = sum_k A[m, k] B[n, k] (both contiguous along k), for
// int8, bf16 and fp16 elements: the one product that the 8-bit linear layer (forward and both gradients) and the
// orthogonalised update are made of.
//
// Every element type is seen as bytes: a K step is 128 bytes of each row (128 int8, 64 bf16 / fp16), two 16-byte
// fragments per lane and step.  A workgroup of WAVES_M x WAVES_N waves owns a BM x BN tile; two LDS stages hold the
// 128-byte pieces of its BM + BN rows, filled by direct global -> LDS loads (16 bytes a lane, 8 rows an instruction)
// while the other stage is multiplied.  One barrier a step: behind it every wave has both finished reading the stage
// that is filled next and seen the arrival of the stage that is read next.
//
// LDS layout: row r keeps its 16-byte chunk c at position c ^ (r & 7).  The direct load writes lane after lane, so the
// permutation is applied to the global chunk a lane asks for; a fragment read then touches all banks evenly (8
// successive lanes read 8 different 16-byte columns).
//
// Operands of a product in a split form (SPLIT): a row holds blocks of 32 elements, first their leading halves (64
// bytes), then their remainders (64 bytes).  A step then carries 32 elements, and the three products lead*lead,
// lead*rest, rest*lead go into one accumulator: fp16 halves of a scaled fp32 value give 22 bits of it.
//
// Lane layout of the results: the B rows are the first operand of the instruction, so a lane of a 16 x 16 block holds
// C[m = lane & 15][n = 4 * (lane >> 4) + 0..3]: four consecutive columns of one row.
#pragma once
#include "common.h"

namespace nt {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void;

enum Kind { I8, BF16, F16, F16_SPLIT };

template <int KIND>
struct Acc {
    using type = f32x4;
};
template <>
struct Acc<I8> {
    using type = i32x4;
};

template <int KIND>
DEV typename Acc<KIND>::type mfma(i32x4 a, i32x4 b, typename Acc<KIND>::type c) {
    if constexpr (KIND == I8)
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
    else if constexpr (KIND == BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

struct Args {
    const char *a, *b;             // 16-byte aligned
    int64_t lda, ldb;              // bytes from row to row: multiples of 16
    int64_t a_batch, b_batch;      // bytes from matrix to matrix (grid z)
    int M, N;                      // rows of a and of b
    int steps;                     // K steps of the whole product
    int wrap;                      // steps after which the B operand starts again (a has several planes along k); == steps otherwise
    int tail;                      // valid bytes of the last step of a plane (a multiple of 16; 128 where rows are padded)
    int tiles_m, tiles_n;
    int lower;                     // C is symmetric: tiles wholly above the diagonal are left out (BM == BN)
};

constexpr int STEP = 128;                                   // bytes of a row per step

// Which tile a workgroup takes.  Workgroups go to the 8 XCDs in turn; each XCD gets a contiguous run of tiles, and
// inside a run the tiles go down bands of 8 tile rows, so that the operands of neighbours meet in one L2.
DEV void tile_of(const Args &g, int id, int n_tiles, int *tm, int *tn) {
    const int xcd = id & 7, q = n_tiles >> 3, r = n_tiles & 7;
    const int t = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (id >> 3);
    const int band = 8 * g.tiles_n, b = t / band, in = t - b * band;
    const int rows = min(8, g.tiles_m - b * 8);
    *tn = in / rows;
    *tm = b * 8 + in - *tn * rows;
}

template <int KIND, int BM, int BN, int WAVES_M, int WAVES_N, class Epilogue>
DEV void gemm_tile(const Args &g, const Epilogue &epi) {
    constexpr int WAVES = WAVES_M * WAVES_N, TM = BM / WAVES_M / 16, TN = BN / WAVES_N / 16;
    constexpr int LOADS_A = BM / 8 / WAVES, LOADS_B = BN / 8 / WAVES, STAGE = (BM + BN) * STEP;
    static_assert(LOADS_A >= 1 && LOADS_B >= 1, "every wave loads whole groups of 8 rows");
    __shared__ __attribute__((aligned(128))) char smem[2 * STAGE];
    int tm, tn;
    tile_of(g, blockIdx.x, g.tiles_m * g.tiles_n, &tm, &tn);
    if (g.lower && tn > tm) return;
    const int m0 = tm * BM, n0 = tn * BN;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WAVES_N, wn = wave % WAVES_N;

    const char *ab = g.a + blockIdx.z * g.a_batch + (int64_t)m0 * g.lda, *bb = g.b + blockIdx.z * g.b_batch + (int64_t)n0 * g.ldb;
    // rows beyond the last read it again (their results are not stored); chunks beyond `tail` lie outside the resource
    // and arrive as zeros.  The step is the scalar offset, which the bounds check leaves out.
    const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc((void *)ab, 0, 0x7fffffff, 0x00020000);
    const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc((void *)bb, 0, 0x7fffffff, 0x00020000);
    const int chunk = ((lane & 7) ^ (lane >> 3)) * 16;
    unsigned va[LOADS_A], vb[LOADS_B];
#pragma unroll
    for (int i = 0; i < LOADS_A; ++i) va[i] = (unsigned)(min((i * WAVES + wave) * 8 + (lane >> 3), g.M - 1 - m0) * (int)g.lda + chunk);
#pragma unroll
    for (int i = 0; i < LOADS_B; ++i) vb[i] = (unsigned)(min((i * WAVES + wave) * 8 + (lane >> 3), g.N - 1 - n0) * (int)g.ldb + chunk);

    auto stage = [&](int s, int buf) {
        char *base = smem + buf * STAGE;
        const int w = s % g.wrap;
        const bool cut = w == g.wrap - 1 && chunk >= g.tail;
#pragma unroll
        for (int i = 0; i < LOADS_A; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_void *)(base + (i * WAVES + wave) * 1024), 16, cut ? 0xfffffff0u : va[i], s * STEP, 0, 0);
#pragma unroll
        for (int i = 0; i < LOADS_B; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_void *)(base + BM * STEP + (i * WAVES + wave) * 1024), 16, cut ? 0xfffffff0u : vb[i], w * STEP, 0, 0);
    };

    typename Acc<KIND>::type acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = typename Acc<KIND>::type{0, 0, 0, 0};

    const int frag = (lane & 15) * STEP, c0 = ((lane >> 4) ^ (lane & 7)) * 16, c1 = ((4 + (lane >> 4)) ^ (lane & 7)) * 16;
    auto compute = [&](int buf) {
        const char *pa = smem + buf * STAGE + wm * TM * 16 * STEP + frag, *pb = smem + buf * STAGE + (BM + wn * TN * 16) * STEP + frag;
        i32x4 a0[TM], b0[TN], a1[TM], b1[TN];
#pragma unroll
        for (int i = 0; i < TM; ++i) a0[i] = *(const i32x4 *)(pa + i * 16 * STEP + c0);
#pragma unroll
        for (int j = 0; j < TN; ++j) b0[j] = *(const i32x4 *)(pb + j * 16 * STEP + c0);
#pragma unroll
        for (int i = 0; i < TM; ++i) a1[i] = *(const i32x4 *)(pa + i * 16 * STEP + c1);
#pragma unroll
        for (int j = 0; j < TN; ++j) b1[j] = *(const i32x4 *)(pb + j * 16 * STEP + c1);
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                if constexpr (KIND == F16_SPLIT) {
                    acc[i][j] = mfma<KIND>(b1[j], a0[i], acc[i][j]);
                    acc[i][j] = mfma<KIND>(b0[j], a1[i], acc[i][j]);
                    acc[i][j] = mfma<KIND>(b0[j], a0[i], acc[i][j]);
                } else {
                    acc[i][j] = mfma<KIND>(b0[j], a0[i], acc[i][j]);
                }
            }
        if constexpr (KIND != F16_SPLIT) {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = mfma<KIND>(b1[j], a1[i], acc[i][j]);
        }
    };

    stage(0, 0);
    for (int s = 0; s < g.steps; ++s) {
        // this wave's part of stage s has arrived, and its reads of the other stage have returned
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (s + 1 < g.steps) stage(s + 1, (s + 1) & 1);
        compute(s & 1);
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int m = m0 + (wm * TM + i) * 16 + (lane & 15), n = n0 + (wn * TN + j) * 16 + (lane >> 4) * 4;
            if (m < g.M && n < g.N) epi(blockIdx.z, m, n, acc[i][j]);
        }
}

template <int KIND, int BM, int BN, int WAVES_M, int WAVES_N, class Epilogue>
static __global__ __launch_bounds__(64 * WAVES_M *WAVES_N) void k_gemm(Args g, Epilogue epi) {
    gemm_tile<KIND, BM, BN, WAVES_M, WAVES_N>(g, epi);
}

// ---- host side -------------------------------------------------------------------------
// Largest tile that still gives most of the 256 compute units one; the small ones trade operand traffic for that.
template <int KIND, int BM, int BN, int WAVES_M, int WAVES_N, class Epilogue>
static int launch(Args g, int batch, const Epilogue &epi, hipStream_t st) {
    g.tiles_m = (g.M + BM - 1) / BM;
    g.tiles_n = (g.N + BN - 1) / BN;
    hipLaunchKernelGGL((k_gemm<KIND, BM, BN, WAVES_M, WAVES_N, Epilogue>), dim3((unsigned)(g.tiles_m * g.tiles_n), 1, (unsigned)batch),
                       dim3(64 * WAVES_M * WAVES_N), 0, st, g, epi);
    DPD_LAUNCH_CHECK();
    return DPD_OK;
}

template <int KIND, class Epilogue>
static int product(const Args &g, int batch, const Epilogue &epi, hipStream_t st) {
    auto tiles = [&](int b) { return (int64_t)((g.M + b - 1) / b) * ((g.N + b - 1) / b) * batch; };
    if (tiles(256) >= 192) return launch<KIND, 256, 256, 2, 4>(g, batch, epi, st);
    if (tiles(128) >= 128) return launch<KIND, 128, 128, 2, 2>(g, batch, epi, st);
    return launch<KIND, 64, 64, 2, 2>(g, batch, epi, st);
}

// A row of an operand may have at most this many bytes: 256 rows of a tile stay inside 32-bit offsets.
constexpr int64_t MAX_ROW_BYTES = (1 << 23) - 128;

static inline int64_t pad_to(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

}  // namespace nt

// ---- element types of the entry points ----------------------------------------------------
typedef float f32x4_t __attribute__((ext_vector_type(4)));

template <class T>
DEV float to_f32(T v) { return (float)v; }
template <class T>
DEV T from_f32(float v) { return (T)v; }           // round to nearest even

// One value of a tensor whose type is known at run time only.
DEV float load_any(const void *p, int type, int64_t i) {
    return type == DPD_F32 ? ((const float *)p)[i] : type == DPD_BF16 ? (float)((const __bf16 *)p)[i] : (float)((const _Float16 *)p)[i];
}

// Four consecutive values of one row; `whole`: all four lie inside the row and the address is aligned for one store.
template <class T>
DEV void store4(T *p, f32x4_t v, int valid, bool whole) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    if (whole && valid >= 4) {
        *(T4 *)p = T4{from_f32<T>(v[0]), from_f32<T>(v[1]), from_f32<T>(v[2]), from_f32<T>(v[3])};
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < valid) p[i] = from_f32<T>(v[i]);
    }
}

static inline int type_size(int type) { return type == DPD_F32 ? 4 : 2; }

// Calls f with a value of the element type that `type` names.
template <class F>
static int with_type(int type, F f) {
    if (type == DPD_F32) return f(float{});
    if (type == DPD_BF16) return f(__bf16{});
    return f(_Float16{});
}
