// Tiled matrix-core product of two row-major operands, C[m, n] = sum_k A[m, k] B[n, k] (both contiguous along k), for
// int8, bf16 and fp16 elements: the one product that the 8-bit linear layer (forward and both gradients) and the
// orthogonalised update are made of.
//
// Every element type is seen as bytes: a K step is 128 bytes of each row (128 int8, 64 bf16 / fp16), two 16-byte
// fragments per lane and step.  A workgroup of WAVES_M x WAVES_N waves owns a BM x BN tile.  STAGES pieces of LDS, each
// for one step of its BM + BN rows, are filled by direct global -> LDS loads (16 bytes a lane, 8 rows an instruction).
// The loop runs half a step ahead of itself: while the first fragments of a step are multiplied the second ones are
// read, and while those are multiplied the first ones of the next step.  One barrier a step, between the halves: behind
// it every wave has read all of this step's stage (which is filled again, STAGES steps ahead) and seen its successor.
// WAVES_K groups of such waves take the steps in turn, each with its part of a stage, and are added at the end.
//
// LDS layout: row r keeps its 16-byte chunk c at position c ^ key(r).  The direct load writes lane after lane, so the
// permutation is applied to the global chunk a lane asks for.  Keys are chosen so that the 16 lanes that read together
// hit 16 different 16-byte columns of the 256-byte bank row, for the row orders of both operands (measured: no conflicts).
//
// Operands of a product in a split form (SPLIT): a row holds blocks of 32 elements, first their leading halves (64
// bytes), then their remainders (64 bytes), held times REST.  A step then carries 32 elements; the product lead*lead goes into
// one accumulator, lead*rest and rest*lead into another, which joins the first divided by REST at the end.  The two halves
// give 22 bits of every scaled value of at least 2^-14, the smallest normal fp16 number, and an absolute 2^-36 below; without
// REST a remainder would be a subnormal below 2^-3 already: in an iteration of 150 x 300, X at unit size, the factors' roundings
// would put rows of a hundredth of the others' size 2.5e-6 off instead of 1.1e-7, rows of a ten-thousandth 2.4e-4.  The second
// accumulator leaves no registers for tiles above 256 x 128.
//
// Lane layout of the results: the B rows are the first operand of the instruction, so a lane of a 16 x 16 block holds
// one row m = lane & 15 and four columns.  The B rows of a pair of blocks are interleaved in fours, so that the pair gives
// a lane eight successive columns: n = 8 * (lane >> 4) + 0..7 of 32.
//
// Bound by the matrix cores, and on large products by the power that they may draw: with zeros for data 4096^3 in bf16 takes
// 80 us, with random data 100 to 106 (1.3 PFLOP/s); int8 4096^3 62 to 66 us, 8192^3 430 to 470 us (2.3 to 2.5 POP/s).  The library's
// products of these sizes take 96, 67 and 441 us.  Small ones are bound by the start of a kernel and the write-back at its end.
#pragma once
#include "common.h"

typedef float f32x4_t __attribute__((ext_vector_type(4)));

extern int g_product_tile;       // dpd_set_option("product_tile", -1 by the rule / 0..10 that tile wherever it applies)

namespace nt {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void;

enum Kind { I8, BF16, F16, F16_SPLIT };

struct Yes {
    static constexpr bool value = true;
};
struct No {
    static constexpr bool value = false;
};

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
    int tail;                      // valid bytes of the last step (a multiple of 16; 128 where rows are padded or wrap < steps)
    int tiles_m, tiles_n;
    int lower;                     // C is symmetric: the tiles above the diagonal are left out (BM == BN)
};

constexpr int STEP = 128;                                   // bytes of a row per step
constexpr float REST = 2048.f;                              // scale of the remainders of a split form: at most half a step of the leading half

// Which tile a workgroup takes.  Workgroups go to the 8 XCDs in turn; each XCD gets a contiguous run of tiles, and
// inside a run the tiles go down bands of 8 tile rows, so that the operands of neighbours meet in one L2.  `lower`: the
// tiles on and below the diagonal only (the last 8 columns of a band are a triangle).
DEV void tile_of(const Args &g, int id, int n_tiles, int *tm, int *tn) {
    const int xcd = id & 7, q = n_tiles >> 3, r = n_tiles & 7;
    int t = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (id >> 3), b = 0;
    if (!g.lower) {
        b = t / (8 * g.tiles_n), t -= b * 8 * g.tiles_n;
        const int rows = min(8, g.tiles_m - b * 8);
        *tn = t / rows;
        *tm = b * 8 + t - *tn * rows;
        return;
    }
    for (;; ++b) {
        const int rows = min(8, g.tiles_m - b * 8), square = rows * 8 * b, size = square + rows * (rows + 1) / 2;
        if (t >= size) {
            t -= size;
            continue;
        }
        if (t < square) {
            *tn = t / rows;
            *tm = b * 8 + t - *tn * rows;
            return;
        }
        t -= square;
        int col = 0;
        while (t >= rows - col) t -= rows - col++;
        *tn = b * 8 + col;
        *tm = b * 8 + col + t;
        return;
    }
}
static inline int64_t tiles_of(const Args &g) { return g.lower ? (int64_t)g.tiles_m * (g.tiles_m + 1) / 2 : (int64_t)g.tiles_m * g.tiles_n; }

// Row of a tile that lane r (0..15) of block j of the B operand stands for: blocks 2q and 2q + 1 share 32 rows.
DEV int b_row(int j, int r) { return (j >> 1) * 32 + (r >> 2) * 8 + (j & 1) * 4 + (r & 3); }
DEV int key_a(int row) { return row & 7; }                                              // 16 successive rows
DEV int key_b(int row) { return ((row >> 1) & 1) | (((row >> 3) & 3) << 1); }           // rows 0..3, 8..11, 16..19, 24..27 (+ 4)

// All but the N newest loads of this wave, and all its LDS reads, have arrived; then all waves of the workgroup.
template <int N>
DEV void wait_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));       // vmcnt(N), lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <int KIND, int BM, int BN, int WAVES_M, int WAVES_N, int WAVES_K, int STAGES, class Epilogue>
DEV void gemm_tile(const Args &g, const Epilogue &epi) {
    constexpr int WAVES = WAVES_M * WAVES_N, TM = BM / WAVES_M / 16, TN = BN / WAVES_N / 16;
    constexpr int LOADS_A = BM / 8 / WAVES, LOADS_B = BN / 8 / WAVES, LOADS = LOADS_A + LOADS_B, PART = (BM + BN) * STEP, STAGE = WAVES_K * PART;
    static_assert(LOADS_A >= 1 && LOADS_B >= 1 && LOADS_A * 8 * WAVES == BM && LOADS_B * 8 * WAVES == BN, "every wave loads whole groups of 8 rows");
    static_assert(TN % 2 == 0 && (TM % 2 == 0 || KIND != F16_SPLIT) && STAGES >= 2 && (STAGES - 1) * LOADS < 64, "pairs of blocks; the wait counter has 6 bits");
    constexpr int PITCH = BM + 8, TURN_BYTES = Epilogue::TURNED ? BN * PITCH * 2 : 0, LDS = STAGES * STAGE > TURN_BYTES ? STAGES * STAGE : TURN_BYTES;
    static_assert(LDS <= 160 * 1024, "LDS of a compute unit");
    __shared__ __attribute__((aligned(256))) char smem[LDS];
    int tm, tn;
    tile_of(g, blockIdx.x, gridDim.x, &tm, &tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const int lane = threadIdx.x & 63, all_waves = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = all_waves / WAVES, wave = all_waves % WAVES, wm = wave / WAVES_N, wn = wave % WAVES_N;
    char *const mine = smem + group * PART;                // this group's part of every stage
    const int steps = (g.steps + WAVES_K - 1) / WAVES_K;   // of a group: group k takes the steps k, k + WAVES_K, ...

    const char *ab = g.a + blockIdx.z * g.a_batch + (int64_t)m0 * g.lda, *bb = g.b + blockIdx.z * g.b_batch + (int64_t)n0 * g.ldb;
    // rows beyond the last read it again (their results are not stored); chunks beyond `tail` lie outside the resource
    // and arrive as zeros.  The step is the scalar offset, which the bounds check leaves out.
    const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc((void *)ab, 0, 0x7fffffff, 0x00020000);
    const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc((void *)bb, 0, 0x7fffffff, 0x00020000);
    unsigned va[LOADS_A], vb[LOADS_B];
    auto chunk_a = [&](int i) { return ((lane & 7) ^ key_a((i * WAVES + wave) * 8 + (lane >> 3))) * 16; };
    auto chunk_b = [&](int i) { return ((lane & 7) ^ key_b((i * WAVES + wave) * 8 + (lane >> 3))) * 16; };
#pragma unroll
    for (int i = 0; i < LOADS_A; ++i) va[i] = (unsigned)(min((i * WAVES + wave) * 8 + (lane >> 3), g.M - 1 - m0) * (int)g.lda + chunk_a(i));
#pragma unroll
    for (int i = 0; i < LOADS_B; ++i) vb[i] = (unsigned)(min((i * WAVES + wave) * 8 + (lane >> 3), g.N - 1 - n0) * (int)g.ldb + chunk_b(i));
    int wrapped = group % g.wrap;                          // step of the B operand that is loaded next
    auto load = [&](int i, int s, int at) {                // 8 rows: part i of LOADS
        if (i < LOADS_A)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_void *)(mine + at + (i * WAVES + wave) * 1024), 16, va[i], (s * WAVES_K + group) * STEP, 0, 0);
        else
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_void *)(mine + at + BM * STEP + ((i - LOADS_A) * WAVES + wave) * 1024), 16, vb[i - LOADS_A],
                                                     wrapped * STEP, 0, 0);
    };
    // chunks that the last step does not have, and steps that do not exist (a group's last): zeros
    const int cut_step = g.tail == STEP && WAVES_K == 1 ? -1 : steps - 1;
    auto before_loads = [&](int s) {
        if (s == cut_step) {
            const int have = s * WAVES_K + group, tail = have < g.steps - 1 ? STEP : have == g.steps - 1 ? g.tail : 0;
#pragma unroll
            for (int i = 0; i < LOADS_A; ++i) va[i] = chunk_a(i) >= tail ? 0xfffffff0u : va[i];
#pragma unroll
            for (int i = 0; i < LOADS_B; ++i) vb[i] = chunk_b(i) >= tail ? 0xfffffff0u : vb[i];
        }
    };
    auto after_loads = [&]() {
        wrapped += WAVES_K;
        while (wrapped >= g.wrap) wrapped -= g.wrap;
    };

    typename Acc<KIND>::type acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = typename Acc<KIND>::type{0, 0, 0, 0};
    constexpr bool SPLIT = KIND == F16_SPLIT;
    f32x4 cross[SPLIT ? TM : 1][SPLIT ? TN : 1];           // the products with remainders
    if constexpr (SPLIT) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) cross[i][j] = f32x4{0, 0, 0, 0};
    }

    // fragment c (0 or 1) of block i of A, of block j of B: the keys do not depend on i and j
    const int r = lane & 15, q = lane >> 4;
    const char *pa = mine + (wm * TM * 16 + r) * STEP, *pb = mine + (BM + wn * TN * 16) * STEP;
    const int ka[2] = {(q ^ key_a(r)) * 16, ((4 + q) ^ key_a(r)) * 16};
    const int kb[2] = {b_row(0, r) * STEP + (q ^ key_b(b_row(0, r))) * 16, b_row(0, r) * STEP + ((4 + q) ^ key_b(b_row(0, r))) * 16};
    i32x4 a0[SPLIT ? 2 : TM], b0[TN], a1[SPLIT ? 2 : TM], b1[TN];
    auto reada = [&](i32x4 *a, int k, int i, int at, int c) { a[k] = *(const i32x4 *)(pa + at + i * 16 * STEP + ka[c]); };
    auto readb = [&](i32x4 *b, int j, int at, int c) { b[j] = *(const i32x4 *)(pb + at + b_row(j, 0) * STEP + kb[c]); };
    auto mul = [&](const i32x4 *a, const i32x4 *b, int i) {
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mfma<KIND>(b[j], a[i], acc[i][j]);
    };
    auto mul3 = [&](int i, int j, int count) {             // blocks j .. j + count - 1 in turn
#pragma unroll
        for (int k = j; k < j + count; ++k) cross[i][k] = mfma<F16_SPLIT>(b1[k], a0[i & 1], cross[i][k]);
#pragma unroll
        for (int k = j; k < j + count; ++k) cross[i][k] = mfma<F16_SPLIT>(b0[k], a1[i & 1], cross[i][k]);
#pragma unroll
        for (int k = j; k < j + count; ++k) acc[i][k] = mfma<KIND>(b0[k], a0[i & 1], acc[i][k]);
    };
    // The order of the instructions is the order written here: in front of the products of block row i the reads of the
    // fragments that the next half needs (early, so that the last of them has arrived by then) and the loads.
    constexpr int READ_ROWS = TM > 2 ? TM - 2 : 1, READS = (TM + TN + READ_ROWS - 1) / READ_ROWS, LOADS_ROW = (LOADS + TM - 1) / TM;
    auto read_part = [&](i32x4 *a, i32x4 *b, int i, int at, int c) {
#pragma unroll
        for (int k = i * READS; k < (i + 1) * READS; ++k) {
            if (k < TM) reada(a, k, k, at, c);
            else if (k < TM + TN) readb(b, k - TM, at, c);
        }
    };
    auto next = [](int at) { return at == (STAGES - 1) * STAGE ? 0 : at + STAGE; };

    // What the epilogue reads: AHEAD block rows together.  Where a wave has few results and its workgroup is alone on the
    // compute unit, all of it in front of the loop, whose first wait it shares (1024 x 4096, update: 17.1 -> 16.3 us, last
    // 14.5 -> 13.6); a wave with many has no registers for that, and a second workgroup hides the wait at the end (there it cost
    // 42.4 -> 45.1 us).
    constexpr int AHEAD = SPLIT ? 2 : TM % 4 == 0 ? 4 : TM;
    constexpr bool EARLY = TM * TN <= 8 && AHEAD == TM && LDS > 80 * 1024;
    static_assert(TM % AHEAD == 0, "whole groups of block rows");
    typename Epilogue::Col col[TN / 2];
    typename Epilogue::Row row[AHEAD];
    typename Epilogue::Pre pre[AHEAD][TN / 2];
    auto read_col = [&]() {
#pragma unroll
        for (int j = 0; j < TN / 2; ++j) col[j] = epi.col(blockIdx.z, n0 + wn * TN * 16 + j * 32 + q * 8);
    };
    auto read_rows = [&](int i0) {
        if (WAVES_K > 1 && group > 0) return;
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int m = m0 + (wm * TM + i0 + k) * 16 + r;
            if (m >= g.M) continue;
            row[k] = epi.row(blockIdx.z, m);
#pragma unroll
            for (int j = 0; j < TN / 2; ++j) {
                const int n = n0 + wn * TN * 16 + j * 32 + q * 8;
                if (n < g.N) pre[k][j] = epi.pre(blockIdx.z, m, n);
            }
        }
    };
    if (EARLY) {
        read_col(), read_rows(0);
        // nothing of it may come behind the loads of the stages: the waits count those
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int s = 0; s < STAGES; ++s)
        if (s < steps) {
            before_loads(s);
#pragma unroll
            for (int i = 0; i < LOADS; ++i) load(i, s, s * STAGE);
            after_loads();
        }
    if (steps >= STAGES) wait_barrier<(STAGES - 1) * LOADS>();
    else wait_barrier<0>();
#pragma unroll
    for (int i = 0; i < (SPLIT ? 1 : TM); ++i) reada(a0, i, i, 0, 0);
#pragma unroll
    for (int j = 0; j < TN; ++j) readb(b0, j, 0, 0);
    if constexpr (SPLIT) {
        reada(a1, 0, 0, 0, 1);
#pragma unroll
        for (int j = 0; j < TN; ++j) readb(b1, j, 0, 1);
    }
    int at = 0;
    auto step = [&](int s, auto more) {                    // more: stage s + STAGES exists
        const int ahead = next(at);
        __builtin_amdgcn_s_waitcnt(0xc07f);                // lgkmcnt(0): the first fragments
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            read_part(a1, b1, i, at, 1);
            mul(a0, b0, i);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (more.value) {
            wait_barrier<(STAGES - 2) * LOADS>();
            before_loads(s + STAGES);
        } else {
            wait_barrier<0>();                             // the last stages: nothing newer is in flight
        }
        auto load_part = [&](int i) {
            if constexpr (more.value) {
#pragma unroll
                for (int k = i * LOADS_ROW; k < (i + 1) * LOADS_ROW; ++k)
                    if (k < LOADS) load(k, s + STAGES, at);
            }
        };
        // behind the last step the reads for the next one find an old stage, and nobody uses them
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            load_part(i);
            read_part(a0, b0, i, ahead, 0);
            mul(a1, b1, i);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (more.value) after_loads();
        at = ahead;
    };
    // The split form needs both halves of both operands at once.  The B fragments of a step stay in registers; the A
    // fragments of block row i + 1 are read while row i is multiplied; in front of the last row everything of this stage
    // has been read, and behind each of its blocks that block's B fragments of the next step are.
    auto step_split = [&](int s, auto more) {
        const int ahead = next(at);
#pragma unroll
        for (int i = 0; i < TM - 1; ++i) {
            reada(a0, (i + 1) & 1, i + 1, at, 0);
            reada(a1, (i + 1) & 1, i + 1, at, 1);
            mul3(i, 0, TN);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (more.value) {
            wait_barrier<(STAGES - 2) * LOADS>();
            before_loads(s + STAGES);
#pragma unroll
            for (int k = 0; k < LOADS; ++k) load(k, s + STAGES, at);
            after_loads();
        } else {
            wait_barrier<0>();
        }
        reada(a0, 0, 0, ahead, 0);
        reada(a1, 0, 0, ahead, 1);
#pragma unroll
        for (int j = 0; j < TN; j += 2) {
            mul3(TM - 1, j, 2);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = j; k < j + 2; ++k) readb(b0, k, ahead, 0), readb(b1, k, ahead, 1);
        }
        at = ahead;
    };
    int s = 0;
    if constexpr (SPLIT) {
        for (; s + STAGES < steps; ++s) step_split(s, Yes{});
        for (; s < steps; ++s) step_split(s, No{});
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] += cross[i][j] * (1.f / REST);
    } else {
        for (; s + STAGES < steps; ++s) step(s, Yes{});
        for (; s < steps; ++s) step(s, No{});
    }
    if constexpr (WAVES_K > 1) {                           // the groups' sums meet in the first one, in order
        static_assert((WAVES_K - 1) * BM * BN * 4 <= STAGES * STAGE, "the partial tiles fit into LDS");
        typedef typename Acc<KIND>::type V;
        V *parts = (V *)smem;
        __syncthreads();
        if (group > 0) {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) parts[(((group - 1) * WAVES + wave) * TM * TN + i * TN + j) * 64 + lane] = acc[i][j];
        }
        __syncthreads();
        if (group > 0 && !Epilogue::TURNED) return;
        if (group == 0) {
#pragma unroll
            for (int k = 0; k < WAVES_K - 1; ++k)
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j) acc[i][j] += parts[((k * WAVES + wave) * TM * TN + i * TN + j) * 64 + lane];
        }
    }
    if (!EARLY) read_col();
    const bool turn = Epilogue::TURNED && !(g.lower && tm == tn);
#pragma unroll
    for (int i0 = 0; i0 < TM; i0 += AHEAD) {
        if (!EARLY) read_rows(i0);
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int i = i0 + k, m = m0 + (wm * TM + i) * 16 + r;
#pragma unroll
            for (int j = 0; j < TN / 2; ++j) {
                const int n = n0 + wn * TN * 16 + j * 32 + q * 8;
                float v[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = (float)acc[i][2 * j][e], v[4 + e] = (float)acc[i][2 * j + 1][e];
                if (WAVES_K > 1 && group > 0) continue;
                if (m < g.M && n < g.N) {
                    epi.put(blockIdx.z, m, n, v, row[k], col[j], pre[k][j]);
                } else if (Epilogue::TURNED) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = 0.f;    // zeros behind the rows of the turned tile
                }
                if constexpr (Epilogue::TURNED) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][2 * j][e] = v[e], acc[i][2 * j + 1][e] = v[4 + e];
                }
            }
            if (Epilogue::TURNED) __builtin_amdgcn_sched_barrier(0);
        }
    }
    // The tile once more, turned: through LDS (free now), as fp16 rows of BM values along m, a pass for each half of the
    // split form.
    if constexpr (Epilogue::TURNED) {
        if (!turn) return;
        constexpr int CHUNKS = BM / 8;
        _Float16 *t = (_Float16 *)smem, *mine_t = t + (wn * TN * 16 + q * 8) * PITCH + wm * TM * 16 + r;
#pragma unroll 1
        for (int half = 0; half < (SPLIT ? 2 : 1); ++half) {
            __syncthreads();
            if (WAVES_K == 1 || group == 0) {
#pragma unroll
                for (int i = 0; i < TM; ++i) {
#pragma unroll
                    for (int j = 0; j < TN; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float v = acc[i][j][e];
                            if (SPLIT) {
                                asm volatile("" : "+v"(v));    // nothing of one pass is kept for the other: registers
                                if (half) v = (v - (float)(_Float16)v) * REST;
                            }
                            mine_t[((j >> 1) * 32 + (j & 1) * 4 + e) * PITCH + i * 16] = (_Float16)v;
                        }
                    __builtin_amdgcn_sched_barrier(0);         // one block row's conversions at a time: registers
                }
            }
            __syncthreads();
            for (int k = threadIdx.x; k < BN * CHUNKS; k += 64 * WAVES * WAVES_K) {
                const int nl = k / CHUNKS, c = k - nl * CHUNKS;
                if (n0 + nl < g.N && m0 + c * 8 < g.M) epi.put_turned(blockIdx.z, n0 + nl, m0 + c * 8, half, *(const f16x8 *)(t + nl * PITCH + c * 8));
            }
        }
    }
}

template <int KIND, int BM, int BN, int WAVES_M, int WAVES_N, int WAVES_K, int STAGES, class Epilogue>
static __global__ __launch_bounds__(64 * WAVES_M *WAVES_N *WAVES_K) void k_gemm(Args g, Epilogue epi) {
    gemm_tile<KIND, BM, BN, WAVES_M, WAVES_N, WAVES_K, STAGES>(g, epi);
}

// ---- host side -------------------------------------------------------------------------
template <int KIND, int BM, int BN, int WAVES_M, int WAVES_N, int WAVES_K, int STAGES, class Epilogue>
static int launch(Args g, int batch, const Epilogue &epi, hipStream_t st) {
    g.tiles_m = (g.M + BM - 1) / BM;
    g.tiles_n = (g.N + BN - 1) / BN;
    const int64_t tiles = tiles_of(g);
    DPD_REQUIRE(tiles * 64 * WAVES_M * WAVES_N * WAVES_K <= UINT32_MAX, DPD_ERR_SHAPE, "a product of %d x %d results is too large for one call", g.M, g.N);
    hipLaunchKernelGGL((k_gemm<KIND, BM, BN, WAVES_M, WAVES_N, WAVES_K, STAGES, Epilogue>), dim3((unsigned)tiles, 1, (unsigned)batch),
                       dim3(64 * WAVES_M * WAVES_N * WAVES_K), 0, st, g, epi);
    DPD_LAUNCH_CHECK();
    return DPD_OK;
}

// Which tile: the one whose rounds over the 256 compute units are estimated to take least.  A round has one workgroup on
// every compute unit, or two where 80 KB of LDS hold one; it takes steps * per + fixed.  Measured with full rounds of 1024 to
// 4096 rows, fp16 operands (int8 and bf16 take the same time a step) and the split form, us; the fixed part of the fourth one's
// split form with an epilogue that stores both orientations (3 x 777 x 1000: 30.4 us, 27.6 with the fifth).  The lines were
// fitted at 12 steps and more and say too little for fewer.  Iterations in the split form with every tile forced in turn, us,
// the rule's against the best: 3 of 777 x 1000 325, 303; 1024 x 4096 408, 405; 2048 x 2048 754, 749; 4096 x 4096 4258, 4086; 8 of
// 500 x 700 286, 275; 300 x 400 122, 102.
struct Round {
    float per, fixed;
};
struct Tile {
    int bm, bn;
    Round one, two;              // one and two workgroups on a compute unit (per == 0: does not fit)
    Round split_one, split_two;
};
constexpr Tile TILES[] = {
    {256, 256, {1.35f, 10.f}, {}, {}, {}},                                    // no registers for two accumulators: not split
    {256, 128, {0.885f, 6.4f}, {}, {1.28f, 4.8f}, {}},
    {192, 192, {0.94f, 7.f}, {}, {}, {}},                                     // nor this one
    {128, 128, {0.48f, 4.4f}, {}, {0.615f, 7.5f}, {}},
    {128, 128, {0.685f, 1.2f}, {0.904f, 5.6f}, {0.7f, 4.f}, {1.33f, 2.2f}},
    {128, 64, {0.32f, 3.1f}, {0.565f, 3.8f}, {0.4175f, 2.8f}, {0.7075f, 4.1f}},
    {96, 96, {0.29f, 4.f}, {}, {}, {}},                                       // an odd number of block rows a wave: not split
    {64, 64, {0.19f, 3.1f}, {}, {0.2475f, 2.9f}, {}},
    {64, 64, {0.208f, 2.9f}, {0.377f, 2.6f}, {0.35f, 0.5f}, {0.39f, 3.8f}},
    {64, 32, {0.131f, 2.9f}, {}, {0.131f, 3.2f}, {}},
    {32, 32, {0.071f, 3.2f}, {}, {0.08f, 3.2f}, {}},
};

static inline int best_tile(const Args &g, int batch, bool split) {
    int best = -1;
    float least = 0.f;
    static_assert(sizeof(TILES) / sizeof(TILES[0]) == 11, "product_tile names every tile");
    if (g_product_tile >= 0) {
        const Tile &t = TILES[g_product_tile];
        if (!(g.lower && t.bm != t.bn) && (split ? t.split_one : t.one).per > 0.f) return g_product_tile;
    }
    for (int i = 0; i < (int)(sizeof(TILES) / sizeof(TILES[0])); ++i) {
        const Tile &t = TILES[i];
        const Round one = split ? t.split_one : t.one, two = split ? t.split_two : t.two;
        if ((g.lower && t.bm != t.bn) || one.per == 0.f) continue;
        Args a = g;
        a.tiles_m = (g.M + t.bm - 1) / t.bm, a.tiles_n = (g.N + t.bn - 1) / t.bn;
        const int64_t tiles = tiles_of(a) * batch, size = two.per > 0.f ? 512 : 256, rest = tiles % size;
        const float c1 = (float)g.steps * one.per + one.fixed, c2 = (float)g.steps * two.per + two.fixed;
        const float cost = (float)(tiles / size) * (size == 512 ? c2 : c1) + (rest == 0 ? 0.f : rest > 256 ? c2 : c1);
        if (best < 0 || cost < least) best = i, least = cost;
    }
    return best;
}

template <int KIND, class Epilogue>
static int product(const Args &g, int batch, const Epilogue &epi, hipStream_t st) {
    constexpr bool SPLIT = KIND == F16_SPLIT;
    const int tile = best_tile(g, batch, SPLIT);
    if constexpr (!SPLIT) {
        if (tile == 0) return launch<KIND, 256, 256, 2, 4, 1, 2>(g, batch, epi, st);
        if (tile == 2) return launch<KIND, 192, 192, 4, 2, 1, 3>(g, batch, epi, st);
        if (tile == 6) return launch<KIND, 96, 96, 2, 3, 2, 3>(g, batch, epi, st);
    }
    switch (tile) {
    case 1: return launch<KIND, 256, 128, 4, 2, 1, 3>(g, batch, epi, st);
    case 3: return launch<KIND, 128, 128, 2, SPLIT ? 2 : 4, SPLIT ? 2 : 1, SPLIT ? 2 : 4>(g, batch, epi, st);
    case 4: return launch<KIND, 128, 128, 2, 4, 1, 2>(g, batch, epi, st);
    case 5: return launch<KIND, 128, 64, 2, 2, 1, 3>(g, batch, epi, st);
    case 7: return launch<KIND, 64, 64, 2, 2, 2, 4>(g, batch, epi, st);
    case 8: return launch<KIND, 64, 64, 2, 2, SPLIT ? 2 : 1, SPLIT ? 2 : 4>(g, batch, epi, st);
    case 9: return launch<KIND, 64, 32, 2, 1, 4, 3>(g, batch, epi, st);
    default: return launch<KIND, 32, 32, 1, 1, 4, 3>(g, batch, epi, st);
    }
}

// A row of an operand may have at most this many bytes: 256 rows of a tile stay inside 32-bit offsets.
constexpr int64_t MAX_ROW_BYTES = (1 << 23) - 128;

static inline int64_t pad_to(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

}  // namespace nt

// ---- element types of the entry points ----------------------------------------------------

template <class T>
DEV float to_f32(T v) { return (float)v; }
template <class T>
DEV T from_f32(float v) { return (T)v; }           // round to nearest even

// One value of a tensor whose type is known at run time only.
DEV float load_any(const void *p, int type, int64_t i) {
    return type == DPD_F32 ? ((const float *)p)[i] : type == DPD_BF16 ? (float)((const __bf16 *)p)[i] : (float)((const _Float16 *)p)[i];
}

// Eight consecutive values of one row, the first `valid` of them; `whole`: the row's address is aligned for 16-byte
// stores at every multiple of eight elements.
template <class T>
DEV void store8(T *p, const float *v, int valid, bool whole) {
    if (whole && valid >= 8) {
        if constexpr (sizeof(T) == 4) {
            *(f32x4_t *)p = f32x4_t{v[0], v[1], v[2], v[3]};
            *((f32x4_t *)p + 1) = f32x4_t{v[4], v[5], v[6], v[7]};
        } else {
            typedef T T8 __attribute__((ext_vector_type(8)));
            T8 o;
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = from_f32<T>(v[i]);
            *(T8 *)p = o;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < valid) p[i] = from_f32<T>(v[i]);
    }
}
template <class T>
DEV void load8(const T *p, float *v, int valid, bool whole) {
    if (whole && valid >= 8) {
        if constexpr (sizeof(T) == 4) {
            const f32x4_t a = *(const f32x4_t *)p, b = *((const f32x4_t *)p + 1);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
        } else {
            typedef T T8 __attribute__((ext_vector_type(8)));
            const T8 a = *(const T8 *)p;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = to_f32(a[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < valid ? to_f32(p[i]) : 0.f;
    }
}
struct None {};

static inline int type_size(int type) { return type == DPD_F32 ? 4 : 2; }

// Calls f with a value of the element type that `type` names.
template <class F>
static int with_type(int type, F f) {
    if (type == DPD_F32) return f(float{});
    if (type == DPD_BF16) return f(__bf16{});
    return f(_Float16{});
}
