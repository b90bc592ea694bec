// dimn_xent.h -- softmax cross entropy of a linear output layer, in pieces of the classes, the logits never kept (gfx950).
//
//   z = x W + b,  lse = log sum_v exp z_v
//   label y:    loss = lse - z_y                          G_v = dloss (exp(z_v - lse) - [v = y])
//   profile t:  loss = sum_v t_v lse - sum_v t_v z_v       G_v = dloss (sum(t) exp(z_v - lse) - t_v)
//   dx = G W^T,  dW = x^T G,  db = sum over rows of G
//
// Everything is one matrix product with different epilogues (k_xent_gemm): C[m][n] = sum_k A[m][k] B[n][k], both operands bfloat16 and
// k-contiguous, float32 accumulation on the bf16 matrix cores.
//   * Forward: A = rows, B = classes.  A workgroup leaves the running maximum and the sum of exponentials of each row over its classes (8 bytes
//     for 256 logits), k_xent_lse joins them.
//   * Backward, per piece of the classes: the logits again, G of the piece in the epilogue -- kept in both memory orders, because each of the
//     two products that read it wants its own inner dimension contiguous --, then dx += G W^T and dW = x^T G of the piece.
//   * float32 operands are split into three bfloat16 terms each (8 + 8 + 8 bits of the 24-bit significand; exact from 2^-110 up), and the six products whose
//     weight is 2^-16 or more are summed: what is left out is below 2^-23 of a product, the rounding of a float32 product itself.  Six passes
//     of the bf16 matrix cores still have 2.7 times the rate of the float32 ones.
//   * Operands that are k-contiguous, aligned and a multiple of 64 long are read in place; everything else is laid out by k_xent_lay.
//   * Of bfloat16 operands G is rounded to bfloat16 too (half a step, 2^-8 of it): it is the operand of two more products, and three planes of it would
//     cost three passes each where x and the kernel hold eight bits themselves.  float32 G keeps its three planes.
// Measured, bfloat16: 4096 x 2048 x 100000 forward 1.38-1.45 ms (1.16-1.2 PFLOP/s; the library's product of the same sizes alone: 1.2);
// 4096 x 2048 x 64000 backward 3.0 ms: logits again 1.10, dx 0.90, dW 0.88 (1.0-1.2 PFLOP/s), layouts 0.11.  float32 1024 x 1024 x 20000: 264 us forward
// (layouts 35, product 224), 159 TFLOP/s (the float32 matrix instructions reach 154 in a product without a softmax behind it); backward 925 us.
#pragma once
#include <type_traits>

#include "dimn_rowops.h"

namespace rowops {

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x4u __attribute__((ext_vector_type(4), aligned(2)));

__device__ __forceinline__ uint16_t to_bf16(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }
__device__ __forceinline__ float from_bf16(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }

// The next term of a float32 number in bfloat16 terms, the first of three unless it is the `last`; what is left of the number stays in `rest`: three
// terms hold every finite one of 2^-110 or more exactly.  Values within half a step of the largest float32 would round to an infinity and take the largest bfloat16
// instead; the remainders are exact either way (Sterbenz; above, 16 bits are left).
// An infinity is the LAST term, its sign the others: so it is multiplied by the other operand's first term alone, which has the operand's own sign
// and is 0 where the operand is.  As the first term it would also meet the second and third ones, which are 0 or have the other sign, and make a
// NaN of inf x 0.5.  What its other terms add is finite and has the sign of the result.  A NaN is every term.
__device__ __forceinline__ uint16_t split_term(float& rest, bool last) {
    if (last) return to_bf16(rest);
    constexpr float top = 3.38953139e38f;                        // (2 - 2^-7) 2^127
    const float size = fabsf(rest);
    const bool inf = size == INFINITY;
    const uint16_t b = to_bf16(inf || size > top ? copysignf(inf ? 1.f : top, rest) : rest);
    rest = inf ? rest : rest - from_bf16(b);
    return b;
}
__device__ __forceinline__ void split3(float x, uint16_t (&b)[3]) {
#pragma unroll
    for (int pl = 0; pl < 3; ++pl) b[pl] = split_term(x, pl == 2);
}

// The rows of a batch that have a gradient: those whose label is a class (profiles: dloss is 0 where all weights are) and whose dloss is not 0.  The
// G of the others is 0, but x may hold anything there, NaN too (padding), and 0 x NaN would reach dW: x^T G takes their x as zeros.
enum { XT_I32 = 0, XT_I64 = 1, XT_F32 = 2, XT_BF16 = 3 };        // DIMN_TARGET_*
// look() only loads, without a branch or a use of what it loads, so that other loads can follow before has() waits.
struct LiveRows {
    const float* dloss;
    const char* label; uint32_t step, high_at, high;      // the labels' words: bytes between them, to the upper one, and its mask; profiles: dloss again
    uint32_t last;                                         // the last class; profiles: every word passes
    struct Row { uint32_t low, high; float dloss; };
    __device__ __forceinline__ Row look(uint32_t row) const {                 // (rows: up to 2^22, so the offsets take 32 bits)
        return {*(const uint32_t*)(label + row * step), *(const uint32_t*)(label + high_at + row * step), *(const float*)((const char*)dloss + row * 4)};
    }
    __device__ __forceinline__ bool has(const Row& r) const { return (r.dloss != 0.f) & (r.low <= last) & ((r.high & high) == 0); }
};

// ---- operand layout -----------------------------------------------------------------------------------------------------------
// to[plane][r][k] = bfloat16 term `plane` of from[r][k], zero for cols <= k < ldk (ldk: a multiple of 64).  T = float: three planes, T = bf16_t: one.
// Copying bounds both; everything moves in 16-byte pieces (64000 x 2048 and 4096 x 2048 bfloat16 transposed: 558 MB in 113 us, 4.9 TB/s).
template <typename T> struct Eight { typedef uint16_t vec __attribute__((ext_vector_type(8), aligned(2))); };
template <> struct Eight<float> { typedef float vec __attribute__((ext_vector_type(8), aligned(4))); };
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

template <typename T>
__device__ __forceinline__ void lay_store(const T (&v)[8], uint16_t* to, int64_t plane) {
    constexpr int PL = sizeof(T) == 4 ? 3 : 1;
    u16x8 o[PL];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if constexpr (PL == 3) {
            uint16_t b[3];
            split3(v[j], b);
            o[0][j] = b[0]; o[1][j] = b[1]; o[2][j] = b[2];
        } else o[0][j] = v[j];
    }
#pragma unroll
    for (int pl = 0; pl < PL; ++pl) *(u16x8*)(to + pl * plane) = o[pl];
}
// One operand to lay out.  Not transposed: from is [r][k] with k contiguous, a thread takes eight k's.  Transposed: from is [k][r] with r contiguous
// (row stride `ld` along k), 64 x 64 tiles through LDS, whose line of 65 (float) / 66 (bfloat16) elements spreads a column over the banks.
// `live`: the k's are rows of the batch, and one without a gradient is laid out as zeros.
struct LayJob {
    const void* from; int64_t ld, rows, cols;
    uint16_t* to; int64_t ldk, plane;
    int32_t transposed, blocks, live;
};
struct LayJobs { LayJob job[4]; int32_t n, first; LiveRows rows; };                    // (one launch for everything a piece needs: each is a few microseconds of copying)
template <typename T>
__global__ __launch_bounds__(256) void k_xent_lay(const LayJobs all) {
    constexpr int LD = sizeof(T) == 4 ? 65 : 66;
    __shared__ T tile[64][LD];
    int block = blockIdx.x + all.first, w = 0;
    while (w + 1 < all.n && block >= all.job[w].blocks) { block -= all.job[w].blocks; ++w; }
    const LayJob& p = all.job[w];
    const T* from = (const T*)p.from;
    if (!p.transposed) {
        const int64_t e = ((int64_t)block * 256 + threadIdx.x) * 8;
        if (e >= p.rows * p.ldk) return;
        const int64_t r = e / p.ldk, k = e - r * p.ldk;
        const T* q = from + r * p.ld + k;
        T v[8];
        if (k + 8 <= p.cols) {
            const typename Eight<T>::vec x = *(const typename Eight<T>::vec*)q;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = x[j];
        } else
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = k + j < p.cols ? q[j] : (T)0;
        lay_store<T>(v, p.to + e, p.plane);
        return;
    }
    const int64_t tiles_k = p.ldk >> 6;
    const int64_t tr = block / tiles_k, tk = block - tr * tiles_k;
    const int64_t r0 = tr * 64, k0 = tk * 64;
    const int q = threadIdx.x & 7, s = threadIdx.x >> 3;         // 8 pieces of eight x 32 lines
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int64_t k = k0 + s + 32 * i, r = r0 + 8 * q;
        const T* f = from + k * p.ld + r;
        T v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        LiveRows::Row row = {0, 0, 1.f};
        if (p.live) row = all.rows.look((uint32_t)(k < p.cols ? k : p.cols - 1));
        if (k < p.cols) {
            if (r + 8 <= p.rows) {
                const typename Eight<T>::vec x = *(const typename Eight<T>::vec*)f;
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = x[j];
            } else
#pragma unroll
                for (int j = 0; j < 8; ++j) if (r + j < p.rows) v[j] = f[j];
        }
        const bool live = !p.live || all.rows.has(row);
#pragma unroll
        for (int j = 0; j < 8; ++j) tile[s + 32 * i][8 * q + j] = live ? v[j] : (T)0;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int64_t r = r0 + s + 32 * i;
        if (r >= p.rows) continue;
        T v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = tile[8 * q + j][s + 32 * i];
        lay_store<T>(v, p.to + r * p.ldk + k0 + 8 * q, p.plane);
    }
}

// ---- the product --------------------------------------------------------------------------------------------------------------
struct XentGemm {
    const uint16_t* A; const uint16_t* B;      // [plane][m][lda], [plane][n][ldb]; 16-byte aligned, lda / ldb multiples of 8
    int64_t lda, ldb, a_plane, b_plane;
    int32_t M, N;                              // columns from N on are not classes / not stored
    int32_t ksteps;                            // steps of the inner dimension: 64 deep (one plane) / 32 deep (three)
    int32_t tiles_m, tiles_n;
    // epilogues over logits: z = C + bias
    const float* bias;                         // [N] or NULL
    const void* target; int64_t target_row;    // labels (int32 / int64 [M]), or a profile [M][..] of float32 / bfloat16 (class 0 of the piece first)
    int32_t target_kind;
    int64_t class0, classes;                   // first class of the piece; classes in all
    // forward
    float2* part;                              // [tiles_n][M]: (maximum, sum of exp(z - maximum))
    float2* part_t;                            // profile: [tiles_n][M]: (sum of t, sum of t z)
    float* picked;                             // labels: [M], z of the label, written by the workgroup that holds it
    // G
    const float* lse; const float* dloss;      // [M]
    const float* tsum;                         // profile: [M]
    uint16_t* G; int64_t ldg, g_plane;         // [plane][M][ldg], columns N .. ldg zero
    uint16_t* GT; int64_t ldgt, gt_plane;      // [plane][N][ldgt], columns M .. ldgt zero
    float* dbias_part; int64_t dbias_ld;       // [WM tiles_m][dbias_ld]: column sums of G over the rows of one wave row (WM of them per tile)
    // result
    void* C; int64_t ldc;                      // epilogue 2: C[m][n], float32 (three planes) or bfloat16 (one)
    float* acc; int64_t acc_split; int32_t acc_first;   // epilogue 3: acc[split][M][N] (+)= C
};
enum { XE_LSE = 0, XE_GRAD = 1, XE_STORE = 2, XE_ADD = 3 };

__device__ __forceinline__ int64_t xent_label(const XentGemm& p, int64_t row) {
    return p.target_kind == XT_I64 ? ((const int64_t*)p.target)[row] : (int64_t)((const int32_t*)p.target)[row];
}
// four consecutive entries of a profile row, 0 from `n` on
__device__ __forceinline__ f32x4 xent_profile4(const void* target, int32_t kind, int64_t ld, int64_t row, int64_t col, int64_t n) {
    f32x4 t = {0.f, 0.f, 0.f, 0.f};
    if (kind == XT_F32) {
        const float* q = (const float*)target + row * ld + col;
        if (col + 4 <= n) t = *(const f32x4u*)q;
        else
#pragma unroll
            for (int r = 0; r < 4; ++r) if (col + r < n) t[r] = q[r];
    } else {
        const uint16_t* q = (const uint16_t*)target + row * ld + col;
        if (col + 4 <= n) {
            const u16x4u v = *(const u16x4u*)q;
#pragma unroll
            for (int r = 0; r < 4; ++r) t[r] = from_bf16(v[r]);
        } else
#pragma unroll
            for (int r = 0; r < 4; ++r) if (col + r < n) t[r] = from_bf16(q[r]);
    }
    return t;
}

typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) const void global_void;

// Tile BM x BN per workgroup, WM x WN waves; k in steps of 64 (PL = 1: bfloat16) or 32 (PL = 3: all three planes of both operands, six products), two
// stages of LDS filled by 16-byte DMA while the other one is multiplied, one barrier per step.  The matrix instruction takes B's rows as its rows and
// A's as its columns, and fragment i / j of a wave holds rows FM q + i of A, 4 FN (q >> 2) + 4 j + (q & 3) of B (q: the instruction's index): a lane
// then owns FM consecutive m's x 4 FN consecutive n's of C.  Sums along n are mostly inside a lane, results leave in 16-byte pieces in BOTH memory
// orders, and G needs no transposition.
// LDS holds the rows in fragment order (row 16 f + q of a wave's part), 128 / 64 bytes each, the 16-byte pieces of a row turned by its number: the
// rows a fragment reads at once are neighbours on different banks, and every address is one register plus a constant.  The DMA writes LDS in lane
// order, so order and turn are made on the global side.
template <int BM, int BN, int WM, int WN, int EPI, int PL>
__global__ __launch_bounds__(64 * WM * WN) void k_xent_gemm(const XentGemm p) {
    constexpr int NW = WM * WN, TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16, ROWS = BM + BN;
    constexpr int DEEP = PL == 1 ? 64 : 32, PIECES = DEEP / 8, LINE = 64 / PIECES;      // k's per step; pieces per row; rows per request
    constexpr int LOADS = PL * ROWS / LINE / NW;
    static_assert(LOADS * LINE * NW == PL * ROWS && BM % LINE == 0, "whole requests per wave");
    __shared__ __attribute__((aligned(1024))) uint16_t lds[2][PL * ROWS * DEEP];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN, li = lane & 15, lj = lane >> 4;
    auto turn = [](int row) { return PL == 1 ? row & 7 : (row >> 2) & 3; };
    // Workgroup b runs on XCD b % 8: each XCD gets a consecutive range of the tiles, ordered in columns of four m tiles, so that the 32
    // workgroups of an XCD at a time share four A and eight B tiles in its L2 (columns of 8: 1 % more time, of 16: 4 %).
    int tile;
    {
        const int total = p.tiles_m * p.tiles_n, b = blockIdx.x, x = b & 7, q = total >> 3, rem = total & 7;
        tile = x * q + (x < rem ? x : rem) + (b >> 3);
    }
    int tm, tn;
    {
        const int per = 4 * p.tiles_n, grp = tile / per, in = tile - grp * per;
        const int h = p.tiles_m - grp * 4 < 4 ? p.tiles_m - grp * 4 : 4;
        tn = in / h;
        tm = grp * 4 + in - tn * h;
    }
    const int m0 = tm * BM, n0 = tn * BN;
    // request c of this wave brings lines [LINE (wave LOADS + c), + LINE) of the stacked planes of [A; B]
    uint32_t off[LOADS];
    auto line_of = [&](int c) { return (wave * LOADS + c) * LINE; };
#pragma unroll
    for (int c = 0; c < LOADS; ++c) {
        const int pos = line_of(c) % ROWS + lane / PIECES;
        const bool isA = line_of(c) % ROWS < BM;
        const int t = isA ? pos : pos - BM, q = t & 15, f = t >> 4;
        int r = isA ? f / FM * TM + q * FM + f % FM : f / FN * TN + (q >> 2) * 4 * FN + 4 * (f % FN) + (q & 3);
        const int piece = (lane % PIECES) ^ turn(t);
        const int lim = isA ? p.M - 1 - m0 : p.N - 1 - n0;       // rows past the end read the last one: their results are never used
        r = r < lim ? r : lim;
        off[c] = (uint32_t)((int64_t)r * (isA ? p.lda : p.ldb) * 2 + piece * 16);
    }
    const char* Abase = (const char*)(p.A + (int64_t)m0 * p.lda);
    const char* Bbase = (const char*)(p.B + (int64_t)n0 * p.ldb);
    const int S = gridDim.y, sp = blockIdx.y;
    const int tbeg = (int)((int64_t)p.ksteps * sp / S), tend = (int)((int64_t)p.ksteps * (sp + 1) / S);
    auto request = [&](int stage, int t) {
        const char* a = Abase + (int64_t)t * (DEEP * 2);
        const char* b = Bbase + (int64_t)t * (DEEP * 2);
#pragma unroll
        for (int c = 0; c < LOADS; ++c) {
            const int plane = line_of(c) / ROWS;
            const bool isA = line_of(c) % ROWS < BM;
            const char* from = isA ? a + plane * p.a_plane * 2 : b + plane * p.b_plane * 2;
            __builtin_amdgcn_global_load_lds((global_void*)(from + off[c]), (lds_void*)&lds[stage][line_of(c) * DEEP], 16, 0, 0);
        }
    };
    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    // fragment f of a part that starts at LDS row `row0` of `plane`, k's 32 kk ..
    auto fragment = [&](int stage, int plane, int row0, int f, int kk) {
        return *(const bf8*)&lds[stage][(plane * ROWS + row0 + 16 * f + li) * DEEP + (((kk * 4 + lj) ^ turn(li)) << 3)];
    };
    auto multiply = [&](int stage) {
        if constexpr (PL == 1) {
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                bf8 a[FM], b[FN];
#pragma unroll
                for (int j = 0; j < FN; ++j) b[j] = fragment(stage, 0, BM + wn * TN, j, kk);
#pragma unroll
                for (int i = 0; i < FM; ++i) a[i] = fragment(stage, 0, wm * TM, i, kk);
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[j], a[i], acc[i][j], 0, 0, 0);
            }
        } else {
            bf8 a[PL][FM], b[PL][FN];
            auto add = [&](const bf8 (&u)[FM], const bf8 (&v)[FN]) {
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[j], u[i], acc[i][j], 0, 0, 0);
            };
#pragma unroll
            for (int s = 0; s < PL; ++s) {
#pragma unroll
                for (int j = 0; j < FN; ++j) b[s][j] = fragment(stage, s, BM + wn * TN, j, 0);
#pragma unroll
                for (int i = 0; i < FM; ++i) a[s][i] = fragment(stage, s, wm * TM, i, 0);
                // (0,0); (0,1) (1,0) (1,1); (0,2) (2,0)
                add(a[0], b[s]);
                if (s > 0) add(a[s], b[0]);
                if (s == 1) add(a[1], b[1]);
            }
        }
    };
    if (tbeg < tend) request(0, tbeg);
    int stage = 0;
    for (int t = tbeg; t + 1 < tend; ++t) {
        __syncthreads();                                         // the stage's bytes have landed (the barrier waits for this wave's requests first) and
        request(stage ^ 1, t + 1);                               // everybody is done with the other stage
        multiply(stage);
        stage ^= 1;
        // Fragments are read one group of products ahead of their use: left alone, the compiler reads two, waits, and multiplies (4-6 % slower)
        if constexpr (PL == 1) {
            constexpr int GROUP = (2 * FM + FN - 2) / (FM - 2);
            __builtin_amdgcn_sched_group_barrier(0x100, FN + 2, 0);
#pragma unroll
            for (int q = 0; q < FM - 2; ++q) {
                __builtin_amdgcn_sched_group_barrier(0x100, GROUP, 0);
                __builtin_amdgcn_sched_group_barrier(0x8, 2 * FN, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x8, 4 * FN, 0);
        } else {
            __builtin_amdgcn_sched_group_barrier(0x100, FM + FN, 0);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                __builtin_amdgcn_sched_group_barrier(0x100, FN, 0);
                __builtin_amdgcn_sched_group_barrier(0x8, FM * FN, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, FM, 0);
                __builtin_amdgcn_sched_group_barrier(0x8, FM * FN, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x8, 2 * FM * FN, 0);
        }
    }
    if (tbeg < tend) {
        __syncthreads();
        multiply(stage);
    }
    // this lane's results: C[mb + i][nb + 4 j + r] in acc[i][j][r]
    const int mb = m0 + wm * TM + li * FM, nb = n0 + wn * TN + lj * 4 * FN;
    if constexpr (EPI == XE_STORE || EPI == XE_ADD) {
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const int64_t m = mb + i;
            if (m >= p.M) continue;
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                const int n = nb + 4 * j;
                if (n >= p.N) continue;
                const f32x4 v = acc[i][j];
                if constexpr (EPI == XE_ADD) {
                    float* q = p.acc + (int64_t)sp * p.acc_split + m * p.N + n;
                    if (n + 4 <= p.N) *(f32x4u*)q = p.acc_first ? v : *(const f32x4u*)q + v;
                    else
#pragma unroll
                        for (int r = 0; r < 4; ++r) if (n + r < p.N) q[r] = p.acc_first ? v[r] : q[r] + v[r];
                } else if constexpr (PL == 3) {
                    float* q = (float*)p.C + m * p.ldc + n;
                    if (n + 4 <= p.N) *(f32x4u*)q = v;
                    else
#pragma unroll
                        for (int r = 0; r < 4; ++r) if (n + r < p.N) q[r] = v[r];
                } else {
                    uint16_t* q = (uint16_t*)p.C + m * p.ldc + n;
                    u16x4u o;
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[r] = to_bf16(v[r]);
                    if (n + 4 <= p.N) *(u16x4u*)q = o;
                    else
#pragma unroll
                        for (int r = 0; r < 4; ++r) if (n + r < p.N) q[r] = o[r];
                }
            }
        }
        return;
    }
    if constexpr (EPI == XE_LSE || EPI == XE_GRAD) {
        // (__expf rounds its scaled argument, 2^-24 |d| of the result: far below a bfloat16 operand's half step, too much for float32 results)
        auto power = [](float d) { if constexpr (PL == 1) return __expf(d); else return expf(d); };
        const bool labels = p.target_kind <= XT_I64;
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            f32x4 b = {0.f, 0.f, 0.f, 0.f};
            const int n = nb + 4 * j;
            if (p.bias) {
                if (n + 4 <= p.N) b = *(const f32x4u*)(p.bias + n);
                else
#pragma unroll
                    for (int r = 0; r < 4; ++r) if (n + r < p.N) b[r] = p.bias[n + r];
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (n + r >= p.N) b[r] = -INFINITY;              // no class: no probability
#pragma unroll
                for (int i = 0; i < FM; ++i) acc[i][j][r] += b[r];
            }
        }
        if constexpr (EPI == XE_LSE) {
            float2* red = (float2*)&lds[0][0];                   // [WN][BM] (maximum, sum), then [WN][BM] (sum t, sum t z)
            __syncthreads();
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                const int mr = wm * TM + li * FM + i;
                const int64_t m = m0 + mr;
                const bool mine = m < p.M;
                float top = -INFINITY, s = 0.f;
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) top = fmaxf(top, acc[i][j][r]);
                if (labels) {
                    const int64_t y = mine ? xent_label(p, m) - p.class0 - nb : -1;
                    if (y >= 0 && y < 4 * FN && nb + y < p.N) {
#pragma unroll
                        for (int j = 0; j < FN; ++j)
#pragma unroll
                            for (int r = 0; r < 4; ++r) if (y == 4 * j + r) p.picked[m] = acc[i][j][r];
                    }
                } else {
                    float st = 0.f, stz = 0.f;
                    if (mine)
#pragma unroll
                        for (int j = 0; j < FN; ++j) {
                            if (nb + 4 * j >= p.N) continue;
                            const f32x4 t = xent_profile4(p.target, p.target_kind, p.target_row, m, nb + 4 * j, p.N);
#pragma unroll
                            for (int r = 0; r < 4; ++r) { st += t[r]; stz += t[r] != 0.f ? t[r] * acc[i][j][r] : 0.f; }
                        }
                    st += __shfl_xor(st, 16); stz += __shfl_xor(stz, 16);
                    st += __shfl_xor(st, 32); stz += __shfl_xor(stz, 32);
                    if (lj == 0) red[(WN + wn) * BM + mr] = make_float2(st, stz);
                }
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s += power(acc[i][j][r] - ref);
                s += __shfl_xor(s, 16);
                s += __shfl_xor(s, 32);
                if (lj == 0) red[wn * BM + mr] = make_float2(top, s);
            }
            __syncthreads();
            for (int mr = tid; mr < BM; mr += 64 * NW) {
                if (m0 + mr >= p.M) break;
                float top = -INFINITY, s = 0.f;
#pragma unroll
                for (int w = 0; w < WN; ++w) top = fmaxf(top, red[w * BM + mr].x);
                const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
                for (int w = 0; w < WN; ++w) { const float2 v = red[w * BM + mr]; s += v.y * power((v.x == -INFINITY ? ref : v.x) - ref); }
                const int64_t at = (int64_t)tn * p.M + m0 + mr;
                p.part[at] = make_float2(top, s);
                if (!labels) {
                    float2 t = make_float2(0.f, 0.f);
#pragma unroll
                    for (int w = 0; w < WN; ++w) { const float2 v = red[(WN + w) * BM + mr]; t.x += v.x; t.y += v.y; }
                    p.part_t[at] = t;
                }
            }
        } else {
            // G in place of the logits: d ts exp(z - lse), minus d t or, at the label, d.  Rows without a target (d = 0) are 0 whatever they hold.
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                const int64_t m = mb + i;
                const bool mine = m < p.M;
                const int64_t label = labels && mine ? xent_label(p, m) : -1;
                const float d = mine && (!labels || (label >= 0 && label < p.classes)) ? p.dloss[m] : 0.f;     // a label that is no class: no gradient
                float lse = mine ? p.lse[m] : 0.f;
                lse = lse == -INFINITY ? 0.f : lse;              // (no class left: every exponential is 0)
                const float scale = labels ? d : (mine ? d * p.tsum[m] : 0.f);
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[i][j][r] = d != 0.f ? scale * power(acc[i][j][r] - lse) : 0.f;
                if (labels) {
                    const int64_t y = label - p.class0 - nb;
                    if (d != 0.f && y >= 0 && y < 4 * FN) {
#pragma unroll
                        for (int j = 0; j < FN; ++j)
#pragma unroll
                            for (int r = 0; r < 4; ++r) acc[i][j][r] -= y == 4 * j + r ? d : 0.f;
                    }
                } else if (d != 0.f) {
#pragma unroll
                    for (int j = 0; j < FN; ++j) {
                        if (nb + 4 * j >= p.N) continue;
                        const f32x4 t = xent_profile4(p.target, p.target_kind, p.target_row, m, nb + 4 * j, p.N);
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[i][j][r] -= d * t[r];
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float s = 0.f;
#pragma unroll
                    for (int i = 0; i < FM; ++i) s += acc[i][j][r];
#pragma unroll
                    for (int o = 1; o < 16; o <<= 1) s += __shfl_xor(s, o);
                    if (li == 0 && nb + 4 * j + r < p.N) p.dbias_part[(int64_t)(tm * WM + wm) * p.dbias_ld + nb + 4 * j + r] = s;
                }
            typedef uint16_t rowvec __attribute__((ext_vector_type(4 * FN)));
            typedef uint16_t colvec __attribute__((ext_vector_type(FM)));
            auto store = [&](auto edges) {
#pragma unroll
            for (int pl = 0; pl < PL; ++pl) {
                uint16_t o[FM][4 * FN];
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < FN; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            float rest = acc[i][j][r];
                            if constexpr (decltype(edges)::value) o[i][4 * j + r] = split_term(rest, pl + 1 == PL);
                            else {
                                o[i][4 * j + r] = to_bf16(rest);
                                rest -= from_bf16(o[i][4 * j + r]);
                            }
                            acc[i][j][r] = rest;
                        }
                uint16_t* G = p.G + pl * p.g_plane;
                uint16_t* GT = p.GT + pl * p.gt_plane;
                if (nb < p.ldg) {                                // (ldg is a multiple of 64, a lane's 4 FN columns lie inside or outside of it)
#pragma unroll
                    for (int i = 0; i < FM; ++i) {
                        if (mb + i >= p.M) continue;
                        rowvec v;
#pragma unroll
                        for (int k = 0; k < 4 * FN; ++k) v[k] = o[i][k];
                        *(rowvec*)(G + (int64_t)(mb + i) * p.ldg + nb) = v;
                    }
                }
                if (mb < p.ldgt) {                               // (so is ldgt)
#pragma unroll
                    for (int k = 0; k < 4 * FN; ++k) {
                        if (nb + k >= p.N) continue;
                        colvec v;
#pragma unroll
                        for (int i = 0; i < FM; ++i) v[i] = o[i][k];
                        *(colvec*)(GT + (int64_t)(nb + k) * p.ldgt + mb) = v;
                    }
                }
            }
            };
            // (split_term's care for values at float32's end and infinities costs 5 % of a product with 800 rows: only where a wave has one)
            float most = 0.f;
            if constexpr (PL == 3)
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < FN; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) most = fmaxf(most, fabsf(acc[i][j][r]));
            if (PL == 3 && __builtin_amdgcn_ballot_w64(most > 3.38953139e38f) != 0) store(std::true_type{});
            else store(std::false_type{});
        }
    }
}

// (maximum, sum) of two disjoint sets of classes.  A set of NaNs has no maximum: its sum says so.
__device__ __forceinline__ float2 join_lse(float2 a, float2 b) {
    const float top = fmaxf(a.x, b.x);
    if (top == -INFINITY) return make_float2(top, a.y + b.y);
    return make_float2(top, a.y * (a.x == -INFINITY ? 1.f : __expf(a.x - top)) + b.y * (b.x == -INFINITY ? 1.f : __expf(b.x - top)));
}

// loss and lse of every row from the partial sums of the class tiles (4096 rows of 391 tiles: 15 us; one row of 1000: 4.1 us): 1024 threads, `per` rows (a power of two up to 64) x 1024 / per strands of tiles
// One call per piece of the classes: what the pieces so far come to waits in `carry`, the last one gives the results.
struct XentRows {
    float4* carry; int32_t first, last;        // [rows] (maximum, sum, sum of t, sum of t z)
    const float2* part; const float2* part_t; const float* picked;
    int64_t tiles, rows, classes;
    int32_t per;
    const void* target; int32_t target_kind;
    float* loss; float* lse;
};
__global__ __launch_bounds__(1024) void k_xent_lse(const XentRows p) {
    __shared__ float2 red[1024], red_t[1024];
    const int in = threadIdx.x & (p.per - 1), strands = 1024 / p.per, strand = threadIdx.x / p.per;
    const int64_t row = (int64_t)blockIdx.x * p.per + in;
    float2 v = make_float2(-INFINITY, 0.f), t = make_float2(0.f, 0.f);
    if (row < p.rows) {
        if (!p.first && strand == 0) { const float4 c = p.carry[row]; v = make_float2(c.x, c.y); t = make_float2(c.z, c.w); }
#pragma unroll 4
        for (int64_t k = strand; k < p.tiles; k += strands) v = join_lse(v, p.part[k * p.rows + row]);
        if (p.part_t) {
#pragma unroll 4
            for (int64_t k = strand; k < p.tiles; k += strands) { const float2 u = p.part_t[k * p.rows + row]; t.x += u.x; t.y += u.y; }
        }
    }
    red[threadIdx.x] = v;
    red_t[threadIdx.x] = t;
    for (int half = strands / 2; half > 0; half >>= 1) {
        __syncthreads();
        if (strand < half) {
            v = join_lse(v, red[threadIdx.x + half * p.per]);
            const float2 u = red_t[threadIdx.x + half * p.per];
            t.x += u.x; t.y += u.y;
            red[threadIdx.x] = v;
            red_t[threadIdx.x] = t;
        }
    }
    if (strand != 0 || row >= p.rows) return;
    if (!p.last) { p.carry[row] = make_float4(v.x, v.y, t.x, t.y); return; }
    const float lse = v.x == -INFINITY ? (v.y == 0.f ? -INFINITY : v.y) : v.x + __logf(v.y);
    p.lse[row] = lse;
    float loss;
    if (p.target_kind <= XT_I64) {
        const int64_t y = p.target_kind == XT_I64 ? ((const int64_t*)p.target)[row] : (int64_t)((const int32_t*)p.target)[row];
        if (y < 0) loss = 0.f;
        else if (y >= p.classes) loss = NAN;
        else { const float z = p.picked[row]; loss = z == -INFINITY ? INFINITY : lse - z; }
    } else if (t.x == 0.f && t.y == 0.f) loss = 0.f;
    else loss = fabsf(t.y) == INFINITY && !isnan(lse) ? -t.y : t.x * lse - t.y;      // (weight on a class that is not there, also where none is: lse = -inf)
    p.loss[row] = loss;
}

// tsum = the sum of every row of a profile, weight = dloss, or 0 where all of the row is; one workgroup per row (64 x 20000 float32: 4.7 us, latency)
__global__ __launch_bounds__(1024) void k_xent_tsum(const void* target, int32_t kind, int64_t target_row, int64_t classes, const float* __restrict__ dloss,
                                                    float* __restrict__ tsum, float* __restrict__ weight) {
    const int64_t row = blockIdx.x;
    __shared__ float red[16];
    __shared__ int some[16];
    const int64_t step = 4 * (int64_t)blockDim.x;
    float s = 0.f;
    bool any = false;
    if (kind == XT_F32) {
        const float* t = (const float*)target + row * target_row;
#pragma unroll 4
        for (int64_t c = (int64_t)threadIdx.x * 4; c < classes; c += step) {
            if (c + 4 <= classes) { const f32x4u v = *(const f32x4u*)(t + c); s += (v[0] + v[1]) + (v[2] + v[3]); any |= v[0] != 0.f || v[1] != 0.f || v[2] != 0.f || v[3] != 0.f; }
            else for (int64_t k = c; k < classes; ++k) { s += t[k]; any |= t[k] != 0.f; }
        }
    } else {
        const uint16_t* t = (const uint16_t*)target + row * target_row;
#pragma unroll 4
        for (int64_t c = (int64_t)threadIdx.x * 4; c < classes; c += step) {
            if (c + 4 <= classes) { const u16x4u v = *(const u16x4u*)(t + c); s += (from_bf16(v[0]) + from_bf16(v[1])) + (from_bf16(v[2]) + from_bf16(v[3])); any |= ((v[0] | v[1] | v[2] | v[3]) & 0x7fff) != 0; }
            else for (int64_t k = c; k < classes; ++k) { s += from_bf16(t[k]); any |= (t[k] & 0x7fff) != 0; }
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    const bool wave_any = __builtin_amdgcn_ballot_w64(any) != 0;
    if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6] = s; some[threadIdx.x >> 6] = wave_any; }
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.f;
        int live = 0;
        for (int w = 0; w < (int)blockDim.x / 64; ++w) { s += red[w]; live |= some[w]; }
        tsum[row] = s;
        weight[row] = live ? dloss[row] : 0.f;
    }
}

// What is left of a backward pass (of a piece of its classes), in one launch: out[m][n] = the sum of the splits' float32 sums for up to two matrices (dx, dW), dbias = the sum of
// the partial column sums, each added in order and rounded once.  A thread takes one element of a small matrix, four consecutive ones of a large one.
struct SplitSum {
    const float* acc; int64_t split; int32_t splits, blocks;     // [splits][rows][cols], `split` elements apart; blocks = 0: nothing to do
    int32_t per;                                                 // 1 / 4 elements per thread
    int64_t rows, cols;
    void* out; int64_t ld;
};
struct XentFinish {
    SplitSum m[2];
    int32_t first;                                               // number of the launch's first workgroup
    const float* part; int64_t part_ld; int32_t parts;
    int64_t classes;
    float* dbias;
};
template <typename T>
__global__ __launch_bounds__(256) void k_xent_finish(const XentFinish p) {
    int block = blockIdx.x + p.first;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        if (block < p.m[w].blocks) {
            const SplitSum& q = p.m[w];
            const int64_t e = ((int64_t)block * 256 + threadIdx.x) * q.per, all = q.rows * q.cols;
            if (e >= all) return;
            int64_t m = e / q.cols, n = e - m * q.cols;
            T* out = (T*)q.out + m * q.ld + n;
            auto rounded = [](float v) -> T { if constexpr (sizeof(T) == 4) return v; else return to_bf16(v); };
            if (q.per == 1) {
                float s = 0.f;
#pragma unroll 8
                for (int k = 0; k < q.splits; ++k) s += q.acc[k * q.split + e];
                *out = rounded(s);
            } else if (n + 4 <= q.cols) {
                typedef T four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
                f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
                for (int k = 0; k < q.splits; ++k) s += *(const f32x4u*)(q.acc + k * q.split + e);
                *(four*)out = (four){rounded(s[0]), rounded(s[1]), rounded(s[2]), rounded(s[3])};
            } else {                                             // the end of a row, or of everything
                for (int64_t i = e; i < e + 4 && i < all; ++i) {
                    float s = 0.f;
                    for (int k = 0; k < q.splits; ++k) s += q.acc[k * q.split + i];
                    ((T*)q.out)[m * q.ld + n] = rounded(s);
                    if (++n == q.cols) { n = 0; ++m; }
                }
            }
            return;
        }
        block -= p.m[w].blocks;
    }
    const int64_t c = (int64_t)block * 256 + threadIdx.x;
    if (c >= p.classes) return;
    float s = 0.f;
#pragma unroll 8
    for (int k = 0; k < p.parts; ++k) s += p.part[k * p.part_ld + c];
    p.dbias[c] = s;
}

}  // namespace rowops
