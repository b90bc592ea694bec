// dimn_norm.h -- layer normalisation over the last axis, forward and backward (gfx950).
//
//   mu = mean(x),  r = 1 / sqrt(mean((x - mu)^2) + eps),  xh = (x - mu) r,  y = xh gamma + beta
//   g = dy gamma,  dx = r (g - mean(g) - xh mean(g xh)),  dgamma = sum over rows of dy xh,  dbeta = sum over rows of dy
//
// Both directions read every element once and write one result per element: HBM bounds them, and everything here serves that.
//   * A row lives in the registers of TPR threads (16, 64, 256 or 1024), E pieces of 16 bytes each, so the mean, the centred sum of
//     squares and the result come from ONE read.  The variance is the centred sum, not E[x^2] - mu^2: nothing cancels for rows far from 0.
//   * Pieces are 16 bytes whatever the alignment: gfx950 takes unaligned 16-byte global accesses, so odd widths and odd row strides
//     need no second kernel.  The piece that would cross the end of a row is moved back to end with it (Columns): guarded element-wise accesses
//     instead put a branch and a wait between the requests of a row -- 50k rows of 2400 bfloat16 ran 175 us with them.
//   * A thread keeps its columns of gamma / beta in registers over all rows it handles (read per row they would cost twice the bytes of a
//     bfloat16 row from L2), and requests the next row before it reduces the current one.
//   * Backward: a thread owns its columns for all rows it handles, so dgamma / dbeta are sums in its registers; a workgroup writes one
//     partial row, k_norm_param_grad adds the partial rows in a fixed order.  No atomics: the same call gives the same bits.
// All arithmetic is float32; a bfloat16 result is rounded once, to nearest even.
// Measured: 50k x 2400 bfloat16 forward 94 us = 5.1 TB/s, float32 backward 271 + 6 us = 5.2 TB/s (a large copy: 5.3); 40 groups of 64 x 256 float32
// 3.8 us forward, 5.5 + 2.5 backward, where the launch is most of it.
#pragma once
#include "dimn_rowops.h"

namespace rowops {

// V consecutive elements of a row, as one access when V > 1
template <typename T, int V> struct Piece;
template <> struct Piece<float, 4> { typedef float raw __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Piece<float, 1> { typedef float raw __attribute__((ext_vector_type(1), aligned(4))); };
template <> struct Piece<bf16_t, 8> { typedef uint16_t raw __attribute__((ext_vector_type(8), aligned(2))); };
template <> struct Piece<bf16_t, 1> { typedef uint16_t raw __attribute__((ext_vector_type(1), aligned(2))); };
template <typename T> constexpr int kWide = sizeof(T) == 2 ? 8 : 4;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16_t from_f32<bf16_t>(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }

// The columns of a thread: piece e covers V columns from first(e).  Only the last piece can cross the end of the row; it is moved back to end with
// the row, and its first `skip` columns (all of them where the thread has no last piece) belong to other threads: they are read, since a full
// piece is one access without a branch, but take no part in sums.  What two threads store to the same column is the same value -- bit by bit, since
// which of them comes last is open: every operation between load and store is written out (no contraction, fmaf where one is meant), or the compiler
// fuses those of a thread's last piece, whose sums are conditional, differently from the others' (2051 float32 columns: the bits of one of them changed
// from call to call).
template <int TPR, int E, int V>
struct Columns {
    int lane, last, skip;
    __device__ __forceinline__ Columns(int width) : lane(threadIdx.x % TPR) {
        const int c = (lane + (E - 1) * TPR) * V;
        last = c < width - V ? c : width - V;
        skip = c - last < V ? c - last : V;
    }
    __device__ __forceinline__ int first(int e) const { return e < E - 1 ? (lane + e * TPR) * V : last; }
    __device__ __forceinline__ bool mine(int e, int i) const { return e < E - 1 || i >= skip; }
};

// a thread's columns of a parameter row (float32; NULL: `none` everywhere)
template <int TPR, int E, int V>
__device__ __forceinline__ void load_params(const float* row, const Columns<TPR, E, V>& col, float none, float (&to)[E * V]) {
    constexpr int W = V < 4 ? V : 4;
#pragma unroll
    for (int k = 0; k < E * V; ++k) to[k] = none;
    if (!row) return;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
        for (int j = 0; j < V; j += W) {
            const typename Piece<float, W>::raw v = *(const typename Piece<float, W>::raw*)(row + col.first(e) + j);
#pragma unroll
            for (int i = 0; i < W; ++i) to[e * V + j + i] = v[i];
        }
}

// the sum of (a, b) over the TPR threads of a row, in every one of them.  `red`: 2 x 16 float2 of LDS for TPR > 64, used alternately (`turn`)
// so that one barrier per sum is enough: nobody writes a slot again before everybody has passed the barrier of the sum between.
template <int TPR>
__device__ __forceinline__ void row_sum2(float& a, float& b, float2* red, int& turn) {
#pragma unroll
    for (int off = (TPR < 64 ? TPR : 64) / 2; off > 0; off >>= 1) { a += __shfl_xor(a, off); b += __shfl_xor(b, off); }
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        float2* slot = red + turn * 16;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = make_float2(a, b);
        __syncthreads();
        a = 0.f; b = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) { const float2 t = slot[w]; a += t.x; b += t.y; }
    }
}

// result times the gate of a float32 plane (general path only)
template <typename T, int V>
__device__ __forceinline__ void apply_gate(const float* gate, float (&f)[V]) {
    if constexpr (sizeof(T) == 4) {
        if (gate) {
            const typename Piece<float, V>::raw k = *(const typename Piece<float, V>::raw*)gate;
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] *= k[i];
        }
    }
}

// grid (workgroups, groups); max(256, TPR) threads; each set of TPR threads takes rows set, set + sets, ... of its group
template <typename T, int TPR, int E, int V>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void k_norm(const NormP p) {
#pragma clang fp contract(off)
    typedef typename Piece<T, V>::raw raw;
    constexpr int BLOCK = TPR < 256 ? 256 : TPR, SETS = BLOCK / TPR;
    __shared__ float2 red[32];
    int turn = 0;
    const Columns<TPR, E, V> col(p.width);
    const int64_t g = blockIdx.y, sets = (int64_t)gridDim.x * SETS;
    const T* x = (const T*)p.x + g * p.x_group;
    T* y = (T*)p.out + g * p.out_group;
    const float n = (float)p.width;
    // TPR > 64: every thread of the workgroup walks the same rows; TPR <= 64: sets of one wave may run out of rows at different times, but the
    // sums stay inside a set
    int64_t r = (int64_t)blockIdx.x * SETS + threadIdx.x / TPR;
    raw next[E];
    auto request = [&](int64_t row) {
        const T* from = x + row * p.x_row;
#pragma unroll
        for (int e = 0; e < E; ++e) next[e] = *(const raw*)(from + col.first(e));
    };
    if (r < p.rows) request(r);
    float ga[E * V], be[E * V];
    load_params(p.gamma ? p.gamma + g * p.width : nullptr, col, 1.f, ga);
    load_params(p.beta ? p.beta + g * p.width : nullptr, col, 0.f, be);
    for (; r < p.rows; r += sets) {
        float v[E * V], s = 0.f, q = 0.f, none = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[e * V + i] = to_f32(next[e][i]);
                s += col.mine(e, i) ? v[e * V + i] : 0.f;
            }
        if (r + sets < p.rows) request(r + sets);
        row_sum2<TPR>(s, none, red, turn);
        const float mu = s / n;                                  // (a division, not a product with 1 / n: the mean of a constant row is that constant)
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = v[e * V + i] - mu;
                v[e * V + i] = d;
                q = col.mine(e, i) ? fmaf(d, d, q) : q;
            }
        none = 0.f;
        row_sum2<TPR>(q, none, red, turn);
        const float rs = 1.f / sqrtf(q / n + p.eps);
        if (threadIdx.x % TPR == 0) { if (p.mean) p.mean[g * p.rows + r] = mu; if (p.rstd) p.rstd[g * p.rows + r] = rs; }
        T* to = y + r * p.out_row;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float f[V];
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = fmaf(v[e * V + i] * rs, ga[e * V + i], be[e * V + i]);
            apply_gate<T, V>(p.gate ? p.gate + g * p.out_group + r * p.out_row + col.first(e) : nullptr, f);
            raw o;
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = from_f32<T>(f[i]);
            if (col.mine(e, V - 1)) *(raw*)(to + col.first(e)) = o;
        }
    }
}

// as k_norm; partial sums of dgamma / dbeta: one row per workgroup (the sets of a workgroup are added through LDS, in order).
// 1024 threads leave 128 registers each: no next row in flight there, and gamma is read again for every row.
template <typename T, int TPR, int E, int V>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void k_norm_grad(const NormP p) {
#pragma clang fp contract(off)
    typedef typename Piece<T, V>::raw raw;
    constexpr int BLOCK = TPR < 256 ? 256 : TPR, SETS = BLOCK / TPR;
    constexpr bool AHEAD = TPR < 1024;
    __shared__ float2 red[32];
    __shared__ float acc[SETS > 1 ? SETS * TPR * V : 1];
    int turn = 0;
    const int D = p.width, lane = threadIdx.x % TPR, set = threadIdx.x / TPR;
    const Columns<TPR, E, V> col(D);
    const int64_t g = blockIdx.y, sets = (int64_t)gridDim.x * SETS;
    const T* x = (const T*)p.x + g * p.x_group;
    const T* dy = (const T*)p.dy + g * p.dy_group;
    T* dx = (T*)p.out + g * p.out_group;
    const float* gamma = p.gamma ? p.gamma + g * D : nullptr;
    const float n = (float)D;
    int64_t r = (int64_t)blockIdx.x * SETS + set;
    raw nx[E], nd[E];
    float nmu = 0.f, nrs = 0.f;
    auto request = [&](int64_t row) {
        const T *fx = x + row * p.x_row, *fd = dy + row * p.dy_row;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            nx[e] = *(const raw*)(fx + col.first(e));
            nd[e] = *(const raw*)(fd + col.first(e));
        }
        nmu = p.mean[g * p.rows + row];
        nrs = p.rstd[g * p.rows + row];
    };
    if (AHEAD && r < p.rows) request(r);
    float ga[E * V], dg[E * V], db[E * V];
    if (AHEAD) load_params(gamma, col, 1.f, ga);
#pragma unroll
    for (int k = 0; k < E * V; ++k) dg[k] = db[k] = 0.f;
    for (; r < p.rows; r += sets) {
        if (!AHEAD) { request(r); load_params(gamma, col, 1.f, ga); }
        float xh[E * V], gy[E * V];
        const float mu = nmu, rs = nrs;
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int k = e * V + i;
                const float d = to_f32(nd[e][i]);
                xh[k] = (to_f32(nx[e][i]) - mu) * rs;
                dg[k] = fmaf(d, xh[k], dg[k]);                   // (columns of other threads: summed, but not handed on below)
                db[k] += d;
                gy[k] = d * ga[k];
                s1 = col.mine(e, i) ? s1 + gy[k] : s1;
                s2 = col.mine(e, i) ? fmaf(gy[k], xh[k], s2) : s2;
            }
        if (AHEAD && r + sets < p.rows) request(r + sets);
        row_sum2<TPR>(s1, s2, red, turn);
        s1 /= n; s2 /= n;
        T* to = dx + r * p.out_row;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float f[V];
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = rs * fmaf(-xh[e * V + i], s2, gy[e * V + i] - s1);
            apply_gate<T, V>(p.gate ? p.gate + g * p.out_group + r * p.out_row + col.first(e) : nullptr, f);
            raw o;
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = from_f32<T>(f[i]);
            if (col.mine(e, V - 1)) *(raw*)(to + col.first(e)) = o;
        }
    }
    if (!p.part) return;
    float* part = p.part + (g * gridDim.x + blockIdx.x) * 2 * (int64_t)D;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float* to = part + which * (int64_t)D;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if constexpr (SETS > 1) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < V; ++i) acc[(set * V + i) * TPR + lane] = which ? db[e * V + i] : dg[e * V + i];
                __syncthreads();
                if (set == 0) {                                  // (LDS rows of a lane's own columns: no need to undo the shift of the last piece)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        float t = 0.f;
#pragma unroll
                        for (int w = 0; w < SETS; ++w) t += acc[(w * V + i) * TPR + lane];
                        if (col.mine(e, i)) to[col.first(e) + i] = t;
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (col.mine(e, i)) to[col.first(e) + i] = which ? db[e * V + i] : dg[e * V + i];
            }
        }
    }
}

// Rows longer than the registers of 1024 threads hold: one workgroup per row at a time, the row read three times (the second and third
// time from L2).  Backward keeps the parameter gradients in the workgroup's own partial row, which nobody else touches.
template <typename T>
__device__ __forceinline__ typename Piece<T, kWide<T>>::raw load_piece(const T* row, int64_t c, int64_t n) {
    typedef typename Piece<T, kWide<T>>::raw raw;
    if (c + kWide<T> <= n) return *(const raw*)(row + c);
    raw v;
#pragma unroll
    for (int i = 0; i < kWide<T>; ++i) v[i] = c + i < n ? row[c + i] : (T)0;
    return v;
}
template <typename T>
__device__ __forceinline__ void store_piece(T* row, int64_t c, int64_t n, const typename Piece<T, kWide<T>>::raw& v) {
    typedef typename Piece<T, kWide<T>>::raw raw;
    if (c + kWide<T> <= n) { *(raw*)(row + c) = v; return; }
#pragma unroll
    for (int i = 0; i < kWide<T>; ++i)
        if (c + i < n) row[c + i] = v[i];
}

template <typename T>
__global__ __launch_bounds__(1024) void k_norm_long(const NormP p) {
    constexpr int V = kWide<T>;
    typedef typename Piece<T, V>::raw raw;
    __shared__ float2 red[32];
    int turn = 0;
    const int D = p.width;
    const int64_t g = blockIdx.y;
    const float n = (float)D;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* x = (const T*)p.x + g * p.x_group + r * p.x_row;
        T* y = (T*)p.out + g * p.out_group + r * p.out_row;
        float s = 0.f, q = 0.f, zero = 0.f;
        for (int64_t c = (int64_t)threadIdx.x * V; c < D; c += 1024 * V) {
            const raw v = load_piece(x, c, D);
#pragma unroll
            for (int i = 0; i < V; ++i) s += to_f32(v[i]);
        }
        row_sum2<1024>(s, zero, red, turn);
        const float mu = s / n;                                // (a division, not a product with 1 / n: the mean of a constant row is that constant)
        for (int64_t c = (int64_t)threadIdx.x * V; c < D; c += 1024 * V) {
            const raw v = load_piece(x, c, D);
#pragma unroll
            for (int i = 0; i < V; ++i) { const float d = to_f32(v[i]) - mu; q += c + i < D ? d * d : 0.f; }
        }
        zero = 0.f;
        row_sum2<1024>(q, zero, red, turn);
        const float rs = 1.f / sqrtf(q / n + p.eps);
        if (threadIdx.x == 0) { if (p.mean) p.mean[g * p.rows + r] = mu; if (p.rstd) p.rstd[g * p.rows + r] = rs; }
        for (int64_t c = (int64_t)threadIdx.x * V; c < D; c += 1024 * V) {
            const raw v = load_piece(x, c, D);
            raw o;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const bool in = c + i < D;
                float f = (to_f32(v[i]) - mu) * rs * (p.gamma && in ? p.gamma[g * D + c + i] : 1.f) + (p.beta && in ? p.beta[g * D + c + i] : 0.f);
                if (p.gate && in) f *= p.gate[g * p.out_group + r * p.out_row + c + i];
                o[i] = from_f32<T>(f);
            }
            store_piece(y, c, D, o);
        }
    }
}

template <typename T>
__global__ __launch_bounds__(1024) void k_norm_grad_long(const NormP p) {
    constexpr int V = kWide<T>;
    typedef typename Piece<T, V>::raw raw;
    __shared__ float2 red[32];
    int turn = 0;
    const int D = p.width;
    const int64_t g = blockIdx.y;
    const float n = (float)D;
    float* part = p.part ? p.part + (g * gridDim.x + blockIdx.x) * 2 * (int64_t)D : nullptr;
    bool first = true;
    for (int64_t r = blockIdx.x; r < p.rows || (first && part); r += gridDim.x) {
        const bool have = r < p.rows;                                // (a workgroup without a row still owes a partial row of zeros)
        const T* x = (const T*)p.x + g * p.x_group + r * p.x_row;
        const T* dy = (const T*)p.dy + g * p.dy_group + r * p.dy_row;
        T* dx = (T*)p.out + g * p.out_group + r * p.out_row;
        const float mu = have ? p.mean[g * p.rows + r] : 0.f, rs = have ? p.rstd[g * p.rows + r] : 0.f;
        float s1 = 0.f, s2 = 0.f;
        for (int64_t c = (int64_t)threadIdx.x * V; c < D; c += 1024 * V) {
            raw v, d;
#pragma unroll
            for (int i = 0; i < V; ++i) { v[i] = 0; d[i] = 0; }
            if (have) { v = load_piece(x, c, D); d = load_piece(dy, c, D); }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (c + i >= D) continue;
                const float f = to_f32(d[i]), xh = (to_f32(v[i]) - mu) * rs, gy = f * (p.gamma ? p.gamma[g * D + c + i] : 1.f);
                s1 += gy;
                s2 += gy * xh;
                if (part) {                                          // this thread's own columns: no other thread reads or writes them
                    part[c + i] = (first ? 0.f : part[c + i]) + f * xh;
                    part[D + c + i] = (first ? 0.f : part[D + c + i]) + f;
                }
            }
        }
        first = false;
        if (!have) break;
        row_sum2<1024>(s1, s2, red, turn);
        s1 /= n; s2 /= n;
        for (int64_t c = (int64_t)threadIdx.x * V; c < D; c += 1024 * V) {
            const raw v = load_piece(x, c, D), d = load_piece(dy, c, D);
            raw o;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const bool in = c + i < D;
                const float xh = (to_f32(v[i]) - mu) * rs, gy = to_f32(d[i]) * (p.gamma && in ? p.gamma[g * D + c + i] : 1.f);
                float f = rs * (gy - s1 - xh * s2);
                if (p.gate && in) f *= p.gate[g * p.out_group + r * p.out_row + c + i];
                o[i] = from_f32<T>(f);
            }
            store_piece(dx, c, D, o);
        }
    }
}

// dgamma / dbeta = the partial rows of a group, added in order (342 of 2 x 1025: 4.3 us; twice the workgroups in front of it would cost it more than they
// save there).  grid (ceil(2 width / 64), groups), 1024 threads: 64 columns x 16 strands of rows.
__global__ __launch_bounds__(1024) void k_norm_param_grad(const float* __restrict__ part, int parts, int32_t width, float* __restrict__ dgamma, float* __restrict__ dbeta) {
    __shared__ float red[16][64];
    const int64_t g = blockIdx.y, n2 = 2 * (int64_t)width;
    const int64_t c = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    const int strand = threadIdx.x >> 6;
    float s = 0.f;
    if (c < n2) {
        const float* from = part + g * parts * n2 + c;
#pragma unroll 8
        for (int k = strand; k < parts; k += 16) s += from[k * n2];
    }
    red[strand][threadIdx.x & 63] = s;
    __syncthreads();
    if (strand == 0 && c < n2) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < 16; ++w) t += red[w][threadIdx.x];
        if (c < width) { if (dgamma) dgamma[g * width + c] = t; }
        else if (dbeta) dbeta[g * width + c - width] = t;
    }
}

}  // namespace rowops
