// dimn_rowops.hip -- the row operators of libdimn on device arrays of the caller: layer normalisation (dimn_norm.h) and the softmax
// cross entropy of a linear output layer (dimn_xent.h).
// No handle: a call names its device and its stream, works on the caller's memory only, and returns when its kernels are queued.
#include "dimn_rowops.h"

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "dimn_norm.h"
#include "dimn_xent.h"
#include "dimn_xent_thin.h"

#define HIPCHK(expr)                                                                            \
    do {                                                                                        \
        hipError_t e_ = (expr);                                                                 \
        if (e_ != hipSuccess)                                                                   \
            return dimn_fail(DIMN_ERR_HIP, "%s failed: %s (%s:%d)", #expr, hipGetErrorString(e_), __FILE__, __LINE__); \
    } while (0)
#define CHK(expr)              \
    do {                       \
        int rc_ = (expr);      \
        if (rc_) return rc_;   \
    } while (0)

namespace {

int64_t ceil_div64(int64_t a, int64_t b) { return (a + b - 1) / b; }

// the caller's current device comes back when the call ends
struct OnDevice {
    int before = -1, now = -1;
    int enter(const char* who, int32_t device) {
        static std::atomic<int> known{0};                        // (a query of ~0.5 us per call; the number does not change while a process lives)
        int n = known.load(std::memory_order_relaxed);
        if (n == 0) {
            if (hipGetDeviceCount(&n) != hipSuccess || n < 1) return dimn_fail(DIMN_ERR_HIP, "%s: no HIP device visible", who);
            known.store(n, std::memory_order_relaxed);
        }
        if (device < 0 || device >= n) return dimn_fail(DIMN_ERR_ARG, "%s: device_id %d out of range (%d devices)", who, device, n);
        (void)hipGetLastError();                                 // (an error that an earlier call of the thread left is not the coming launches')
        HIPCHK(hipGetDevice(&before));
        now = device;
        if (before != now) HIPCHK(hipSetDevice(now));
        return DIMN_OK;
    }
    ~OnDevice() { if (now >= 0 && before != now) (void)hipSetDevice(before); }
};

// compute units of a device (256 on MI355X), asked once per device
int compute_units(int dev) {
    static std::atomic<int> known[64];
    if (dev < 0 || dev >= 64) return 256;
    int n = known[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 1) n = 256;
        known[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

int current_device() {
    int dev = 0;
    return hipGetDevice(&dev) == hipSuccess ? dev : 0;
}

// ---- layer normalisation: which kernel a width takes -----------------------------------------------------------------------
// `tpr` threads hold a row in `e` pieces of `v` elements (16 bytes; 1 for rows shorter than that); tpr = 0: the row does not fit the registers
// (k_norm_long).  As few threads per row as the registers allow: sums then need fewer steps and more rows are in flight.  The limits keep a thread
// below 256 registers, 128 at 1024 threads (backward holds gamma, two gradient sums, two row values and the next row's pieces per element).
struct NormForm { int tpr, e, v; };
NormForm norm_form(int32_t type, bool grad, int32_t width) {
    const bool bf = type == DIMN_TYPE_BF16;
    const int v = bf ? 8 : 4;
    if (width < v) return {16, 1, 1};
    const int nv = (int)ceil_div64(width, v);
    const int most = bf ? (grad ? 3 : 5) : 6, most1k = bf ? 2 : 4;
    if (nv <= 32) return {16, (int)ceil_div64(nv, 16), v};
    for (int tpr : {64, 256})
        if (nv <= tpr * most) return {tpr, (int)ceil_div64(nv, tpr), v};
    if (nv <= 1024 * most1k) return {1024, (int)ceil_div64(nv, 1024), v};
    return {0, 0, v};
}

// workgroups per group: enough to fill the device, every one with the same number of rows (the last one apart)
int64_t norm_blocks(const NormForm& f, bool grad, int64_t groups, int64_t rows) {
    if (rows == 0) return 1;
    const int sets = f.tpr == 0 ? 1 : std::max(1, 256 / f.tpr);
    const int64_t per_cu = grad ? 2 : 4;
    const int64_t budget = std::max<int64_t>(1, per_cu * compute_units(current_device()) / (f.tpr == 1024 || f.tpr == 0 ? 2 : 1) / std::max<int64_t>(1, groups));
    const int64_t all = ceil_div64(rows, sets);
    const int64_t each = ceil_div64(all, budget);
    return std::max<int64_t>(1, ceil_div64(all, each));
}

template <typename T, bool GRAD, int TPR, int E, int V>
void norm_launch_one(dim3 grid, hipStream_t st, const NormP& p) {
    if constexpr (GRAD) hipLaunchKernelGGL((rowops::k_norm_grad<T, TPR, E, V>), grid, dim3(TPR < 256 ? 256 : TPR), 0, st, p);
    else hipLaunchKernelGGL((rowops::k_norm<T, TPR, E, V>), grid, dim3(TPR < 256 ? 256 : TPR), 0, st, p);
}
template <typename T, bool GRAD>
void norm_launch(const NormForm& f, dim3 grid, hipStream_t st, const NormP& p) {
    constexpr bool bf = sizeof(T) == 2;
    constexpr int V = rowops::kWide<T>;
    if (f.v == 1) { norm_launch_one<T, GRAD, 16, 1, 1>(grid, st, p); return; }
    switch (f.tpr * 16 + f.e) {
#define FORM(TPR, E) case TPR * 16 + E: norm_launch_one<T, GRAD, TPR, E, V>(grid, st, p); return
        FORM(16, 1); FORM(16, 2);
        FORM(64, 1); FORM(64, 2); FORM(64, 3);
        FORM(256, 2); FORM(256, 3);
        FORM(1024, 2);
    }
    if constexpr (bf && GRAD) {                                  // (the other forms hold more pieces on a quarter of the threads)
        switch (f.tpr * 16 + f.e) { FORM(256, 1); FORM(1024, 1); }
    }
    if constexpr (!bf || !GRAD) {
        switch (f.tpr * 16 + f.e) { FORM(64, 4); FORM(64, 5); FORM(256, 4); FORM(256, 5); }
    }
    if constexpr (!bf) {
        switch (f.tpr * 16 + f.e) { FORM(64, 6); FORM(256, 6); FORM(1024, 3); FORM(1024, 4); }
    }
#undef FORM
    if constexpr (GRAD) hipLaunchKernelGGL((rowops::k_norm_grad_long<T>), grid, dim3(1024), 0, st, p);
    else hipLaunchKernelGGL((rowops::k_norm_long<T>), grid, dim3(1024), 0, st, p);
}

constexpr int64_t kGridY = 65535;

}  // namespace

int64_t norm_workspace_floats(int32_t type, int64_t groups, int64_t rows, int32_t width) {
    return groups * norm_blocks(norm_form(type, true, width), true, groups, rows) * 2 * (int64_t)width;
}

// p with its group-th plane first
static NormP norm_from(const NormP& p, int64_t group, int64_t parts, int size) {
    NormP q = p;
    auto move = [&](const void* base, int64_t stride) { return base ? (const char*)base + group * stride * size : nullptr; };
    q.x = move(p.x, p.x_group);
    q.dy = move(p.dy, p.dy_group);
    q.out = const_cast<char*>((const char*)move(p.out, p.out_group));
    if (p.gate) q.gate = p.gate + group * p.out_group;
    if (p.gamma) q.gamma = p.gamma + group * p.width;
    if (p.beta) q.beta = p.beta + group * p.width;
    if (p.mean) q.mean = p.mean + group * p.rows;
    if (p.rstd) q.rstd = p.rstd + group * p.rows;
    if (p.part) q.part = p.part + group * parts * 2 * p.width;
    return q;
}

int norm_forward(hipStream_t st, int32_t type, int64_t groups, const NormP& p) {
    if (groups == 0 || p.rows == 0) return DIMN_OK;
    const NormForm f = norm_form(type, false, p.width);
    const int64_t blocks = norm_blocks(f, false, groups, p.rows);
    for (int64_t g0 = 0; g0 < groups; g0 += kGridY) {
        const dim3 grid((unsigned)blocks, (unsigned)std::min(kGridY, groups - g0));
        const NormP q = norm_from(p, g0, 0, type == DIMN_TYPE_BF16 ? 2 : 4);
        if (type == DIMN_TYPE_BF16) norm_launch<bf16_t, false>(f, grid, st, q);
        else norm_launch<float, false>(f, grid, st, q);
    }
    HIPCHK(hipGetLastError());
    return DIMN_OK;
}

int norm_backward(hipStream_t st, int32_t type, int64_t groups, NormP p, float* dgamma, float* dbeta, float* workspace) {
    if (groups == 0) return DIMN_OK;
    const NormForm f = norm_form(type, true, p.width);
    const int64_t blocks = norm_blocks(f, true, groups, p.rows);
    p.part = dgamma || dbeta ? workspace : nullptr;
    if (p.rows == 0 && !p.part) return DIMN_OK;
    for (int64_t g0 = 0; g0 < groups; g0 += kGridY) {
        const dim3 grid((unsigned)blocks, (unsigned)std::min(kGridY, groups - g0));
        const NormP q = norm_from(p, g0, blocks, type == DIMN_TYPE_BF16 ? 2 : 4);      // (rows = 0: the kernels write partial rows of zeros)
        if (type == DIMN_TYPE_BF16) norm_launch<bf16_t, true>(f, grid, st, q);
        else norm_launch<float, true>(f, grid, st, q);
        if (p.part)
            hipLaunchKernelGGL(rowops::k_norm_param_grad, dim3((unsigned)ceil_div64(2 * (int64_t)p.width, 64), grid.y), dim3(1024), 0, st, q.part, (int)blocks, p.width,
                               dgamma ? dgamma + g0 * p.width : nullptr, dbeta ? dbeta + g0 * p.width : nullptr);
    }
    HIPCHK(hipGetLastError());
    return DIMN_OK;
}

static int norm_check(const char* who, int32_t type, int64_t groups, int64_t rows, int64_t width) {
    if (type != DIMN_TYPE_F32 && type != DIMN_TYPE_BF16) return dimn_fail(DIMN_ERR_UNSUP, "%s: element type %d (DIMN_TYPE_F32 or DIMN_TYPE_BF16)", who, type);
    if (groups < 0 || rows < 0 || groups > INT32_MAX || rows > INT32_MAX) return dimn_fail(DIMN_ERR_ARG, "%s: %lld groups of %lld rows", who, (long long)groups, (long long)rows);
    if (width < 1 || width > (1 << 26)) return dimn_fail(DIMN_ERR_ARG, "%s: width %lld not in 1..2^26", who, (long long)width);
    return DIMN_OK;
}

extern "C" int dimn_layer_norm(int32_t device_id, void* stream, int32_t type, int64_t groups, int64_t rows, int64_t width, const void* x, int64_t x_group, int64_t x_row,
                               const float* gamma, const float* beta, float eps, void* y, int64_t y_group, int64_t y_row, float* mean, float* rstd) {
    CHK(norm_check("dimn_layer_norm", type, groups, rows, width));
    if (!(eps >= 0.f)) return dimn_fail(DIMN_ERR_ARG, "dimn_layer_norm: eps %g is negative or not a number", (double)eps);
    if (groups == 0 || rows == 0) return DIMN_OK;
    if (!x || !y) return dimn_fail(DIMN_ERR_ARG, "dimn_layer_norm: null array");
    OnDevice on;
    CHK(on.enter("dimn_layer_norm", device_id));
    NormP p{};
    p.x = x; p.x_group = x_group; p.x_row = x_row; p.out = y; p.out_group = y_group; p.out_row = y_row;
    p.gamma = gamma; p.beta = beta; p.mean = mean; p.rstd = rstd; p.rows = rows; p.width = (int32_t)width; p.eps = eps;
    return norm_forward((hipStream_t)stream, type, groups, p);
}

extern "C" int dimn_layer_norm_grad_workspace(int32_t device_id, int32_t type, int64_t groups, int64_t rows, int64_t width, int64_t* bytes) {
    CHK(norm_check("dimn_layer_norm_grad_workspace", type, groups, rows, width));
    if (!bytes) return dimn_fail(DIMN_ERR_ARG, "dimn_layer_norm_grad_workspace: null");
    OnDevice on;
    CHK(on.enter("dimn_layer_norm_grad_workspace", device_id));
    *bytes = norm_workspace_floats(type, groups, rows, (int32_t)width) * 4;
    return DIMN_OK;
}

extern "C" int dimn_layer_norm_grad(int32_t device_id, void* stream, int32_t type, int64_t groups, int64_t rows, int64_t width, const void* dy, int64_t dy_group, int64_t dy_row,
                                    const void* x, int64_t x_group, int64_t x_row, const float* mean, const float* rstd, const float* gamma,
                                    void* dx, int64_t dx_group, int64_t dx_row, float* dgamma, float* dbeta, void* workspace, int64_t workspace_bytes) {
    CHK(norm_check("dimn_layer_norm_grad", type, groups, rows, width));
    if (groups == 0) return DIMN_OK;
    if (rows > 0 && (!dy || !x || !mean || !rstd || !dx)) return dimn_fail(DIMN_ERR_ARG, "dimn_layer_norm_grad: null array");
    OnDevice on;
    CHK(on.enter("dimn_layer_norm_grad", device_id));
    if (dgamma || dbeta) {
        const int64_t need = norm_workspace_floats(type, groups, rows, (int32_t)width) * 4;
        if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)
            return dimn_fail(DIMN_ERR_ARG, "dimn_layer_norm_grad: a 16-byte aligned workspace of %lld bytes is needed, got %lld", (long long)need, (long long)workspace_bytes);
    }
    NormP p{};
    p.x = x; p.x_group = x_group; p.x_row = x_row; p.dy = dy; p.dy_group = dy_group; p.dy_row = dy_row; p.out = dx; p.out_group = dx_group; p.out_row = dx_row;
    p.gamma = gamma; p.mean = const_cast<float*>(mean); p.rstd = const_cast<float*>(rstd); p.rows = rows; p.width = (int32_t)width;
    return norm_backward((hipStream_t)stream, type, groups, p, dgamma, dbeta, (float*)workspace);
}

// ---- softmax cross entropy of a linear output layer -----------------------------------------------------------------------------
namespace {
using rowops::XentGemm;

int64_t up(int64_t a, int64_t b) { return ceil_div64(a, b) * b; }

// tile shapes of k_xent_gemm: 256 x 256 (float32: 256 x 128; 8 waves), 128 x 128 (4), 64 x 128 (4); wm: waves along m; step: microseconds of one step
// when every CU has a workgroup (128 x 128 bfloat16: two)
struct Tile { int bm, bn, wm, per_cu; double step; };
constexpr Tile kTiles[2][3] = {{{256, 256, 2, 1, 0.9}, {128, 128, 2, 2, 0.6}, {64, 128, 1, 2, 0.4}}, {{256, 128, 4, 1, 1.5}, {128, 128, 2, 1, 1.0}, {64, 128, 1, 2, 0.9}}};
int64_t tile_count(const Tile& t, int64_t M, int64_t N) { return ceil_div64(M, t.bm) * ceil_div64(N, t.bn); }
// the tile that needs the least time in whole rounds; small ones where the large leave CUs idle (1581 x 2880 x 877 float32 logits: 128 x 128 149 us,
// 64 x 128 92; the same in bfloat16: 50 and 33)
int pick_tile(bool f32, int64_t M, int64_t N, int ncu) {
    if (M <= 64) return 2;
    const Tile* t = kTiles[f32];
    auto cost = [&](const Tile& x) { return (double)ceil_div64(tile_count(x, M, N), (int64_t)ncu * x.per_cu) * x.step; };
    const int best = cost(t[0]) <= cost(t[1]) ? 0 : 1;
    return cost(t[2]) < cost(t[best]) ? 2 : best;
}

// A piece's operands take up to 1 GiB: 4096 x 2048 x 64000 / x 100000 bfloat16 backward 3.02 / 4.66 ms (512 MiB:
// 3.09 / 4.88, 192 MiB: 3.17 / 5.02, 4 GiB: 2.93 / 4.78 -- but that keeps as much as the logits).
constexpr int64_t kBudget = (int64_t)1 << 30;

// what a call needs: operand forms, pieces of the classes, and where everything lies in the workspace
struct XentPlan {
    const dimn_output_loss* d;
    bool grad, f32, labels, out_in;           // out_in: the kernel is stored [classes][width]
    int planes, deep, ncu;                    // deep: k's of one step
    int64_t N, H, V, Hp, Np, P;               // Hp, Np: width / rows rounded up to 64; P: classes per piece
    bool x_direct, w_direct, wt_direct;
    int t_logits;
    int64_t tiles_m, tiles_n;                 // logits
    int t_dx, splits, t_dw, dw_splits;
    bool thin; int nf; int64_t blocks;        // few rows: dimn_xent_thin.h; 16 nf rows per block
    size_t x, xt, w, wt, g, gt, part, part_t, picked, carry, tsum, weight, dbias, acc, acc_w, bytes;

    // The largest piece allowed, or a smaller one whose 256 x 256 tiles fill the device in whole rounds: a piece of 84 class tiles at 16 row tiles
    // takes 6 rounds of 256 workgroups where 96 class tiles take the same six (64000 classes: 16 rounds instead of 18, 8 instead of 9 for dW).
    int64_t best_piece(int64_t most) const {
        const int64_t tm = ceil_div64(N, 256) * (f32 ? 2 : 1), th = ceil_div64(H, 256) * (f32 ? 2 : 1);
        auto rounds = [&](int64_t tiles) { return ceil_div64(tiles, ncu); };
        auto cost = [&](int64_t tiles_v) { return (double)rounds(tiles_v * tm) * H + (grad ? (double)rounds(tiles_v * th) * N : 0.0); };
        const int64_t all = ceil_div64(V, 256), top = most / 256;
        int64_t best = top;
        double least = 1e300;
        for (int64_t t = top; t >= 1 && t >= top / 4; --t) {
            const int64_t full = all / t, rest = all - full * t;
            const double c = full * cost(t) + (rest ? cost(rest) : 0.0) + 2e-3 * (double)ncu * (full + (rest ? 1 : 0));
            if (c < least) { least = c; best = t; }
        }
        return best * 256;
    }
    // Ranges of the inner dimension of an M x N product: its rounds get shorter, its sums are written and read once more (at 4 TB/s).
    int split_count(int tile, int64_t M, int64_t N_, int64_t steps) const {
        const Tile& x = kTiles[f32][tile];
        const int64_t tiles = tile_count(x, M, N_), slots = (int64_t)ncu * x.per_cu, most = std::max<int64_t>(1, std::min<int64_t>(32, steps / 8));
        double least = 1e300;
        int best = 1;
        for (int64_t k = 1; k <= most; ++k) {
            const double c = (double)ceil_div64(tiles * k, slots) * (double)steps / (double)k * x.step + (k > 1 ? 4.0 + (double)(k * M * N_) * 8 / 4e6 : 0.0);
            if (c < least) { least = c; best = (int)k; }
        }
        return best;
    }
    // Which form is faster: estimates in microseconds from both forms' measured times over 16 .. 2048 rows, widths of 64 .. 4096 and 300 .. 50000
    // classes (launches, laying out operands, a product's rate, the latency of a step where there are few tiles); backward, a least-squares fit.  Over 98
    // shapes of 40 .. 800 rows each (profiles/xent_forms.txt) the form taken costs 1.1 / 0.7 % more than the better one forward (float32 / bfloat16; 31 %
    // at worst) and 1.7 / 2.1 % backward (46 %), on average; a fit to those shapes alone comes to 0.5 / 1.5 and 1.1 / 0.9 % (tools/xent_forms.py).
    bool prefers_thin() const {
#ifdef DIMN_XENT_FORM      // (tools/xent_forms.py times either form at every shape)
        return DIMN_XENT_FORM;
#endif
        const double hv = (double)H * (double)V, work = hv * (double)N, steps = (f32 ? 2.0 : 0.5) * (double)(Hp / 64);
        double t, g;
        if (!grad) {
            t = work * (f32 ? 25e-6 : 10.5e-6) * 1e-3;
            g = (x_direct ? 0 : 5) + (w_direct ? 0 : 5 + hv * (f32 ? 3.9e-6 : 0.9e-6));
            g += std::max(work * (f32 ? 8e-6 : 2.1e-6) * 1e-3, steps) - 4;
        } else {
            const double weights = hv * 1e-6, gs = (double)N * (double)V * 1e-6, padded = (double)Hp * (double)V * (double)up(N, 128);
            t = (f32 ? 24 : 22) + hv * (double)up(N, f32 ? 32 : 64) * (f32 ? 70e-9 : 20e-9) + (f32 ? 0 : 0.5) * weights + (f32 ? 3.9 : 3.3) * gs;
            g = (f32 ? 41 : 33) + padded * (f32 ? 28e-9 : 6e-9) + (f32 ? 4.6 : 2.0) * weights + (f32 ? 5.7 : 1.8) * gs + (f32 ? 0.027 : 0.001) * (double)Hp;
        }
        return t < g;
    }
    size_t take(int64_t n) { const size_t at = bytes; bytes += (size_t)up(n, 256); return at; }
    void make(const dimn_output_loss* desc, bool with_grad, int compute_units) {
        d = desc; grad = with_grad; ncu = compute_units;
        N = d->rows; H = d->width; V = d->classes;
        f32 = d->type == DIMN_TYPE_F32;
        labels = d->target_kind <= DIMN_TARGET_I64;
        out_in = d->kernel_in == 1;
        planes = f32 ? 3 : 1;
        deep = f32 ? 32 : 64;
        Hp = up(H, 64); Np = up(N, 64);
        const int64_t far = 1 << 22;          // (operand rows are reached by 32-bit offsets inside a tile of 256)
        auto aligned = [](const void* p) { return ((uintptr_t)p & 15) == 0; };
        x_direct = !f32 && H % 64 == 0 && aligned(d->x) && d->x_row % 8 == 0 && d->x_row <= far && d->x_row >= 0;
        w_direct = !f32 && out_in && H % 64 == 0 && aligned(d->kernel) && d->kernel_out % 8 == 0 && d->kernel_out <= far && d->kernel_out >= 0;
        wt_direct = !f32 && !out_in && V % 64 == 0 && aligned(d->kernel) && d->kernel_in % 8 == 0 && d->kernel_in <= far && d->kernel_in >= 0;
        // bytes of the workspace that a class of a piece takes: its operands, and what its tiles leave per row (forward: 8 or 16 bytes for 128 classes or
        // more) or per 64 rows (backward: a sum for dbias)
        const int64_t per_class = 2 * planes * ((w_direct ? 0 : Hp) + (grad ? (wt_direct ? 0 : H) + N + Np : 0)) + (grad ? Np / 16 : Np / (labels ? 16 : 8));
        P = std::max<int64_t>(256, kBudget / std::max<int64_t>(1, per_class) / 256 * 256);
        P = std::min({P, far, up(V, 256), std::max<int64_t>(256, ((int64_t)1 << 20) / std::max<int64_t>(1, ceil_div64(N, 256)) * 256)});      // (the last: a launch has fewer than 2^32 threads, whatever its tiles)
        if (P < V && (grad || !w_direct)) P = best_piece(P);
        t_logits = pick_tile(f32, N, std::min(P, V), ncu);
        tiles_m = ceil_div64(N, kTiles[f32][t_logits].bm);
        tiles_n = ceil_div64(std::min(P, V), kTiles[f32][t_logits].bn);
        bytes = 0;
        // Few rows (and at least four of everything the class-contiguous forms take four at a time): no operand is laid out.  Its backward pass keeps G of
        // all classes: no more of it than a piece takes, or 2 GiB (a narrow float32 layer would use this form with any number of rows, 65536 x 32 x 100000:
        // 24 GiB; up to there it is worth its memory, 8000 x 32 x 48000: 2.1 against 2.8 ms).
        thin = V >= 4 && H >= 4 && (!grad || (f32 ? 4 : 2) * N * V <= std::max(2 * kBudget, P * per_class)) && prefers_thin();
        if (thin) {
            // 64 rows per block read the kernel least often, 32 give twice the workgroups.  float32, bound by the matrix instructions: up to 32, half the
            // registers (64 / 80 x 1344 x 28165 logits 82 / 120 us, with 64 rows 94 / 143), 16 where a third of two blocks of 32 would be no rows (48: 75, 81 us)
            tiles_n = ceil_div64(V, out_in ? 32 : 64);
            nf = N <= 16 || (f32 && N > 32 && N <= 48) ? 1 : (N <= 32 || f32 || tiles_n * ceil_div64(N, 64) < 2 * ncu ? 2 : 4);
            blocks = ceil_div64(N, 16 * nf);
            if (!grad) {
                part = take(8 * tiles_n * N);
                part_t = labels ? 0 : take(8 * tiles_n * N);
                picked = take(4 * N);
                return;
            }
            g = take((f32 ? 4 : 2) * N * V);
            tsum = take(4 * N);
            weight = labels ? 0 : take(4 * N);
            dbias = take(4 * blocks * V);
            const int64_t wgs = ceil_div64(H, out_in ? 64 : 32) * blocks, chunks = V / 64;
            splits = (int)std::max<int64_t>(1, std::min<int64_t>({(int64_t)64, ceil_div64(4 * ncu, wgs), chunks / 2}));
            acc = splits > 1 ? take(4 * (int64_t)splits * N * H) : 0;
            const int64_t wt_wgs = ceil_div64(H, 64) * ceil_div64(V, 256);        // (dW: 64 x 256 of the product per workgroup, either way round)
            dw_splits = (int)std::max<int64_t>(1, std::min<int64_t>({(int64_t)32, 2 * ncu / wt_wgs, N / 128}));
            acc_w = dw_splits > 1 ? take(4 * (int64_t)dw_splits * H * V) : 0;
            return;
        }
        x = x_direct ? 0 : take(2 * planes * N * Hp);
        w = w_direct ? 0 : take(2 * planes * P * Hp);
        if (!grad) {
            part = take(8 * tiles_n * N);
            part_t = labels ? 0 : take(8 * tiles_n * N);
            picked = take(4 * N);
            carry = P < V ? take(16 * N) : 0;
            return;
        }
        xt = take(2 * planes * H * Np);
        wt = wt_direct ? 0 : take(2 * planes * H * P);
        g = take(2 * planes * N * P);
        gt = take(2 * planes * P * Np);
        tsum = take(4 * N);
        weight = labels ? 0 : take(4 * N);
        dbias = take(4 * tiles_m * kTiles[f32][t_logits].wm * std::min(P, V));
        // dx has few tiles and a long inner dimension, so has dW of a narrow layer: ranges of it, each with float32 sums of its own
        const int64_t pv = std::min(P, V);
        auto tile_for = [&](int64_t M, int64_t N_, int64_t steps) {        // (the large tile if a few ranges of k fill the device with it)
            const int64_t most = std::min<int64_t>(4, std::max<int64_t>(1, steps / 8));
            return M > 64 && tile_count(kTiles[f32][0], M, N_) * most >= ncu * 3 / 4 ? 0 : pick_tile(f32, M, N_, ncu);
        };
        const int64_t steps = up(pv, 64) / deep, steps_w = Np / deep;
        t_dx = tile_for(N, H, steps);
        splits = split_count(t_dx, N, H, steps);
        const int64_t wm = d->kernel_in == 1 ? pv : H, wn = d->kernel_in == 1 ? H : pv;
        t_dw = pick_tile(f32, wm, wn, ncu);
        dw_splits = split_count(t_dw, wm, wn, steps_w);
        acc_w = dw_splits > 1 ? take(4 * (int64_t)dw_splits * H * pv) : 0;
        acc = take(4 * (int64_t)splits * N * H);
    }
};

template <int EPI>
void xent_gemm(bool f32, int tile, int splits, XentGemm& p, hipStream_t st) {
    const Tile& t = kTiles[f32][tile];
    p.tiles_m = (int)ceil_div64(p.M, t.bm);
    p.tiles_n = (int)ceil_div64(p.N, t.bn);
    const dim3 grid((unsigned)(p.tiles_m * p.tiles_n), (unsigned)splits);
    if (f32) {
        if (tile == 0) hipLaunchKernelGGL((rowops::k_xent_gemm<256, 128, 4, 2, EPI, 3>), grid, dim3(512), 0, st, p);
        else if (tile == 1) hipLaunchKernelGGL((rowops::k_xent_gemm<128, 128, 2, 2, EPI, 3>), grid, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((rowops::k_xent_gemm<64, 128, 1, 4, EPI, 3>), grid, dim3(256), 0, st, p);
    } else {
        if (tile == 0) hipLaunchKernelGGL((rowops::k_xent_gemm<256, 256, 2, 4, EPI, 1>), grid, dim3(512), 0, st, p);
        else if (tile == 1) hipLaunchKernelGGL((rowops::k_xent_gemm<128, 128, 2, 2, EPI, 1>), grid, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((rowops::k_xent_gemm<64, 128, 1, 4, EPI, 1>), grid, dim3(256), 0, st, p);
    }
}

// `blocks` workgroups of 256 threads, in as many launches as keep each below 2^32 threads
template <typename F>
void in_launches(int64_t blocks, F&& launch) {
    constexpr int64_t most = 1 << 23;
    for (int64_t b = 0; b < blocks; b += most) launch(b, (unsigned)std::min(most, blocks - b));
}

// Operands to lay out, gathered and launched together
struct Lay {
    rowops::LayJobs jobs{};
    void add(bool transposed, const void* from, int64_t ld, int64_t rows, int64_t cols, uint16_t* to, int64_t ldk, int64_t plane, bool live = false) {
        rowops::LayJob& j = jobs.job[jobs.n++];
        j = {from, ld, rows, cols, to, ldk, plane, transposed, (int32_t)(transposed ? ceil_div64(rows, 64) * (ldk / 64) : ceil_div64(rows * ldk, 2048)), live};
    }
    void launch(bool f32, hipStream_t st) {
        int64_t blocks = 0;
        for (int i = 0; i < jobs.n; ++i) blocks += jobs.job[i].blocks;
        in_launches(blocks, [&](int64_t first, unsigned count) {
            jobs.first = (int32_t)first;
            if (f32) hipLaunchKernelGGL(rowops::k_xent_lay<float>, dim3(count), dim3(256), 0, st, jobs);
            else hipLaunchKernelGGL(rowops::k_xent_lay<bf16_t>, dim3(count), dim3(256), 0, st, jobs);
        });
        jobs.n = 0;
    }
};

const void* at(const dimn_output_loss* d, const void* base, int64_t elements) { return (const char*)base + elements * (d->type == DIMN_TYPE_F32 ? 4 : 2); }

// the logits' operands of the piece that starts at class c0 and has pv classes
void xent_logits(const XentPlan& q, char* ws, int64_t c0, int64_t pv, XentGemm& p, Lay& lay) {
    const dimn_output_loss* d = q.d;
    p = XentGemm{};
    if (q.x_direct) { p.A = (const uint16_t*)d->x; p.lda = d->x_row; }
    else {
        p.A = (const uint16_t*)(ws + q.x); p.lda = q.Hp; p.a_plane = q.N * q.Hp;
        if (c0 == 0) lay.add(false, d->x, d->x_row, q.N, q.H, (uint16_t*)(ws + q.x), q.Hp, p.a_plane);
    }
    if (q.w_direct) { p.B = (const uint16_t*)at(d, d->kernel, c0 * d->kernel_out); p.ldb = d->kernel_out; }
    else {
        p.B = (const uint16_t*)(ws + q.w); p.ldb = q.Hp; p.b_plane = q.P * q.Hp;
        if (q.out_in) lay.add(false, at(d, d->kernel, c0 * d->kernel_out), d->kernel_out, pv, q.H, (uint16_t*)(ws + q.w), q.Hp, p.b_plane);
        else lay.add(true, at(d, d->kernel, c0), d->kernel_in, pv, q.H, (uint16_t*)(ws + q.w), q.Hp, p.b_plane);
    }
    p.M = (int)q.N; p.N = (int)pv;
    p.ksteps = (int)(q.Hp / q.deep);
    p.bias = d->bias ? d->bias + c0 : nullptr;
    p.target = d->target; p.target_row = d->target_row; p.target_kind = d->target_kind;
    if (!q.labels) p.target = (const char*)d->target + c0 * (d->target_kind == DIMN_TARGET_F32 ? 4 : 2);
    p.class0 = c0; p.classes = q.V;
}

// workgroups of `units` x the row blocks (thin_place)
int64_t thin_groups(const XentPlan& q, int64_t units) { return (units < 64 ? units : up(units, 8)) * q.blocks; }
template <typename T> constexpr int kRows = sizeof(T) == 2 ? 4 : 2;      // the largest XentPlan::nf
// k_xent_thin with four waves over `k` elements of the inner dimension.  Chunks in fours pay where a wave has several rounds of them: k-contiguous from
// 64 chunks on (128 x 2922 x 25664 float32 dx: 356 us one by one, 295 in fours; 64 x 800 x 50000 bfloat16 logits: 27 and 33), class-contiguous
// float32 from 512 (128 x 25664 logits, 1000 wide: 106 and 96 us; 500 wide: 53 and 55).  Class-contiguous bfloat16 gains
// nothing (12 x 2000 x 40000: 37 and 41 us).  float32 keeps a second round in flight (295 against 313 us), bfloat16 does
// better with the registers (64 x 1500 x 20000: 21 against 23).
template <typename T, bool VC, int NF, int EPI>
void thin_launch(const rowops::Thin& p, int64_t k, unsigned groups, int tiles, int ranges, int blocks, hipStream_t st) {
    constexpr int FOURS = VC ? (sizeof(T) == 4 ? 1 : 0) : (sizeof(T) == 4 ? 2 : 1);
    if constexpr (FOURS > 0)
        if (k >= (VC ? 512 : (sizeof(T) == 2 ? 2048 : 1024))) {
            hipLaunchKernelGGL((rowops::k_xent_thin<T, VC, NF, EPI, 4, FOURS>), dim3(groups), dim3(256), 0, st, p, tiles, ranges, blocks);
            return;
        }
    hipLaunchKernelGGL((rowops::k_xent_thin<T, VC, NF, EPI, 4, 0>), dim3(groups), dim3(256), 0, st, p, tiles, ranges, blocks);
}
// the logits' product: epilogue XE_LSE or XE_GRAD
template <typename T, int EPI>
void xent_thin(const XentPlan& q, const rowops::Thin& p, hipStream_t st) {
    const unsigned groups = (unsigned)thin_groups(q, q.tiles_n);
    const int tiles = (int)q.tiles_n, blocks = (int)q.blocks;
    // sixteen waves per workgroup while that leaves CUs to spare and every wave still has chunks of k
    const bool deep = q.nf <= 2 && q.tiles_n * q.blocks <= q.ncu && q.H >= 512;
#define THIN(VC, NF)                                                                                                                              \
    do {                                                                                                                                          \
        if (NF <= 2 && deep) hipLaunchKernelGGL((rowops::k_xent_thin<T, VC, NF <= 2 ? NF : 1, EPI, 16, 0>), dim3(groups), dim3(1024), 0, st, p, tiles, 1, blocks);  \
        else thin_launch<T, VC, NF, EPI>(p, q.H, groups, tiles, 1, blocks, st);                                                                  \
    } while (0)
    if (q.out_in) { if (q.nf == 1) THIN(false, 1); else if (q.nf == 2) THIN(false, 2); else THIN(false, kRows<T>); }
    else { if (q.nf == 1) THIN(true, 1); else if (q.nf == 2) THIN(true, 2); else THIN(true, kRows<T>); }
#undef THIN
}
rowops::Thin xent_thin_logits(const XentPlan& q) {
    const dimn_output_loss* d = q.d;
    rowops::Thin p{};
    p.A = d->x; p.lda = d->x_row;
    p.B = d->kernel; p.ldb = q.out_in ? d->kernel_out : d->kernel_in;
    p.M = q.N; p.N = q.V; p.K = q.H;
    p.bias = d->bias; p.target = d->target; p.target_row = d->target_row; p.target_kind = d->target_kind;
    return p;
}
// the rows with a gradient; of a profile their sums are made here (ws + tsum), and their dloss stands at ws + weight
rowops::LiveRows xent_live(const XentPlan& q, char* ws, const float* dloss, hipStream_t st) {
    const dimn_output_loss* d = q.d;
    const unsigned threads = q.N < 1 << 20 ? 1024 : 256;        // (a launch has fewer than 2^32 of them; so many rows fill the device anyhow)
    float* weight = (float*)(ws + q.weight);
    if (!q.labels) hipLaunchKernelGGL(rowops::k_xent_tsum, dim3((unsigned)q.N), dim3(threads), 0, st, d->target, d->target_kind, d->target_row, q.V, dloss, (float*)(ws + q.tsum), weight);
    if (!q.labels) return {weight, (const char*)weight, 4, 0, 0, UINT32_MAX};
    if (d->target_kind == DIMN_TARGET_I64) return {dloss, (const char*)d->target, 8, 4, UINT32_MAX, (uint32_t)(q.V - 1)};
    return {dloss, (const char*)d->target, 4, 0, 0, (uint32_t)(q.V - 1)};
}
rowops::SplitSum split_sum(const float* acc, int splits, int64_t rows, int64_t cols, void* out, int64_t ld) {
    const int32_t per = rows * cols >= 1 << 20 ? 4 : 1;          // (4096 x 2048 bfloat16, two splits: 32 us one by one, 21 by four)
    return {acc, rows * cols, splits, (int32_t)ceil_div64(rows * cols, 256 * per), per, rows, cols, out, ld};
}
void xent_finish(bool f32, rowops::XentFinish& f, hipStream_t st) {
    in_launches((int64_t)f.m[0].blocks + f.m[1].blocks + (f.dbias && f.parts ? ceil_div64(f.classes, 256) : 0), [&](int64_t first, unsigned count) {
        f.first = (int32_t)first;
        if (f32) hipLaunchKernelGGL(rowops::k_xent_finish<float>, dim3(count), dim3(256), 0, st, f);
        else hipLaunchKernelGGL(rowops::k_xent_finish<bf16_t>, dim3(count), dim3(256), 0, st, f);
    });
}
// the bias gradient of `classes` classes from `parts` rows of partial sums in the workspace
void finish_bias(rowops::XentFinish& f, const XentPlan& q, char* ws, int64_t classes, int parts, float* dbias) {
    f.part = (const float*)(ws + q.dbias); f.part_ld = classes; f.parts = parts; f.classes = classes; f.dbias = dbias;
}
template <typename T>
void xent_thin_backward(const XentPlan& q, char* ws, const float* dloss, const float* lse, void* dx, int64_t dx_row, void* dkernel, int64_t dk_in, int64_t dk_out, float* dbias, hipStream_t st) {
    const dimn_output_loss* d = q.d;
    T* G = (T*)(ws + q.g);
    const rowops::LiveRows live = xent_live(q, ws, dloss, st);
    rowops::Thin p = xent_thin_logits(q);
    p.lse = lse; p.dloss = live.dloss; p.tsum = (float*)(ws + q.tsum);
    p.G = G; p.ldg = q.V;
    p.dbias_part = dbias ? (q.blocks == 1 ? dbias : (float*)(ws + q.dbias)) : nullptr;
    xent_thin<T, rowops::XE_GRAD>(q, p, st);
    // dx[n][h] = sum over the classes: the classes are the inner dimension now
    rowops::Thin a{};
    a.A = G; a.lda = q.V; a.B = d->kernel; a.ldb = p.ldb;
    a.M = q.N; a.N = q.H; a.K = q.V; a.acc = (float*)(ws + q.acc);
    a.C = dx; a.ldc = dx_row;
    rowops::ThinDw w{};
    w.n = q.N;
    if (dk_in == 1) { w.P = G; w.ldp = q.V; w.Q = d->x; w.ldq = d->x_row; w.na = q.V; w.nb = q.H; w.ldc = dk_out; }
    else { w.P = d->x; w.ldp = d->x_row; w.Q = G; w.ldq = q.V; w.na = q.H; w.nb = q.V; w.ldc = dk_in; }
    w.C = dkernel;
    w.tiles_b = (int)ceil_div64(w.nb, 256);
    w.tiles = w.tiles_b * (int)ceil_div64(w.na, 64);
    w.ranges = q.dw_splits;
    w.acc = (float*)(ws + q.acc_w);
    w.live = live;
    const bool vc = q.out_in;
    const int tiles = (int)ceil_div64(q.H, vc ? 64 : 32), dx_groups = (int)thin_groups(q, (int64_t)tiles * q.splits);
    const dim3 grid((unsigned)(dx_groups + w.tiles * w.ranges));
    const int ranges = q.splits, blocks = (int)q.blocks;
    if (grid.x <= 8 * (unsigned)q.ncu) {
#define BOTH(NF, EPI)                                                                                                                                      \
    do {                                                                                                                                                   \
        if (vc) hipLaunchKernelGGL((rowops::k_xent_thin_both<T, true, NF, EPI>), grid, dim3(256), 0, st, a, w, dx_groups, tiles, ranges, blocks);          \
        else hipLaunchKernelGGL((rowops::k_xent_thin_both<T, false, NF, EPI>), grid, dim3(256), 0, st, a, w, dx_groups, tiles, ranges, blocks);            \
    } while (0)
        if (ranges == 1) { if (q.nf == 1) BOTH(1, rowops::XE_STORE); else if (q.nf == 2) BOTH(2, rowops::XE_STORE); else BOTH(kRows<T>, rowops::XE_STORE); }
        else { if (q.nf == 1) BOTH(1, rowops::XE_ADD); else if (q.nf == 2) BOTH(2, rowops::XE_ADD); else BOTH(kRows<T>, rowops::XE_ADD); }
#undef BOTH
    } else {
#define DX(NF, EPI)                                                                                                                                        \
    do {                                                                                                                                                   \
        if (vc) thin_launch<T, true, NF, EPI>(a, q.V / ranges, (unsigned)dx_groups, tiles, ranges, blocks, st);                                           \
        else thin_launch<T, false, NF, EPI>(a, q.V / ranges, (unsigned)dx_groups, tiles, ranges, blocks, st);                                             \
    } while (0)
        if (ranges == 1) { if (q.nf == 1) DX(1, rowops::XE_STORE); else if (q.nf == 2) DX(2, rowops::XE_STORE); else DX(kRows<T>, rowops::XE_STORE); }
        else { if (q.nf == 1) DX(1, rowops::XE_ADD); else if (q.nf == 2) DX(2, rowops::XE_ADD); else DX(kRows<T>, rowops::XE_ADD); }
#undef DX
        const dim3 gw((unsigned)(w.tiles * w.ranges));
        hipLaunchKernelGGL((rowops::k_xent_thin_dw<T>), gw, dim3(256), 0, st, w);
    }
    rowops::XentFinish f{};
    if (q.splits > 1) f.m[0] = split_sum((const float*)(ws + q.acc), q.splits, q.N, q.H, dx, dx_row);
    if (w.ranges > 1) f.m[1] = split_sum(w.acc, w.ranges, w.na, w.nb, w.C, w.ldc);
    if (q.blocks > 1) finish_bias(f, q, ws, q.V, (int)q.blocks, dbias);
    xent_finish(q.f32, f, st);
}

int xent_check(const char* who, const dimn_output_loss* d) {
    if (!d) return dimn_fail(DIMN_ERR_ARG, "%s: null description", who);
    if (d->type != DIMN_TYPE_F32 && d->type != DIMN_TYPE_BF16) return dimn_fail(DIMN_ERR_UNSUP, "%s: element type %d (DIMN_TYPE_F32 or DIMN_TYPE_BF16)", who, d->type);
    if (d->target_kind < DIMN_TARGET_I32 || d->target_kind > DIMN_TARGET_BF16) return dimn_fail(DIMN_ERR_UNSUP, "%s: target kind %d", who, d->target_kind);
    const int64_t most = 1 << 22;
    if (d->rows < 0 || d->rows > most || d->width < 1 || d->width > most || d->classes < 1 || d->classes > most)
        return dimn_fail(DIMN_ERR_ARG, "%s: %lld rows, width %lld, %lld classes (each up to 2^22, the latter two at least 1)", who, (long long)d->rows, (long long)d->width, (long long)d->classes);
    if (ceil_div64(d->rows, 64) * ceil_div64(d->classes, 128) > INT32_MAX || ceil_div64(d->width, 64) * ceil_div64(std::max(d->rows, d->classes), 64) > INT32_MAX)
        return dimn_fail(DIMN_ERR_ARG, "%s: %lld rows, width %lld, %lld classes are too many tiles for one launch", who, (long long)d->rows, (long long)d->width, (long long)d->classes);
    if (d->kernel_in != 1 && d->kernel_out != 1) return dimn_fail(DIMN_ERR_ARG, "%s: one of the kernel's strides (%lld, %lld) has to be 1", who, (long long)d->kernel_in, (long long)d->kernel_out);
    if (d->rows > 0 && (!d->x || !d->kernel || !d->target)) return dimn_fail(DIMN_ERR_ARG, "%s: null array", who);
    return DIMN_OK;
}
int xent_space(const char* who, const XentPlan& q, const void* workspace, int64_t bytes) {
    if (!workspace || ((uintptr_t)workspace & 255) || bytes < (int64_t)q.bytes)
        return dimn_fail(DIMN_ERR_ARG, "%s: a 256-byte aligned workspace of %lld bytes is needed, got %lld", who, (long long)q.bytes, (long long)bytes);
    return DIMN_OK;
}
}  // namespace

extern "C" int dimn_linear_cross_entropy_workspace(const dimn_output_loss* d, int32_t grad, int64_t* bytes) {
    const char* who = "dimn_linear_cross_entropy_workspace";
    CHK(xent_check(who, d));
    if (!bytes) return dimn_fail(DIMN_ERR_ARG, "%s: null", who);
    if (d->rows == 0) { *bytes = 0; return DIMN_OK; }            // (nothing to plan: a plan divides by the number of row blocks)
    OnDevice on;
    CHK(on.enter(who, d->device_id));
    XentPlan q;
    q.make(d, grad != 0, compute_units(d->device_id));
    *bytes = (int64_t)q.bytes;
    return DIMN_OK;
}

extern "C" int dimn_linear_cross_entropy(const dimn_output_loss* d, void* stream, float* loss, float* lse, void* workspace, int64_t workspace_bytes) {
    const char* who = "dimn_linear_cross_entropy";
    CHK(xent_check(who, d));
    if (d->rows == 0) return DIMN_OK;
    if (!loss || !lse) return dimn_fail(DIMN_ERR_ARG, "%s: null array", who);
    OnDevice on;
    CHK(on.enter(who, d->device_id));
    hipStream_t st = (hipStream_t)stream;
    XentPlan q;
    q.make(d, false, compute_units(d->device_id));
    CHK(xent_space(who, q, workspace, workspace_bytes));
    char* ws = (char*)workspace;
    rowops::XentRows r{};
    r.part = (const float2*)(ws + q.part);
    r.part_t = q.labels ? nullptr : (const float2*)(ws + q.part_t);
    r.picked = (const float*)(ws + q.picked);
    r.rows = q.N; r.classes = q.V;
    r.target = d->target; r.target_kind = d->target_kind;
    r.carry = (float4*)(ws + q.carry);
    r.loss = loss; r.lse = lse;
    auto join = [&](int64_t tiles, bool first, bool last) {
        r.tiles = tiles; r.first = first; r.last = last;
        r.per = 1;                                               // rows per workgroup: fewer, with more strands over the tiles each, while a strand has more than two
        while (r.per < 64 && 2 * r.per <= q.N && (r.per < 4 || 1024 / (2 * r.per) * 2 >= tiles)) r.per *= 2;
        hipLaunchKernelGGL(rowops::k_xent_lse, dim3((unsigned)ceil_div64(q.N, r.per)), dim3(1024), 0, st, r);
    };
    if (q.thin) {
        rowops::Thin p = xent_thin_logits(q);
        p.part = (float2*)(ws + q.part);
        p.part_t = q.labels ? nullptr : (float2*)(ws + q.part_t);
        p.picked = (float*)(ws + q.picked);
        if (q.f32) xent_thin<float, rowops::XE_LSE>(q, p, st);
        else xent_thin<bf16_t, rowops::XE_LSE>(q, p, st);
        join(q.tiles_n, true, true);
    } else for (int64_t c0 = 0; c0 < q.V; c0 += q.P) {
        const int64_t pv = std::min(q.P, q.V - c0);
        XentGemm p;
        Lay lay;
        xent_logits(q, ws, c0, pv, p, lay);
        lay.launch(q.f32, st);
        p.part = (float2*)(ws + q.part);
        if (!q.labels) p.part_t = (float2*)(ws + q.part_t);
        p.picked = (float*)(ws + q.picked);
        xent_gemm<rowops::XE_LSE>(q.f32, q.t_logits, 1, p, st);
        join(ceil_div64(pv, kTiles[q.f32][q.t_logits].bn), c0 == 0, c0 + pv == q.V);
    }
    HIPCHK(hipGetLastError());
    return DIMN_OK;
}

extern "C" int dimn_linear_cross_entropy_grad(const dimn_output_loss* d, void* stream, const float* dloss, const float* lse, void* dx, int64_t dx_row,
                                              void* dkernel, int64_t dkernel_in, int64_t dkernel_out, float* dbias, void* workspace, int64_t workspace_bytes) {
    const char* who = "dimn_linear_cross_entropy_grad";
    CHK(xent_check(who, d));
    if (d->rows == 0) return dimn_fail(DIMN_ERR_ARG, "%s: no rows", who);
    if (!dkernel || !dloss || !lse || !dx) return dimn_fail(DIMN_ERR_ARG, "%s: null array", who);
    if (dkernel_in != 1 && dkernel_out != 1) return dimn_fail(DIMN_ERR_ARG, "%s: one of the strides of dkernel (%lld, %lld) has to be 1", who, (long long)dkernel_in, (long long)dkernel_out);
    OnDevice on;
    CHK(on.enter(who, d->device_id));
    hipStream_t st = (hipStream_t)stream;
    XentPlan q;
    q.make(d, true, compute_units(d->device_id));
    CHK(xent_space(who, q, workspace, workspace_bytes));
    char* ws = (char*)workspace;
    if (q.thin) {
        if (q.f32) xent_thin_backward<float>(q, ws, dloss, lse, dx, dx_row, dkernel, dkernel_in, dkernel_out, dbias, st);
        else xent_thin_backward<bf16_t>(q, ws, dloss, lse, dx, dx_row, dkernel, dkernel_in, dkernel_out, dbias, st);
        HIPCHK(hipGetLastError());
        return DIMN_OK;
    }
    const rowops::LiveRows live = xent_live(q, ws, dloss, st);
    Lay lay;
    lay.jobs.rows = live;
    uint16_t* xt = (uint16_t*)(ws + q.xt);
    const int64_t xt_plane = q.H * q.Np;
    lay.add(true, d->x, d->x_row, q.H, q.N, xt, q.Np, xt_plane, true);
    const bool dk_out_in = dkernel_in == 1;
    for (int64_t c0 = 0; c0 < q.V; c0 += q.P) {
        const int64_t pv = std::min(q.P, q.V - c0), ldg = up(pv, 64);
        XentGemm p;
        xent_logits(q, ws, c0, pv, p, lay);
        uint16_t* wt = (uint16_t*)(ws + q.wt);
        const int64_t wt_plane = q.H * ldg;
        if (!q.wt_direct) {
            if (q.out_in) lay.add(true, at(d, d->kernel, c0 * d->kernel_out), d->kernel_out, q.H, pv, wt, ldg, wt_plane);
            else lay.add(false, at(d, d->kernel, c0), d->kernel_in, q.H, pv, wt, ldg, wt_plane);
        }
        lay.launch(q.f32, st);
        p.lse = lse; p.dloss = live.dloss; p.tsum = (float*)(ws + q.tsum);
        p.G = (uint16_t*)(ws + q.g); p.ldg = ldg; p.g_plane = q.N * ldg;
        p.GT = (uint16_t*)(ws + q.gt); p.ldgt = q.Np; p.gt_plane = pv * q.Np;
        p.dbias_part = (float*)(ws + q.dbias); p.dbias_ld = pv;
        xent_gemm<rowops::XE_GRAD>(q.f32, q.t_logits, 1, p, st);
        // dx += G W^T
        XentGemm a{};
        a.A = p.G; a.lda = ldg; a.a_plane = p.g_plane;
        if (q.wt_direct) { a.B = (const uint16_t*)at(d, d->kernel, c0); a.ldb = d->kernel_in; }
        else { a.B = wt; a.ldb = ldg; a.b_plane = wt_plane; }
        a.M = (int)q.N; a.N = (int)q.H;
        a.ksteps = (int)(ldg / q.deep);
        a.acc = (float*)(ws + q.acc); a.acc_split = q.N * q.H; a.acc_first = c0 == 0;
        xent_gemm<rowops::XE_ADD>(q.f32, q.t_dx, q.splits, a, st);
        // dW of the piece
        XentGemm w{};
        w.ksteps = (int)(q.Np / q.deep);
        const uint16_t *gt = p.GT, *xa = xt;
        if (dk_out_in) {
            w.A = gt; w.lda = q.Np; w.a_plane = p.gt_plane; w.M = (int)pv;
            w.B = xa; w.ldb = q.Np; w.b_plane = xt_plane; w.N = (int)q.H;
            w.C = const_cast<void*>(at(d, dkernel, c0 * dkernel_out)); w.ldc = dkernel_out;
        } else {
            w.A = xa; w.lda = q.Np; w.a_plane = xt_plane; w.M = (int)q.H;
            w.B = gt; w.ldb = q.Np; w.b_plane = p.gt_plane; w.N = (int)pv;
            w.C = const_cast<void*>(at(d, dkernel, c0)); w.ldc = dkernel_in;
        }
        rowops::XentFinish f{};
        if (q.dw_splits > 1) {
            w.acc = (float*)(ws + q.acc_w); w.acc_split = (int64_t)w.M * w.N; w.acc_first = 1;
            xent_gemm<rowops::XE_ADD>(q.f32, q.t_dw, q.dw_splits, w, st);
            f.m[0] = split_sum(w.acc, q.dw_splits, w.M, w.N, w.C, w.ldc);
        } else xent_gemm<rowops::XE_STORE>(q.f32, q.t_dw, 1, w, st);
        if (c0 + pv == q.V) f.m[1] = split_sum((const float*)(ws + q.acc), q.splits, q.N, q.H, dx, dx_row);
        if (dbias) finish_bias(f, q, ws, pv, (int)(q.tiles_m * kTiles[q.f32][q.t_logits].wm), dbias + c0);
        xent_finish(q.f32, f, st);
    }
    HIPCHK(hipGetLastError());
    return DIMN_OK;
}
