// linear.hip -- the entry points of the fully connected layers (include/umr_nn.h): argument checks, and the plan of every product --
// which kernel, how many parts.  The kernels are in linear_kernels.h, compiled once for each type (linear_f32 / _bf16 / _f16.hip).
#include "linear_shared.h"

namespace umr_linear {
namespace {

// Which kernel, and how many parts of the contraction.
Plan plan(int kind, long nq, long np, long nc, int G, int dtype) {
    Plan pl;
    const int es = dtype == UMR_F32 ? 4 : 2;
    // Few rows, streamed weights against tiles: fp32 8192 x 8192 of 32 rows 67 / 139 us forward, 74 / 130 dx, of 64 rows 125 / 143, 107 /
    // 132; bf16 of 64 rows 57 / 75, 45 / 80; at 1024 x 1024 the two are within 5 us of each other.
    pl.few = kind != GRAD_WEIGHT && nq <= 64;
    // A short contraction, outer products against the best tile: up to 16 rows 1024 x 1024 4.7 / 5.5 us, 8192 x 8192 45 / 100, bf16 29 /
    // 73.  Beyond, the longer column gathers have to be paid for by a large result: fp32 of 32 rows 1024 x 1024 6.8 / 5.2, 2048 x 2048
    // 9.6 / 9.8, 4096 x 4096 19 / 26, of 64 rows 9.7 / 6.1, 13.2 / 12.5, 30 / 34, 8192 x 8192 114 / 127; bf16 4096 x 4096 of 32 rows 20.8 /
    // 21.4, of 64 34 / 21.
    pl.outer = kind == GRAD_WEIGHT && np >= 64 && nq >= 64 && ceil_div(nq, 64) <= 65535 &&
               (nc <= 16 || (nc <= (dtype == UMR_F32 ? 64 : 32) && (double)nq * np * G >= 8388608.));
    pl.tile = 0;
    long groups, step;
    if (pl.few) {
        groups = ceil_div(np, kind == FORWARD ? 32 : 64) * G;
        step = 64 / es * FEW_WAVES * 4;                       // at least 4 loads deep in every wave
    } else {
        // Rounds of the 256 CUs times the work of a tile, where a smaller tile reads more for each product.  Measured, 64 / 128 / 256
        // wide: fp32 10000 x 1011 x 350 78 / 110 us, 4096^3 1240 / 1170 us; bf16 8192 x 4096 x 4096 - / 370 / 300 us, 32 heads of
        // 333 x 512 x 1024 40 / 35 / 45 us; fp16 777 x 1001 x 515 12 / 19 us.  The widest tile starts and ends most slowly, so it has
        // to find a contraction of 512: 8192 x 8192 of 128 fp32 199 / 219 us, 256 343 / 353, 512 651 / 630; bf16 of 64 - / 71 / 104,
        // 256 - / 111 / 133, 512 - / 176 / 173.
        const int widest = (dtype == UMR_F32 ? T128x128 : T256x256) - (nc < 512);
        double best = 0;
        groups = 1;
        for (int i = T64x64; i <= widest; ++i) {
            const long w = TILE[i], n = ceil_div(nq, w) * ceil_div(np, w) * G;
            const double cost = (double)ceil_div(n, 256) * (w * w + (dtype == UMR_F32 ? 16 : 128) * w);
            if (i == T64x64 || cost < best) { best = cost; pl.tile = i; groups = n; }
        }
        step = 128 / es * 4;
    }
    long S = pl.outer ? 1 : groups > 0 ? 256 / groups : 1;
    const long most = nc / step;
    S = S < most ? S : most;
    S = S < 1 ? 1 : S > 64 ? 64 : S;
    const long unit = pl.few ? 64 / es : 128 / es;
    pl.c_split = ceil_div(ceil_div(nc > 0 ? nc : 1, S), unit) * unit;
    pl.S = (int)ceil_div(nc > 0 ? nc : 1, pl.c_split);
    return pl;
}

size_t plan_bytes(const Plan &pl, long nq, long np, int G) { return pl.S > 1 ? (size_t)pl.S * G * nq * np * sizeof(float) : 0; }

bool sizes_ok(long M, long N, long K, int G, int dtype) {
    const long lim = 1L << 27;                                // (a launch has at most 2^32 threads)
    if (M < 0 || N < 0 || K < 0 || G < 1 || G > 65535 || M >= lim || N >= lim || K >= lim) return false;
    if (dtype != UMR_F32 && dtype != UMR_BF16 && dtype != UMR_F16) return false;
    const long wide = N > K ? N : K;
    return (double)M * G * wide < 7e13 && (double)G * N * K < 7e13;
}

int run(int kind, Product pr, const Epilogue &e, int dtype, void *workspace, size_t workspace_bytes, hipStream_t st) {
    if (pr.nq == 0 || pr.np == 0) return UMR_OK;              // nothing to write
    const Plan pl = plan(kind, pr.nq, pr.np, pr.nc, pr.G, dtype);
    if (plan_bytes(pl, pr.nq, pr.np, pr.G) > workspace_bytes || (pl.S > 1 && !workspace)) return UMR_ERR_ARG;
    if (dtype == UMR_F32) return run_product<float>(kind, pl, pr, e, workspace, st);
    if (dtype == UMR_BF16) return run_product<bf16_t>(kind, pl, pr, e, workspace, st);
    return run_product<f16_t>(kind, pl, pr, e, workspace, st);
}

bool strides_ok(long row, long head) { return row >= 0 && head >= 0; }

long act_grad_rows(long M, long N, int G) {                  // rows per workgroup of k_linear_act_grad
    const long cols = ceil_div(N, 256) * G;
    const long blocks = ceil_div(2048, cols > 0 ? cols : 1);
    long rows = ceil_div(M, blocks);
    return rows < 32 ? 32 : rows;
}

}  // namespace
}  // namespace umr_linear

using namespace umr_linear;

extern "C" {

size_t umr_linear_forward_workspace_bytes(long M, long N, long K, int G, int dtype) {
    if (!sizes_ok(M, N, K, G, dtype) || M == 0 || N == 0) return 0;
    return plan_bytes(plan(FORWARD, M, N, K, G, dtype), M, N, G);
}
size_t umr_linear_grad_input_workspace_bytes(long M, long N, long K, int G, int dtype) {
    if (!sizes_ok(M, N, K, G, dtype) || M == 0 || K == 0) return 0;
    return plan_bytes(plan(GRAD_INPUT, M, K, N, G, dtype), M, K, G);
}
size_t umr_linear_grad_weight_workspace_bytes(long M, long N, long K, int G, int dtype) {
    if (!sizes_ok(M, N, K, G, dtype) || N == 0 || K == 0) return 0;
    return plan_bytes(plan(GRAD_WEIGHT, N, K, M, G, dtype), N, K, G);
}
size_t umr_linear_grad_act_workspace_bytes(long M, long N, int G) {
    if (!sizes_ok(M, N, 0, G, UMR_F32) || M == 0) return 0;
    const long blocks = ceil_div(M, act_grad_rows(M, N, G));
    return blocks > 1 ? (size_t)blocks * 2 * G * N * sizeof(float) : 0;
}

int umr_linear_forward(const void *x, long x_row, long x_head, const void *w, long w_row, long w_head, const void *bias, const void *residual,
                       long r_row, long r_head, void *y, void *z, long M, long N, long K, int G, int dtype, int act, float slope,
                       void *workspace, size_t workspace_bytes, void *stream) {
    if (!sizes_ok(M, N, K, G, dtype) || act < UMR_ACT_NONE || act > UMR_ACT_SILU || !strides_ok(x_row, x_head) || !strides_ok(w_row, w_head) ||
        (residual && !strides_ok(r_row, r_head)) || (act == UMR_ACT_LEAKY_RELU && !(slope >= 0.f)))
        return UMR_ERR_ARG;
    if (M == 0 || N == 0) return UMR_OK;
    if (!y || (K > 0 && (!x || !w))) return UMR_ERR_ARG;
    Product pr = {{w, w_row, w_head}, {x, x_row, x_head}, N, M, K, 0, G, 1};
    Epilogue e = {bias, residual, r_row, r_head, y, z, (long)G * N, N, act, slope, nullptr};
    return run(FORWARD, pr, e, dtype, workspace, workspace_bytes, (hipStream_t)stream);
}

int umr_linear_grad_input(const void *dz, long dz_row, long dz_head, const void *w, long w_row, long w_head, void *dx, long M, long N, long K,
                          int G, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
    if (!sizes_ok(M, N, K, G, dtype) || !strides_ok(dz_row, dz_head) || !strides_ok(w_row, w_head)) return UMR_ERR_ARG;
    if (M == 0 || K == 0) return UMR_OK;
    if (!dx || (N > 0 && (!dz || !w))) return UMR_ERR_ARG;
    Product pr = {{w, w_row, w_head}, {dz, dz_row, dz_head}, K, M, N, 0, G, 1};
    Epilogue e = {nullptr, nullptr, 0, 0, dx, nullptr, (long)G * K, K, UMR_ACT_NONE, 0.f, nullptr};
    return run(GRAD_INPUT, pr, e, dtype, workspace, workspace_bytes, (hipStream_t)stream);
}

int umr_linear_grad_weight(const void *dz, long dz_row, long dz_head, const void *x, long x_row, long x_head, void *dw, long M, long N, long K,
                           int G, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
    if (!sizes_ok(M, N, K, G, dtype) || !strides_ok(dz_row, dz_head) || !strides_ok(x_row, x_head)) return UMR_ERR_ARG;
    if (N == 0 || K == 0) return UMR_OK;
    if (!dw || (M > 0 && (!dz || !x))) return UMR_ERR_ARG;
    Product pr = {{x, x_row, x_head}, {dz, dz_row, dz_head}, K, N, M, 0, G, 1};
    Epilogue e = {nullptr, nullptr, 0, 0, dw, nullptr, K, N * K, UMR_ACT_NONE, 0.f, nullptr};
    return run(GRAD_WEIGHT, pr, e, dtype, workspace, workspace_bytes, (hipStream_t)stream);
}

int umr_linear_grad_act(const void *gy, long g_row, long g_head, const void *z, void *dz, void *db, void *dr, long M, long N, int G, int dtype,
                        int act, float slope, void *workspace, size_t workspace_bytes, void *stream) {
    if (!sizes_ok(M, N, 0, G, dtype) || act < UMR_ACT_NONE || act > UMR_ACT_SILU || !strides_ok(g_row, g_head) ||
        (act == UMR_ACT_LEAKY_RELU && !(slope >= 0.f)) || (M > 0 && N > 0 && ((act == UMR_ACT_NONE) != (dz == nullptr) || (dz && !z))))
        return UMR_ERR_ARG;
    if (N == 0 || (M == 0 && !db && !dr) || (!dz && !db && !dr)) return UMR_OK;
    if (M > 0 && !gy) return UMR_ERR_ARG;
    const long rows = M > 0 ? act_grad_rows(M, N, G) : 32, blocks = M > 0 ? ceil_div(M, rows) : 1;
    float *part = nullptr;
    if (blocks > 1 && (db || dr)) {
        if (!workspace || workspace_bytes < (size_t)blocks * 2 * G * N * sizeof(float)) return UMR_ERR_ARG;
        part = (float *)workspace;
    }
    if (blocks > 65535) return UMR_ERR_ARG;
    const ActGrad a = {gy, z, g_row, g_head, dz, db, dr, part, M, N, rows, blocks, G, act, slope};
    if (dtype == UMR_F32) return run_act_grad<float>(a, (hipStream_t)stream);
    if (dtype == UMR_BF16) return run_act_grad<bf16_t>(a, (hipStream_t)stream);
    return run_act_grad<f16_t>(a, (hipStream_t)stream);
}

}  // extern "C"
