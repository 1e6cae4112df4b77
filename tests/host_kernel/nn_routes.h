// nn_routes.h -- TEST INFRASTRUCTURE, compiled through nn_tu.cpp (-DUMR_TU='"nn_routes.h"'): the plan of a product of csrc/linear.hip,
// and every tile of csrc/linear_kernels.h at sizes that its plan would give to another kernel.
#include "../../umr_amd/csrc/linear.hip"
#include "../../umr_amd/csrc/linear_kernels.h"

namespace umr_linear {
template int run_product<float>(int, const Plan &, Product, Epilogue, void *, hipStream_t);
template int run_product<bf16_t>(int, const Plan &, Product, Epilogue, void *, hipStream_t);
template int run_product<f16_t>(int, const Plan &, Product, Epilogue, void *, hipStream_t);
template int run_act_grad<float>(const ActGrad &, hipStream_t);
template int run_act_grad<bf16_t>(const ActGrad &, hipStream_t);
template int run_act_grad<f16_t>(const ActGrad &, hipStream_t);
}  // namespace umr_linear

// a product with tiles of 64, at most `most` workgroups a launch
template <class T> static int in_launches_of(long most, int kind, Product pr, const Epilogue &e) {
    return launch_tile<T, 2, 2, 1, 1>(kind, pr, e, nullptr, most);
}

extern "C" {
// 0: few rows, 1: outer products, else the edge of the tile; parts: of the contraction.  Sizes of the product, not of the layer.
int nn_route(int kind, long nq, long np, long nc, int G, int dtype, int *parts) {
    const Plan pl = plan(kind, nq, np, nc, G, dtype);
    *parts = pl.S;
    return pl.few ? 0 : pl.outer ? 1 : TILE[pl.tile];
}

// out[q,g,p] = act(sum_c Q[q,g,c] P[g,p,c] + bias[g,p]) + res[q,g,p] (GRAD_WEIGHT: out[g,q,p]) with tiles of `tile`, whatever the plan says;
// most > 0: with tiles of 64 and at most that many workgroups a launch
int nn_run_tile(int kind, int tile, int dtype, const void *P, long p_row, long p_head, const void *Q, long q_row, long q_head, const void *bias,
                const void *res, long r_row, long r_head, void *out, void *z, long nq, long np, long nc, int G, int act, float slope, long most) {
    Plan pl = {};
    for (int i = 0; i < 3; ++i)
        if (TILE[i] == tile) pl.tile = i;
    pl.S = 1;
    pl.c_split = ceil_div(nc, 64) * 64;
    Product pr = {{P, p_row, p_head}, {Q, q_row, q_head}, np, nq, nc, 0, G, 1};
    const bool weight = kind == GRAD_WEIGHT;
    const Epilogue e = {bias, res, r_row, r_head, out, z, weight ? np : (long)G * np, weight ? nq * np : np, act, slope, nullptr};
    if (most) {
        pr.S = pl.S;
        pr.c_split = pl.c_split;
        return dtype == UMR_F32 ? in_launches_of<float>(most, kind, pr, e)
                                : dtype == UMR_BF16 ? in_launches_of<bf16_t>(most, kind, pr, e) : in_launches_of<f16_t>(most, kind, pr, e);
    }
    if (dtype == UMR_F32) return run_product<float>(kind, pl, pr, e, nullptr, nullptr);
    if (dtype == UMR_BF16) return run_product<bf16_t>(kind, pl, pr, e, nullptr, nullptr);
    return run_product<f16_t>(kind, pl, pr, e, nullptr, nullptr);
}
}
