// linear_bf16.hip -- the kernels of linear_kernels.h for bf16.
#include "linear_kernels.h"

namespace umr_linear {
template int run_product<bf16_t>(int, const Plan &, Product, Epilogue, void *, hipStream_t);
template int run_act_grad<bf16_t>(const ActGrad &, hipStream_t);
}  // namespace umr_linear
