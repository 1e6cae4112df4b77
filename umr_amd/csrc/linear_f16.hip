// linear_f16.hip -- the kernels of linear_kernels.h for f16.
#include "linear_kernels.h"

namespace umr_linear {
template int run_product<f16_t>(int, const Plan &, Product, Epilogue, void *, hipStream_t);
template int run_act_grad<f16_t>(const ActGrad &, hipStream_t);
}  // namespace umr_linear
