// linear_f32.hip -- the kernels of linear_kernels.h for float.
#include "linear_kernels.h"

namespace umr_linear {
template int run_product<float>(int, const Plan &, Product, Epilogue, void *, hipStream_t);
template int run_act_grad<float>(const ActGrad &, hipStream_t);
}  // namespace umr_linear
