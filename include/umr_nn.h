/*
 * umr_nn.h -- C ABI of libumr_hip.so, second part: the network-side operators (fully connected layers with their epilogue and
 * their gradients, one layer for many heads at once, the balance loss over camera hypotheses).  Same conventions as umr_hip.h
 * (caller owns every buffer, work is enqueued on `stream`, nothing is allocated or synchronised inside, status 0 / UMR_ERR_ARG /
 * UMR_ERR_LAUNCH), with these differences:
 *   - `dtype` names the type of every tensor passed as void*: UMR_F32, UMR_BF16 or UMR_F16; all sums are fp32
 *   - a matrix operand is described by its element strides (row, head); its last dimension has stride 1.  Strides of 0 are
 *     allowed in operands that are read (a broadcast), outputs are dense
 *   - outputs and workspaces overlap nothing else of the call (parts of a result may be written twice, with the same bits)
 *   - sizes may be 0 (an empty product is 0); M, N, K < 2^27, G < 65536, M * G * max(N, K) < 2^46; M * N, M * K and N * K of one head
 *     < 2^35 (a larger one is UMR_ERR_ARG where its tiles are more than a launch holds)
 */
#ifndef UMR_NN_H
#define UMR_NN_H

#include <stddef.h>

#include "umr_hip.h" /* UMR_OK, UMR_ERR_ARG, UMR_ERR_LAUNCH */

#ifdef __cplusplus
extern "C" {
#endif

#define UMR_F32 0
#define UMR_BF16 1
#define UMR_F16 2

#define UMR_ACT_NONE 0
#define UMR_ACT_RELU 1
#define UMR_ACT_LEAKY_RELU 2 /* slope >= 0 */
#define UMR_ACT_TANH 3
#define UMR_ACT_GELU 4 /* z Phi(z), the exact form */
#define UMR_ACT_SILU 5

/* y[m,g,:] = act(z[m,g,:]) + r[m,g,:],   z[m,g,n] = sum_k x[m,g,k] w[g,n,k] + b[g,n]        m < M, g < G, n < N, k < K
 *   x [M,G,K] by strides, w [G,N,K] by strides, bias [G,N] dense or NULL, residual [M,G,N] by strides or NULL
 *   y [M,G,N] dense; z [M,G,N] dense or NULL: what umr_linear_grad_act needs of the pre-activation -- fp32 for none, tanh, gelu and
 *   silu, `dtype` (its sign matters) for relu and leaky relu
 * G = 1 is an ordinary fully connected layer.  `workspace` may be NULL where umr_linear_forward_workspace_bytes is 0. */
size_t umr_linear_forward_workspace_bytes(long M, long N, long K, int G, int dtype);
int umr_linear_forward(const void *x, long x_row, long x_head, const void *w, long w_row, long w_head, const void *bias,
                       const void *residual, long r_row, long r_head, void *y, void *z, long M, long N, long K, int G, int dtype,
                       int act, float slope, void *workspace, size_t workspace_bytes, void *stream);

/* dz = gy * act'(z) and the sums over the rows:  db[g,n] = sum_m dz[m,g,n],  dr[g,n] = sum_m gy[m,g,n]
 *   gy [M,G,N] by strides; z [M,G,N] dense: the forward call's z (for relu and leaky relu any tensor of type `dtype` with its sign:
 *   the output of a call without residual), NULL where act is UMR_ACT_NONE; dz [M,G,N] dense, NULL where act is UMR_ACT_NONE (dz is gy then);
 *   db, dr [G,N] dense or NULL.  Sums run in a fixed order.  At a kink the derivative is the one of the negative side. */
size_t umr_linear_grad_act_workspace_bytes(long M, long N, int G);
int umr_linear_grad_act(const void *gy, long g_row, long g_head, const void *z, void *dz, void *db, void *dr, long M, long N, int G,
                        int dtype, int act, float slope, void *workspace, size_t workspace_bytes, void *stream);

/* dx[m,g,k] = sum_n dz[m,g,n] w[g,n,k]:  dz [M,G,N] and w [G,N,K] by strides, dx [M,G,K] dense */
size_t umr_linear_grad_input_workspace_bytes(long M, long N, long K, int G, int dtype);
int umr_linear_grad_input(const void *dz, long dz_row, long dz_head, const void *w, long w_row, long w_head, void *dx, long M, long N,
                          long K, int G, int dtype, void *workspace, size_t workspace_bytes, void *stream);

/* dw[g,n,k] = sum_m dz[m,g,n] x[m,g,k]:  dz [M,G,N] and x [M,G,K] by strides, dw [G,N,K] dense */
size_t umr_linear_grad_weight_workspace_bytes(long M, long N, long K, int G, int dtype);
int umr_linear_grad_weight(const void *dz, long dz_row, long dz_head, const void *x, long x_row, long x_head, void *dw, long M, long N,
                           long K, int G, int dtype, void *workspace, size_t workspace_bytes, void *stream);

/* Balance loss over E choices (1 <= E <= UMR_BALANCE_MAX_CHOICES).  Rows t < T with scores z[t,:] (T x E, dense), T * k < 2^31, of which k
 * choices inds[t,:] (T x k, dense, k >= 1) were taken:
 *     p[t,:] = softmax(z[t,:])        over the valid rows, n of them:
 *     counts[e] = #{(t,j): inds[t,j] = e},   f_e = counts[e] / (n k),   P_e = mean_t p[t,e],      loss = E sum_e f_e P_e
 * A row is valid where mask[t] is non-zero (mask NULL: every row) and not all of its scores are -inf; other rows are not read
 * into anything, whatever they hold, and have gradient 0.  An index outside 0 .. E-1 counts for no choice.  Without a valid row
 * the loss is 0.  A NaN or +inf in a valid row makes loss and gradient NaN, as softmax does.
 *   loss [1] fp32, counts [E] int64; coef [E + 1] fp32: what the backward call needs (f_e less their mean, then E / n).
 * backward: dz[t,e] = grad * (E / n) * p[t,e] * (f_e - sum_i f_i p[t,i]),  grad [1] fp32 on the device, dz (T x E) in `dtype`. */
#define UMR_BALANCE_MAX_CHOICES 1024
size_t umr_balance_workspace_bytes(long T, int E);
int umr_balance_forward(const void *z, const long long *inds, const unsigned char *mask, float *loss, long long *counts, float *coef,
                        long T, int E, int k, int dtype, void *workspace, size_t workspace_bytes, void *stream);
int umr_balance_backward(const void *z, const unsigned char *mask, const float *coef, const float *grad, void *dz, long T, int E,
                         int dtype, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* UMR_NN_H */
