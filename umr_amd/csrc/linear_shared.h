// linear_shared.h -- what the entry points (linear.hip) and the kernels of each type (linear_kernels.h) agree on.
#pragma once
#include "nn_common.h"

namespace umr_linear {

struct Epilogue {
    const void *bias;               // [G, np] or NULL
    const void *res;                // [nq, G, np] by strides or NULL
    long r_row, r_head;
    void *out, *z;                  // z: NULL or dense like out: T for a kinked activation, fp32 for the others
    long o_row, o_head;
    int act;
    float slope;
    float *part;                    // not NULL: fp32 sums to part[split][head][q][p] and nothing else
};

struct Operand {
    const void *data;
    long row, head;                 // element strides: between rows of the tensor as it lies in memory, and between heads
};

struct Product {
    Operand P, Q;
    long np, nq, nc;
    long c_split;                   // contraction per split (a multiple of the kernel's step); the last one is shorter
    int G, S;
};

enum Kind { FORWARD = 0, GRAD_INPUT = 1, GRAD_WEIGHT = 2 };

inline long ceil_div(long a, long b) { return (a + b - 1) / b; }

constexpr int FEW_WAVES = 8;          // waves of a workgroup of the kernels for few rows

enum Tile { T64x64, T128x128, T256x256 };
constexpr int TILE[] = {64, 128, 256};

struct Plan {
    bool few, outer;
    int tile, S;
    long c_split;
};

struct ActGrad {
    const void *gy, *z;
    long g_row, g_head;
    void *dz, *db, *dr;
    float *part;
    long M, N, rows, blocks;
    int G, act;
    float slope;
};

// one product, one act' pass; defined for float, bf16_t and f16_t in linear_f32.hip, linear_bf16.hip and linear_f16.hip
template <class T> int run_product(int kind, const Plan &pl, Product pr, Epilogue e, void *workspace, hipStream_t st);
template <class T> int run_act_grad(const ActGrad &a, hipStream_t st);

}  // namespace umr_linear
