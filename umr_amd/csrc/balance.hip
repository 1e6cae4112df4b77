// balance.hip -- balance loss over E choices with the count of every choice, and its gradient (include/umr_nn.h).
//
//     f_e = counts[e] / (n k),   P_e = mean over the n valid rows of softmax(z)[e],   loss = E sum_e f_e P_e
//     d loss / d z[t,e] = E / n * p[t,e] (f_e - sum_i f_i p[t,i])
//
// (as sum_i p[t,i] = 1, any constant may be taken off all f_e: with their mean taken off, the difference of the two terms loses no
// digits when the choices are used almost evenly).
//
// Both directions are one pass over the scores.  A row is shared by LPR lanes (a power of two), each with 16-byte pieces of it, so
// that a wave reads whole lines whatever E is; the softmax's maximum and sum are butterflies over those lanes, in fp32.  Forward: a
// lane adds up its columns over its rows in registers, lanes and waves meet in a fixed order, choices are counted with integer
// LDS atomics; one workgroup joins the workgroups' parts in part order (in double).  Nothing depends on the order of arrival.
// 2^19 x 128 bf16 with 8 choices a row: rows 53 us (168 MB, 3.2 TB/s), fold and join 5 each, backward 64 us (268 MB, 4.2 TB/s).  In the
// rows the vector unit is busy 63 % of the time (the exponentials alone are 7 us of it) and the waves wait 61 % of theirs: a row's loads
// start when the one before is done.
#include "nn_common.h"

namespace {

constexpr int WG = 256, ROWS_WG = 1024;                  // threads of a workgroup, backward and forward

template <class T, int LPR, int J> struct Row {          // one row's pieces in LPR lanes: lane s holds elements (j LPR + s) V .. + V
    static constexpr int V = 16 / (int)sizeof(T);
    float x[J][V], r;                                    // softmax = x r

    // E a multiple of V (uniform): whole pieces, without the branches of a cut one
    __device__ __forceinline__ void load(const T *z, int E, int s) {
        if (E % V == 0) {
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int e0 = (j * LPR + s) * V;
                const u32x4 v = load16B(z + (e0 < E ? e0 : 0));
#pragma unroll
                for (int i = 0; i < V; ++i) x[j][i] = e0 < E ? elem_of<T>(v, i) : -INFINITY;
            }
        } else {
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int e0 = (j * LPR + s) * V;
                const u32x4 v = load16B_n(z + e0, E - e0);
#pragma unroll
                for (int i = 0; i < V; ++i) x[j][i] = e0 + i < E ? elem_of<T>(v, i) : -INFINITY;
            }
        }
    }

    // false: nothing to choose from (every score -inf)
    __device__ __forceinline__ bool softmax() {
        float m = -INFINITY;                             // (a NaN is left out; it comes back through the exponentials)
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) m = fmaxf(m, x[j][i]);
        m = group_max<LPR>(m);
        float none = 0.f;
        if (__any(m == -INFINITY)) {                     // a row without a maximum: all -inf, or NaN among them
            float nans = 0.f;
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i) nans += x[j][i] != x[j][i] ? 1.f : 0.f;
            nans = group_sum<LPR>(nans);                 // (every lane takes part)
            none = m == -INFINITY && nans == 0.f ? 1.f : 0.f;
        }
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                // 2^((x - m) log2 e): off by |x - m| 2^-24 of its value and a unit of the exponential, i.e. far below 2^-24 of the
                // row's sum wherever |x - m| is large.  Behind the row's end: exp(-inf) = 0.
                x[j][i] = exp2_of((x[j][i] - m) * 1.44269504088896341f);
                sum += x[j][i];
            }
        r = 1.f / group_sum<LPR>(sum);
        return none == 0.f;
    }
};

// f_e, the loss and what the backward call needs, from the sums over all rows.  One workgroup; usage[] and count[] in LDS.
__device__ __forceinline__ void finish(const double *usage, const int *count, long n, float *loss, long long *counts, float *coef, int E, int k,
                                       double *red, long *all) {
    const int t = threadIdx.x, threads = blockDim.x;
    const double per = n > 0 ? 1.0 / (double)n : 0.0;
    double s = 0.0;
    long c = 0;
    for (int e = t; e < E; e += threads) {
        counts[e] = count[e];
        c += count[e];
        s += (double)count[e] * per / (double)k * usage[e] * per;
    }
    red[t] = s;
    all[t] = c;
    __syncthreads();
    for (int o = threads / 2; o > 0; o >>= 1) {              // (a power of two)
        if (t < o) { red[t] += red[t + o]; all[t] += all[t + o]; }
        __syncthreads();
    }
    for (int e = t; e < E; e += threads) coef[e] = (float)(((double)count[e] - (double)all[0] / E) * per / (double)k);
    if (t == 0) {
        loss[0] = (float)(red[0] * E);
        coef[E] = (float)(E * per);
    }
}

template <class T, int LPR, int J>
__global__ __launch_bounds__(ROWS_WG) void k_balance_rows(const T *z, const long long *inds, const unsigned char *mask, float *part_p, int *part_c,
                                                     float *loss, long long *counts, float *coef, long T_rows, int E, int k, long rows) {
    constexpr int V = 16 / (int)sizeof(T), RPW = 64 / LPR, W = LPR * V * J;      // rows per wave, columns a row's lanes hold (>= E)
    __shared__ float usage[ROWS_WG / 64][W];
    __shared__ int hist[W + 1];                                                  // [E]: the number of valid rows
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, s = lane % LPR, sub = lane / LPR;
    for (int e = t; e < W + 1; e += ROWS_WG) hist[e] = 0;
    __syncthreads();
    const long r0 = blockIdx.x * rows, r1 = r0 + rows < T_rows ? r0 + rows : T_rows;
    float acc[J][V];
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) acc[j][i] = 0.f;
    for (long b = r0 + wave * RPW; b < r1; b += RPW * (ROWS_WG / 64)) {               // (uniform per wave: the butterflies need every lane)
        const long row = b + sub;
        const bool here = row < r1;
        const long safe = here ? row : r1 - 1;
        Row<T, LPR, J> r;
        r.load(z + safe * E, E, s);
        const long long chosen = s < k ? inds[safe * k + s] : -1;                // (on its way while the softmax is made)
        const bool counts_here = here && (!mask || mask[safe]);
        const bool some = r.softmax();
        if (!counts_here || !some) continue;
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) acc[j][i] = fmaf(r.x[j][i], r.r, acc[j][i]);
        if (s == 0) atomicAdd(&hist[W], 1);
        if (chosen >= 0 && chosen < E) atomicAdd(&hist[(int)chosen], 1);
        for (int i = s + LPR; i < k; i += LPR) {
            const long long e = inds[row * k + i];
            if (e >= 0 && e < E) atomicAdd(&hist[(int)e], 1);
        }
    }
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
#pragma unroll
            for (int o = 32; o >= LPR; o >>= 1) acc[j][i] += __shfl_xor(acc[j][i], o, UMR_WAVE);
            if (sub == 0) usage[wave][(j * LPR + s) * V + i] = acc[j][i];
        }
    __syncthreads();
    if (part_p) {
        for (int e = t; e < E; e += ROWS_WG) {
            float v = usage[0][e];
#pragma unroll
            for (int w = 1; w < ROWS_WG / 64; ++w) v += usage[w][e];
            part_p[(long)blockIdx.x * E + e] = v;
            part_c[(long)blockIdx.x * (E + 1) + e] = hist[e];
        }
        if (t == 0) part_c[(long)blockIdx.x * (E + 1) + E] = hist[W];
        return;
    }
    __shared__ double sums[W], red[ROWS_WG];
    __shared__ long all[ROWS_WG];                                          // the only workgroup: finish here
    for (int e = t; e < E; e += ROWS_WG) {
        double v = 0.0;
#pragma unroll
        for (int w = 0; w < ROWS_WG / 64; ++w) v += usage[w][e];
        sums[e] = v;
    }
    __syncthreads();
    finish(sums, hist, hist[W], loss, counts, coef, E, k, red, all);
}

// Many parts first become one of 32, in part order: read by one workgroup alone, 512 parts of 128 choices took 28 us.
constexpr int FOLD = 32;
__global__ __launch_bounds__(256) void k_balance_fold(const float *part_p, const int *part_c, int blocks, float *to_p, int *to_c, int E) {
    const int b0 = blockIdx.x * FOLD, b1 = b0 + FOLD < blocks ? b0 + FOLD : blocks, e = blockIdx.y * 256 + threadIdx.x;
    if (e > E) return;
    int c = 0;
#pragma unroll 8
    for (int b = b0; b < b1; ++b) c += part_c[(long)b * (E + 1) + e];
    to_c[(long)blockIdx.x * (E + 1) + e] = c;
    if (e == E) return;
    float s = 0.f;
#pragma unroll 8
    for (int b = b0; b < b1; ++b) s += part_p[(long)b * E + e];
    to_p[(long)blockIdx.x * E + e] = s;
}

// Joins the parts: 1024 threads, the columns side by side and as many runs of parts as fit, each in part order.
__global__ __launch_bounds__(1024) void k_balance_join(const float *part_p, const int *part_c, int blocks, float *loss, long long *counts, float *coef,
                                                       int E, int k) {
    __shared__ double sum[1024], red[1024];
    __shared__ long all[1024];
    __shared__ int cnt[1024], total[UMR_BALANCE_MAX_CHOICES];
    __shared__ double usage[UMR_BALANCE_MAX_CHOICES];
    __shared__ int nvalid[1024];
    const int t = threadIdx.x, runs = 1024 / E > 0 ? 1024 / E : 1, run = t / E, e = t % E;
    double s = 0.0;
    int c = 0;
    if (run < runs) {
        const int per = (blocks + runs - 1) / runs, b0 = run * per, b1 = b0 + per < blocks ? b0 + per : blocks;
#pragma unroll 16
        for (int b = b0; b < b1; ++b) { s += part_p[(long)b * E + e]; c += part_c[(long)b * (E + 1) + e]; }
    }
    int v = 0;
    for (int b = t; b < blocks; b += 1024) v += part_c[(long)b * (E + 1) + E];
    sum[t] = s; cnt[t] = c; nvalid[t] = v;
    __syncthreads();
    for (int o = 512; o > 0; o >>= 1) {
        if (t < o) nvalid[t] += nvalid[t + o];
        __syncthreads();
    }
    if (t < E) {
        double a = 0.0;
        int b = 0;
        for (int r = 0; r < runs; ++r) { a += sum[r * E + t]; b += cnt[r * E + t]; }
        usage[t] = a; total[t] = b;
    }
    __syncthreads();
    finish(usage, total, nvalid[0], loss, counts, coef, E, k, red, all);
}

template <class T, int LPR, int J>
__global__ __launch_bounds__(WG) void k_balance_backward(const T *__restrict__ z, const unsigned char *__restrict__ mask, const float *__restrict__ coef,
                                                         const float *__restrict__ grad, T *__restrict__ dz,
                                                         long T_rows, int E) {
    constexpr int V = 16 / (int)sizeof(T), RPW = 64 / LPR;
    const int t = threadIdx.x, lane = t & 63, s = lane % LPR, sub = lane / LPR;
    const long wave = (long)blockIdx.x * (WG / 64) + (t >> 6), waves = (long)gridDim.x * (WG / 64);
    float f[J][V];
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = (j * LPR + s) * V + i;
            f[j][i] = e < E ? coef[e] : 0.f;
        }
    const float scale = grad[0] * coef[E];
    for (long b = wave * RPW; b < T_rows; b += waves * RPW) {
        const long row = b + sub;
        const bool here = row < T_rows;
        Row<T, LPR, J> r;
        r.load(z + (here ? row : T_rows - 1) * E, E, s);
        const bool some = r.softmax();
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) dot = fmaf(f[j][i], r.x[j][i], dot);
        dot = group_sum<LPR>(dot) * r.r;
        if (!here) continue;
        const float up = scale * r.r;
        const bool valid = some && (!mask || mask[row]);
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int i0 = 0; i0 < V; i0 += 4) {
                const int e0 = (j * LPR + s) * V + i0;
                float v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = valid ? up * r.x[j][i0 + i] * (f[j][i0 + i] - dot) : 0.f;
                store4(dz + row * E + e0, E - e0, v);
            }
    }
}

// lanes per row and pieces per lane: the fewest lanes that hold a row in one piece each, then more pieces
#define UMR_BALANCE_SHAPES(T, E, CALL)                                                   \
    {                                                                                    \
        const int pieces = ((E) + 16 / (int)sizeof(T) - 1) / (16 / (int)sizeof(T));      \
        if (pieces <= 1) CALL(T, 1, 1)                                                   \
        else if (pieces <= 2) CALL(T, 2, 1)                                              \
        else if (pieces <= 4) CALL(T, 4, 1)                                              \
        else if (pieces <= 8) CALL(T, 8, 1)                                              \
        else if (pieces <= 16) CALL(T, 16, 1)                                            \
        else if (pieces <= 32) CALL(T, 32, 1)                                            \
        else if (pieces <= 64) CALL(T, 64, 1)                                            \
        else if (pieces <= 128) CALL(T, 64, 2)                                           \
        else if constexpr (sizeof(T) == 4) CALL(T, 64, 4)                                \
    }

long rows_per_group(long T, int E) {
    // a workgroup's 16 waves take 16 bytes a lane, 16 KB of scores, at a time: at least twice in fp32, once in 16 bits; at most 512
    // workgroups, whose parts one workgroup joins
    long rows = (T + 511) / 512, least = 32768 / (4 * (E < 4 ? 4 : E));
    if (least < 32) least = 32;
    return rows < least ? least : rows;
}

bool balance_ok(long T, int E, int dtype) {
    return T >= 0 && T < (1L << 40) && E >= 1 && E <= UMR_BALANCE_MAX_CHOICES && (dtype == UMR_F32 || dtype == UMR_BF16 || dtype == UMR_F16);
}

long groups_of(long T, int E) { const long r = rows_per_group(T, E); return T > 0 ? (T + r - 1) / r : 1; }

long folds_of(long groups) { return groups > 2 * FOLD ? (groups + FOLD - 1) / FOLD : 0; }

}  // namespace

extern "C" {

size_t umr_balance_workspace_bytes(long T, int E) {
    if (!balance_ok(T, E, UMR_F32)) return 0;
    const long g = groups_of(T, E);
    return g > 1 ? (size_t)(g + folds_of(g)) * (2 * E + 1) * 4 : 0;
}

int umr_balance_forward(const void *z, const long long *inds, const unsigned char *mask, float *loss, long long *counts, float *coef, long T, int E,
                        int k, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
    if (!balance_ok(T, E, dtype) || k < 1 || !loss || !counts || !coef || (T > 0 && (!z || !inds)) || T * (double)k >= 2147483648.0) return UMR_ERR_ARG;
    const long rows = rows_per_group(T, E), groups = groups_of(T, E);
    if (groups > 1 && (!workspace || workspace_bytes < umr_balance_workspace_bytes(T, E))) return UMR_ERR_ARG;
    float *pp = groups > 1 ? (float *)workspace : nullptr;
    int *pc = groups > 1 ? (int *)workspace + groups * E : nullptr;
    const hipStream_t st = (hipStream_t)stream;
#define UMR_CALL(TT, LPR, J)                                                                                                               \
    UMR_LAUNCH((k_balance_rows<TT, LPR, J>), (unsigned)groups, ROWS_WG, 0, st, (const TT *)z, inds, mask, pp, pc, loss, counts, coef, T, E, k, rows);
    if (dtype == UMR_F32) UMR_BALANCE_SHAPES(float, E, UMR_CALL)
    else if (dtype == UMR_BF16) UMR_BALANCE_SHAPES(bf16_t, E, UMR_CALL)
    else UMR_BALANCE_SHAPES(f16_t, E, UMR_CALL)
#undef UMR_CALL
    if (umr_launch_status() != UMR_OK) return UMR_ERR_LAUNCH;
    if (groups > 1) {
        long parts = groups;
        if (const long folds = folds_of(groups)) {
            float *to_p = (float *)(pc + groups * (E + 1));
            int *to_c = (int *)(to_p + folds * E);
            UMR_LAUNCH(k_balance_fold, dim3((unsigned)folds, (unsigned)(E / 256 + 1)), 256, 0, st, (const float *)pp, (const int *)pc, (int)groups, to_p, to_c, E);
            if (umr_launch_status() != UMR_OK) return UMR_ERR_LAUNCH;
            pp = to_p;
            pc = to_c;
            parts = folds;
        }
        UMR_LAUNCH(k_balance_join, 1, 1024, 0, st, (const float *)pp, (const int *)pc, (int)parts, loss, counts, coef, E, k);
        return umr_launch_status();
    }
    return UMR_OK;
}

int umr_balance_backward(const void *z, const unsigned char *mask, const float *coef, const float *grad, void *dz, long T, int E, int dtype,
                         void *stream) {
    if (!balance_ok(T, E, dtype) || !coef || !grad || (T > 0 && (!z || !dz))) return UMR_ERR_ARG;
    if (T == 0) return UMR_OK;
    const hipStream_t st = (hipStream_t)stream;
    const long want = (T + 15) / 16;
    const unsigned grid = (unsigned)(want < 4096 ? want : 4096);
#define UMR_CALL(TT, LPR, J) UMR_LAUNCH((k_balance_backward<TT, LPR, J>), grid, WG, 0, st, (const TT *)z, mask, coef, grad, (TT *)dz, T, E);
    if (dtype == UMR_F32) UMR_BALANCE_SHAPES(float, E, UMR_CALL)
    else if (dtype == UMR_BF16) UMR_BALANCE_SHAPES(bf16_t, E, UMR_CALL)
    else UMR_BALANCE_SHAPES(f16_t, E, UMR_CALL)
#undef UMR_CALL
    return umr_launch_status();
}

}  // extern "C"
