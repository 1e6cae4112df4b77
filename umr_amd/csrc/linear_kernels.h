// linear_kernels.h -- fully connected layers with bias, activation and residual in the product's epilogue, and their gradients
// (include/umr_nn.h).  With the heads g < G as an outer index, all three products are
//
//     out[q, p] = sum_c Q[q, c] P[p, c]            q < nq, p < np (p runs along memory in `out`), c < nc
//
//     forward     y  = x w^T     q = m, p = n, c = k      both operands have the contraction along memory ("fast")
//     gradient    dx = dz w      q = m, p = k, c = n      P is w, whose rows are the contraction ("slow")
//     gradient    dw = dz^T x    q = n, p = k, c = m      both slow
//
// One kernel family for few rows q (the weights are read once, from memory to the matrix unit without LDS) and one tiled through
// LDS for many.  Both can split the contraction over workgroups; the parts are then added in part order by a second launch, so
// results do not depend on the order of arrival.  All sums are fp32 (the matrix unit's accumulators), one rounding at the end.
#pragma once
#include "linear_shared.h"

namespace umr_linear {
namespace {

// ------------------------------------------------------------------------------------------------ epilogue
__host__ __device__ __forceinline__ bool kinked(int act) { return act == UMR_ACT_RELU || act == UMR_ACT_LEAKY_RELU; }

// exp and the normal distribution, both to a few steps of the value itself, also where Phi is tiny (0.5 (1 + erf) has no digit left
// at -6).  EXACT (fp32 results): the library's functions.  Otherwise (results of 16 bits) exp is one v_exp_f32, and the tail Phi(-a) =
// exp(-a^2 / 2) t q(t), t = 1 / (1 + 0.346 a), shares it with phi: q is a minimax fit of degree 6 to the Mills ratio over a <= 14, within
// 2e-8 of Phi and 7e-6 relative, where half a step of the result is 2^-11 or 2^-8 of it.
template <bool EXACT> __device__ __forceinline__ float exp_of(float x) { return EXACT ? expf(x) : exp2_of(x * 1.44269504088896341f); }
template <bool EXACT> __device__ __forceinline__ float normal_cdf(float z, float gauss) {       // gauss = exp(-z^2 / 2)
    if (EXACT) return 0.5f * erfcf(z * -0.70710678118654752f);
    const float t = __builtin_amdgcn_rcpf(1.f + 0.346f * fabsf(z));
    const float q = 0.138244497f + t * (0.134363111f + t * (0.147132262f + t * (-0.0041666107f + t * (0.229732837f + t * (-0.189794395f + t * 0.0444883194f)))));
    const float tail = gauss * (t * q);
    return z < 0.f ? tail : 1.f - tail;
}

template <bool EXACT> __device__ __forceinline__ float act_value(float z, int act, float slope) {
    switch (act) {                  // (uniform)
        case UMR_ACT_RELU: return z > 0.f ? z : z != z ? z : 0.f;
        case UMR_ACT_LEAKY_RELU: return z > 0.f ? z : slope * z;
        case UMR_ACT_TANH: return tanhf(z);
        case UMR_ACT_GELU: return z * normal_cdf<EXACT>(z, EXACT ? 0.f : exp_of<EXACT>(-0.5f * z * z));
        case UMR_ACT_SILU: return z / (1.f + exp_of<EXACT>(-z));
        default: return z;
    }
}

template <bool EXACT> __device__ __forceinline__ float act_slope(float z, int act, float slope) {      // act'(z)
    switch (act) {
        case UMR_ACT_RELU: return z <= 0.f ? 0.f : 1.f;            // (a NaN hides no gradient)
        case UMR_ACT_LEAKY_RELU: return z > 0.f ? 1.f : slope;
        case UMR_ACT_TANH: {        // 1 - tanh^2 without the difference, which has no digits left where tanh rounds to 1
            const float e = exp_of<EXACT>(-2.f * fabsf(z)), d = 1.f + e;
            return 4.f * e / (d * d);
        }
        case UMR_ACT_GELU: { const float e = exp_of<EXACT>(-0.5f * z * z); return normal_cdf<EXACT>(z, e) + z * e * 0.39894228040143268f; }
        case UMR_ACT_SILU: { const float s = 1.f / (1.f + exp_of<EXACT>(-z)); return s * (1.f + z * (1.f - s)); }
        default: return 1.f;
    }
}

// n <= 4 neighbours of one row from their pre-activations: z, activation, residual, store at element o
template <class T> __device__ __forceinline__ void finish_row(const Epilogue &e, float (&v)[4], const float (&res)[4], long o, long n) {
    // what the backward call needs of z: all of it in fp32 for a smooth activation (rounded to 16 bits it would add to the
    // rounding of dz), the sign for a kinked one
    if (e.z) {
        if (kinked(e.act)) store4((T *)e.z + o, n, v);
        else store4((float *)e.z + o, n, v);
    }
    if (e.act != UMR_ACT_NONE) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = act_value<sizeof(T) == 4>(v[i], e.act, e.slope);
    }
    if (e.res) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += res[i];
    }
    store4((T *)e.out + o, n, v);
}

// ... from their sums
template <class T> __device__ __forceinline__ void finish4(const Epilogue &e, float (&v)[4], long q, long p, long np, int g) {
    const long n = np - p;
    if (e.bias) {
        float b[4];
        load4((const T *)e.bias + g * np + p, n, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += b[i];
    }
    float r[4] = {0.f, 0.f, 0.f, 0.f};
    if (e.res) load4((const T *)e.res + q * e.r_row + g * e.r_head + p, n, r);
    finish_row<T>(e, v, r, q * e.o_row + g * e.o_head + p, n);
}

template <class T>
__device__ __forceinline__ void emit4(const Epilogue &e, float (&v)[4], long q, long p, long nq, long np, int g, int G, int split) {
    if (q >= nq || p >= np) return;
    if (e.part) store4(e.part + (((long)split * G + g) * nq + q) * np + p, np - p, v);
    else finish4<T>(e, v, q, p, np, g);
}

// The parts of a split contraction, added in part order, and the epilogue.  One thread per 4 neighbours.
template <class T> __global__ __launch_bounds__(256) void k_linear_join(Epilogue e, const float *part, int S, long nq, long np, int G) {
    const long p4 = (np + 3) / 4, total = nq * G * p4, plane = (long)G * nq * np;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const long p = (i % p4) * 4, q = (i / p4) % nq;
        const int g = (int)(i / p4 / nq);
        const float *src = part + ((long)g * nq + q) * np + p;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < S; ++s) {
            float t[4];
            load4(src + s * plane, np - p, t);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += t[j];
        }
        finish4<T>(e, v, q, p, np, g);
    }
}

// ------------------------------------------------------------------------------------------------ many rows: tiles through LDS
// A tile is TQ x TP results; the contraction advances by 128 bytes a row (32 fp32, 64 of 16 bits).  In LDS a row is 128 bytes +
// 16 of padding: 8 lanes that read the same chunk of 8 rows meet 32 different banks.  An fp32 operand whose contraction is slow
// keeps memory's order [c][row] (the fp32 matrix instructions take one value per lane, so any order serves); a 16-bit one is
// transposed in registers on its way in (8 x 2 or 8 x 4 values per thread).  Two buffers, one barrier per step; the loads of
// the next step are in flight while the matrix unit works.
//
// The loop has no guarded loads.  The last tile of a dimension starts early enough to end with it (its overlap is computed twice, to
// the same bits); a matrix smaller than a tile repeats its last row, whose results are dropped.  A last step that is not whole
// loads 16 bytes that end with the row and moves them into place, and zeros behind them, when they go to LDS.
//
// 256 x 256 (16 bits): 8 waves of 128 x 64, one workgroup a CU; bf16 8192 x 4096 x 4096 forward with gelu, z and residual 394 us (698
// TFLOP/s), dx 406, dw 350.  The matrix unit is busy 30, 28 and 32 % of the time and the waves wait 47, 53 and 38 % of theirs: LDS carries
// 256 KB a step and the loads' latency shows.  128 x 128: fp32 4096^3 1180 us (116 TFLOP/s, matrix unit 74 % busy).  64 x 64 where larger
// tiles would leave CUs idle: fp32 10000 x 1011 x 350 93 us (49 % busy).
constexpr int ROW_BYTES = 144;
constexpr long NEAR = 1L << 22;                               // rows closer than this many elements: a tile's offsets fit 32 bits

// v: the 16 bytes that end with the row's last element, `valid` of them wanted (> 0): those first, zeros behind
template <class T> __device__ __forceinline__ u32x4 ending_chunk(u32x4 v, int valid) {
    constexpr int V = 16 / (int)sizeof(T);
    const int words = sizeof(T) == 4 ? V - valid : (V - valid) / 2;
    u32x4 r;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        unsigned x = 0u;
#pragma unroll
        for (int o = 0; o < 4; ++o)
            if (k + o < 4 && words == o) x = v[(k + o) & 3];
        r[k] = x;
    }
    if (sizeof(T) == 2 && ((V - valid) & 1)) {
#pragma unroll
        for (int k = 0; k < 4; ++k) r[k] = (r[k] >> 16) | (k < 3 ? r[(k + 1) & 3] << 16 : 0u);
    }
    return r;
}

template <class T, int R, bool SLOW, int NT> struct Stager {  // R rows of one operand, NT threads
    static constexpr bool WORDS = sizeof(T) == 4;
    static constexpr int ES = (int)sizeof(T), V = 16 / ES, BC = 128 / ES;
    static constexpr int N = R * 8 / NT;                      // 16-byte pieces per thread
    static constexpr int W = N / 2;                           // 16 bits, slow: 32-bit words per contraction row of a thread's 8 x N block
    static constexpr int SLOW_ROW = (R + 8) * 4;              // bytes of one c-row of an fp32 slow tile: halves of a wave (4 c-rows
                                                              // apart) read different banks
    static constexpr int BYTES = SLOW && WORDS ? (BC * SLOW_ROW > R * ROW_BYTES ? BC * SLOW_ROW : R * ROW_BYTES) : R * ROW_BYTES;
    u32x4 r[N];
    unsigned off[SLOW ? 1 : N];                               // byte offset of this thread's piece in the tile's first step

    static __device__ __forceinline__ int chunk(int t) { return t & 7; }                               // fast: which 16 bytes of a row
    static __device__ __forceinline__ int c_row(int t, int u) { return WORDS ? (t + NT * u) / (R / 4) : (t / (R / N)) * 8 + u; }   // slow
    static __device__ __forceinline__ int column(int t) { return WORDS ? (t % (R / 4)) * 4 : (t % (R / N)) * N; }

    // a tile's pieces lie within 32-bit offsets of its corner (true for rows of less than 2^22 elements), and a slow operand has
    // as many rows as the tile: what load and load_last need
    static __device__ __forceinline__ bool near(long ld, long n) { return ld < NEAR && (!SLOW || n >= R); }

    // a tile of `rows` rows (fewer than R: the last is repeated)
    __device__ __forceinline__ void start(long ld, long rows, int t) {
        if constexpr (!SLOW) {
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int row = (t + NT * u) >> 3;
                off[u] = (unsigned)((row < rows ? row : (int)rows - 1) * (unsigned)ld + chunk(t) * V) * ES;
            }
        } else off[0] = (unsigned)(c_row(t, 0) * (unsigned)ld + column(t)) * ES;
    }
    static __device__ __forceinline__ const T *at(const T *p, unsigned bytes) { return (const T *)((const char *)p + bytes); }
    __device__ __forceinline__ void take(int j, const T *p) {     // slow, 16 bits: N neighbours of contraction row j
        if constexpr (W == 2) { const u32x2 v = *(const u32x2_any *)p; r[j / 2][(j % 2) * 2] = v[0]; r[j / 2][(j % 2) * 2 + 1] = v[1]; }
        else r[j / 4][j % 4] = *(const u32_any *)p;
    }

    // a whole step; corner: the tile's first row at this contraction (uniform)
    __device__ __forceinline__ void load(const T *corner, long ld) {
        if constexpr (!SLOW) {
#pragma unroll
            for (int u = 0; u < N; ++u) r[u] = load16B(at(corner, off[u]));
        } else if constexpr (WORDS) {
#pragma unroll
            for (int u = 0; u < N; ++u) r[u] = load16B(at(corner + (long)(u * (NT / (R / 4))) * ld, off[0]));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) take(j, at(corner + j * ld, off[0]));
        }
    }
    // the last step, `left` contraction values, fewer than BC; c: of the whole row, nc of them.  Everything read lies within the
    // operand: a fast row that is cut is read as the 16 bytes that end with it, a slow operand's last c-row is repeated.
    template <bool TINY> __device__ __forceinline__ void load_last(const T *corner, long ld, int left, long nc, int t) {   // TINY: nc may be below V
        if constexpr (!SLOW) {
            const int back = chunk(t) * V + V - left;         // > 0: this chunk would end behind the row
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const T *p = at(corner, off[u]);
                r[u] = !TINY || nc >= V ? load16B(p - (back > 0 ? back : 0)) : load16B_n(p, chunk(t) == 0 ? nc : 0);
            }
        } else if constexpr (WORDS) {
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int c = c_row(t, u) < left ? c_row(t, u) : left - 1;
                r[u] = load16B(corner + c * ld + column(t));
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) take(j, corner + (c_row(t, j) < left ? c_row(t, j) : left - 1) * ld + column(t));
        }
    }
    // any step of an operand that is not near(): in 64 bits, element by element
    __device__ __forceinline__ void load_far(const T *corner, long ld, int left, long rows, int t) {
        if constexpr (!SLOW) {
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int row = (t + NT * u) >> 3;
                r[u] = load16B_n(corner + (row < rows ? row : rows - 1) * ld + chunk(t) * V, left - chunk(t) * V);
            }
        } else if constexpr (WORDS) {
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int c = c_row(t, u) < left ? c_row(t, u) : left - 1;
#pragma unroll
                for (int i = 0; i < 4; ++i) r[u][i] = as_u32(corner[c * ld + (column(t) + i < rows ? column(t) + i : rows - 1)]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int c = c_row(t, j) < left ? c_row(t, j) : left - 1;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const long col = column(t) + 2 * w;
                    const unsigned lo = corner[c * ld + (col < rows ? col : rows - 1)].bits, hi = corner[c * ld + (col + 1 < rows ? col + 1 : rows - 1)].bits;
                    r[(j * W + w) / 4][(j * W + w) % 4] = lo | (hi << 16);
                }
            }
        }
    }
    // ... made whole: `left` contraction values, zeros behind them
    __device__ __forceinline__ void trim(int left, bool cut, int t) {      // cut: rows were read as load_last does
        if constexpr (!SLOW) {
            const int valid = left - chunk(t) * V;
#pragma unroll
            for (int u = 0; u < N; ++u)
                if (valid <= 0) r[u] = u32x4{0u, 0u, 0u, 0u};
                else if (valid < V && cut) r[u] = ending_chunk<T>(r[u], valid);
        } else if constexpr (WORDS) {
#pragma unroll
            for (int u = 0; u < N; ++u)
                if (c_row(t, u) >= left) r[u] = u32x4{0u, 0u, 0u, 0u};
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c_row(t, j) >= left) {
#pragma unroll
                    for (int w = 0; w < W; ++w) r[(j * W + w) / 4][(j * W + w) % 4] = 0u;
                }
        }
    }
    __device__ __forceinline__ void put(char *lds, int t) const {
        if constexpr (!SLOW) {
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int idx = t + NT * u;
                *(u32x4 *)(lds + (idx >> 3) * ROW_BYTES + (idx & 7) * 16) = r[u];
            }
        } else if constexpr (WORDS) {
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int idx = t + NT * u;
                *(u32x4 *)(lds + (idx / (R / 4)) * SLOW_ROW + (idx % (R / 4)) * 16) = r[u];
            }
        } else {
            const int cg = t / (R / N), col = (t % (R / N)) * N;
#pragma unroll
            for (int i = 0; i < N; ++i) {                     // neighbour i: its 8 contraction values
                u32x4 v;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int a = 2 * k * W + i / 2, b = (2 * k + 1) * W + i / 2;
                    const unsigned lo = r[a / 4][a % 4], hi = r[b / 4][b % 4];
                    v[k] = (i & 1) ? (lo >> 16) | (hi & 0xffff0000u) : (lo & 0xffffu) | (hi << 16);
                }
                *(u32x4 *)(lds + (col + i) * ROW_BYTES + cg * 16) = v;
            }
        }
    }

    // chunk `grp` (32 bytes of contraction per row: 16 for each half of the wave) of row `row`
    static __device__ __forceinline__ u32x4 fragment(const char *lds, int row, int grp, int half) {
        if constexpr (SLOW && WORDS) {
            u32x4 v;
#pragma unroll
            for (int s = 0; s < 4; ++s) v[s] = *(const unsigned *)(lds + (grp * 8 + half * 4 + s) * SLOW_ROW + row * 4);
            return v;
        } else {
            return *(const u32x4 *)(lds + row * ROW_BYTES + grp * 32 + half * 16);
        }
    }
};

// Workgroup -> tile, split and head.  Workgroups go to the 8 XCDs in turn, each with its own L2: an XCD gets a run of neighbours in
// the order [head][split][tile], and within a head tiles go down 8 rows of tiles before they move right, so that the workgroups
// that share an L2 at a time share rows of both operands.
struct Place { int q, p, split, g; };
__device__ __forceinline__ Place place_of(long wg, long total, int tq, int tp, int S) {
    const long per = total / 8, rest = total % 8, xcd = wg % 8, i = wg / 8;
    const long id = xcd * per + (xcd < rest ? xcd : rest) + i;
    const int tiles = tq * tp;
    Place w;
    w.g = (int)(id / ((long)tiles * S));
    const long in_head = id - (long)w.g * tiles * S;
    w.split = (int)(in_head / tiles);
    const int tile = (int)(in_head - (long)w.split * tiles);
    const int band = tile / (8 * tp), q0 = band * 8, h = tq - q0 < 8 ? tq - q0 : 8, in = tile - band * 8 * tp;
    w.q = q0 + in % h;
    w.p = in / h;
    return w;
}

// FQ x FP blocks of 32 x 32 results per wave, NQ x NP waves
template <class T, bool PSLOW, bool QSLOW, int NQ, int NP, int FQ, int FP>
__global__ __launch_bounds__(64 * NQ * NP, 2) void k_linear_tile(Product pr, Epilogue e, int tq, int tp) {
    constexpr int TQ = NQ * FQ * 32, TP = NP * FP * 32, NT = 64 * NQ * NP;
    constexpr bool BIG = FQ * FP >= 8;                        // (its registers are all in use: near() operands only, see run_product)
    typedef Stager<T, TP, PSLOW, NT> SP;
    typedef Stager<T, TQ, QSLOW, NT> SQ;
    constexpr int BC = SP::BC;
    __shared__ __attribute__((aligned(16))) char lds[2 * SP::BYTES + 2 * SQ::BYTES];
    char *const lds_p = lds, *const lds_q = lds + 2 * SP::BYTES;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, half = lane >> 5, l32 = lane & 31;
    const int wq = (wave / NP) * (FQ * 32), wp = (wave % NP) * (FP * 32);
    const Place w = place_of(blockIdx.x, gridDim.x, tq, tp, pr.S);
    const int split = w.split, g = w.g;
    const long q0 = pr.nq < TQ ? 0 : (long)w.q * TQ + TQ <= pr.nq ? (long)w.q * TQ : pr.nq - TQ;
    const long p0 = pr.np < TP ? 0 : (long)w.p * TP + TP <= pr.np ? (long)w.p * TP : pr.np - TP;
    const long cb = split * pr.c_split, ce = cb + pr.c_split < pr.nc ? cb + pr.c_split : pr.nc;
    const T *P = (const T *)pr.P.data + g * pr.P.head, *Q = (const T *)pr.Q.data + g * pr.Q.head;

    f32x16 acc[FP][FQ];
#pragma unroll
    for (int a = 0; a < FP; ++a)
#pragma unroll
        for (int b = 0; b < FQ; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.f;

    if (cb < ce) {
        SP sp;
        SQ sq;
        const long ldp = pr.P.row, ldq = pr.Q.row, rows_p = pr.np < TP ? pr.np : TP, rows_q = pr.nq < TQ ? pr.nq : TQ;
        const bool near_p = BIG || SP::near(ldp, pr.np), near_q = BIG || SQ::near(ldq, pr.nq);
        const T *P0 = P + (PSLOW ? p0 : p0 * ldp), *Q0 = Q + (QSLOW ? q0 : q0 * ldq);
        sp.start(ldp, rows_p, t);
        sq.start(ldq, rows_q, t);
        auto fetch = [&](long c) {                            // (every branch is uniform)
            const int left = (int)(ce - c < BC ? ce - c : BC);
            const T *cp = P0 + (PSLOW ? c * ldp : c), *cq = Q0 + (QSLOW ? c * ldq : c);
            if (near_p && near_q && left == BC) {
                sp.load(cp, ldp);
                sq.load(cq, ldq);
            } else {
                if (near_p) sp.template load_last<!BIG>(cp, ldp, left, pr.nc, t);
                else if constexpr (!BIG) sp.load_far(cp, ldp, left, rows_p, t);
                if (near_q) sq.template load_last<!BIG>(cq, ldq, left, pr.nc, t);
                else if constexpr (!BIG) sq.load_far(cq, ldq, left, rows_q, t);
            }
        };
        auto store = [&](int buf, long c) {
            if (c + BC > ce) {
                sp.trim((int)(ce - c), near_p && pr.nc >= SP::V, t);
                sq.trim((int)(ce - c), near_q && pr.nc >= SP::V, t);
            }
            sp.put(lds_p + buf * SP::BYTES, t);
            sq.put(lds_q + buf * SQ::BYTES, t);
        };
        fetch(cb);
        store(0, cb);
        __syncthreads();
        int buf = 0;
        for (long c = cb; c < ce; c += BC, buf ^= 1) {
            const bool more = c + BC < ce;
            if (more) fetch(c + BC);
            // the next group's fragments are read while this one's are used (BIG: two waves a SIMD take turns instead)
            constexpr int SETS = BIG ? 1 : 2;
            u32x4 fp[SETS][FP], fq[SETS][FQ];
            auto fragments = [&](int set, int grp) {
#pragma unroll
                for (int a = 0; a < FP; ++a) fp[set][a] = SP::fragment(lds_p + buf * SP::BYTES, wp + a * 32 + l32, grp, half);
#pragma unroll
                for (int b = 0; b < FQ; ++b) fq[set][b] = SQ::fragment(lds_q + buf * SQ::BYTES, wq + b * 32 + l32, grp, half);
            };
            if (!BIG) fragments(0, 0);
#pragma unroll
            for (int grp = 0; grp < 4; ++grp) {
                const int set = grp % SETS;
                if (BIG) fragments(0, grp);
                else if (grp < 3) fragments(set ^ 1, grp + 1);
                // BIG puts the next step into LDS in the middle of this one's products, to be done when they end (dw of 8192 rows,
                // 4096 x 4096: 364 -> 332 us); the smaller tiles have a second workgroup on the CU to fill that gap
                if (BIG && grp == 2 && more) store(buf ^ 1, c + BC);
                if (!BIG) UMR_SCHED_FENCE();
#pragma unroll
                for (int a = 0; a < FP; ++a)
#pragma unroll
                    for (int b = 0; b < FQ; ++b) acc[a][b] = mma32(T{}, fp[set][a], fq[set][b], acc[a][b]);
                if (!BIG) UMR_SCHED_FENCE();
            }
            if (!BIG && more) store(buf ^ 1, c + BC);
            __syncthreads();
        }
    }
    // 32 rows at a time go through the wave's own part of LDS, so that 8 or 16 lanes store (and read the residual of) one row
    // together: 128 bytes and more of it, where the accumulators' own layout would touch 16 or 32 bytes of 32 rows at once.
    constexpr int COLS = FP * 32, LANES = COLS / 4, ITS = 32 * LANES / 64;
    float *own = (float *)lds + wave * 32 * (COLS + 4);
    const bool inside = pr.nq >= TQ && pr.np >= TP;           // (uniform) no results to drop
    const long p = p0 + wp + (lane % LANES) * 4, n = inside ? 4 : pr.np - p;
    const int row0 = lane / LANES;
    float bias[4] = {0.f, 0.f, 0.f, 0.f};
    if (e.bias && !e.part && n > 0) load4((const T *)e.bias + g * pr.np + p, n, bias);
#pragma unroll
    for (int b = 0; b < FQ; ++b) {
        const long q = q0 + wq + b * 32 + row0;
        float res[ITS][4];
        if (e.res && !e.part) {
            const T *src = (const T *)e.res + q * e.r_row + g * e.r_head + p;
#pragma unroll
            for (int k = 0; k < ITS; ++k)
                if (inside) load4(src + k * (64 / LANES) * e.r_row, 4, res[k]);
                else if (q + k * (64 / LANES) < pr.nq) load4(src + k * (64 / LANES) * e.r_row, n, res[k]);
        }
#pragma unroll
        for (int a = 0; a < FP; ++a)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                *(f32x4 *)(own + l32 * (COLS + 4) + a * 32 + 8 * r + 4 * half) =
                    f32x4{acc[a][b][4 * r], acc[a][b][4 * r + 1], acc[a][b][4 * r + 2], acc[a][b][4 * r + 3]};
        UMR_WAVE_LDS_HANDOVER();
#pragma unroll
        for (int k = 0; k < ITS; ++k) {
            const int row = row0 + k * (64 / LANES);
            const f32x4 s = *(const f32x4 *)(own + row * (COLS + 4) + (lane % LANES) * 4);
            float v[4] = {s[0] + bias[0], s[1] + bias[1], s[2] + bias[2], s[3] + bias[3]};
            const long qq = q + k * (64 / LANES);
            if (inside) {
                if (e.part) store4(e.part + (((long)split * pr.G + g) * pr.nq + qq) * pr.np + p, 4, v);
                else finish_row<T>(e, v, res[k], qq * e.o_row + g * e.o_head + p, 4);
            } else if (qq < pr.nq && n > 0) {
                if (e.part) store4(e.part + (((long)split * pr.G + g) * pr.nq + qq) * pr.np + p, n, v);
                else finish_row<T>(e, v, res[k], qq * e.o_row + g * e.o_head + p, n);
            }
        }
        UMR_WAVE_LDS_HANDOVER();
    }
}

// ------------------------------------------------------------------------------------------------ few rows: weights straight to the matrix unit
// q <= 16 QT.  A workgroup owns 32 (fast) or 64 (slow) columns p; its 8 waves share out the contraction, add up in LDS and finish.
// The weights are the traffic: each byte is loaded once, 16 bytes a lane, and goes to the matrix unit from registers; the rows of
// Q come from L2 again for every workgroup.  fp32 8192 x 8192: 48 us at one row (5.6 TB/s of weights), 50 at 16, 67 at 32, 125 at 64
// (16 waves: 50, 54, 71, 113; at 4096 x 4096 18, 19, 24, 37 against 17, 19, 22, 35 with 8); bf16 34 us at 16 rows.  The slow form (dx): 43 us at 16 rows, part of the weights still in the memory-side cache.
template <class T, int QT> __global__ __launch_bounds__(64 * FEW_WAVES) void k_linear_few(Product pr, Epilogue e) {
    constexpr int V = 16 / (int)sizeof(T), PT = 2, STEP = 4 * V, U = QT > 2 ? 1 : 2;     // STEP: contraction of one wave load (64 bytes a row)
    __shared__ __attribute__((aligned(16))) float red[FEW_WAVES][16 * QT][36];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, l16 = lane & 15, h = lane >> 4;
    const int split = blockIdx.y, g = blockIdx.z;
    const long p0 = (long)blockIdx.x * 32;
    const long sb = split * pr.c_split, se = sb + pr.c_split < pr.nc ? sb + pr.c_split : pr.nc;
    long per = (se - sb + FEW_WAVES - 1) / FEW_WAVES;
    per = (per + STEP - 1) / STEP * STEP;
    const long cb = sb + wave * per, ce = cb + per < se ? cb + per : se;
    const T *P = (const T *)pr.P.data + g * pr.P.head, *Q = (const T *)pr.Q.data + g * pr.Q.head;
    const T *prow[PT], *qrow[QT];
#pragma unroll
    for (int a = 0; a < PT; ++a) {
        const long p = p0 + a * 16 + l16;
        prow[a] = P + (p < pr.np ? p : pr.np - 1) * pr.P.row + h * V;
    }
#pragma unroll
    for (int b = 0; b < QT; ++b) {
        const long q = b * 16 + l16;
        qrow[b] = Q + (q < pr.nq ? q : pr.nq - 1) * pr.Q.row + h * V;
    }
    f32x4 acc[PT][QT];
#pragma unroll
    for (int a = 0; a < PT; ++a)
#pragma unroll
        for (int b = 0; b < QT; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    struct Block { u32x4 p[U][PT], q[U][QT]; };               // U wave loads of each row; two of them take turns
    auto load = [&](Block &k, long c) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int a = 0; a < PT; ++a) k.p[u][a] = load16B(prow[a] + c + u * STEP);
#pragma unroll
            for (int b = 0; b < QT; ++b) k.q[u][b] = load16B(qrow[b] + c + u * STEP);
        }
        UMR_SCHED_FENCE();
    };
    auto use = [&](const Block &k) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int a = 0; a < PT; ++a)
#pragma unroll
                for (int b = 0; b < QT; ++b) acc[a][b] = mma16(T{}, k.p[u][a], k.q[u][b], acc[a][b]);
        UMR_SCHED_FENCE();
    };
    const long blocks = ce > cb ? (ce - cb) / (U * STEP) : 0;
    long c = cb + blocks * (U * STEP);
    if (blocks > 0) {
        Block even, odd;
        // workgroups start at different places and wrap around: started together, all would ask L2 for the
        // same few lines of Q at once (fp32 8192 x 8192: one row 69 -> 51 us, 32 rows 97 -> 67; with 64 rows the lines are many
        // anyway, and what neighbours share in the cache counts for more: 8192 x 12000 164 us against 174 with the stagger)
        const long start = QT <= 2 ? blockIdx.x % blocks : 0;
        auto place = [&](long i) { return cb + (i + start < blocks ? i + start : i + start - blocks) * (U * STEP); };
        load(even, place(0));
        long i = 0;
        for (; i + 2 < blocks; i += 2) {
            load(odd, place(i + 1));
            use(even);
            load(even, place(i + 2));
            use(odd);
        }
        if (i + 1 < blocks) {
            load(odd, place(i + 1));
            use(even);
            use(odd);
        } else use(even);
    }
    for (; c < ce; c += STEP) {
        const long left = ce - c - h * V;
        u32x4 fp[PT], fq[QT];
#pragma unroll
        for (int a = 0; a < PT; ++a) fp[a] = load16B_n(prow[a] + c, left);
#pragma unroll
        for (int b = 0; b < QT; ++b) fq[b] = load16B_n(qrow[b] + c, left);
#pragma unroll
        for (int a = 0; a < PT; ++a)
#pragma unroll
            for (int b = 0; b < QT; ++b) acc[a][b] = mma16(T{}, fp[a], fq[b], acc[a][b]);
    }
#pragma unroll
    for (int a = 0; a < PT; ++a)
#pragma unroll
        for (int b = 0; b < QT; ++b) *(f32x4 *)&red[wave][b * 16 + l16][a * 16 + 4 * h] = acc[a][b];
    __syncthreads();
    for (int i = t; i < 16 * QT * 8; i += 64 * FEW_WAVES) {
        const int q = i >> 3, p = (i & 7) * 4;
        f32x4 s = *(const f32x4 *)&red[0][q][p];
#pragma unroll
        for (int w = 1; w < FEW_WAVES; ++w) {
            const f32x4 o = *(const f32x4 *)&red[w][q][p];
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] += o[j];
        }
        float v[4] = {s[0], s[1], s[2], s[3]};
        emit4<T>(e, v, q, p0 + p, pr.nq, pr.np, g, pr.G, split);
    }
}

template <class T, int QT> __global__ __launch_bounds__(64 * FEW_WAVES) void k_linear_few_slow(Product pr, Epilogue e) {
    constexpr bool WORDS = sizeof(T) == 4;
    constexpr int V = 16 / (int)sizeof(T), STEP = 4 * V;      // a wave step: STEP contraction rows x 64 columns
    __shared__ __attribute__((aligned(16))) float red[FEW_WAVES][16 * QT][68];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, l16 = lane & 15, h = lane >> 4;
    const int split = blockIdx.y, g = blockIdx.z;
    const long p0 = (long)blockIdx.x * 64, p = p0 + 4 * l16;  // this lane's 4 columns
    const long sb = split * pr.c_split, se = sb + pr.c_split < pr.nc ? sb + pr.c_split : pr.nc;
    long per = (se - sb + FEW_WAVES - 1) / FEW_WAVES;
    per = (per + STEP - 1) / STEP * STEP;
    const long cb = sb + wave * per, ce = cb + per < se ? cb + per : se;
    const T *P = (const T *)pr.P.data + g * pr.P.head + p, *Q = (const T *)pr.Q.data + g * pr.Q.head;
    const T *qrow[QT];
#pragma unroll
    for (int b = 0; b < QT; ++b) {
        const long q = b * 16 + l16;
        qrow[b] = Q + (q < pr.nq ? q : pr.nq - 1) * pr.Q.row + h * V;
    }
    f32x4 acc[4][QT];                                         // [column of the lane][row block]
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < QT; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    const bool full_cols = p0 + 64 <= pr.np;
    for (long c = cb; c < ce; c += STEP) {
        const bool full = c + STEP <= ce && full_cols;
        u32x4 fq[QT], w[4];                                   // w[column]: its V contraction values
#pragma unroll
        for (int b = 0; b < QT; ++b) fq[b] = full ? load16B(qrow[b] + c) : load16B_n(qrow[b] + c, ce - c - h * V);
        if constexpr (WORDS) {
            u32x4 row[4];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const long cc = c + 4 * h + s;
                row[s] = full ? load16B(P + cc * pr.P.row) : load16B_n(P + cc * pr.P.row, cc < ce ? pr.np - p : 0);
            }
#pragma unroll
            for (int a = 0; a < 4; ++a) w[a] = u32x4{row[0][a], row[1][a], row[2][a], row[3][a]};
        } else {
            u32x2 row[8];
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                const long cc = c + 8 * h + s;
                const T *src = P + cc * pr.P.row;
                if (full) row[s] = *(const u32x2_any *)src;
                else {
                    const u32x4 v = load16B_n(src, cc < ce ? (pr.np - p < 4 ? pr.np - p : 4) : 0);
                    row[s] = u32x2{v[0], v[1]};
                }
            }
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const unsigned lo = row[2 * k][a / 2], hi = row[2 * k + 1][a / 2];
                    w[a][k] = (a & 1) ? (lo >> 16) | (hi & 0xffff0000u) : (lo & 0xffffu) | (hi << 16);
                }
        }
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int b = 0; b < QT; ++b) acc[a][b] = mma16(T{}, w[a], fq[b], acc[a][b]);
    }
    // register r of acc[a]: column 4 (4 h + r) + a
#pragma unroll
    for (int b = 0; b < QT; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) *(f32x4 *)&red[wave][b * 16 + l16][16 * h + 4 * r] = f32x4{acc[0][b][r], acc[1][b][r], acc[2][b][r], acc[3][b][r]};
    __syncthreads();
    for (int i = t; i < 16 * QT * 16; i += 64 * FEW_WAVES) {
        const int q = i >> 4, pp = (i & 15) * 4;
        f32x4 s = *(const f32x4 *)&red[0][q][pp];
#pragma unroll
        for (int w = 1; w < FEW_WAVES; ++w) {
            const f32x4 o = *(const f32x4 *)&red[w][q][pp];
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] += o[j];
        }
        float v[4] = {s[0], s[1], s[2], s[3]};
        emit4<T>(e, v, q, p0 + pp, pr.nq, pr.np, g, pr.G, split);
    }
}

// ------------------------------------------------------------------------------------------------ a short contraction: outer products
// dw of few rows m: the result is all the traffic.  A wave makes 64 x 64 results from registers, without LDS or barriers; both
// operands are slow, so that a lane gathers the contraction values of one column (they come from L2).  Here the operand whose
// columns run along memory is the matrix instruction's second: 32 lanes then hold 32 neighbours (of 16 bits: 32 pairs of them) and a
// store of 4 bytes a lane writes two whole lines of 128 bytes.  8192 x 8192 fp32 of 16 rows: 54 us, streamed 46 (5.9 TB/s; results of
// 64 MB and more are streamed: they do not fit the caches, and what was there stays); 64 x 64 tiles through LDS 100.
template <class T, bool STREAM> __global__ __launch_bounds__(256) void k_linear_outer(Product pr, T *out, long o_row, long o_head) {
    constexpr bool WORDS = sizeof(T) == 4;
    constexpr int V = 16 / (int)sizeof(T), STEP = 2 * V;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l32 = lane & 31, half = lane >> 5, g = blockIdx.z;
    long p0 = (long)blockIdx.x * 256 + wave * 64, q0 = (long)blockIdx.y * 64;
    if (p0 >= pr.np) return;
    p0 = p0 + 64 <= pr.np ? p0 : pr.np - 64;                  // (np, nq >= 64: the last tiles overlap, with the same bits)
    q0 = q0 + 64 <= pr.nq ? q0 : pr.nq - 64;
    const T *P = (const T *)pr.P.data + g * pr.P.head + p0, *Q = (const T *)pr.Q.data + g * pr.Q.head + q0;
    f32x16 acc[2][2];                                         // [p half][q half]; 16 bits: of the p's, the even and the odd ones
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.f;
    for (long c = 0; c < pr.nc; c += STEP) {
        u32x4 fp[2], fq[2];
        if constexpr (WORDS) {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const long cc = c + half * V + s, row = cc < pr.nc ? cc : pr.nc - 1;
                const unsigned keep = cc < pr.nc ? 0xffffffffu : 0u;
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    fp[a][s] = as_u32(P[row * pr.P.row + a * 32 + l32]) & keep;
                    fq[a][s] = as_u32(Q[row * pr.Q.row + a * 32 + l32]) & keep;
                }
            }
        } else {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                unsigned p[2], q[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const long cc = c + half * V + 2 * s + j, row = cc < pr.nc ? cc : pr.nc - 1;
                    const unsigned keep = cc < pr.nc ? 0xffffffffu : 0u;
                    p[j] = *(const u32_any *)(P + row * pr.P.row + 2 * l32) & keep;
                    q[j] = *(const u32_any *)(Q + row * pr.Q.row + 2 * l32) & keep;
                }
                fp[0][s] = (p[0] & 0xffffu) | (p[1] << 16);
                fp[1][s] = (p[0] >> 16) | (p[1] & 0xffff0000u);
                fq[0][s] = (q[0] & 0xffffu) | (q[1] << 16);
                fq[1][s] = (q[0] >> 16) | (q[1] & 0xffff0000u);
            }
        }
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int b = 0; b < 2; ++b) acc[a][b] = mma32(T{}, fq[b], fp[a], acc[a][b]);
    }
    out += g * o_head + p0;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int i = 8 * (r / 4) + 4 * half + r % 4;
            T *row = out + (q0 + (WORDS ? b * 32 + i : 2 * i + b)) * o_row;
            if constexpr (WORDS) {
#pragma unroll
                for (int a = 0; a < 2; ++a) store_word<STREAM>(row + a * 32 + l32, as_u32(acc[a][b][r]));
            } else store_word<STREAM>(row + 2 * l32, (unsigned)from_f32<T>(acc[0][b][r]).bits | ((unsigned)from_f32<T>(acc[1][b][r]).bits << 16));
        }
}

// ------------------------------------------------------------------------------------------------ act' and the sums over the rows
template <int N> struct Count { static constexpr int value = N; };

// One pass over gy and z.  A wave takes 256 columns (4 a lane) of the rows r0 + wave, r0 + wave + 4, ...; sums meet in LDS, and
// over the row blocks in k_linear_colsum, both in a fixed order.  The lanes at the right edge take the last 4 columns, some of them
// twice, so that every load is 4 wide and none is behind a branch.  8192 x 4096 gelu in bf16: 61 us, 268 MB at 4.4 TB/s.
template <class T>
__global__ __launch_bounds__(256) void k_linear_act_grad(const T *__restrict__ gy, long g_row, long g_head, const void *__restrict__ z, T *__restrict__ dz, T *db, T *dr, float *part,
                                                         long M, long N, int G, long rows, int act, float slope) {
    __shared__ __attribute__((aligned(16))) float red[2][4][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = blockIdx.z;
    const long first = (long)blockIdx.x * 256, want = first + lane * 4;
    const long n = want + 4 <= N || N < 4 ? want : N - 4, left = N - n;
    const long r0 = (long)blockIdx.y * rows, r1 = r0 + rows < M ? r0 + rows : M;
    float sz[4] = {0.f, 0.f, 0.f, 0.f}, sg[4] = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](auto count, long m, long wide) {           // rows m, m + 4, ..: every load before the first use
        constexpr int B = decltype(count)::value;
        float gv[B][4], zv[B][4];
#pragma unroll
        for (int k = 0; k < B; ++k) load4(gy + (m + 4 * k) * g_row + g * g_head + n, wide, gv[k]);
        if (dz) {
#pragma unroll
            for (int k = 0; k < B; ++k) {
                const long o = ((m + 4 * k) * G + g) * N + n;
                if (kinked(act)) load4((const T *)z + o, wide, zv[k]);
                else load4((const float *)z + o, wide, zv[k]);
            }
        }
#pragma unroll
        for (int k = 0; k < B; ++k) {
#pragma unroll
            for (int i = 0; i < 4; ++i) sg[i] += gv[k][i];
            if (dz) {
#pragma unroll
                for (int i = 0; i < 4; ++i) gv[k][i] *= act_slope<sizeof(T) == 4>(zv[k][i], act, slope);
                // dz in the operator's own type: the operand of both gradient products (16-bit matrix instructions take 16 bits).
                // This second rounding puts dx and dw 1.4 times as far from 64 bits as their own rounding alone would (bf16 2.35e-3
                // against 1.66e-3 in the norm, fp16 2.9e-4 against 2.1e-4; a layer that rounds z too, 2.42e-3 and 3.0e-4); the halves of
                // an fp32 dz would take both products twice.  The sums over the rows have it in fp32.
                store4(dz + ((m + 4 * k) * G + g) * N + n, wide, gv[k]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) sz[i] += gv[k][i];
        }
    };
    if (N >= 4) {                                             // (uniform)
        if (want < N) {
            long m = r0 + wave;
            for (; m + 12 < r1; m += 16) add(Count<4>{}, m, 4);
            for (; m < r1; m += 4) add(Count<1>{}, m, 4);
        }
    } else if (left > 0) {
        for (long m = r0 + wave; m < r1; m += 4) add(Count<1>{}, m, left);
    }
    if (!db && !dr) return;                                   // (uniform)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long k = n + i - first;                         // its column of this workgroup (the edge lane's first may be another's)
        if (want < N && k >= 0 && k < 256) { red[0][wave][k] = sz[i]; red[1][wave][k] = sg[i]; }
    }
    __syncthreads();
    const int i = threadIdx.x;
    const long col = first + i;
    if (col >= N) return;
    const float a = ((red[0][0][i] + red[0][1][i]) + red[0][2][i]) + red[0][3][i];
    const float b = ((red[1][0][i] + red[1][1][i]) + red[1][2][i]) + red[1][3][i];
    if (part) {
        part[((long)blockIdx.y * 2 * G + g) * N + col] = a;
        part[((long)blockIdx.y * 2 * G + G + g) * N + col] = b;
    } else {
        if (db) db[g * N + col] = from_f32<T>(a);
        if (dr) dr[g * N + col] = from_f32<T>(b);
    }
}

template <class T> __global__ __launch_bounds__(256) void k_linear_colsum(const float *part, int blocks, T *db, T *dr, long cols) {
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < cols; i += (long)gridDim.x * 256) {
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            T *out = which ? dr : db;
            if (!out) continue;
            float s = 0.f;
#pragma unroll 8
            for (int b = 0; b < blocks; ++b) s += part[((long)b * 2 + which) * cols + i];
            out[i] = from_f32<T>(s);
        }
    }
}

// ------------------------------------------------------------------------------------------------ launches
// the product from head g0 on (not of a split contraction: its parts lie head by head in one plane)
template <class T> void from_head(Product &pr, Epilogue &e, long g0) {
    pr.P.data = (const T *)pr.P.data + g0 * pr.P.head;
    pr.Q.data = (const T *)pr.Q.data + g0 * pr.Q.head;
    if (e.bias) e.bias = (const T *)e.bias + g0 * pr.np;
    if (e.res) e.res = (const T *)e.res + g0 * e.r_head;
    e.out = (T *)e.out + g0 * e.o_head;
    if (e.z && kinked(e.act)) e.z = (T *)e.z + g0 * e.o_head;
    else if (e.z) e.z = (float *)e.z + g0 * e.o_head;
}

// `most`: workgroups of a launch, whose threads are counted in 32 bits.  More heads than fit take several launches.
template <class T, int NQ, int NP, int FQ, int FP>
int launch_tile(int kind, const Product &all, const Epilogue &epilogue, hipStream_t st, long most = 0xffffffffL / (64 * NQ * NP)) {
    const long tq = ceil_div(all.nq, NQ * FQ * 32), tp = ceil_div(all.np, NP * FP * 32), head = tq * tp * all.S;
    const long at_once = most / head < all.G ? most / head : all.G;
    if (at_once < 1 || (at_once < all.G && all.S > 1)) return UMR_ERR_ARG;
    constexpr int NT = 64 * NQ * NP;
    for (long g0 = 0; g0 < all.G; g0 += at_once) {
        Product pr = all;
        Epilogue e = epilogue;
        from_head<T>(pr, e, g0);
        pr.G = (int)(all.G - g0 < at_once ? all.G - g0 : at_once);
        const unsigned grid = (unsigned)(head * pr.G);
        if (kind == FORWARD) UMR_LAUNCH((k_linear_tile<T, false, false, NQ, NP, FQ, FP>), grid, NT, 0, st, pr, e, (int)tq, (int)tp);
        else if (kind == GRAD_INPUT) UMR_LAUNCH((k_linear_tile<T, true, false, NQ, NP, FQ, FP>), grid, NT, 0, st, pr, e, (int)tq, (int)tp);
        else UMR_LAUNCH((k_linear_tile<T, true, true, NQ, NP, FQ, FP>), grid, NT, 0, st, pr, e, (int)tq, (int)tp);
        if (umr_launch_status() != UMR_OK) return UMR_ERR_LAUNCH;
    }
    return UMR_OK;
}

template <class T, int QT> int launch_few(int kind, const Product &pr, const Epilogue &e, hipStream_t st) {
    const dim3 grid((unsigned)ceil_div(pr.np, kind == FORWARD ? 32 : 64), pr.S, pr.G);
    if (kind == FORWARD) UMR_LAUNCH((k_linear_few<T, QT>), grid, 64 * FEW_WAVES, 0, st, pr, e);
    else UMR_LAUNCH((k_linear_few_slow<T, QT>), grid, 64 * FEW_WAVES, 0, st, pr, e);
    return umr_launch_status();
}

}  // namespace

template <class T> int run_product(int kind, const Plan &pl, Product pr, Epilogue e, void *workspace, hipStream_t st) {
    pr.S = pl.S;
    pr.c_split = pl.c_split;
    Epilogue first = e;
    first.part = pl.S > 1 ? (float *)workspace : nullptr;
    int rc;
    if (pl.outer) {
        const dim3 grid((unsigned)ceil_div(pr.np, 256), (unsigned)ceil_div(pr.nq, 64), pr.G);
        const bool stream = (double)pr.nq * pr.np * pr.G * sizeof(T) >= 64e6;
        if (stream) UMR_LAUNCH((k_linear_outer<T, true>), grid, 256, 0, st, pr, (T *)e.out, e.o_row, e.o_head);
        else UMR_LAUNCH((k_linear_outer<T, false>), grid, 256, 0, st, pr, (T *)e.out, e.o_row, e.o_head);
        rc = umr_launch_status();
    } else if (pl.few) {
        rc = pr.nq <= 16 ? launch_few<T, 1>(kind, pr, first, st) : pr.nq <= 32 ? launch_few<T, 2>(kind, pr, first, st) : launch_few<T, 4>(kind, pr, first, st);
    } else {
        rc = UMR_ERR_ARG;
        const bool near = pr.P.row < NEAR && pr.Q.row < NEAR && pr.np >= 256 && pr.nq >= 256 && pr.nc >= 8;
        if (pl.tile == T256x256 && !near) rc = launch_tile<T, 2, 2, 2, 2>(kind, pr, first, st);
        else if (pl.tile == T64x64) rc = launch_tile<T, 2, 2, 1, 1>(kind, pr, first, st);
        else if (pl.tile == T128x128) rc = launch_tile<T, 2, 2, 2, 2>(kind, pr, first, st);
        else if constexpr (sizeof(T) == 2) rc = launch_tile<T, 2, 4, 4, 2>(kind, pr, first, st);
    }
    if (rc != UMR_OK || pl.S == 1) return rc;
    const long work = ceil_div(pr.nq * pr.G * ceil_div(pr.np, 4), 256);
    UMR_LAUNCH((k_linear_join<T>), (unsigned)(work < 8192 ? work : 8192), 256, 0, st, e, (const float *)workspace, pl.S, pr.nq, pr.np, pr.G);
    return umr_launch_status();
}

template <class T> int run_act_grad(const ActGrad &a, hipStream_t st) {
    const dim3 grid((unsigned)ceil_div(a.N, 256), (unsigned)a.blocks, (unsigned)a.G);
    UMR_LAUNCH((k_linear_act_grad<T>), grid, 256, 0, st, (const T *)a.gy, a.g_row, a.g_head, a.z, (T *)a.dz, (T *)a.db, (T *)a.dr, a.part, a.M, a.N,
               a.G, a.rows, a.act, a.slope);
    if (umr_launch_status() != UMR_OK) return UMR_ERR_LAUNCH;
    if (a.part) {
        const long cols = a.G * a.N, work = ceil_div(cols, 256);
        UMR_LAUNCH((k_linear_colsum<T>), (unsigned)(work < 8192 ? work : 8192), 256, 0, st, (const float *)a.part, (int)a.blocks, (T *)a.db, (T *)a.dr, cols);
    }
    return umr_launch_status();
}

}  // namespace umr_linear
