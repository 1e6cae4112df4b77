// linear.hip -- fully connected layers with bias, activation and residual in the product's epilogue, and their gradients
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
#include "nn_common.h"

namespace {

// ------------------------------------------------------------------------------------------------ epilogue
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

__host__ __device__ __forceinline__ bool kinked(int act) { return act == UMR_ACT_RELU || act == UMR_ACT_LEAKY_RELU; }

__device__ __forceinline__ float act_value(float z, int act, float slope) {
    switch (act) {                  // (uniform)
        case UMR_ACT_RELU: return z > 0.f ? z : z != z ? z : 0.f;
        case UMR_ACT_LEAKY_RELU: return z > 0.f ? z : slope * z;
        case UMR_ACT_TANH: return tanhf(z);
        case UMR_ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
        case UMR_ACT_SILU: return z / (1.f + expf(-z));
        default: return z;
    }
}

__device__ __forceinline__ float act_slope(float z, int act, float slope) {      // act'(z)
    switch (act) {
        case UMR_ACT_RELU: return z > 0.f ? 1.f : 0.f;
        case UMR_ACT_LEAKY_RELU: return z > 0.f ? 1.f : slope;
        case UMR_ACT_TANH: { const float t = tanhf(z); return 1.f - t * t; }
        case UMR_ACT_GELU: return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * expf(-0.5f * z * z) * 0.39894228040143268f;
        case UMR_ACT_SILU: { const float s = 1.f / (1.f + expf(-z)); return s * (1.f + z * (1.f - s)); }
        default: return 1.f;
    }
}

// 4 neighbours of one row from their sums: bias, z, activation, residual, store
template <class T> __device__ __forceinline__ void finish4(const Epilogue &e, float (&v)[4], long q, long p, long np, int g) {
    const long n = np - p, o = q * e.o_row + g * e.o_head + p;
    if (e.bias) {
        float b[4];
        load4((const T *)e.bias + g * np + p, n, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += b[i];
    }
    // what the backward call needs of z: all of it in fp32 for a smooth activation (rounded to 16 bits it would add to the
    // rounding of dz), the sign for a kinked one
    if (e.z) {
        if (kinked(e.act)) store4((T *)e.z + o, n, v);
        else store4((float *)e.z + o, n, v);
    }
    if (e.act != UMR_ACT_NONE) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = act_value(v[i], e.act, e.slope);
    }
    if (e.res) {
        float r[4];
        load4((const T *)e.res + q * e.r_row + g * e.r_head + p, n, r);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += r[i];
    }
    store4((T *)e.out + o, n, v);
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

// ------------------------------------------------------------------------------------------------ operands
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

// ------------------------------------------------------------------------------------------------ many rows: tiles through LDS
// A tile is TQ x TP results; the contraction advances by 128 bytes a row (32 fp32, 64 of 16 bits).  In LDS a row is 128 bytes +
// 16 of padding: 8 lanes that read the same chunk of 8 rows meet 32 different banks.  An fp32 operand whose contraction is slow
// keeps memory's order [c][row] (the fp32 matrix instructions take one value per lane, so any order serves); a 16-bit one is
// transposed in registers on its way in (8 x 2 or 8 x 4 values per thread).  Two buffers, one barrier per step; the loads of
// the next step are in flight while the matrix unit works.
constexpr int ROW_BYTES = 144;

template <class T, int R, bool SLOW> struct Stager {          // R rows of one operand, 256 threads
    static constexpr bool WORDS = sizeof(T) == 4;
    static constexpr int ES = (int)sizeof(T), V = 16 / ES, BC = 128 / ES;
    static constexpr int N = R / 32;                          // 16-byte pieces per thread
    static constexpr int SLOW_ROW = (R + 8) * 4;              // bytes of one c-row of an fp32 slow tile: halves of a wave (4 c-rows
                                                              // apart) read different banks
    static constexpr int BYTES = SLOW && WORDS ? (BC * SLOW_ROW > R * ROW_BYTES ? BC * SLOW_ROW : R * ROW_BYTES) : R * ROW_BYTES;
    u32x4 r[N];

    // rows r0 .. of `n` rows; contraction c0 .. below c1.  Rows past the end repeat the last one (their results are dropped),
    // contraction past the end is zero.
    __device__ __forceinline__ void load(const T *base, long ld, long r0, long n, long c0, long c1, int t) {
        if constexpr (!SLOW) {
            const bool full = c0 + BC <= c1;
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int idx = t + 256 * u, ch = idx & 7;
                long row = r0 + (idx >> 3);
                row = row < n ? row : n - 1;
                const T *src = base + row * ld + c0 + ch * V;
                r[u] = full ? load16B(src) : load16B_n(src, c1 - c0 - ch * V);
            }
        } else if constexpr (WORDS) {
            const bool full = c0 + BC <= c1 && r0 + R <= n;
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int idx = t + 256 * u, c = idx / (R / 4), col = (idx % (R / 4)) * 4;
                const T *src = base + (c0 + c) * ld + r0 + col;
                r[u] = full ? load16B(src) : load16B_n(src, c0 + c < c1 ? n - r0 - col : 0);
            }
        } else {
            // thread: 8 contraction rows x N neighbours; r holds them row by row (N elements each)
            constexpr int W = N / 2;                          // 32-bit words per contraction row
            const int cg = t / (R / N), col = (t % (R / N)) * N;
            const bool full = c0 + BC <= c1 && r0 + R <= n;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const long c = c0 + cg * 8 + j;
                const T *src = base + c * ld + r0 + col;
                if (full) {
                    if constexpr (W == 2) { const u32x2 v = *(const u32x2_any *)src; r[j / 2][(j % 2) * 2] = v[0]; r[j / 2][(j % 2) * 2 + 1] = v[1]; }
                    else r[j / 4][j % 4] = *(const u32_any *)src;
                } else {
                    const long left = c < c1 ? n - r0 - col : 0;
#pragma unroll
                    for (int w = 0; w < W; ++w) {
                        const unsigned lo = 2 * w < left ? src[2 * w].bits : 0u, hi = 2 * w + 1 < left ? src[2 * w + 1].bits : 0u;
                        r[(j * W + w) / 4][(j * W + w) % 4] = lo | (hi << 16);
                    }
                }
            }
        }
    }

    __device__ __forceinline__ void put(char *lds, int t) const {
        if constexpr (!SLOW) {
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int idx = t + 256 * u;
                *(u32x4 *)(lds + (idx >> 3) * ROW_BYTES + (idx & 7) * 16) = r[u];
            }
        } else if constexpr (WORDS) {
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int idx = t + 256 * u;
                *(u32x4 *)(lds + (idx / (R / 4)) * SLOW_ROW + (idx % (R / 4)) * 16) = r[u];
            }
        } else {
            constexpr int W = N / 2;
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

// Workgroup -> tile.  Workgroups go to the 8 XCDs in turn, each with its own L2: an XCD gets a run of neighbouring tiles, and within
// a run tiles go down 8 rows of tiles before they move right, so that a run shares rows of both operands.
__device__ __forceinline__ void tile_of(int wg, int tq, int tp, int &q, int &p) {
    const int total = tq * tp, per = total / 8, rest = total % 8, xcd = wg % 8, i = wg / 8;
    const int id = xcd * per + (xcd < rest ? xcd : rest) + i;
    const int band = id / (8 * tp), q0 = band * 8, h = tq - q0 < 8 ? tq - q0 : 8, in = id - band * 8 * tp;
    q = q0 + in % h;
    p = in / h;
}

template <class T, bool PSLOW, bool QSLOW, int TQ, int TP>
__global__ __launch_bounds__(256) void k_linear_tile(Product pr, Epilogue e, int tq, int tp) {
    typedef Stager<T, TP, PSLOW> SP;
    typedef Stager<T, TQ, QSLOW> SQ;
    constexpr int FQ = TQ / 64, FP = TP / 64, BC = SP::BC;
    __shared__ __attribute__((aligned(16))) char lds_p[2][SP::BYTES];
    __shared__ __attribute__((aligned(16))) char lds_q[2][SQ::BYTES];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, half = lane >> 5, l32 = lane & 31;
    const int wq = (wave >> 1) * (TQ / 2), wp = (wave & 1) * (TP / 2);
    int iq, ip;
    tile_of(blockIdx.x, tq, tp, iq, ip);
    const int split = blockIdx.y, g = blockIdx.z;
    const long q0 = (long)iq * TQ, p0 = (long)ip * TP;
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
        sp.load(P, pr.P.row, p0, pr.np, cb, ce, t);
        sq.load(Q, pr.Q.row, q0, pr.nq, cb, ce, t);
        sp.put(lds_p[0], t);
        sq.put(lds_q[0], t);
        __syncthreads();
        int buf = 0;
        for (long c = cb; c < ce; c += BC, buf ^= 1) {
            const bool more = c + BC < ce;
            if (more) {
                sp.load(P, pr.P.row, p0, pr.np, c + BC, ce, t);
                sq.load(Q, pr.Q.row, q0, pr.nq, c + BC, ce, t);
            }
            const int left = (int)(ce - c < BC ? ce - c : BC);
#pragma unroll
            for (int grp = 0; grp < 4; ++grp) {
                if (grp * (BC / 4) >= left) break;            // (uniform) a short last step, or a short contraction
                u32x4 fp[FP], fq[FQ];
#pragma unroll
                for (int a = 0; a < FP; ++a) fp[a] = SP::fragment(lds_p[buf], wp + a * 32 + l32, grp, half);
#pragma unroll
                for (int b = 0; b < FQ; ++b) fq[b] = SQ::fragment(lds_q[buf], wq + b * 32 + l32, grp, half);
#pragma unroll
                for (int a = 0; a < FP; ++a)
#pragma unroll
                    for (int b = 0; b < FQ; ++b) acc[a][b] = mma32(T{}, fp[a], fq[b], acc[a][b]);
            }
            if (more) {
                sp.put(lds_p[buf ^ 1], t);
                sq.put(lds_q[buf ^ 1], t);
            }
            __syncthreads();
        }
    }
#pragma unroll
    for (int b = 0; b < FQ; ++b)
#pragma unroll
        for (int a = 0; a < FP; ++a)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = acc[a][b][4 * r + i];
                emit4<T>(e, v, q0 + wq + b * 32 + l32, p0 + wp + a * 32 + 8 * r + 4 * half, pr.nq, pr.np, g, pr.G, split);
            }
}

// ------------------------------------------------------------------------------------------------ few rows: weights straight to the matrix unit
// q <= 16 QT.  A workgroup owns 32 (fast) or 64 (slow) columns p; its 8 waves share out the contraction, add up in LDS and finish.
// The weights are the traffic: each byte is loaded once, 16 bytes a lane, and goes to the matrix unit from registers; the rows of
// Q come from L2 again for every workgroup.
constexpr int FEW_WAVES = 8;

template <class T, int QT> __global__ __launch_bounds__(64 * FEW_WAVES) void k_linear_few(Product pr, Epilogue e) {
    constexpr int V = 16 / (int)sizeof(T), PT = 2, STEP = 4 * V, U = QT > 2 ? 2 : 4;    // STEP: contraction of one wave load (64 bytes a row)
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
    long c = cb;
    for (; c + U * STEP <= ce; c += U * STEP) {
        u32x4 fp[U][PT], fq[U][QT];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int a = 0; a < PT; ++a) fp[u][a] = load16B(prow[a] + c + u * STEP);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int b = 0; b < QT; ++b) fq[u][b] = load16B(qrow[b] + c + u * STEP);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int a = 0; a < PT; ++a)
#pragma unroll
                for (int b = 0; b < QT; ++b) acc[a][b] = mma16(T{}, fp[u][a], fq[u][b], acc[a][b]);
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

// ------------------------------------------------------------------------------------------------ act' and the sums over the rows
// One pass over gy and z.  A wave takes 256 columns (4 a lane) of the rows r0 + wave, r0 + wave + 4, ...; sums meet in LDS, and
// over the row blocks in k_linear_colsum, both in a fixed order.
template <class T>
__global__ __launch_bounds__(256) void k_linear_act_grad(const T *gy, long g_row, long g_head, const void *z, T *dz, T *db, T *dr, float *part,
                                                         long M, long N, int G, long rows, int act, float slope) {
    __shared__ __attribute__((aligned(16))) float red[2][4][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = blockIdx.z;
    const long n = (long)blockIdx.x * 256 + lane * 4, left = N - n;
    const long r0 = (long)blockIdx.y * rows, r1 = r0 + rows < M ? r0 + rows : M;
    float sz[4] = {0.f, 0.f, 0.f, 0.f}, sg[4] = {0.f, 0.f, 0.f, 0.f};
    if (left > 0) {
#pragma unroll 4
        for (long m = r0 + wave; m < r1; m += 4) {
            float gv[4], zv[4];
            load4(gy + m * g_row + g * g_head + n, left, gv);
#pragma unroll
            for (int i = 0; i < 4; ++i) sg[i] += gv[i];
            if (dz) {
                const long o = (m * G + g) * N + n;
                if (kinked(act)) load4((const T *)z + o, left, zv);
                else load4((const float *)z + o, left, zv);
#pragma unroll
                for (int i = 0; i < 4; ++i) gv[i] *= act_slope(zv[i], act, slope);
                // dz in the operator's own type: the operand of both gradient products (16-bit matrix instructions take 16 bits)
                store4(dz + o, left, gv);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) sz[i] += gv[i];
        }
    }
    if (!db && !dr) return;                                   // (uniform)
#pragma unroll
    for (int i = 0; i < 4; ++i) { red[0][wave][lane * 4 + i] = sz[i]; red[1][wave][lane * 4 + i] = sg[i]; }
    __syncthreads();
    const int i = threadIdx.x;
    const long col = (long)blockIdx.x * 256 + i;
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
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= cols) return;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        T *out = which ? dr : db;
        if (!out) continue;
        float s = 0.f;
        for (int b = 0; b < blocks; ++b) s += part[((long)b * 2 + which) * cols + i];
        out[i] = from_f32<T>(s);
    }
}

// ------------------------------------------------------------------------------------------------ plans and launches
enum { FORWARD = 0, GRAD_INPUT = 1, GRAD_WEIGHT = 2 };

inline long ceil_div(long a, long b) { return (a + b - 1) / b; }

struct Plan {
    bool few;
    int tile, S;
    long c_split;
};

// Which kernel, and how many parts of the contraction.
Plan plan(int kind, long nq, long np, long nc, int G, int dtype) {
    Plan pl;
    const int es = dtype == UMR_F32 ? 4 : 2;
    pl.few = kind != GRAD_WEIGHT && nq <= 64;
    long groups, step;
    if (pl.few) {
        groups = ceil_div(np, kind == FORWARD ? 32 : 64) * G;
        pl.tile = 0;
        step = 64 / es * FEW_WAVES * 4;                       // at least 4 loads deep in every wave
    } else {
        pl.tile = ceil_div(nq, 128) * ceil_div(np, 128) * G >= 256 ? 128 : 64;
        groups = ceil_div(nq, pl.tile) * ceil_div(np, pl.tile) * G;
        step = 128 / es * 4;
    }
    long S = groups > 0 ? 256 / groups : 1;
    const long most = nc / step;
    S = S < most ? S : most;
    S = S < 1 ? 1 : S > 64 ? 64 : S;
    const long unit = pl.few ? 64 / es : 128 / es;
    pl.c_split = ceil_div(ceil_div(nc > 0 ? nc : 1, S), unit) * unit;
    pl.S = (int)ceil_div(nc > 0 ? nc : 1, pl.c_split);
    return pl;
}

size_t plan_bytes(const Plan &pl, long nq, long np, int G) { return pl.S > 1 ? (size_t)pl.S * G * nq * np * sizeof(float) : 0; }

template <class T, int TILE> int launch_tile(int kind, const Product &pr, const Epilogue &e, hipStream_t st) {
    const long tq = ceil_div(pr.nq, TILE), tp = ceil_div(pr.np, TILE);
    if (tq * tp > 0x7fffffffL) return UMR_ERR_ARG;
    const dim3 grid((unsigned)(tq * tp), pr.S, pr.G);
    if (kind == FORWARD) UMR_LAUNCH((k_linear_tile<T, false, false, TILE, TILE>), grid, 256, 0, st, pr, e, (int)tq, (int)tp);
    else if (kind == GRAD_INPUT) UMR_LAUNCH((k_linear_tile<T, true, false, TILE, TILE>), grid, 256, 0, st, pr, e, (int)tq, (int)tp);
    else UMR_LAUNCH((k_linear_tile<T, true, true, TILE, TILE>), grid, 256, 0, st, pr, e, (int)tq, (int)tp);
    return umr_launch_status();
}

template <class T, int QT> int launch_few(int kind, const Product &pr, const Epilogue &e, hipStream_t st) {
    const dim3 grid((unsigned)ceil_div(pr.np, kind == FORWARD ? 32 : 64), pr.S, pr.G);
    if (kind == FORWARD) UMR_LAUNCH((k_linear_few<T, QT>), grid, 64 * FEW_WAVES, 0, st, pr, e);
    else UMR_LAUNCH((k_linear_few_slow<T, QT>), grid, 64 * FEW_WAVES, 0, st, pr, e);
    return umr_launch_status();
}

template <class T> int run_typed(int kind, const Plan &pl, Product pr, Epilogue e, void *workspace, hipStream_t st) {
    pr.S = pl.S;
    pr.c_split = pl.c_split;
    Epilogue first = e;
    first.part = pl.S > 1 ? (float *)workspace : nullptr;
    int rc;
    if (pl.few) {
        rc = pr.nq <= 16 ? launch_few<T, 1>(kind, pr, first, st) : pr.nq <= 32 ? launch_few<T, 2>(kind, pr, first, st) : launch_few<T, 4>(kind, pr, first, st);
    } else {
        rc = pl.tile == 128 ? launch_tile<T, 128>(kind, pr, first, st) : launch_tile<T, 64>(kind, pr, first, st);
    }
    if (rc != UMR_OK || pl.S == 1) return rc;
    const long work = ceil_div(pr.nq * pr.G * ceil_div(pr.np, 4), 256);
    UMR_LAUNCH((k_linear_join<T>), (unsigned)(work < 8192 ? work : 8192), 256, 0, st, e, (const float *)workspace, pl.S, pr.nq, pr.np, pr.G);
    return umr_launch_status();
}

bool sizes_ok(long M, long N, long K, int G, int dtype) {
    const long lim = 0x7fffffffL - 256;
    if (M < 0 || N < 0 || K < 0 || G < 1 || G > 65535 || M > lim || N > lim || K > lim) return false;
    if (dtype != UMR_F32 && dtype != UMR_BF16 && dtype != UMR_F16) return false;
    const long wide = N > K ? N : K;
    return (double)M * G * wide < 7e13 && (double)G * N * K < 7e13;
}

int run(int kind, Product pr, const Epilogue &e, int dtype, void *workspace, size_t workspace_bytes, hipStream_t st) {
    if (pr.nq == 0 || pr.np == 0) return UMR_OK;              // nothing to write
    const Plan pl = plan(kind, pr.nq, pr.np, pr.nc, pr.G, dtype);
    if (plan_bytes(pl, pr.nq, pr.np, pr.G) > workspace_bytes || (pl.S > 1 && !workspace)) return UMR_ERR_ARG;
    if (dtype == UMR_F32) return run_typed<float>(kind, pl, pr, e, workspace, st);
    if (dtype == UMR_BF16) return run_typed<bf16_t>(kind, pl, pr, e, workspace, st);
    return run_typed<f16_t>(kind, pl, pr, e, workspace, st);
}

bool strides_ok(long row, long head) { return row >= 0 && head >= 0; }

long act_grad_rows(long M, long N, int G) {                  // rows per workgroup of k_linear_act_grad
    const long cols = ceil_div(N, 256) * G;
    const long blocks = ceil_div(1024, cols > 0 ? cols : 1);
    long rows = ceil_div(M, blocks);
    return rows < 32 ? 32 : rows;
}

}  // namespace

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
    const dim3 grid((unsigned)ceil_div(N, 256), (unsigned)blocks, (unsigned)G);
    const hipStream_t st = (hipStream_t)stream;
    const long cols = (long)G * N;
#define UMR_ACT_GRAD(T)                                                                                                                   \
    {                                                                                                                                     \
        UMR_LAUNCH((k_linear_act_grad<T>), grid, 256, 0, st, (const T *)gy, g_row, g_head, z, (T *)dz, (T *)db, (T *)dr, part, M, N, G, rows, act, slope); \
        if (umr_launch_status() != UMR_OK) return UMR_ERR_LAUNCH;                                                                         \
        if (part) UMR_LAUNCH((k_linear_colsum<T>), (unsigned)ceil_div(cols, 256), 256, 0, st, (const float *)part, (int)blocks, (T *)db, (T *)dr, cols); \
    }
    if (dtype == UMR_F32) UMR_ACT_GRAD(float)
    else if (dtype == UMR_BF16) UMR_ACT_GRAD(bf16_t)
    else UMR_ACT_GRAD(f16_t)
#undef UMR_ACT_GRAD
    return umr_launch_status();
}

}  // extern "C"
