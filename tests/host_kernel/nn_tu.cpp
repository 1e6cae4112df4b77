// nn_tu.cpp -- TEST INFRASTRUCTURE: the network-side operators (-DUMR_TU='"../../umr_amd/csrc/<name>.hip"') on the wave64 emulator
// of wave_emu.h, with the matrix instructions restated from their operand layout.  tests/host_nn.py builds libumr_nn_host.so.
#include "wave_emu.h"
#include "../../umr_amd/csrc/nn_common.h"

namespace emu_mma {
// operands of the wave's lanes; two sets, so that a lane may go on to its next instruction while others still read this one's
struct Slots { u32x4 a[2][emu::MAX_THREADS], b[2][emu::MAX_THREADS]; unsigned char turn[emu::MAX_THREADS]; };
static thread_local Slots g;

// chunk element e of a lane's 16 bytes, in fp32
template <class T> static inline float element(u32x4 v, int e) { return elem_of<T>(v, e); }

// ROWS = 32: row l % 32, lane half l / 32 holds one chunk; ROWS = 16: row l % 16, quarter l / 16.  c[r] of lane l += sum over all
// chunks and their elements of a[row of register r] * b[column l % ROWS]
template <class T, int ROWS, class C> static inline C mma(u32x4 a, u32x4 b, C c, int regs) {
    emu::Block *blk = emu::g_block;
    const int t = blk->cur, w0 = t & ~63, lane = t & 63;
    const int set = g.turn[t];
    g.turn[t] ^= 1;
    g.a[set][t] = a;
    g.b[set][t] = b;
    (void)emu::collect(emu::K_FENCE, 0, 0);
    constexpr int V = 16 / (int)sizeof(T), PARTS = 64 / ROWS;
    for (int r = 0; r < regs; ++r) {
        const int row = ROWS == 32 ? 8 * (r / 4) + 4 * (lane / 32) + r % 4 : 4 * (lane / 16) + r;
        float s = c[r];
        for (int e = 0; e < V; ++e)
            for (int part = 0; part < PARTS; ++part)
                s += element<T>(g.a[set][w0 + part * ROWS + row], e) * element<T>(g.b[set][w0 + part * ROWS + lane % ROWS], e);
        c[r] = s;
    }
    return c;
}
}  // namespace emu_mma
template <class T> f32x16 mma32(T, u32x4 a, u32x4 b, f32x16 c) { return emu_mma::mma<T, 32>(a, b, c, 16); }
template <class T> f32x4 mma16(T, u32x4 a, u32x4 b, f32x4 c) { return emu_mma::mma<T, 16>(a, b, c, 4); }

#include UMR_TU
