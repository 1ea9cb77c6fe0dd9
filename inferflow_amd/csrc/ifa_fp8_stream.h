// ifa_fp8_stream.h -- products of a few rows in 8-bit floating point: sixteen matrix rows against TILES x 16 activation rows, the blocks of 128 columns one after the other or shared out
// to waves.  Bound by the matrix's bytes: they go from memory to registers, DEPTH blocks asked for while DEPTH blocks are multiplied.
// One row, 4096 x 11008 from memory: 10.6 us, 4.3 TB/s with the launch's start and end (a large copy: 4.9); two blocks asked for at a time or 32 matrix rows a workgroup: no faster.
#pragma once
#include "ifa_fp8.h"

namespace ifa8 {

// acc[i][j][r] += the sums over blocks first, first + step, ... of matrix row n0[i] + 4 (l / 16) + r and activation row of tile j, lane l % 16.  w[i] / sw[i]: the lane's matrix row and its
// row of block scales (the same in all lanes); a[j] / sa[j]: the lane's activation row and its scales.  Columns beyond `cols` are neither read nor counted.
template <bool WIDE, int DEPTH, int MATS, int TILES, bool ENDS = true>
__device__ __forceinline__ void stream_blocks(const uint8_t *const (&w)[MATS], const float *const (&sw)[MATS], const uint8_t *const (&a)[TILES], const float *const (&sa)[TILES], int cols,
                                              int first, int step, f32x4 (&acc)[MATS][TILES])
{
    const int lane = threadIdx.x & 63, k_lane = 16 * (lane >> 4), whole = cols / BLOCK;
    struct Group { u32x4 w[DEPTH][MATS][2], a[DEPTH][TILES][2]; float sw[DEPTH][MATS], sa[DEPTH][TILES]; };
    auto ask = [&](Group &G, int kb0) {          // (past the last whole block of a last group: that block again, not used)
#pragma unroll
        for (int d = 0; d < DEPTH; d++) {
            const int kb = min(kb0 + d * step, whole - 1);
            const size_t k = (size_t)kb * BLOCK + k_lane;
#pragma unroll
            for (int i = 0; i < MATS; i++) {
                G.w[d][i][0] = *reinterpret_cast<const u32x4 *>(w[i] + k); G.w[d][i][1] = *reinterpret_cast<const u32x4 *>(w[i] + k + 64);
                G.sw[d][i] = sw[i][kb];
            }
        }
#pragma unroll
        for (int d = 0; d < DEPTH; d++) {
            const int kb = min(kb0 + d * step, whole - 1);
            const size_t k = (size_t)kb * BLOCK + k_lane;
#pragma unroll
            for (int j = 0; j < TILES; j++) {
                G.a[d][j][0] = *reinterpret_cast<const u32x4 *>(a[j] + k); G.a[d][j][1] = *reinterpret_cast<const u32x4 *>(a[j] + k + 64);
                G.sa[d][j] = sa[j][kb];
            }
        }
    };
    auto one = [&](const u32x4 (&gw)[MATS][2], const u32x4 (&ga)[TILES][2], const float (&gsw)[MATS], const float (&gsa)[TILES]) {
        Operand<WIDE> av[TILES], wv[MATS];
#pragma unroll
        for (int i = 0; i < MATS; i++) wv[i].set(gw[i][0], gw[i][1]);
#pragma unroll
        for (int j = 0; j < TILES; j++) {
            av[j].set(ga[j][0], ga[j][1]);
#pragma unroll
            for (int i = 0; i < MATS; i++) {
                const f32x4 p = mfma128(wv[i], av[j]);
                const float f = gsw[i] * gsa[j];
#pragma unroll
                for (int r = 0; r < 4; r++) acc[i][j][r] = fmaf(p[r], f, acc[i][j][r]);
            }
        }
    };
    if (first < whole) {
        // a group asked for while the one before it is multiplied; with ENDS none beyond the last (a request that may or may not have gone out would have the compiler wait for all: the ends
        // stand apart.  One row, 11008 x 4096: 14.3 -> 12.2 us)
        Group G[2];
        const int groups = (whole - first + DEPTH * step - 1) / (DEPTH * step);
        auto at = [&](int g) { return first + g * DEPTH * step; };
        // The condition below always holds with DEPTH 1, and stays: without it hipcc 7.2 takes the second half of an 8-bit operand for one that nobody has written where it copies the operand behind the loop's
        // requests (16-bit outputs; its assembly shows "kill: def" of registers by others), and the sums are wrong.
        auto go = [&](const Group &X, int g) {
#pragma unroll
            for (int d = 0; d < DEPTH; d++) if (at(g) + d * step < whole) one(X.w[d], X.a[d], X.sw[d], X.sa[d]);
        };
        ask(G[0], at(0));
        if constexpr (!ENDS) {          // (the other form's copies of the loop take more registers than four waves a SIMD have: gate and up of 53 rows' experts 22.7 -> 33 us)
            int kb = first;
            while (true) {
                ask(G[1], kb + DEPTH * step);
#pragma unroll
                for (int d = 0; d < DEPTH; d++) if (kb + d * step < whole) one(G[0].w[d], G[0].a[d], G[0].sw[d], G[0].sa[d]);
                kb += DEPTH * step;
                if (kb >= whole) break;
                ask(G[0], kb + DEPTH * step);
#pragma unroll
                for (int d = 0; d < DEPTH; d++) if (kb + d * step < whole) one(G[1].w[d], G[1].a[d], G[1].sw[d], G[1].sa[d]);
                kb += DEPTH * step;
                if (kb >= whole) break;
            }
        } else if (groups == 1) go(G[0], 0);
        else {
            ask(G[1], at(1));
            int g = 0;
            while (true) {
                if (g + 2 >= groups) { go(G[0], g); go(G[1], g + 1); break; }
                go(G[0], g); ask(G[0], at(g + 2)); g++;
                if (g + 2 >= groups) { go(G[1], g); go(G[0], g + 1); break; }
                go(G[1], g); ask(G[1], at(g + 2)); g++;
            }
        }
    }
    if (whole * BLOCK < cols && whole % step == first) {          // the part of a block behind them
        const int k = whole * BLOCK + k_lane;
        const u32x4 zero = {0u, 0u, 0u, 0u};
        u32x4 gw[MATS][2], ga[TILES][2];
        float gsw[MATS], gsa[TILES];
#pragma unroll
        for (int i = 0; i < MATS; i++) {
            gw[i][0] = k < cols ? *reinterpret_cast<const u32x4 *>(w[i] + k) : zero; gw[i][1] = k + 64 < cols ? *reinterpret_cast<const u32x4 *>(w[i] + k + 64) : zero;
            gsw[i] = sw[i][whole];
        }
#pragma unroll
        for (int j = 0; j < TILES; j++) {
            ga[j][0] = k < cols ? *reinterpret_cast<const u32x4 *>(a[j] + k) : zero; ga[j][1] = k + 64 < cols ? *reinterpret_cast<const u32x4 *>(a[j] + k + 64) : zero;
            gsa[j] = sa[j][whole];
        }
        one(gw, ga, gsw, gsa);
    }
}

// the sums of WAVES waves added up in wave 0 in the order of the waves
template <int WAVES, int MATS, int TILES>
__device__ __forceinline__ void join_waves(f32x4 (&acc)[MATS][TILES], f32x4 *red)      // red: [WAVES - 1][MATS][TILES][64]
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (wave > 0) {
#pragma unroll
        for (int i = 0; i < MATS; i++)
#pragma unroll
            for (int j = 0; j < TILES; j++) red[((wave - 1) * MATS * TILES + i * TILES + j) * 64 + lane] = acc[i][j];
    }
    __syncthreads();
    if (wave == 0) {
#pragma unroll
        for (int v = 0; v < WAVES - 1; v++)
#pragma unroll
            for (int i = 0; i < MATS; i++)
#pragma unroll
                for (int j = 0; j < TILES; j++) {
                    const f32x4 o = red[(v * MATS * TILES + i * TILES + j) * 64 + lane];
#pragma unroll
                    for (int r = 0; r < 4; r++) acc[i][j][r] += o[r];
                }
    }
}

} // namespace ifa8
