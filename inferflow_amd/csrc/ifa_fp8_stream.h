// ifa_fp8_stream.h -- products of a few rows in 8-bit floating point: sixteen matrix rows against TILES x 16 activation rows by one workgroup, whose
// waves share out the blocks of 128 columns.
#pragma once
#include "ifa_fp8.h"

namespace ifa8 {

constexpr int STREAM_WAVES = 4;

// acc[i][j][r] += the sums of matrix row n0[i] + 4 (l / 16) + r and activation row of tile j, lane l % 16.  w[i] / sw[i]: the lane's matrix row and its row of block
// scales (uniform); a[j] / sa[j]: the lane's activation row and its scales.  Columns beyond `cols` are neither read nor counted.
template <bool WIDE, int MATS, int TILES>
__device__ __forceinline__ void stream_blocks(const uint8_t *const (&w)[MATS], const float *const (&sw)[MATS], const uint8_t *const (&a)[TILES], const float *const (&sa)[TILES], int cols,
                                              int first, int step, f32x4 (&acc)[MATS][TILES])
{
    const int lane = threadIdx.x & 63, k_lane = 32 * (lane >> 4), nb = (cols + BLOCK - 1) / BLOCK;
#pragma unroll 2
    for (int kb = first; kb < nb; kb += step) {
        const int k = kb * BLOCK + k_lane;
        const u32x4 zero = {0u, 0u, 0u, 0u};
        const bool in0 = k < cols, in1 = k + 16 < cols;
        Operand<WIDE> av[TILES], wv[MATS];
        float s[TILES];
#pragma unroll
        for (int i = 0; i < MATS; i++) {
            const u32x4 lo = in0 ? *reinterpret_cast<const u32x4 *>(w[i] + k) : zero, hi = in1 ? *reinterpret_cast<const u32x4 *>(w[i] + k + 16) : zero;
            wv[i].set(lo, hi);
        }
#pragma unroll
        for (int j = 0; j < TILES; j++) {
            const u32x4 lo = in0 ? *reinterpret_cast<const u32x4 *>(a[j] + k) : zero, hi = in1 ? *reinterpret_cast<const u32x4 *>(a[j] + k + 16) : zero;
            av[j].set(lo, hi);
            s[j] = sa[j][kb];
        }
#pragma unroll
        for (int i = 0; i < MATS; i++) {
            const float ws = sw[i][kb];
#pragma unroll
            for (int j = 0; j < TILES; j++) {
                const f32x4 p = mfma128(wv[i], av[j]);
                const float f = ws * s[j];
#pragma unroll
                for (int r = 0; r < 4; r++) acc[i][j][r] = fmaf(p[r], f, acc[i][j][r]);
            }
        }
    }
}

// the waves' sums added up in wave 0 in the order of the waves
template <int MATS, int TILES>
__device__ __forceinline__ void join_waves(f32x4 (&acc)[MATS][TILES], f32x4 *red)      // red: [STREAM_WAVES - 1][MATS][TILES][64]
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
        for (int v = 0; v < STREAM_WAVES - 1; v++)
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
