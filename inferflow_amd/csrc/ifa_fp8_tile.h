// ifa_fp8_tile.h -- products of many rows in 8-bit floating point: output tiles of BM matrix rows x BN activation rows, the blocks of 128 columns through two buffers in LDS.
//   * both operands go from memory to LDS directly, a wave 8 rows x 128 bytes a request; images are [rows][128 bytes] with the eight 16-byte pieces of row r at slot
//     c ^ ((r >> 1) & 7), so that sixteen lanes that read one piece of sixteen rows meet no bank twice (the permutation sits in the requests' source addresses);
//   * a wave multiplies (BM / WM) x (BN / WN) values of a block as 16 x 16 products over all its 128 columns and adds each, times the two scales, to its 32-bit sums: four
//     multiply-adds beside the 32 cycles of a product;
//   * the requests are inline assembly without results (the compiler would wait for all of them in front of every read of LDS); the waits and barriers stand beside them.
// Columns beyond the last block's end: the requests stay inside their row, and both operands' values there are taken as zero.  Rows beyond the last: repeated, not stored.
#pragma once
#include "ifa_fp8.h"

namespace ifa8 {

typedef __attribute__((address_space(3))) char lds_char;

// 64 lanes' 16 bytes each to 1024 consecutive bytes of LDS from `to` (the same in all lanes); arrive behind arrive_all()
__device__ __forceinline__ void request16(const void *from, uint32_t to)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "m0");
}
__device__ __forceinline__ void request16(const void *base, uint32_t offset, uint32_t to)      // (base: the same in all lanes)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base) : "m0");
}
__device__ __forceinline__ void arrive_all()      // this wave's requests are in LDS, then everybody's
{
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
__device__ __forceinline__ int slot_of(int row, int piece) { return piece ^ ((row >> 1) & 7); }

template <int BM, int BN, int WM, int WN> struct Tile {
    static constexpr int WAVES = WM * WN, TM = BM / (16 * WM), TN = BN / (16 * WN), WI = BM / (8 * WAVES), AI = BN / (8 * WAVES), BUF = (BM + BN) * BLOCK, SMEM = 2 * BUF;
    static_assert(WI * 8 * WAVES == BM && AI * 8 * WAVES == BN && TM * 16 * WM == BM && TN * 16 * WN == BN, "whole rows and products a wave");
};

// One tile's sums.  The tile's matrix rows are wbase + woff(r), its activation rows asrc(r); wrow(m): the first of the 16 tile rows of product m of this wave; sw(m, b): the matrix scale of that
// product's rows in block b (ONE_SCALE: the same for all m); sa: of activation row `lane` of this wave's (a lane below 16 TN).
// The sums of a block are taken over one group of products behind it (p), so that no multiply-add waits for the product in front of it.
template <bool WIDE, bool ONE_SCALE, class T, class WOff, class ASrc, class WRow, class SW>
__device__ __forceinline__ void tile_sums(char *smem, int cols, const uint8_t *wbase, WOff woff, ASrc asrc, WRow wrow, SW sw, const float *sa, int arow0, f32x4 (&acc)[T::TM][T::TN])
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_char *)smem;
    const int nb = (cols + BLOCK - 1) / BLOCK, rest = cols - (nb - 1) * BLOCK;
    uint32_t wo[T::WI];
    const uint8_t *ap[T::AI];
    constexpr int WROWS = T::WI * 8 * T::WAVES;
    auto w_piece = [&](int j) { const int r = (wave * T::WI + j) * 8 + (lane >> 3); return 16 * slot_of(r, lane & 7); };
    auto a_piece = [&](int j) { const int r = (wave * T::AI + j) * 8 + (lane >> 3); return 16 * slot_of(r, lane & 7); };
#pragma unroll
    for (int j = 0; j < T::WI; j++) wo[j] = woff((wave * T::WI + j) * 8 + (lane >> 3)) + w_piece(j);
#pragma unroll
    for (int j = 0; j < T::AI; j++) ap[j] = asrc((wave * T::AI + j) * 8 + (lane >> 3)) + a_piece(j);
    auto request = [&](int b, uint32_t to) {
        if (b + 1 < nb || rest == BLOCK) {
#pragma unroll
            for (int j = 0; j < T::WI; j++) request16(wbase + (size_t)b * BLOCK, wo[j], to + (wave * T::WI + j) * 1024);
#pragma unroll
            for (int j = 0; j < T::AI; j++) request16(ap[j] + (size_t)b * BLOCK, to + WROWS * BLOCK + (wave * T::AI + j) * 1024);
        } else {
#pragma unroll
            for (int j = 0; j < T::WI; j++) request16(wbase + (size_t)b * BLOCK, wo[j] - max(0, w_piece(j) + 16 - rest), to + (wave * T::WI + j) * 1024);
#pragma unroll
            for (int j = 0; j < T::AI; j++) request16(ap[j] + (size_t)b * BLOCK - max(0, a_piece(j) + 16 - rest), to + WROWS * BLOCK + (wave * T::AI + j) * 1024);
        }
    };
    const int i = lane & 15, g = lane >> 4;
    auto read = [&](const char *image, int row, int k_end) {      // the lane's pieces g and g + 4 of a row
        const char *at = image + row * BLOCK;
        u32x4 lo = *reinterpret_cast<const u32x4 *>(at + 16 * slot_of(row, g)), hi = *reinterpret_cast<const u32x4 *>(at + 16 * slot_of(row, g + 4));
        const u32x4 zero = {0u, 0u, 0u, 0u};
        if (k_end < BLOCK) { if (16 * g >= k_end) lo = zero; if (16 * g + 64 >= k_end) hi = zero; }
        Operand<WIDE> o;
        o.set(lo, hi);
        return o;
    };
    auto block = [&](const char *buf, int b, int k_end, float scale) {
        Operand<WIDE> av[T::TN];
        float s[T::TN];
#pragma unroll
        for (int j = 0; j < T::TN; j++) {
            av[j] = read(buf + WROWS * BLOCK, arow0 + 16 * j + i, k_end);
            s[j] = __shfl(scale, 16 * j + i, 64);
            if (ONE_SCALE) s[j] *= sw(0, b);
        }
        Operand<WIDE> wnext = read(buf, wrow(0) + i, k_end);
        f32x4 p[2][T::TN];
        auto add = [&](int m, int j) {
            const float f = ONE_SCALE ? s[j] : s[j] * sw(m, b);
#pragma unroll
            for (int r = 0; r < 4; r++) acc[m][j][r] = fmaf(p[m & 1][j][r], f, acc[m][j][r]);
        };
#pragma unroll
        for (int m = 0; m < T::TM; m++) {
            const Operand<WIDE> wv = wnext;
            if (m + 1 < T::TM) wnext = read(buf, wrow(m + 1) + i, k_end);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < T::TN; j++) {
                p[m & 1][j] = mfma128(wv, av[j]);
                if (m > 0) add(m - 1, j);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int j = 0; j < T::TN; j++) add(T::TM - 1, j);
    };
    float scale = sa[0];
    request(0, lds0);
    arrive_all();
    for (int b = 0; b + 1 < nb; b++) {
        const float next = sa[b + 1];
        request(b + 1, lds0 + ((b + 1) & 1) * T::BUF);
        block(smem + (b & 1) * T::BUF, b, BLOCK, scale);
        scale = next;
        arrive_all();
    }
    block(smem + ((nb - 1) & 1) * T::BUF, nb - 1, rest, scale);
}

// A wave's sums by way of LDS, so that they leave in whole lines: f(t, n, v) with N consecutive values of activation row t from matrix row n on (both counted from the wave's first).  Every wave
// has its part of the buffers; all of them are through with the last block.
template <class T, int N, class F> __device__ __forceinline__ void tile_out(char *smem, const f32x4 (&acc)[T::TM][T::TN], F f)
{
    constexpr int PART = T::SMEM / T::WAVES, ROW = T::TM * 64, ROWS = PART / ROW / 16 * 16 < T::TN * 16 ? PART / ROW / 16 * 16 : T::TN * 16, PIECES = T::TM * 4;      // 16-byte pieces a row
    static_assert(ROWS >= 16 && (PIECES & (PIECES - 1)) == 0 && PIECES >= 16, "a part of 16 rows at least");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    char *const part = smem + wave * PART;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int t0 = 0; t0 < T::TN * 16; t0 += ROWS) {
#pragma unroll
        for (int j = 0; j < ROWS / 16; j++) {
            if (t0 / 16 + j >= T::TN) break;
#pragma unroll
            for (int m = 0; m < T::TM; m++) *reinterpret_cast<f32x4 *>(part + (16 * j + i) * ROW + 16 * ((4 * m + g) ^ i)) = acc[m][t0 / 16 + j];
        }
        constexpr int LANES = T::TM * 16 / N;          // of a row
#pragma unroll 4
        for (int k = lane; k < ROWS * LANES; k += 64) {
            const int t = k / LANES, c = k % LANES;
            if (t0 + t >= T::TN * 16) break;
            float v[N];
#pragma unroll
            for (int q = 0; q < N / 4; q++) {
                const f32x4 x = *reinterpret_cast<const f32x4 *>(part + t * ROW + 16 * ((c * (N / 4) + q) ^ (t & 15)));
#pragma unroll
                for (int r = 0; r < 4; r++) v[4 * q + r] = x[r];
            }
            f(t0 + t, c * N, v);
        }
    }
}

// Workgroups are dealt to the eight XCDs in turn: the place of a workgroup among those of its XCD, so that an XCD works on neighbouring tiles whose operands its L2 shares
__device__ __forceinline__ int xcd_place(int id, int all)
{
    const int xcd = id & 7, q = all >> 3, r = all & 7;
    return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (id >> 3);
}

} // namespace ifa8
