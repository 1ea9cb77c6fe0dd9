// ifa_linear_fp8.hip -- matrix products in 8-bit floating point with a scale for each block of 128:
//   C[t][n] (+)= sum_b sa[t][b] sw[n / 128][b] (sum_{k in block b} a[t][k] w[n][k]) + bias[n]
// The inner sums run on the matrix cores over exactly one block, their products with the two scales and the outer sum in 32-bit floats: the partial sum of a block
// never meets another block's before it has its scale.  16-bit outputs take the 8-bit instructions, 32-bit outputs exact halves (ifa_fp8.h).
#include <algorithm>
#include "ifa_host.h"
#include "ifa_fp8_stream.h"
#include "ifa_fp8_tile.h"

using namespace ifa8;

namespace {

template <int DT> __device__ __forceinline__ void store_out(typename Elem<DT>::type *c, float v, int accumulate)
{
    if (accumulate) v += (float)*c;
    *c = (typename Elem<DT>::type)v;
}

template <int DT, int MATS, int TILES, int WAVES, int DEPTH>
__global__ void __launch_bounds__(64 * WAVES) k_linear_fp8_stream(const uint8_t *__restrict__ w, const float *__restrict__ sw, int rows, int cols, const uint8_t *__restrict__ a, size_t lda,
                                                                        const float *__restrict__ sa, size_t lds, int tokens, const bf16_t *__restrict__ bias, int accumulate,
                                                                        typename Elem<DT>::type *__restrict__ c, size_t ldc)
{
    __shared__ f32x4 red[(WAVES - 1) * MATS * TILES * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n0 = blockIdx.x * 16 * MATS, t0 = blockIdx.y * 16 * TILES;
    const uint8_t *wr[MATS], *ar[TILES];
    const float *swr[MATS], *sar[TILES];
    f32x4 acc[MATS][TILES];
#pragma unroll
    for (int i = 0; i < MATS; i++) {
        wr[i] = w + (size_t)min(n0 + 16 * i + (lane & 15), rows - 1) * cols;
        swr[i] = sw + (size_t)(min(n0 + 16 * i, rows - 1) / BLOCK) * blocks_of(cols);
#pragma unroll
        for (int j = 0; j < TILES; j++) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
#pragma unroll
    for (int j = 0; j < TILES; j++) {
        const size_t t = min(t0 + 16 * j + (lane & 15), tokens - 1);
        ar[j] = a + t * lda;
        sar[j] = sa + t * lds;
    }
    stream_blocks<DT == IFA_F32, DEPTH, MATS, TILES>(wr, swr, ar, sar, cols, wave, WAVES, acc);
    join_waves<WAVES, MATS, TILES>(acc, red);
    if (wave > 0) return;
#pragma unroll
    for (int j = 0; j < TILES; j++) {
        const int t = t0 + 16 * j + (lane & 15);
        if (t >= tokens) continue;
#pragma unroll
        for (int i = 0; i < MATS; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int n = n0 + 16 * i + 4 * (lane >> 4) + r;
                if (n < rows) store_out<DT>(c + (size_t)t * ldc + n, acc[i][j][r] + (bias ? ifa32::bf2f(bias[n]) : 0.0f), accumulate);
            }
    }
}

struct LinearJob {
    const uint8_t *wbase, *abase;
    const float *swr, *sa;
    int cols, row_cols, last_row, last_token, nw, tw, part;          // (nw, tw: the wave's first rows)
    uint32_t lda;
    bool idle;
    __device__ __forceinline__ uint32_t woff(int r) const { return (uint32_t)min(r, last_row) * (uint32_t)row_cols; }
    __device__ __forceinline__ uint32_t asrc(int r) const { return (uint32_t)min(r, last_token) * lda; }
    __device__ __forceinline__ const float *sw(int) const { return swr; }
};

template <int DT, class T, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN, 2) k_linear_fp8_tile(const uint8_t *__restrict__ w, const float *__restrict__ sw, int rows, int cols, const uint8_t *__restrict__ a, size_t lda,
                                                                     const float *__restrict__ sa, size_t lds, int tokens, const bf16_t *__restrict__ bias, int accumulate,
                                                                     typename Elem<DT>::type *__restrict__ c, size_t ldc, int tiles_t, int tiles_n, int whole, int parts,
                                                                     float *__restrict__ planes)
{
    constexpr int BM = T::TM * 16 * WM, BN = T::TN * 16 * WN, BAND = 8;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave % WM, wn = wave / WM;
    // bands of eight activation tiles, the tiles of a band fastest; the parts of the columns one behind the other
    const int tiles = tiles_t * tiles_n, nb = (cols + BLOCK - 1) / BLOCK;
    const Share share(tiles * parts);
    auto job = [&](int k) {
        LinearJob J;
        const int place = share.at(k), part = place / tiles, at = place - part * tiles, band = at / (BAND * tiles_n), within = at % (BAND * tiles_n), band_t = min(BAND, tiles_t - band * BAND);
        const int t0 = (band * BAND + within % band_t) * BN, n0 = within / band_t * BM;
        const int b0 = (int)((long long)part * nb / parts), b1 = (int)((long long)(part + 1) * nb / parts);
        J.part = part; J.nw = n0 + wm * (BM / WM); J.tw = t0 + wn * (BN / WN);
        J.cols = min(cols, b1 * BLOCK) - b0 * BLOCK; J.row_cols = cols; J.last_row = rows - 1 - n0; J.last_token = tokens - 1 - t0; J.lda = (uint32_t)lda;
        J.wbase = w + (size_t)n0 * cols + (size_t)b0 * BLOCK; J.abase = a + (size_t)t0 * lda + (size_t)b0 * BLOCK;
        J.swr = sw + (size_t)(min(J.nw, rows - 1) / BLOCK) * blocks_of(cols) + b0;
        J.sa = sa + (size_t)min(J.tw + lane % (16 * T::TN), tokens - 1) * lds + b0;
        J.idle = J.tw >= tokens || J.nw >= rows;
        return J;
    };
    tile_run<false, DT == IFA_F32, 1, true, T, WM>(smem, 1, job, [&](const LinearJob &J, const f32x4 (&acc)[T::TM][T::TN], char *buffer) {
        const int tw = J.tw, nw = J.nw, part = J.part;
        if (parts > 1) {
            float *const plane = planes + (size_t)part * tokens * rows;
            tile_out<T, false, 4>(buffer, acc, [&](int t, int n, float *v) {
                t += tw; n += nw;
                if (t >= tokens || n >= rows) return;
                float *d = plane + (size_t)t * rows + n;
                if (rows % 4 == 0) *reinterpret_cast<u32x4 *>(d) = pack<IFA_F32>(v);
                else for (int e = 0; e < 4; e++) if (n + e < rows) d[e] = v[e];
            });
            return;
        }
        constexpr int N = VEC<DT>;
        if (whole) tile_out<T, false, N>(buffer, acc, [&](int t, int n, float *v) {
            t += tw; n += nw;
            if (t >= tokens || n >= rows) return;
            typename Elem<DT>::type *d = c + (size_t)t * ldc + n;
            if (bias) {
#pragma unroll
                for (int e = 0; e < N; e++) v[e] += ifa32::bf2f(bias[n + e]);
            }
            if (accumulate) {
                float old[N];
                unpack<DT>(*reinterpret_cast<const u32x4 *>(d), old);
#pragma unroll
                for (int e = 0; e < N; e++) v[e] += old[e];
            }
            *reinterpret_cast<u32x4 *>(d) = pack<DT>(v);
        });
        else tile_out<T, false, 1>(buffer, acc, [&](int t, int n, float *v) {          // (rows that do not start on 16 bytes: a lane a value, so that a store is of neighbours all the same)
            t += tw; n += nw;
            if (t < tokens && n < rows) store_out<DT>(c + (size_t)t * ldc + n, v[0] + (bias ? ifa32::bf2f(bias[n]) : 0.0f), accumulate);
        });
    });
}

// the parts' sums one after the other, then what a tile's output is
template <int DT>
__global__ void __launch_bounds__(256) k_linear_fp8_join(const float *__restrict__ planes, int parts, size_t all, int rows, const bf16_t *__restrict__ bias, int accumulate,
                                                         typename Elem<DT>::type *__restrict__ c, size_t ldc)
{
    const size_t id = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (id >= all) return;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (rows % 4 == 0) {
#pragma unroll 4
        for (int k = 0; k < parts; k++) {
            float o[4];
            unpack<IFA_F32>(*reinterpret_cast<const u32x4 *>(planes + (size_t)k * all + id), o);
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] += o[e];
        }
    } else {
        for (int k = 0; k < parts; k++)
            for (int e = 0; e < 4; e++) if (id + e < all) v[e] += planes[(size_t)k * all + id + e];
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (id + e >= all) break;
        const size_t t = (id + e) / rows;
        const int n = (int)(id + e - t * rows);
        store_out<DT>(c + t * ldc + n, v[e] + (bias ? ifa32::bf2f(bias[n]) : 0.0f), accumulate);
    }
}

struct Product {
    const uint8_t *w; const float *sw; size_t rows, cols; const uint8_t *a; size_t lda; const float *sa; size_t lds, tokens; const bf16_t *bias; int accumulate; void *c; size_t ldc;
    float *ws; size_t ws_bytes;
};

template <int DT, int MATS, int TILES, int WAVES, int DEPTH>
int launch_stream(const Product &P, hipStream_t s)
{
    hipLaunchKernelGGL((k_linear_fp8_stream<DT, MATS, TILES, WAVES, DEPTH>), dim3((unsigned)((P.rows + 16 * MATS - 1) / (16 * MATS)), (unsigned)((P.tokens + 16 * TILES - 1) / (16 * TILES))), dim3(64 * WAVES), 0, s, P.w, P.sw,
                       (int)P.rows, (int)P.cols, P.a, P.lda, P.sa, P.lds, (int)P.tokens, P.bias, P.accumulate, (typename Elem<DT>::type *)P.c, P.ldc);
    IFA_LAUNCH_CHECK();
    return IFA_OK;
}

template <int DT, int BM, int BN, int WM, int WN>
int launch_tile(const Product &P, int parts, hipStream_t s)
{
    typedef Tile<BM, BN, WM, WN> T;
    const auto fn = k_linear_fp8_tile<DT, T, WM, WN>;
    const size_t tt = (P.tokens + BN - 1) / BN, tn = (P.rows + BM - 1) / BM;
    IFA_REQUIRE(tt * tn * parts < (1u << 31), "ifa_linear_fp8: too many tiles");
    IFA_REQUIRE(parts == 1 || ((size_t)parts <= blocks_of(P.cols) && P.ws && parts * P.tokens * P.rows * 4 <= P.ws_bytes), "ifa_linear_fp8: %d parts in a workspace of %zu bytes", parts, P.ws_bytes);
    const bool whole = P.rows % VEC<DT> == 0 && P.ldc % VEC<DT> == 0 && ((uintptr_t)P.c & 15) == 0;          // 16 bytes of output at a time
    if (T::SMEM > 64 * 1024) IFA_HIP_CHECK(hipFuncSetAttribute((const void *)fn, hipFuncAttributeMaxDynamicSharedMemorySize, T::SMEM));
    hipLaunchKernelGGL(fn, dim3((unsigned)(tt * tn * parts)), dim3(64 * WM * WN), T::SMEM, s, P.w, P.sw, (int)P.rows, (int)P.cols, P.a, P.lda, P.sa, P.lds, (int)P.tokens, P.bias, P.accumulate,
                       (typename Elem<DT>::type *)P.c, P.ldc, (int)tt, (int)tn, (int)whole, parts, P.ws);
    if (parts > 1)
        hipLaunchKernelGGL((k_linear_fp8_join<DT>), dim3(ifa_cdiv((P.tokens * P.rows + 3) / 4, 256)), dim3(256), 0, s, P.ws, parts, P.tokens * P.rows, (int)P.rows, P.bias, P.accumulate,
                           (typename Elem<DT>::type *)P.c, P.ldc);
    IFA_LAUNCH_CHECK();
    return IFA_OK;
}

// ---- which kernel.  Up to 16 rows: the stream.  From there on what takes least by these figures (us, measured with weights from memory): a stream of 32 rows a workgroup 2.3 and 8.6e-4 for each
// workgroup and block of columns, or 0.14 for each block; tiles a step (a block) and beside the steps, with one, two or three workgroups on a compute unit; parts of the columns the join and the
// planes' way to memory and back.  Against the fastest of 16 choices at 28 sizes from 19 to 2385 rows, 258 to 11008 matrix rows, 656 to 11840 columns, 16- and 32-bit outputs: 4.5 % behind on average, 30 %
// at worst (19 rows, 258 x 11840, where the stream is taken for slower than it is).
// 256 x 256 tiles of 32-bit outputs do not fit the registers.
struct TileCost { int bm, bn, per_cu; double step[3], beside; };
enum { T_256x256, T_256x128, T_128x128, T_128x64, T_128x32, N_TILES };
constexpr TileCost TILE_COST[2][N_TILES] = {{{256, 256, 1, {1.78}, 9.0}, {256, 128, 1, {1.05}, 7.0}, {128, 128, 2, {0.80, 1.19}, 5.5}, {128, 64, 3, {0.55, 0.75, 1.35}, 5.5}, {128, 32, 3, {0.58, 0.83, 1.1}, 3.7}},
                                            {{256, 256, 0, {}, 0.0}, {256, 128, 1, {1.5}, 7.0}, {128, 128, 2, {1.0, 1.8}, 5.5}, {128, 64, 3, {0.65, 1.0, 1.75}, 5.5}, {128, 32, 3, {0.6, 0.9, 1.25}, 3.7}}};
struct Plan { int form, parts; double us; };          // form: a tile, or -1: the stream

Plan choose(bool wide, size_t rows, size_t cols, size_t lda, size_t tokens, size_t ws_bytes)
{
    if (tokens <= 16 || cols > (1u << 22) || lda > (1u << 22)) return {-1, 1, 0.0};          // (a tile's offsets have 32 bits)
    const double out = (double)tokens * rows;
    const size_t nb = blocks_of(cols);
    Plan best = {-1, 1, 2.3 + std::max(8.6e-4 * ((rows + 15) / 16) * ((tokens + 31) / 32) * nb, 0.14 * nb)};
    for (int k = 0; k < N_TILES; k++) {
        const TileCost &C = TILE_COST[wide][k];
        if (C.per_cu == 0) continue;
        const size_t tiles = ((rows + C.bm - 1) / C.bm) * ((tokens + C.bn - 1) / C.bn), slots = 256 * C.per_cu;
        for (int parts = 1; parts <= 16 && (parts == 1 || (nb >= 2 * (size_t)parts && parts * out * 4 <= (double)ws_bytes)); parts++) {
            const size_t n = tiles * parts, rounds = n / slots, rest = n % slots;
            const double steps = (double)((nb + parts - 1) / parts);
            double us = rounds * (steps * C.step[C.per_cu - 1] + C.beside) + (rest ? steps * C.step[(rest + 255) / 256 - 1] + C.beside : 0.0);
            if (parts > 1) us += 2.5 + parts * out * 2e-6;
            if (us < best.us) best = {k, parts, us};
        }
    }
    return best;
}

bool sizes_known(size_t rows, size_t cols, size_t tokens) { return rows > 0 && cols > 0 && tokens > 0 && cols % 16 == 0 && rows < (1u << 26) && cols < (1u << 30) && tokens <= 1000000; }

template <int DT>
int linear(const Product &P, hipStream_t s)
{
    const Plan plan = choose(DT == IFA_F32, P.rows, P.cols, P.lda, P.tokens, P.ws ? P.ws_bytes : 0);
    switch (plan.form) {
    case T_256x256: if constexpr (DT != IFA_F32) return launch_tile<DT, 256, 256, 2, 4>(P, plan.parts, s); [[fallthrough]];
    case T_256x128: return launch_tile<DT, 256, 128, 2, 4>(P, plan.parts, s);
    case T_128x128: return launch_tile<DT, 128, 128, 2, 2>(P, plan.parts, s);
    case T_128x64: return launch_tile<DT, 128, 64, 2, 2>(P, plan.parts, s);
    case T_128x32: return launch_tile<DT, 128, 32, 2, 2>(P, plan.parts, s);
    }
    // sixteen waves where there is a workgroup for each compute unit at most: one row, 4096 x 4096 6.4 -> 5.5 us, 4096 x 11008 13.1 -> 12.7; 11008 x 4096 12.2 -> 13.2
    if (P.tokens <= 16) return P.rows <= 4096 && P.cols >= 16 * BLOCK ? launch_stream<DT, 1, 1, 16, 1>(P, s) : launch_stream<DT, 1, 1, 8, 1>(P, s);
    return launch_stream<DT, 1, 2, 8, 1>(P, s);
}

} // namespace

extern "C" {

size_t ifa_linear_fp8_workspace_bytes(size_t rows, size_t cols, size_t tokens) 
{
    if (!sizes_known(rows, cols, tokens)) return 0;
    size_t most = 0;
    for (int wide = 0; wide < 2; wide++) {
        const Plan plan = choose(wide, rows, cols, cols, tokens, (size_t)256 << 20);
        if (plan.parts > 1) most = std::max(most, (size_t)plan.parts * tokens * rows * 4);
    }
    return most;
}

int ifa_linear_fp8_plan(size_t rows, size_t cols, size_t lda, size_t tokens, int c_dtype, size_t ws_bytes, int *tile_rows, int *tile_tokens, int *parts)
{
    IFA_REQUIRE(tile_rows && tile_tokens && parts, "ifa_linear_fp8_plan: null pointer");
    if (!elem_known(c_dtype)) return ifa_fail(IFA_ERR_DTYPE, "ifa_linear_fp8_plan: output dtype %d (F32, F16 or BF16)", c_dtype);
    IFA_REQUIRE(sizes_known(rows, cols, tokens) && lda >= cols && lda % 16 == 0, "ifa_linear_fp8_plan: %zu x %zu over %zu rows (columns in whole 16s)", rows, cols, tokens);
    const Plan plan = choose(c_dtype == IFA_F32, rows, cols, lda, tokens, ws_bytes);
    *tile_rows = plan.form < 0 ? 0 : TILE_COST[0][plan.form].bm;
    *tile_tokens = plan.form < 0 ? 0 : TILE_COST[0][plan.form].bn;
    *parts = plan.parts;
    return IFA_OK;
}

int ifa_linear_fp8(const void *w_e4m3, const void *w_scale_f32, size_t rows, size_t cols, const void *a_e4m3, size_t lda, const void *a_scale_f32, size_t lds, size_t tokens,
                   const void *bias_bf16, int accumulate, int c_dtype, void *c, size_t ldc, void *ws, size_t ws_bytes, ifa_stream stream)
{
    IFA_REQUIRE(w_e4m3 && w_scale_f32 && a_e4m3 && a_scale_f32 && c, "ifa_linear_fp8: null pointer");
    if (!elem_known(c_dtype)) return ifa_fail(IFA_ERR_DTYPE, "ifa_linear_fp8: output dtype %d (F32, F16 or BF16)", c_dtype);
    IFA_REQUIRE(sizes_known(rows, cols, tokens), "ifa_linear_fp8: %zu x %zu over %zu rows (columns in whole 16s)", rows,
                cols, tokens);
    IFA_REQUIRE(lda >= cols && lda % 16 == 0 && lds >= blocks_of(cols) && ldc >= rows, "ifa_linear_fp8: row strides");
    IFA_REQUIRE((((uintptr_t)w_e4m3 | (uintptr_t)a_e4m3 | (uintptr_t)ws) & 15) == 0 && (((uintptr_t)w_scale_f32 | (uintptr_t)a_scale_f32) & 3) == 0 && ((uintptr_t)bias_bf16 & 1) == 0
                    && (uintptr_t)c % elem_bytes(c_dtype) == 0, "ifa_linear_fp8: misaligned pointer");
    const Product P = {(const uint8_t *)w_e4m3, (const float *)w_scale_f32, rows, cols, (const uint8_t *)a_e4m3, lda, (const float *)a_scale_f32, lds, tokens, (const bf16_t *)bias_bf16, accumulate, c,
                       ldc, (float *)ws, ws_bytes};
    return c_dtype == IFA_F32 ? linear<IFA_F32>(P, ifa_s(stream)) : c_dtype == IFA_F16 ? linear<IFA_F16>(P, ifa_s(stream)) : linear<IFA_BF16>(P, ifa_s(stream));
}

} // extern "C"
