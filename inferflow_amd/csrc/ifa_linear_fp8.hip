// ifa_linear_fp8.hip -- matrix products in 8-bit floating point with a scale for each block of 128:
//   C[t][n] (+)= sum_b sa[t][b] sw[n / 128][b] (sum_{k in block b} a[t][k] w[n][k]) + bias[n]
// The inner sums run on the matrix cores over exactly one block, their products with the two scales and the outer sum in 32-bit floats: the partial sum of a block
// never meets another block's before it has its scale.  16-bit outputs take the 8-bit instructions, 32-bit outputs exact halves (ifa_fp8.h).
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

template <int DT, int TILES, int WAVES, int DEPTH>
__global__ void __launch_bounds__(64 * WAVES) k_linear_fp8_stream(const uint8_t *__restrict__ w, const float *__restrict__ sw, int rows, int cols, const uint8_t *__restrict__ a, size_t lda,
                                                                        const float *__restrict__ sa, size_t lds, int tokens, const bf16_t *__restrict__ bias, int accumulate,
                                                                        typename Elem<DT>::type *__restrict__ c, size_t ldc)
{
    __shared__ f32x4 red[(WAVES - 1) * TILES * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n0 = blockIdx.x * 16, t0 = blockIdx.y * 16 * TILES;
    const uint8_t *wr[1] = {w + (size_t)min(n0 + (lane & 15), rows - 1) * cols};
    const float *swr[1] = {sw + (size_t)(n0 / BLOCK) * blocks_of(cols)};
    const uint8_t *ar[TILES];
    const float *sar[TILES];
    f32x4 acc[1][TILES];
#pragma unroll
    for (int j = 0; j < TILES; j++) {
        const size_t t = min(t0 + 16 * j + (lane & 15), tokens - 1);
        ar[j] = a + t * lda;
        sar[j] = sa + t * lds;
        acc[0][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    stream_blocks<DT == IFA_F32, DEPTH, 1, TILES>(wr, swr, ar, sar, cols, wave, WAVES, acc);
    join_waves<WAVES, 1, TILES>(acc, red);
    if (wave > 0) return;
#pragma unroll
    for (int j = 0; j < TILES; j++) {
        const int t = t0 + 16 * j + (lane & 15);
        if (t >= tokens) continue;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int n = n0 + 4 * (lane >> 4) + r;
            if (n < rows) store_out<DT>(c + (size_t)t * ldc + n, acc[0][j][r] + (bias ? ifa32::bf2f(bias[n]) : 0.0f), accumulate);
        }
    }
}

template <int DT, class T, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN, 2) k_linear_fp8_tile(const uint8_t *__restrict__ w, const float *__restrict__ sw, int rows, int cols, const uint8_t *__restrict__ a, size_t lda,
                                                                     const float *__restrict__ sa, size_t lds, int tokens, const bf16_t *__restrict__ bias, int accumulate,
                                                                     typename Elem<DT>::type *__restrict__ c, size_t ldc, int tiles_t, int tiles_n, int whole)
{
    constexpr int BM = T::TM * 16 * WM, BN = T::TN * 16 * WN, BAND = 8;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave % WM, wn = wave / WM;
    // bands of eight activation tiles, the tiles of a band fastest
    const int at = xcd_place(blockIdx.x, tiles_t * tiles_n), band = at / (BAND * tiles_n), within = at % (BAND * tiles_n), band_t = min(BAND, tiles_t - band * BAND);
    const int t0 = (band * BAND + within % band_t) * BN, n0 = within / band_t * BM;
    f32x4 acc[T::TM][T::TN];
#pragma unroll
    for (int j = 0; j < T::TN; j++)
#pragma unroll
        for (int m = 0; m < T::TM; m++) acc[m][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int nw = n0 + wm * (BM / WM), tw = t0 + wn * (BN / WN);          // the wave's first rows
    const float *swr = sw + (size_t)(min(nw, rows - 1) / BLOCK) * blocks_of(cols);
    tile_sums<DT == IFA_F32, true, T>(
        smem, cols, w + (size_t)n0 * cols, [&](int r) { return (uint32_t)min(r, rows - 1 - n0) * (uint32_t)cols; }, [&](int r) { return a + (size_t)min(t0 + r, tokens - 1) * lda; },
        [&](int m) { return wm * (BM / WM) + 16 * m; }, [&](int, int b) { return swr[b]; }, sa + (size_t)min(tw + lane, tokens - 1) * lds, wn * (BN / WN), acc);
    constexpr int N = VEC<DT>;
    tile_out<T, N>(smem, acc, [&](int t, int n, float *v) {
        t += tw; n += nw;
        if (t >= tokens || n >= rows) return;
        typename Elem<DT>::type *d = c + (size_t)t * ldc + n;
        if (whole) {
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
        } else {
#pragma unroll
            for (int e = 0; e < N; e++)
                if (n + e < rows) store_out<DT>(d + e, v[e] + (bias ? ifa32::bf2f(bias[n + e]) : 0.0f), accumulate);
        }
    });
}

struct Product {
    const uint8_t *w; const float *sw; size_t rows, cols; const uint8_t *a; size_t lda; const float *sa; size_t lds, tokens; const bf16_t *bias; int accumulate; void *c; size_t ldc;
};

template <int DT, int TILES, int WAVES, int DEPTH>
int launch_stream(const Product &P, hipStream_t s)
{
    hipLaunchKernelGGL((k_linear_fp8_stream<DT, TILES, WAVES, DEPTH>), dim3((unsigned)((P.rows + 15) / 16), (unsigned)((P.tokens + 16 * TILES - 1) / (16 * TILES))), dim3(64 * WAVES), 0, s, P.w, P.sw,
                       (int)P.rows, (int)P.cols, P.a, P.lda, P.sa, P.lds, (int)P.tokens, P.bias, P.accumulate, (typename Elem<DT>::type *)P.c, P.ldc);
    IFA_LAUNCH_CHECK();
    return IFA_OK;
}

template <int DT, int BM, int BN, int WM, int WN>
int launch_tile(const Product &P, hipStream_t s)
{
    typedef Tile<BM, BN, WM, WN> T;
    const auto fn = k_linear_fp8_tile<DT, T, WM, WN>;
    const size_t tt = (P.tokens + BN - 1) / BN, tn = (P.rows + BM - 1) / BM;
    if (P.cols > (1u << 22)) return launch_stream<DT, 4, 8, 1>(P, s);          // (a tile's offsets have 32 bits)
    IFA_REQUIRE(tt * tn < (1u << 31), "ifa_linear_fp8: too many tiles");
    const bool whole = P.rows % VEC<DT> == 0 && P.ldc % VEC<DT> == 0 && ((uintptr_t)P.c & 15) == 0;          // 16 bytes of output at a time
    if (T::SMEM > 64 * 1024) IFA_HIP_CHECK(hipFuncSetAttribute((const void *)fn, hipFuncAttributeMaxDynamicSharedMemorySize, T::SMEM));
    hipLaunchKernelGGL(fn, dim3((unsigned)(tt * tn)), dim3(64 * WM * WN), T::SMEM, s, P.w, P.sw, (int)P.rows, (int)P.cols, P.a, P.lda, P.sa, P.lds, (int)P.tokens, P.bias, P.accumulate,
                       (typename Elem<DT>::type *)P.c, P.ldc, (int)tt, (int)tn, (int)whole);
    IFA_LAUNCH_CHECK();
    return IFA_OK;
}

template <int DT>
int linear(const Product &P, hipStream_t s)
{
    if (P.tokens <= 16) return launch_stream<DT, 1, 8, 1>(P, s);
    if (P.tokens <= 32) return launch_stream<DT, 2, 8, 1>(P, s);
    if (P.tokens <= 64) return launch_stream<DT, 4, 8, 1>(P, s);
    if (DT != IFA_F32 && P.tokens > 256 && P.rows > 512) return launch_tile<DT, 256, 256, 2, 4>(P, s);
    return launch_tile<DT, 128, 128, 2, 2>(P, s);
}

} // namespace

extern "C" {

size_t ifa_linear_fp8_workspace_bytes(size_t rows, size_t cols, size_t tokens) { return 0; }

int ifa_linear_fp8(const void *w_e4m3, const void *w_scale_f32, size_t rows, size_t cols, const void *a_e4m3, size_t lda, const void *a_scale_f32, size_t lds, size_t tokens,
                   const void *bias_bf16, int accumulate, int c_dtype, void *c, size_t ldc, void *ws, size_t ws_bytes, ifa_stream stream)
{
    IFA_REQUIRE(w_e4m3 && w_scale_f32 && a_e4m3 && a_scale_f32 && c, "ifa_linear_fp8: null pointer");
    if (!elem_known(c_dtype)) return ifa_fail(IFA_ERR_DTYPE, "ifa_linear_fp8: output dtype %d (F32, F16 or BF16)", c_dtype);
    IFA_REQUIRE(rows > 0 && cols > 0 && tokens > 0 && cols % 16 == 0 && rows < (1u << 30) && cols < (1u << 30) && tokens <= 1000000, "ifa_linear_fp8: %zu x %zu over %zu rows (columns in whole 16s)", rows,
                cols, tokens);
    IFA_REQUIRE(lda >= cols && lda % 16 == 0 && lds >= blocks_of(cols) && ldc >= rows, "ifa_linear_fp8: row strides");
    IFA_REQUIRE((((uintptr_t)w_e4m3 | (uintptr_t)a_e4m3 | (uintptr_t)ws) & 15) == 0 && (((uintptr_t)w_scale_f32 | (uintptr_t)a_scale_f32) & 3) == 0 && ((uintptr_t)bias_bf16 & 1) == 0
                    && (uintptr_t)c % elem_bytes(c_dtype) == 0, "ifa_linear_fp8: misaligned pointer");
    const Product P = {(const uint8_t *)w_e4m3, (const float *)w_scale_f32, rows, cols, (const uint8_t *)a_e4m3, lda, (const float *)a_scale_f32, lds, tokens, (const bf16_t *)bias_bf16, accumulate, c,
                       ldc};
    return c_dtype == IFA_F32 ? linear<IFA_F32>(P, ifa_s(stream)) : c_dtype == IFA_F16 ? linear<IFA_F16>(P, ifa_s(stream)) : linear<IFA_BF16>(P, ifa_s(stream));
}

} // extern "C"
