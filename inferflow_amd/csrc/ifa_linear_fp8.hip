// ifa_linear_fp8.hip -- matrix products in 8-bit floating point with a scale for each block of 128:
//   C[t][n] (+)= sum_b sa[t][b] sw[n / 128][b] (sum_{k in block b} a[t][k] w[n][k]) + bias[n]
// The inner sums run on the matrix cores over exactly one block, their products with the two scales and the outer sum in 32-bit floats: the partial sum of a block
// never meets another block's before it has its scale.  16-bit outputs take the 8-bit instructions, 32-bit outputs exact halves (ifa_fp8.h).
#include "ifa_host.h"
#include "ifa_fp8_stream.h"

using namespace ifa8;

namespace {

template <int DT> __device__ __forceinline__ void store_out(typename Elem<DT>::type *c, float v, int accumulate)
{
    if (accumulate) v += (float)*c;
    *c = (typename Elem<DT>::type)v;
}

template <int DT, int TILES>
__global__ void __launch_bounds__(64 * STREAM_WAVES) k_linear_fp8_stream(const uint8_t *__restrict__ w, const float *__restrict__ sw, int rows, int cols, const uint8_t *__restrict__ a, size_t lda,
                                                                        const float *__restrict__ sa, size_t lds, int tokens, const bf16_t *__restrict__ bias, int accumulate,
                                                                        typename Elem<DT>::type *__restrict__ c, size_t ldc)
{
    __shared__ f32x4 red[(STREAM_WAVES - 1) * TILES * 64];
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
    stream_blocks<DT == IFA_F32, 1, TILES>(wr, swr, ar, sar, cols, wave, STREAM_WAVES, acc);
    join_waves<1, TILES>(acc, red);
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

template <int DT>
int linear(const void *w, const void *sw, size_t rows, size_t cols, const void *a, size_t lda, const void *sa, size_t lds, size_t tokens, const void *bias, int accumulate, void *c, size_t ldc,
           void *ws, size_t ws_bytes, hipStream_t s)
{
    typedef typename Elem<DT>::type T;
#define IFA_STREAM(TILES)                                                                                                                                                  \
    hipLaunchKernelGGL((k_linear_fp8_stream<DT, TILES>), dim3((unsigned)((rows + 15) / 16), (unsigned)((tokens + 16 * TILES - 1) / (16 * TILES))), dim3(64 * STREAM_WAVES), 0, s, \
                       (const uint8_t *)w, (const float *)sw, (int)rows, (int)cols, (const uint8_t *)a, lda, (const float *)sa, lds, (int)tokens, (const bf16_t *)bias, accumulate,  \
                       (T *)c, ldc)
    if (tokens <= 16) IFA_STREAM(1);
    else if (tokens <= 32) IFA_STREAM(2);
    else IFA_STREAM(4);
#undef IFA_STREAM
    IFA_LAUNCH_CHECK();
    return IFA_OK;
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
    auto f = c_dtype == IFA_F32 ? linear<IFA_F32> : c_dtype == IFA_F16 ? linear<IFA_F16> : linear<IFA_BF16>;
    return f(w_e4m3, w_scale_f32, rows, cols, a_e4m3, lda, a_scale_f32, lds, tokens, bias_bf16, accumulate, c, ldc, ws, ws_bytes, ifa_s(stream));
}

} // extern "C"
