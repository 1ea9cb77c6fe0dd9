// ifa_fp8_rows.hip -- what leaves rows in 8-bit floating point: the norm in front of a sub-layer (with the residual's addition) and the gated activation.
//   row t, block b of 128 columns:  s = max(max |v| / 448, 2^-126),  q = e4m3(v / s)
//   norm:        x <- x + m (rounded to x's type),  v = x / sqrt(mean(x^2) + eps) * (w_offset + w)
//   activation:  v = act(gate) * up
// Both are bound by memory: a thread keeps its pieces of 16 bytes in registers, so that every value comes once and leaves once; a block of 128 columns
// is 32 (32-bit) or 16 (16-bit values) neighbouring lanes, whose maximum takes four or five steps between lanes.
// Measured: norm with the residual, 4096 x 4096 in 32 bits 44.5 us, 4.9 TB/s (a large copy: 4.9), 2048 x 8192 bf16 33.3 us, 3.5 TB/s (its weights come two bytes at a time behind the row's sum); activation, 2051 x 11008 bf16 22.7 us, 5.0 TB/s; few rows 2.5 us, a launch's start and end.
#include "ifa_host.h"
#include "ifa_fp8.h"

using namespace ifa8;

namespace {

template <int DT, int PIECES>
__global__ void __launch_bounds__(1024) k_norm_add_fp8(typename Elem<DT>::type *__restrict__ x, size_t ldx, int cols, const typename Elem<DT>::type *__restrict__ m, size_t ldm,
                                                       const bf16_t *__restrict__ w, float w_offset, float eps, typename Elem<DT>::type *__restrict__ h, size_t ldh,
                                                       uint8_t *__restrict__ q, size_t ldq, float *__restrict__ scale, size_t lds)
{
    constexpr int N = VEC<DT>;
    __shared__ float red[17];
    const size_t t = blockIdx.x;
    float v[PIECES][N];
    float sum = 0.0f;
#pragma unroll
    for (int p = 0; p < PIECES; p++) {
        const int c = N * (threadIdx.x + p * blockDim.x);
        u32x4 a = {0u, 0u, 0u, 0u}, b = a;
        if (c < cols) {
            a = *reinterpret_cast<const u32x4 *>(x + t * ldx + c);
            if (m) b = *reinterpret_cast<const u32x4 *>(m + t * ldm + c);
        }
        unpack<DT>(a, v[p]);
        if (m) {
            float add[N];
            unpack<DT>(b, add);
#pragma unroll
            for (int e = 0; e < N; e++) v[p][e] += add[e];
            const u32x4 r = pack<DT>(v[p]);
            if (c < cols) *reinterpret_cast<u32x4 *>(x + t * ldx + c) = r;
        }
#pragma unroll
        for (int e = 0; e < N; e++) sum = fmaf(v[p][e], v[p][e], sum);
    }
    const float rinv = 1.0f / sqrtf(ifa32::block_sum(sum, red) / (float)cols + eps);
#pragma unroll
    for (int p = 0; p < PIECES; p++) {
        const int c = N * (threadIdx.x + p * blockDim.x);
        uint32_t most = 0u;
        if (c < cols) {
#pragma unroll
            for (int e = 0; e < N; e++) { v[p][e] = v[p][e] * rinv * (w_offset + (w ? ifa32::bf2f(w[c + e]) : 0.0f)); most = dpp_max(most, abs_bits(v[p][e])); }
        }
        most = group_max<BLOCK / N>(most);
        if (c < cols) {
            const float s = scale_of(most), inv = 1.0f / s;
            uint32_t *dst = reinterpret_cast<uint32_t *>(q + t * ldq + c);
            dst[0] = quantise4(v[p], inv);
            if constexpr (N == 8) dst[1] = quantise4(v[p] + 4, inv);
            if (c % BLOCK == 0) scale[t * lds + c / BLOCK] = s;
            if (h) *reinterpret_cast<u32x4 *>(h + t * ldh + c) = pack<DT>(v[p]);
        }
    }
}

// a thread a piece; pieces of a row padded to whole blocks so that a block's lanes stay together
template <int DT, int KIND>
__global__ void __launch_bounds__(256) k_glu_fp8(float limit, const typename Elem<DT>::type *__restrict__ gu, size_t ld, int cols, int pieces, size_t all,
                                                 uint8_t *__restrict__ q, size_t ldq, float *__restrict__ scale, size_t lds)
{
    constexpr int N = VEC<DT>;
    const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x;
    const size_t t = id / pieces;
    const int c = (int)(id % pieces) * N;
    const bool live = id < all && c < cols;
    float v[N];
    uint32_t most = 0u;
    if (live) {
        unpack<DT>(*reinterpret_cast<const u32x4 *>(gu + t * ld + c), v);
        if constexpr (KIND != 4) {
            float u[N];
            unpack<DT>(*reinterpret_cast<const u32x4 *>(gu + t * ld + cols + c), u);
#pragma unroll
            for (int e = 0; e < N; e++) v[e] = gated<KIND>(limit, v[e], u[e]);
        }
#pragma unroll
        for (int e = 0; e < N; e++) most = dpp_max(most, abs_bits(v[e]));
    }
    most = group_max<BLOCK / N>(most);
    if (live) {
        const float s = scale_of(most), inv = 1.0f / s;
        uint32_t *dst = reinterpret_cast<uint32_t *>(q + t * ldq + c);
        dst[0] = quantise4(v, inv);
        if constexpr (N == 8) dst[1] = quantise4(v + 4, inv);
        if (c % BLOCK == 0) scale[t * lds + c / BLOCK] = s;
    }
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

template <int DT>
int norm_add(void *x, size_t ldx, size_t rows, size_t cols, const void *m, size_t ldm, const void *w, float w_offset, float eps, void *h, size_t ldh, void *q, size_t ldq, void *scale,
             size_t lds, hipStream_t s)
{
    typedef typename Elem<DT>::type T;
    const size_t pieces = cols / VEC<DT>;
#define IFA_NORM(P)                                                                                                                                                        \
    hipLaunchKernelGGL((k_norm_add_fp8<DT, P>), dim3((unsigned)rows), dim3((unsigned)((pieces + 64 * P - 1) / (64 * P) * 64)), 0, s, (T *)x, ldx, (int)cols, (const T *)m, ldm, \
                       (const bf16_t *)w, w_offset, eps, (T *)h, ldh, (uint8_t *)q, ldq, (float *)scale, lds)
    // threads of a row: few rows want all their requests at once, many rows several workgroups on a compute unit.  us 1024 / 512 at most, rows of 4096 32-bit columns: 4096 48.4 / 45.3, 1024 13.2 / 12.0,
    // 512 7.7 / 7.6, 256 5.4 / 5.5, 1 3.3 / 3.6; 2048 rows of 8192 bf16 35.9 / 34.7, 64 5.1 / 5.2
    const size_t most = rows > 512 ? 512 : 1024;
    if (pieces <= most) IFA_NORM(1);
    else if (pieces <= 2 * most) IFA_NORM(2);
    else if (pieces <= 4 * most) IFA_NORM(4);
    else IFA_NORM(8);
#undef IFA_NORM
    IFA_LAUNCH_CHECK();
    return IFA_OK;
}

template <int DT>
int glu(int kind, float limit, const void *gu, size_t ld, size_t rows, size_t cols, void *q, size_t ldq, void *scale, size_t lds, hipStream_t s)
{
    typedef typename Elem<DT>::type T;
    const size_t pieces = blocks_of(cols) * (BLOCK / VEC<DT>), all = rows * pieces;
    const auto fn = kind == 0 ? k_glu_fp8<DT, 0> : kind == 1 ? k_glu_fp8<DT, 1> : kind == 2 ? k_glu_fp8<DT, 2> : kind == 3 ? k_glu_fp8<DT, 3> : k_glu_fp8<DT, 4>;
    hipLaunchKernelGGL(fn, dim3((unsigned)((all + 255) / 256)), dim3(256), 0, s, limit, (const T *)gu, ld, (int)cols, (int)pieces, all, (uint8_t *)q, ldq,
                       (float *)scale, lds);
    IFA_LAUNCH_CHECK();
    return IFA_OK;
}

} // namespace

extern "C" {

int ifa_norm_add_fp8(int dtype, void *x, size_t ldx, size_t rows, size_t cols, const void *m, size_t ldm, const void *w_bf16, float w_offset, float eps, void *h, size_t ldh,
                     void *q_e4m3, size_t ldq, void *scale_f32, size_t lds, ifa_stream stream)
{
    IFA_REQUIRE(x && q_e4m3 && scale_f32, "ifa_norm_add_fp8: null pointer");
    if (!elem_known(dtype)) return ifa_fail(IFA_ERR_DTYPE, "ifa_norm_add_fp8: dtype %d (F32, F16 or BF16)", dtype);
    const size_t n = 16 / elem_bytes(dtype);
    IFA_REQUIRE(rows > 0 && rows < (1u << 22) && cols > 0 && cols % 16 == 0 && cols <= 32768, "ifa_norm_add_fp8: %zu rows (fewer than 2^22) of %zu columns (whole 16s up to 32768)", rows, cols);
    IFA_REQUIRE(ldx >= cols && ldx % n == 0 && (!m || (ldm >= cols && ldm % n == 0)) && (!h || (ldh >= cols && ldh % n == 0)) && ldq >= cols && ldq % 16 == 0 && lds >= blocks_of(cols),
                "ifa_norm_add_fp8: row strides (rows of whole 16 bytes)");
    IFA_REQUIRE(aligned16(x) && aligned16(m) && aligned16(h) && aligned16(q_e4m3) && ((uintptr_t)w_bf16 & 1) == 0 && ((uintptr_t)scale_f32 & 3) == 0, "ifa_norm_add_fp8: misaligned pointer");
    IFA_REQUIRE(h != x && (!m || m != x), "ifa_norm_add_fp8: x is a buffer of its own");
    auto f = dtype == IFA_F32 ? norm_add<IFA_F32> : dtype == IFA_F16 ? norm_add<IFA_F16> : norm_add<IFA_BF16>;
    return f(x, ldx, rows, cols, m, ldm, w_bf16, w_offset, eps, h, ldh, q_e4m3, ldq, scale_f32, lds, ifa_s(stream));
}

int ifa_glu_fp8(int kind, float limit, int dtype, const void *gate_up, size_t ld, size_t rows, size_t cols, void *q_e4m3, size_t ldq, void *scale_f32, size_t lds, ifa_stream stream)
{
    IFA_REQUIRE(gate_up && q_e4m3 && scale_f32, "ifa_glu_fp8: null pointer");
    if (!elem_known(dtype)) return ifa_fail(IFA_ERR_DTYPE, "ifa_glu_fp8: dtype %d (F32, F16 or BF16)", dtype);
    const size_t n = 16 / elem_bytes(dtype);
    IFA_REQUIRE(kind >= 0 && kind <= 4, "ifa_glu_fp8: kind %d", kind);
    IFA_REQUIRE(rows > 0 && cols > 0 && cols % 16 == 0 && cols < (1u << 30) && rows < (1u << 31) && rows * (blocks_of(cols) * BLOCK / n) < 0xFFFFFF00u, "ifa_glu_fp8: %zu rows of %zu columns (whole 16s, fewer than 2^32 pieces of 16 bytes)", rows, cols);
    IFA_REQUIRE(ld >= cols * (kind == 4 ? 1 : 2) && ld % n == 0 && ldq >= cols && ldq % 16 == 0 && lds >= blocks_of(cols), "ifa_glu_fp8: row strides (rows of whole 16 bytes)");
    IFA_REQUIRE(aligned16(gate_up) && aligned16(q_e4m3) && ((uintptr_t)scale_f32 & 3) == 0, "ifa_glu_fp8: misaligned pointer");
    auto f = dtype == IFA_F32 ? glu<IFA_F32> : dtype == IFA_F16 ? glu<IFA_F16> : glu<IFA_BF16>;
    return f(kind, limit, gate_up, ld, rows, cols, q_e4m3, ldq, scale_f32, lds, ifa_s(stream));
}

} // extern "C"
