// ifa_moe_fp8.hip -- mixture of experts whose matrices and activations are 8-bit floating point, and the router that chooses by groups of experts.
//   router   score_e = sigmoid(z_e) or softmax(z)_e, choice_e = score_e + correction_e; a group's value is the sum of its best one or two choices; of the groups with
//            the largest values the `top` largest choices are taken (the lower index wins a tie everywhere); weight = score [/ (sum of the taken + eps)] * scale
//   experts  y[t] (+)= sum_k wgt[t][k] * Down_e q(act(Gate_e a[t]) * (Up_e a[t])),  e = idx[t][k];  q: rows in e4m3 with a scale for each 128 columns
#include <algorithm>
#include "ifa_host.h"
#include "ifa_fp8_stream.h"

using namespace ifa8;

namespace {

// One wave per row.  Scores and choices in 64 bits: two experts whose choices differ by less than a 32-bit rounding are told apart as the formula does.
__global__ void __launch_bounds__(64) k_moe_route_groups(const float *__restrict__ logits, size_t ld, int n_all, int top, int score_kind, int groups, int kept, int best_of, int renorm,
                                                         float renorm_eps, float wgt_scale, const float *__restrict__ corr, int *__restrict__ idx, float *__restrict__ wgt)
{
    extern __shared__ double sc[];          // [n_all] scores, [n_all] choices
    double *ch = sc + n_all;
    const int lane = threadIdx.x, each = n_all / groups;
    const size_t t = blockIdx.x;
    const float *z = logits + t * ld;
    auto logit = [&](int e) { const float v = z[e]; return v == v ? v : -INFINITY; };
    double mx = 0.0, all = 1.0;
    if (score_kind == 0) {
        float m = -INFINITY;
        for (int e = lane; e < n_all; e += 64) m = fmaxf(m, logit(e));
        mx = (double)ifa32::wave_max(m);
        all = 0.0;
        for (int e = lane; e < n_all; e += 64) all += exp((double)logit(e) - mx);
        for (int o = 32; o > 0; o >>= 1) all += __shfl_xor(all, o, 64);
    }
    for (int e = lane; e < n_all; e += 64) {
        const float v = logit(e);
        const double s = score_kind == 0 ? exp((double)v - mx) / all : 1.0 / (1.0 + exp(-(double)v));
        const double c = s + (corr ? (double)corr[e] : 0.0);
        sc[e] = s;
        ch[e] = v > -INFINITY && c == c ? c : -INFINITY;
    }
    __syncthreads();
    if (groups > 1) {
        double value = -INFINITY;          // lane g: of group g
        if (lane < groups) {
            double b0 = -INFINITY, b1 = -INFINITY;
            for (int e = lane * each; e < (lane + 1) * each; e++) { const double c = ch[e]; if (c > b0) { b1 = b0; b0 = c; } else if (c > b1) b1 = c; }
            value = b0 + (best_of > 1 && b1 > -INFINITY ? b1 : 0.0);
        }
        int better = 0;
        for (int g = 0; g < groups; g++) { const double o = __shfl(value, g, 64); better += o > value || (o == value && g < lane); }
        if (lane < groups && better >= kept) for (int e = lane * each; e < (lane + 1) * each; e++) ch[e] = -INFINITY;
        __syncthreads();
    }
    double sum = 0.0, mine = 0.0;
    int at = -1;
    for (int k = 0; k < top; k++) {
        double best = -INFINITY; int bi = n_all;
        for (int e = lane; e < n_all; e += 64) { const double v = ch[e]; if (v > best) { best = v; bi = e; } }
        for (int o = 32; o > 0; o >>= 1) {
            const double ov = __shfl_xor(best, o, 64); const int oi = __shfl_xor(bi, o, 64);
            if (ov > best || (ov == best && oi < bi)) { best = ov; bi = oi; }
        }
        const bool found = bi < n_all;
        const double s = found ? sc[bi] : 0.0;
        sum += s;
        if (lane == k) { at = found ? bi : -1; mine = s; }
        if (found && lane == 0) ch[bi] = -INFINITY;
        __syncthreads();
    }
    if (lane < top) {
        if (renorm) { const double den = sum + (double)renorm_eps; mine = den > 0.0 ? mine / den : 0.0; }
        idx[t * top + lane] = at;
        wgt[t * top + lane] = (float)(mine * (double)wgt_scale);
    }
}

// ONE workgroup: the pairs (row, choice) sorted by expert.  place_row[at] = the row of the pair at sorted place `at`, pair_at[p] = the place of pair p (-1: none), tiles = {expert, first
// place, places} of at most `tile` places of one expert.  A pair's place within its expert's range is a matter of order alone: no value depends on it.
__global__ void __launch_bounds__(1024) k_moe_fp8_sort(const int *__restrict__ idx, int pairs, int experts, int top, int tile, int *__restrict__ place_row, int *__restrict__ pair_at,
                                                       int *__restrict__ tiles, int *__restrict__ n_tiles)
{
    extern __shared__ int cnt[];          // [experts] counts, then cursors; [experts] first places
    int *off = cnt + experts;
    for (int e = threadIdx.x; e < experts; e += blockDim.x) cnt[e] = 0;
    __syncthreads();
    for (int p = threadIdx.x; p < pairs; p += blockDim.x) { const int e = idx[p]; if (e >= 0 && e < experts) atomicAdd(&cnt[e], 1); }
    __syncthreads();
    if (threadIdx.x == 0) {
        int o = 0, nt = 0;
        for (int e = 0; e < experts; e++) {
            off[e] = o;
            for (int r = 0; r < cnt[e]; r += tile) { tiles[3 * nt] = e; tiles[3 * nt + 1] = o + r; tiles[3 * nt + 2] = min(tile, cnt[e] - r); nt++; }
            o += cnt[e];
            cnt[e] = 0;
        }
        *n_tiles = nt;
    }
    __syncthreads();
    for (int p = threadIdx.x; p < pairs; p += blockDim.x) {
        const int e = idx[p];
        if (e < 0 || e >= experts) { pair_at[p] = -1; continue; }
        const int at = off[e] + atomicAdd(&cnt[e], 1);
        place_row[at] = p / top; pair_at[p] = at;
    }
}

// act[at][n] = act(Gate_e a) (Up_e a) for the places of a tile; grid (16 columns each, tiles)
template <int TILES>
__global__ void __launch_bounds__(64 * STREAM_WAVES) k_moe_fp8_up(const uint8_t *__restrict__ gu, const float *__restrict__ sgu, int width, int ff, const uint8_t *__restrict__ a, size_t lda,
                                                                 const float *__restrict__ sa, size_t lds, const int *__restrict__ place_row, const int *__restrict__ tiles,
                                                                 const int *__restrict__ n_tiles, int kind, float limit, float *__restrict__ act)
{
    if ((int)blockIdx.y >= *n_tiles) return;
    __shared__ f32x4 red[(STREAM_WAVES - 1) * 2 * TILES * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n0 = blockIdx.x * 16, e = tiles[3 * blockIdx.y], at0 = tiles[3 * blockIdx.y + 1], n_at = tiles[3 * blockIdx.y + 2];
    const size_t n = min(n0 + (lane & 15), ff - 1), wb = blocks_of(width), fb = blocks_of(ff);
    const uint8_t *wr[2] = {gu + ((size_t)e * 2 * ff + n) * width, gu + ((size_t)(e * 2 + 1) * ff + n) * width};
    const float *swr[2] = {sgu + ((size_t)e * 2 * fb + n0 / BLOCK) * wb, sgu + ((size_t)(e * 2 + 1) * fb + n0 / BLOCK) * wb};
    const uint8_t *ar[TILES];
    const float *sar[TILES];
    f32x4 acc[2][TILES];
#pragma unroll
    for (int j = 0; j < TILES; j++) {
        const size_t t = place_row[at0 + min(16 * j + (lane & 15), n_at - 1)];
        ar[j] = a + t * lda;
        sar[j] = sa + t * lds;
        acc[0][j] = acc[1][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    stream_blocks<false, 2, TILES>(wr, swr, ar, sar, width, wave, STREAM_WAVES, acc);
    join_waves<2, TILES>(acc, red);
    if (wave > 0) return;
#pragma unroll
    for (int j = 0; j < TILES; j++) {
        const int at = 16 * j + (lane & 15);
        if (at >= n_at) continue;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int c = n0 + 4 * (lane >> 4) + r;
            if (c < ff) act[(size_t)(at0 + at) * ff + c] = ifa32::glu_of(kind, limit, acc[0][j][r], acc[1][j][r]);
        }
    }
}

// rows of 32-bit activations in places that the tiles hold, into e4m3: a workgroup of two rows of lanes a block
__global__ void __launch_bounds__(256) k_moe_fp8_quantise(const float *__restrict__ act, int ff, const int *__restrict__ tiles, const int *__restrict__ n_tiles, uint8_t *__restrict__ q, float *__restrict__ s)
{
    if ((int)blockIdx.y >= *n_tiles) return;
    const int at0 = tiles[3 * blockIdx.y + 1], n_at = tiles[3 * blockIdx.y + 2], fb = (int)blocks_of(ff);
    for (int i = blockIdx.x * 8 + (threadIdx.x >> 5); i < n_at * fb; i += gridDim.x * 8) {
        const size_t at = at0 + i / fb;
        const int b = i % fb, c = b * BLOCK + 4 * (threadIdx.x & 31);
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (c < ff) unpack<IFA_F32>(*reinterpret_cast<const u32x4 *>(act + at * ff + c), v);
        uint32_t most = 0u;
#pragma unroll
        for (int e = 0; e < 4; e++) most = dpp_max(most, abs_bits(v[e]));
        most = group_max<32>(most);
        const float sc = scale_of(most);
        if (c < ff) *reinterpret_cast<uint32_t *>(q + at * ff + c) = quantise4(v, 1.0f / sc);
        if ((threadIdx.x & 31) == 0) s[at * fb + b] = sc;
    }
}

// out[at][c] = Down_e q[at]; grid (16 columns each, tiles)
template <bool WIDE, int TILES>
__global__ void __launch_bounds__(64 * STREAM_WAVES) k_moe_fp8_down(const uint8_t *__restrict__ down, const float *__restrict__ sdown, int width, int ff, const uint8_t *__restrict__ q,
                                                                   const float *__restrict__ s, const int *__restrict__ tiles, const int *__restrict__ n_tiles, float *__restrict__ out)
{
    if ((int)blockIdx.y >= *n_tiles) return;
    __shared__ f32x4 red[(STREAM_WAVES - 1) * TILES * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n0 = blockIdx.x * 16, e = tiles[3 * blockIdx.y], at0 = tiles[3 * blockIdx.y + 1], n_at = tiles[3 * blockIdx.y + 2];
    const size_t wb = blocks_of(width), fb = blocks_of(ff);
    const uint8_t *wr[1] = {down + ((size_t)e * width + min(n0 + (lane & 15), width - 1)) * ff};
    const float *swr[1] = {sdown + ((size_t)e * wb + n0 / BLOCK) * fb};
    const uint8_t *ar[TILES];
    const float *sar[TILES];
    f32x4 acc[1][TILES];
#pragma unroll
    for (int j = 0; j < TILES; j++) {
        const size_t at = at0 + min(16 * j + (lane & 15), n_at - 1);
        ar[j] = q + at * ff;
        sar[j] = s + at * fb;
        acc[0][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    stream_blocks<WIDE, 1, TILES>(wr, swr, ar, sar, ff, wave, STREAM_WAVES, acc);
    join_waves<1, TILES>(acc, red);
    if (wave > 0) return;
#pragma unroll
    for (int j = 0; j < TILES; j++) {
        const int at = 16 * j + (lane & 15);
        if (at < n_at) *reinterpret_cast<f32x4 *>(out + (size_t)(at0 + at) * width + n0 + 4 * (lane >> 4)) = acc[0][j];      // (width % 16 == 0)
    }
}

// y[t][c] (+)= sum over the row's choices, in their order
template <int DT>
__global__ void __launch_bounds__(256) k_moe_fp8_join(const float *__restrict__ out, const int *__restrict__ pair_at, const float *__restrict__ wgt, int top, int width, size_t all,
                                                      typename Elem<DT>::type *__restrict__ y, size_t ldy, int accumulate)
{
    const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= all) return;
    const size_t t = id / (width / 4);
    const int c = (int)(id % (width / 4)) * 4;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = 0; k < top; k++) {
        const int at = pair_at[t * top + k];
        if (at < 0) continue;
        const f32x4 v = *reinterpret_cast<const f32x4 *>(out + (size_t)at * width + c);
        const float f = wgt[t * top + k];
#pragma unroll
        for (int r = 0; r < 4; r++) sum[r] = fmaf(f, v[r], sum[r]);
    }
#pragma unroll
    for (int r = 0; r < 4; r++) {
        typename Elem<DT>::type *d = y + t * ldy + c + r;
        *d = (typename Elem<DT>::type)(accumulate ? (float)*d + sum[r] : sum[r]);
    }
}

// ---- workspace
size_t up16(size_t n) { return (n + 255) / 256 * 256; }
struct Work {
    size_t lists, tiles, act, q, s, out, bytes;
    Work(size_t rows, size_t top, size_t width, size_t ff, size_t experts)
    {
        const size_t pairs = rows * top, n_tiles = pairs / 16 + std::min(pairs, experts) + 1;
        size_t o = 0;
        auto take = [&](size_t n) { const size_t at = o; o += up16(n); return at; };
        lists = take(8 * pairs + 16);          // place_row, pair_at; the number of tiles
        tiles = take(12 * n_tiles);
        act = take(4 * pairs * ff);
        q = take(pairs * ff);
        s = take(4 * pairs * blocks_of(ff));
        out = take(4 * pairs * width);
        bytes = o;
    }
};

} // namespace

extern "C" {

int ifa_moe_route_groups_f32(int score_kind, int groups, int groups_kept, int group_best, int renorm, float renorm_eps, float wgt_scale, const void *logits_f32, size_t ld, size_t rows, int n_all,
                             int top, const void *correction_f32, int *idx_dev, void *wgt_f32, ifa_stream stream)
{
    IFA_REQUIRE(logits_f32 && idx_dev && wgt_f32, "ifa_moe_route_groups_f32: null pointer");
    IFA_REQUIRE(score_kind == 0 || score_kind == 1, "ifa_moe_route_groups_f32: score kind %d", score_kind);
    IFA_REQUIRE(rows > 0 && rows < (1u << 31) && n_all > 0 && n_all <= 1024 && ld >= (size_t)n_all, "ifa_moe_route_groups_f32: %zu rows of %d experts (1024 at most)", rows, n_all);
    IFA_REQUIRE(groups > 0 && groups <= 64 && n_all % groups == 0 && groups_kept > 0 && groups_kept <= groups && (group_best == 1 || group_best == 2),
                "ifa_moe_route_groups_f32: %d of %d groups by their best %d", groups_kept, groups, group_best);
    IFA_REQUIRE(top > 0 && top <= 64 && top <= groups_kept * (n_all / groups), "ifa_moe_route_groups_f32: %d of %d experts", top, groups_kept * (n_all / groups));
    hipLaunchKernelGGL(k_moe_route_groups, dim3((unsigned)rows), dim3(64), 2 * (size_t)n_all * sizeof(double), ifa_s(stream), (const float *)logits_f32, ld, n_all, top, score_kind, groups,
                       groups_kept, group_best, renorm, renorm_eps, wgt_scale, (const float *)correction_f32, idx_dev, (float *)wgt_f32);
    IFA_LAUNCH_CHECK();
    return IFA_OK;
}

size_t ifa_moe_experts_fp8_workspace_bytes(size_t rows, int top, int width, int ff, int experts)
{
    if (rows == 0 || rows > (1u << 24) || top <= 0 || width <= 0 || ff <= 0 || experts <= 0) return 0;
    return Work(rows, top, width, ff, experts).bytes;
}

int ifa_moe_experts_fp8(int glu_kind, float limit, const void *a_e4m3, size_t lda, const void *a_scale_f32, size_t lds, size_t rows, int width, int ff, int experts, int top,
                        const void *gate_up_e4m3, const void *gate_up_scale_f32, const void *down_e4m3, const void *down_scale_f32, const int *idx_dev, const void *wgt_f32, void *ws,
                        size_t ws_bytes, int y_dtype, void *y, size_t ldy, int accumulate, ifa_stream stream)
{
    IFA_REQUIRE(a_e4m3 && a_scale_f32 && gate_up_e4m3 && gate_up_scale_f32 && down_e4m3 && down_scale_f32 && idx_dev && wgt_f32 && ws && y, "ifa_moe_experts_fp8: null pointer");
    if (!elem_known(y_dtype)) return ifa_fail(IFA_ERR_DTYPE, "ifa_moe_experts_fp8: output dtype %d (F32, F16 or BF16)", y_dtype);
    IFA_REQUIRE(glu_kind >= 0 && glu_kind <= 3, "ifa_moe_experts_fp8: activation %d", glu_kind);
    IFA_REQUIRE(rows > 0 && width > 0 && ff > 0 && width % 16 == 0 && ff % 16 == 0 && experts > 0 && experts <= 1024 && top > 0 && top <= 64 && rows * top <= 1000000 && width <= 65536 && ff <= 65536,
                "ifa_moe_experts_fp8: %zu rows x %d of %d experts, %d x %d (whole 16s)", rows, top, experts, width, ff);
    IFA_REQUIRE(lda >= (size_t)width && lda % 16 == 0 && lds >= blocks_of(width) && ldy >= (size_t)width, "ifa_moe_experts_fp8: row strides");
    IFA_REQUIRE((((uintptr_t)a_e4m3 | (uintptr_t)gate_up_e4m3 | (uintptr_t)down_e4m3 | (uintptr_t)ws) & 15) == 0 && (((uintptr_t)a_scale_f32 | (uintptr_t)gate_up_scale_f32 | (uintptr_t)down_scale_f32) & 3) == 0
                    && (uintptr_t)y % elem_bytes(y_dtype) == 0, "ifa_moe_experts_fp8: misaligned pointer");
    const Work W(rows, top, width, ff, experts);
    IFA_REQUIRE(ws_bytes >= W.bytes, "ifa_moe_experts_fp8: workspace of %zu bytes (%zu needed)", ws_bytes, W.bytes);
    uint8_t *base = (uint8_t *)ws;
    const int pairs = (int)(rows * top);
    int *place_row = (int *)(base + W.lists), *pair_at = place_row + pairs, *n_tiles = pair_at + pairs, *tiles = (int *)(base + W.tiles);
    float *act = (float *)(base + W.act), *s = (float *)(base + W.s), *out = (float *)(base + W.out);
    uint8_t *q = base + W.q;
    const hipStream_t st = ifa_s(stream);
    const int tile = pairs / experts >= 32 ? 64 : 16;
    const unsigned max_tiles = (unsigned)(pairs / tile + std::min(pairs, experts));
    hipLaunchKernelGGL(k_moe_fp8_sort, dim3(1), dim3(1024), 2 * experts * sizeof(int), st, idx_dev, pairs, experts, top, tile, place_row, pair_at, tiles, n_tiles);
    const dim3 g_up((unsigned)((ff + 15) / 16), max_tiles), g_down((unsigned)(width / 16), max_tiles), b(64 * STREAM_WAVES);
    IFA_REQUIRE(max_tiles < 65536, "ifa_moe_experts_fp8: too many rows");
#define IFA_UP(T) hipLaunchKernelGGL((k_moe_fp8_up<T>), g_up, b, 0, st, (const uint8_t *)gate_up_e4m3, (const float *)gate_up_scale_f32, width, ff, (const uint8_t *)a_e4m3, lda, \
                                     (const float *)a_scale_f32, lds, place_row, tiles, n_tiles, glu_kind, limit, act)
#define IFA_DOWN(W, T) hipLaunchKernelGGL((k_moe_fp8_down<W, T>), g_down, b, 0, st, (const uint8_t *)down_e4m3, (const float *)down_scale_f32, width, ff, q, s, tiles, n_tiles, out)
    if (tile == 16) IFA_UP(1); else IFA_UP(4);
    hipLaunchKernelGGL(k_moe_fp8_quantise, dim3((unsigned)std::min<size_t>((blocks_of(ff) * tile + 7) / 8, 64), max_tiles), dim3(256), 0, st, act, ff, tiles, n_tiles, q, s);
    if (y_dtype == IFA_F32) { if (tile == 16) IFA_DOWN(true, 1); else IFA_DOWN(true, 4); }
    else if (tile == 16) IFA_DOWN(false, 1); else IFA_DOWN(false, 4);
#undef IFA_UP
#undef IFA_DOWN
    const size_t all = rows * (width / 4);
#define IFA_JOIN(DT) hipLaunchKernelGGL((k_moe_fp8_join<DT>), dim3(ifa_cdiv(all, 256)), dim3(256), 0, st, out, pair_at, (const float *)wgt_f32, top, width, all, (Elem<DT>::type *)y, ldy, accumulate)
    if (y_dtype == IFA_F32) IFA_JOIN(IFA_F32); else if (y_dtype == IFA_F16) IFA_JOIN(IFA_F16); else IFA_JOIN(IFA_BF16);
#undef IFA_JOIN
    IFA_LAUNCH_CHECK();
    return IFA_OK;
}

} // extern "C"
