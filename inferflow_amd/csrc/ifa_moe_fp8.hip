// ifa_moe_fp8.hip -- mixture of experts whose matrices and activations are 8-bit floating point, and the router that chooses by groups of experts.
//   router   score_e = sigmoid(z_e) or softmax(z)_e, choice_e = score_e + correction_e; a group's value is the sum of its best one or two choices; of the groups with
//            the largest values the `top` largest choices are taken (the lower index wins a tie everywhere); weight = score [/ (sum of the taken + eps)] * scale
//   experts  y[t] (+)= sum_k wgt[t][k] * Down_e q(act(Gate_e a[t]) * (Up_e a[t])),  e = idx[t][k];  q: rows in e4m3 with a scale for each 128 columns
#include <algorithm>
#include <cmath>
#include "ifa_host.h"
#include "ifa_fp8_stream.h"
#include "ifa_fp8_tile.h"

using namespace ifa8;

namespace {

// ---- the router.  One wave per row, four rows a workgroup; lane l holds the choices of experts l, l + 64, ...  Scores and choices in 64 bits: two experts whose choices differ by less than a 32-bit
// rounding are told apart as the formula does.  Bound by instructions (64-bit exponentials and quotients, a maximum over the wave for each expert taken), not by the logits' bytes; so the
// choices are kept as integers that order like them, and the maximum is one of their upper halves (a comparison of 32 bits a step between lanes) unless two are equal there.
// 8191 rows of 256 experts, 8 of 4 groups of 8: 14.2 us (735 vector instructions a wave, issued in three quarters of the busy cycles; the logits alone take 2 us); one to 64 rows 3.4 us and the launch.
constexpr int ROUTE_ROWS = 4;

__device__ __forceinline__ uint64_t order_of(double v)          // orders like v; 0: no choice
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return v > -INFINITY ? ((u >> 63) ? ~u : u | 0x8000000000000000ull) : 0ull;          // (false for a NaN)
}
__device__ __forceinline__ double value_of(uint64_t o) { return __builtin_bit_cast(double, (o >> 63) ? o & 0x7FFFFFFFFFFFFFFFull : ~o); }
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v)
{
    v = group_max<16>(v);
    v = dpp_max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false));          // rows 1 and 3: the row in front of them too
    v = dpp_max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false));          // rows 2 and 3: the half in front of them
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint64_t read_lane(uint64_t v, int lane)
{
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
__device__ __forceinline__ bool set_in(uint64_t mask) { return __builtin_amdgcn_inverse_ballot_w64(mask); }          // this lane's bit
template <int CTRL> __device__ __forceinline__ uint64_t dpp_u64(uint64_t v)
{
    return ((uint64_t)(uint32_t)__builtin_amdgcn_mov_dpp((int)(v >> 32), CTRL, 0xF, 0xF, true) << 32) | (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, true);
}

template <int PER>
__global__ void __launch_bounds__(64 * ROUTE_ROWS) k_moe_route_groups(const float *__restrict__ logits, size_t ld, int rows, int n_all, int top, int score_kind, int groups, int kept, int best_of,
                                                                      int renorm, float renorm_eps, float wgt_scale, const float *__restrict__ corr, int *__restrict__ idx, float *__restrict__ wgt)
{
    __shared__ uint64_t grp[ROUTE_ROWS][64 * PER];          // a row's choices, for its groups
    __shared__ double sc[ROUTE_ROWS][64 * PER];              // and its scores
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, each = n_all / groups;
    const size_t t = (size_t)blockIdx.x * ROUTE_ROWS + wave;
    if (t >= (size_t)rows) return;
    const float *z = logits + t * ld;
    float v[PER], c[PER];
#pragma unroll
    for (int j = 0; j < PER; j++) {
        const int e = min(lane + 64 * j, n_all - 1);          // (all loads at once: none waits for a comparison)
        v[j] = z[e];
        c[j] = corr ? corr[e] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < PER; j++) if (lane + 64 * j >= n_all || !(v[j] == v[j])) v[j] = -INFINITY;
    double s[PER];
    if (score_kind == 0) {
        float m = -INFINITY;
#pragma unroll
        for (int j = 0; j < PER; j++) m = fmaxf(m, v[j]);
        const double mx = (double)ifa32::wave_max(m);
        double all = 0.0;
#pragma unroll
        for (int j = 0; j < PER; j++) { s[j] = exp((double)v[j] - mx); all += lane + 64 * j < n_all ? s[j] : 0.0; }
        for (int o = 32; o > 0; o >>= 1) all += __shfl_xor(all, o, 64);
        all = 1.0 / all;
#pragma unroll
        for (int j = 0; j < PER; j++) s[j] *= all;
    } else {
#pragma unroll
        for (int j = 0; j < PER; j++) s[j] = 1.0 / (1.0 + exp(-(double)v[j]));
    }
    uint32_t hi[PER], lo[PER];
#pragma unroll
    for (int j = 0; j < PER; j++) {
        const uint64_t o = v[j] > -INFINITY ? order_of(s[j] + (double)c[j]) : 0ull;
        hi[j] = (uint32_t)(o >> 32); lo[j] = (uint32_t)o;
        sc[wave][lane + 64 * j] = s[j];
        if (groups > 1) grp[wave][lane + 64 * j] = o;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");          // (a wave reads what it has written itself)
    if (groups > 1) {
        // a group's best two by `per` neighbouring lanes, each over its part of the group
        const int per = 64 >> (32 - __builtin_clz(groups - 1)), g = lane / per;
        uint64_t b0 = 0, b1 = 0;
        if (g < groups)
            for (int e = g * each + lane % per; e < (g + 1) * each; e += per) { const uint64_t o = grp[wave][e]; if (o > b0) { b1 = b0; b0 = o; } else if (o > b1) b1 = o; }
        auto merge = [&](uint64_t p0, uint64_t p1) { b1 = max(min(b0, p0), max(b1, p1)); b0 = max(b0, p0); };
        if (per > 1) merge(dpp_u64<0xB1>(b0), dpp_u64<0xB1>(b1));
        if (per > 2) merge(dpp_u64<0x4E>(b0), dpp_u64<0x4E>(b1));
        if (per > 4) merge(dpp_u64<0x141>(b0), dpp_u64<0x141>(b1));
        if (per > 8) merge(dpp_u64<0x128>(b0), dpp_u64<0x128>(b1));
        if (per > 16) merge(__shfl_xor(b0, 16, 64), __shfl_xor(b1, 16, 64));
        const double value = b0 == 0 ? -INFINITY : value_of(b0) + (best_of > 1 && b1 != 0 ? value_of(b1) : 0.0);
        int better = 0;
        for (int o = 0; o < groups; o++) {
            const double other = __builtin_bit_cast(double, read_lane(__builtin_bit_cast(uint64_t, value), o * per));
            const uint64_t behind = o * per + per < 64 ? ~0ull << (o * per + per) : 0ull;          // (lanes of groups of a larger index: an equal value is better there)
            better += set_in(__ballot(other > value) | (__ballot(other >= value) & behind));
        }
        const uint64_t stays = __ballot(better < kept);
#pragma unroll
        for (int j = 0; j < PER; j++)
            if (!((stays >> (min((lane + 64 * j) / each, groups - 1) * per)) & 1)) hi[j] = 0;
    }
    int at = -1;
    for (int k = 0; k < top; k++) {
        uint32_t m = hi[0];
#pragma unroll
        for (int j = 1; j < PER; j++) m = dpp_max(m, hi[j]);
        m = wave_max_u32(m);
        if (m == 0) break;          // (a choice's upper half is not 0)
        uint64_t who[PER];
        int n = 0, e = -1;
#pragma unroll
        for (int j = 0; j < PER; j++) { who[j] = __ballot(hi[j] == m); n += __popcll(who[j]); }
        if (n > 1) {          // the same upper half: by the lower ones
            uint32_t l = 0;
#pragma unroll
            for (int j = 0; j < PER; j++) if (hi[j] == m) l = dpp_max(l, lo[j]);
            l = wave_max_u32(l);
#pragma unroll
            for (int j = 0; j < PER; j++) who[j] = __ballot(hi[j] == m && lo[j] == l);
        }
#pragma unroll
        for (int j = 0; j < PER; j++)
            if (who[j]) {
                if (e < 0) { e = 64 * j + __builtin_ctzll(who[j]); who[j] &= -who[j]; }          // (the lowest index of equals)
                else who[j] = 0;
            }
#pragma unroll
        for (int j = 0; j < PER; j++) if (set_in(who[j])) hi[j] = 0;
        if (lane == k) at = e;
    }
    double mine = at >= 0 ? sc[wave][at] : 0.0;
    if (renorm) {
        double sum = mine;
        auto add = [&](uint64_t o) { sum += __builtin_bit_cast(double, o); };
        add(dpp_u64<0xB1>(__builtin_bit_cast(uint64_t, sum)));
        add(dpp_u64<0x4E>(__builtin_bit_cast(uint64_t, sum)));
        add(dpp_u64<0x141>(__builtin_bit_cast(uint64_t, sum)));
        if (top > 8) add(dpp_u64<0x128>(__builtin_bit_cast(uint64_t, sum)));
        for (int o = 16; o < top; o <<= 1) sum += __shfl_xor(sum, o, 64);          // (the lanes behind the last choice hold 0)
        const double den = sum + (double)renorm_eps;
        mine = den > 0.0 ? mine / den : 0.0;
    }
    if (lane < top) {
        idx[t * top + lane] = at;
        wgt[t * top + lane] = (float)(mine * (double)wgt_scale);
    }
}

// ---- one to a few rows, two launches: every (row, choice) pair streams its expert's matrices.
// act[p][n] = act(Gate_e a) (Up_e a) of pair p; grid (16 columns each, pairs), the blocks of columns shared out to the waves
// Bound by the matrices' bytes and a launch's start and end: 6 experts of 2048 x 1408, 34.6 MB, 11.9 us (7.0 at a copy's rate; 10.2 with sums by the 8-bit instructions, see ifa_moe_experts_fp8).
constexpr int PAIR_WAVES = 8;
__global__ void __launch_bounds__(64 * PAIR_WAVES) k_moe_fp8_up_pairs(const uint8_t *__restrict__ gu, const float *__restrict__ sgu, int width, int ff, int experts, int top,
                                                                      const uint8_t *__restrict__ a, size_t lda, const float *__restrict__ sa, size_t lds, const int *__restrict__ idx, int kind,
                                                                      float limit, float *__restrict__ act)
{
    __shared__ f32x4 red[(PAIR_WAVES - 1) * 2 * 64];
    const int p = blockIdx.y, e = idx[p];
    if (e < 0 || e >= experts) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n0 = blockIdx.x * 16;
    const size_t n = n0 + (lane & 15), wb = blocks_of(width), fb = blocks_of(ff), t = p / top;          // (ff in whole 16s)
    const uint8_t *wr[2] = {gu + ((size_t)e * 2 * ff + n) * width, gu + ((size_t)(e * 2 + 1) * ff + n) * width};
    const float *swr[2] = {sgu + ((size_t)e * 2 * fb + n0 / BLOCK) * wb, sgu + ((size_t)(e * 2 + 1) * fb + n0 / BLOCK) * wb};
    const uint8_t *ar[1] = {a + t * lda};
    const float *sar[1] = {sa + t * lds};
    f32x4 acc[2][1];
    acc[0][0] = acc[1][0] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    stream_blocks<true, 1, 2, 1>(wr, swr, ar, sar, width, wave, PAIR_WAVES, acc);
    join_waves<PAIR_WAVES, 2, 1>(acc, red);
    if (wave > 0 || (lane & 15)) return;          // (the sixteen activation rows of the products are one and the same)
    float v[4] = {acc[0][0][0], acc[0][0][1], acc[0][0][2], acc[0][0][3]};
    gated_all(kind, limit, v, {acc[1][0][0], acc[1][0][1], acc[1][0][2], acc[1][0][3]});
    *reinterpret_cast<u32x4 *>(act + (size_t)p * ff + n0 + 4 * (lane >> 4)) = pack<IFA_F32>(v);
}

// 32-bit activations of pairs into e4m3 in LDS: item it = block it % fb of pair pair(it / fb) (-1: zeros); [items] blocks of 128 bytes and their scales.  Half a wave an item.
template <class Pair> __device__ __forceinline__ void quantise_items(const float *__restrict__ act, int ff, int fb, int items, Pair pair, char *q, float *sc)
{
    for (int it = threadIdx.x >> 5; it < items; it += blockDim.x >> 5) {
        const int k = it / fb, b = it - k * fb, p = pair(k), c = b * BLOCK + 4 * (threadIdx.x & 31);
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (p >= 0 && c < ff) unpack<IFA_F32>(*reinterpret_cast<const u32x4 *>(act + (size_t)p * ff + c), v);
        uint32_t most = 0u;
#pragma unroll
        for (int r = 0; r < 4; r++) most = dpp_max(most, abs_bits(v[r]));
        most = group_max<32>(most);
        const float s = scale_of(most);
        *reinterpret_cast<uint32_t *>(q + it * BLOCK + 4 * (threadIdx.x & 31)) = quantise4(v, 1.0f / s);
        if ((threadIdx.x & 31) == 0) sc[it] = p >= 0 ? s : 0.0f;
    }
}

// y[t][c] (+)= sum_k wgt Down_e q(act[t, k]); grid (8 columns each, rows).  Of the sixteen matrix rows of a product eight are of one choice's expert and eight, the same columns, of another's; their
// activations are its columns 0 and 1 (with sixteen columns of one expert 2048 columns are 128 workgroups, half of the compute units: 14 us).  A workgroup quantises its row's activations into LDS
// itself (again in every workgroup: a launch of its own would take longer), its first weights on their way meanwhile.  6 experts of 2048 x 1408, 17.3 MB: 9.8 us (3.5 at a copy's rate; the rest is
// the chain index, activations, maximum, first product).
template <int DT, int AHEAD>
__global__ void __launch_bounds__(64 * PAIR_WAVES) k_moe_fp8_down_pairs(const uint8_t *__restrict__ down, const float *__restrict__ sdown, int width, int ff, int experts, int top,
                                                                        const float *__restrict__ act, const int *__restrict__ idx, const float *__restrict__ wgt,
                                                                        typename Elem<DT>::type *__restrict__ y, size_t ldy, int accumulate)
{
    constexpr bool WIDE = DT == IFA_F32;
    extern __shared__ __attribute__((aligned(16))) char smem[];          // [2 pairs of choices * fb] blocks of 128 bytes, their scales
    __shared__ f32x4 red[(PAIR_WAVES - 1) * 64];
    __shared__ int expert[64];
    __shared__ float weight[64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, n0 = blockIdx.x * 8, fb = (int)blocks_of(ff), both = (top + 1) / 2, items = both * fb, p0 = blockIdx.y * top;
    const size_t wb = blocks_of(width);
    float *const sc = reinterpret_cast<float *>(smem + (size_t)2 * items * BLOCK);
    if (threadIdx.x < 2 * both) {
        const int e = (int)threadIdx.x < top ? idx[p0 + threadIdx.x] : -1;
        expert[threadIdx.x] = e >= 0 && e < experts ? e : -1;
        weight[threadIdx.x] = (int)threadIdx.x < top ? wgt[p0 + threadIdx.x] : 0.0f;
    }
    __syncthreads();
    // item: block item % fb of choices 2 k and 2 k + 1, k = item / fb.  A lane's matrix row: column n0 + lane % 8 of choice 2 k + (lane / 8) % 2; its results': choice 2 k + lane / 32
    const u32x4 zero = {0u, 0u, 0u, 0u};
    struct Group { u32x4 w[AHEAD][2]; float f[AHEAD]; };
    auto ask = [&](Group &G, int first) {
#pragma unroll
        for (int d = 0; d < AHEAD; d++) {
            const int it = first + d * PAIR_WAVES, k = it < items ? it / fb : 0, b = it - k * fb, c = b * BLOCK + 16 * g;
            const int e = it < items ? expert[2 * k + ((lane >> 3) & 1)] : -1, er = it < items ? expert[2 * k + (lane >> 5)] : -1;
            const uint8_t *w = down + ((size_t)max(e, 0) * width + n0 + (lane & 7)) * ff + c;
            G.w[d][0] = e >= 0 && c < ff ? *reinterpret_cast<const u32x4 *>(w) : zero;
            G.w[d][1] = e >= 0 && c + 64 < ff ? *reinterpret_cast<const u32x4 *>(w + 64) : zero;
            G.f[d] = er >= 0 ? sdown[((size_t)er * wb + n0 / BLOCK) * fb + b] * weight[2 * k + (lane >> 5)] : 0.0f;
        }
    };
    Group G[2];
    ask(G[0], wave);
    quantise_items(act, ff, fb, 2 * items, [&](int k) { return expert[k] >= 0 ? p0 + k : -1; }, smem, sc);
    __syncthreads();
    f32x4 acc[1][1];
    acc[0][0] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    auto go = [&](const Group &G, int first) {
#pragma unroll
        for (int d = 0; d < AHEAD; d++) {
            const int it = first + d * PAIR_WAVES;
            if (it >= items) break;
            const int k = it / fb, b = it - k * fb;
            Operand<WIDE> av, wv;
            const char *q = smem + ((2 * k + (lane & 1)) * fb + b) * BLOCK + 16 * g;
            av.set(*reinterpret_cast<const u32x4 *>(q), *reinterpret_cast<const u32x4 *>(q + 64));
            wv.set(G.w[d][0], G.w[d][1]);
            const f32x4 x = mfma128(wv, av);
            const float s = sc[(2 * k + (lane >> 5)) * fb + b];
            if (expert[2 * k + (lane >> 5)] >= 0)          // (a choice that is none: whatever its weight is)
#pragma unroll
                for (int r = 0; r < 4; r++) acc[0][0][r] = fmaf(x[r], G.f[d] * s, acc[0][0][r]);
        }
    };
    for (int it = wave; it < items; it += 2 * AHEAD * PAIR_WAVES) {
        ask(G[1], it + AHEAD * PAIR_WAVES);
        go(G[0], it);
        ask(G[0], it + 2 * AHEAD * PAIR_WAVES);
        go(G[1], it + AHEAD * PAIR_WAVES);
    }
    join_waves<PAIR_WAVES, 1, 1>(acc, red);
    if (wave > 0) return;
    // lane 0 / 16: columns 0 .. 3 / 4 .. 7 of the first choices; lane 33 / 49: of the second ones
#pragma unroll
    for (int r = 0; r < 4; r++) acc[0][0][r] += __shfl(acc[0][0][r], (lane + 33) & 63, 64);
    if (lane != 0 && lane != 16) return;
    typename Elem<DT>::type *d = y + (size_t)blockIdx.y * ldy + n0 + 4 * g;
#pragma unroll
    for (int r = 0; r < 4; r++) d[r] = (typename Elem<DT>::type)(accumulate ? (float)d[r] + acc[0][0][r] : acc[0][0][r]);
}

// ---- a few rows for each expert, three launches: a workgroup finds the pairs of its expert itself, in their order, and streams its part of the expert's matrices past all of them.
constexpr int LIST_MAX = 2048;          // pairs of a step
constexpr int LIST_WAVES = 4;
// pairs p with idx[p] == e in list[0 .. n); every thread gets n
template <int WAVES> __device__ __forceinline__ int list_pairs(const int *__restrict__ idx, int pairs, int e, uint16_t *list, int *counts)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int n = 0;
    for (int p0 = 0; p0 < pairs; p0 += 64 * WAVES) {
        const int p = p0 + threadIdx.x;
        const bool mine = p < pairs && idx[p] == e;
        const uint64_t who = __ballot(mine);
        if (lane == 0) counts[wave] = __popcll(who);
        __syncthreads();
        int at = n;
#pragma unroll
        for (int w = 0; w < WAVES; w++) { if (w < wave) at += counts[w]; n += counts[w]; }
        if (mine) list[at + __popcll(who & ((1ull << lane) - 1))] = (uint16_t)p;
        __syncthreads();
    }
    return n;
}

// act[p] of the expert's pairs; grid (16 columns each, experts), the blocks of columns shared out to the waves.  (A workgroup of 128 columns, a wave 16 of them, could quantise them too: few workgroups,
// 22.6 + 3.4 -> 32.5 us for 53 rows of four of 32 experts, 2048 x 704.)  Bound by the matrices' bytes, 92 MB there: 22 us, 4.2 TB/s.
template <int TILES>
__device__ __forceinline__ void up_list(const uint16_t *list, int n, const uint8_t *const (&wr)[2], const float *const (&swr)[2], int n0, int width, int ff, int top, const uint8_t *a, size_t lda,
                                        const float *sa, size_t lds, int kind, float limit, float *act, f32x4 *red)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15;
    const uint8_t *ar[TILES];
    const float *sar[TILES];
    f32x4 acc[2][TILES];
#pragma unroll
    for (int j = 0; j < TILES; j++) {
        const size_t t = list[min(16 * j + i, n - 1)] / top;
        ar[j] = a + t * lda; sar[j] = sa + t * lds;
        acc[0][j] = acc[1][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    stream_blocks<true, 1, 2, TILES, false>(wr, swr, ar, sar, width, wave, LIST_WAVES, acc);
    join_waves<LIST_WAVES, 2, TILES>(acc, red);
    if (wave == 0) {
#pragma unroll
        for (int j = 0; j < TILES; j++) {
            if (16 * j + i >= n) continue;
            float v[4] = {acc[0][j][0], acc[0][j][1], acc[0][j][2], acc[0][j][3]};
            gated_all(kind, limit, v, {acc[1][j][0], acc[1][j][1], acc[1][j][2], acc[1][j][3]});
            *reinterpret_cast<u32x4 *>(act + (size_t)list[16 * j + i] * ff + n0 + 4 * (lane >> 4)) = pack<IFA_F32>(v);
        }
    }
    __syncthreads();          // (`red` is read)
}
__global__ void __launch_bounds__(64 * LIST_WAVES) k_moe_fp8_up_list(const uint8_t *__restrict__ gu, const float *__restrict__ sgu, int width, int ff, int pairs, int top,
                                                                     const uint8_t *__restrict__ a, size_t lda, const float *__restrict__ sa, size_t lds, const int *__restrict__ idx, int kind,
                                                                     float limit, float *__restrict__ act)
{
    __shared__ uint16_t list[LIST_MAX];
    __shared__ int counts[LIST_WAVES];
    __shared__ f32x4 red[(LIST_WAVES - 1) * 2 * 2 * 64];
    const int e = blockIdx.y, n = list_pairs<LIST_WAVES>(idx, pairs, e, list, counts), lane = threadIdx.x & 63, n0 = blockIdx.x * 16;          // (ff in whole 16s)
    const size_t r0 = n0 + (lane & 15), wb = blocks_of(width), fb = blocks_of(ff);
    const uint8_t *wr[2] = {gu + ((size_t)e * 2 * ff + r0) * width, gu + ((size_t)(e * 2 + 1) * ff + r0) * width};
    const float *swr[2] = {sgu + ((size_t)e * 2 * fb + n0 / BLOCK) * wb, sgu + ((size_t)(e * 2 + 1) * fb + n0 / BLOCK) * wb};
    for (int at = 0; at < n; at += 32) {
        if (n - at <= 16) up_list<1>(list + at, n - at, wr, swr, n0, width, ff, top, a, lda, sa, lds, kind, limit, act, red);
        else up_list<2>(list + at, n - at, wr, swr, n0, width, ff, top, a, lda, sa, lds, kind, limit, act, red);
    }
}

// out[p] of the expert's pairs, 16 at a time; grid (128 columns, experts), a wave 16 columns and all their blocks.  The workgroup quantises the pairs' activations into LDS itself.  46 MB: 16.4 us, 2.8 TB/s.
constexpr int DOWN_WAVES = 8;
constexpr int DOWN_FF = 4096;          // at most: 16 rows in LDS
template <bool WIDE>
__global__ void __launch_bounds__(64 * DOWN_WAVES) k_moe_fp8_down_list(const uint8_t *__restrict__ down, const float *__restrict__ sdown, int width, int ff, int pairs, const int *__restrict__ idx,
                                                                       const float *__restrict__ act, float *__restrict__ out)
{
    constexpr int AHEAD = 3;
    extern __shared__ __attribute__((aligned(16))) char smem[];          // [16 * fb] blocks of 128 bytes, their scales
    __shared__ uint16_t list[LIST_MAX];
    __shared__ int counts[DOWN_WAVES];
    const int e = blockIdx.y, lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15, n0 = blockIdx.x * 16 * DOWN_WAVES + 16 * (threadIdx.x >> 6), fb = (int)blocks_of(ff);
    float *const sc = reinterpret_cast<float *>(smem + (size_t)16 * fb * BLOCK);
    const bool live = n0 < width;          // (width in whole 16s)
    const uint8_t *const w = down + ((size_t)e * width + (live ? n0 : 0) + i) * ff;
    const float *const sw = sdown + ((size_t)e * blocks_of(width) + (live ? n0 : 0) / BLOCK) * fb;
    const u32x4 zero = {0u, 0u, 0u, 0u};
    struct Group { u32x4 w[AHEAD][2]; float f[AHEAD]; };
    auto ask = [&](Group &G, int b0) {
#pragma unroll
        for (int d = 0; d < AHEAD; d++) {
            const int b = min(b0 + d, fb - 1), c = b * BLOCK + 16 * g;
            G.w[d][0] = c < ff ? *reinterpret_cast<const u32x4 *>(w + c) : zero;
            G.w[d][1] = c + 64 < ff ? *reinterpret_cast<const u32x4 *>(w + c + 64) : zero;
            G.f[d] = sw[b];
        }
    };
    const int n = list_pairs<DOWN_WAVES>(idx, pairs, e, list, counts);
    for (int at = 0; at < n; at += 16) {
        const int here = min(n - at, 16);
        Group G[2];
        ask(G[0], 0);
        if (at > 0) __syncthreads();          // (the rows before are read)
        quantise_items(act, ff, fb, here * fb, [&](int k) { return (int)list[at + k]; }, smem, sc);
        __syncthreads();
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
        const int row = min(i, here - 1) * fb;
        auto go = [&](const Group &G, int b0) {
#pragma unroll
            for (int d = 0; d < AHEAD; d++) {
                const int b = b0 + d;
                if (b >= fb) break;
                Operand<WIDE> av, wv;
                const char *q = smem + (row + b) * BLOCK + 16 * g;
                av.set(*reinterpret_cast<const u32x4 *>(q), *reinterpret_cast<const u32x4 *>(q + 64));
                wv.set(G.w[d][0], G.w[d][1]);
                const f32x4 x = mfma128(wv, av);
                const float f = G.f[d] * sc[row + b];
#pragma unroll
                for (int r = 0; r < 4; r++) acc[r] = fmaf(x[r], f, acc[r]);
            }
        };
        for (int b = 0; b < fb; b += 2 * AHEAD) {
            ask(G[1], b + AHEAD);
            go(G[0], b);
            ask(G[0], b + 2 * AHEAD);
            go(G[1], b + AHEAD);
        }
        if (live && i < here) *reinterpret_cast<f32x4 *>(out + (size_t)list[at + i] * width + n0 + 4 * g) = acc;
    }
}

// ---- many rows: the pairs sorted by expert.  k_moe_fp8_count leaves, for each block of `per` pairs, how many of them chose each expert, and in pair_at[p] the expert of pair p (-1: none); k_moe_fp8_place
// adds these counts up and gives the pairs their places from what was counted (idx is looked at once: if it changed meanwhile, places counted by one idx and given out by another would run past the
// lists): place_row[at] = the row of the pair at sorted place `at`, pair_at[p] = the place of pair p (-1: none), tiles = {expert, first place, places} of at most `tile` places of one
// expert, *n_tiles.  (A workgroup alone took 31 us for 18000 pairs.)  A pair's place within its block's part of an expert's range is a matter of order alone: no value depends on it.
__global__ void __launch_bounds__(1024) k_moe_fp8_count(const int *__restrict__ idx, int pairs, int experts, int per, int *__restrict__ counts, int *__restrict__ pair_at)
{
    __shared__ int cnt[1024];
    cnt[threadIdx.x] = 0;
    __syncthreads();
    const int p0 = blockIdx.x * per;
    for (int p = p0 + threadIdx.x; p < min(p0 + per, pairs); p += 1024) {
        const int e = idx[p];
        const bool known = e >= 0 && e < experts;
        if (known) atomicAdd(&cnt[e], 1);
        pair_at[p] = known ? e : -1;
    }
    __syncthreads();
    if ((int)threadIdx.x < experts) counts[blockIdx.x * experts + threadIdx.x] = cnt[threadIdx.x];
}
// what stands in front of a thread's value among 1024 threads' values; part: 17 ints
__device__ __forceinline__ int scan_1024(int v, int *part)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
    for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(x, d, 64); if (lane >= d) x += o; }
    if (lane == 63) part[wave] = x;
    __syncthreads();
    int in_front = 0;
    for (int w = 0; w < 16; w++) if (w < wave) in_front += part[w];
    if (threadIdx.x == 1023) part[16] = in_front + x;
    __syncthreads();
    return in_front + x - v;
}
__global__ void __launch_bounds__(1024) k_moe_fp8_place(int pairs, int experts, int top, int tile, int per, const int *__restrict__ counts, int *__restrict__ place_row,
                                                        int *__restrict__ pair_at, int *__restrict__ tiles, int *__restrict__ n_tiles)
{
    __shared__ int cursor[1024], part[17], part2[17];
    const int e = threadIdx.x, blocks = gridDim.x;
    int before = 0, all = 0;
    if (e < experts)
        for (int b = 0; b < blocks; b++) { const int c = counts[b * experts + e]; all += c; if (b < (int)blockIdx.x) before += c; }
    const int first = scan_1024(all, part);
    cursor[e] = first + before;
    if (blockIdx.x == 0) {
        const int nt = (all + tile - 1) / tile, t0 = scan_1024(nt, part2);
        for (int k = 0; k < nt; k++) { int *t = tiles + 3 * (t0 + k); t[0] = e; t[1] = first + k * tile; t[2] = min(tile, all - k * tile); }
        if (e == 0) *n_tiles = part2[16];
    }
    __syncthreads();
    const int p0 = blockIdx.x * per;
    for (int p = p0 + threadIdx.x; p < min(p0 + per, pairs); p += 1024) {
        const int x = pair_at[p];
        if (x < 0) continue;
        const int at = atomicAdd(&cursor[x], 1);
        place_row[at] = p / top; pair_at[p] = at;
    }
}

// Tiles of 128 or 192 places of one expert (places_for).  A workgroup of eight waves, one a compute unit.
template <int PLACES> using MoeTile = Tile<256, PLACES, 2, 4>;

// tile and block of columns at a place among those that there are (the empty tiles behind them are dealt to nobody): tiles of one expert side by side, full and other ones in turn for a workgroup
__device__ __forceinline__ void moe_place(int at, int n_tiles, int blocks, int &tile, int &block)
{
    constexpr int BAND = 8;
    const int band = at / (BAND * blocks), within = at % (BAND * blocks), in_band = min(BAND, n_tiles - band * BAND);
    block = within / in_band;
    tile = band * BAND + (within + block / 4) % in_band;
}

struct UpJob {
    const uint8_t *wbase, *abase, *a;
    const float *sg, *su, *sa;
    const int *rows;          // of the tile's places
    int cols, n0, ff, at0, n_at, block;
    size_t lda;
    bool idle;
    __device__ __forceinline__ uint32_t woff(int r) const { return (uint32_t)((r < BLOCK ? 0 : ff) + min(n0 + (r & (BLOCK - 1)), ff - 1)) * (uint32_t)cols; }
    __device__ __forceinline__ const uint8_t *asrc(int r) const { return a + (size_t)rows[min(r, n_at - 1)] * lda; }
    __device__ __forceinline__ const float *sw(int h) const { return h ? su : sg; }
};
struct DownJob {
    const uint8_t *wbase, *abase;
    const float *sd, *sa;
    int cols, last_row, at0, n_at, nw;          // (nw: the wave's first column)
    bool idle;
    __device__ __forceinline__ uint32_t woff(int r) const { return (uint32_t)min(r, last_row) * (uint32_t)cols; }
    __device__ __forceinline__ uint32_t asrc(int r) const { return (uint32_t)min(r, n_at - 1) * (uint32_t)cols; }
    __device__ __forceinline__ const float *sw(int) const { return sd; }
};

// a tile of 128 gate rows and the 128 up rows of the same columns: one block of the activations, which leave it quantised.  Bound by the products and a tile's ends (16 blocks of columns
// between them): 17100 pairs of 64 experts, 2048 x 1408, 300 us (181 with sums by the 8-bit instructions, see ifa_moe_experts_fp8).  With 192 places eleven registers are laid aside for the ends of a tile, once a tile
template <int PLACES>
__global__ void __launch_bounds__(512, 2) k_moe_fp8_up_tile(const uint8_t *__restrict__ gu, const float *__restrict__ sgu, int width, int ff, const uint8_t *__restrict__ a, size_t lda,
                                                            const float *__restrict__ sa, size_t lds, const int *__restrict__ place_row, const int *__restrict__ tiles,
                                                            const int *__restrict__ n_tiles, int kind, float limit, uint8_t *__restrict__ q, float *__restrict__ s)
{
    typedef MoeTile<PLACES> T;
    constexpr int MINE = 16 * T::TN;          // places of a wave
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave & 1, wn = wave >> 1, g = lane >> 4, i = lane & 15, fb = (int)blocks_of(ff);
    const int n = *n_tiles;
    const Share share(n * fb);
    if (share.count == 0) return;
    const size_t wb = blocks_of(width);
    auto job = [&](int k) {
        UpJob J;
        int tile;
        moe_place(share.at(k), n, fb, tile, J.block);
        const int e = tiles[3 * tile];
        J.at0 = tiles[3 * tile + 1]; J.n_at = tiles[3 * tile + 2]; J.n0 = J.block * BLOCK; J.cols = width; J.ff = ff; J.a = a; J.lda = lda; J.abase = nullptr;
        J.rows = place_row + J.at0;
        J.wbase = gu + (size_t)e * 2 * ff * width;
        J.sg = sgu + ((size_t)e * 2 * fb + J.block) * wb; J.su = J.sg + fb * wb;
        J.sa = sa + (size_t)J.rows[min(MINE * wn + (fresh(lane) & 63) % MINE, J.n_at - 1)] * lds;
        J.idle = MINE * wn >= J.n_at;
        return J;
    };
    tile_run<true, true, 2, false, T, 2>(smem, share.count, job, [&](const UpJob &J, f32x4 (&acc)[T::TM][T::TN], char *buffer) {
        const int n0 = J.n0, n_at = J.n_at, at0 = J.at0, block = J.block, lane = fresh(threadIdx.x) & 63, g = lane >> 4, i = lane & 15;
        uint32_t *const most = reinterpret_cast<uint32_t *>(buffer + PLACES * BLOCK);          // [2 waves][PLACES], behind the tile's quantised rows
        const bool whole = n0 + BLOCK <= ff;
        uint32_t mine[T::TN];
#pragma unroll
        for (int j = 0; j < T::TN; j++) {
            mine[j] = 0u;
            float v[16], u[16];
#pragma unroll
            for (int k = 0; k < 16; k++) { v[k] = acc[k / 4][j][k % 4]; u[k] = acc[k / 4 + 4][j][k % 4]; }
            gated_all(kind, limit, v, u);
#pragma unroll
            for (int k = 0; k < 16; k++) {
                if (!whole && n0 + 64 * wm + 16 * (k / 4) >= ff) v[k] = 0.0f;          // (ff in whole 16s)
                acc[k / 4][j][k % 4] = v[k];
                mine[j] = dpp_max(mine[j], abs_bits(v[k]));
            }
            mine[j] = dpp_max(mine[j], (uint32_t)__shfl_xor((int)mine[j], 16, 64));
            mine[j] = dpp_max(mine[j], (uint32_t)__shfl_xor((int)mine[j], 32, 64));
            if (g == 0) most[wm * PLACES + MINE * wn + 16 * j + i] = mine[j];
        }
        lds_barrier();
#pragma unroll
        for (int j = 0; j < T::TN; j++) {
            const int at = MINE * wn + 16 * j + i;
            const float sc = scale_of(dpp_max(most[at], most[PLACES + at])), inv = 1.0f / sc;
            if (wm == 0 && g == 0 && at < n_at) s[(size_t)(at0 + at) * fb + block] = sc;
#pragma unroll
            for (int m = 0; m < 4; m++) {
                const float v[4] = {acc[m][j][0], acc[m][j][1], acc[m][j][2], acc[m][j][3]};
                *reinterpret_cast<uint32_t *>(buffer + at * BLOCK + 16 * ((4 * wm + m) ^ (at & 7)) + 4 * g) = quantise4(v, inv);
            }
        }
        lds_barrier();
#pragma unroll
        for (int k = fresh(threadIdx.x) & 511; k < PLACES * 8; k += 64 * T::WAVES) {
            const int at = k >> 3, piece = k & 7;
            if (at < n_at && n0 + 16 * piece < ff) *reinterpret_cast<u32x4 *>(q + (size_t)(at0 + at) * ff + n0 + 16 * piece) = *reinterpret_cast<const u32x4 *>(buffer + at * BLOCK + 16 * (piece ^ (at & 7)));
        }
    });
}

template <bool WIDE, int PLACES>
__global__ void __launch_bounds__(512, 2) k_moe_fp8_down_tile(const uint8_t *__restrict__ down, const float *__restrict__ sdown, int width, int ff, const uint8_t *__restrict__ q,
                                                              const float *__restrict__ s, const int *__restrict__ tiles, const int *__restrict__ n_tiles, float *__restrict__ out)
{
    typedef MoeTile<PLACES> T;
    constexpr int MINE = 16 * T::TN;          // places of a wave
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave & 1, wn = wave >> 1;
    const int n = *n_tiles, blocks = (width + 255) / 256;
    const Share share(n * blocks);
    if (share.count == 0) return;
    const size_t wb = blocks_of(width), fb = blocks_of(ff);
    auto job = [&](int k) {
        DownJob J;
        int tile, block;
        moe_place(share.at(k), n, blocks, tile, block);
        const int e = tiles[3 * tile], n0 = block * 256;
        J.at0 = tiles[3 * tile + 1]; J.n_at = tiles[3 * tile + 2]; J.nw = n0 + 128 * wm; J.cols = ff; J.last_row = width - 1 - n0;
        J.wbase = down + ((size_t)e * width + n0) * ff; J.abase = q + (size_t)J.at0 * ff;
        J.sd = sdown + ((size_t)e * wb + min(J.nw, width - 1) / BLOCK) * fb;
        J.sa = s + (size_t)(J.at0 + min(MINE * wn + (fresh(lane) & 63) % MINE, J.n_at - 1)) * fb;
        J.idle = MINE * wn >= J.n_at || J.nw >= width;
        return J;
    };
    tile_run<true, WIDE, 1, true, T, 2>(smem, share.count, job, [&](const DownJob &J, const f32x4 (&acc)[T::TM][T::TN], char *buffer) {
        tile_out<T, true, 4>(buffer, acc, [&](int t, int n, float *v) {
            if (MINE * wn + t < J.n_at && J.nw + n < width) *reinterpret_cast<u32x4 *>(out + (size_t)(J.at0 + MINE * wn + t) * width + J.nw + n) = pack<IFA_F32>(v);          // (width in whole 16s)
        });
    });
}

// y[t][c] (+)= sum over the row's choices, in their order.  Bound by the pairs' rows: 140 MB and 12 of results 30 us, 5 TB/s
template <int DT>
__global__ void __launch_bounds__(256) k_moe_fp8_join(const float *__restrict__ out, const int *__restrict__ pair_at, const int *__restrict__ idx, int experts, const float *__restrict__ wgt, int top, int width, size_t all,
                                                      typename Elem<DT>::type *__restrict__ y, size_t ldy, int accumulate)
{
    const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= all) return;
    const size_t t = id / (width / 4);
    const int c = (int)(id % (width / 4)) * 4;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = 0; k < top; k++) {
        const int p = (int)t * top + k, at = pair_at ? pair_at[p] : (idx[p] >= 0 && idx[p] < experts ? p : -1);          // (no places: the pairs' own order)
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
size_t up256(size_t n) { return (n + 255) / 256 * 256; }
struct Work {
    size_t lists, counts, tiles, act, q, s, out, bytes;
    int per, blocks;          // k_moe_fp8_count's
    Work(size_t rows, size_t top, size_t width, size_t ff, size_t experts)
    {
        const size_t pairs = rows * top, n_tiles = pairs / 128 + std::min(pairs, experts) + 1;
        per = (int)std::max<size_t>(2048, (pairs + 255) / 256);
        blocks = (int)((pairs + per - 1) / per);
        size_t o = 0;
        auto take = [&](size_t n) { const size_t at = o; o += up256(n); return at; };
        lists = take(8 * pairs + 16);          // place_row, pair_at; the number of tiles
        counts = take(4 * blocks * experts);
        tiles = take(12 * n_tiles);
        act = take(pairs <= LIST_MAX ? 4 * pairs * ff : 0);
        q = take(pairs * ff);
        s = take(4 * pairs * blocks_of(ff));
        out = take(4 * pairs * width);
        bytes = o;
    }
};

// Places of a tile: what takes least by these figures (us, measured: a step, that is a block of 128 columns, and beside the steps), with the experts' rows scattered about their mean as independent choices
// would be.  A tile that is not full has waves that only fetch; they leave 0.6 of a step's time to those that do not.  step: by the 8-bit instructions (down, 16-bit outputs), exact: on exact
// halves (gate and up; down, 32-bit outputs).  us 128 / 192, bfloat16 outputs, rows: 64 experts of 2048 x 1408, top 6, 1024 182 / 210, 1400 272 / 225, 2048 313 / 335, 2600 380 / 379, 3001 419 / 412, 4096
// 540 / 508; 8 of 4096 x 4096, top 2, 400 140 / 156, 1100 293 / 233; 128 of 7168 x 2048, top 8, 600 1129 / 1274, 2048 2062 / 1865, 4096 3433 / 3231; 32-bit outputs, the first of these, 1024 200 / 229, 3001
// 496 / 456.  At these eleven sizes of bfloat16 the choice is 0.7 % behind the faster one on average.
int places_for(int width, int ff, int experts, int pairs, bool wide)
{
    constexpr struct { int places; double step, exact, beside; } FORMS[2] = {{128, 1.1, 1.6, 5.5}, {192, 1.4, 2.1, 6.5}};
    constexpr double SHARE[7] = {0.07, 0.12, 0.20, 0.22, 0.20, 0.12, 0.07};          // of experts (k - 3) / 2 deviations from the mean
    const double mean = (double)pairs / experts;
    int best = 128;
    double least = 1e30;
    for (const auto &F : FORMS) {
        double us = 0.0;
        for (int down = 0; down < 2; down++) {
            const double steps = (double)blocks_of(down ? ff : width), blocks = down ? (width + 255) / 256 : (double)blocks_of(ff), step = down && !wide ? F.step : F.exact;
            double time = 0.0, tiles = 0.0;          // an expert's
            for (int k = 0; k < 7; k++) {
                const double n = std::max(1.0, mean + 0.5 * (k - 3) * std::sqrt(mean)), full = std::floor(n / F.places), rest = n - full * F.places, live = std::ceil(4.0 * rest / F.places);
                time += SHARE[k] * (full * (F.beside + steps * step) + (rest > 0.0 ? F.beside + steps * step * (0.4 + 0.15 * live) : 0.0));
                tiles += SHARE[k] * (full + (rest > 0.0 ? 1.0 : 0.0));
            }
            const double rounds = experts * tiles * blocks / 256, each = time / tiles;
            us += std::max((rounds + 0.5) * each, rounds < 3.0 ? std::ceil(rounds - 0.02) * each : 0.0);
        }
        if (us < least) { least = us; best = F.places; }
    }
    return best;
}

// what fits the kernels' 32-bit offsets, lists and grids
bool sizes_known(size_t rows, int top, int width, int ff, int experts)
{
    return rows > 0 && rows <= 1000000 && top > 0 && top <= 64 && rows * top <= 1000000 && width > 0 && width <= 65536 && width % 16 == 0 && ff > 0 && ff <= 65536 && ff % 16 == 0 && experts > 0
           && experts <= 1024 && 2 * (size_t)ff * width < (1ull << 32) && rows * ((size_t)width / 4) < 0xFFFFFF00u;
}

} // namespace

extern "C" {

int ifa_moe_route_groups_f32(int score_kind, int groups, int groups_kept, int group_best, int renorm, float renorm_eps, float wgt_scale, const void *logits_f32, size_t ld, size_t rows, int n_all,
                             int top, const void *correction_f32, int *idx_dev, void *wgt_f32, ifa_stream stream)
{
    IFA_REQUIRE(logits_f32 && idx_dev && wgt_f32, "ifa_moe_route_groups_f32: null pointer");
    IFA_REQUIRE(score_kind == 0 || score_kind == 1, "ifa_moe_route_groups_f32: score kind %d", score_kind);
    IFA_REQUIRE(rows > 0 && rows < (1u << 25) && n_all > 0 && n_all <= 1024 && ld >= (size_t)n_all, "ifa_moe_route_groups_f32: %zu rows (fewer than 2^25) of %d experts (1024 at most)", rows, n_all);
    IFA_REQUIRE(groups > 0 && groups <= 64 && n_all % groups == 0 && groups_kept > 0 && groups_kept <= groups && (group_best == 1 || group_best == 2),
                "ifa_moe_route_groups_f32: %d of %d groups by their best %d", groups_kept, groups, group_best);
    IFA_REQUIRE(top > 0 && top <= 64 && top <= groups_kept * (n_all / groups), "ifa_moe_route_groups_f32: %d of %d experts", top, groups_kept * (n_all / groups));
    const int per = (n_all + 63) / 64;
    const auto fn = per <= 1 ? k_moe_route_groups<1> : per <= 2 ? k_moe_route_groups<2> : per <= 4 ? k_moe_route_groups<4> : per <= 8 ? k_moe_route_groups<8> : k_moe_route_groups<16>;
    hipLaunchKernelGGL(fn, dim3(ifa_cdiv(rows, ROUTE_ROWS)), dim3(64 * ROUTE_ROWS), 0, ifa_s(stream), (const float *)logits_f32, ld, (int)rows, n_all, top, score_kind, groups, groups_kept,
                       group_best, renorm, renorm_eps, wgt_scale, (const float *)correction_f32, idx_dev, (float *)wgt_f32);
    IFA_LAUNCH_CHECK();
    return IFA_OK;
}

size_t ifa_moe_experts_fp8_workspace_bytes(size_t rows, int top, int width, int ff, int experts)
{
    if (!sizes_known(rows, top, width, ff, experts)) return 0;
    return Work(rows, top, width, ff, experts).bytes;
}

int ifa_moe_experts_fp8(int glu_kind, float limit, const void *a_e4m3, size_t lda, const void *a_scale_f32, size_t lds, size_t rows, int width, int ff, int experts, int top,
                        const void *gate_up_e4m3, const void *gate_up_scale_f32, const void *down_e4m3, const void *down_scale_f32, const int *idx_dev, const void *wgt_f32, void *ws,
                        size_t ws_bytes, int y_dtype, void *y, size_t ldy, int accumulate, ifa_stream stream)
{
    IFA_REQUIRE(a_e4m3 && a_scale_f32 && gate_up_e4m3 && gate_up_scale_f32 && down_e4m3 && down_scale_f32 && idx_dev && wgt_f32 && ws && y, "ifa_moe_experts_fp8: null pointer");
    if (!elem_known(y_dtype)) return ifa_fail(IFA_ERR_DTYPE, "ifa_moe_experts_fp8: output dtype %d (F32, F16 or BF16)", y_dtype);
    IFA_REQUIRE(glu_kind >= 0 && glu_kind <= 3, "ifa_moe_experts_fp8: activation %d", glu_kind);
    IFA_REQUIRE(sizes_known(rows, top, width, ff, experts),
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
    const size_t few_lds = (size_t)2 * ((top + 1) / 2) * blocks_of(ff) * (BLOCK + 4);
    // one or two rows, or up to four of small matrices: a stream for each pair.  us pairs / lists, rows x choices of experts, width x ff: 1 x 6 of 64, 2048 x 1408 22.3 / 32.9, 2 31.3 / 40.5, 4 53.6 / 47.1;
    // 4 x 4 of 16, 1024 x 704 15.9 / 16.8, 8 27.7 / 18.5; 2 x 2 of 8, 4096 x 4096 50 / 44, 3 71 / 56; 1 x 8 of 128, 7168 x 2048 85 / 105, 2 166 / 169, 3 246 / 223
    const double bytes = 3.0 * width * ff;
    // Gate and up run on exact halves whatever the output's type (ifa_fp8.h): they decide which e4m3 value an activation becomes, and the 8-bit instructions' error would move one in some thousands to its
    // neighbour, 1e-3 of the output and more -- as much as a bfloat16's rounding adds.  Down: on exact halves for a 32-bit output, by the 8-bit instructions in front of a rounding to 16 bits.
    const bool wide = y_dtype == IFA_F32;
    if ((rows <= 2 || (rows <= 4 && bytes <= 4e6)) && few_lds <= 48 * 1024) {
        hipLaunchKernelGGL(k_moe_fp8_up_pairs, dim3(ff / 16, pairs), dim3(64 * PAIR_WAVES), 0, st, (const uint8_t *)gate_up_e4m3, (const float *)gate_up_scale_f32, width, ff, experts, top,
                           (const uint8_t *)a_e4m3, lda, (const float *)a_scale_f32, lds, idx_dev, glu_kind, limit, act);
#define IFA_DOWN(DT) hipLaunchKernelGGL((k_moe_fp8_down_pairs<DT, 3>), dim3(width / 8, (unsigned)rows), dim3(64 * PAIR_WAVES), few_lds, st, (const uint8_t *)down_e4m3, (const float *)down_scale_f32, \
                                        width, ff, experts, top, act, idx_dev, (const float *)wgt_f32, (Elem<DT>::type *)y, ldy, accumulate)
        if (y_dtype == IFA_F32) IFA_DOWN(IFA_F32); else if (y_dtype == IFA_F16) IFA_DOWN(IFA_F16); else IFA_DOWN(IFA_BF16);
#undef IFA_DOWN
        IFA_LAUNCH_CHECK();
        return IFA_OK;
    }
    // lists go through an expert's matrices once for each 32 of its rows, tiles once for each 128 or 192 but with two launches more about them.  us lists / tiles, rows: 64 experts of 2048 x 1408, top 6,
    // 64 128 / 131, 100 139 / 131, 256 216 / 135; 32 of 2048 x 704, top 4, 96 45 / 52, 160 56 / 54; 16 of 1024 x 704, top 4, 64 27 / 38, 128 39 / 40, 256 59 / 45; 8 of 4096 x 4096, top 2, 48 110 / 120, 64 134 / 122;
    // 128 of 7168 x 2048, top 8, 64 997 / 983, 128 1111 / 1001, 256 1457 / 1030
    const bool many = pairs > LIST_MAX || ff > DOWN_FF || (double)pairs / experts >= (experts * bytes > 256e6 ? 12.0 : experts * bytes > 64e6 ? 15.0 : 30.0);
    if (many) {
        const int places = places_for(width, ff, experts, pairs, wide), max_tiles = pairs / places + std::min(pairs, experts);
        const int lds_bytes = places == 192 ? MoeTile<192>::SMEM : MoeTile<128>::SMEM;
        const size_t g_up = blocks_of(ff) * max_tiles, g_down = (size_t)((width + 255) / 256) * max_tiles;
        int *counts = (int *)(base + W.counts);
        hipLaunchKernelGGL(k_moe_fp8_count, dim3(W.blocks), dim3(1024), 0, st, idx_dev, pairs, experts, W.per, counts, pair_at);
        hipLaunchKernelGGL(k_moe_fp8_place, dim3(W.blocks), dim3(1024), 0, st, pairs, experts, top, places, W.per, counts, place_row, pair_at, tiles, n_tiles);
        const auto up_fn = places == 192 ? k_moe_fp8_up_tile<192> : k_moe_fp8_up_tile<128>;
        const auto fn = places == 192 ? (wide ? k_moe_fp8_down_tile<true, 192> : k_moe_fp8_down_tile<false, 192>) : wide ? k_moe_fp8_down_tile<true, 128> : k_moe_fp8_down_tile<false, 128>;
        IFA_HIP_CHECK(hipFuncSetAttribute((const void *)up_fn, hipFuncAttributeMaxDynamicSharedMemorySize, lds_bytes));
        IFA_HIP_CHECK(hipFuncSetAttribute((const void *)fn, hipFuncAttributeMaxDynamicSharedMemorySize, lds_bytes));
        hipLaunchKernelGGL(up_fn, dim3((unsigned)std::min<size_t>(g_up, 256)), dim3(512), lds_bytes, st, (const uint8_t *)gate_up_e4m3, (const float *)gate_up_scale_f32, width, ff, (const uint8_t *)a_e4m3, lda,
                           (const float *)a_scale_f32, lds, place_row, tiles, n_tiles, glu_kind, limit, q, s);
        hipLaunchKernelGGL(fn, dim3((unsigned)std::min<size_t>(g_down, 256)), dim3(512), lds_bytes, st, (const uint8_t *)down_e4m3, (const float *)down_scale_f32, width, ff, q, s, tiles, n_tiles, out);
    } else {
        hipLaunchKernelGGL(k_moe_fp8_up_list, dim3(ff / 16, experts), dim3(64 * LIST_WAVES), 0, st, (const uint8_t *)gate_up_e4m3, (const float *)gate_up_scale_f32, width, ff, pairs, top,
                           (const uint8_t *)a_e4m3, lda, (const float *)a_scale_f32, lds, idx_dev, glu_kind, limit, act);
        const auto fn = wide ? k_moe_fp8_down_list<true> : k_moe_fp8_down_list<false>;
        const size_t list_lds = 16 * blocks_of(ff) * (BLOCK + 4);
        IFA_HIP_CHECK(hipFuncSetAttribute((const void *)fn, hipFuncAttributeMaxDynamicSharedMemorySize, 16 * DOWN_FF / BLOCK * (BLOCK + 4)));
        hipLaunchKernelGGL(fn, dim3(ifa_cdiv(width, 16 * DOWN_WAVES), experts), dim3(64 * DOWN_WAVES), list_lds, st, (const uint8_t *)down_e4m3, (const float *)down_scale_f32, width, ff, pairs,
                           idx_dev, act, out);
        pair_at = nullptr;
    }
    const size_t all = rows * (width / 4);
#define IFA_JOIN(DT) hipLaunchKernelGGL((k_moe_fp8_join<DT>), dim3(ifa_cdiv(all, 256)), dim3(256), 0, st, out, pair_at, idx_dev, experts, (const float *)wgt_f32, top, width, all, (Elem<DT>::type *)y, ldy, \
                                        accumulate)
    if (y_dtype == IFA_F32) IFA_JOIN(IFA_F32); else if (y_dtype == IFA_F16) IFA_JOIN(IFA_F16); else IFA_JOIN(IFA_BF16);
#undef IFA_JOIN
    IFA_LAUNCH_CHECK();
    return IFA_OK;
}

} // extern "C"
