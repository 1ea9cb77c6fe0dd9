// ifa_fp8_tile.h -- products of many rows in 8-bit floating point: output tiles of BM matrix rows x BN activation rows, the blocks of 128 columns through two buffers in LDS.
//   * both operands go from memory to LDS directly, a wave 8 rows x 128 bytes a request; images are [rows][128 bytes] with the eight 16-byte pieces of row r at slot
//     c ^ ((r >> 1) & 7), so that sixteen lanes that read one piece of sixteen rows meet no bank twice (the permutation sits in the requests' source addresses);
//   * a wave multiplies (BM / WM) x (BN / WN) values of a block as 16 x 16 products over all its 128 columns and adds each, times the two scales, to its 32-bit sums: four
//     multiply-adds beside the 32 cycles of a product;
//   * a buffer is asked for again in two parts, each as soon as everybody has read it: the activations, the scales and the matrix rows of a wave's first products in the middle of the block, the
//     other matrix rows at its end.  So every request has one and a half blocks' products to arrive under (one block's: 2.1 us a block of a 256 x 256 tile instead of 1.8; two and a half, a third buffer
//     of 256 x 128 tiles: 1.13 instead of 1.11);
//   * the requests are inline assembly without results (the compiler would wait for all of them in front of every read of LDS); the waits and barriers stand beside them.
// Measured: 256 x 256 tiles, 4096 rows of 4096 x 16384 2.25-2.32 PFLOP/s, where the chip's power limit lowers its clock (a lone workgroup 1.46 us a block, 0.85 of them products); 11008 x 4096 1.9
// (688 tiles on 256 compute units).
// Columns beyond the last block's end: the requests stay inside their row, and zeros are written over what they brought.  Rows beyond the last: repeated, not stored.
#pragma once
#include "ifa_fp8.h"

namespace ifa8 {

typedef __attribute__((address_space(3))) char lds_char;

// 64 lanes' 16 bytes each to 1024 consecutive bytes of LDS from `to` (the same in all lanes), if `on` (the same in all lanes) is not 0 -- a branch inside, so that the compiler sees none and keeps
// the products around it in their order; they have arrived behind arrive<n>() where n younger requests of the wave may be under way
__device__ __forceinline__ void request16(const void *from, uint32_t to, int on)
{
    asm volatile("s_cmp_eq_u32 %2, 0\n\ts_cbranch_scc1 .Lrequest%=\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n.Lrequest%=:" ::"s"(to), "v"(from), "s"(__builtin_amdgcn_readfirstlane(on)) : "scc", "m0");
}
__device__ __forceinline__ void request16(const void *base, uint32_t offset, uint32_t to, int on)      // (base: the same in all lanes)
{
    asm volatile("s_cmp_eq_u32 %3, 0\n\ts_cbranch_scc1 .Lrequest%=\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n.Lrequest%=:" ::"s"(to), "v"(offset), "s"(base), "s"(__builtin_amdgcn_readfirstlane(on))
                 : "scc", "m0");
}
__device__ __forceinline__ void request4(const void *from, uint32_t to, int on)      // 64 lanes' 4 bytes each to 256 bytes
{
    asm volatile("s_cmp_eq_u32 %2, 0\n\ts_cbranch_scc1 .Lrequest%=\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off\n.Lrequest%=:" ::"s"(to), "v"(from), "s"(__builtin_amdgcn_readfirstlane(on)) : "scc", "m0");
}
template <int N> __device__ __forceinline__ void arrive()      // this wave's requests but the last N, and everybody's; everybody's reads of LDS in front of it are done
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// v, as if it were computed anew here: what hangs on it is not kept in registers from tile to tile (the mask behind it says how large it is)
__device__ __forceinline__ int fresh(int v) { asm volatile("" : "+v"(v)); return v; }
__device__ __forceinline__ int slot_of(int row, int piece) { return piece ^ ((row >> 1) & 7); }

template <int BM, int BN, int WM, int WN> struct Tile {
    static constexpr int STAGES = 2, WAVES = WM * WN, TM = BM / (16 * WM), TN = BN / (16 * WN), WI = BM / (8 * WAVES), AI = BN / (8 * WAVES), DATA = (BM + BN) * BLOCK, SCALES = 2 * 256 * WAVES;
    static constexpr int BUF = DATA + SCALES;          // a buffer: the rows, the waves' activation scales, their matrix scales
    static constexpr int OUT = BUF > WAVES * TM * 1024 ? BUF : WAVES * TM * 1024;          // the last buffer, while sums leave: 16 rows of each wave at least
    static constexpr int SMEM = (STAGES - 1) * BUF + OUT;
    static_assert(WI * 8 * WAVES == BM && AI * 8 * WAVES == BN && TM * 16 * WM == BM && TN * 16 * WN == BN, "whole rows and products a wave");
    static_assert(WI % 2 == 0 && TM % 2 == 0 && TM >= 4 && (BM / (16 * WM)) % 4 == 0 && TN <= 4 && BM == 128 * WM || BM == 64 * WM, "halves of a wave's matrix rows");
};

// A workgroup's tiles one after the other: job(k), k < jobs, says what tile k is made of, done(J, acc, buffer) takes its sums.  A Job has: wbase and woff(r), the tile's matrix rows (32-bit offsets); asrc(r),
// its activation rows (A32: 32-bit offsets from abase); cols; sw(h), the row of block scales of half h; sa, that of the lane's activation row (lane % (16 TN) of this wave's); idle, whether none of the wave's
// activation rows is one: it asks for its part and waits with the others, no more (the chip is at its power limit in the products).
// Wave (wm, wn)'s products m = 0 .. TM - 1 have matrix rows wm BM / WM + 16 m on; NSC 2: in two halves, m < TM / 2 from the tile's rows wm BM / (2 WM) on, the others BM / 2 further on, with matrix scales of
// their own.
// MANY: the next tile's first block is asked for in front of done(), which has the second buffer to itself; its second block behind done().  Otherwise there is one tile, and done() has both buffers.  Experts' gate and up, 16 blocks, 5.5
// tiles a workgroup, with the 8-bit instructions: 208 -> 194 us; what hangs on the lane alone is computed anew in each of these parts (fresh): kept across the blocks' loop it would take 40 registers.
// A block's products (each over the wave's TN activation tiles) run without a break from block to block: a product's sums are taken in front of the one that takes its registers, TN products later.  The
// barrier at a block's end stands in front of its last product, whose operands are read by then: under it the next block's first operands come from LDS.
template <bool MANY, bool WIDE, int NSC, bool A32, class T, int WM, class Jobs, class Done> __device__ __forceinline__ void tile_run(char *smem, int jobs, Jobs job, Done done)
{
    constexpr int WROWS = T::WI * 8 * T::WAVES, AROWS = T::AI * 8 * T::WAVES, WH = T::WI / 2, FIRST = T::AI + WH + 2;          // requests of a block's first part; WH of the second
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave % WM, wn = wave / WM;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_char *)smem;
    int nb, rest;
    bool idle;
    const uint8_t *wbase, *abase;
    const float *swl, *sa;
    // the rows of product m of wave row k: wrow(k, m) on.  Which rows a wave asks for: of its WI requests of 8 rows the first WH are of the first half of somebody's products
    auto wrow = [&](int k, int m) { return NSC == 1 ? k * (WROWS / WM) + 16 * m : (m < T::TM / 2 ? 0 : WROWS / 2) + k * (WROWS / (2 * WM)) + 16 * (m % (T::TM / 2)); };
    auto w_row8 = [&](int j) {          // the first of the 8 rows of request j
        const int u = wave * WH + j % WH, k = u / T::TM, r = u % T::TM;          // (TM requests of 8 rows are half of a wave row's products)
        return wrow(k, (j / WH) * (T::TM / 2) + r / 2) + 8 * (r & 1);
    };
    uint32_t wo[T::WI], ao[A32 ? T::AI : 1];
    const uint8_t *ap[A32 ? 1 : T::AI];
    auto take = [&](const auto &J) {
        const int lane = fresh(threadIdx.x) & 63, sub = lane >> 3;
        nb = (J.cols + BLOCK - 1) / BLOCK; rest = J.cols - (nb - 1) * BLOCK; idle = J.idle; wbase = J.wbase; abase = J.abase; sa = J.sa;
        swl = J.sw(lane & (NSC - 1));
#pragma unroll
        for (int j = 0; j < T::WI; j++) { const int r = w_row8(j) + sub; wo[j] = J.woff(r) + 16 * slot_of(r, lane & 7); }
#pragma unroll
        for (int j = 0; j < T::AI; j++) {
            const int r = (wave * T::AI + j) * 8 + sub;
            if constexpr (A32) ao[j] = J.asrc(r) + 16 * slot_of(r, lane & 7);
            else ap[j] = J.asrc(r) + 16 * slot_of(r, lane & 7);
        }
    };
    // in front of the last block's requests: pieces beyond the rows' end are their last one instead
    auto draw_back = [&]() {
        const int lane = fresh(threadIdx.x) & 63, sub = lane >> 3;
        auto back = [&](int r) { return (uint32_t)max(0, 16 * slot_of(r, lane & 7) + 16 - rest); };
#pragma unroll
        for (int j = 0; j < T::WI; j++) wo[j] -= back(w_row8(j) + sub);
#pragma unroll
        for (int j = 0; j < T::AI; j++) { if constexpr (A32) ao[j] -= back((wave * T::AI + j) * 8 + sub); else ap[j] -= back((wave * T::AI + j) * 8 + sub); }
    };
    const uint32_t sc0 = lds0 + T::DATA + wave * 256;
    auto ask_first = [&](int b, int slot, int k, int on) {          // request k of FIRST of block b into buffer `slot`
        if (k == 0) request4(sa + b, sc0 + slot * T::BUF, on);
        else if (k == 1) request4(swl + b, sc0 + slot * T::BUF + T::SCALES / 2, on);
        else if (k < 2 + T::AI) {
            const int j = k - 2;
            const uint32_t to = lds0 + slot * T::BUF + WROWS * BLOCK + (wave * T::AI + j) * 1024;
            if constexpr (A32) request16(abase + (size_t)b * BLOCK, ao[j], to, on);
            else request16(ap[j] + (size_t)b * BLOCK, to, on);
        } else request16(wbase + (size_t)b * BLOCK, wo[k - 2 - T::AI], lds0 + slot * T::BUF + w_row8(k - 2 - T::AI) * BLOCK, on);
    };
    auto ask_second = [&](int b, int slot, int k, int on) { request16(wbase + (size_t)b * BLOCK, wo[WH + k], lds0 + slot * T::BUF + w_row8(WH + k) * BLOCK, on); };
    auto ask = [&](int b) {          // (in front of the blocks' loop: b < STAGES)
        if (b + 1 == nb && rest < BLOCK) draw_back();
#pragma unroll
        for (int k = 0; k < FIRST; k++) ask_first(b, b, k, 1);
#pragma unroll
        for (int k = 0; k < WH; k++) ask_second(b, b, k, 1);
    };
    auto clear = [&](int b, int slot, bool second) {          // (the last block's columns that are none; everybody's requests of this part have arrived)
        if (b + 1 < nb || rest == BLOCK) return;
        char *const buf = smem + slot * T::BUF;
        for (int k = threadIdx.x; k < (WROWS / 2 + (second ? 0 : AROWS)) * 8; k += 64 * T::WAVES) {
            const int q = k >> 3, half = WROWS / 2, u = q / 8, r = q < half ? wrow(u / T::TM, (second ? T::TM / 2 : 0) + u % T::TM / 2) + 8 * (u & 1) + (q & 7) : WROWS + q - half;
            if (16 * (k & 7) >= rest) *reinterpret_cast<u32x4 *>(buf + r * BLOCK + 16 * slot_of(r < WROWS ? r : r - WROWS, k & 7)) = u32x4{0u, 0u, 0u, 0u};
        }
        lds_barrier();
    };
    int i, piece;          // (a product's rows start at multiples of 16: their slots are those of 0 .. 15)
    auto read = [&](const char *rows16) {      // the lane's pieces g and g + 4 of its row
        Operand<WIDE> o;
        o.set(*reinterpret_cast<const u32x4 *>(rows16 + piece), *reinterpret_cast<const u32x4 *>(rows16 + (piece ^ 64)));
        return o;
    };
    f32x4 acc[T::TM][T::TN];
    Operand<WIDE> av[T::TN], wq[2];          // (a product's matrix rows are asked for two products ahead)
    f32x4 p[T::TN];
    float s[NSC][T::TN], last[T::TN];          // the scales of this block and, for its last product, of the one before
    auto read_scales = [&](int slot) {
        const float *at = reinterpret_cast<const float *>(smem + slot * T::BUF + T::DATA + wave * 256);
#pragma unroll
        for (int h = 0; h < NSC; h++)
#pragma unroll
            for (int j = 0; j < T::TN; j++) s[h][j] = at[16 * j + i] * at[T::SCALES / 8 + h];
    };
    auto add = [&](int m, int j, float f) {
#pragma unroll
        for (int r = 0; r < 4; r++) acc[m][j][r] = fmaf(p[j][r], f, acc[m][j][r]);
        asm volatile("" : "+v"(acc[m][j]));          // (here: the compiler takes them behind the next branch otherwise, the products kept in registers until then)
    };
    const int arow = WROWS * BLOCK + wn * T::TN * 16 * BLOCK;
    constexpr int YOUNGER = (T::STAGES - 1) * (FIRST + WH);          // requests behind those that a barrier waits for, as long as there are blocks to ask for
    auto sums = [&]() {
        i = fresh(threadIdx.x) & 15;
        piece = i * BLOCK + 16 * slot_of(i, (fresh(threadIdx.x) & 63) >> 4);
        if (nb >= T::STAGES) arrive<YOUNGER>(); else arrive<0>();
        clear(0, 0, false);
        clear(0, 0, true);
        int slot = 0;
        if (idle) {
            for (int b = 0; b < nb; b++) {
                const int next = slot + 1 == T::STAGES ? 0 : slot + 1, more = b + T::STAGES < nb;
                if (b + T::STAGES - 1 < nb) arrive<YOUNGER>(); else arrive<0>();
                if (b > 0) clear(b, slot, true);
                if (b + T::STAGES + 1 == nb && rest < BLOCK) draw_back();
#pragma unroll
                for (int k = 0; k < FIRST; k++) ask_first(b + T::STAGES, slot, k, more);
                if (more) arrive<YOUNGER>();
                else if (b + 1 < nb) { arrive<WH>(); clear(b + 1, next, false); }
#pragma unroll
                for (int k = 0; k < WH; k++) ask_second(b + T::STAGES, slot, k, more);
                slot = next;
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < T::TN; j++) av[j] = read(smem + arow + 16 * j * BLOCK);
        wq[0] = read(smem + wrow(wm, 0) * BLOCK);
        wq[1] = read(smem + wrow(wm, 1) * BLOCK);
        read_scales(0);
#pragma unroll
        for (int j = 0; j < T::TN; j++) { last[j] = 0.0f; p[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f}; }
        // Product m reads the rows of product m + 2 behind itself; the middle of a block is MID, where the first half's rows are read and the second's are about to be, its end END, the same the other way
        // round (their barriers stand inside the products, so that the reads before have time to arrive).  Between MID and END the requests of a block's first part go out, one beside a product, behind
        // END those of the second.
        constexpr int MID = T::TM / 2 - 2, END = T::TM - 2, SLOTS = (END - MID - 1) * T::TN, EACH = (FIRST + SLOTS - 1) / SLOTS, EACH2 = (WH + T::TN - 1) / T::TN;
        for (int b = 0; b < nb; b++) {
            const int next = slot + 1 == T::STAGES ? 0 : slot + 1;
            const char *const cur = smem + slot * T::BUF, *const nxt = smem + next * T::BUF;
            const int more = b + T::STAGES < nb;
#pragma unroll
            for (int m = 0; m < T::TM; m++) {
                const Operand<WIDE> wv = wq[m & 1];
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < T::TN; j++) {
                    if (m == MID && j == T::TN / 2) {          // the block's second part is there; its first one is read, scales and activations too
                        if (b + T::STAGES - 1 < nb) arrive<YOUNGER>(); else arrive<0>();
                        if (b > 0) clear(b, slot, true);
                        if (b + T::STAGES + 1 == nb && rest < BLOCK) draw_back();
                    }
                    if (m == END && j == T::TN / 2) {          // the next block's first part is there; this one's second is read
                        if (b + T::STAGES < nb) arrive<YOUNGER>();
                        else if (b + 1 < nb) { arrive<WH>(); clear(b + 1, next, false); }
                    }
                    if (m > 0) add(m - 1, j, s[m - 1 < T::TM / 2 ? 0 : NSC - 1][j]);
                    else add(T::TM - 1, j, last[j]);
                    p[j] = mfma128(wv, av[j]);
                    if (m + 1 == T::TM) av[j] = read(nxt + arow + 16 * j * BLOCK);          // (behind the last block: what is there, not used)
                    if (j == T::TN - 1) wq[m & 1] = m + 2 < T::TM ? read(cur + wrow(wm, m + 2) * BLOCK) : read(nxt + wrow(wm, m + 2 - T::TM) * BLOCK);
                    if (m > MID && m < END) {
#pragma unroll
                        for (int k = ((m - MID - 1) * T::TN + j) * EACH; k < ((m - MID - 1) * T::TN + j + 1) * EACH; k++) if (k < FIRST) ask_first(b + T::STAGES, slot, k, more);
                    } else if (m > END) {
#pragma unroll
                        for (int k = ((m - END - 1) * T::TN + j) * EACH2; k < ((m - END - 1) * T::TN + j + 1) * EACH2; k++) if (k < WH) ask_second(b + T::STAGES, slot, k, more);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
#pragma unroll
            for (int j = 0; j < T::TN; j++) last[j] = s[NSC - 1][j];
            read_scales(next);
            slot = next;
        }
#pragma unroll
        for (int j = 0; j < T::TN; j++) add(T::TM - 1, j, last[j]);
    };
    auto J = job(0);
    take(J);
    ask(0);
    if (nb > 1) ask(1);
    for (int k = 0;;) {
#pragma unroll
        for (int m = 0; m < T::TM; m++)
#pragma unroll
            for (int j = 0; j < T::TN; j++) acc[m][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        sums();
        lds_barrier();          // (everybody has read the last block)
        if constexpr (!MANY) { done(J, acc, smem); break; }
        const bool more = ++k < jobs;
        const auto now = J;
        if (more) { J = job(k); take(J); ask(0); }
        done(now, acc, smem + T::BUF);
        if (!more) break;
        lds_barrier();          // (done() has read its buffer)
        if (nb > 1) ask(1);
    }
}

// A wave's sums by way of LDS, so that they leave in whole lines: f(t, n, v) with N consecutive values of activation row t from matrix row n on (both counted from the wave's first).  Every wave
// has its part of the buffers.
template <class T, bool MANY, int N, class F> __device__ __forceinline__ void tile_out(char *buffer, const f32x4 (&acc)[T::TM][T::TN], F f)
{
    constexpr int PART = (MANY ? T::OUT : T::SMEM) / T::WAVES / 1024 * 1024, ROW = T::TM * 64, ROWS = PART / ROW / 16 * 16 < T::TN * 16 ? PART / ROW / 16 * 16 : T::TN * 16, PIECES = T::TM * 4;      // 16-byte pieces a row
    static_assert(ROWS >= 16 && (PIECES & (PIECES - 1)) == 0 && PIECES >= 16, "a part of 16 rows at least");
    const int lane = fresh(threadIdx.x) & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    char *const part = buffer + wave * PART;
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
            if constexpr (N == 1) v[0] = *reinterpret_cast<const float *>(part + t * ROW + 16 * ((c >> 2) ^ (t & 15)) + 4 * (c & 3));
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

// Workgroups are dealt to the eight XCDs in turn; each XCD has a range of the `all` places, so that it works on neighbouring tiles whose operands its L2 shares, and its workgroups take them in turn
struct Share {
    int first, count, each;          // this workgroup's places: first + k each, k < count
    __device__ __forceinline__ Share(int all)
    {
        const int xcd = blockIdx.x & 7, rank = blockIdx.x >> 3, q = all >> 3, r = all & 7, mine = q + (xcd < r), from = xcd * q + min(xcd, r);
        each = ((int)gridDim.x - xcd + 7) >> 3;          // workgroups of the XCD
        first = from + rank;
        count = rank < mine ? (mine - rank + each - 1) / each : 0;
    }
    __device__ __forceinline__ int at(int k) const { return first + k * each; }
};

} // namespace ifa8
