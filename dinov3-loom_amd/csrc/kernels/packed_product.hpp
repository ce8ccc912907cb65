// The products of the feed-forward half of a packed block
// (include/dinov3_packed.h): rows of x times rows of one or two weight matrices,
// in 16 bits or in 4 with a scale per 32 values, with a bias, or gated (act(g) u of
// the two). One tile kernel in bytes: a piece of 16 bytes of a row is 8 values
// or a block of 32, a stage in LDS holds 8 pieces of each of a tile's rows, and a
// matrix instruction (32 x 32 outputs, either way 8 passes) takes one piece per
// lane of each side.
#pragma once
#include <type_traits>
#include <algorithm>

#include "packed_four.hpp"

namespace dhx {

// What a launcher hands on; strides are in bytes but that of out. xs_stride: from 32
// blocks' scales of all rows to the next 32's.
struct Product {
    uint32_t activation, rows, pieces, outputs, sequences;
    const void *x, *w, *up;             // up: gated only
    const void *xs, *ws, *us;           // scales: 4-bit only
    const float *bias, *up_bias;
    void* out;
    const int32_t* starts;
    uint64_t x_stride, w_stride, xs_stride, ws_stride, out_stride;
};

#define DHX_PRODUCT_PARAMS Addr x_, Addr w_, Addr up_, int rows, int pieces, int outputs, uint32_t x_stride, uint32_t w_stride, Addr starts_, Addr xs_, Addr ws_, Addr us_, Addr bias_, Addr up_bias_, Addr out_, uint64_t out_stride, int sequences, int activation, uint64_t xs_stride, uint32_t ws_stride

template <class K>
hipError_t enqueue_product(K kernel, dim3 grid, dim3 block, hipStream_t s, const Product& p) {
    return enqueue(kernel, grid, block, 0, s, p.x, p.w, p.up, (int)p.rows, (int)p.pieces, (int)p.outputs, (uint32_t)p.x_stride,
                   (uint32_t)p.w_stride, p.starts, p.xs, p.ws, p.us, p.bias, p.up_bias, p.out, p.out_stride, (int)p.sequences,
                   (int)p.activation, p.xs_stride, (uint32_t)p.ws_stride);
}

// --- device pieces ---------------------------------------------------------

typedef int int8v_t __attribute__((ext_vector_type(8)));

// Products of one piece per lane of each side. Four bits: scale byte KK of a lane's
// word is its piece's.
template <class T, bool FOUR, int KK>
__device__ __forceinline__ float16_t product32(uint4_t a, uint4_t b, float16_t c, uint32_t a_scale, uint32_t b_scale) {
    if constexpr (FOUR) {
        const int8v_t wide_a = {(int)a[0], (int)a[1], (int)a[2], (int)a[3]}, wide_b = {(int)b[0], (int)b[1], (int)b[2], (int)b[3]};
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide_a, wide_b, c, 4, 4, KK, (int)a_scale, KK, (int)b_scale);
    } else {
        typedef typename Num<T>::v8 v8;
        return Num<T>::mfma(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c);
    }
}

// The same with 16 x 16 outputs, of 4 bits; the scale is a word's lowest byte.
__device__ __forceinline__ float4_t product16(uint4_t a, uint4_t b, float4_t c, uint32_t a_scale, uint32_t b_scale) {
    const int8v_t wide_a = {(int)a[0], (int)a[1], (int)a[2], (int)a[3]}, wide_b = {(int)b[0], (int)b[1], (int)b[2], (int)b[3]};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide_a, wide_b, c, 4, 4, 0, (int)a_scale, 0, (int)b_scale);
}

// The lane's number, from no register that would have to hold it.
__device__ __forceinline__ int lane_anew() {
    int lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    asm volatile("" : "+v"(lane));
    return lane;
}

template <int ACT>
__device__ __forceinline__ float activated(float g) {
    // e^-g past the range of float32 is infinite, and its reciprocal 0.
    if constexpr (ACT == DHX_SILU) return g * fast_rcp(1.0f + fast_exp2(-kLog2e * g));
    if constexpr (ACT == DHX_SIGMOID) return fast_rcp(1.0f + fast_exp2(-kLog2e * g));
    if constexpr (ACT == DHX_RELU) return g < 0.0f ? 0.0f : g;  // NaN stays
    if constexpr (ACT == DHX_GELU) {
        // g (1 + erf x) / 2 = max(g, 0) - |g| erfc(|x|) / 2, x = g / sqrt 2: no difference of near
        // values where g is negative, so what is left there is as exact as erfc is: e^(-x^2)
        // times a polynomial in 1 / (1 + c |g|), fitted to |g| <= 14 with a relative error of at
        // most 1.5e-7 near 0 and 5e-5, a tenth of half a step of f16, far from it. (2299 rows, 1000 ->
        // 2728 with 4-bit weights 17.5 us; with a step more, which leaves 1.6e-6, 17.8; with
        // Abramowitz and Stegun's formula 7.1.26, a step less and 1e-2 off at -8, 17.35; erff
        // took 3 us more than that.)
        const float t = fast_rcp(fmaf(0.29225f, fabsf(g), 1.0f));
        float p = fmaf(fmaf(-0.0862025083f, t, 0.268044585f), t, -0.0729217612f);
        p = fmaf(fmaf(fmaf(p, t, 0.169077223f), t, 0.104507711f), t, 0.117494752f);
        const float half = p * t * fast_exp2(-0.5f * kLog2e * g * g);
        return fmaf(-fabsf(g), half, fmaxf(g, 0.0f));
    }
    // (1 + tanh u) / 2 = 1 / (1 + e^-2u), 2 sqrt(2 / pi) = 1.5957691
    if constexpr (ACT == DHX_GELU_TANH) return g * fast_rcp(1.0f + fast_exp2(-kLog2e * 1.5957691f * fmaf(0.044715f * g * g, g, g)));
}

// f(activation as a constant) for the activation of the call.
template <class F>
__device__ __forceinline__ void with_activation(int activation, F f) {
    switch (activation) {
        case DHX_SILU: f(std::integral_constant<int, DHX_SILU>{}); break;
        case DHX_GELU: f(std::integral_constant<int, DHX_GELU>{}); break;
        case DHX_GELU_TANH: f(std::integral_constant<int, DHX_GELU_TANH>{}); break;
        case DHX_RELU: f(std::integral_constant<int, DHX_RELU>{}); break;
        default: f(std::integral_constant<int, DHX_SIGMOID>{});
    }
}

// Tile of BM rows of x and BN rows of weights (gated: 32 of gate, 32 of up in turn,
// so that a lane holds both sums of an output), waves of WM x WN each. NST stages
// of 8 pieces in LDS, NST - 1 of them on their way while one is multiplied (a
// variable each, so that the compiler can tell the stage that is read from those
// being filled: one that may be both would make each read wait for all loads). A
// lane multiplies piece 4 (lane / 32) + kk in step kk: a block of 4 bits then finds
// its scale in byte kk of the half's own word of the row's 8. Scales come 32 bytes
// per row at a time, for four stages, with the first of them (16 bytes at a time a
// row's line would be asked for twice as often: 16384 rows, 4096 -> 4096, take 199 us
// then, 190 so). Those of x lie [32 blocks][row][32], so that a load's rows are one piece.
template <class T, bool FOUR, bool GATED, int BM, int BN, int WM, int WN, int NST, int PER_SIMD>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN), PER_SIMD) void packed_product_kernel(DHX_PRODUCT_PARAMS) {
    typedef typename Num<T>::v4 v4;
    constexpr int WAVES = (BM / WM) * (BN / WN), THREADS = 64 * WAVES;
    constexpr int XL = BM / 8 / WAVES, WL = BN / 8 / WAVES;  // loads of 8 rows per wave and stage
    constexpr int SCALE_LOADS = (BM + BN) / 32, SL = FOUR ? (SCALE_LOADS + WAVES - 1) / WAVES : 0;  // per wave and four stages
    constexpr int MB = WM / 32, NB = WN / 32, KK = 4;
    // Turns of four stages end after two where those are the last, but in the largest
    // tile (with four bits), whose registers do not fit then: up to three stages of zeros
    // are multiplied there.
    constexpr int TURNS = FOUR || NST == 4 ? 4 : 2;
    constexpr bool BREAK = MB * NB < 8;
    constexpr int BO = GATED ? BN / 2 : BN;  // outputs of a tile
    constexpr int WS = BM * 128, SS = WS + BN * 128, STAGE = SS + (FOUR ? (BM + BN) * 32 : 0);  // x, weights, scales
    static_assert(NST == 2 || NST == 4, "which of two stages a buffer holds is a constant");
    static_assert(XL * 8 * WAVES == BM && WL * 8 * WAVES == BN && BM % 64 == 0 && BN % 64 == 0 && BN <= THREADS, "whole loads");
    static_assert(!GATED || NB % 2 == 0, "both sums of an output in one lane");
    __shared__ __attribute__((aligned(16))) char s0[STAGE], s1[SS], s2[NST > 2 ? SS : 16], s3[NST > 2 ? SS : 16];
    __shared__ __attribute__((aligned(16))) float sBias[BN];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Tiles in XCD-contiguous order, four row blocks at a time, so that the tiles
    // that an XCD has under way share rows of x and rows of weights in its L2.
    const int n_tiles = (outputs + BO - 1) / BO, total = n_tiles * ((rows + BM - 1) / BM);
    const int per = (total + 7) >> 3, g = blockIdx.x, t = (g & 7) * per + (g >> 3);
    if ((g >> 3) >= per || t >= total) return;
    constexpr int GROUP = 4;
    const int block = t / (GROUP * n_tiles), in_block = t - block * GROUP * n_tiles;
    const int tall = min(GROUP, total / n_tiles - block * GROUP), across = in_block / tall;
    const int row0 = (block * GROUP + in_block - across * tall) * BM, col0 = across * BO;
    int first = 0, end = rows;  // the rows that count
    if (starts_.a) {
        first = start_at(starts_, 0, rows);
        end = start_at(starts_, sequences, rows);
        if (row0 >= end || row0 + BM <= first) return;
    }
    const int steps = (pieces + 7) / 8;

    // Weight row r of the tile: which matrix, and which of its rows.
    auto of_up = [&](int r) { return GATED && (r & 32) != 0; };
    auto column = [&](int r) { return GATED ? (r >> 6) * 32 + (r & 31) : r; };
    // Buffers of the tile's rows: a load's address is one register per lane and one
    // of the wave, and a lane beyond the end fetches zeros. A wave loads rows of one
    // of the matrices.
    static_assert(!GATED || 32 % (WL * 8) == 0, "of gate or of up");
    const int columns = min(BO, outputs - col0);
    auto rows_of = [&](Addr base, int row, int n, uint32_t stride) {
        return __builtin_amdgcn_make_buffer_rsrc((void*)(base.a + (uint64_t)row * stride), 0, (int)((uint32_t)(n - 1) * stride + pieces * 16),
                                                 kBufferRsrcWord3);
    };
    const __amdgpu_buffer_rsrc_t x_rows = rows_of(x_, row0, min(BM, rows - row0), x_stride);
    const __amdgpu_buffer_rsrc_t w_rows = rows_of(of_up(wave * WL * 8) ? up_ : w_, col0, columns, w_stride);

    // Lane -> row lane / 8 of a load's 8, the piece that the swizzle puts at slot
    // lane % 8; rows behind the last one fetch that one.
    uint32_t xo[XL], wo[WL];
    const int l32 = lane & 31, hi = lane >> 5;
#pragma unroll
    for (int j = 0; j < XL; ++j) {
        const int r = (wave * XL + j) * 8 + (lane >> 3);
        xo[j] = (uint32_t)min(r, rows - 1 - row0) * x_stride + ((lane & 7) ^ slot_of<64>(r)) * 16;
    }
#pragma unroll
    for (int j = 0; j < WL; ++j) {
        const int r = (wave * WL + j) * 8 + (lane >> 3);
        wo[j] = (uint32_t)min(column(r), columns - 1) * w_stride + ((lane & 7) ^ slot_of<64>(r)) * 16;
    }
    // A load of scales takes the 32 bytes (four stages) of 32 rows, those of x first;
    // with more waves than loads some are made twice, so that every wave has as many
    // on their way. A row's halves change places every 8 rows, which spreads the reads
    // over the banks.
    const char* so[SL > 0 ? SL : 1];
    int sto[SL > 0 ? SL : 1];
    const int half = (lane & 1) ^ ((lane >> 4) & 1);
    if constexpr (FOUR) {
#pragma unroll
        for (int j = 0; j < SL; ++j) {
            const int load = (wave * SL + j) % SCALE_LOADS, r = load * 32 + (lane >> 1);
            sto[j] = load * 1024;
            if (r < BM) {
                so[j] = (const char*)xs_ + (uint64_t)(row0 + min(r, rows - 1 - row0)) * 32 + half * 16;
            } else {
                const int c = col0 + min(column(r - BM), columns - 1);
                so[j] = (of_up(r - BM) ? (const char*)us_ : (const char*)ws_) + (uint64_t)c * ws_stride + half * 16;
            }
        }
    }
    auto move_scales = [&](int s) __attribute__((always_inline)) {
        if constexpr (FOUR) {
            const int group = min(s, steps - 1) >> 2;
            const bool there = group * 32 + half * 16 < pieces;  // a row of weights' may end between
#pragma unroll
            for (int j = 0; j < SL; ++j) {
                const uint64_t step = sto[j] < BM * 32 ? (uint64_t)group * xs_stride : (uint64_t)(group * 32);
                dma16(there ? so[j] + step : (const char*)&kZeros, s0 + SS + sto[j]);
            }
        }
    };
    auto buffer_load = [](const __amdgpu_buffer_rsrc_t& from, char* to, uint32_t lane_at, int at) __attribute__((always_inline)) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)to, 16, (int)lane_at, at, 0, 0);
    };
    // Stage s, also the last one, whose pieces may not all exist, and stages behind
    // it, which have none: such lanes pass the buffer's end and fetch zeros. (One code
    // for all stages: with the tail apart its registers did not fit.) turn: s % 4, a
    // constant.
    static_assert(XL % 2 == 0 || XL == 1, "rows 16 apart have their pieces at the same slots");
    auto chunk = [&](int j) { return (lane & 7) ^ slot_of<64>((j & 1) * 8 + (lane >> 3)); };
    const int chunk_x = chunk(wave * XL), chunk_w = chunk(wave * WL);  // of a wave's even loads; bit 1 differs in odd ones
    // Load n of a wave's XL + WL of a stage, the scales with the first.
    auto move_one = [&](char* to, int s, int turn, int n) __attribute__((always_inline)) {
        const int left = pieces - s * 8;
        if (n == 0 && turn == 0) move_scales(s);
        if (n < XL) buffer_load(x_rows, to + (wave * XL + n) * 1024, (chunk_x ^ (n & 1) * 2) < left ? xo[n < XL ? n : 0] : ~15u, s * 128);
        const int j = n - XL;
        if (j >= 0)
            buffer_load(w_rows, to + WS + (wave * WL + j) * 1024, (chunk_w ^ (j & 1) * 2) < left ? wo[j >= 0 ? j : 0] : ~15u, s * 128);
    };
    auto move = [&](char* to, int s, int turn) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < XL + WL; ++n) move_one(to, s, turn, n);
    };

    const int wm = wave / (BN / WN) * WM, wn = wave % (BN / WN) * WN;
    const int frag = l32 * 128 + (((hi * 4) ^ slot_of<64>(l32)) << 4);
    float16_t acc[MB][NB] = {};
    uint4_t fx[2][MB], fw[2][NB];
    // Fragment n of MB + NB.
    auto load_one = [&](const char* from, int kk, int set, int n) __attribute__((always_inline)) {
        const int at = frag ^ (kk << 4);
        if (n < MB) fx[set][n < MB ? n : 0] = *(const uint4_t*)(from + (wm + n * 32) * 128 + at);
        else fw[set][n < MB ? 0 : n - MB] = *(const uint4_t*)(from + WS + (wn + (n - MB) * 32) * 128 + at);
    };
    auto load = [&](const char* from, int kk, int set) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < MB + NB; ++n) load_one(from, kk, set, n);
    };
    // The scales of stage s: two stages in a ring take them from LDS stage by stage,
    // four take those of four stages at once, since their place is filled anew before
    // the last of them. Their places are kept from the compiler, which would read two
    // at once: such a read, unlike the others, it lets wait for all loads.
    constexpr int SETS = NST == 2 ? 2 : 4;
    uint32_t scale_x[SETS][MB], scale_w[SETS][NB];
    int scale_at[MB + NB];
    if constexpr (FOUR) {
#pragma unroll
        for (int i = 0; i < MB + NB; ++i) {
            scale_at[i] = SS + ((i < MB ? wm + i * 32 : BM + wn + (i - MB) * 32) + l32) * 32 + ((lane >> 3) & 1) * 16 + (NST == 2 ? hi * 4 : 0);
            asm volatile("" : "+v"(scale_at[i]));
        }
    }
    // Behind the last piece there are no scales (and zeros for values).
    auto scale_mask = [&](int s) __attribute__((always_inline)) {
        const int left = pieces - s * 8 - hi * 4;
        return left >= 4 ? ~0u : (1u << (8 * max(left, 0))) - 1;
    };
    auto put_scale = [&](int i, int set, uint32_t v) __attribute__((always_inline)) {
        if (i < MB) scale_x[set][i] = v;
        else scale_w[set][i - MB] = v;
    };
    auto load_scales = [&](int s, int turn) __attribute__((always_inline)) {
        if constexpr (FOUR && NST == 2) {
            const uint32_t mask = scale_mask(s);
#pragma unroll
            for (int i = 0; i < MB + NB; ++i)
                put_scale(i, turn & 1, *(const uint32_t*)(s0 + (scale_at[i] ^ ((turn & 2) * 8)) + (turn & 1) * 8) & mask);
        }
        if constexpr (FOUR && NST == 4) {
#pragma unroll
            for (int i = 0; i < MB + NB; ++i)
#pragma unroll
                for (int pair = 0; pair < 2; ++pair) {
                    const uint4_t v = *(const uint4_t*)(s0 + (scale_at[i] ^ (pair * 16)));
                    put_scale(i, 2 * pair, (hi ? v[1] : v[0]) & scale_mask(s + 2 * pair));
                    put_scale(i, 2 * pair + 1, (hi ? v[3] : v[2]) & scale_mask(s + 2 * pair + 1));
                }
        }
    };
    // The products of step kk; between them the reads of the next step's fragments, in
    // the first half, and loads d0 .. d1-1 of a stage. (With all reads and loads in front
    // of the products the matrix units wait while they are issued: gated, 12864 rows, 384
    // -> 1536, 44.8 us, so 38.1; linear, 4 bits, 16384 rows, 4096 -> 4096, 186 and 172;
    // loads only between the products 42.0 and 178.)
    auto multiply = [&](auto kk, int scales, auto read, auto fetch, int d0, int d1) __attribute__((always_inline)) {
        constexpr int STEP = decltype(kk)::value, N = MB * NB, HALF = (N + 1) / 2;
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int k = 0; k < NB; ++k) {
                const int m = i * NB + k;
                acc[i][k] = product32<T, FOUR, STEP>(fw[STEP & 1][k], fx[STEP & 1][i], acc[i][k], FOUR ? scale_w[scales][k] : 0, FOUR ? scale_x[scales][i] : 0);
                __builtin_amdgcn_sched_barrier(0);
                if (m < HALF) {
#pragma unroll
                    for (int r = m * (MB + NB) / HALF; r < (m + 1) * (MB + NB) / HALF; ++r) read(r);
                }
#pragma unroll
                for (int n = d0 + m * (d1 - d0) / N; n < d0 + (m + 1) * (d1 - d0) / N; ++n) fetch(n);
                __builtin_amdgcn_sched_barrier(0);
            }
    };
    move(s0, 0, 0);
    if (tid < BN) {
        const float* bias = of_up(tid) ? up_bias_ : bias_;
        sBias[tid] = bias && col0 + column(tid) < outputs ? bias[col0 + column(tid)] : 0.f;
    }
    if constexpr (NST > 2) {
        move(s1, 1, 1);
        move(s2, 2, 0);
    }
    // Opens stage s: it has landed (the NST - 2 stages behind it may be on their way,
    // with their scales), and every wave has read the one before, whose place stage
    // s + NST - 1 takes. turn: s % 4, a constant.
    auto open = [&](auto turn) __attribute__((always_inline)) {
        constexpr int TURN = decltype(turn)::value;
        wait_vm<(NST - 2) * (XL + WL) + (NST == 4 && TURN >= 2 ? SL : 0)>();
        wait_lgkm();
        barrier();
    };
    // Multiplies a stage; the next one's first fragments are read between its last
    // products, and the loads of the stage that takes its place begin there too, in
    // large tiles the half of them (in small ones that gained nothing).
    constexpr int ALL = XL + WL, FIRST = MB * NB >= 4 ? ALL / 2 : ALL;
    auto step = [&](auto turn, char* before, char* now, const char* next, int s) __attribute__((always_inline)) {
        constexpr int TURN = decltype(turn)::value, SET = NST == 2 ? TURN & 1 : TURN, NEXT = (TURN + 1) & 3;
        auto read = [&](const char* from, int kk) { return [&, from, kk](int r) __attribute__((always_inline)) { load_one(from, kk, kk & 1, r); }; };
        auto fetch = [&](char* to, int ahead) {
            return [&, to, ahead](int n) __attribute__((always_inline)) { move_one(to, s + ahead, (TURN + ahead) & 3, n); };
        };
        if (NST == 2 && (TURN & 1) == 0) load_scales(s + 1, TURN + 1);
        multiply(std::integral_constant<int, 0>{}, SET, read(now, 1), fetch(before, NST - 1), FIRST, ALL);
        multiply(std::integral_constant<int, 1>{}, SET, read(now, 2), [](int) {}, 0, 0);
        multiply(std::integral_constant<int, 2>{}, SET, read(now, 3), [](int) {}, 0, 0);
        open(std::integral_constant<int, NEXT>{});
        if (NST == 2 && (TURN & 1) == 1) load_scales(s + 1, NEXT);
        multiply(std::integral_constant<int, 3>{}, SET, read(next, 0), fetch(now, NST), 0, FIRST);
        if (NST == 4 && TURN == 3) load_scales(s + 1, 0);
    };
    open(std::integral_constant<int, 0>{});
#pragma unroll
    for (int n = 0; n < FIRST; ++n) move_one(NST == 2 ? s1 : s3, NST - 1, NST - 1, n);
    load(s0, 0, 0);
    load_scales(0, 0);
    for (int s = 0; s < steps; s += TURNS) {  // an odd number of stages: one of zeros behind them
        step(std::integral_constant<int, 0>{}, NST > 2 ? s3 : s1, s0, s1, s);
        step(std::integral_constant<int, 1>{}, s0, s1, NST > 2 ? s2 : s0, s + 1);
        if constexpr (TURNS > 2) {
            if (BREAK && s + 2 >= steps) break;
            step(std::integral_constant<int, 2>{}, s1, NST > 2 ? s2 : s0, NST > 2 ? s3 : s1, s + 2);
            step(std::integral_constant<int, 3>{}, NST > 2 ? s2 : s0, NST > 2 ? s3 : s1, s0, s + 3);
        }
    }
    wait_vm<0>();  // no load may come when the LDS holds outputs, or is another workgroup's
    barrier();

    // Lane: row l32 of a block, columns 8 g + 4 hi .. +3 of its 32 in register group
    // g; both halves exchange groups, so that each holds 8 columns at once. A wave's
    // 32 rows go through its own part of the LDS, from where they are stored as whole
    // lines, through the L2 as WtOut's (common.hpp). us, 32-byte pieces straight from
    // registers, whole lines, and those through the L2: linear, 4 bits, 16384 rows, 4096 ->
    // 4096, 192, 180, 178; gated, 12864 rows, 384 -> 1536, 46.6, 44.1, 41.7, 2299 rows, 1000
    // -> 2728 with 4 bits 20.7, 20.6, 18.5. (Pieces through the L2 257, 52.6 and 19.5.)
    constexpr int ROW = (GATED ? WN / 2 : WN) * 2, PITCH = ROW + 16, LANES = ROW / 16;  // bytes; lanes of a stored row
    static_assert(WAVES * 32 * PITCH <= SS, "the first stage's buffer holds them");
    char* const mine = s0 + wave * 32 * PITCH;
    const uint32_t out_bytes = (uint32_t)out_stride * 2;
    const __amdgpu_buffer_rsrc_t out_rows = __builtin_amdgcn_make_buffer_rsrc(
        (void*)(out_.a + (uint64_t)row0 * out_bytes), 0, (int)((uint32_t)(min(BM, rows - row0) - 1) * out_bytes + outputs * 2), kBufferRsrcWord3);
    auto bias4 = [&](int k, int g) { return *(const float4_t*)(sBias + wn + k * 32 + 8 * g + 4 * hi); };
    auto put = [&](int column, v4 lo, v4 up) __attribute__((always_inline)) {
        *(half8_t*)(mine + l32 * PITCH + (column + hi * 8) * 2) = frag_swap(__builtin_bit_cast(half4_t, lo), __builtin_bit_cast(half4_t, up));
    };
    auto store = [&](int i) __attribute__((always_inline)) {
        wave_lds_sync();
#pragma unroll
        for (int j = 0; j < 32 * LANES / 64; ++j) {
            const int r = j * (64 / LANES) + lane / LANES, row = row0 + wm + i * 32 + r;
            const int col = col0 + (GATED ? wn / 2 : wn) + lane % LANES * 8;
            const bool there = row >= first && row < end && col < outputs;
            const uint32_t at = there ? (uint32_t)(row - row0) * out_bytes + col * 2 : ~15u;  // past the end: not stored
            const uint4_t piece = *(const uint4_t*)(mine + r * PITCH + lane % LANES * 16);
            constexpr int kSc1 = 16;
            __builtin_amdgcn_raw_buffer_store_b128(piece, out_rows, (int)at, 0, kSc1);
        }
        wave_lds_sync();
    };
    auto rounded = [](float4_t v) {
        v4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (T)v[e];
        return o;
    };
    auto group = [](const float16_t& v, int g) { return float4_t{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]}; };
    if constexpr (GATED) {
        with_activation(activation, [&](auto act) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < MB; ++i) {
#pragma unroll
                for (int k = 0; k < NB; k += 2)
#pragma unroll
                    for (int kk = 0; kk < 2; ++kk) {
                        v4 o[2];
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const float4_t a = group(acc[i][k], 2 * kk + q) + bias4(k, 2 * kk + q);
                            float4_t u = group(acc[i][k + 1], 2 * kk + q) + bias4(k + 1, 2 * kk + q);
#pragma unroll
                            for (int e = 0; e < 4; ++e) u[e] *= activated<decltype(act)::value>(a[e]);
                            o[q] = rounded(u);
                        }
                        put(k * 16 + kk * 16, o[0], o[1]);
                    }
                store(i);
            }
        });
    } else {
#pragma unroll
        for (int i = 0; i < MB; ++i) {
#pragma unroll
            for (int k = 0; k < NB; ++k)
#pragma unroll
                for (int kk = 0; kk < 2; ++kk)
                    put(k * 32 + kk * 16, rounded(group(acc[i][k], 2 * kk) + bias4(k, 2 * kk)), rounded(group(acc[i][k], 2 * kk + 1) + bias4(k, 2 * kk + 1)));
            store(i);
        }
    }
}

template <class T, bool FOUR, bool GATED, int BM, int BN, int WM, int WN, int NST, int PER_SIMD>
hipError_t launch_tiles(const Product& p, hipStream_t s) {
    constexpr uint64_t BO = GATED ? BN / 2 : BN;
    const uint64_t total = ((uint64_t)p.rows + BM - 1) / BM * ((p.outputs + BO - 1) / BO);
    return enqueue_product(packed_product_kernel<T, FOUR, GATED, BM, BN, WM, WN, NST, PER_SIMD>, dim3((unsigned)((total + 7) / 8 * 8)),
                           dim3(64 * (BM / WM) * (BN / WN)), s, p);
}

// The end of a workgroup of few rows: its waves' parts of 16 outputs of 16 XB rows from
// row0 on are joined in LDS, and the rows in first .. end-1 are stored. A lane's part:
// row 16 m + lane % 16, columns 4 (lane / 16) .. +3.
constexpr int kFewProductWaves = 8;
template <class T, bool GATED, int XB>
__device__ __forceinline__ void store_few(float (*sum)[kFewProductWaves][16 * XB][20], const float4_t (*acc)[XB], int col0, int row0, int first,
                                          int end, int outputs, int activation, Addr bias_, Addr up_bias_, Addr out_, uint64_t out_stride) {
    constexpr int AB = GATED ? 2 : 1;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
#pragma unroll
    for (int a = 0; a < AB; ++a)
#pragma unroll
        for (int m = 0; m < XB; ++m) *(float4_t*)&sum[a][wave][m * 16 + (lane & 15)][4 * (lane >> 4)] = acc[a][m];
    lds_barrier();
    const int r = tid >> 2, row = row0 + r, c = (tid & 3) * 4, col = col0 + c;
    if (r < 16 * XB && row >= first && row < end && col < outputs) {
        float4_t v[AB] = {};
#pragma unroll
        for (int a = 0; a < AB; ++a) {
#pragma unroll
            for (int i = 0; i < kFewProductWaves; ++i) v[a] += *(const float4_t*)&sum[a][i][r][c];
            const float* bias = a ? up_bias_ : bias_;
            if (bias) v[a] += *(const float4_t*)(bias + col);
        }
        typename Num<T>::v4 o;
        if constexpr (GATED) {
            with_activation(activation, [&](auto act) __attribute__((always_inline)) {
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = (T)(v[1][e] * activated<decltype(act)::value>(v[0][e]));
            });
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (T)v[0][e];
        }
        *(typename Num<T>::v4*)((T*)out_ + (uint64_t)row * out_stride + col) = o;
    }
}

// Few rows against 4-bit weights, which are all there is to read: a workgroup takes
// 16 outputs at a time (gated: and both of their sums) and 16 XB rows, its
// waves share the columns out in steps of QUADS * 4 blocks and join their sums in LDS.
// Weights go straight into registers; a wave quantises its own columns of x into its
// own LDS while they are on their way, so that one launch does it all. Where every wave
// has no more than one step, a workgroup takes further outputs with the x it has.
#define DHX_FEW_PARAMS Addr x_, Addr w_, Addr up_, int rows, int inputs, int outputs, uint32_t x_stride, uint32_t w_stride, Addr starts_, Addr ws_, Addr us_, Addr bias_, Addr up_bias_, Addr out_, uint64_t out_stride, int sequences, int activation, uint32_t ws_stride

template <class T, bool GATED, int XB, int QUADS>
__global__ __launch_bounds__(64 * kFewProductWaves) void packed_product_few_kernel(DHX_FEW_PARAMS) {
    typedef typename Num<T>::v8 v8;
    constexpr int AB = GATED ? 2 : 1, ROWS = 16 * XB, WAVES = kFewProductWaves;
    constexpr int LANES = 16 * QUADS, SIDE = 64 / LANES;      // of a row, rows side by side
    constexpr int LOADS = ROWS / SIDE < 4 ? ROWS / SIDE : 4;  // of x on their way at a time
    static_assert(ROWS % (LOADS * SIDE) == 0, "no row behind the last");
    constexpr int PITCH = QUADS * 64 + 16, SCALES = QUADS * 4;  // bytes of a row's codes, and of its scales
    __shared__ __attribute__((aligned(16))) char all_codes[WAVES * ROWS * PITCH], all_scales[WAVES * ROWS * SCALES];
    __shared__ __attribute__((aligned(16))) float sum[AB][WAVES][ROWS][20];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, part = lane >> 4;
    char *const codes = all_codes + wave * ROWS * PITCH, *const scales = all_scales + wave * ROWS * SCALES;
    const int row0 = blockIdx.y * ROWS, mine = min(rows - row0, ROWS);
    const char* x0 = (const char*)x_ + (uint64_t)row0 * x_stride;
    const int pieces = (inputs + 31) >> 5, steps = (pieces + 4 * QUADS - 1) / (4 * QUADS), blocks = (outputs + 15) >> 4;
    int first = 0, end = rows;  // the rows that count
    if (starts_.a) {
        first = start_at(starts_, 0, rows);
        end = start_at(starts_, sequences, rows);
    }
    // A lane's blocks: 4 kk + part, kk = 0 .. QUADS-1, of a step's.
    uint4_t fw[AB][QUADS];
    uint32_t sw[AB][QUADS];
    auto load_weights = [&](int block, int s) __attribute__((always_inline)) {
        const int col = min(block * 16 + l16, outputs - 1), left = pieces - s * 4 * QUADS - part;
#pragma unroll
        for (int a = 0; a < AB; ++a) {
            const char *w = (const char*)(a ? up_ : w_) + (uint64_t)col * w_stride + part * 16, *ws = (const char*)(a ? us_ : ws_) + (uint64_t)col * ws_stride;
#pragma unroll
            for (int kk = 0; kk < QUADS; ++kk) {
                const bool in = 4 * kk < left;
                fw[a][kk] = in ? *(const uint4_t*)(w + (s * QUADS + kk) * 64) : uint4_t{};
                sw[a][kk] = in ? *(const uint32_t*)(ws + (s * QUADS + kk) * 4) >> (8 * part) : 0;
            }
        }
    };
    auto quantise = [&](int s) __attribute__((always_inline)) {
        const int at = s * QUADS * 128 + lane % LANES * 8;  // the lane's first column of x
        wave_lds_sync();  // the step before has been read
#pragma unroll
        for (int r0 = 0; r0 < ROWS; r0 += LOADS * SIDE) {
            if (r0 >= mine) break;  // what stands in the other rows is multiplied, and not stored
            v8 v[LOADS];
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int r = r0 + i * SIDE + lane / LANES;
                v[i] = r < mine && at < inputs ? *(const v8*)(x0 + (uint64_t)r * x_stride + at * 2) : v8{};
            }
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int r = r0 + i * SIDE + lane / LANES;
                const FourBits got = four_bits<T>(v[i]);
                *(uint32_t*)(codes + r * PITCH + lane % LANES * 4) = got.codes;
                if ((lane & 3) == 0) scales[r * SCALES + lane % LANES / 4] = (char)got.scale;
            }
        }
        wave_lds_sync();
    };
    if (wave < steps) {
        load_weights(blockIdx.x, wave);
        quantise(wave);
    }
    for (int block = blockIdx.x; block < blocks; block += gridDim.x) {
        float4_t acc[AB][XB] = {};
        for (int s = wave; s < steps; s += WAVES) {
            if (s != wave) {
                load_weights(block, s);
                quantise(s);
            }
#pragma unroll
            for (int m = 0; m < XB; ++m)
#pragma unroll
                for (int kk = 0; kk < QUADS; ++kk) {
                    const int r = m * 16 + l16;
                    const uint4_t fx = *(const uint4_t*)(codes + r * PITCH + (kk * 4 + part) * 16);
                    const uint32_t sx = *(const uint32_t*)(scales + r * SCALES + kk * 4) >> (8 * part);
#pragma unroll
                    for (int a = 0; a < AB; ++a) acc[a][m] = product16(fw[a][kk], fx, acc[a][m], sw[a][kk], sx);
                }
        }
        if (wave < steps && block + (int)gridDim.x < blocks) load_weights(block + gridDim.x, wave);
        store_few<T, GATED, XB>(sum, acc, block * 16, row0, first, min(end, rows), outputs, activation, bias_, up_bias_, out_, out_stride);
        lds_barrier();  // the sums have been read
    }
}

// Whether the few-rows kernel takes a call, by its pairs of 16 rows and 16 outputs, of
// which a gated one has two products. us against tiles (with their launch that quantises
// x), linear: 1024 -> 1024, 1 row 3.2 and 5.9, 64 rows (256 pairs) 3.5 and 6.9; 4096 ->
// 4096, 1 row 4.8 and 10.0, 32 rows (512) 10.7 and 11.4, 48 rows (768) 13.6 and 11.8; 4096
// -> 16384 (1024), 8 rows 12.5 and 13.0, 16 rows 14.2 and 13.3; 16384 -> 128, 512 rows (256)
// 25.0 and 29.6, 1000 rows (504) 45.2 and 31.2; short rows: 384 -> 384, 1024 rows (1536)
// 4.7 and 5.9, 2048 rows 6.9 and 6.1; 1024 -> 1024, 256 rows (1024) 5.1 and 7.0, 512 rows
// 7.2 and 7.1; 2048 -> 2048, 128 rows (1024) 7.6 and 9.0, 256 rows 11.5 and 9.3. Gated:
// 4096 -> 512, 128 rows (256) 9.5 and 12.6, 256 rows 15.0 and 12.8; 1024 -> 2728, 64 rows
// (684) 6.6 and 7.3, 128 rows 8.5 and 7.4; 384 -> 1536, 128 rows (768) 5.0 and 6.3, 256
// rows 6.3 and 6.4.
inline bool few_product(uint64_t rows, uint64_t inputs, uint64_t outputs, bool gated) {
    const uint64_t blocks = (outputs + 15) / 16, all = (rows + 15) / 16 * blocks * (gated ? 2 : 1);
    if (rows <= 8) return blocks <= 256 || inputs <= 4096;
    if (all <= 256 || (all <= 512 && (gated || inputs <= 4096))) return true;
    return all <= 2048 && inputs <= 2048 && all * inputs <= 2048 * 1024;
}

// p.x is the call's own here, in 16 bits, and p.pieces the columns of it. Two
// workgroups of 16 rows run on a CU, one of 32. A workgroup that takes several blocks of
// 16 outputs quantises its rows once for all of them, so that one round of workgroups is
// better than one for every block (32 rows: 1024 -> 1024, 256 rows 5.1 us and 6.0; 384 ->
// 1152, 512 rows 6.3 and 8.6).
template <class T, bool GATED, int XB, int QUADS>
hipError_t launch_few(const Product& p, hipStream_t s) {
    uint32_t blocks = (p.outputs + 15) / 16;
    const uint32_t row_blocks = (p.rows + 16 * XB - 1) / (16 * XB), at_once = XB == 1 ? 512 : 256;
    if (p.pieces <= 128 * QUADS * kFewProductWaves) blocks = std::min(blocks, std::max(1u, at_once / row_blocks));
    return enqueue(packed_product_few_kernel<T, GATED, XB, QUADS>, dim3(blocks, row_blocks),
                   dim3(64 * kFewProductWaves), 0, s, p.x, p.w, p.up,
                   (int)p.rows, (int)p.pieces, (int)p.outputs, (uint32_t)p.x_stride, (uint32_t)p.w_stride, p.starts, p.ws, p.us, p.bias,
                   p.up_bias, p.out, p.out_stride, (int)p.sequences, (int)p.activation, (uint32_t)p.ws_stride);
}
template <class T, bool GATED, int XB>
hipError_t launch_few_columns(const Product& p, hipStream_t s) {
    if (p.pieces <= 1024) return launch_few<T, GATED, XB, 1>(p, s);
    if constexpr (XB == 1) {
        if (p.pieces > 2048) return launch_few<T, GATED, 1, 4>(p, s);
    }
    return launch_few<T, GATED, XB, 2>(p, s);
}
// Blocks of 16 rows take half as long as those of 32 to be quantised, and read the weights
// twice as often. us of 16 and 32 rows: 1024 -> 1024, 64 rows (256 pairs of 16 rows and 16
// outputs) 3.5 and 4.3, 128 rows 4.6 and 4.3; gated, 128 rows 5.8 and 5.3; short rows: 640
// -> 640, 256 rows (640) 4.4 and 4.7, 896 -> 2048, 128 rows (1024) 5.0 and 4.9; long ones:
// 4096 -> 512, 256 rows (512) 11.1 and 11.6, 2048 -> 2048, 64 rows (512) 6.7 and 6.5.
template <class T, bool GATED>
hipError_t launch_few_rows(const Product& p, hipStream_t s) {
    const uint64_t all = (p.rows + 15) / 16 * ((p.outputs + 15) / 16);
    if (p.rows <= 16 || all <= 256 || p.pieces <= 768 || p.pieces > 2048) return launch_few_columns<T, GATED, 1>(p, s);
    return launch_few_columns<T, GATED, 2>(p, s);
}

// The tile of a call, from the number of workgroups that each would make and the
// number of its stages. us on MI355X (two of 128 x 128 or smaller tiles run on a CU, one
// of 256 x 256 and of those with four stages; products with 4-bit weights hold the
// launch that quantises x):
// - 256 x 256 where they fill the CUs once or in rounds of which the last is not
//   mostly empty: gated, 4096 -> 8192, 1024 rows (256 tiles) 116, 128 x 128 148; 512 rows
//   (128 tiles) 98 and 77; 1024 -> 2728, 2048 rows (176) 27.4 and 30.5, 4096 rows (352)
//   55.9 and 51.8; 384 -> 1536, 12864 rows (612) 41.4 and 44.5; four bits, two stages
//   (384 -> 1536, 4096 rows) 17.4 and 15.1; gated, waves of 64 x 128, which hold whole
//   lines of outputs (128 x 64: 8192 rows, 4096 -> 8192, 860 and 844);
// - long rows and a CU for every tile: four stages in flight, of the smallest such tile:
//   gated, 4096 -> 8192, 48 rows, 64 x 64 34.1 (two stages 49.9), 128 rows, 128 x 64 38.9
//   (55.6), 256 rows, 128 x 128 49.4 (60.8; four bits 20.8 and 19.2); short rows gain
//   nothing (384 -> 1536, 256 rows, 4.8 and 4.4);
// - else the smallest of which two rounds run at once: linear, four bits, 1024 -> 1024,
//   2048 rows, 64 x 64 8.9, 128 x 128 9.8, 4096 rows 12.2 and 11.9; gated, 384 -> 1536,
//   1024 rows, 64 x 64 7.0, 128 x 64 6.4, 2048 rows 13.3, 10.2 and (128 x 128) 10.1.
template <class T, bool FOUR, bool GATED>
hipError_t launch_product(const Product& p, hipStream_t s) {
    auto count = [&](uint64_t m, uint64_t n) { return (p.rows + m - 1) / m * ((p.outputs + n - 1) / n) * (GATED ? 2 : 1); };
    const uint64_t largest = (p.rows + 255ull) / 256 * ((p.outputs + (GATED ? 127 : 255)) / (GATED ? 128 : 256));
    const uint32_t steps = (p.pieces + 7) / 8;
    constexpr int WM = GATED ? 32 : 64, WN = GATED ? 64 : 32;  // of a 128 x 64 tile: a wave of the gated one holds both sums
    const bool fills = largest <= 256 ? largest >= 160 : largest * 4 >= (largest + 255) / 256 * 256 * 3;
    // (With 4 bits that tile takes stages by fours.)
    if (fills && (!FOUR || (steps + 3) / 4 * 16 <= steps * 5))
        return launch_tiles<T, FOUR, GATED, 256, 256, GATED ? 64 : 128, GATED ? 128 : 64, 2, 2>(p, s);
    if (steps >= 12) {
        if (count(64, 64) <= 256) return launch_tiles<T, FOUR, GATED, 64, 64, 32, GATED ? 64 : 32, 4, GATED ? 1 : 2>(p, s);
        if (count(128, 64) <= 256) return launch_tiles<T, FOUR, GATED, 128, 64, WM, WN, 4, 1>(p, s);
        if constexpr (!FOUR)
            if (count(128, 128) <= 256) return launch_tiles<T, FOUR, GATED, 128, 128, 64, 64, 4, 1>(p, s);
    }
    if (count(64, 64) <= 512) return launch_tiles<T, FOUR, GATED, 64, 64, 32, GATED ? 64 : 32, 2, GATED ? 2 : 4>(p, s);
    if (count(128, 64) <= 512) return launch_tiles<T, FOUR, GATED, 128, 64, WM, WN, 2, 2>(p, s);
    return launch_tiles<T, FOUR, GATED, 128, 128, 64, 64, 2, 2>(p, s);
}

// x of a call, quantised into its workspace (codes, then scales) on the stream: the
// launch of it, and where the product finds it.
uint64_t quantised_rows_bytes(uint64_t rows, uint64_t columns);
hipError_t quantise_rows(uint32_t type, const void* x, uint64_t x_stride, uint64_t rows, uint32_t columns, void* workspace, Product* product,
                         hipStream_t s);

}  // namespace dhx
