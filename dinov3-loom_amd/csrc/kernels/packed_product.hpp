// The products of the feed-forward half of a packed block
// (include/dinov3_packed.h): rows of x times rows of one or two weight matrices,
// in 16 bits or in 4 with a scale per 32 values, with a bias, or gated (act(g) u of
// the two). One tile kernel in bytes: a piece of 16 bytes of a row is 8 values
// or a block of 32, a stage in LDS holds 8 pieces of each of a tile's rows, and a
// matrix instruction (32 x 32 outputs, either way 8 passes) takes one piece per
// lane of each side.
#pragma once
#include <type_traits>

#include "packed.hpp"

namespace dhx {

// What a launcher hands on; strides are in bytes but that of out.
struct Product {
    uint32_t type, activation, rows, pieces, outputs, sequences;
    const void *x, *w, *up;             // up: gated only
    const void *xs, *ws, *us;           // scales: 4-bit only
    const float *bias, *up_bias;
    void* out;
    const int32_t* starts;
    uint64_t x_stride, w_stride, xs_stride, ws_stride, out_stride;
};

#define DHX_PRODUCT_PARAMS Addr x_, Addr w_, Addr up_, int rows, int pieces, int outputs, uint32_t x_stride, uint32_t w_stride, Addr starts_, Addr xs_, Addr ws_, Addr us_, Addr bias_, Addr up_bias_, Addr out_, uint64_t out_stride, int sequences, int activation, uint32_t xs_stride, uint32_t ws_stride

template <class K>
hipError_t enqueue_product(K kernel, dim3 grid, dim3 block, hipStream_t s, const Product& p) {
    return enqueue(kernel, grid, block, 0, s, p.x, p.w, p.up, (int)p.rows, (int)p.pieces, (int)p.outputs, (uint32_t)p.x_stride,
                   (uint32_t)p.w_stride, p.starts, p.xs, p.ws, p.us, p.bias, p.up_bias, p.out, p.out_stride, (int)p.sequences,
                   (int)p.activation, (uint32_t)p.xs_stride, (uint32_t)p.ws_stride);
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

template <int ACT>
__device__ __forceinline__ float activated(float g) {
    // e^-g past the range of float32 is infinite, and its reciprocal 0.
    if constexpr (ACT == DHX_SILU) return g * fast_rcp(1.0f + fast_exp2(-kLog2e * g));
    if constexpr (ACT == DHX_SIGMOID) return fast_rcp(1.0f + fast_exp2(-kLog2e * g));
    if constexpr (ACT == DHX_RELU) return g < 0.0f ? 0.0f : g;  // NaN stays
    if constexpr (ACT == DHX_GELU) return 0.5f * g * (1.0f + erff(0.70710678f * g));
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
// being filled). A lane multiplies piece 4 (lane / 32) + kk in step kk: a block of 4
// bits then finds its scale in byte kk of the half's own word of the row's 8.
// Scales come 16 bytes per row at a time, for two stages.
template <class T, bool FOUR, bool GATED, int BM, int BN, int WM, int WN, int NST, int PER_SIMD>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN), PER_SIMD) void packed_product_kernel(DHX_PRODUCT_PARAMS) {
    typedef typename Num<T>::v8 v8;
    typedef typename Num<T>::v4 v4;
    constexpr int WAVES = (BM / WM) * (BN / WN), THREADS = 64 * WAVES;
    constexpr int XL = BM / 8 / WAVES, WL = BN / 8 / WAVES;  // loads of 8 rows per wave and stage
    constexpr int SCALE_LOADS = (BM + BN) / 64, SL = FOUR ? (SCALE_LOADS + WAVES - 1) / WAVES : 0;
    constexpr int MB = WM / 32, NB = WN / 32, KK = 4;
    constexpr int BO = GATED ? BN / 2 : BN;  // outputs of a tile
    constexpr int RINGS = NST > 2 ? 3 : 2;   // of scales, each for two stages
    static_assert(NST % 2 == 0, "a stage's half of its scales is a constant");
    static_assert(XL * 8 * WAVES == BM && WL * 8 * WAVES == BN && BM % 64 == 0 && BN % 64 == 0 && BN <= THREADS, "whole loads");
    static_assert(!GATED || NB % 2 == 0, "both sums of an output in one lane");
    __shared__ __attribute__((aligned(16))) char sX0[BM * 128], sX1[BM * 128], sX2[NST > 2 ? BM * 128 : 16], sX3[NST > 2 ? BM * 128 : 16];
    __shared__ __attribute__((aligned(16))) char sW0[BN * 128], sW1[BN * 128], sW2[NST > 2 ? BN * 128 : 16], sW3[NST > 2 ? BN * 128 : 16];
    __shared__ __attribute__((aligned(16))) char sScale[FOUR ? RINGS * (BM + BN) * 16 : 16];
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
    const int steps = (pieces + 7) / 8, whole = pieces / 8;
    const char* x0 = (const char*)x_ + (uint64_t)row0 * x_stride;

    // Weight row r of the tile: which matrix, and which of its rows.
    auto of_up = [&](int r) { return GATED && (r & 32) != 0; };
    auto column = [&](int r) { return GATED ? (r >> 6) * 32 + (r & 31) : r; };
    const char *w0 = (const char*)w_ + (uint64_t)col0 * w_stride, *up0 = (const char*)up_ + (uint64_t)col0 * w_stride;

    // Lane -> row lane / 8 of a load's 8, the piece that the swizzle puts at slot
    // lane % 8; rows behind the last one fetch that one.
    uint32_t xo[XL], wo[WL];
    const int lr = lane >> 3, l32 = lane & 31, hi = lane >> 5;
    auto chunk = [&](int r) { return (lane & 7) ^ slot_of<64>(r); };
#pragma unroll
    for (int j = 0; j < XL; ++j) {
        const int r = (wave * XL + j) * 8 + lr;
        xo[j] = (uint32_t)min(r, rows - 1 - row0) * x_stride + chunk(r) * 16;
    }
#pragma unroll
    for (int j = 0; j < WL; ++j) {
        const int r = (wave * WL + j) * 8 + lr;
        wo[j] = (uint32_t)min(column(r), outputs - 1 - col0) * w_stride + chunk(r) * 16;
    }
    auto w_base = [&](int j) { return of_up((wave * WL + j) * 8) ? up0 : w0; };
    // A load of scales takes 64 rows, those of x first; with more waves than loads
    // some are made twice, so that every wave has as many on their way.
    const char* so[SL > 0 ? SL : 1];
    int sto[SL > 0 ? SL : 1];
    if constexpr (FOUR) {
#pragma unroll
        for (int j = 0; j < SL; ++j) {
            const int load = (wave * SL + j) % SCALE_LOADS, r = load * 64 + lane;
            sto[j] = load * 1024;
            if (load * 64 < BM) {
                so[j] = (const char*)xs_ + (uint64_t)(row0 + min(r, rows - 1 - row0)) * xs_stride;
            } else {
                const int c = col0 + min(column(r - BM), outputs - 1 - col0);
                so[j] = (of_up(r - BM) ? (const char*)us_ : (const char*)ws_) + (uint64_t)c * ws_stride;
            }
        }
    }
    auto move_scales = [&](int pair) __attribute__((always_inline)) {
        if constexpr (FOUR) {
#pragma unroll
            for (int j = 0; j < SL; ++j) dma16(so[j] + pair * 16, sScale + pair % RINGS * (BM + BN) * 16 + sto[j]);
        }
    };
    auto move_whole = [&](char* sx, char* sw, int s) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < XL; ++j) dma16(x0 + s * 128 + xo[j], sx + (wave * XL + j) * 1024);
#pragma unroll
        for (int j = 0; j < WL; ++j) dma16(w_base(j) + s * 128 + wo[j], sw + (wave * WL + j) * 1024);
    };
    auto move = [&](char* sx, char* sw, int s) __attribute__((always_inline)) {
        if ((s & 1) == 0) move_scales(s >> 1);
        if (s < whole) {
            move_whole(sx, sw, s);
            return;
        }
        const char* zeros = (const char*)&kZeros;
#pragma unroll
        for (int j = 0; j < XL; ++j) {
            const bool in = s * 8 + chunk((wave * XL + j) * 8 + lr) < pieces;
            dma16(in ? x0 + s * 128 + xo[j] : zeros, sx + (wave * XL + j) * 1024);
        }
#pragma unroll
        for (int j = 0; j < WL; ++j) {
            const bool in = s * 8 + chunk((wave * WL + j) * 8 + lr) < pieces;
            dma16(in ? w_base(j) + s * 128 + wo[j] : zeros, sw + (wave * WL + j) * 1024);
        }
    };

    const int wm = wave / (BN / WN) * WM, wn = wave % (BN / WN) * WN;
    const int frag = l32 * 128 + (((hi * 4) ^ slot_of<64>(l32)) << 4);
    float16_t acc[MB][NB] = {};
    uint4_t fx[2][MB], fw[2][NB];
    uint32_t scale_x[2][MB], scale_w[2][NB];  // of even and odd stages
    auto load = [&](const char* sx, const char* sw, int kk, int set) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MB; ++i) fx[set][i] = *(const uint4_t*)(sx + (wm + i * 32) * 128 + (frag ^ (kk << 4)));
#pragma unroll
        for (int i = 0; i < NB; ++i) fw[set][i] = *(const uint4_t*)(sw + (wn + i * 32) * 128 + (frag ^ (kk << 4)));
    };
    auto load_scales = [&](int s, int odd) __attribute__((always_inline)) {
        if constexpr (FOUR) {
            const char* from = sScale + (s >> 1) % RINGS * (BM + BN) * 16 + odd * 8 + l32 * 16 + hi * 4;
            // Behind the last piece there are no scales (and zeros for values).
            const int left = pieces - s * 8 - hi * 4;
            const uint32_t mask = left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1;
#pragma unroll
            for (int i = 0; i < MB; ++i) scale_x[odd][i] = *(const uint32_t*)(from + (wm + i * 32) * 16) & mask;
#pragma unroll
            for (int i = 0; i < NB; ++i) scale_w[odd][i] = *(const uint32_t*)(from + (BM + wn + i * 32) * 16) & mask;
        }
    };
    auto multiply = [&](auto kk, int set, int odd) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int k = 0; k < NB; ++k)
                acc[i][k] = product32<T, FOUR, decltype(kk)::value>(fw[set][k], fx[set][i], acc[i][k], FOUR ? scale_w[odd][k] : 0, FOUR ? scale_x[odd][i] : 0);
    };
    move(sX0, sW0, 0);
    if (tid < BN) {
        const float* bias = of_up(tid) ? up_bias_ : bias_;
        sBias[tid] = bias && col0 + column(tid) < outputs ? bias[col0 + column(tid)] : 0.f;
    }
    if (NST > 2 && steps > 1) move(sX1, sW1, 1);
    if (NST > 2 && steps > 2) move(sX2, sW2, 2);
    // Opens stage s: it has landed (the NST - 2 stages behind it may be on their way,
    // one of them with scales), and every wave has read the one before, whose place
    // stage s + NST - 1 takes.
    auto open = [&](auto fast, char* free_x, char* free_w, int s) __attribute__((always_inline)) {
        if (fast || s + NST - 2 < steps) wait_vm<(NST - 2) * (XL + WL) + (NST > 2 ? SL : 0)>();
        else wait_vm<0>();
        wait_lgkm();
        barrier();
        const int next = s + NST - 1;
        if constexpr (fast) {
            if ((next & 1) == 0) move_scales(next >> 1);
            move_whole(free_x, free_w, next);
        } else if (next < steps) {
            move(free_x, free_w, next);
        }
    };
    auto step = [&](auto fast, char* sx, char* sw, const char* next_x, const char* next_w, int s, int odd) __attribute__((always_inline)) {
        auto inner = [&](auto kk) __attribute__((always_inline)) {
            load(sx, sw, kk + 1, (kk + 1) & 1);
            __builtin_amdgcn_sched_barrier(0);  // the reads go ahead of the products they pass under
            multiply(kk, kk & 1, odd);
            __builtin_amdgcn_sched_barrier(0);
        };
        inner(std::integral_constant<int, 0>{});
        inner(std::integral_constant<int, 1>{});
        inner(std::integral_constant<int, 2>{});
        if (fast || s + 1 < steps) {
            open(fast, sx, sw, s + 1);
            load(next_x, next_w, 0, 0);
            load_scales(s + 1, 1 - odd);
        }
        __builtin_amdgcn_sched_barrier(0);
        multiply(std::integral_constant<int, 3>{}, 1, odd);
    };
    open(std::false_type{}, NST == 2 ? sX1 : sX3, NST == 2 ? sW1 : sW3, 0);
    load(sX0, sW0, 0, 0);
    load_scales(0, 0);
    int s = 0;
    auto turn_of_stages = [&](auto fast) __attribute__((always_inline)) {
        step(fast, sX0, sW0, sX1, sW1, s, 0);
        if (fast || s + 1 < steps) step(fast, sX1, sW1, NST > 2 ? sX2 : sX0, NST > 2 ? sW2 : sW0, s + 1, 1);
        if constexpr (NST > 2) {
            if (fast || s + 2 < steps) step(fast, sX2, sW2, sX3, sW3, s + 2, 0);
            if (fast || s + 3 < steps) step(fast, sX3, sW3, sX0, sW0, s + 3, 1);
        }
        s += NST;
    };
    while (s + 2 * NST <= whole) turn_of_stages(std::true_type{});
    while (s < steps) turn_of_stages(std::false_type{});

    // Lane: row l32 of a block, columns 8 g + 4 hi .. +3 of its 32 in register group
    // g; both halves exchange groups, so that each stores 8 columns at once.
    auto bias4 = [&](int k, int g) { return *(const float4_t*)(sBias + wn + k * 32 + 8 * g + 4 * hi); };
    auto store = [&](int i, int col, v4 lo, v4 up) __attribute__((always_inline)) {
        const int row = row0 + wm + i * 32 + l32;
        const v8 piece = __builtin_bit_cast(v8, frag_swap(__builtin_bit_cast(half4_t, lo), __builtin_bit_cast(half4_t, up)));
        if (row >= first && row < end && col + hi * 8 < outputs) *(v8*)((T*)out_ + (uint64_t)row * out_stride + col + hi * 8) = piece;
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
            for (int i = 0; i < MB; ++i)
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
                        store(i, col0 + (wn + k * 32) / 2 + kk * 16, o[0], o[1]);
                    }
        });
    } else {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int k = 0; k < NB; ++k)
#pragma unroll
                for (int kk = 0; kk < 2; ++kk)
                    store(i, col0 + wn + k * 32 + kk * 16, rounded(group(acc[i][k], 2 * kk) + bias4(k, 2 * kk)),
                          rounded(group(acc[i][k], 2 * kk + 1) + bias4(k, 2 * kk + 1)));
    }
}

template <class T, bool FOUR, bool GATED, int BM, int BN, int WM, int WN, int NST, int PER_SIMD>
hipError_t launch_tiles(const Product& p, hipStream_t s) {
    constexpr uint64_t BO = GATED ? BN / 2 : BN;
    const uint64_t total = ((uint64_t)p.rows + BM - 1) / BM * ((p.outputs + BO - 1) / BO);
    return enqueue_product(packed_product_kernel<T, FOUR, GATED, BM, BN, WM, WN, NST, PER_SIMD>, dim3((unsigned)((total + 7) / 8 * 8)),
                           dim3(64 * (BM / WM) * (BN / WN)), s, p);
}

// x of a call, quantised into its workspace (codes, then scales) on the stream: the
// launch of it, and where the product finds it.
uint64_t quantised_rows_bytes(uint64_t rows, uint64_t columns);
hipError_t quantise_rows(uint32_t type, const void* x, uint64_t x_stride, uint64_t rows, uint32_t columns, void* workspace, Product* product,
                         hipStream_t s);

}  // namespace dhx
