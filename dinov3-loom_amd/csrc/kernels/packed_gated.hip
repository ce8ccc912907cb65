// The gated projections of a feed-forward block on packed batches
// (include/dinov3_packed.h): out = act(x Wg^T + bg) (x Wu^T + bu), one product
// kernel whose tiles hold rows of both matrices (packed_product.hpp), with weights in
// 16 bits, or in 4 behind the kernel that quantises x (packed_quantise.hip). Few rows
// have kernels of their own, of which the one for 4 bits quantises x as well.
#include "packed_product.hpp"

namespace dhx {

// Few rows against weights in 16 bits: a workgroup takes 16 outputs and both of their
// sums, of 16 XB rows; its waves take steps of 64 columns in turn and join their sums in
// LDS, so that long rows do not make one workgroup's chain. Bound by the weights'
// bytes where these fill the CUs (4096 -> 8192, 1 row: 134 MB in 25.7 us, 5.2 TB/s), by a
// CU's own reads where few outputs leave the others idle. Operands are fetched a step
// ahead into registers, in whole lines, and change lanes through LDS that is the wave's own:
// fetched as the matrix instruction wants them, 16 rows side by side, a load takes four
// times as long (4096 -> 512, 16 rows 13.4 us and 6.9; 16384 -> 512 44.5 and 18.5). Steps
// of 64 columns leave room for two workgroups on a CU; one, with steps of 128 and the
// sums beside the operands, took longer (32 rows: 2048 -> 2048, 64 rows 7.6 and 6.7; 4096 ->
// 8192, 32 rows 31.5 and 30.7).
template <class T, int XB>
__global__ __launch_bounds__(64 * kFewProductWaves) void packed_gated_few_kernel(Addr x_, Addr w_, Addr up_, int rows, int pieces, int outputs, uint32_t x_stride, uint32_t w_stride, Addr starts_, Addr bias_, Addr up_bias_, Addr out_, uint64_t out_stride, int sequences, int activation) {
    typedef typename Num<T>::v8 v8;
    constexpr int PITCH = 128 + 16;
    typedef float Sums[kFewProductWaves][16 * XB][20];
    __shared__ __attribute__((aligned(16))) char tiles[kFewProductWaves][(2 + XB) * 16 * PITCH];
    static_assert(sizeof tiles >= 2 * sizeof(Sums), "the sums follow in the same place");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    char* const tile = tiles[wave];
    const int l16 = lane & 15, part = lane >> 4;
    const int row0 = blockIdx.y * 16 * XB, col0 = blockIdx.x * 16, steps = (pieces + 7) >> 3;
    int first = 0, end = rows;  // the rows that count
    if (starts_.a) {
        first = start_at(starts_, 0, rows);
        end = start_at(starts_, sequences, rows);
    }
    auto rows_of = [&](Addr base, int row, int n, uint32_t stride) {
        return __builtin_amdgcn_make_buffer_rsrc((void*)(base.a + (uint64_t)row * stride), 0, (int)((uint32_t)(n - 1) * stride + pieces * 16),
                                                 kBufferRsrcWord3);
    };
    const int columns = min(16, outputs - col0), mine = min(16 * XB, rows - row0);
    const __amdgpu_buffer_rsrc_t x_rows = rows_of(x_, row0, mine, x_stride);
    const __amdgpu_buffer_rsrc_t w_rows[2] = {rows_of(w_, col0, columns, w_stride), rows_of(up_, col0, columns, w_stride)};
    // A load takes 128 bytes of 8 rows, eight lanes to a row; rows behind the last one
    // fetch that one.
    uint32_t xo[XB][2], wo[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = i * 8 + (lane >> 3);
        wo[i] = (uint32_t)min(r, columns - 1) * w_stride;
#pragma unroll
        for (int m = 0; m < XB; ++m) xo[m][i] = (uint32_t)min(m * 16 + r, mine - 1) * x_stride;
    }
    uint4_t fetched[2][2 + XB][2];
    auto load = [&](auto slot, int s) __attribute__((always_inline)) {
        const int piece = s * 8 + (lane & 7);  // those behind the last one are zeros
        auto from = [&](const __amdgpu_buffer_rsrc_t& r, uint32_t at) __attribute__((always_inline)) {
            return __builtin_bit_cast(uint4_t, __builtin_amdgcn_raw_buffer_load_b128(r, (int)(piece < pieces ? at + piece * 16 : ~15u), 0, 0));
        };
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            fetched[slot][0][i] = from(w_rows[0], wo[i]);
            fetched[slot][1][i] = from(w_rows[1], wo[i]);
#pragma unroll
            for (int m = 0; m < XB; ++m) fetched[slot][2 + m][i] = from(x_rows, xo[m][i]);
        }
    };
    float4_t acc[2][XB] = {};
    auto multiply = [&](auto slot) __attribute__((always_inline)) {
        wave_lds_sync();  // the step before has been read
#pragma unroll
        for (int g = 0; g < 2 + XB; ++g)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                *(uint4_t*)(tile + (g * 16 + i * 8 + (lane >> 3)) * PITCH + (lane & 7) * 16) = fetched[slot][g][i];
        wave_lds_sync();
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            v8 f[2 + XB];
#pragma unroll
            for (int g = 0; g < 2 + XB; ++g) f[g] = *(const v8*)(tile + (g * 16 + l16) * PITCH + (kk * 4 + part) * 16);
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int m = 0; m < XB; ++m) acc[a][m] = Num<T>::mfma16(f[a], f[2 + m], acc[a][m]);
        }
    };
    constexpr std::integral_constant<int, 0> even{};
    constexpr std::integral_constant<int, 1> odd{};
    load(even, wave);
    for (int s = wave; s < steps; s += 2 * kFewProductWaves) {
        load(odd, s + kFewProductWaves);
        __builtin_amdgcn_sched_barrier(0);  // loads are not put off until they are used
        multiply(even);
        __builtin_amdgcn_sched_barrier(0);
        load(even, s + 2 * kFewProductWaves);
        __builtin_amdgcn_sched_barrier(0);
        multiply(odd);
        __builtin_amdgcn_sched_barrier(0);
    }
    lds_barrier();  // every wave has read its operands
    store_few<T, true, XB>((Sums*)tiles, acc, col0, row0, first, end, outputs, activation, bias_, up_bias_, out_, out_stride);
}

// Blocks of 16 rows to a workgroup of the few-rows kernel, 0 for tiles. By pairs of 16 (or
// 32) rows and 16 outputs, in us of tiles, of 16 rows and of 32:
// - up to 256 pairs of 16 rows: 136 -> 4096, 16 rows (256 pairs) 3.7, 3.0, 3.3; 1024 -> 1024,
//   64 rows (256) 6.8, 3.7, 4.2; 4096 -> 512, 128 rows (256) 19.4, 7.3, 8.8; 16384 -> 512, 1
//   row 63.1, 17.5, 22.5; and one block of rows, but for short rows of many outputs: 1024 ->
//   16384, 1 row (1024) 13.3, 12.5, 12.7; 384 -> 8096 (506) 5.7, 4.7, 5.5, -> 16384 (1024)
//   7.1, 8.1, 9.3;
// - up to 256 pairs of 32 rows: 384 -> 384, 256 rows (192) 4.2, 4.2, 3.9; 600 -> 800, 160
//   rows (250) 5.2, 5.1, 4.7; 4096 -> 512, 256 rows (256) 19.4, 11.3, 9.2; and one such
//   block, but for short rows: 2048 -> 8192, 24 rows (512) 13.8, 20.6, 12.5; 384 -> 8096,
//   24 rows (506) 5.8, 8.4, 5.8, -> 16384 7.3, 14.0, 9.7;
// - up to 512 of long rows, whose weights caches hold for the next block of rows: 2048 ->
//   2048, 128 rows (512) 11.5, 12.8, 9.8; 4096 -> 1024, 256 rows (512) 19.4, 19.8, 14.9; but
//   4096 -> 4096, 64 rows (512) 20.0, 41.1, 22.6; 1024 -> 2728, 64 rows (342) 7.6, 9.5, 7.5.
int few_gated(uint64_t rows, uint64_t inputs, uint64_t outputs) {
    const uint64_t blocks = (outputs + 15) / 16, narrow = (rows + 15) / 16 * blocks, wide = (rows + 31) / 32 * blocks;
    if (narrow <= 256 || (rows <= 16 && (blocks <= 512 || inputs >= 1024))) return 1;
    if (wide <= 256 || (rows <= 32 && inputs >= 1024)) return 2;
    return wide <= 512 && inputs >= 2048 && inputs * outputs <= 1 << 22 ? 2 : 0;
}

template <class T>
hipError_t launch_few_gated(const Product& p, int blocks, hipStream_t s) {
    return enqueue(blocks == 1 ? packed_gated_few_kernel<T, 1> : packed_gated_few_kernel<T, 2>,
                   dim3((p.outputs + 15) / 16, (p.rows + 16 * blocks - 1) / (16 * blocks)), dim3(64 * kFewProductWaves), 0, s, p.x, p.w, p.up,
                   (int)p.rows, (int)p.pieces, (int)p.outputs, (uint32_t)p.x_stride, (uint32_t)p.w_stride, p.starts, p.bias, p.up_bias, p.out,
                   p.out_stride, (int)p.sequences, (int)p.activation);
}

uint64_t packed_gated_bytes(const dhx_packed_gated& p) {
    return p.gate_scales && !few_product(p.rows, p.inputs, p.outputs, true) ? quantised_rows_bytes(p.rows, p.inputs) : 0;
}

hipError_t launch_packed_gated(const dhx_packed_gated& p, hipStream_t s) {
    Product a{};
    a.activation = p.activation;
    a.rows = (uint32_t)p.rows;
    a.outputs = p.outputs;
    a.sequences = p.sequences;
    a.w = p.gate;
    a.up = p.up;
    a.bias = p.gate_bias;
    a.up_bias = p.up_bias;
    a.out = p.out;
    a.starts = p.starts;
    a.out_stride = p.out_stride;
    if (p.gate_scales) {
        a.ws = p.gate_scales;
        a.us = p.up_scales;
        a.w_stride = p.w_stride;
        a.ws_stride = p.scales_stride;
        if (few_product(p.rows, p.inputs, p.outputs, true)) {
            a.x = p.x;
            a.x_stride = p.x_stride * 2;
            a.pieces = p.inputs;
            return p.type == DHX_F16 ? launch_few_rows<half_t, true>(a, s) : launch_few_rows<bf16_t, true>(a, s);
        }
        const hipError_t err = quantise_rows(p.type, p.x, p.x_stride, p.rows, p.inputs, p.workspace, &a, s);
        if (err != hipSuccess) return err;
        return p.type == DHX_F16 ? launch_product<half_t, true, true>(a, s) : launch_product<bf16_t, true, true>(a, s);
    }
    a.x = p.x;
    a.x_stride = p.x_stride * 2;
    a.w_stride = p.w_stride * 2;
    a.pieces = p.inputs / 8;
    if (const int blocks = few_gated(p.rows, p.inputs, p.outputs))
        return p.type == DHX_F16 ? launch_few_gated<half_t>(a, blocks, s) : launch_few_gated<bf16_t>(a, blocks, s);
    return p.type == DHX_F16 ? launch_product<half_t, false, true>(a, s) : launch_product<bf16_t, false, true>(a, s);
}

}  // namespace dhx
