// Rows of a packed batch to 4-bit codes with a scale per block of 32 values, and
// back (include/dinov3_packed.h). Every value is read once and every code written
// once, or the other way round; there is little arithmetic, so both are bound by
// memory. A lane takes 8 values (16 bytes), four lanes a block. Codes and values are
// stored through the L2 (WtOut, common.hpp): 8192 rows of 4096 to codes and back 36.7
// us without, 34.5 so (168 MB, 4.9 TB/s), 2299 of 1000 5.9 and 5.5.
#include <algorithm>

#include "packed_four.hpp"

namespace dhx {
namespace {

#define DHX_QUANTISE_PARAMS Addr x_, Addr codes_, Addr scales_, int rows, int columns, uint64_t x_stride, uint64_t codes_stride, uint64_t scales_stride, uint64_t group_stride, Addr starts_, int sequences, int block_rows

// Whether the rows of the call hold `row`.
__device__ __forceinline__ bool counts(const int32_t* starts, int sequences, int rows, int64_t row) {
    return !starts || (row >= start_at(starts, 0, rows) && row < start_at(starts, sequences, rows));
}

// A workgroup takes block_rows rows at a time; an item is 8 columns of a row. The
// items of a row are whole blocks and, behind them, what fills the scales up to 16.
template <class T>
__global__ __launch_bounds__(256) void packed_quantise_kernel(DHX_QUANTISE_PARAMS) {
    typedef typename Num<T>::v8 v8;
    const int blocks = (columns + 31) >> 5, per_row = ((blocks + 15) & ~15) * 4;
    for (int64_t row0 = (int64_t)blockIdx.x * block_rows; row0 < rows; row0 += (int64_t)gridDim.x * block_rows) {
        const __amdgpu_buffer_rsrc_t code_rows = __builtin_amdgcn_make_buffer_rsrc((void*)(codes_.a + row0 * codes_stride), 0, -1, kBufferRsrcWord3);
        const int n = (int)min((int64_t)block_rows, rows - row0) * per_row;
        for (int i = threadIdx.x; i < n; i += 256) {  // n is a multiple of 64: whole waves
            const int r = i / per_row, piece = i - r * per_row;
            const int64_t row = row0 + r;
            v8 v = {};
            const bool in = counts(starts_, sequences, rows, row);
            if (in && piece * 8 < columns) v = *(const v8*)((const T*)x_ + row * x_stride + piece * 8);
            const FourBits got = four_bits<T>(v);
            if (!in) continue;
            if (piece < blocks * 4) {
                constexpr int kSc1 = 16;
                __builtin_amdgcn_raw_buffer_store_b32(got.codes, code_rows, (int)((uint32_t)r * (uint32_t)codes_stride + piece * 4), 0, kSc1);
            }
            if ((piece & 3) == 0) {
                const int b = piece >> 2;
                *((uint8_t*)scales_ + (b >> 5) * group_stride + row * scales_stride + (b & 31)) = b < blocks ? (uint8_t)got.scale : 0;
            }
        }
    }
}

template <class T>
__global__ __launch_bounds__(256) void packed_dequantise_kernel(DHX_QUANTISE_PARAMS) {
    typedef typename Num<T>::v8 v8;
    const int per_row = columns >> 3;
    for (int64_t row0 = (int64_t)blockIdx.x * block_rows; row0 < rows; row0 += (int64_t)gridDim.x * block_rows) {
        const WtOut x_rows((const T*)x_ + row0 * x_stride, ~0u);
        const int n = (int)min((int64_t)block_rows, rows - row0) * per_row;
        for (int i = threadIdx.x; i < n; i += 256) {
            const int r = i / per_row, piece = i - r * per_row;
            const int64_t row = row0 + r;
            if (!counts(starts_, sequences, rows, row)) continue;
            const uint32_t c = *(const uint32_t*)((const char*)codes_ + row * codes_stride + piece * 4);
            const float scale = scale_of(*((const uint8_t*)scales_ + row * scales_stride + (piece >> 2)));
            v8 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2_t two = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c >> (8 * e), scale, 0);
                v[2 * e] = (T)two[0];
                v[2 * e + 1] = (T)two[1];
            }
            x_rows.store((uint32_t)r * (uint32_t)x_stride * 2 + piece * 16, v);
        }
    }
}

constexpr uint64_t kMostBlocks = 1u << 21;  // a launch has fewer than 2^32 threads; workgroups take further rows in turn

template <class K>
hipError_t launch(K kernel, const dhx_packed_quantisation& p, uint64_t group_stride, uint64_t per_row, hipStream_t s) {
    const int block_rows = (int)std::max<uint64_t>(256 / per_row, 1);
    const uint64_t blocks = std::min<uint64_t>((p.rows + block_rows - 1) / block_rows, kMostBlocks);
    return enqueue(kernel, dim3((unsigned)blocks), dim3(256), 0, s, p.x, p.codes, p.scales, (int)p.rows, (int)p.columns, p.x_stride,
                   p.codes_stride, p.scales_stride, group_stride, p.starts, (int)p.sequences, block_rows);
}

}  // namespace

hipError_t launch_packed_quantise(const dhx_packed_quantisation& p, hipStream_t s, uint64_t group_stride) {
    const uint64_t per_row = scale_bytes(p.columns) * 4;
    return p.type == DHX_F16 ? launch(packed_quantise_kernel<half_t>, p, group_stride, per_row, s)
                             : launch(packed_quantise_kernel<bf16_t>, p, group_stride, per_row, s);
}

hipError_t launch_packed_dequantise(const dhx_packed_quantisation& p, hipStream_t s) {
    const uint64_t per_row = p.columns / 8;
    return p.type == DHX_F16 ? launch(packed_dequantise_kernel<half_t>, p, 32, per_row, s)
                             : launch(packed_dequantise_kernel<bf16_t>, p, 32, per_row, s);
}

}  // namespace dhx
