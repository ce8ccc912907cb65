// A projection whose weights are held in 4 bits, on packed batches
// (include/dinov3_packed.h). Two kernels: x is quantised into the workspace
// (packed_quantise.hip), then the product of both sides' codes (packed_product.hpp);
// few rows have a kernel that does both.
#include "packed_product.hpp"

namespace dhx {

// Scales as the product reads them, [32 blocks][row][32].
uint64_t quantised_rows_bytes(uint64_t rows, uint64_t columns) { return rows * (code_bytes(columns) + (blocks_of(columns) + 31) / 32 * 32); }

hipError_t quantise_rows(uint32_t type, const void* x, uint64_t x_stride, uint64_t rows, uint32_t columns, void* workspace, Product* product,
                         hipStream_t s) {
    dhx_packed_quantisation q{};
    q.type = type;
    q.rows = rows;
    q.columns = columns;
    q.x = const_cast<void*>(x);
    q.x_stride = x_stride;
    q.codes = static_cast<uint8_t*>(workspace);
    q.codes_stride = code_bytes(columns);
    q.scales = q.codes + rows * q.codes_stride;
    q.scales_stride = 32;
    product->x = q.codes;
    product->x_stride = q.codes_stride;
    product->xs = q.scales;
    product->xs_stride = rows * 32;
    product->pieces = (uint32_t)blocks_of(columns);
    return launch_packed_quantise(q, s, rows * 32);
}

uint64_t packed_quantised_linear_bytes(const dhx_packed_quantised_linear& p) {
    return few_product(p.rows, p.inputs, p.outputs, false) ? 0 : quantised_rows_bytes(p.rows, p.inputs);
}

hipError_t launch_packed_quantised_linear(const dhx_packed_quantised_linear& p, hipStream_t s) {
    Product a{};
    a.rows = (uint32_t)p.rows;
    a.outputs = p.outputs;
    a.sequences = p.sequences;
    a.w = p.w;
    a.ws = p.w_scales;
    a.bias = p.bias;
    a.out = p.y;
    a.starts = p.starts;
    a.w_stride = p.w_stride;
    a.ws_stride = p.scales_stride;
    a.out_stride = p.y_stride;
    if (few_product(p.rows, p.inputs, p.outputs, false)) {
        a.x = p.x;
        a.x_stride = p.x_stride * 2;
        a.pieces = p.inputs;
        return p.type == DHX_F16 ? launch_few_rows<half_t, false>(a, s) : launch_few_rows<bf16_t, false>(a, s);
    }
    const hipError_t err = quantise_rows(p.type, p.x, p.x_stride, p.rows, p.inputs, p.workspace, &a, s);
    if (err != hipSuccess) return err;
    return p.type == DHX_F16 ? launch_product<half_t, true, false>(a, s) : launch_product<bf16_t, true, false>(a, s);
}

}  // namespace dhx
