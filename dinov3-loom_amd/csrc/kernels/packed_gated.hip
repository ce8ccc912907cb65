// The gated projections of a feed-forward block on packed batches
// (include/dinov3_packed.h): out = act(x Wg^T + bg) (x Wu^T + bu), one product
// kernel whose tiles hold rows of both matrices (packed_product.hpp), with weights in
// 16 bits, or in 4 behind the kernel that quantises x (packed_quantise.hip); few rows
// against 4 bits have a kernel that does both.
#include "packed_product.hpp"

namespace dhx {

uint64_t packed_gated_bytes(const dhx_packed_gated& p) {
    return p.gate_scales && !few_product(p.rows, p.inputs, p.outputs, true) ? quantised_rows_bytes(p.rows, p.inputs) : 0;
}

hipError_t launch_packed_gated(const dhx_packed_gated& p, hipStream_t s) {
    Product a{};
    a.type = p.type;
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
    return p.type == DHX_F16 ? launch_product<half_t, false, true>(a, s) : launch_product<bf16_t, false, true>(a, s);
}

}  // namespace dhx
