// The operators on packed batches behind the C ABI of include/dinov3_packed.h:
// argument checks, then the launch on the caller's stream.
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>
#include <utility>

#include "../../include/dinov3_packed.h"
#include "engine_internal.hpp"
#include "errors.hpp"
#include "kernels/packed.hpp"

namespace {

using dhx::Error;

// No size or stride reaches past this, so that a row number and the bytes
// that a tile of 256 rows spans fit in 32 bits.
constexpr uint64_t kMaxRows = 0x7fffffff - 256;
constexpr uint64_t kMaxStride = 1u << 22;
// A launch has fewer than 2^32 threads: 256 to each 32 rows of a projection, 512
// to a tile of 256 x 256, and 256 to each row tile of attention.
constexpr uint64_t kMaxLinearRows = 1u << 27, kMaxLinearTiles = 1u << 22, kMaxRowTiles = 1u << 23;

void positive(uint64_t v, const char* what) {
    if (v == 0) throw Error(std::string(what) + " must be positive");
}

void eights(uint64_t v, const char* what) {
    if (v == 0 || v % 8 != 0) throw Error(std::string(what) + " must be a positive multiple of 8");
}

void most(uint64_t v, uint64_t limit, const char* what) {
    if (v > limit) throw Error(std::string(what) + " must be at most " + std::to_string(limit));
}

// `needed` false: there are no rows to read or write, and a null is fine.
void pointer(const void* p, uint64_t align, const char* what, bool needed = true) {
    if (!p && !needed) return;
    if (!p) throw Error(std::string(what) + " is a null device pointer");
    if (reinterpret_cast<uintptr_t>(p) % align != 0)
        throw Error(std::string(what) + " must be " + std::to_string(align) + "-byte aligned");
}

void stride(uint64_t v, uint64_t least, const char* what) {
    if (v % 8 != 0) throw Error(std::string(what) + " must be a multiple of 8");
    if (v < least) throw Error(std::string(what) + " must be at least " + std::to_string(least));
    most(v, kMaxStride, what);
}

void type_of(uint32_t type) {
    if (type != DHX_F16 && type != DHX_BF16) throw Error("type must be DHX_F16 or DHX_BF16");
}

void workspace(const void* p, uint64_t have, uint64_t need) {
    if (need == 0) return;
    if (have < need)
        throw Error("the workspace has " + std::to_string(have) + " bytes, the call needs " + std::to_string(need));
    pointer(p, 16, "workspace");
}

void linear_sizes(const dhx_packed_linear& p) {
    type_of(p.type);
    positive(p.sequences, "sequences");
    most(p.sequences, kMaxRows, "sequences");
    most(p.rows, kMaxLinearRows, "rows");
    eights(p.inputs, "inputs");
    eights(p.outputs, "outputs");
    eights(p.rank, "rank");
    positive(p.adapters, "adapters");
    most(p.inputs, kMaxStride, "inputs");
    most(p.outputs, kMaxStride, "outputs");
    most(p.rank, 256, "rank");
    most(p.adapters, kMaxRows, "adapters");
    most(((p.rows + 255) / 256) * ((p.outputs + 255) / 256), kMaxLinearTiles,
         "the number of tiles of 256 x 256 outputs");
}

void linear_check(const dhx_packed_linear& p) {
    linear_sizes(p);
    pointer(p.x, 16, "x", p.rows > 0);
    pointer(p.w, 16, "w");
    if (p.bias) pointer(p.bias, 16, "bias");
    pointer(p.a, 16, "a");
    pointer(p.b, 16, "b");
    pointer(p.scale, 4, "scale");
    pointer(p.y, 16, "y", p.rows > 0);
    pointer(p.starts, 4, "starts");
    pointer(p.adapter, 4, "adapter");
    stride(p.x_stride, p.inputs, "x_stride");
    stride(p.w_stride, p.inputs, "w_stride");
    stride(p.y_stride, p.outputs, "y_stride");
    workspace(p.workspace, p.workspace_bytes, dhx::packed_linear_bytes(p));
}

void rotation_check(const dhx_packed_rotation& p) {
    type_of(p.type);
    if (p.neighbours > 1) throw Error("neighbours must be 0 or 1");
    most(p.rows, kMaxRows, "rows");
    positive(p.heads, "heads");
    eights(p.head_dim, "head_dim");
    const bool part = (uint64_t)p.rotated * 2 == p.head_dim || p.rotated == p.head_dim;
    if (p.rotated == 0 || p.rotated % (part ? 8 : 16) != 0)
        throw Error("rotated must be a positive multiple of 16, or a multiple of 8 that is head_dim or half of it");
    if (p.rotated > p.head_dim) throw Error("rotated must be at most head_dim");
    positive(p.places, "places");
    most(p.places, kMaxRows, "places");
    most((uint64_t)p.heads * p.head_dim, kMaxStride, "heads * head_dim");
    pointer(p.x, 16, "x", p.rows > 0);
    pointer(p.out, 16, "out", p.rows > 0);
    pointer(p.cos, 16, "cos");
    pointer(p.sin, 16, "sin");
    pointer(p.index, 4, "index", p.rows > 0);
    stride(p.x_stride, (uint64_t)p.heads * p.head_dim, "x_stride");
    stride(p.out_stride, (uint64_t)p.heads * p.head_dim, "out_stride");
    if (p.rows > 0 && p.x == p.out && p.x_stride != p.out_stride) throw Error("in place, out_stride must be x_stride");
}

dhx_packed_attention with_head_strides(const dhx_packed_attention& p) {
    dhx_packed_attention a = p;
    for (uint64_t* s : {&a.q_head_stride, &a.k_head_stride, &a.v_head_stride, &a.out_head_stride})
        if (*s == 0) *s = p.head_dim;
    return a;
}

void attention_sizes(const dhx_packed_attention& p) {
    type_of(p.type);
    if (p.causal > 1) throw Error("causal must be 0 or 1");
    if (p.reserved != 0) throw Error("reserved must be 0");
    positive(p.sequences, "sequences");
    most(p.sequences, kMaxRows, "sequences");
    positive(p.kv_heads, "kv_heads");
    positive(p.heads, "heads");
    most(p.heads, 65536, "heads");
    if (p.heads % p.kv_heads != 0) throw Error("heads must be a multiple of kv_heads");
    eights(p.head_dim, "head_dim");
    most(p.head_dim, 128, "head_dim");
    most(p.q_rows, kMaxRows, "q_rows");
    most(p.k_rows, kMaxRows, "k_rows");
    const uint64_t rows = p.q_rows * (p.heads / p.kv_heads);
    most(rows, kMaxRows, "q_rows * (heads / kv_heads)");
    most(p.q_rows + p.k_rows, kMaxRows, "q_rows + k_rows");
    most((rows / 32 + p.sequences) * p.kv_heads, kMaxRowTiles, "the number of row tiles");
}

void attention_check(const dhx_packed_attention& p) {
    attention_sizes(p);
    if (!(p.scale > 0) || !std::isfinite(p.scale)) throw Error("scale must be positive and finite");
    if (p.scale > 1048576.0f) throw Error("scale must be at most 2^20");  // times a row's first maximum it stays finite
    pointer(p.q, 16, "q", p.q_rows > 0);
    pointer(p.k, 16, "k", p.k_rows > 0);
    pointer(p.v, 16, "v", p.k_rows > 0);
    pointer(p.out, 16, "out", p.q_rows > 0);
    if (p.lse) pointer(p.lse, 4, "lse");
    pointer(p.q_starts, 4, "q_starts");
    pointer(p.k_starts, 4, "k_starts");
    stride(p.q_stride, p.head_dim, "q_stride");
    stride(p.k_stride, p.head_dim, "k_stride");
    stride(p.v_stride, p.head_dim, "v_stride");
    stride(p.out_stride, p.head_dim, "out_stride");
    // Heads may lie behind each other in a row, or each in a matrix of its own.
    for (uint64_t s : {p.q_head_stride, p.k_head_stride, p.v_head_stride, p.out_head_stride}) {
        if (s % 8 != 0) throw Error("head strides must be multiples of 8");
        if (s < p.head_dim) throw Error("head strides must be at least head_dim");
        if (s > (1ull << 40)) throw Error("head strides must be at most 2^40");
    }
    const uint64_t inner = (p.heads - 1) * p.out_head_stride + p.head_dim;
    const uint64_t outer = (p.q_rows ? p.q_rows - 1 : 0) * p.out_stride + p.head_dim;
    if (p.heads > 1 && p.out_stride < inner && p.out_head_stride < outer)
        throw Error("out_stride and out_head_stride make heads overlap");
    workspace(p.workspace, p.workspace_bytes, dhx::packed_attention_cut(p).bytes);
}

// Starts may be missing in the calls of the feed-forward half: then all rows count.
void optional_starts(const int32_t* starts, uint32_t sequences) {
    most(sequences, kMaxRows, "sequences");
    if (starts) {
        positive(sequences, "sequences");
        pointer(starts, 4, "starts");
    } else if (sequences != 0) {
        throw Error("starts is a null device pointer");
    }
}

void norm_check(const dhx_packed_norm& p) {
    type_of(p.type);
    if (p.stream_type != p.type && p.stream_type != DHX_F32) throw Error("stream_type must be type or DHX_F32");
    for (uint32_t kind : {p.post, p.pre})
        if (kind > DHX_NORM_LAYER) throw Error("post and pre must be DHX_NORM_NONE, DHX_NORM_RMS or DHX_NORM_LAYER");
    most(p.rows, kMaxRows, "rows");
    eights(p.channels, "channels");
    most(p.channels, 32768, "channels");
    for (float eps : {p.post_eps, p.pre_eps})
        if (!(eps >= 0) || !std::isfinite(eps)) throw Error("post_eps and pre_eps must be finite and not negative");
    optional_starts(p.starts, p.sequences);
    const bool work = p.rows > 0;
    pointer(p.x, 16, "x", work);
    stride(p.x_stride, p.channels, "x_stride");
    if (p.y) {
        pointer(p.y, 16, "y");
        pointer(p.x_out, 16, "x_out", work);
        stride(p.y_stride, p.channels, "y_stride");
        stride(p.x_out_stride, p.channels, "x_out_stride");
        if (work && p.x == p.x_out && p.x_stride != p.x_out_stride) throw Error("in place, x_out_stride must be x_stride");
        if (work && p.y == p.x_out && (p.type != p.stream_type || p.y_stride != p.x_out_stride))
            throw Error("x_out in the place of y must have its type, and x_out_stride be y_stride");
    } else if (work && (p.post != DHX_NORM_NONE || p.pre == DHX_NORM_NONE || p.scale || p.gate || p.x_out)) {
        throw Error("without y there are no post, scale, gate and x_out, and pre is needed");
    }
    if (p.pre != DHX_NORM_NONE) {
        pointer(p.h, 16, "h", work);
        stride(p.h_stride, p.channels, "h_stride");
        if (p.h && p.h == p.y && p.h_stride != p.y_stride) throw Error("in place, h_stride must be y_stride");
        if (work && p.h == p.x && (p.type != p.stream_type || p.h_stride != p.x_stride))
            throw Error("h in the place of x must have its type, and h_stride be x_stride");
        if (work && p.h == p.x_out) throw Error("h and x_out must not be the same");
    } else if (p.h) {
        throw Error("h needs a norm in pre");
    }
    const std::pair<const float*, const char*> vectors[] = {{p.post_weight, "post_weight"}, {p.post_bias, "post_bias"},
                                                            {p.pre_weight, "pre_weight"},   {p.pre_bias, "pre_bias"},
                                                            {p.scale, "scale"},             {p.gate, "gate"}};
    for (const auto& [v, what] : vectors) pointer(v, 16, what, false);
    if (p.post == DHX_NORM_NONE && (p.post_weight || p.post_bias)) throw Error("post_weight and post_bias need a norm in post");
    if (p.pre == DHX_NORM_NONE && (p.pre_weight || p.pre_bias)) throw Error("pre_weight and pre_bias need a norm in pre");
    if (p.gate) {
        if (!p.starts) throw Error("gate needs starts");
        stride(p.gate_stride, p.channels, "gate_stride");
    }
}

// A stride in bytes, of codes or scales.
void byte_stride(uint64_t v, uint64_t least, const char* what) {
    if (v % 16 != 0) throw Error(std::string(what) + " must be a multiple of 16");
    if (v < least) throw Error(std::string(what) + " must be at least " + std::to_string(least));
    most(v, 2 * kMaxStride, what);
}

void quantisation_check(const dhx_packed_quantisation& p) {
    type_of(p.type);
    if (p.reserved != 0) throw Error("reserved must be 0");
    most(p.rows, kMaxRows, "rows");
    eights(p.columns, "columns");
    most(p.columns, kMaxStride, "columns");
    optional_starts(p.starts, p.sequences);
    pointer(p.x, 16, "x", p.rows > 0);
    pointer(p.codes, 16, "codes", p.rows > 0);
    pointer(p.scales, 16, "scales", p.rows > 0);
    stride(p.x_stride, p.columns, "x_stride");
    byte_stride(p.codes_stride, dhx::code_bytes(p.columns), "codes_stride");
    byte_stride(p.scales_stride, dhx::scale_bytes(p.columns), "scales_stride");
}

// What the two products of the feed-forward half have in common.
void product_sizes(uint32_t type, uint64_t rows, uint32_t inputs, uint32_t outputs) {
    type_of(type);
    most(rows, kMaxLinearRows, "rows");
    eights(inputs, "inputs");
    eights(outputs, "outputs");
    most(inputs, kMaxStride, "inputs");
    most(outputs, kMaxStride, "outputs");
    most(((rows + 255) / 256) * ((outputs + 127) / 128), kMaxLinearTiles / 2, "the number of tiles of 256 x 128 outputs");
}

void quantised_linear_sizes(const dhx_packed_quantised_linear& p) { product_sizes(p.type, p.rows, p.inputs, p.outputs); }

void quantised_linear_check(const dhx_packed_quantised_linear& p) {
    quantised_linear_sizes(p);
    optional_starts(p.starts, p.sequences);
    pointer(p.x, 16, "x", p.rows > 0);
    pointer(p.w, 16, "w");
    pointer(p.w_scales, 16, "w_scales");
    pointer(p.bias, 16, "bias", false);
    pointer(p.y, 16, "y", p.rows > 0);
    stride(p.x_stride, p.inputs, "x_stride");
    stride(p.y_stride, p.outputs, "y_stride");
    byte_stride(p.w_stride, dhx::code_bytes(p.inputs), "w_stride");
    byte_stride(p.scales_stride, dhx::scale_bytes(p.inputs), "scales_stride");
    workspace(p.workspace, p.workspace_bytes, dhx::packed_quantised_linear_bytes(p));
}

void gated_sizes(const dhx_packed_gated& p) {
    product_sizes(p.type, p.rows, p.inputs, p.outputs);
    if (!p.gate_scales != !p.up_scales) throw Error("gate_scales and up_scales come together");
}

void gated_check(const dhx_packed_gated& p) {
    gated_sizes(p);
    if (p.activation > DHX_SIGMOID) throw Error("activation must be one of DHX_SILU to DHX_SIGMOID");
    if (p.reserved != 0) throw Error("reserved must be 0");
    optional_starts(p.starts, p.sequences);
    pointer(p.x, 16, "x", p.rows > 0);
    pointer(p.gate, 16, "gate");
    pointer(p.up, 16, "up");
    pointer(p.gate_bias, 16, "gate_bias", false);
    pointer(p.up_bias, 16, "up_bias", false);
    pointer(p.out, 16, "out", p.rows > 0);
    stride(p.x_stride, p.inputs, "x_stride");
    stride(p.out_stride, p.outputs, "out_stride");
    if (p.gate_scales) {
        pointer(p.gate_scales, 16, "gate_scales");
        pointer(p.up_scales, 16, "up_scales");
        byte_stride(p.w_stride, dhx::code_bytes(p.inputs), "w_stride");
        byte_stride(p.scales_stride, dhx::scale_bytes(p.inputs), "scales_stride");
    } else {
        stride(p.w_stride, p.inputs, "w_stride");
    }
    workspace(p.workspace, p.workspace_bytes, dhx::packed_gated_bytes(p));
}

// The caller's current device again on every way out.
class KeepDevice {
public:
    explicit KeepDevice(int device) : device_(device) {
        if (hipGetDevice(&prev_) != hipSuccess) prev_ = -1;
        err_ = prev_ == device_ ? hipSuccess : hipSetDevice(device_);
    }
    ~KeepDevice() {
        if (prev_ >= 0 && prev_ != device_) (void)hipSetDevice(prev_);
    }
    KeepDevice(const KeepDevice&) = delete;
    KeepDevice& operator=(const KeepDevice&) = delete;
    hipError_t error() const { return err_; }

private:
    int device_, prev_ = -1;
    hipError_t err_;
};

template <class F>
int guarded(dhx_engine* e, F&& f) {
    try {
        f();
        return 0;
    } catch (const std::exception& ex) {
        if (e) dhx::engine_set_error(e, ex.what());
        else dhx::set_global_error(ex.what());
        return 1;
    }
}

// Checks, then queues one operator; `work` false: nothing to do.
template <class P, class Check, class Launch>
int run(dhx_engine* e, const P* p, void* stream, Check check, Launch launch) {
    return guarded(e, [&] {
        if (!p) throw Error("null argument");
        const bool work = check(*p);
        if (!e) throw Error("null engine");
        dhx::engine_ensure_usable(e);
        if (!work) return;
        const KeepDevice keep(dhx::engine_device(e));
        dhx::engine_check(e, keep.error(), "hipSetDevice");
        dhx::engine_check(e, launch(*p, static_cast<hipStream_t>(stream)), "kernel launch");
    });
}

}  // namespace

extern "C" {

int dhx_packed_linear_workspace(const dhx_packed_linear* p, uint64_t* bytes) {
    return guarded(nullptr, [&] {
        if (!p || !bytes) throw Error("null argument");
        linear_sizes(*p);
        *bytes = dhx::packed_linear_bytes(*p);
    });
}

int dhx_packed_linear_run(dhx_engine* e, const dhx_packed_linear* p, void* stream) {
    return run(
        e, p, stream,
        [](const dhx_packed_linear& a) {
            linear_check(a);
            return a.rows > 0;
        },
        dhx::launch_packed_linear);
}

int dhx_packed_rotation_run(dhx_engine* e, const dhx_packed_rotation* p, void* stream) {
    return run(
        e, p, stream,
        [](const dhx_packed_rotation& a) {
            rotation_check(a);
            return a.rows > 0;
        },
        dhx::launch_packed_rotation);
}

int dhx_packed_attention_workspace(const dhx_packed_attention* p, uint64_t* bytes) {
    return guarded(nullptr, [&] {
        if (!p || !bytes) throw Error("null argument");
        attention_sizes(*p);
        *bytes = dhx::packed_attention_cut(*p).bytes;
    });
}

int dhx_packed_attention_run(dhx_engine* e, const dhx_packed_attention* p, void* stream) {
    return run(
        e, p, stream,
        [](const dhx_packed_attention& a) {
            attention_check(with_head_strides(a));
            return a.q_rows > 0;
        },
        [](const dhx_packed_attention& a, hipStream_t s) { return dhx::launch_packed_attention(with_head_strides(a), s); });
}

int dhx_packed_norm_run(dhx_engine* e, const dhx_packed_norm* p, void* stream) {
    return run(
        e, p, stream,
        [](const dhx_packed_norm& a) {
            norm_check(a);
            return a.rows > 0;
        },
        dhx::launch_packed_norm);
}

int dhx_packed_quantise_run(dhx_engine* e, const dhx_packed_quantisation* p, void* stream) {
    return run(
        e, p, stream,
        [](const dhx_packed_quantisation& a) {
            quantisation_check(a);
            return a.rows > 0;
        },
        [](const dhx_packed_quantisation& a, hipStream_t s) { return dhx::launch_packed_quantise(a, s); });
}

int dhx_packed_dequantise_run(dhx_engine* e, const dhx_packed_quantisation* p, void* stream) {
    return run(
        e, p, stream,
        [](const dhx_packed_quantisation& a) {
            quantisation_check(a);
            return a.rows > 0;
        },
        dhx::launch_packed_dequantise);
}

int dhx_packed_quantised_linear_workspace(const dhx_packed_quantised_linear* p, uint64_t* bytes) {
    return guarded(nullptr, [&] {
        if (!p || !bytes) throw Error("null argument");
        quantised_linear_sizes(*p);
        *bytes = dhx::packed_quantised_linear_bytes(*p);
    });
}

int dhx_packed_quantised_linear_run(dhx_engine* e, const dhx_packed_quantised_linear* p, void* stream) {
    return run(
        e, p, stream,
        [](const dhx_packed_quantised_linear& a) {
            quantised_linear_check(a);
            return a.rows > 0;
        },
        dhx::launch_packed_quantised_linear);
}

int dhx_packed_gated_workspace(const dhx_packed_gated* p, uint64_t* bytes) {
    return guarded(nullptr, [&] {
        if (!p || !bytes) throw Error("null argument");
        gated_sizes(*p);
        *bytes = dhx::packed_gated_bytes(*p);
    });
}

int dhx_packed_gated_run(dhx_engine* e, const dhx_packed_gated* p, void* stream) {
    return run(
        e, p, stream,
        [](const dhx_packed_gated& a) {
            gated_check(a);
            return a.rows > 0;
        },
        dhx::launch_packed_gated);
}

}  // extern "C"
