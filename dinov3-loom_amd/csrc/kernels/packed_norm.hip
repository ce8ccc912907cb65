// The residual step behind a block of a packed batch, with the norms before and
// behind it (include/dinov3_packed.h): x' = x + gate[s] scale post(y), h =
// pre(x'). Each row of x and y is read once and held in registers through both
// norms (over 16384 channels partly in scratch), x' and h are written once, and there is
// little arithmetic, so the kernel is bound by memory (few rows: by one row's chain of
// loads, sums and stores).
#include <algorithm>
#include <climits>
#include <type_traits>

#include "packed.hpp"

namespace dhx {
namespace {

#define DHX_NORM_PARAMS Addr x_, Addr y_, Addr x_out_, Addr h_, int rows, int channels, uint64_t x_stride, uint64_t y_stride, Addr starts_, Addr scale_, Addr gate_, Addr post_weight_, Addr post_bias_, Addr pre_weight_, Addr pre_bias_, uint64_t x_out_stride, uint64_t h_stride, uint64_t gate_stride, int sequences, int post, int pre, float post_eps, float pre_eps

// The sum of v over the G lanes (G <= 64: of a wave, else all of the workgroup) that
// hold a row, in all of them, by the same tree in each: inside rows of 16 lanes by
// moves between lanes (G at least 8), then across them. part: a float for each of 16
// waves, zeros behind the last.
template <int G>
__device__ __forceinline__ float row_sum(float v, float* part) {
    auto move = [](float a, auto ctrl) {
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, a), decltype(ctrl)::value, 0xf, 0xf, false));
    };
    v += move(v, std::integral_constant<int, 0xb1>{});   // quad_perm 1, 0, 3, 2
    v += move(v, std::integral_constant<int, 0x4e>{});   // quad_perm 2, 3, 0, 1
    v += move(v, std::integral_constant<int, 0x141>{});  // row_half_mirror
    if constexpr (G >= 16) v += move(v, std::integral_constant<int, 0x140>{});  // row_mirror
    if constexpr (G >= 32) v += __shfl_xor(v, 16);
    if constexpr (G >= 64) v = half_pair_sum(v);
    if constexpr (G > 64) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        if (lane == 0) part[wave] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int w = 0; w < 16; ++w) v += part[w];
    }
    return v;
}

// The value of a row's first lane (of those of row_sum), in all of them.
template <int G>
__device__ __forceinline__ float row_first(float v, float* part) {
    if constexpr (G < 64) {
        int first = __builtin_bit_cast(int, v);
        first = __builtin_amdgcn_update_dpp(first, first, 0x000, 0xf, 0xf, false);  // quad_perm 0, 0, 0, 0
        first = __builtin_amdgcn_update_dpp(first, first, 0x114, 0xf, 0xa, false);  // row_shr:4 into lanes 4-7 and 12-15
        if constexpr (G >= 16) first = __builtin_amdgcn_update_dpp(first, first, 0x118, 0xf, 0xc, false);  // row_shr:8 into lanes 8-15
        if constexpr (G >= 32) first = __builtin_amdgcn_update_dpp(first, first, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
        return __builtin_bit_cast(float, first);
    }
    if constexpr (G == 64) return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
    if (threadIdx.x == 0) *part = v;
    __syncthreads();
    return *part;
}

// The last sequence that does not begin behind row0 + mine, one of the ROWS rows
// from row0 on that a wave holds; -1: none.
template <int ROWS>
__device__ __forceinline__ int sequence_of(const int32_t* starts, int sequences, int rows, int row0, int mine) {
    int at = -1;
    if (sequences <= 64) {
        const int lane = threadIdx.x & 63, first = lane < sequences ? start_at(starts, lane, rows) : INT_MAX;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int n = __builtin_popcountll(__ballot(first <= row0 + r));
            if (mine == r) at = n - 1;
        }
    } else {
        for (int r = 0; r < ROWS; ++r) {
            const int last = wave_last(sequences, row0 + r, [&](int s) { return (int64_t)start_at(starts, s, rows); });
            if (mine == r) at = last;
        }
    }
    return at;
}

template <class S>
__device__ __forceinline__ void load8(const S* p, float (&v)[8]) {
    if constexpr (std::is_same_v<S, float>) {
        const float4_t a = *(const float4_t*)p, b = *(const float4_t*)(p + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < 4 ? a[e] : b[e - 4];
    } else {
        const typename Num<S>::v8 a = *(const typename Num<S>::v8*)p;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)a[e];
    }
}
// 8 values from element `at` of rows on: 16-bit ones through the L2 (12864 rows of 384
// channels 11.0 us, 11.5 without), float32 ones, of which an instruction stores half a
// line only, not (5,000,000 values 14.0 us, through it 17.5).
template <class S>
struct Rows {
    S* first;
    WtOut through;
    __device__ __forceinline__ explicit Rows(S* p) : first(p), through(p, ~0u) {}
    __device__ __forceinline__ void store8(uint32_t at, const float (&v)[8]) const {
        if constexpr (std::is_same_v<S, float>) {
            *(float4_t*)(first + at) = float4_t{v[0], v[1], v[2], v[3]};
            *(float4_t*)(first + at + 4) = float4_t{v[4], v[5], v[6], v[7]};
        } else {
            typename Num<S>::v8 a;
#pragma unroll
            for (int e = 0; e < 8; ++e) a[e] = (S)v[e];
            through.store(at * 2, a);
        }
    }
};

// A channel vector's piece; ones or zeros where there is no vector.
__device__ __forceinline__ void vector8(const float* vector, int c, float none, float (&v)[8]) {
    if (vector) {
        load8(vector + c, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = none;
    }
}

// One over the row's root of its mean square, of P pieces of 8 channels a lane
// (zeros where a piece does not exist); for LayerNorm of the deviations from the
// mean, which it leaves in v.
// A mean is off by some 30 roundings of itself (8 values of a lane, 6 steps across lanes, 16
// waves), which deviations far smaller than the mean would show: a float32 row of one
// value would have some, and its norm nothing else. Where the mean is more than 128 times
// the deviations, which are exact so near to it, these are therefore taken from the first
// of them, so that nothing is left of a row of one value, and then from their own mean.
// Other rows pay a comparison (12864 rows of 384 channels 10.84 us without it and with;
// most where both norms wait for several waves: 4882 rows of 1024 12.5 and 13.0, 24 rows of
// 8192 4.23 and 4.45; holding the mean between every row's least and largest value took
// 11.4, 14.5 and 4.69).
// part: 48 floats, of which the last 16 are any.
template <int G, int P>
__device__ __forceinline__ float inverse(float (&v)[P][8], const bool (&there)[P], int kind, float eps, int channels, float* part) {
    const float each = 1.0f / (float)channels;
    auto less = [&](float mean) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[p][e] = there[p] ? v[p][e] - mean : 0.f;
    };
    auto mean_of = [&]() __attribute__((always_inline)) {
        float sum = 0.f;
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += v[p][e];
        return row_sum<G>(sum, part) / (float)channels;
    };
    auto square = [&]() __attribute__((always_inline)) {
        float sum = 0.f;
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf(v[p][e], v[p][e], sum);
        return row_sum<G>(sum, part + 16);
    };
    float mean = 0.f;
    if (kind == DHX_NORM_LAYER) {
        mean = mean_of();
        less(mean);
    }
    float all = square();
    if (kind == DHX_NORM_LAYER) {
        const bool near = mean != 0.f && all * each <= mean * mean * 0x1p-14f;
        if (__any(near)) {
            const float first = row_first<G>(v[0][0], part + 32);
            less(near ? first : 0.f);
            const float more = mean_of();
            less(near ? more : 0.f);
            all = square();
        }
    }
    return rsqrtf(fmaf(all, each, eps));
}

// T: y and h, S: x and x'. G lanes (over 64: those of the workgroup, however many)
// hold a row, P pieces of 8 channels each: piece p of lane l is G p + l of the row.
template <class T, class S, int G, int P>
__global__ __launch_bounds__(G <= 64 ? 256 : G) void packed_norm_kernel(DHX_NORM_PARAMS) {
    constexpr int ROWS = G <= 64 ? 256 / G : 1, WAVE_ROWS = G <= 64 ? 64 / G : 1;
    __shared__ float part[G > 64 ? 96 : 1];  // for each norm 16 waves' sums, of two kinds, and a value
    const S* x = x_;
    const T* y = y_;
    const int tid = threadIdx.x, lanes = G <= 64 ? G : blockDim.x, lane = G <= 64 ? tid % G : tid, in_wave = G <= 64 ? (tid & 63) / G : 0;
    const int pieces = channels >> 3;
    bool there[P];
    int at[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        there[p] = lanes * p + lane < pieces;
        at[p] = (lanes * p + lane) * 8;
    }
    if (G > 64 && tid < 96 && tid % 16 >= lanes >> 6) part[tid] = 0.f;
    for (int64_t first = (int64_t)blockIdx.x * ROWS; first < rows; first += (int64_t)gridDim.x * ROWS) {
        const int in_block = G <= 64 ? tid / G : 0;
        const int64_t row = first + in_block;
        const Rows<S> x_rows((S*)x_out_ + first * x_out_stride);
        const Rows<T> h_rows((T*)h_ + first * h_stride);
        const int32_t* starts = starts_;
        bool in = row < rows;
        int s = 0;
        if (gate_.a) {
            s = sequence_of<WAVE_ROWS>(starts, sequences, rows, (int)(row - in_wave), in_wave);
            in = in && s >= 0 && row < start_at(starts, s + 1, rows);
        } else if (starts_.a) {
            in = in && row >= start_at(starts, 0, rows) && row < start_at(starts, sequences, rows);
        }
        float v[P][8], z[P][8];
#pragma unroll
        for (int p = 0; p < P; ++p) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[p][e] = z[p][e] = 0.f;
            if (in && there[p]) {
                load8(x + row * x_stride + at[p], v[p]);
                if (y) load8(y + row * y_stride + at[p], z[p]);
            }
        }
        // x' = x + (y' r) by + plus
        auto step_vectors = [&](int p, float (&by)[8], float (&plus)[8]) __attribute__((always_inline)) {
            const int c = there[p] ? at[p] : 0;
            float scale[8], gate[8];
            vector8(post_weight_, c, 1.f, by);
            vector8(post_bias_, c, 0.f, plus);
            vector8(scale_, c, 1.f, scale);
            vector8(gate_.a ? (const float*)gate_ + max(s, 0) * gate_stride : nullptr, c, 1.f, gate);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                scale[e] *= gate[e];
                by[e] *= scale[e];
                plus[e] *= scale[e];
            }
        };
        auto pre_vectors = [&](int p, float (&by)[8], float (&plus)[8]) __attribute__((always_inline)) {
            const int c = there[p] ? at[p] : 0;
            vector8(pre_weight_, c, 1.f, by);
            vector8(pre_bias_, c, 0.f, plus);
        };
        // With one piece per lane the vectors are loaded in front of the first sum, so that
        // one latency is waited for; those of more pieces would not fit in registers.
        float by[8], plus[8], pre_by[8], pre_plus[8];
        if constexpr (P == 1) {
            if (y) step_vectors(0, by, plus);
            if (pre != DHX_NORM_NONE) pre_vectors(0, pre_by, pre_plus);
        }
        if (y) {
            const float r = post != DHX_NORM_NONE ? inverse<G, P>(z, there, post, post_eps, channels, part) : 1.f;
#pragma unroll
            for (int p = 0; p < P; ++p) {
                if constexpr (P > 1) step_vectors(p, by, plus);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[p][e] = there[p] ? v[p][e] + fmaf(z[p][e] * r, by[e], plus[e]) : 0.f;
                if (in && there[p]) x_rows.store8(in_block * (uint32_t)x_out_stride + at[p], v[p]);
            }
        }
        if (pre != DHX_NORM_NONE) {
            const float r = inverse<G, P>(v, there, pre, pre_eps, channels, part + (G > 64 ? 48 : 0));
#pragma unroll
            for (int p = 0; p < P; ++p) {
                if constexpr (P > 1) pre_vectors(p, pre_by, pre_plus);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[p][e] = fmaf(v[p][e] * r, pre_by[e], pre_plus[e]);
                if (in && there[p]) h_rows.store8(in_block * (uint32_t)h_stride + at[p], v[p]);
            }
        }
        if (G > 64) __syncthreads();  // part, for the next row
    }
}

constexpr uint64_t kMostBlocks = 1u << 21;  // a launch has fewer than 2^32 threads; workgroups take further rows in turn

template <class T, class S, int G, int P>
hipError_t launch(const dhx_packed_norm& p, hipStream_t s) {
    constexpr int ROWS = G <= 64 ? 256 / G : 1;
    const uint32_t threads = G <= 64 ? 256 : (p.channels / 8 + 64 * P - 1) / (64 * P) * 64;
    const uint64_t blocks = std::min<uint64_t>((p.rows + ROWS - 1) / ROWS, kMostBlocks);
    return enqueue(packed_norm_kernel<T, S, G, P>, dim3((unsigned)blocks), dim3(threads), 0, s, p.x, p.y, p.x_out, p.h, (int)p.rows,
                   (int)p.channels, p.x_stride, p.y_stride, p.starts, p.scale, p.gate, p.post_weight, p.post_bias, p.pre_weight,
                   p.pre_bias, p.x_out_stride, p.h_stride, p.gate_stride, (int)p.sequences, (int)p.post, (int)p.pre, p.post_eps,
                   p.pre_eps);
}

template <class T, class S>
hipError_t launch_pieces(const dhx_packed_norm& p, hipStream_t s) {
    const uint32_t pieces = p.channels / 8;
    // A lane per piece, and as few lanes as that leaves idle: 39 MB of 384 channels, 64
    // lanes 11.1 us, 32 lanes of two pieces 13.2, 128 lanes 18.4; of 2048, 256 lanes
    // 11.3, 128 of two 11.5, 64 of four 19.5, 512 lanes 15.2. A workgroup has at most 1024
    // lanes, so that longer rows are two and four pieces a lane, and four do not fit in a
    // lane's 128 registers: 31 to 35 of them are kept in scratch (128 to 144 bytes a lane),
    // and 39 MB of 32768 channels take 20.2 us where as many bytes of 4096 take 11.2, one
    // row 17 us and 3.1.
    if (pieces <= 8) return launch<T, S, 8, 1>(p, s);
    if (pieces <= 16) return launch<T, S, 16, 1>(p, s);
    if (pieces <= 32) return launch<T, S, 32, 1>(p, s);
    if (pieces <= 64) return launch<T, S, 64, 1>(p, s);
    if (pieces <= 1024) return launch<T, S, 1024, 1>(p, s);
    if (pieces <= 2048) return launch<T, S, 1024, 2>(p, s);
    return launch<T, S, 1024, 4>(p, s);
}

template <class T>
hipError_t launch_type(const dhx_packed_norm& p, hipStream_t s) {
    return p.stream_type == DHX_F32 ? launch_pieces<T, float>(p, s) : launch_pieces<T, T>(p, s);
}

}  // namespace

hipError_t launch_packed_norm(const dhx_packed_norm& p, hipStream_t s) {
    return p.type == DHX_F16 ? launch_type<half_t>(p, s) : launch_type<bf16_t>(p, s);
}

}  // namespace dhx
