// Launchers and shared device pieces of the operators on packed batches
// (include/dinov3_packed.h). As in launch.hpp the launchers assume checked
// arguments (csrc/packed.cpp); the row numbers that the kernels read from
// device memory (starts, adapter ids, table indices) are held inside their
// arrays by the kernels themselves.
#pragma once
#include "../../../include/dinov3_packed.h"
#include "launch.hpp"

namespace dhx {

typedef __bf16 bf16_t;
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

// The two 16-bit types the operators take.
template <class T>
struct Num;
template <>
struct Num<half_t> {
    typedef half4_t v4;
    typedef half8_t v8;
    static __device__ __forceinline__ float16_t mfma(v8 a, v8 b, float16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ float4_t mfma16(v8 a, v8 b, float4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Num<bf16_t> {
    typedef bf16x4_t v4;
    typedef bf16x8_t v8;
    static __device__ __forceinline__ float16_t mfma(v8 a, v8 b, float16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ float4_t mfma16(v8 a, v8 b, float4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};

// How a launch is cut; the workspace function and the launcher decide alike.
struct AttentionCut {
    bool few;         // 32-row tiles whose waves share the keys out
    int tile;         // rows of a tile (not few)
    int waves;        // of a workgroup
    uint32_t splits;  // parts of the longest sequence's keys (few only)
    uint64_t span;    // key blocks of 32 in a part
    uint64_t slots;   // workgroups per key head
    uint64_t bytes;   // of workspace
};
AttentionCut packed_attention_cut(const dhx_packed_attention& p);
hipError_t launch_packed_attention(const dhx_packed_attention& p, hipStream_t s);

uint64_t packed_linear_bytes(const dhx_packed_linear& p);
hipError_t launch_packed_linear(const dhx_packed_linear& p, hipStream_t s);

hipError_t launch_packed_rotation(const dhx_packed_rotation& p, hipStream_t s);

hipError_t launch_packed_norm(const dhx_packed_norm& p, hipStream_t s);

// group_stride: from the scales of a row's 32 blocks to those of the next 32 (32: a
// row's scales are one piece).
hipError_t launch_packed_quantise(const dhx_packed_quantisation& p, hipStream_t s, uint64_t group_stride = 32);
hipError_t launch_packed_dequantise(const dhx_packed_quantisation& p, hipStream_t s);

uint64_t packed_quantised_linear_bytes(const dhx_packed_quantised_linear& p);
hipError_t launch_packed_quantised_linear(const dhx_packed_quantised_linear& p, hipStream_t s);

uint64_t packed_gated_bytes(const dhx_packed_gated& p);
hipError_t launch_packed_gated(const dhx_packed_gated& p, hipStream_t s);

// 4-bit rows: a block of 32 values has 16 bytes of codes and a scale byte; a row of
// scales is read 16 bytes at a time.
constexpr uint64_t blocks_of(uint64_t columns) { return (columns + 31) / 32; }
constexpr uint64_t code_bytes(uint64_t columns) { return blocks_of(columns) * 16; }
constexpr uint64_t scale_bytes(uint64_t columns) { return (blocks_of(columns) + 15) / 16 * 16; }

// --- device pieces ---------------------------------------------------------

// 16 bytes of zeros in global memory: what a lane of a DMA load fetches for a
// piece that does not exist (a row behind its sequence, a channel behind a
// head's last).
static __device__ const uint4_t kZeros = {0, 0, 0, 0};

// One DMA load of a wave: each lane's 16 bytes from its own address to LDS at
// `to` (wave-uniform) + 16 * lane.
__device__ __forceinline__ void dma16(const void* from, void* to) {
    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)(uintptr_t)from,
                                     (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// Of the two values in a word, bits 15 and 31: the value is not finite (its
// exponent is ones only). Other bits hold anything.
template <class T>
__device__ __forceinline__ uint32_t not_finite(uint32_t two) {
    constexpr uint32_t EXP = __is_same(T, half_t) ? 0x7c00u : 0x7f80u;
    return (two & (EXP * 0x10001u)) + (0x8000u - EXP) * 0x10001u;
}
template <class T>
__device__ __forceinline__ bool any_not_finite(typename Num<T>::v8 v) {
    const uint4_t w = __builtin_bit_cast(uint4_t, v);
    return ((not_finite<T>(w[0]) | not_finite<T>(w[1]) | not_finite<T>(w[2]) | not_finite<T>(w[3])) & 0x80008000u) != 0;
}

// s_waitcnt vmcnt(N) that the compiler's own wait insertion can see.
template <int N>
__device__ __forceinline__ void wait_vm() {
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_lgkm() {
    __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4));
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Chunk c of LDS row r sits at slot c ^ slot_of(r). 128-byte rows (two per
// pass over the 64 banks): f((r / 2) % 8), f(t) = 4 (t % 2) + t / 2. 256-byte
// rows: 4 (r % 4) + (r / 4) % 4. Either way 16 consecutive rows at one chunk
// (K reads) and 4 consecutive rows at 4 aligned chunks (V transpose reads)
// cover every bank once, rows 8 apart differ in bit 1 and rows 16 apart agree.
template <int PITCH>
__device__ __forceinline__ int slot_of(int r) {
    if constexpr (PITCH == 64) {
        const int t = (r >> 1) & 7;
        return ((t & 1) << 2) | (t >> 1);
    } else {
        return ((r & 3) << 2) | ((r >> 2) & 3);
    }
}
template <int PITCH>
__device__ __forceinline__ int lds_at(int r, int ch) {
    return r * PITCH + (((ch >> 3) ^ slot_of<PITCH>(r)) << 3) + (ch & 7);
}

// Row `s` of a starts array, held inside 0 .. rows.
__device__ __forceinline__ int start_at(const int32_t* starts, int s, int rows) {
    return min(max(starts[s], 0), rows);
}

// The last s of 0 .. n-1 with key(s) <= x, where key does not decrease; -1 if
// there is none. 64 values are looked at in each round, one per lane, so a
// batch of up to 64 sequences costs one load's latency. The result lies inside
// the range whatever key returns.
template <class Key>
__device__ __forceinline__ int wave_last(int n, int64_t x, Key key) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = n;
    while (true) {
        const int step = (hi - lo + 63) >> 6, s = lo + lane * step;
        const int count = __builtin_popcountll(__ballot(s < hi && key(s) <= x));
        if (count == 0) return -1;
        lo = __builtin_amdgcn_readfirstlane(lo + (count - 1) * step);
        if (step == 1) return lo;
        hi = min(hi, lo + step);
    }
}

// Sum over the lanes up to this one: within rows of 16 lanes, then from row to
// row (data-parallel moves between lanes, no LDS).
__device__ __forceinline__ uint32_t wave_sum_to(uint32_t v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
    return v;
}

}  // namespace dhx
