// A projection with low-rank adapters on packed batches
// (include/dinov3_packed.h): y = x W^T + bias + scale_a (x A_a^T) B_a^T, a the
// adapter of the row's sequence.
//
// Two kernels. The first finds each row's adapter and computes u = scale_a x
// A_a^T (rank columns), rounded to the operands' type. The second is the
// product over all columns of x, continued over those of u: a tile's rows
// belong to runs of rows with one adapter, and run j adds rank columns
// [u of the run's rows, 0 elsewhere] . B_a^T. So adapters cost the product
// rank columns per run in a tile, and no pass over y. A value of B that is not
// finite would make 0 . B of the other rows not a number: the product takes zeros
// for such values, and their part of the run's own rows is added behind it
// (not_finite_part).
#include <algorithm>
#include <type_traits>
#include "packed.hpp"

namespace dhx {
namespace {

constexpr int kNoAdapter = -1;   // a row of a sequence without adapter
constexpr int kNoSequence = -2;  // a row of no sequence: its y stays as it was

// The few-rows kernel takes the product up to 64 rows, and up to 512 where a tile
// would walk many columns alone and the few-rows kernel's workgroups (16 columns
// of y and 64 rows) find a CU each. us, against tiles: 4096 columns to 1024, 256
// rows, 21.7 and 30.5 (256 workgroups; rank 64 25.6 and 39.6), 384 rows 35.9 and
// 30.7 (384); 2048 to 2048, 128 rows, 16.0 and 19.5 (256); 1536 to 384, 512 rows,
// 15.4 and 16.7 (192); but 384 to 1152, 128 rows, 10.1 and 9.8 (144).
constexpr uint64_t kFewRows = 64, kMostFewRows = 512, kLongColumns = 1024;
bool few_rows(const dhx_packed_linear& p) {
    return p.rows <= kFewRows || (p.rows <= kMostFewRows && p.inputs >= kLongColumns &&
                                  (p.rows + 63) / 64 * ((p.outputs + 15) / 16) <= 256);
}
constexpr int kMostParts = 4;

struct Workspace {
    uint64_t u, bytes;  // ids, int32 [rows], are at 0
    uint32_t parts;     // sums of u over parts of the columns, float32 [parts][rows][rank]; 1: u itself, [rows][rank]
};
Workspace layout(const dhx_packed_linear& p) {
    Workspace w{};
    w.u = (p.rows * 4 + 255) / 256 * 256;
    // A run's columns in parts where rows are few: a CU reads no more than about
    // 40 GB/s of A, and 24 single tokens' adapters (4096 columns, rank 16) would
    // keep 24 of them busy.
    w.parts = few_rows(p) ? (uint32_t)std::min<uint64_t>(std::max<uint32_t>(p.inputs / 1024, 1), kMostParts) : 1;
    w.bytes = w.u + p.rows * p.rank * (w.parts > 1 ? 4 * w.parts : 2);
    return w;
}

// The products of 16 AB rows of one matrix and 16 XB rows of another along all
// their columns, shared out to the WAVES waves of a workgroup by steps of 64
// columns. A wave moves its own steps into its own LDS, NST - 1 of them ahead,
// so there is no barrier. (Loaded straight into registers, a 16x16x32 operand
// takes 16 bytes of 16 rows per quarter-wave, 16 cache lines each: 32 rows of
// 4096 columns out of L2 then cost 9.2 us, as much as 33 MB of weights out of
// HBM; a DMA load takes whole lines of 8 rows.)
template <class T, int AB, int XB, int WAVES, int NST>
struct Stream {
    typedef typename Num<T>::v8 v8;
    static constexpr int ROWS = 16 * (AB + XB), STAGE = ROWS * 64, LOADS = ROWS / 8;
    const char *a, *x;    // first rows
    uint32_t at[LOADS];   // byte offsets of the lane's row in each load
    int lane, wave;

    // a_at(r), x_at(r): byte offset of row r.
    template <class A, class X>
    __device__ __forceinline__ Stream(const T* a_, const T* x_, int lane_, int wave_, A a_at, X x_at)
        : a((const char*)a_), x((const char*)x_), lane(lane_), wave(wave_) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int r = j * 8 + (lane >> 3);
            at[j] = j < 2 * AB ? a_at(r) : x_at(r - 16 * AB);
        }
    }
    __device__ __forceinline__ void move(T* to, int step, int columns) const {
        const bool whole = step * 64 + 64 <= columns;
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int c = (lane & 7) ^ slot_of<64>(j * 8 + (lane >> 3));
            const char* p = (j < 2 * AB ? a : x) + step * 128;
            if (whole) dma16(p + (at[j] + c * 16), to + j * 512);
            else dma16(step * 64 + c * 8 < columns ? p + (at[j] + c * 16) : (const char*)&kZeros, to + j * 512);
        }
    }
    __device__ __forceinline__ void use(const T* from, float4_t (&acc)[AB][XB]) const {
        const int frag = (lane & 15) * 64 + (((lane >> 4) ^ slot_of<64>(lane & 15)) << 3);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            v8 fa[AB], fx[XB];
#pragma unroll
            for (int i = 0; i < AB; ++i) fa[i] = *(const v8*)(from + i * 1024 + (frag ^ (kk << 5)));
#pragma unroll
            for (int i = 0; i < XB; ++i) fx[i] = *(const v8*)(from + (AB + i) * 1024 + (frag ^ (kk << 5)));
#pragma unroll
            for (int i = 0; i < AB; ++i)
#pragma unroll
                for (int k = 0; k < XB; ++k) acc[i][k] = Num<T>::mfma16(fa[i], fx[k], acc[i][k]);
        }
    }
    // s0 .. s3: this wave's stages (NST of them).
    __device__ __forceinline__ void run(T* s0, T* s1, T* s2, T* s3, int columns, float4_t (&acc)[AB][XB]) const {
        const int steps = (columns + 63) / 64, n = (steps - wave + WAVES - 1) / WAVES;
        auto column = [&](int i) { return wave + i * WAVES; };
        auto step = [&](const T* from, T* free, int i) __attribute__((always_inline)) {
            wait_lgkm();  // the stage before has been read
            if (i + NST - 1 < n) {
                move(free, column(i + NST - 1), columns);
                wait_vm<(NST - 1) * LOADS>();
            } else {
                wait_vm<0>();
            }
            use(from, acc);
        };
        if (n > 0) move(s0, column(0), columns);
        if (n > 1) move(s1, column(1), columns);
        if (NST > 3 && n > 2) move(s2, column(2), columns);
        for (int i = 0; i < n; i += NST) {
            step(s0, NST > 3 ? s3 : s2, i);
            if (i + 1 < n) step(s1, s0, i + 1);
            if (i + 2 < n) step(s2, s1, i + 2);
            if (NST > 3 && i + 3 < n) step(s3, s2, i + 3);
        }
    }
};

// The lane's number, from no register that would have to hold it.
__device__ __forceinline__ int lane_id() { return __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)); }

// --- u = scale x A^T ---------------------------------------------------------

#define DHX_SHRINK_PARAMS Addr starts_, Addr adapter_, Addr x_, Addr a_, Addr scale_, int sequences, int rows, int adapters, int inputs, int rank, Addr ids_, Addr u_, uint64_t x_stride

// The adapter of `row` (per lane, row0 + lane % TILE), or one of the two above. A
// lane holds the first row of one of 64 sequences, those from the one of row0 on,
// and a row's sequence is the last one that does not begin behind it: one load's
// latency for batches of up to 64 sequences. Rows behind the window (only where
// sequences in it are empty) are searched.
template <int TILE>
__device__ __forceinline__ int adapter_of(int row, int row0, const int32_t* starts, const int32_t* adapter, int sequences,
                                          int rows, int adapters) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    if (sequences > 64) base = max(0, wave_last(sequences, row0, [&](int s) { return (int64_t)start_at(starts, s, rows); }));
    const int s = min(base + lane, sequences - 1);
    const int from = start_at(starts, s, rows), to = start_at(starts, s + 1, rows), id = adapter[s];
    int at = 0;
#pragma unroll
    for (int r = 0; r < TILE; ++r) {
        const int n = __builtin_popcountll(__ballot(base + lane < sequences && from <= row0 + r));
        if (lane % TILE == r) at = max(n - 1, 0);
    }
    int lo = __shfl(from, at), hi = __shfl(to, at), mine = __shfl(id, at);
    if (at == 63 && row >= hi && base + 64 < sequences) {
        int a = base + 63, b = sequences - 1;
        while (a < b) {  // the last sequence that does not begin behind the row
            const int mid = a + (b - a + 1) / 2;
            if (start_at(starts, mid, rows) <= row) a = mid;
            else b = mid - 1;
        }
        lo = start_at(starts, a, rows);
        hi = start_at(starts, a + 1, rows);
        mine = adapter[a];
    }
    if (row < lo || row >= hi) return kNoSequence;
    return (uint32_t)mine < (uint32_t)adapters ? mine : kNoAdapter;
}

// A workgroup takes 32 rows and, of the runs of rows with one adapter among
// them, every gridDim.y-th, and of the columns of x one of gridDim.z parts (of
// several, the sums of u are left to the product); its waves share those out and
// join their sums in LDS. RB: blocks of 16 columns of u at a time.
template <class T, int RB, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void packed_shrink_kernel(DHX_SHRINK_PARAMS) {
    typedef typename Num<T>::v4 v4;
    constexpr int COLS = 16 * RB, XB = 2, TILE = 16 * XB;
    typedef Stream<T, RB, XB, WAVES, 4> S;
    __shared__ __attribute__((aligned(16))) T s0[WAVES * S::STAGE], s1[WAVES * S::STAGE], s2[WAVES * S::STAGE], s3[WAVES * S::STAGE];
    __shared__ float sum[WAVES][TILE][COLS + 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int at = lane % TILE, l16 = lane & 15, part = lane >> 4;
    const int row0 = blockIdx.x * TILE;
    // This workgroup's part of the columns, in whole steps.
    const int per = ((inputs + 63) / 64 + gridDim.z - 1) / gridDim.z * 64, column0 = min((int)blockIdx.z * per, inputs);
    const int columns = min(per, inputs - column0);
    int id = adapter_of<TILE>(row0 + at, row0, starts_, adapter_, sequences, rows, adapters);
    if (row0 + at >= rows) id = kNoSequence;
    if (blockIdx.y == 0 && blockIdx.z == 0 && wave == 0 && lane < TILE && row0 + at < rows) ((int32_t*)ids_)[row0 + at] = id;
    const int before = __shfl(id, max(at - 1, 0));
    const uint64_t starts = __ballot(lane < TILE && id >= 0 && (at == 0 || id != before));
    const int run = __popcll(starts & (~0ull >> (63 - at))) - 1;  // of this lane's row, if id >= 0
    const int runs = __popcll(starts);
    for (int j = blockIdx.y; j < runs; j += gridDim.y) {
        const uint64_t mine = __ballot(lane < TILE && id >= 0 && run == j);
        const int some = __ffsll((long long)mine) - 1, a = __builtin_amdgcn_readfirstlane(__shfl(id, some));
        const float scale = ((const float*)scale_)[a];
        for (int r0 = 0; r0 < rank; r0 += COLS) {
            // Rows outside the run fetch its first one: no more than is needed.
            const S stream(
                (const T*)a_ + ((uint64_t)a * rank + r0) * inputs + column0, (const T*)x_ + (uint64_t)row0 * x_stride + column0, lane, wave,
                [&](int r) { return (uint32_t)min(r, rank - 1 - r0) * (uint32_t)inputs * 2; },
                [&](int r) { return (uint32_t)(mine >> r & 1 ? r : some) * (uint32_t)x_stride * 2; });
            float4_t acc[RB][XB] = {};
            stream.run(s0 + wave * S::STAGE, s1 + wave * S::STAGE, s2 + wave * S::STAGE, s3 + wave * S::STAGE, columns, acc);
            // Lane: row 16 x + l16, columns 16 i + 4 part .. +3.
            __syncthreads();
#pragma unroll
            for (int i = 0; i < RB; ++i)
#pragma unroll
                for (int x = 0; x < XB; ++x) *(float4_t*)&sum[wave][16 * x + l16][16 * i + 4 * part] = acc[i][x];
            __syncthreads();
            for (int i = tid; i < TILE * (COLS / 4); i += 64 * WAVES) {  // a row of the tile, 4 columns
                const int tr = i / (COLS / 4), c = i % (COLS / 4) * 4;
                if (!(mine >> tr & 1) || r0 + c >= rank) continue;
                float4_t v = {};
#pragma unroll
                for (int w = 0; w < WAVES; ++w) v += *(const float4_t*)&sum[w][tr][c];
                const uint64_t to = (uint64_t)(row0 + tr) * rank + r0 + c;
                if (gridDim.z > 1) {
                    *(float4_t*)((float*)u_ + (uint64_t)blockIdx.z * rows * rank + to) = scale * v;
                    continue;
                }
                v4 out;
#pragma unroll
                for (int e = 0; e < 4; ++e) out[e] = (T)(scale * v[e]);
                *(v4*)((T*)u_ + to) = out;
            }
        }
    }
}

// --- y = [x, u] [W, B]^T + bias ----------------------------------------------

#define DHX_LINEAR_PARAMS Addr x_, Addr w_, Addr ids_, Addr u_, Addr b_, int rows, int inputs, int outputs, int rank, Addr bias_, Addr y_, uint64_t x_stride, uint64_t w_stride, uint64_t y_stride

// The runs of rows with one adapter among `n` rows from row0 on (n at most the
// workgroup's threads): each row's run in run[] (-1: no adapter, -2: no
// sequence), each run's adapter in list[]; returns their number, and in `bare`
// whether a row has no adapter. count: one int per wave.
template <int THREADS>
__device__ __forceinline__ int find_runs(const int32_t* ids, int row0, int n, int rows, int* run, int* list, int* count, bool& bare) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const bool in = tid < n && row0 + tid < rows;
    const int mine = in ? ids[row0 + tid] : kNoSequence;
    const int before = in && tid > 0 ? ids[row0 + tid - 1] : kNoSequence;
    const bool first = mine >= 0 && mine != before;
    const uint64_t flags = __ballot(first);
    const int none = __any(mine == kNoAdapter) << 16;  // above the number of runs
    if (lane == 0) count[wave] = __popcll(flags) + none;
    __syncthreads();
    int at = __popcll(flags & (~0ull >> (63 - lane))) - 1, all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        if (w < wave) at += count[w] & 0xffff;
        all += count[w];
    }
    all = __builtin_amdgcn_readfirstlane(all);
    bare = all >> 16 != 0;
    if (tid < n) {
        run[tid] = mine >= 0 ? at : mine;
        if (first) list[at] = mine;
    }
    __syncthreads();
    return all & 0xffff;
}

// The values of a row of B (`rank8` pieces of 8) that are not finite, times those
// of u (piece i: u_at(i)): what a product leaves out that takes zeros for them.
template <class T, class U>
__device__ __forceinline__ float not_finite_part(const T* b, int rank8, U u_at) {
    typedef typename Num<T>::v8 v8;
    float sum = 0.f;
#pragma unroll 1
    for (int i = 0; i < rank8; ++i) {
        const v8 vb = *(const v8*)(b + 8 * i);
        if (!any_not_finite<T>(vb)) continue;
        const v8 vu = u_at(i);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float f = (float)vb[e];
            if (!__builtin_isfinite(f)) sum = fmaf((float)vu[e], f, sum);
        }
    }
    return sum;
}
template <class T>
__device__ __forceinline__ typename Num<T>::v8 zeros_for_not_finite(typename Num<T>::v8 v) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (!__builtin_isfinite((float)v[e])) v[e] = (T)0.f;
    return v;
}

// Chunk c of LDS row r of a stage, 64 columns (128-byte rows, as in packed.hpp)
// or 128 (256-byte rows) or 32 (64-byte rows, four per pass over the banks).
template <int BK>
__device__ __forceinline__ int stage_slot(int r) {
    if constexpr (BK == 32) return (r >> 2) & 3;
    else return slot_of<BK>(r);
}

// Tile BM x BN in steps of BK columns, waves of WM x WN each. NST stages in
// LDS, NST - 1 of them on their way while one is multiplied (a variable each, so
// that the compiler can tell the stage that is read from those being filled);
// the last fragments of a stage are multiplied behind the barrier that opens
// the next one, whose first fragments are on their way by then.
template <class T, int BM, int BN, int WM, int WN, int BK, int NST, bool PRE, int PER_SIMD>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN), PER_SIMD) void packed_linear_kernel(DHX_LINEAR_PARAMS) {
    typedef typename Num<T>::v8 v8;
    typedef typename Num<T>::v4 v4;
    constexpr int WAVES = (BM / WM) * (BN / WN), THREADS = 64 * WAVES;
    constexpr int CH = BK / 8, LR = 64 / CH;  // chunks of a stage row, rows of a DMA load
    constexpr int XL = BM / LR / WAVES, WL = BN / LR / WAVES;
    constexpr int MB = WM / 32, NB = WN / 32, KK = BK / 16;
    static_assert(!PRE || NST % 2 == 0, "the fragments' sets take turns with the stages");
    static_assert(NB <= 2, "a lane's columns of 32 rows are the bits of a word");
    static_assert(XL * LR * WAVES == BM && WL * LR * WAVES == BN && BM <= THREADS && BN <= THREADS, "whole loads");
    constexpr int XS = BM * BK, WS = BN * BK;
    __shared__ __attribute__((aligned(16))) T sX0[XS], sX1[XS], sX2[NST > 2 ? XS : 8], sX3[NST > 3 ? XS : 8];
    __shared__ __attribute__((aligned(16))) T sW0[WS], sW1[WS], sW2[NST > 2 ? WS : 8], sW3[NST > 3 ? WS : 8];
    __shared__ int sRun[BM], sList[BM], sCount[WAVES];
    __shared__ __attribute__((aligned(16))) float sBias[BN];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Tiles in XCD-contiguous order, four row blocks at a time, so that the tiles
    // that an XCD has under way share rows of x and rows of W in its L2.
    const int n_tiles = (outputs + BN - 1) / BN, total = n_tiles * ((rows + BM - 1) / BM);
    const int per = (total + 7) >> 3, g = blockIdx.x, t = (g & 7) * per + (g >> 3);
    if ((g >> 3) >= per || t >= total) return;
    constexpr int GROUP = 4;
    const int block = t / (GROUP * n_tiles), in_block = t - block * GROUP * n_tiles;
    const int tall = min(GROUP, total / n_tiles - block * GROUP), across = in_block / tall;
    const int row0 = (block * GROUP + in_block - across * tall) * BM, col0 = across * BN;
    const int k_steps = (inputs + BK - 1) / BK, whole = inputs / BK;
    const T *x0 = (const T*)x_ + (uint64_t)row0 * x_stride, *w0 = (const T*)w_ + (uint64_t)col0 * w_stride;

    // Lane -> row lane / CH of a load's LR, the chunk that the swizzle puts at
    // slot lane % CH; rows behind the last one fetch that one.
    uint32_t xo[XL], wo[WL];
    int frag;  // the element of a stage that the lane's first fragment begins at
    auto place = [&](int lane) __attribute__((always_inline)) {
        const int lr = lane / CH, l32 = lane & 31, hi = lane >> 5;
        frag = l32 * BK + ((hi ^ stage_slot<BK>(l32)) << 3);
        auto chunk = [&](int r) { return (lane % CH) ^ stage_slot<BK>(r); };
#pragma unroll
        for (int j = 0; j < XL; ++j) {
            const int r = (wave * XL + j) * LR + lr;
            xo[j] = (uint32_t)min(r, rows - 1 - row0) * (uint32_t)x_stride + chunk(r) * 8;
        }
#pragma unroll
        for (int j = 0; j < WL; ++j) {
            const int r = (wave * WL + j) * LR + lr;
            wo[j] = (uint32_t)min(r, outputs - 1 - col0) * (uint32_t)w_stride + chunk(r) * 8;
        }
    };
    place(lane);
    auto move_whole = [&](T* sx, T* sw, int s) __attribute__((always_inline)) {
        const T *px = x0 + s * BK, *pw = w0 + s * BK;
#pragma unroll
        for (int j = 0; j < XL; ++j) dma16(px + xo[j], sx + (wave * XL + j) * 512);
#pragma unroll
        for (int j = 0; j < WL; ++j) dma16(pw + wo[j], sw + (wave * WL + j) * 512);
    };
    // Any stage: whole ones, the last columns of x and W, and those of u and B,
    // where chunk c belongs to run c / (rank / 8): turn = ceil(2^18 / (rank / 8))
    // divides every c below 2^13 by it exactly.
    int runs = 0;
    const int rank8 = rank >> 3;
    const uint32_t turn = ((1u << 18) + rank8 - 1) / rank8;
    auto move = [&](T* sx, T* sw, int s) __attribute__((always_inline)) {
        if (s < whole) {
            move_whole(sx, sw, s);
            return;
        }
        const T* zeros = (const T*)&kZeros;
        // What follows is taken anew in each of these few stages: held through the
        // whole ones it would cost them registers.
        int lane = lane_id();
        asm volatile("" : "+v"(lane));
        const int lr = lane / CH;
        auto chunk = [&](int r) { return (lane % CH) ^ stage_slot<BK>(r); };
        if (s < k_steps) {
#pragma unroll
            for (int j = 0; j < XL; ++j) {
                const bool in = s * BK + chunk((wave * XL + j) * LR + lr) * 8 < inputs;
                dma16(in ? x0 + s * BK + xo[j] : zeros, sx + (wave * XL + j) * 512);
            }
#pragma unroll
            for (int j = 0; j < WL; ++j) {
                const bool in = s * BK + chunk((wave * WL + j) * LR + lr) * 8 < inputs;
                dma16(in ? w0 + s * BK + wo[j] : zeros, sw + (wave * WL + j) * 512);
            }
            return;
        }
        const T *u0 = (const T*)u_ + (uint64_t)row0 * rank, *b = (const T*)b_;
        const uint64_t adapter = (uint64_t)outputs * rank;
        const int c0 = (s - k_steps) * CH;
#pragma unroll
        for (int j = 0; j < XL; ++j) {
            const int r = (wave * XL + j) * LR + lr;
            const uint32_t c = c0 + chunk(r), i = (c * turn) >> 18;
            const bool in = i < (uint32_t)runs && sRun[r] == (int)i;  // no row behind the last has a run
            dma16(in ? u0 + (uint32_t)(r * rank + (c - i * rank8) * 8) : zeros, sx + (wave * XL + j) * 512);
        }
#pragma unroll
        for (int j = 0; j < WL; ++j) {
            const int r = (wave * WL + j) * LR + lr;
            const uint32_t c = c0 + chunk(r), i = (c * turn) >> 18;
            const T* pb = b + (uint64_t)(uint32_t)(col0 + min(r, outputs - 1 - col0)) * rank + (c - i * rank8) * 8;
            dma16(i < (uint32_t)runs ? pb + sList[i] * adapter : zeros, sw + (wave * WL + j) * 512);
        }
    };

    const int wm = wave / (BN / WN) * WM, wn = wave % (BN / WN) * WN;
    float16_t acc[MB][NB] = {};
    constexpr int SETS = PRE ? 2 * KK : 2;
    v8 fx[SETS][MB], fw[SETS][NB];
    auto load = [&](const T* sx, const T* sw, int kk, int set) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MB; ++i) fx[set][i] = *(const v8*)(sx + (wm + i * 32) * BK + (frag ^ (kk << 4)));
#pragma unroll
        for (int i = 0; i < NB; ++i) fw[set][i] = *(const v8*)(sw + (wn + i * 32) * BK + (frag ^ (kk << 4)));
    };
    auto multiply = [&](int set) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int k = 0; k < NB; ++k) acc[i][k] = Num<T>::mfma(fw[set][k], fx[set][i], acc[i][k]);
    };
    move(sX0, sW0, 0);
    if (tid < BN) sBias[tid] = bias_.a && col0 + tid < outputs ? ((const float*)bias_)[col0 + tid] : 0.f;
    bool bare;
    runs = find_runs<THREADS>(ids_, row0, BM, rows, sRun, sList, sCount, bare);
    const int steps = k_steps + (runs * rank8 + CH - 1) / CH;
    if (NST > 2 && steps > 1) move(sX1, sW1, 1);
    if (NST > 3 && steps > 2) move(sX2, sW2, 2);
    // Opens stage s: it has landed (the NST - 2 stages behind it may be on their
    // way), and every wave has read the one before, whose place stage s + NST - 1
    // takes.
    // FAST: s + 2 (NST - 1) <= whole, so that there is a next stage, NST - 1 of
    // them on their way, and the one to fetch is whole.
    auto open = [&](auto fast, T* free_x, T* free_w, int s) __attribute__((always_inline)) {
        if (fast || s + NST - 2 < steps) wait_vm<(NST - 2) * (XL + WL)>();
        else wait_vm<0>();
        wait_lgkm();
        barrier();
        if constexpr (fast) move_whole(free_x, free_w, s + NST - 1);
        else if (s + NST - 1 < steps) move(free_x, free_w, s + NST - 1);
    };
    auto step = [&](auto fast, T* sx, T* sw, const T* next_x, const T* next_w, int s, int odd) __attribute__((always_inline)) {
        if constexpr (PRE) {
            if (fast || s + 1 < steps) {
                open(fast, sx, sw, s + 1);
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) load(next_x, next_w, kk, (1 - odd) * KK + kk);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) multiply(odd * KK + kk);
        } else {
#pragma unroll
            for (int kk = 0; kk < KK - 1; ++kk) {
                load(sx, sw, kk + 1, (kk + 1) & 1);
                __builtin_amdgcn_sched_barrier(0);  // the reads go ahead of the products they pass under
                multiply(kk & 1);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (fast || s + 1 < steps) {
                open(fast, sx, sw, s + 1);
                load(next_x, next_w, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
            multiply((KK - 1) & 1);
        }
    };
    open(std::false_type{}, NST == 2 ? sX1 : NST == 3 ? sX2 : sX3, NST == 2 ? sW1 : NST == 3 ? sW2 : sW3, 0);
#pragma unroll
    for (int kk = 0; kk < (PRE ? KK : 1); ++kk) load(sX0, sW0, kk, kk);
    int s = 0;
    auto turn_of_stages = [&](auto fast) __attribute__((always_inline)) {
        step(fast, sX0, sW0, sX1, sW1, s, 0);
        if (fast || s + 1 < steps) step(fast, sX1, sW1, NST > 2 ? sX2 : sX0, NST > 2 ? sW2 : sW0, s + 1, 1);
        if constexpr (NST > 2)
            if (fast || s + 2 < steps) step(fast, sX2, sW2, NST > 3 ? sX3 : sX0, NST > 3 ? sW3 : sW0, s + 2, 0);
        if constexpr (NST > 3)
            if (fast || s + 3 < steps) step(fast, sX3, sW3, sX0, sW0, s + 3, 1);
        s += NST;
    };
    while (s + 2 * NST <= whole) turn_of_stages(std::true_type{});
    while (s < steps) turn_of_stages(std::false_type{});

    // Rows that a run's B does not belong to are multiplied by it, as zeros. A
    // value of B that is not finite leaves none of its column's sums finite, those
    // of its own rows (u times it) nor the others (0 times it), so some of the rows
    // tell, and all of them where they are not finite (rows of x may not be). Such
    // a tile is computed once more, with zeros for those values. (us, without this
    // check and with it: 12864 rows, 384 x 1152, 28.3 and 28.4; 7823 rows, 1536 x
    // 384, 25.6 and 25.75; 16384 rows, 4096 x 4096, 502 and 502; with a NaN in one of
    // eight adapters the first takes 87, with all of every eighth request's x NaN as
    // long as without. Checked in front of the stores it cost 0.5, and the pipelined
    // walk run twice registers.)
    const bool mixed = runs > 1 || (runs == 1 && bare);
    if (mixed) {
        float odd = 0.f;  // no number, if a sum is not finite
#pragma unroll
        for (int k = 0; k < NB; ++k)
#pragma unroll
            for (int r = 0; r < 16; ++r) odd = fmaf(acc[0][k][r], 0.f, odd);
        bool mine = __any(odd != 0.f);
        if (__builtin_expect(mine, 0)) {  // a column without a finite sum?
            uint32_t none = ~0u;
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                uint32_t here = 0;
#pragma unroll
                for (int k = 0; k < NB; ++k)
#pragma unroll
                    for (int r = 0; r < 16; ++r) here |= (uint32_t)!__builtin_isfinite(acc[i][k][r]) << (16 * k + r);
                none &= here;
            }
#pragma unroll
            for (int i = 16; i; i >>= 1) none &= __shfl_xor(none, i);
            mine = __any(none != 0);
        }
        if (lane_id() == 0) sCount[wave] = mine;
    }
    for (bool again = false;; again = true) {
        // As in move: taken anew, not held through the walk.
        int last = lane_id();
        asm volatile("" : "+v"(last));
        const int r32 = last & 31, half = last >> 5;
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            const int row = row0 + wm + i * 32 + r32;
            const bool there = sRun[wm + i * 32 + r32] != kNoSequence;
            T* py = (T*)y_ + (uint64_t)row * y_stride;
#pragma unroll
            for (int k = 0; k < NB; ++k)
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    const int n = col0 + wn + k * 32 + kk * 16;
                    v4 o[2];
#pragma unroll
                    for (int q = 0; q < 2; ++q) {  // columns n + 8q + 4hi .. +3
                        const float4_t add = *(const float4_t*)(sBias + wn + k * 32 + kk * 16 + 8 * q + 4 * half);
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[q][e] = (T)(acc[i][k][8 * kk + 4 * q + e] + add[e]);
                    }
                    const v8 piece = __builtin_bit_cast(v8, frag_swap(__builtin_bit_cast(half4_t, o[0]), __builtin_bit_cast(half4_t, o[1])));
                    if (there && n + half * 8 < outputs) *(v8*)(py + n + half * 8) = piece;
                }
        }
        if (!mixed || again) return;
        wait_lgkm();
        barrier();  // behind the stores: they are on their way
        int any = 0;
#pragma unroll
        for (int n = 0; n < BN / WN; ++n) {  // in all rows of its columns
            int all = 1;
#pragma unroll
            for (int m = 0; m < BM / WM; ++m) all &= sCount[m * (BN / WN) + n];
            any |= all;
        }
        if (__builtin_expect(!__builtin_amdgcn_readfirstlane(any), 1)) return;
        // The same products in the same order, a stage at a time.
        place(last);
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int k = 0; k < NB; ++k) acc[i][k] = float16_t{};
#pragma unroll 1
        for (int s = 0; s < steps; ++s) {
            move(sX0, sW0, s);
            wait_vm<0>();
            barrier();
            if (s >= k_steps) {
#pragma unroll 1
                for (int i = (wave * 64 + last) * 8; i < WS; i += THREADS * 8) *(v8*)(sW0 + i) = zeros_for_not_finite<T>(*(const v8*)(sW0 + i));
                wait_lgkm();
                barrier();
            }
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                load(sX0, sW0, kk, kk & 1);
                multiply(kk & 1);
            }
            wait_lgkm();
            barrier();  // read by every wave
        }
        // What the zeros left out of the run's own rows.
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            const int row = row0 + wm + i * 32 + r32, run = sRun[wm + i * 32 + r32];
            if (run < 0) continue;
            const T *u = (const T*)u_ + (uint64_t)row * rank, *b = (const T*)b_ + (uint64_t)sList[run] * outputs * rank;
#pragma unroll
            for (int k = 0; k < NB; ++k)
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    const int col = col0 + wn + k * 32 + 8 * g4 + 4 * half;
                    if (col >= outputs) continue;
#pragma unroll 1
                    for (int e = 0; e < 4; ++e) {
                        const float part = not_finite_part<T>(b + (uint64_t)(col + e) * rank, rank8, [&](int at) { return *(const v8*)(u + 8 * at); });
#pragma unroll
                        for (int to = 0; to < 4; ++to) acc[i][k][4 * g4 + to] += to == e ? part : 0.f;
                    }
                }
        }
    }
}

// Few rows: a workgroup takes 16 columns of y and 16 MB rows, so that W, which
// is all there is to read, streams through as many workgroups as it can; the
// four waves share the columns of x and u out and join their sums in LDS.
constexpr int kFewWaves = 4;
template <class T, int MB>
__global__ __launch_bounds__(64 * kFewWaves) void packed_linear_few_kernel(DHX_LINEAR_PARAMS, int parts) {
    typedef typename Num<T>::v8 v8;
    constexpr int NST = MB == 4 ? 3 : 4, ROWS = 16 * MB;
    typedef Stream<T, 1, MB, kFewWaves, NST> S;
    constexpr int LDS = kFewWaves * S::STAGE;
    __shared__ __attribute__((aligned(16))) T s0[LDS], s1[LDS], s2[LDS], s3[NST > 3 ? LDS : 8];
    __shared__ float sum[kFewWaves][ROWS][20];
    __shared__ int sRun[ROWS], sList[ROWS], sCount[kFewWaves], sOdd;  // sOdd: some value of B is not finite
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, part = lane >> 4;
    const int col0 = blockIdx.x * 16, row0 = blockIdx.y * ROWS;
    const int col = min(col0 + l16, outputs - 1);
    const S stream(
        (const T*)w_ + (uint64_t)col0 * w_stride, (const T*)x_ + (uint64_t)row0 * x_stride, lane, wave,
        [&](int r) { return (uint32_t)min(r, outputs - 1 - col0) * (uint32_t)w_stride * 2; },
        [&](int r) { return (uint32_t)min(r, rows - 1 - row0) * (uint32_t)x_stride * 2; });
    float4_t acc[1][MB] = {};
    stream.run(s0 + wave * S::STAGE, s1 + wave * S::STAGE, s2 + wave * S::STAGE, s3 + (NST > 3 ? wave * S::STAGE : 0), inputs, acc);
    if (tid == 0) sOdd = 0;
    bool bare;
    const int runs = find_runs<64 * kFewWaves>(ids_, row0, ROWS, rows, sRun, sList, sCount, bare), rank8 = rank >> 3;
    const T *u = (const T*)u_, *b = (const T*)b_;
    auto u_at = [&](uint64_t at) {  // 8 values
        if (parts == 1) return *(const v8*)(u + at);
        float4_t v[kMostParts][2] = {};
#pragma unroll
        for (int z = 0; z < kMostParts; ++z) {
            const float4_t* p = (const float4_t*)((const float*)u_ + (uint64_t)min(z, parts - 1) * rows * rank + at);
            v[z][0] = p[0];
            v[z][1] = p[1];
        }
        float4_t all[2] = {v[0][0], v[0][1]};
#pragma unroll
        for (int z = 1; z < kMostParts; ++z)
            if (z < parts) {
                all[0] += v[z][0];
                all[1] += v[z][1];
            }
        v8 sum;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] = (T)all[e / 4][e % 4];
        return sum;
    };
    for (int s = wave; s * 4 < runs * rank8; s += kFewWaves) {
        const int c = s * 4 + part, i = c / rank8, off = (c - i * rank8) * 8;
        const bool in = i < runs;
        v8 fb = in ? *(const v8*)(b + ((uint64_t)sList[i] * outputs + col) * rank + off) : v8{};
        v8 fu[MB];
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            const int r = m * 16 + l16;
            fu[m] = in && sRun[r] == i ? u_at((uint64_t)(row0 + r) * rank + off) : v8{};
        }
        if (__builtin_expect(__any(any_not_finite<T>(fb)), 0)) {  // behind the loads of u: they are on their way together
            fb = zeros_for_not_finite<T>(fb);
            sOdd = 1;
        }
#pragma unroll
        for (int m = 0; m < MB; ++m) acc[0][m] = Num<T>::mfma16(fb, fu[m], acc[0][m]);
    }
    // Lane: row 16 m + l16, columns 4 part .. +3.
#pragma unroll
    for (int m = 0; m < MB; ++m) *(float4_t*)&sum[wave][m * 16 + l16][4 * part] = acc[0][m];
    __syncthreads();
    const int r = tid >> 2, c = (tid & 3) * 4, row = row0 + r, odd = sOdd;
    if (r >= ROWS || row >= rows || col0 + c >= outputs || sRun[r] == kNoSequence) return;
    float4_t v = {};
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) v += *(const float4_t*)&sum[w][r][c];
    const float* bias = bias_;
    if (bias) v += *(const float4_t*)(bias + col0 + c);
    if (__builtin_expect(odd, 0) && sRun[r] >= 0) {
        const T* row_of_b = b + ((uint64_t)sList[sRun[r]] * outputs + col0 + c) * rank;
#pragma unroll 1
        for (int e = 0; e < 4; ++e) {
            const float part = not_finite_part<T>(row_of_b + e * rank, rank8, [&](int i) { return u_at((uint64_t)row * rank + 8 * i); });
#pragma unroll
            for (int to = 0; to < 4; ++to) v[to] += to == e ? part : 0.f;
        }
    }
    typename Num<T>::v4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (T)v[e];
    *(typename Num<T>::v4*)((T*)y_ + (uint64_t)row * y_stride + col0 + c) = o;
}

template <class T, int BM, int BN, int WM, int WN, int BK, int NST, bool PRE, int PER_SIMD>
hipError_t tiles(const dhx_packed_linear& p, Addr ids, Addr u, hipStream_t s) {
    const uint64_t total = ((p.rows + BM - 1) / BM) * ((p.outputs + BN - 1) / BN);
    return enqueue(packed_linear_kernel<T, BM, BN, WM, WN, BK, NST, PRE, PER_SIMD>, dim3((unsigned)((total + 7) / 8 * 8)),
                   dim3(64 * (BM / WM) * (BN / WN)), 0, s, p.x, p.w, ids, u, p.b, (int)p.rows, (int)p.inputs, (int)p.outputs,
                   (int)p.rank, p.bias, p.y, p.x_stride, p.w_stride, p.y_stride);
}

template <class T, int MB>
hipError_t few(const dhx_packed_linear& p, Addr ids, Addr u, uint32_t parts, hipStream_t s) {
    return enqueue(packed_linear_few_kernel<T, MB>, dim3((p.outputs + 15) / 16, (unsigned)((p.rows + 16 * MB - 1) / (16 * MB))),
                   dim3(64 * kFewWaves), 0, s, p.x, p.w, ids, u, p.b, (int)p.rows, (int)p.inputs, (int)p.outputs, (int)p.rank,
                   p.bias, p.y, p.x_stride, p.w_stride, p.y_stride, (int)parts);
}

template <class T>
hipError_t launch(const dhx_packed_linear& p, hipStream_t s) {
    const Workspace w = layout(p);
    const Addr ids(p.workspace), u(static_cast<const char*>(p.workspace) + w.u);
    // Two waves on a tile of 32 rows where tiles are many and rows short: 12864
    // rows of 384 columns 7.1 us (four waves 9.2); else four: 16384 rows of 4096
    // 48 (62 with two). Taller tiles were slower everywhere. Runs go side by side
    // while there are few tiles.
    const unsigned row_tiles = (unsigned)((p.rows + 31) / 32);
    const unsigned side = row_tiles >= 128 ? 1 : (unsigned)std::min<uint64_t>(32, p.sequences * 32 / p.rows + 2);
    auto shrink = [&](auto kernel, int waves) {
        return enqueue(kernel, dim3(row_tiles, side, w.parts), dim3(64 * waves), 0, s, p.starts, p.adapter, p.x, p.a, p.scale,
                       (int)p.sequences, (int)p.rows, (int)p.adapters, (int)p.inputs, (int)p.rank, ids, u, p.x_stride);
    };
    const bool narrow = row_tiles >= 256 && p.inputs <= 512;
    const hipError_t err = narrow ? p.rank <= 16 ? shrink(packed_shrink_kernel<T, 1, 2>, 2) : shrink(packed_shrink_kernel<T, 2, 2>, 2)
                                  : p.rank <= 16 ? shrink(packed_shrink_kernel<T, 1, 4>, 4) : shrink(packed_shrink_kernel<T, 2, 4>, 4);
    if (err != hipSuccess) return err;
    // Times in us, whole calls on MI355X. For few rows W alone counts: 64 rows,
    // 4096 x 4096, 22 (64 x 64 tiles 31). Then the largest tile of which there are
    // enough for the 256 CUs: 16384 rows, 4096 x 4096, 498 with 256 x 256 (128 x
    // 128 597), 4096 rows 130 (152; 256 tiles); 12864 rows, 384 x 1152, 29 (31; 255
    // tiles), 8192 rows, 1024 x 1024, 38 (30; 128 tiles); 1024 rows, 4096 x 4096,
    // 128 x 128 53.5 (256 tiles), 128 x 64 52.1 (512); 7823 rows, 1536 x 384, 29.1
    // (186), 28.9 (372), 64 x 64 28.1 (738); 256 rows, 4096 x 4096, 64 x 64 in four
    // stages 31 (256 tiles), in two 43.
    if (p.rows <= 16) return few<T, 1>(p, ids, u, w.parts, s);
    if (p.rows <= 32) return few<T, 2>(p, ids, u, w.parts, s);
    if (few_rows(p)) return few<T, 4>(p, ids, u, w.parts, s);
    auto count = [&](uint64_t m, uint64_t n) { return (p.rows + m - 1) / m * ((p.outputs + n - 1) / n); };
    if (count(256, 256) >= 224) return tiles<T, 256, 256, 128, 64, 64, 2, false, 2>(p, ids, u, s);
    if (count(128, 128) >= 300) return tiles<T, 128, 128, 64, 64, 64, 2, false, 2>(p, ids, u, s);
    if (count(128, 64) >= 400) return tiles<T, 128, 64, 64, 32, 64, 2, true, 2>(p, ids, u, s);
    if (count(64, 64) >= 512) return tiles<T, 64, 64, 32, 32, 64, 2, true, 4>(p, ids, u, s);
    return tiles<T, 64, 64, 32, 32, 64, 4, true, 2>(p, ids, u, s);
}

}  // namespace

uint64_t packed_linear_bytes(const dhx_packed_linear& p) { return layout(p).bytes; }

hipError_t launch_packed_linear(const dhx_packed_linear& p, hipStream_t s) {
    return p.type == DHX_F16 ? launch<half_t>(p, s) : launch<bf16_t>(p, s);
}

}  // namespace dhx
