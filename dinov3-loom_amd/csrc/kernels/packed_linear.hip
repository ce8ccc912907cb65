// A projection with low-rank adapters on packed batches
// (include/dinov3_packed.h): y = x W^T + bias + scale_a (x A_a^T) B_a^T, a the
// adapter of the row's sequence.
//
// Two kernels. The first finds each row's adapter and computes u = scale_a x
// A_a^T (rank columns), rounded to the operands' type. The second is the
// product over all columns of x, continued over those of u: a tile's rows
// belong to runs of rows with one adapter, and run j adds rank columns
// [u of the run's rows, 0 elsewhere] . B_a^T. So adapters cost the product
// rank columns per run in a tile, and no pass over y.
#include "packed.hpp"

namespace dhx {
namespace {

constexpr int kThreads = 256;
constexpr int kNoAdapter = -1;   // a row of a sequence without adapter
constexpr int kNoSequence = -2;  // a row of no sequence: its y stays as it was

struct Workspace {
    uint64_t ids, u, bytes;  // int32 [rows]; [rows][rank]
};
Workspace layout(const dhx_packed_linear& p) {
    Workspace w{};
    w.u = (p.rows * 4 + 255) / 256 * 256;
    w.bytes = w.u + p.rows * p.rank * 2;
    return w;
}

// --- u = scale x A^T ---------------------------------------------------------

#define DHX_SHRINK_PARAMS Addr starts_, Addr adapter_, Addr x_, Addr a_, Addr scale_, int sequences, int rows, int adapters, int inputs, int rank, Addr ids_, Addr u_, uint64_t x_stride

// The adapter of `row` (per lane), as above. The sequences of the tile's first
// and last rows are found by the whole wave, a lane's own between them.
__device__ __forceinline__ int adapter_of(int row, int first, int last, const int32_t* starts, const int32_t* adapter,
                                          int sequences, int rows, int adapters) {
    auto at = [&](int s) { return (int64_t)start_at(starts, s, rows); };
    int lo = max(wave_last(sequences, first, at), 0), hi = max(wave_last(sequences, last, at), lo);
    while (lo < hi) {  // the last s whose first row is not behind `row`
        const int mid = lo + (hi - lo + 1) / 2;
        if (start_at(starts, mid, rows) <= row) lo = mid;
        else hi = mid - 1;
    }
    if (row < start_at(starts, lo, rows) || row >= start_at(starts, lo + 1, rows)) return kNoSequence;
    const int id = adapter[lo];
    return (uint32_t)id < (uint32_t)adapters ? id : kNoAdapter;
}

// A workgroup takes 32 rows and, of the runs of rows with one adapter among
// them, every gridDim.y-th; its four waves share the columns of x out and join
// their sums in LDS. Both operands come straight from memory: A is read once
// per run, x once per run and tile, out of the caches after the first.
template <class T>
__global__ __launch_bounds__(kThreads) void packed_shrink_kernel(DHX_SHRINK_PARAMS) {
    typedef typename Num<T>::v8 v8;
    typedef typename Num<T>::v4 v4;
    __shared__ float sum[4][32][33];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, hi = lane >> 5;
    const int row0 = blockIdx.x * 32, row = min(row0 + l32, rows - 1);
    int id = adapter_of(row, row0, min(row0 + 31, rows - 1), starts_, adapter_, sequences, rows, adapters);
    if (row0 + l32 >= rows) id = kNoSequence;
    if (blockIdx.y == 0 && wave == 0 && hi == 0 && row0 + l32 < rows) ((int32_t*)ids_)[row] = id;
    const int before = __shfl(id, (lane & 32) | ((l32 - 1) & 31));
    const uint32_t starts = (uint32_t)__ballot(hi == 0 && id >= 0 && (l32 == 0 || id != before));
    const int run = __popc(starts & (0xffffffffu >> (31 - l32))) - 1;  // of this lane's row, if id >= 0
    const int runs = __popc(starts);
    const T* px = (const T*)x_ + (uint64_t)row * x_stride;
    const int steps = (inputs + 15) / 16;
    for (int j = blockIdx.y; j < runs; j += gridDim.y) {
        const uint64_t mine = __ballot(hi == 0 && id >= 0 && run == j);
        const int a = __shfl(id, __ffsll((long long)mine) - 1);
        const float scale = ((const float*)scale_)[a];
        for (int r0 = 0; r0 < rank; r0 += 32) {
            const int ra = min(r0 + l32, rank - 1);
            const T* pa = (const T*)a_ + ((uint64_t)a * rank + ra) * inputs;
            float16_t acc = {};
            for (int s = wave; s < steps; s += 4) {
                const int ch = s * 16 + hi * 8;
                const bool in = ch < inputs;
                const v8 fa = in ? *(const v8*)(pa + ch) : v8{}, fx = in ? *(const v8*)(px + ch) : v8{};
                acc = Num<T>::mfma(fa, fx, acc);
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < 16; ++r) sum[wave][l32][8 * (r >> 2) + 4 * hi + (r & 3)] = acc[r];
            __syncthreads();
            // Thread -> row tid / 8 of the tile, 4 columns.
            const int tr = tid >> 3, c = (tid & 7) * 4;
            const bool write = (mine >> tr & 1) && r0 + c < rank;
            if (write) {
                v4 out;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    out[e] = (T)(scale * ((sum[0][tr][c + e] + sum[1][tr][c + e]) + (sum[2][tr][c + e] + sum[3][tr][c + e])));
                *(v4*)((T*)u_ + (uint64_t)(row0 + tr) * rank + r0 + c) = out;
            }
        }
    }
}

// --- y = [x, u] [W, B]^T + bias ----------------------------------------------

#define DHX_LINEAR_PARAMS Addr x_, Addr w_, Addr ids_, Addr u_, Addr b_, int rows, int inputs, int outputs, int rank, Addr bias_, Addr y_, uint64_t x_stride, uint64_t w_stride, uint64_t y_stride

// Elements of a 64-column stage row: 128 bytes, swizzled as in packed.hpp.
constexpr int kBK = 64;

// Tile BM x BN, waves of WM x WN each.
template <class T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(kThreads, 2) void packed_linear_kernel(DHX_LINEAR_PARAMS) {
    typedef typename Num<T>::v8 v8;
    typedef typename Num<T>::v4 v4;
    static_assert((BM / WM) * (BN / WN) * 64 == kThreads, "four waves");
    constexpr int XL = BM / 32, WL = BN / 32;  // DMA loads of a wave per stage, 8 rows each
    constexpr int MB = WM / 32, NB = WN / 32;
    __shared__ __attribute__((aligned(16))) T sX0[BM * kBK], sX1[BM * kBK];
    __shared__ __attribute__((aligned(16))) T sW0[BN * kBK], sW1[BN * kBK];
    __shared__ int sRun[BM], sList[BM], sCount[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, hi = lane >> 5;
    const int n_tiles = (outputs + BN - 1) / BN, total = n_tiles * ((rows + BM - 1) / BM);
    const int per = (total + 7) >> 3, g = blockIdx.x, t = (g & 7) * per + (g >> 3);
    if ((g >> 3) >= per || t >= total) return;
    const int row0 = (t / n_tiles) * BM, col0 = (t % n_tiles) * BN;

    // Runs of rows with one adapter: each row's run, each run's adapter.
    const int32_t* ids = ids_;
    const int mine = tid < BM && row0 + tid < rows ? ids[row0 + tid] : kNoSequence;
    const int before = tid > 0 && tid < BM && row0 + tid < rows ? ids[row0 + tid - 1] : kNoSequence;
    const uint64_t flags = __ballot(mine >= 0 && mine != before);
    if (lane == 0) sCount[wave] = __popcll(flags);
    __syncthreads();
    int run = __popcll(flags & (~0ull >> (63 - lane))) - 1, runs = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < wave) run += sCount[w];
        runs += sCount[w];
    }
    if (tid < BM) {
        sRun[tid] = mine >= 0 ? run : -1;
        if (mine >= 0 && mine != before) sList[run] = mine;
    }
    __syncthreads();

    const int k_steps = (inputs + kBK - 1) / kBK;
    const int virtual_chunks = runs * (rank >> 3), steps = k_steps + (virtual_chunks + 7) / 8, rank8 = rank >> 3;
    const T *x = x_, *w = w_, *u = u_, *b = b_;
    const T *x0 = x + (uint64_t)row0 * x_stride, *w0 = w + (uint64_t)col0 * w_stride;
    // Lane -> row lane / 8 of each load's 8, the chunk that the swizzle puts at
    // slot lane % 8.
    const int lr = lane >> 3;
    auto move = [&](T* sx, T* sw, int s) {
        const bool real = s < k_steps;
        const int chunk0 = real ? s * 8 : (s - k_steps) * 8;
#pragma unroll
        for (int j = 0; j < XL; ++j) {
            const int r = wave * (BM / 4) + j * 8 + lr, c = chunk0 + ((lane & 7) ^ slot_of<64>(r));
            const int rr = min(r, rows - 1 - row0);
            const T* p = (const T*)&kZeros;
            if (real) {
                if (c * 8 < inputs) p = x0 + ((uint32_t)rr * (uint32_t)x_stride + c * 8);
            } else if (c < virtual_chunks && sRun[r] == c / rank8) {
                p = u + ((uint64_t)(row0 + rr) * rank + (c % rank8) * 8);
            }
            dma16(p, sx + (wave * (BM / 4) + j * 8) * kBK);
        }
#pragma unroll
        for (int j = 0; j < WL; ++j) {
            const int r = wave * (BN / 4) + j * 8 + lr, c = chunk0 + ((lane & 7) ^ slot_of<64>(r));
            const int rr = min(r, outputs - 1 - col0);
            const T* p = (const T*)&kZeros;
            if (real) {
                if (c * 8 < inputs) p = w0 + ((uint32_t)rr * (uint32_t)w_stride + c * 8);
            } else if (c < virtual_chunks) {
                p = b + (((uint64_t)sList[c / rank8] * outputs + col0 + rr) * rank + (c % rank8) * 8);
            }
            dma16(p, sw + (wave * (BN / 4) + j * 8) * kBK);
        }
    };

    const int wm = wave / (BN / WN) * WM, wn = wave % (BN / WN) * WN;
    const int frag = lds_at<64>(l32, hi * 8);
    float16_t acc[MB][NB] = {};
    auto step = [&](const T* sx, const T* sw, T* next_x, T* next_w, int s) {
        wait_vm<0>();
        wait_lgkm();
        barrier();
        if (s + 1 < steps) move(next_x, next_w, s + 1);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            v8 fx[MB], fw[NB];
#pragma unroll
            for (int i = 0; i < MB; ++i) fx[i] = *(const v8*)(sx + (wm + i * 32) * kBK + (frag ^ (kk << 4)));
#pragma unroll
            for (int i = 0; i < NB; ++i) fw[i] = *(const v8*)(sw + (wn + i * 32) * kBK + (frag ^ (kk << 4)));
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int k = 0; k < NB; ++k) acc[i][k] = Num<T>::mfma(fw[k], fx[i], acc[i][k]);
        }
    };
    move(sX0, sW0, 0);
    for (int s = 0; s < steps; s += 2) {
        step(sX0, sW0, sX1, sW1, s);
        if (s + 1 < steps) step(sX1, sW1, sX0, sW0, s + 1);
    }

    const float* bias = bias_;
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        const int row = row0 + wm + i * 32 + l32;
        if (row >= rows || ids[row] == kNoSequence) continue;
        T* py = (T*)y_ + (uint64_t)row * y_stride;
#pragma unroll
        for (int k = 0; k < NB; ++k)
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                const int n = col0 + wn + k * 32 + kk * 16;
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = acc[i][k][8 * kk + e];
                // v[4g + e]: column n + 8g + 4hi + e.
#pragma unroll
                for (int gq = 0; gq < 2; ++gq) {
                    const int c = n + 8 * gq + 4 * hi;
                    if (c >= outputs) continue;
                    v4 o;
                    const float4_t add = bias ? *(const float4_t*)(bias + c) : float4_t{};
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = (T)(v[4 * gq + e] + add[e]);
                    *(v4*)(py + c) = o;
                }
            }
    }
}

template <class T>
hipError_t launch(const dhx_packed_linear& p, hipStream_t s) {
    const Workspace w = layout(p);
    const Addr ids(p.workspace), u(static_cast<const char*>(p.workspace) + w.u);
    const unsigned tiles = (unsigned)((p.rows + 31) / 32);
    // Runs side by side while there are few tiles: enough workgroups for the chip.
    const unsigned side = tiles >= 512 ? 1 : tiles >= 128 ? 4 : 32;
    hipError_t err = enqueue(packed_shrink_kernel<T>, dim3(tiles, side), dim3(kThreads), 0, s, p.starts, p.adapter, p.x, p.a,
                             p.scale, (int)p.sequences, (int)p.rows, (int)p.adapters, (int)p.inputs, (int)p.rank, ids, u, p.x_stride);
    if (err != hipSuccess) return err;
    constexpr int BM = 128, BN = 128;
    const uint64_t total = ((p.rows + BM - 1) / BM) * ((p.outputs + BN - 1) / BN);
    return enqueue(packed_linear_kernel<T, BM, BN, 64, 64>, dim3((unsigned)((total + 7) / 8 * 8)), dim3(kThreads), 0, s, p.x, p.w, ids, u,
                   p.b, (int)p.rows, (int)p.inputs, (int)p.outputs, (int)p.rank, p.bias, p.y, p.x_stride, p.w_stride, p.y_stride);
}

}  // namespace

uint64_t packed_linear_bytes(const dhx_packed_linear& p) { return layout(p).bytes; }

hipError_t launch_packed_linear(const dhx_packed_linear& p, hipStream_t s) {
    return p.type == DHX_F16 ? launch<half_t>(p, s) : launch<bf16_t>(p, s);
}

}  // namespace dhx
