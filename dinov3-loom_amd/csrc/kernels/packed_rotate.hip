// The position rotation of packed rows (include/dinov3_packed.h): out = (x1
// cos - x2 sin, x2 cos + x1 sin) per pair, with the angles of the row's own
// table row. Each value of x is read once and written once and there is no
// arithmetic to speak of, so the kernel is bound by memory: 16-byte pieces, a
// piece of x1 and its partner of x2 per thread, or pieces of 8 bytes where
// rotated is no multiple of 16 (the second half then begins between two 16-byte
// pieces; 12864 rows of 12 heads of 80: 40 rotated 11.4 us, 48 11.0). The table rows are shared by a row's heads and by rows at the same
// place of other sequences, and come from the caches.
#include <algorithm>
#include <type_traits>

#include "packed.hpp"

namespace dhx {
namespace {

// Work items (a pair of pieces of 8 or 4 values, or a copied piece of 8) of a workgroup: whole
// rows, about one item per thread. (Four per thread: 12864 rows of 12 heads of
// 64 9.7 us instead of 8.0, 8192 rows of 40 heads of 128 40 instead of 36; stores
// that bypass the caches 10.0 and 77.)
constexpr int kItems = 256, kMostThreads = 1024;
constexpr uint64_t kMostBlocks = 1u << 21;  // a launch has fewer than 2^32 threads; workgroups take further rows in turn

#define DHX_ROTATE_PARAMS Addr x_, Addr out_, Addr cos_, Addr sin_, Addr index_, uint64_t x_stride, uint64_t out_stride, int rows, int places, int heads, int head_dim, int rotated, int copy, int block_rows

// PAIRS: of an item, 8 or 4; rotated is a multiple of 2 PAIRS.
template <class T, bool NEIGHBOURS, int PAIRS>
__global__ __launch_bounds__(kMostThreads) void packed_rotate_kernel(DHX_ROTATE_PARAMS) {
    typedef typename Num<T>::v8 v8;
    typedef std::conditional_t<PAIRS == 8, v8, typename Num<T>::v4> Piece;
    constexpr int HALF = PAIRS / 2;
    const T* x = x_;
    T* out = out_;
    const float *cos = cos_, *sin = sin_;
    const int32_t* index = index_;
    // Per head `turn` items of two pieces each, then the copied pieces (left
    // out in place).
    const int turn = rotated / (2 * PAIRS), rest = copy ? (head_dim - rotated) / 8 : 0, per_head = turn + rest;
    const int per_row = heads * per_head;
    for (int64_t row0 = (int64_t)blockIdx.x * block_rows; row0 < rows; row0 += (int64_t)gridDim.x * block_rows) {
        const int n = (int)min((int64_t)block_rows, rows - row0) * per_row;
        for (int i = threadIdx.x; i < n; i += blockDim.x) {
            const int r = i / per_row, in_row = i - r * per_row, h = in_row / per_head, j = in_row - h * per_head;
            const int64_t row = row0 + r;
            const T* px = x + row * x_stride + h * head_dim;
            T* po = out + row * out_stride + h * head_dim;
            if (j >= turn) {
                const int c = rotated + (j - turn) * 8;
                *(v8*)(po + c) = *(const v8*)(px + c);
                continue;
            }
            const int place = index[row];
            const bool turned = (uint32_t)place < (uint32_t)places;
            if (!turned && !copy) continue;
            // Halves: the pieces P j and rotated/2 + P j (P = PAIRS), angles P j ..
            // P j + P-1. Neighbours: the pieces 2P j and 2P j + P, the same angles.
            const int c1 = NEIGHBOURS ? 2 * PAIRS * j : PAIRS * j, c2 = NEIGHBOURS ? 2 * PAIRS * j + PAIRS : rotated / 2 + PAIRS * j;
            Piece a = *(const Piece*)(px + c1), b = *(const Piece*)(px + c2);
            if (turned) {
                const float4_t* pc = (const float4_t*)(cos + (size_t)place * (rotated / 2) + PAIRS * j);
                const float4_t* ps = (const float4_t*)(sin + (size_t)place * (rotated / 2) + PAIRS * j);
                float4_t c[PAIRS / 4], s[PAIRS / 4];
#pragma unroll
                for (int i = 0; i < PAIRS / 4; ++i) {
                    c[i] = pc[i];
                    s[i] = ps[i];
                }
                Piece u, w;
#pragma unroll
                for (int e = 0; e < PAIRS; ++e) {
                    const float ce = c[e / 4][e % 4], se = s[e / 4][e % 4];
                    const int n = 2 * (e % HALF);
                    const float x1 = NEIGHBOURS ? (float)(e < HALF ? a[n] : b[n]) : (float)a[e];
                    const float x2 = NEIGHBOURS ? (float)(e < HALF ? a[n + 1] : b[n + 1]) : (float)b[e];
                    const T y1 = (T)(x1 * ce - x2 * se), y2 = (T)(x2 * ce + x1 * se);
                    if constexpr (NEIGHBOURS) {
                        (e < HALF ? u : w)[n] = y1;
                        (e < HALF ? u : w)[n + 1] = y2;
                    } else {
                        u[e] = y1;
                        w[e] = y2;
                    }
                }
                a = u;
                b = w;
            }
            *(Piece*)(po + c1) = a;
            *(Piece*)(po + c2) = b;
        }
    }
}

template <class T, bool NEIGHBOURS, int PAIRS>
hipError_t launch(const dhx_packed_rotation& p, hipStream_t s) {
    const int copy = p.x != p.out;
    const int per_row = (int)p.heads * (int)(p.rotated / (2 * PAIRS) + (copy ? (p.head_dim - p.rotated) / 8 : 0));
    const int block_rows = per_row >= kItems ? 1 : kItems / per_row;
    const uint64_t blocks = std::min<uint64_t>((p.rows + block_rows - 1) / block_rows, kMostBlocks);
    const int threads = std::min(kMostThreads, (per_row * block_rows + 63) / 64 * 64);
    return enqueue(packed_rotate_kernel<T, NEIGHBOURS, PAIRS>, dim3((unsigned)blocks), dim3((unsigned)threads), 0, s, p.x, p.out, p.cos,
                   p.sin, p.index, p.x_stride, p.out_stride, (int)p.rows, (int)p.places, (int)p.heads, (int)p.head_dim,
                   (int)p.rotated, copy, block_rows);
}

template <class T>
hipError_t launch_type(const dhx_packed_rotation& p, hipStream_t s) {
    if (p.rotated % 16 == 0) return p.neighbours ? launch<T, true, 8>(p, s) : launch<T, false, 8>(p, s);
    return p.neighbours ? launch<T, true, 4>(p, s) : launch<T, false, 4>(p, s);
}

}  // namespace

hipError_t launch_packed_rotation(const dhx_packed_rotation& p, hipStream_t s) {
    return p.type == DHX_F16 ? launch_type<half_t>(p, s) : launch_type<bf16_t>(p, s);
}

}  // namespace dhx
