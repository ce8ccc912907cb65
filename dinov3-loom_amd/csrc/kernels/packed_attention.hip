// Softmax attention on packed batches (include/dinov3_packed.h): every
// sequence of its own length, grouped heads, causal or not, any number of
// queries against any number of keys.
//
// The queries of the heads that share a key head are the rows of one matrix:
// row r of a sequence is its token r / group, head r % group of the group. A
// tile of rows walks the keys once, with the running maximum and sum of the
// softmax, and everything is computed transposed so that a lane owns one row:
//   S^T = K . Q^T      (MFMA a = K rows from LDS, b = Q^T held in registers)
//   O^T += V^T . P^T   (MFMA a = V^T rows, LDS transpose reads of the V block;
//                       b = P^T straight from the S^T accumulators)
// Lane l holds row l % 32 and 16 of every 32 keys, lane l ^ 32 the other 16.
// exp(scale (s - m)) is one FMA and v_exp_f32 per score, with m the running
// maximum of the raw scores, moved only when a block's weights against it sum
// past e^8 (its maximum is then needed, and O is rescaled); the sum keeps the
// float32 weights, P is rounded to the type of V for its product.
//
// K and V blocks come by DMA straight into LDS, 128- or 256-byte rows whose
// 16-byte chunks are XOR-swizzled by the row, so that the row reads of K and
// the transpose reads of V spread over all banks.
#include <algorithm>

#include "packed.hpp"

namespace dhx {
namespace {

constexpr int kThreads = 256;
constexpr float kLazySum = 2980.957987f;  // e^8, the slack of the running maximum
constexpr float kNoMax = -1e30f;          // running maximum of a row that has seen no key

// D: head channels as the kernel multiplies them (a multiple of 32; channels
// from head_dim on are zero in Q and K and dropped from O).
template <int D>
struct Geo {
    static constexpr int PITCH = D <= 64 ? 64 : 128;  // elements of a K or V row in LDS
    static constexpr int CH = PITCH / 8;              // 16-byte chunks of it
    static constexpr int ROWS = 64 / CH;              // rows that one DMA load moves
    static constexpr int KK = D / 16;                 // MFMA steps of S
    static constexpr int CT = D / 32;                 // 32-channel blocks of O
};

template <class T>
__device__ __forceinline__ typename Num<T>::v4 read_tr(const T* p) {
    const short4_t v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)p);
    return __builtin_bit_cast(typename Num<T>::v4, v);
}

#define DHX_PACKED_ATTENTION_PARAMS Addr q_starts_, Addr k_starts_, Addr q_, Addr k_, Addr v_, int sequences, int group, int kv_heads, int head_dim, int q_rows, int k_rows, int causal, int slots, int splits, float c, Addr out_, Addr lse_, Addr part_, uint64_t q_stride, uint64_t k_stride, uint64_t v_stride, uint64_t out_stride, uint64_t q_head, uint64_t k_head, uint64_t v_head, uint64_t out_head

// Tile and key head of a workgroup. Workgroups go round the 8 XCDs, each with
// its own L2, so the key heads are dealt to the XCDs (an XCD walks one head's
// keys and values at a time) and, where there are fewer than 8, a head's items
// in turn to the XCDs that share it.
struct Place {
    int head, item;
};
__host__ __device__ inline int xcd_share(int kv_heads) { return kv_heads % 8 == 0 ? 8 : kv_heads % 4 == 0 ? 4 : kv_heads % 2 == 0 ? 2 : 1; }
__device__ __forceinline__ Place place_of(int g, int slots, int kv_heads) {
    const int share = xcd_share(kv_heads), m = 8 / share, per = (slots + m - 1) / m;
    const int x = g & 7, i = g >> 3, h = i / per;
    return Place{x % share + share * h, (i - h * per) * m + x / share};
}

// A workgroup's rows and its sequence.
struct Tile {
    int q0, lq, k0, lk;  // the sequence's first query row and key row and their numbers
    int row0;            // first row of the tile within the sequence, in rows of the group
};

// Finds the tile of 2^SHIFT rows of slot `slot`: sequence s has the slots from
// starts[s] * group / 2^SHIFT + s on, at least as many as it has tiles. False if the
// slot has no rows. For up to 64 sequences a lane holds one of them: one load's
// latency. (Tiles handed out by the keys they see, most first, were no faster:
// 145 us against 145 for ten ragged prompts, 94 against 95 for 39 images of
// 201 to 4101 tokens, and their search cost 1.5 us.)
template <int SHIFT>
__device__ __forceinline__ bool find_tile(Tile& t, int slot, const int32_t* q_starts, const int32_t* k_starts, int sequences,
                                          int group, int q_rows, int k_rows) {
    const int lane = threadIdx.x & 63;
    int s = 0;
    auto base = [&](int s) { return (int64_t)((uint32_t)start_at(q_starts, s, q_rows) * (uint32_t)group >> SHIFT) + s; };
    if (sequences > 64) s = max(wave_last(sequences, slot, base), 0);
    const int mine = min(s + lane, sequences - 1);  // of many only the first counts
    const int q0 = start_at(q_starts, mine, q_rows), q1 = start_at(q_starts, mine + 1, q_rows);
    const int k0 = start_at(k_starts, mine, k_rows), k1 = start_at(k_starts, mine + 1, k_rows);
    const int64_t from = (int64_t)((uint32_t)q0 * (uint32_t)group >> SHIFT) + mine;
    const int j = sequences > 64 ? 0 : max(__builtin_popcountll(__ballot(lane < sequences && from <= slot)) - 1, 0);
    t.q0 = __builtin_amdgcn_readlane(q0, j);
    t.lq = max(0, __builtin_amdgcn_readlane(q1, j) - t.q0);
    t.k0 = __builtin_amdgcn_readlane(k0, j);
    t.lk = max(0, __builtin_amdgcn_readlane(k1, j) - t.k0);
    const int64_t row0 = ((int64_t)slot - (int64_t)((uint32_t)t.q0 * (uint32_t)group >> SHIFT) - (s + j)) << SHIFT;
    if (row0 < 0 || row0 >= (int64_t)t.lq * group) return false;
    t.row0 = (int)row0;
    return true;
}

// The running state of one lane's row.
template <class T, int D>
struct Row {
    typename Num<T>::v8 qf[Geo<D>::KK];
    float16_t o[Geo<D>::CT];
    float m = kNoMax, l = 0.f;  // l: the sum of this lane's keys only, the other half is in lane ^ 32
    int limit;  // keys 0 .. limit-1 of the sequence are seen
};

// Loads of a 32-key block for one wave's lane: which LDS elements it reads.
struct LaneAt {
    int k, v;
};
template <int PITCH>
__device__ __forceinline__ LaneAt lane_at(int lane) {
    const int l32 = lane & 31, hi = lane >> 5;
    return LaneAt{lds_at<PITCH>(l32, hi * 8), lds_at<PITCH>(4 * hi + ((lane & 15) >> 2), 16 * ((lane >> 4) & 1) + 4 * (lane & 3))};
}

// A weight of zero times a value that is not finite is not zero, and in a block
// that some lane does not wholly see such a value may be none of its row's
// business. So they leave zeros behind in the operands of the product, and reach
// the rows that see their keys apart: the product of their places (1 or 0) and
// the keys seen (1 or 0) tells which channels of which rows get an infinity or
// no number.
template <class T, int D>
__device__ __forceinline__ void add_not_finite(Row<T, D>& st, typename Num<T>::v8 (&va)[Geo<D>::CT][2], int key0, int hi) {
    using G = Geo<D>;
    typedef typename Num<T>::v8 v8;
    uint32_t all = 0;
#pragma unroll
    for (int ct = 0; ct < G::CT; ++ct)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int w = 0; w < 4; ++w) all |= not_finite<T>(__builtin_bit_cast(uint4_t, va[ct][ks])[w]);
    if (__builtin_expect(!__any((all & 0x80008000u) != 0), 1)) return;
    const int left = st.limit - key0 - 4 * hi;
    v8 seen[2];
#pragma unroll
    for (int r = 0; r < 16; ++r) seen[r / 8][r % 8] = (T)(8 * (r >> 2) + (r & 3) < left ? 1.f : 0.f);
#pragma unroll
    for (int ct = 0; ct < G::CT; ++ct)
#pragma unroll
        for (int kind = 0; kind < 3; ++kind) {
            __builtin_amdgcn_sched_barrier(0);  // one at a time: this is no place for registers
            const float what = kind == 0 ? __builtin_inff() : kind == 1 ? -__builtin_inff() : __builtin_nanf("");
            float16_t f = {};
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                v8 here;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float v = (float)va[ct][ks][e];
                    const bool is = kind < 2 ? v == what : v != v;
                    here[e] = (T)(is ? 1.f : 0.f);
                    if (is) va[ct][ks][e] = (T)0.f;
                }
                f = Num<T>::mfma(here, seen[ks], f);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) st.o[ct][r] += f[r] > 0.f ? what : 0.f;
        }
}

// One step over a 32-key block at sK, sV (32 rows), whose first key is key0 of
// the sequence. mask (wave-uniform): some lane does not see all of its keys.
template <class T, int D>
__device__ __forceinline__ void attend(Row<T, D>& st, const T* sK, const T* sV, int key0, bool mask, float c, LaneAt at,
                                       int hi) {
    using G = Geo<D>;
    typedef typename Num<T>::v8 v8;
    float16_t s = {};
#pragma unroll
    for (int kk = 0; kk < G::KK; ++kk) s = Num<T>::mfma(*(const v8*)(sK + (at.k ^ (kk << 4))), st.qf[kk], s);
    v8 va[G::CT][2];
#pragma unroll
    for (int ct = 0; ct < G::CT; ++ct)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            const T* p = sV + ks * 16 * G::PITCH;
            va[ct][ks] = __builtin_shufflevector(read_tr(p + (at.v ^ (ct << 5))),
                                                 read_tr(p + (at.v ^ (ct << 5) ^ 16) + 8 * G::PITCH), 0, 1, 2, 3, 4, 5, 6, 7);
        }
    if (mask) {
        const int left = st.limit - key0 - 4 * hi;
#pragma unroll
        for (int r = 0; r < 16; ++r)
            if (8 * (r >> 2) + (r & 3) >= left) s[r] = -__builtin_inff();
    }
    float p[16];
    auto weights = [&](float m) {
        const float mc = m * c;
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            p[r] = fast_exp2(fmaf(s[r], c, -mc));
            sum += p[r];
        }
        return sum;
    };
    float sum = weights(st.m);
    if (__any(!(sum <= kLazySum))) {
        float mx = s[0], both = half_pair_sum(sum);
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
        const bool grow = !(both <= kLazySum);  // alike in both halves of the row
        const float m = grow ? fmaxf(half_pair_max(mx), st.m) : st.m, alpha = fast_exp2((st.m - m) * c);
        st.l *= alpha;
#pragma unroll
        for (int ct = 0; ct < G::CT; ++ct) st.o[ct] *= alpha;
        st.m = m;
        sum = weights(m);
    }
    st.l += sum;
    v8 pb[2];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int e = 0; e < 8; ++e) pb[ks][e] = (T)p[8 * ks + e];
    if (mask) add_not_finite<T, D>(st, va, key0, hi);
#pragma unroll
    for (int ct = 0; ct < G::CT; ++ct)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) st.o[ct] = Num<T>::mfma(va[ct][ks], pb[ks], st.o[ct]);
}

// This wave's share of a block of KB keys of one matrix: LOADS DMA loads of
// ROWS rows each, the wave's rows being first .. first + LOADS * ROWS - 1.
template <int D, int LOADS>
struct Mover {
    using G = Geo<D>;
    const char* base;  // of the sequence's first key, this head
    uint64_t pitch;    // bytes between rows
    int row, chunk[LOADS];
    bool full;         // every chunk of a row exists
    __device__ __forceinline__ Mover(const void* first_key, uint64_t stride, int head_dim, int first, int lane)
        : base((const char*)first_key), pitch(stride * 2), row(first + lane / G::CH), full(head_dim == G::PITCH) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) chunk[j] = (lane % G::CH) ^ slot_of<G::PITCH>(row + j * G::ROWS);
    }
    // Keys key0 .. of the block, `left` of them in the sequence, to LDS at `to`
    // (the wave's own rows' place).
    template <class T>
    __device__ __forceinline__ void move(int key0, int left, int block, int head_dim, T* to) const {
        const char* tile = base + (uint64_t)key0 * pitch;
        if (full && left >= block) {
#pragma unroll
            for (int j = 0; j < LOADS; ++j)
                dma16(tile + ((uint32_t)(row + j * G::ROWS) * (uint32_t)pitch + chunk[j] * 16), to + j * 512);
        } else {
#pragma unroll
            for (int j = 0; j < LOADS; ++j) {
                const int r = row + j * G::ROWS;
                const bool there = r < left && chunk[j] * 8 < head_dim;
                dma16(there ? tile + ((uint32_t)r * (uint32_t)pitch + chunk[j] * 16) : (const char*)&kZeros, to + j * 512);
            }
        }
    }
};

// Q fragments of row r of the tile's sequence (zeros behind its last row and
// its last channel) and the keys it sees.
template <class T, int D>
__device__ __forceinline__ void load_row(Row<T, D>& st, const T* q, const Tile& t, int r, int group, int head_dim,
                                         int causal, uint64_t q_stride, uint64_t q_head, int hi) {
    typedef typename Num<T>::v8 v8;
    const int token = r / group, h = r - token * group;
    const bool there = token < t.lq;
    const T* p = q + (uint64_t)(t.q0 + token) * q_stride + h * q_head;
#pragma unroll
    for (int kk = 0; kk < Geo<D>::KK; ++kk) {
        const int ch = kk * 16 + hi * 8;
        st.qf[kk] = there && ch < head_dim ? *(const v8*)(p + ch) : v8{};
    }
#pragma unroll
    for (int ct = 0; ct < Geo<D>::CT; ++ct) st.o[ct] = float16_t{};
    st.limit = !there ? 0 : causal ? min(max(token + 1 + t.lk - t.lq, 0), t.lk) : t.lk;
}

// O / l of one lane's row, in 16-byte pieces; `head0` the group's first head.
template <class T, int D>
__device__ __forceinline__ void store_row(const Row<T, D>& st, T* out, float* lse, const Tile& t, int r, int group,
                                          int head0, int heads, int head_dim, float c, uint64_t out_stride,
                                          uint64_t out_head, int hi) {
    typedef typename Num<T>::v4 v4;
    typedef typename Num<T>::v8 v8;
    const int token = r / group, h = r - token * group;
    const bool there = token < t.lq;
    const float inv = st.l != 0.f ? 1.0f / st.l : 0.f;  // a sum that is not a number stays one, also below
    T* p = out + (uint64_t)(t.q0 + token) * out_stride + h * out_head;
#pragma unroll
    for (int ct = 0; ct < Geo<D>::CT; ++ct)
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            v4 g0, g1;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                g0[e] = (T)(st.o[ct][8 * kk + e] * inv);
                g1[e] = (T)(st.o[ct][8 * kk + 4 + e] * inv);
            }
            const v8 piece = __builtin_bit_cast(v8, frag_swap(__builtin_bit_cast(half4_t, g0), __builtin_bit_cast(half4_t, g1)));
            const int ch = ct * 32 + kk * 16 + hi * 8;
            if (there && ch < head_dim) *(v8*)(p + ch) = piece;
        }
    if (lse && there && hi == 0)
        lse[(uint64_t)(t.q0 + token) * heads + head0 + h] = st.l != 0.f ? (st.m * c + __log2f(st.l)) * kLn2 : -__builtin_inff();
}

// A tile of 32 WAVES rows, 32 per wave; the waves of a group share blocks of 16
// WAVES keys, the next one on its way while one is used. GROUPS > 1: so many such
// groups take the blocks in turn and join at the end, which shortens a tile's
// chain where it has a CU to itself.
template <class T, int D, int GROUPS, int WAVES>
__global__ __launch_bounds__(64 * WAVES * GROUPS, D <= 64 ? 4 : 2) void packed_attention_kernel(DHX_PACKED_ATTENTION_PARAMS) {
    using G = Geo<D>;
    constexpr int KB = 16 * WAVES, LOADS = KB / WAVES / G::ROWS, BLK = KB * G::PITCH;
    __shared__ __attribute__((aligned(16))) T sK0[GROUPS * BLK], sK1[GROUPS * BLK];
    __shared__ __attribute__((aligned(16))) T sV0[GROUPS * BLK], sV1[GROUPS * BLK];
    __shared__ float2_t sML[GROUPS > 1 ? GROUPS - 1 : 1][WAVES][32];
    const Place at = place_of(blockIdx.x, slots, kv_heads);
    if (at.head >= kv_heads || at.item >= slots) return;
    Tile t;
    // From the last slot on: a causal prompt's longest tiles begin first.
    if (!find_tile<WAVES == 4 ? 7 : 6>(t, slots - 1 - at.item, q_starts_, k_starts_, sequences, group, q_rows, k_rows)) return;
    const int tid = threadIdx.x, lane = tid & 63, all_waves = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wave = all_waves % WAVES, part = all_waves / WAVES;
    const int l32 = lane & 31, hi = lane >> 5;
    const int head0 = at.head * group;

    Row<T, D> st;
    const int first = t.row0 + wave * 32, row = first + l32;
    load_row(st, (const T*)q_ + head0 * q_head, t, row, group, head_dim, causal, q_stride, q_head, hi);
    // Keys that the tile's last row sees, those that all rows of this wave see,
    // and those that any of them sees.
    const int rows = t.lq * group, last = min(t.row0 + 32 * WAVES - 1, rows - 1), wave_last_row = min(first + 31, rows - 1);
    auto seen = [&](int r) { return causal ? min(max(r / group + 1 + t.lk - t.lq, 0), t.lk) : t.lk; };
    const int keys = seen(last), all = seen(min(first, rows - 1)), any = first < rows ? seen(wave_last_row) : 0;
    const int blocks = (keys + KB - 1) / KB;

    const Mover<D, LOADS> mk((const T*)k_ + (uint64_t)t.k0 * k_stride + at.head * k_head, k_stride, head_dim, wave * (KB / WAVES), lane);
    const Mover<D, LOADS> mv((const T*)v_ + (uint64_t)t.k0 * v_stride + at.head * v_head, v_stride, head_dim, wave * (KB / WAVES), lane);
    const LaneAt la = lane_at<G::PITCH>(lane);
    T *k0 = sK0 + part * BLK, *k1 = sK1 + part * BLK, *v0 = sV0 + part * BLK, *v1 = sV1 + part * BLK;
    auto move = [&](T* k, T* v, int b) {
        mk.move(b * KB, t.lk - b * KB, KB, head_dim, k + wave * (KB / WAVES) * G::PITCH);
        mv.move(b * KB, t.lk - b * KB, KB, head_dim, v + wave * (KB / WAVES) * G::PITCH);
    };
    auto step = [&](T* k, T* v, T* next_k, T* next_v, int b) {
        wait_vm<0>();  // block b has landed, and no wave reads the other block any more
        wait_lgkm();
        barrier();
        if (b + GROUPS < blocks) move(next_k, next_v, b + GROUPS);
#pragma unroll(D <= 64 ? 1 : 2)
        for (int i = 0; i < KB; i += 32) {
            const int key0 = b * KB + i;
            if (key0 >= any) break;
            attend<T, D>(st, k + i * G::PITCH, v + i * G::PITCH, key0, key0 + 32 > all, c, la, hi);
        }
    };
    // Every wave takes part in every step's barrier, also without a block.
    if (part < blocks) move(k0, v0, part);
    for (int b = 0; b < blocks; b += 2 * GROUPS) {
        step(k0, v0, k1, v1, b + part);
        if (b + GROUPS < blocks) step(k1, v1, k0, v0, b + GROUPS + part);
    }
    st.l = half_pair_sum(st.l);
    if constexpr (GROUPS > 1) {
        // The other groups' O through their own blocks, as float32 [row][channels],
        // a quarter (of PITCH) of them in each, 16-byte pieces swizzled by the row.
        constexpr int WIDE = G::PITCH / 4, PIECES = WIDE / 4;
        auto piece = [&](int of, int ct, int g4) __attribute__((always_inline)) {
            const int ch = ct * 32 + 8 * g4, at = ch / WIDE;
            float* o = (float*)((at == 0 ? sK0 : at == 1 ? sV0 : at == 2 ? sK1 : sV1) + of * BLK) + wave * 32 * WIDE;
            return (float4_t*)(o + l32 * WIDE + (((ch % WIDE / 4 + hi) ^ (l32 % PIECES)) << 2));
        };
        wait_lgkm();
        barrier();  // every wave has read its last block
        if (part > 0) {
            if (hi == 0) sML[part - 1][wave][l32] = float2_t{st.m, st.l};
#pragma unroll
            for (int ct = 0; ct < G::CT; ++ct)
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4)
                    *piece(part, ct, g4) =
                        float4_t{st.o[ct][4 * g4], st.o[ct][4 * g4 + 1], st.o[ct][4 * g4 + 2], st.o[ct][4 * g4 + 3]};
        }
        __syncthreads();
        if (part > 0) return;
#pragma unroll
        for (int of = 1; of < GROUPS; ++of) {
            const float2_t other = sML[of - 1][wave][l32];
            const float m = fmaxf(st.m, other[0]), mine = fast_exp2((st.m - m) * c), its = fast_exp2((other[0] - m) * c);
            st.l = st.l * mine + other[1] * its;
            st.m = m;
#pragma unroll
            for (int ct = 0; ct < G::CT; ++ct)
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    const float4_t o = *piece(of, ct, g4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) st.o[ct][4 * g4 + e] = st.o[ct][4 * g4 + e] * mine + o[e] * its;
                }
        }
    }
    store_row(st, (T*)out_ + head0 * out_head, (float*)lse_, t, row, group, head0, group * kv_heads, head_dim, c, out_stride,
              out_head, hi);
}

// Item `item` of all (sequence, tile, part), in that order: its tile and part.
// False behind the last one. The search goes on from the 64 sequences that it found
// the last item in (a workgroup's items come in order), so a workgroup walks the
// sequences once, whatever the number of its items. (From the first ones for each
// item, 4096 single tokens with 200 keys each, 32 heads of 128 on 8, took 1659 us
// instead of 818, 16384 with 16 keys, 6 heads of 64, 6180 instead of 852.)
struct Item {
    Tile t;
    int part, parts;
    int s0 = 0;           // the 64 sequences, and the items in front of them
    uint32_t before = 0;
};
__device__ __forceinline__ bool find_item(Item& it, uint32_t item, const int32_t* q_starts, const int32_t* k_starts, int sequences,
                                          int group, int q_rows, int k_rows, int splits, int span) {
    const int lane = threadIdx.x & 63;
    item -= it.before;
    for (; it.s0 < sequences; it.s0 += 64) {
        const int s0 = it.s0, s = min(s0 + lane, sequences - 1);
        const int q0 = start_at(q_starts, s, q_rows), q1 = start_at(q_starts, s + 1, q_rows);
        const int k0 = start_at(k_starts, s, k_rows), k1 = start_at(k_starts, s + 1, k_rows);
        const int lq = s0 + lane < sequences ? max(0, q1 - q0) : 0, lk = max(0, k1 - k0);
        const uint32_t tiles = ((uint32_t)lq * (uint32_t)group + 31) >> 5;
        const uint32_t parts = max(1, min(splits, (((lk + 31) >> 5) + span - 1) / span));
        const uint32_t to = wave_sum_to(tiles * parts);
        const uint64_t behind = __ballot(to > item);
        if (behind == 0) {
            const uint32_t all = __builtin_amdgcn_readlane(to, 63);
            item -= all;
            it.before += all;
            continue;
        }
        const int j = __builtin_ctzll(behind);
        const uint32_t n = __builtin_amdgcn_readlane(parts, j);
        const uint32_t in = item - (__builtin_amdgcn_readlane(to, j) - (uint32_t)__builtin_amdgcn_readlane(tiles, j) * n);
        it.t = Tile{__builtin_amdgcn_readlane(q0, j), __builtin_amdgcn_readlane(lq, j), __builtin_amdgcn_readlane(k0, j),
                    __builtin_amdgcn_readlane(lk, j), (int)(in / n * 32)};
        it.part = (int)(in % n);
        it.parts = (int)n;
        return (uint32_t)it.t.row0 < (uint32_t)(it.t.lq * group);
    }
    return false;
}

// A tile of 32 rows whose NW waves each walk key blocks of their own (every
// NW-th block of 32, through a ring of two blocks in LDS that no other wave
// touches, so without barriers) and join at the end. For launches whose rows
// are too few to fill the chip with 128-row tiles, single tokens among them;
// several workgroups may also share a sequence's keys, a part of `span` blocks
// each, and leave their sums in the workspace for packed_join_kernel: of part
// p, row i and head h D float32 of O at ((p * q_rows + i) * heads + h) * D, and
// (m, l) likewise behind all of those. A workgroup takes items until there are
// none, so an item costs nothing that is not there; gridDim.x counts the
// workgroups of a key head.
template <class T, int D, int NW>
__global__ __launch_bounds__(64 * NW, 1) void packed_attention_few_kernel(DHX_PACKED_ATTENTION_PARAMS, int span) {
    using G = Geo<D>;
    constexpr int LOADS = 32 / G::ROWS, BLK = 32 * G::PITCH;
    __shared__ __attribute__((aligned(16))) T sK0[NW * BLK], sK1[NW * BLK];
    __shared__ __attribute__((aligned(16))) T sV0[NW * BLK], sV1[NW * BLK];
    __shared__ float2_t sML[NW][32];
    const Place at = place_of(blockIdx.x, slots, kv_heads);
    if (at.head >= kv_heads || at.item >= slots) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, hi = lane >> 5;
    const int head0 = at.head * group, heads = group * kv_heads;
    Item it;
    // Starts that decrease may make any number of items, more than 32 bits count;
    // none beyond what these rows and sequences can have otherwise is taken.
    const uint32_t all_rows_of_group = (uint32_t)q_rows * (uint32_t)group;
    const uint32_t most = min(all_rows_of_group / 32 + (uint32_t)sequences, all_rows_of_group) * (uint32_t)splits;
    for (uint32_t item = at.item; item < most; item += slots) {
    if (!find_item(it, item, q_starts_, k_starts_, sequences, group, q_rows, k_rows, splits, span)) return;
    const Tile& t = it.t;

    Row<T, D> st;
    const int row = t.row0 + l32, rows = t.lq * group, last = min(t.row0 + 31, rows - 1);
    load_row(st, (const T*)q_ + head0 * q_head, t, row, group, head_dim, causal, q_stride, q_head, hi);
    auto seen = [&](int r) { return causal ? min(max(r / group + 1 + t.lk - t.lq, 0), t.lk) : t.lk; };
    const int all = seen(t.row0), blocks = (seen(last) + 31) >> 5;
    const int lo = min(it.part * span, blocks), hi_block = it.part == it.parts - 1 ? blocks : min(lo + span, blocks);

    const Mover<D, LOADS> mk((const T*)k_ + (uint64_t)t.k0 * k_stride + at.head * k_head, k_stride, head_dim, 0, lane);
    const Mover<D, LOADS> mv((const T*)v_ + (uint64_t)t.k0 * v_stride + at.head * v_head, v_stride, head_dim, 0, lane);
    const LaneAt la = lane_at<G::PITCH>(lane);
    T *k0 = sK0 + wave * BLK, *k1 = sK1 + wave * BLK, *v0 = sV0 + wave * BLK, *v1 = sV1 + wave * BLK;
    auto move = [&](T* k, T* v, int b) {
        mk.move(b * 32, t.lk - b * 32, 32, head_dim, k);
        mv.move(b * 32, t.lk - b * 32, 32, head_dim, v);
    };
    auto step = [&](const T* k, const T* v, T* next_k, T* next_v, int b) {
        wait_lgkm();  // the other block has been read
        if (b + NW < hi_block) {
            move(next_k, next_v, b + NW);
            wait_vm<2 * LOADS>();
        } else {
            wait_vm<0>();
        }
        attend<T, D>(st, k, v, b * 32, b * 32 + 32 > all, c, la, hi);
    };
    int b = lo + wave;
    if (b < hi_block) move(k0, v0, b);
    wait_vm<0>();  // Q too, which no counted wait behind DMA loads would prove
    for (; b < hi_block; b += 2 * NW) {
        step(k0, v0, k1, v1, b);
        if (b + NW < hi_block) step(k1, v1, k0, v0, b + NW);
    }

    st.l = half_pair_sum(st.l);
    if constexpr (NW > 1) {
        // Join: each wave's O in its own first blocks as float32 [row][channel]
        // (half of the channels in each), 16-byte pieces swizzled by the row.
        constexpr int HALF = G::PITCH / 2, PIECES = HALF / 4;
        wait_lgkm();
        if (hi == 0) sML[wave][l32] = float2_t{st.m, st.l};
#pragma unroll
        for (int ct = 0; ct < G::CT; ++ct) {
            float* o = (float*)(ct * 32 < HALF ? k0 : v0) + l32 * HALF;
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const int piece = (ct * 32 % HALF) / 4 + 2 * g4 + hi;
                *(float4_t*)(o + ((piece ^ (l32 % PIECES)) << 2)) =
                    float4_t{st.o[ct][4 * g4], st.o[ct][4 * g4 + 1], st.o[ct][4 * g4 + 2], st.o[ct][4 * g4 + 3]};
            }
        }
        __syncthreads();
        if (wave == 0) {
            float m = kNoMax, l = 0.f, part[NW];
#pragma unroll
            for (int w = 0; w < NW; ++w) m = fmaxf(m, sML[w][l32][0]);
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                part[w] = fast_exp2((sML[w][l32][0] - m) * c);
                l += part[w] * sML[w][l32][1];
            }
            st.m = m;
            st.l = l;
#pragma unroll
            for (int ct = 0; ct < G::CT; ++ct)
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    const int piece = (ct * 32 % HALF) / 4 + 2 * g4 + hi;
                    float4_t sum = {};
#pragma unroll
                    for (int w = 0; w < NW; ++w) {
                        const float* o = (const float*)((ct * 32 < HALF ? sK0 : sV0) + w * BLK) + l32 * HALF;
                        sum += part[w] * *(const float4_t*)(o + ((piece ^ (l32 % PIECES)) << 2));
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) st.o[ct][4 * g4 + e] = sum[e];
                }
        }
    }
    if (NW == 1 || wave == 0) {
        if (splits == 1) {
            store_row(st, (T*)out_ + head0 * out_head, (float*)lse_, t, row, group, head0, heads, head_dim, c, out_stride, out_head, hi);
        } else if (row < rows) {
            const int token = row / group, h = row - token * group;
            const uint64_t all_rows = (uint64_t)q_rows * heads, at_row = (uint64_t)(t.q0 + token) * heads + head0 + h;
            float* o = (float*)part_ + (it.part * all_rows + at_row) * D;
            float2_t* ml = (float2_t*)((float*)part_ + (uint64_t)splits * all_rows * D) + at_row;
            if (hi == 0) ml[it.part * all_rows] = float2_t{st.m, st.l};
            if (it.part == 0)  // the parts that the sequence does not have
                for (int i = it.parts + hi; i < splits; i += 2) ml[i * all_rows] = float2_t{kNoMax, 0.f};
            if (st.l != 0.f) {  // else the part is not read
#pragma unroll
                for (int ct = 0; ct < G::CT; ++ct)
#pragma unroll
                    for (int g4 = 0; g4 < 4; ++g4)
                        *(float4_t*)(o + ct * 32 + 8 * g4 + 4 * hi) =
                            float4_t{st.o[ct][4 * g4], st.o[ct][4 * g4 + 1], st.o[ct][4 * g4 + 2], st.o[ct][4 * g4 + 3]};
            }
        }
    }
    if constexpr (NW > 1) __syncthreads();  // the blocks may be filled again
    }
}

#define DHX_JOIN_PARAMS Addr part_, Addr q_starts_, Addr out_, Addr lse_, int sequences, int q_rows, int heads, int head_dim, int splits, float c, uint64_t out_stride, uint64_t out_head

// One wave per row and head: the splits' parts, weighted by 2^(c (m - max m)). A
// split without a sum (its keys are not seen, or weigh nothing) has stored no O.
// Groups of lanes take a split each, four floats per lane, eight loads on their
// way.
template <class T, int D>
__global__ __launch_bounds__(kThreads) void packed_join_kernel(DHX_JOIN_PARAMS) {
    constexpr int LANES = D > 64 ? 32 : D / 4, SIDE = 64 / LANES, DEEP = 8;
    typedef typename Num<T>::v4 v4;
    const int lane = threadIdx.x & 63;
    const uint64_t all = (uint64_t)q_rows * heads;
    for (uint64_t r = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < all; r += (uint64_t)gridDim.x * 4) {
        const int row = (int)(r / heads), head = (int)(r - (uint64_t)row * heads);
        const int32_t* starts = q_starts_;
        if (row < start_at(starts, 0, q_rows) || row >= start_at(starts, sequences, q_rows)) continue;
        const float* part = part_;
        const float2_t* ml = (const float2_t*)(part + (uint64_t)splits * all * D) + r;
        const int ch = (lane % LANES) * 4;
        const float* mine = part + r * D + min(ch, D - 4);
        float m = kNoMax, l = 0.f;
        float4_t o = {};
        for (int s0 = 0; s0 < splits; s0 += 64) {
            const float2_t at = s0 + lane < splits ? ml[(s0 + lane) * all] : float2_t{kNoMax, 0.f};
            const uint64_t some = __ballot(at[1] != 0.f);  // also one that is not a number
            if (some == 0) continue;
            const int first = __builtin_ctzll(some), n = 64 - __builtin_clzll(some);
            float top = fmaxf(m, at[0]);
#pragma unroll
            for (int i = 32; i; i >>= 1) top = fmaxf(top, __shfl_xor(top, i));
            const float w = some >> lane & 1 ? fast_exp2((at[0] - top) * c) : 0.f, before = fast_exp2((m - top) * c);
            m = top;
            l = l * before + w * at[1];
            o *= before;
            for (int j0 = 0; j0 < n; j0 += SIDE * DEEP) {
                float4_t p[DEEP];
                float pw[DEEP];
#pragma unroll
                for (int d = 0; d < DEEP; ++d) {
                    const int j = j0 + d * SIDE + lane / LANES;
                    const int from = j < n && (some >> j & 1) ? j : first;
                    p[d] = *(const float4_t*)(mine + (uint64_t)(s0 + from) * all * D);
                    const float wj = __shfl(w, from);
                    pw[d] = from == j ? wj : 0.f;
                }
#pragma unroll
                for (int d = 0; d < DEEP; ++d) o += pw[d] * p[d];
            }
        }
#pragma unroll
        for (int i = 32; i; i >>= 1) l += __shfl_xor(l, i);
#pragma unroll
        for (int i = LANES; i < 64; i <<= 1)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], i);
        const float inv = l != 0.f ? 1.0f / l : 0.f;
        if (lane < LANES && ch < head_dim) {
            v4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = (T)(o[e] * inv);
            *(v4*)((T*)out_ + (uint64_t)row * out_stride + head * out_head + ch) = y;
        }
        if (lse_.a && lane == 0) ((float*)lse_)[r] = l != 0.f ? (m * c + __log2f(l)) * kLn2 : -__builtin_inff();
    }
}

template <class T, int D>
hipError_t launch(const dhx_packed_attention& p, const AttentionCut& cut, hipStream_t s) {
    const int group = (int)(p.heads / p.kv_heads), share = xcd_share((int)p.kv_heads), m = 8 / share;
    const uint64_t grid = 8 * (p.kv_heads / share) * ((cut.slots + m - 1) / m);
    const float c = p.scale * kLog2e;
    auto tile = [&](auto kernel, int groups) {
        return enqueue(kernel, dim3((unsigned)grid), dim3(64 * groups), 0, s, p.q_starts, p.k_starts, p.q, p.k, p.v,
                       (int)p.sequences, group, (int)p.kv_heads, (int)p.head_dim, (int)p.q_rows, (int)p.k_rows, (int)p.causal,
                       (int)cut.slots, 1, c, p.out, p.lse, p.workspace, p.q_stride, p.k_stride, p.v_stride, p.out_stride,
                       p.q_head_stride, p.k_head_stride, p.v_head_stride, p.out_head_stride);
    };
    if (!cut.few) {
        if constexpr (D <= 64) {
            if (cut.tile == 64) return tile(packed_attention_kernel<T, D, 8, 2>, 16);
            if (cut.waves == 16) return tile(packed_attention_kernel<T, D, 4, 4>, 16);
        } else {
            if (cut.tile == 64) return tile(packed_attention_kernel<T, D, 4, 2>, 8);
        }
        return cut.waves == 8 ? tile(packed_attention_kernel<T, D, 2, 4>, 8) : tile(packed_attention_kernel<T, D, 1, 4>, 4);
    }
    auto few = [&](auto kernel, int waves) {
        return enqueue(kernel, dim3((unsigned)grid), dim3(64 * waves), 0, s, p.q_starts, p.k_starts, p.q, p.k, p.v, (int)p.sequences,
                       group, (int)p.kv_heads, (int)p.head_dim, (int)p.q_rows, (int)p.k_rows, (int)p.causal, (int)cut.slots,
                       (int)cut.splits, c, p.out, p.lse, p.workspace, p.q_stride, p.k_stride, p.v_stride, p.out_stride,
                       p.q_head_stride, p.k_head_stride, p.v_head_stride, p.out_head_stride, (int)cut.span);
    };
    const hipError_t err = cut.waves == 4 ? few(packed_attention_few_kernel<T, D, 4>, 4) : few(packed_attention_few_kernel<T, D, 2>, 2);
    if (err != hipSuccess || cut.splits == 1) return err;
    const uint64_t joins = std::min<uint64_t>((p.q_rows * p.heads + 3) / 4, 1u << 20);
    return enqueue(packed_join_kernel<T, D>, dim3((unsigned)joins), dim3(kThreads), 0, s, p.workspace, p.q_starts,
                   p.out, p.lse, (int)p.sequences, (int)p.q_rows, (int)p.heads, (int)p.head_dim, (int)cut.splits,
                   c, p.out_stride, p.out_head_stride);
}

int padded_dim(uint32_t head_dim) { return head_dim <= 32 ? 32 : head_dim <= 64 ? 64 : head_dim <= 96 ? 96 : 128; }

template <class T>
hipError_t launch_type(const dhx_packed_attention& p, const AttentionCut& cut, hipStream_t s) {
    switch (padded_dim(p.head_dim)) {
        case 32: return launch<T, 32>(p, cut, s);
        case 64: return launch<T, 64>(p, cut, s);
        case 96: return launch<T, 96>(p, cut, s);
        default: return launch<T, 128>(p, cut, s);
    }
}

}  // namespace

// How a launch is cut (times in us on MI355X; causal where heads are grouped).
//
// Few-rows kernel: sequences of at most 32 rows have no use for taller tiles:
// single tokens of 48 requests with 32 heads of 128 on 8, 116.6k keys together, 94
// against 657. And launches of few tiles (in tiles of 64 rows) leave CUs idle
// that parts of the keys fill. Against the best of the others, heads of 64: 1029
// rows and keys of 6 heads 12.2 and 16.0 (102 tiles), five images of 201 tokens
// 7.2 and 7.9 (108), 16384 keys of 1029 rows 132 and 138; but 256 tokens, 32 heads
// on 8, 15.0 and 9.1 (128), 1400 rows and keys, 6 heads, 27.3 and 21.4 (132). Wide
// heads have the chain of a tile shortened by half tiles already, and parts pay
// only along more blocks than there are tiles: 32 heads of 128 on 8, 64 tokens
// (32 tiles) behind 2048 keys 18.5 and 24.6, 1024 keys 15.8 and 16.2; 128 (64)
// behind 4096 37 and 44, 2048 26.1 and 24.6, 512 12.6 and 11.8; 256 (128) behind
// 8192 108 and 80, 256 16.8 and 9.9.
constexpr uint64_t kFewRows = 32, kFewTiles = 112, kLeastParted = 16;
// Tiles of 64 rows, their keys shared by twice the groups, where there is a CU
// for each: a tile's chain is half as long, but a second round of them costs more
// than that. Wide heads, against 128 rows: 512 tokens, 32 heads of 128 on 8, 12.2
// and 14.5 (256 tiles), behind 8192 keys 86 and 121; 1024 tokens, 16 heads of 80,
// 15.7 and 19.6 (256); but 1029 of them 29.6 and 19.8 (272). Heads up to 64, whose
// 128 rows can have four groups too, only along many blocks, for the eight groups
// have to join: 300 tokens, 32 heads on 8, behind 8192 keys 77 and 96 (160), 4096
// 45 and 52, 3000 37 and 39, 2048 29 and 28, 1024 21.5 and 18.3.
constexpr uint64_t kCUs = 256, kEightGroups = 96;
// Where tiles of 128 rows are few enough to run at once, the time of one counts,
// and groups of waves share its keys: 2048 causal tokens, 32 heads of 128 on 8,
// 46.5 with two groups, 52.0 with one (520 tiles), 4096 tokens 154 against 148
// (1032); ragged prompts with 16 heads of 80 28.0, 29.6 (400); 4101 rows and keys,
// 6 heads of 64, 42.1 with four, 50.3 with two, 72.3 with one (198). Four groups
// along blocks enough: 2000 rows and keys 27.2, 31.6 (two), twice 1029 18.9, 19.8,
// three times 581 (19 blocks) 14.6, 13.6.
constexpr uint64_t kShareTiles = 600, kFourGroups = 32;
// Four waves share a tile's keys, without parts, where at most 256 items have
// few enough blocks: 201 x 201, 6 heads, 6.9 (two waves 7.8); four queries and
// 1029 keys of 16 images, 12 heads of 64, 14.3 (16.3); 581 x 581, 6 heads, 9.4
// (13.8; 114 items). Else two: their
// workgroups are more and their joins smaller. A part then has a 384th of all
// blocks and no fewer than 4: one token, 1000 keys, 32 heads of 128 on 8, 11.4
// (16 blocks 17.2), 8192 keys 15.6 with 8 blocks (64 blocks 43); the 48 requests
// above 93 with 64 blocks (8 blocks 103).
constexpr uint64_t kPartShare = 384, kLeastSpan = 4, kMostParts = 256;
// Workgroups of a launch at most: beyond what runs at once an item's own
// workgroup balances unequal ones, beyond this they only wait.
constexpr uint64_t kFewGroups = 2048;

AttentionCut packed_attention_cut(const dhx_packed_attention& p) {
    AttentionCut cut{};
    cut.splits = 1;
    if (p.q_rows == 0) return cut;  // nothing is launched, and there is no tile to share keys out to
    const uint64_t group = p.heads / p.kv_heads, rows = p.q_rows * group;
    const uint64_t longest = std::min<uint64_t>(p.longest_q ? p.longest_q : p.q_rows, p.q_rows) * group;
    const uint64_t keys = std::min<uint64_t>(p.longest_k ? p.longest_k : p.k_rows, p.k_rows), blocks = (keys + 31) / 32;
    // Tiles of 64 rows, if each sequence behind the first one ends in the middle of one.
    const uint64_t halves = (rows + 32 * (uint64_t)p.sequences + 31) / 64 * p.kv_heads;
    const bool wide = p.head_dim > 64;  // else a wave's state leaves room for twice the waves
    cut.few = longest <= kFewRows || (halves <= kFewTiles && (!wide || blocks > std::max(halves, kLeastParted)));
    if (!cut.few) {
        const bool half = halves <= kCUs && (wide || blocks >= kEightGroups);
        cut.slots = rows / (half ? 64 : 128) + p.sequences;
        const uint64_t count = cut.slots * p.kv_heads;
        cut.tile = half ? 64 : 128;
        if (half) cut.waves = wide ? 8 : 16;
        else cut.waves = count > kShareTiles ? 4 : count <= kCUs && blocks >= kFourGroups && !wide ? 16 : 8;
        return cut;
    }
    const uint64_t tiles = std::min<uint64_t>(rows / 32 + p.sequences, rows);
    const uint64_t items = tiles * p.kv_heads;
    cut.waves = items <= 256 && (blocks <= 16 || (items >= 96 && blocks <= 40)) ? 4 : 2;
    if (cut.waves == 2) {
        // Blocks that all tiles walk, if each sequence has its share of both.
        const uint64_t per_sequence = (rows + 32ull * p.sequences - 1) / (32ull * p.sequences);
        const uint64_t work = (p.k_rows + 31) / 32 * per_sequence * p.kv_heads;
        cut.span = std::min<uint64_t>(std::max<uint64_t>(work / kPartShare, kLeastSpan), 1u << 20);
        const uint64_t most = std::min<uint64_t>(kMostParts, std::max<uint64_t>(1, (1ull << 30) / tiles));
        cut.splits = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>((blocks + cut.span - 1) / cut.span, most));
    }
    if (cut.splits == 1) cut.span = 1u << 20;
    else cut.bytes = cut.splits * p.q_rows * p.heads * (padded_dim(p.head_dim) + 2) * 4;
    cut.slots = std::max<uint64_t>(1, std::min<uint64_t>(tiles * cut.splits, kFewGroups / p.kv_heads));
    return cut;
}

hipError_t launch_packed_attention(const dhx_packed_attention& p, hipStream_t s) {
    const AttentionCut cut = packed_attention_cut(p);
    return p.type == DHX_F16 ? launch_type<half_t>(p, cut, s) : launch_type<bf16_t>(p, cut, s);
}

}  // namespace dhx
