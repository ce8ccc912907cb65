/*
 * dinov3_packed.h -- operators on packed batches, on device memory (no
 * counterpart in the reference, whose kernels take images of one size and one
 * set of weights per launch).
 *
 * A packed batch holds the rows of many sequences (images of different sizes,
 * prompts, single tokens) back to back. `starts` is an array of sequences + 1
 * int32 in device memory: sequence s has the rows starts[s] .. starts[s+1]-1,
 * none if the two are equal. The array must not decrease; it is read by the
 * kernels only, so it may change between the replays of a captured graph.
 * Whatever it holds, every call ends and no kernel reads or writes outside 0 ..
 * rows-1 (a value outside is taken as the nearest end). Rows in front of starts[0] and from
 * starts[sequences] on belong to no sequence: their outputs are left as they
 * were.
 *
 * Conventions, as in dinov3_engine.h: 0 = success; otherwise the message is in
 * dhx_last_error(engine), or dhx_last_error(NULL) for the workspace functions
 * and where no engine is given. Every argument is checked before anything is
 * queued: a refused call changes nothing and leaves the engine usable, a
 * failed launch poisons it. The launches are queued on `stream`, a hipStream_t
 * of the engine's GPU, and the call returns without waiting. The memory is the
 * caller's, so NULL is the caller's default stream here (HIP's null stream, on
 * which PyTorch works unless told otherwise), not the engine's own: a program
 * that works on engine regions passes dhx_stream(engine) and the addresses that
 * dhx_address gives. It allocates nothing, records nothing and keeps no address,
 * so it may be captured into a HIP graph. The caller's current device is left
 * as it was.
 *
 * Matrices are row-major with a distance between rows (`_stride`, in
 * elements); rows, strides and addresses are multiples of 16 bytes, so sizes
 * along a row are multiples of 8 elements. Outputs must not overlap inputs,
 * but where said. Sums, softmax statistics and angles are float32; an output
 * is rounded once, to the nearest value of its type, and so is what stands
 * between two products (the adapters' a x, the weights of attention), as said.
 *
 * A workspace belongs to the caller: 16-byte aligned device memory of at least
 * the bytes that the workspace function returns for the same sizes and hints.
 * Its content is not read between calls. Calls that may run at the same time
 * (other streams, captured graphs that are replayed side by side) need one each.
 */
#ifndef DINOV3_PACKED_H
#define DINOV3_PACKED_H
#include <stdint.h>
#include "dinov3_engine.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { DHX_F16 = 0, DHX_BF16 = 1 };

/* A projection that all sequences share, and beside it the low-rank adapter
 * of each sequence's own request:
 *   y[t] = w x[t] + bias + scale[a] b[a] (a[a] x[t]),  a = adapter[s]
 * for every row t of sequence s. An id outside 0 .. adapters-1 (-1, say) means
 * no adapter. The rank-sized product scale[a] a[a] x[t] is held in the type of
 * x between its two kernels (one rounding; a value past the type's range
 * becomes infinite there). An adapter has no effect on rows of others, whatever
 * it holds; a value of b that is not finite enters its own rows as its product
 * with theirs. Rows and adapters of any number, also a request per row. */
typedef struct dhx_packed_linear {
    uint32_t type; /* DHX_F16 or DHX_BF16: x, w, a, b, y */
    uint32_t sequences;
    uint64_t rows; /* of x and y */
    uint32_t inputs, outputs, rank, adapters;
    const void *x;        /* [rows][inputs] */
    const void *w;        /* [outputs][inputs] */
    const float *bias;    /* [outputs]; NULL: none */
    const void *a;        /* [adapters][rank][inputs] */
    const void *b;        /* [adapters][outputs][rank] */
    const float *scale;   /* [adapters] */
    void *y;              /* [rows][outputs] */
    uint64_t x_stride, w_stride, y_stride;
    const int32_t *starts;  /* [sequences + 1] */
    const int32_t *adapter; /* [sequences] */
    void *workspace;
    uint64_t workspace_bytes;
} dhx_packed_linear;

int dhx_packed_linear_workspace(const dhx_packed_linear *p, uint64_t *bytes);
int dhx_packed_linear_run(dhx_engine *e, const dhx_packed_linear *p, void *stream);

/* The position rotation of each row's heads, with the angles of the row's own
 * place: out = (x1 cos - x2 sin, x2 cos + x1 sin) for the pairs (x1, x2) of the
 * first `rotated` channels of every head, with cos and sin of row index[t] of
 * the tables. `rotated` is a multiple of 16, or a multiple of 8 that is head_dim
 * or half of it (40 of heads of 80). The pairs are the channels (j, j +
 * rotated/2) or, with `neighbours`, (2j, 2j + 1); angle j is column j of the
 * tables. Channels from
 * `rotated` on are copied, and so is a row whose index is outside 0 ..
 * places-1 (the CLS and register rows of an image, say). out may be x itself
 * with the same stride (in place), for the q and k heads at the front of packed
 * QKV rows, say. */
typedef struct dhx_packed_rotation {
    uint32_t type; /* DHX_F16 or DHX_BF16: x, out */
    uint32_t neighbours;
    uint64_t rows;
    uint32_t heads, head_dim, rotated, places;
    const void *x; /* [rows][heads][head_dim] */
    void *out;     /* [rows][heads][head_dim] */
    uint64_t x_stride, out_stride;
    const float *cos, *sin; /* [places][rotated / 2] */
    const int32_t *index;   /* [rows] */
} dhx_packed_rotation;

int dhx_packed_rotation_run(dhx_engine *e, const dhx_packed_rotation *p, void *stream);

/* Softmax attention inside each sequence:
 *   out[i, h] = sum_j softmax_j(scale q[i, h] . k[j, g]) v[j, g],
 * head h reading the key and value head g = h / (heads / kv_heads). Sequence s
 * has the queries of q_starts and the keys of k_starts, in any numbers. With
 * `causal`, query i of lq sees the keys j <= i + lk - lq (the last query sees
 * all of them, as for a prompt, its next part or one new token), else all. A
 * query that sees no key gets zeros, and -infinity in lse. Keys and values that
 * a query does not see have no effect on it, whatever they hold; a product q . k
 * that is infinity or not a number makes the query's outputs and lse not a number,
 * and a value that is not finite makes its channel not finite (an infinity or not
 * a number) for the queries that see it. A key whose product q . k lies below
 * -1e30 weighs nothing (its value should be finite); a query whose products all
 * do counts as one that sees no key.
 * The weights are rounded to the type of v for their product with it (f16 loses
 * those under 2^-25 of a row's largest); their sum keeps float32. Products, and
 * scale times them, are float32 too.
 * longest_q and longest_k, the rows of the longest sequence (0: not known),
 * only choose how the work is cut: a wrong number costs time, not results. */
typedef struct dhx_packed_attention {
    uint32_t type;   /* DHX_F16 or DHX_BF16: q, k, v, out */
    uint32_t causal; /* 0 or 1 */
    uint32_t sequences, heads, kv_heads, head_dim; /* head_dim: a multiple of 8, to 128 */
    uint64_t q_rows, k_rows; /* of q and out; of k and v */
    uint32_t longest_q, longest_k;
    float scale;             /* positive, at most 2^20 */
    uint32_t reserved;       /* 0 */
    const void *q;           /* row i, head h at q + i q_stride + h q_head_stride */
    const void *k, *v;
    void *out;
    uint64_t q_stride, k_stride, v_stride, out_stride;
    uint64_t q_head_stride, k_head_stride, v_head_stride, out_head_stride; /* 0: head_dim */
    float *lse;              /* [q_rows][heads]: log(sum_j exp(scale q . k)); NULL: not wanted */
    const int32_t *q_starts, *k_starts; /* [sequences + 1] */
    void *workspace;
    uint64_t workspace_bytes;
} dhx_packed_attention;

int dhx_packed_attention_workspace(const dhx_packed_attention *p, uint64_t *bytes);
int dhx_packed_attention_run(dhx_engine *e, const dhx_packed_attention *p, void *stream);

#ifdef __cplusplus
}
#endif
#endif
