/* libccsm_train: the operators of a training step as calls of their own, on device memory.
 *
 * What the reference leaves to torch.nn (PengNi/ccsmeth v0.5.0): nn.Embedding (models.py:35, 91), nn.Linear with an activation behind it
 * (utils/attention.py:34-36, 69; models.py:61, 147) and autograd's saved activations (train_multigpu.py:283-312).  Here each is a plain
 * function on row-major matrices, in fp32, fp16 or bf16, forward and backward:
 *
 *   ccsm_train_linear_forward      z = x w^T + bias;  y = act(z) + residual                    x (rows, inner), w (outer, inner), y (rows, outer)
 *   ccsm_train_linear_backward     d = dy act'(z);  dx = d w;  dw = d^T x;  dbias = column sums of d
 *   ccsm_train_embedding_forward   y[i] = scale table[ids[i]]
 *   ccsm_train_embedding_backward  dtable[v] = scale * sum over {i: ids[i] = v} of dy[i]
 *   ccsm_train_act8_pack / _unpack an activation kept in 8 bits; linear_backward takes x and z in that form too
 *
 * Conventions: every pointer is device memory of `device`; all matrices of a call share one type; `ld*` are row strides in elements (at
 * least the row's width); rows, columns and strides may be odd and bases need the alignment of one element only (rows of whole, aligned
 * 16-byte pieces are fastest).  At most 0x7fffff00 rows and 0x00ffff00 columns; a contraction along rows (linear_forward over `inner` with
 * more than 64 rows, dx over `outer`) has at most 8421504 columns in 16 bits and 4210752 in fp32; linear_backward takes up to 534773728
 * rows for each 256 columns of `outer`.  Work is enqueued on `stream` (NULL = the default stream) and never waits for the GPU, so every
 * call can be captured into a graph; nothing is kept from one call for the next.  `workspace` is scratch of at least *_workspace() bytes,
 * 256-byte aligned, used until the enqueued work is done: calls that may run at the same time, two captured graphs among them, need one
 * each. The current device is the caller's again when a call returns.  Sums, activations and their slopes are computed in 32 bits or more
 * and rounded once, with one exception: linear_backward in 16 bits takes d = dy act'(z) rounded to its type into dx and dw (not into dbias)
 * where an activation meets products in tiles (ccsm_train_linear_backward_way), so that those gradients carry two roundings, sqrt 2 times
 * the error of one.  fp16's d is brought into the type's range by a power of two first (a d below 2^-28 of dy's largest finite magnitude A
 * is off by up to 2^-39 A).  Smaller products keep d to 2^-16.  fp32 products are made of bf16 pieces; what is left out is below 2^-22 of
 * each product, 2^-25 in the mean.  Infinities and NaN of operands give what they give in the formulas above.  Results do not depend on
 * timing (no floating-point atomics).  Outputs share no memory with inputs or each other, except y the residual (same base and stride);
 * columns of the same rows are apart, other views whose ranges of memory meet count as shared.  Zero rows (or tokens) are allowed:
 * gradients of weights are then zero.  Refusals: CCSM_ERR_INVALID_ARG (text in ccsm_train_ops_last_error), CCSM_ERR_CAPACITY for a
 * workspace that is too small.
 */
#ifndef CCSM_TRAIN_OPS_H_
#define CCSM_TRAIN_OPS_H_

#include "ccsm.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum { CCSM_TYPE_F32 = 0, CCSM_TYPE_F16 = 1, CCSM_TYPE_BF16 = 2 } ccsm_type;
typedef enum { CCSM_ID_U8 = 0, CCSM_ID_I32 = 1, CCSM_ID_I64 = 2 } ccsm_id_type;
/* gelu = z (1 + erf(z / sqrt 2)) / 2; silu = z / (1 + e^-z); relu's slope at 0 is 0 */
typedef enum { CCSM_ACT_NONE = 0, CCSM_ACT_RELU = 1, CCSM_ACT_TANH = 2, CCSM_ACT_SIGMOID = 3, CCSM_ACT_GELU = 4, CCSM_ACT_SILU = 5 } ccsm_activation;
/* An activation in 8 bits: each block of 32 consecutive values of a row is divided by 2^e, the least power of two (e >= -126) that brings its
 * largest finite magnitude to at most 127 (INT8) or 448 (E4M3), and rounded to the nearest code, ties to even.  The block's scale byte is
 * e + 127.  A code stands for exactly code * 2^e, a value of the type that was packed (where rounding up would leave that type's range, the
 * code below it is taken).  Infinities and NaN are held as NaN (INT8 code -128, E4M3 0x7f) and do not enter e. */
typedef enum { CCSM_CODE_NONE = 0, CCSM_CODE_INT8 = 1, CCSM_CODE_E4M3 = 2 } ccsm_code8;

/* A matrix that a forward pass has kept: code NONE: `data` in the call's type, `ld` its row stride.  Otherwise `data` = codes (bytes; ld a
 * multiple of 32, at least the width rounded up to 32) and `scales` = scale bytes (lds at least width / 32 rounded up), both 16-byte aligned. */
typedef struct {
    const void* data;
    int64_t ld;
    int32_t code;
    const uint8_t* scales;
    int64_t lds;
} ccsm_saved;

typedef struct {
    int32_t type, activation;
    int64_t rows;
    int32_t inner, outer;
    const void* x; int64_t ldx;
    const void* w; int64_t ldw;
    const void* bias;                   /* (outer) or NULL */
    const void* residual; int64_t ldr;  /* (rows, outer) or NULL */
    void* y; int64_t ldy;
    void* preact; int64_t ldp;          /* (rows, outer): z, for the backward pass; or NULL */
} ccsm_linear;

typedef struct {
    int32_t type, activation;
    int64_t rows;
    int32_t inner, outer;
    const void* dy; int64_t lddy;
    ccsm_saved x;                       /* read for dw */
    const void* w; int64_t ldw;         /* read for dx */
    ccsm_saved preact;                  /* read unless the activation is NONE */
    void* dx; int64_t lddx;             /* each of the three outputs may be NULL: it is not computed */
    void* dw; int64_t lddw;
    void* dbias;
} ccsm_linear_grad;

const char* ccsm_train_ops_last_error(void);

/* *_workspace: the bytes of scratch that the call needs (0: none, workspace may be NULL).  It depends on sizes, types and strides, and on
 * pointers only through their alignment. */
size_t ccsm_train_linear_workspace(const ccsm_linear* p);
ccsm_status ccsm_train_linear_forward(int device, const ccsm_linear* p, void* workspace, size_t workspace_bytes, void* stream);

size_t ccsm_train_linear_backward_workspace(const ccsm_linear_grad* p);
ccsm_status ccsm_train_linear_backward(int device, const ccsm_linear_grad* p, void* workspace, size_t workspace_bytes, void* stream);

/* Which kernels such a call takes, for tests and profiles; nothing is launched.  way[0]: the edge of the products' tiles (256 or 128; 0: the kernel for
 * small products and few rows, or none); way[1], way[2]: into how many parts the contraction is split (forward: way[1]; backward: of dx, of dw;
 * 0: no tiles); way[3]: operands staged in front. */
ccsm_status ccsm_train_linear_way(const ccsm_linear* p, int32_t* way);
ccsm_status ccsm_train_linear_backward_way(const ccsm_linear_grad* p, int32_t* way);

/* ids outside [0, rows) are no tokens (padding): their row of y is zero and they have no gradient.  y (tokens, width) = scale table[ids]. */
ccsm_status ccsm_train_embedding_forward(int device, int type, int id_type, int64_t tokens, const void* ids, int64_t rows, int32_t width,
                                         const void* table, int64_t ldt, float scale, void* y, int64_t ldy, void* stream);
/* dtable (rows, width) is written whole.  A row's sum has one order, which depends on the sizes and the ids alone (tokens are sorted by id on the
 * GPU, stably; tables of few rows are added up without). */
size_t ccsm_train_embedding_backward_workspace(int type, int64_t tokens, int64_t rows, int32_t width);
ccsm_status ccsm_train_embedding_backward(int device, int type, int id_type, int64_t tokens, const void* ids, int64_t rows, int32_t width,
                                          const void* dy, int64_t lddy, float scale, void* dtable, int64_t ldt, void* workspace,
                                          size_t workspace_bytes, void* stream);

/* x (rows, width) -> codes (rows, ldc bytes), scales (rows, lds bytes): layout as in ccsm_saved; the codes between width and its next
 * multiple of 32 are written as 0. */
ccsm_status ccsm_train_act8_pack(int device, int type, int code, int64_t rows, int32_t width, const void* x, int64_t ldx, void* codes,
                                 int64_t ldc, uint8_t* scales, int64_t lds, void* stream);
/* The values that the codes stand for, rounded to `type`. */
ccsm_status ccsm_train_act8_unpack(int device, int type, int64_t rows, int32_t width, const ccsm_saved* s, void* y, int64_t ldy, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* CCSM_TRAIN_OPS_H_ */
