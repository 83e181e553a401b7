/*
 * hgemm_sm100_train.h - C ABI of the training operators of the B200 (sm_100a)
 * HGEMM library (libhgemm_train_sm100.so): the gated feed-forward block and
 * its gradient, softmax cross entropy from hidden states and its gradient,
 * and the orthogonalised update of a weight matrix.
 *
 * The reference has no counterpart (its library is inference-only). The
 * conventions are those of hgemm_sm100.h: plain device pointers, sizes and a
 * stream, status codes (HGEMM_SM100_OK / _ERR_*), no exceptions, launches
 * asynchronous on the given stream on the current device, nothing allocated,
 * no state kept between calls, thread-safe. Workspaces are the caller's; any
 * contents do, two calls that may overlap need one each.
 *
 * Matrices are row-major with FP16 or BF16 elements (one type per call) and
 * FP32 accumulation. Bases of matrices must be 16-byte aligned (except where it
 * says otherwise), those of other arrays to their elements; leading dimensions, hidden
 * and inner sizes multiples of 8 elements (the Python layer pads other sizes).
 * Token counts, vocabularies and the sides of an orthogonalised matrix take
 * any value from 1 on.
 */
#ifndef HGEMM_SM100_TRAIN_H_
#define HGEMM_SM100_TRAIN_H_

#include <stddef.h>
#include <stdint.h>

#include "hgemm_sm100.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { HGEMM_SM100_TRAIN_F16 = 0, HGEMM_SM100_TRAIN_BF16 = 1 };

/* Common part of every call. `tile` forces the tile of all products: 0 = the
 * library chooses; else columns (a multiple of 64 up to 256), plus
 * HGEMM_SM100_TRAIN_TILE_PAIR for CTA pairs (256 rows instead of 128).
 * `splits` forces into how many parts the long sums (y, dx) are cut: 0 = the
 * library chooses, at most 16; for a small orthogonalised matrix the CTAs of
 * its cluster (1, 2, 4, 8 or 16). Workspace queries take both into account. */
#define HGEMM_SM100_TRAIN_TILE_PAIR 0x1000
typedef struct HgemmSm100TrainCommon {
    int32_t dtype;        /* HGEMM_SM100_TRAIN_F16 / _BF16                     */
    int32_t tile;         /* 0 = choose                                       */
    int32_t flags;        /* 0, or HGEMM_SM100_FLAG_TEST_INJECT_TX (tests)    */
    int32_t splits;       /* 0 = choose                                       */
    int32_t* status;      /* device int32 set when a kernel wait runs out; NULL
                             = the library's own word                         */
    uint64_t timeout_ns;  /* per-wait limit inside the kernels; 0 = 2 s       */
} HgemmSm100TrainCommon;

/* Gated feed-forward block, forward: h = silu(x Wg^T) * (x Wu^T), y = h Wd^T.
 * silu / slope (both or neither), for the gradient: silu(g) and u silu'(g) with
 * g = x Wg^T, u = x Wu^T, the factors that turn dh into du and dg. */
typedef struct HgemmSm100FfnForward {
    HgemmSm100TrainCommon common;
    const void* x;         /* [tokens x ldx]                                  */
    const void* gate;      /* Wg [inter x hidden]                             */
    const void* up;        /* Wu [inter x hidden]                             */
    const void* down;      /* Wd [out x inter]                                */
    void* y;               /* [tokens x out]                                  */
    void* h;               /* [tokens x inter]                                */
    void* silu;            /* [tokens x inter] or NULL                        */
    void* slope;          /* [tokens x inter] or NULL                        */
    void* workspace;       /* hgemm_sm100_ffn_forward_workspace bytes (may be 0) */
    uint64_t workspace_bytes;
    int64_t tokens, hidden, inter, out, ldx;
} HgemmSm100FfnForward;
size_t hgemm_sm100_ffn_forward_workspace(const HgemmSm100FfnForward* args);
int hgemm_sm100_ffn_forward(const HgemmSm100FfnForward* args, void* stream);

/* Its gradient. dh = dy Wd, du = dh silu, dg = dh slope (rounded to the
 * call's type, as operands of the products); dx = dg Wg + du Wu, dgate = dg^T x,
 * dup = du^T x, ddown = dy^T h. Outputs that are NULL are not computed. */
typedef struct HgemmSm100FfnBackward {
    HgemmSm100TrainCommon common;
    const void* dy;        /* [tokens x lddy]                                 */
    const void* x;         /* [tokens x ldx]                                  */
    const void* gate;
    const void* up;
    const void* down;
    const void* silu;      /* [tokens x inter], from the forward call         */
    const void* slope;
    const void* h;
    void* dgate_pre;       /* scratch [tokens x inter]: dg                    */
    void* dup_pre;         /* scratch [tokens x inter]: du                    */
    void* dx;              /* [tokens x hidden] or NULL                       */
    void* dgate;           /* [inter x hidden] or NULL                        */
    void* dup;             /* [inter x hidden] or NULL                        */
    void* ddown;           /* [out x inter] or NULL                           */
    void* workspace;       /* hgemm_sm100_ffn_backward_workspace bytes (may be 0) */
    uint64_t workspace_bytes;
    int64_t tokens, hidden, inter, out, ldx, lddy;
} HgemmSm100FfnBackward;
size_t hgemm_sm100_ffn_backward_workspace(const HgemmSm100FfnBackward* args);
int hgemm_sm100_ffn_backward(const HgemmSm100FfnBackward* args, void* stream);

/* Softmax cross entropy of logits z = x W^T that are never stored.
 * loss[t] = log(sum_v exp z[t, v]) - z[t, target[t]], 0 where target[t] is
 * `ignore_index`, NaN where it is outside the vocabulary otherwise. */
enum { HGEMM_SM100_LOSS_NONE = 0, HGEMM_SM100_LOSS_MEAN = 1, HGEMM_SM100_LOSS_SUM = 2 };
typedef struct HgemmSm100LossForward {
    HgemmSm100TrainCommon common;
    const void* x;         /* [tokens x ldx]                                  */
    const void* weight;    /* W [vocab x hidden]                              */
    const int64_t* target; /* [tokens]                                        */
    float* loss;           /* NONE: [tokens]; MEAN (over the tokens whose target
                              is not ignore_index; NaN without any), SUM: [1] */
    float* lse;            /* [tokens]: log(sum_v exp z), for the gradient    */
    void* workspace;       /* hgemm_sm100_loss_forward_workspace bytes        */
    uint64_t workspace_bytes;
    int64_t tokens, hidden, vocab, ldx, ignore_index;
    int32_t reduction;     /* HGEMM_SM100_LOSS_*                              */
    int32_t reserved;
} HgemmSm100LossForward;
size_t hgemm_sm100_loss_forward_workspace(const HgemmSm100LossForward* args);
int hgemm_sm100_loss_forward(const HgemmSm100LossForward* args, void* stream);

/* Its gradient for an incoming gradient dloss ([tokens] for NONE, else [1]):
 * dz = (softmax(z) - onehot(target)) * row factor, dx = dz W, dweight = dz^T x.
 * The vocabulary is taken in pieces; of dz only one piece exists at a time.
 * Rows whose target is `ignore_index` get zeros in dx and add nothing to
 * dweight, even where x or dloss hold infinity or NaN there. */
typedef struct HgemmSm100LossBackward {
    HgemmSm100TrainCommon common;
    const void* x;
    const void* weight;
    const int64_t* target;
    const float* lse;
    const float* dloss;
    void* dx;              /* [tokens x hidden] or NULL                       */
    void* dweight;         /* [vocab x hidden] or NULL                        */
    void* workspace;       /* hgemm_sm100_loss_backward_workspace bytes       */
    uint64_t workspace_bytes;
    int64_t tokens, hidden, vocab, ldx, ignore_index;
    int64_t piece;         /* vocabulary entries per piece; 0 = choose         */
    int32_t reduction;
    int32_t reserved;
} HgemmSm100LossBackward;
size_t hgemm_sm100_loss_backward_workspace(const HgemmSm100LossBackward* args);
int hgemm_sm100_loss_backward(const HgemmSm100LossBackward* args, void* stream);

/* X = g / (|g|_F + eps); `steps` times X <- a X + (b A + c A A) X with A = X X^T
 * (X^T X from the right where rows > cols); out = X. `batch` matrices, each
 * normalised by itself. Elements inside the steps are FP16 (scaled by a power
 * of two), sums FP32. */
typedef struct HgemmSm100Orthogonalize {
    HgemmSm100TrainCommon common;
    const void* g;         /* [batch][rows x ldg], batch_stride elements apart,
                              2-byte aligned, any ldg >= cols                 */
    void* out;             /* [batch][rows x cols], 2-byte aligned            */
    void* workspace;       /* hgemm_sm100_orthogonalize_workspace bytes (0 for
                              small matrices), 256-byte aligned               */
    uint64_t workspace_bytes;
    int64_t batch, rows, cols, ldg, batch_stride;
    int32_t steps;         /* >= 0                                            */
    int32_t reserved;
    float a, b, c;
    float reserved2;
    double eps;
} HgemmSm100Orthogonalize;
size_t hgemm_sm100_orthogonalize_workspace(const HgemmSm100Orthogonalize* args);
int hgemm_sm100_orthogonalize(const HgemmSm100Orthogonalize* args, void* stream);

/* Reads (and with clear != 0 resets) this library's own status word on the
 * current device. Synchronises the device; for tests and debugging. */
int hgemm_sm100_train_read_status(int32_t* value, int clear);

#ifdef __cplusplus
}
#endif

#endif /* HGEMM_SM100_TRAIN_H_ */
