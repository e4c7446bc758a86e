/*
 * fpa.h -- C ABI of the MI355X (gfx950) First Passage Attention library, libfpa.so.
 *
 * Plain C: device pointers, element strides and sizes; no torch or HIP types in
 * the signatures (the stream is passed as the opaque hipStream_t pointer value,
 * NULL = the default stream).  Every buffer is owned by the caller: the library
 * never allocates device memory.  Calls only enqueue work on `stream` and never
 * synchronise the host; they are re-entrant (no global mutable state besides the
 * thread-local error message).
 *
 * Reference interfaces replaced (yliu-fort/first-passage-attention, kernel.py):
 *   fpa_fwd  <- _forward (kernel.py:398-412) with _block_stats (387-395) and the
 *               _stats / _fwd Triton kernels (83-100, 103-162);
 *   fpa_bwd  <- _FirstPassageAttention.backward (kernel.py:424-451) with the
 *               _bwd_delta/_bwd_kv/_bwd_dphi_diag/_bwd_q/_bwd_dphi kernels
 *               (165-370) and the dbeta sum at kernel.py:450 (four kernels here:
 *               delta, key side, query side, phi/beta combine);
 *   fpa_state_floats / fpa_bwd_workspace_bytes <- the scratch allocations of
 *               kernel.py:390-392, 406-407, 430-436, sized so the caller owns them;
 *   fpa_fwd_workspace_bytes: no counterpart in the reference (the scratch of this
 *               forward's split row tiles, see FpaFwdArgs.workspace);
 *   fpa_field_fwd <- Field.forward (kernel.py:502-509): the fp32 projection of x
 *               to (delta, g, h), W = cumsum_t delta, phi = W + g, psi = W + h;
 *   fpa_field_bwd <- the autograd backward of those operations (dx, dW, dbias
 *               from dphi, dpsi), which the reference leaves to torch.
 * Error behaviour mirrors the validation of first_passage_attention
 * (kernel.py:467-486): invalid shapes or dtypes return FPA_ERR_INVALID with the
 * reference's message available from fpa_last_error().
 */
#ifndef FPA_H
#define FPA_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* dtype of q, k, v, o, do, dq, dk, dv */
#define FPA_F16 0
#define FPA_F32 1
/* of the pages of a cache only: 8-bit floating point (4 exponent and 3 mantissa bits, no infinities),
 * each row with a power of two of its own */
#define FPA_E4M3 2

/* phase bits (FpaFwdArgs.phases / FpaBwdArgs.phases) */
#define FPA_FWD_STATS 1    /* block statistics of phi                      */
#define FPA_FWD_MAIN 2     /* the forward kernel (o, lse)                  */
#define FPA_FWD_MERGE 4    /* o and lse of the split row tiles             */
#define FPA_BWD_DELTA 1    /* Delta_t = sum_d dO o                         */
#define FPA_BWD_KEYS 2     /* key side: dk, dv, dpsi, dbeta partials, ...  */
#define FPA_BWD_QUERIES 4  /* query side: dq, query-block soft-min sums;
                              KEYS | QUERIES runs both sides as one kernel */
#define FPA_BWD_PHI 8      /* dphi and dbeta (one kernel)                  */
#define FPA_BWD_BETA 16    /* same kernel as FPA_BWD_PHI                   */

/* status codes */
#define FPA_OK 0
#define FPA_ERR_INVALID 1     /* invalid argument (shape, dtype, tau, stride)        */
#define FPA_ERR_UNSUPPORTED 2 /* valid for the reference but not built (e.g. D > 256, T > 8388608) */
#define FPA_ERR_HIP 3         /* a HIP runtime call failed                            */

/* Forward arguments.  Tensors are (B, H, T, D) for q/k/v/o and (B, H, T) for
 * phi/psi, addressed with element strides s*[0..3] = (b, h, t, d); the d stride
 * must be 1.  phi, psi, beta are float32; beta is (H,) contiguous.  lse and
 * state are contiguous float32 buffers the forward fills and the backward reads:
 * lse holds 2*B*H*TP floats (TP = T rounded up to 64): for fp16 the base-2
 * log-sum-exp of each query row in the first B*H*TP; for fp32 the row's running
 * maximum there and log2 of its sum in the second half.  state holds
 * fpa_state_floats(B, H, T) floats (block statistics).  */
typedef struct {
    int64_t B, H, T, D;
    int32_t dtype;
    float tau;
    const void *q;  int64_t sq[4];
    const void *k;  int64_t sk[4];
    const void *v;  int64_t sv[4];
    const float *phi; int64_t sphi[3];
    const float *psi; int64_t spsi[3];
    const float *beta;
    void *o;        int64_t so[4];
    float *lse;
    float *state;
    int32_t phases;  /* 0: everything.  Otherwise a bitmask of the kernels to enqueue
                        (FPA_FWD_STATS | FPA_FWD_MAIN | FPA_FWD_MERGE), for per-kernel
                        timing only. */
    void *workspace; /* fpa_fwd_workspace_bytes(...) bytes of device memory, 256-byte
                        aligned, contents on entry irrelevant; or NULL.  When the launch
                        would be short of workgroups, the heaviest row tiles are split in
                        two halves of their key range that run side by side, and a merge
                        kernel combines them through this scratch; with NULL (or a shape
                        that needs none) every row tile runs whole.  Same results up to
                        rounding either way.  Needed only until the call's work ends.  */
} FpaFwdArgs;

/* Backward arguments: the forward's inputs, o, lse and state, the incoming
 * gradient do (strided like q), and the outputs.  dq, dk, dv have the dtype of
 * q and strides sdq/sdk/sdv; dphi, dpsi are float32 (B, H, T) contiguous; dbeta is
 * float32 (H,).  workspace is fpa_bwd_workspace_bytes(...) bytes of device memory,
 * 256-byte aligned; its contents on entry do not matter.                        */
typedef struct {
    int64_t B, H, T, D;
    int32_t dtype;
    float tau;
    const void *q;  int64_t sq[4];
    const void *k;  int64_t sk[4];
    const void *v;  int64_t sv[4];
    const float *beta;
    const void *o;  int64_t so[4];
    const void *dout; int64_t sdo[4];
    const float *lse;
    const float *state;
    void *dq;       int64_t sdq[4];
    void *dk;       int64_t sdk[4];
    void *dv;       int64_t sdv[4];
    float *dphi;
    float *dpsi;
    float *dbeta;
    void *workspace;
    int32_t phases;  /* 0: everything.  Otherwise a bitmask of FPA_BWD_* kernels to enqueue,
                        for per-kernel timing only: a partial run reads the workspace
                        left by an earlier full run and leaves skipped outputs unwritten. */
} FpaBwdArgs;

/* Field prologue of the layer (kernel.py:492-509).  x is (B, T, C) with a unit feature stride,
 * fp16 or fp32; the projection (3H outputs, H <= 32) is computed in fp32. */
typedef struct {
    int64_t B, T, C, H;
    int32_t dtype;          /* of x: FPA_F16 or FPA_F32 */
    const void *x;
    int64_t sx[2];          /* element strides of b and t */
    const float *weight;    /* (3H, C) row-major: Field.proj.weight */
    const float *bias;      /* (3H,): Field.proj.bias */
    float *phi;             /* (B, H, T) contiguous */
    float *psi;             /* (B, H, T) contiguous */
    void *workspace;        /* fpa_field_workspace_bytes(), 256-byte aligned */
} FpaFieldFwdArgs;

typedef struct {
    int64_t B, T, C, H;
    int32_t dtype;          /* of x and dx */
    const void *x;
    int64_t sx[2];
    const float *weight;    /* (3H, C) */
    const float *dphi;      /* (B, H, T) contiguous */
    const float *dpsi;      /* (B, H, T) contiguous */
    void *dx;               /* (B, T, C) like x, or NULL to skip it */
    int64_t sdx[2];
    float *dweight;         /* (3H, C) */
    float *dbias;           /* (3H,) */
    void *workspace;        /* fpa_field_workspace_bytes(), 256-byte aligned */
} FpaFieldBwdArgs;

/* Bytes of scratch of fpa_field_fwd and fpa_field_bwd (the larger of the two). */
int64_t fpa_field_workspace_bytes(int64_t B, int64_t T, int64_t C, int64_t H);

/* Enqueue the Field forward (phi, psi) on `stream`. */
int fpa_field_fwd(const FpaFieldFwdArgs *args, void *stream);

/* Enqueue the Field backward (dx, dweight, dbias) on `stream`.  Deterministic. */
int fpa_field_bwd(const FpaFieldBwdArgs *args, void *stream);

/* Floats of the forward state (block statistics) for a (B, H, T) problem. */
int64_t fpa_state_floats(int64_t B, int64_t H, int64_t T);

/* Floats of lse for a (B, H, T) problem (2 * B * H * TP). */
int64_t fpa_lse_floats(int64_t B, int64_t H, int64_t T);

/* Bytes of forward scratch for a (B, H, T, D) problem: 0 when its forward splits no
 * row tile (see FpaFwdArgs.workspace). */
int64_t fpa_fwd_workspace_bytes(int64_t B, int64_t H, int64_t T, int64_t D, int32_t dtype);

/* Bytes of backward scratch for a (B, H, T, D) problem. */
int64_t fpa_bwd_workspace_bytes(int64_t B, int64_t H, int64_t T, int64_t D, int32_t dtype);

/* Enqueue the forward on `stream` (a hipStream_t, NULL for the default stream). */
int fpa_fwd(const FpaFwdArgs *args, void *stream);

/* Enqueue the backward on `stream`. */
int fpa_bwd(const FpaBwdArgs *args, void *stream);

/* The backward without a caller workspace, for callers that cannot allocate device memory (code
 * under HIP graph capture, tight serving loops, harnesses that forbid hipMalloc).  No counterpart
 * in the reference.  Same arguments and results as fpa_bwd (args->workspace is ignored; should the
 * partial sums of a small launch's split tiles not fit, every tile runs whole, the same results to
 * rounding); the scratch is a static device array of FPA_NOALLOC_SCRATCH_BYTES per GPU, held until
 * the process ends.  Problems whose fpa_bwd_workspace_bytes exceed it return FPA_ERR_UNSUPPORTED before any
 * launch.  Calls that overlap on one GPU (two streams, two threads) share that array and race:
 * serialise them.  Allocates nothing (no hipMalloc or allocating library routine).            */
#define FPA_NOALLOC_SCRATCH_BYTES (64ll << 20)
int fpa_bwd_noalloc(const FpaBwdArgs *args, void *stream);

/* ---------------------------------------------------------------------------
 * Serving: a paged cache, attention of new tokens against it, drafted tokens.  No counterpart in the
 * reference, which has the training forward and backward only.
 *
 * A page holds 64 positions of every head.  Tables name a sequence's pages in order (int32; entries behind
 * its last page are not read); lengths, starts and counts are int32 in device memory.  Nothing is checked
 * that only the device knows: a page outside the pool is never touched (appends to it are dropped; what is read
 * from it, and every attention row that would need it, is NaN), and so is a position outside the table.
 * --------------------------------------------------------------------------- */

/* The pages, every buffer contiguous and 16-byte aligned. */
typedef struct {
    int64_t pages, H, D;
    int32_t store;      /* FPA_F16, FPA_F32 or FPA_E4M3 */
    void *k;            /* (pages, H, 64, D) */
    void *v;            /* (pages, H, D, 64): V of a page transposed */
    float *phi, *psi;   /* (pages, H, 64) */
    float *phi_min;     /* (pages, H): min of phi over the page's written positions */
    int8_t *k_exp;      /* (pages, H, 64), FPA_E4M3 only: a row of k or v is its codes times 2^exp */
    int8_t *v_exp;
} FpaPages;

/* Writes positions start[b] + i, i < counts[b] (at most N; N without counts) of B sequences.  k, v: (B, H, N, D)
 * with a unit d stride and 16-byte aligned rows, of the pages' type, or fp16 or fp32 for FPA_E4M3; phi, psi
 * (B, H, N).  Positions of one page must not be written by two sequences of a call.
 * e4m3: exp = clamp(ceil(log2(max |row| / 448)), -60, 60), -60 for a row of zeros; codes are rounded to nearest
 * even and saturate, NaN stays NaN.                                                              */
typedef struct {
    FpaPages cache;
    int64_t B, N, P;    /* table is (B, P) */
    int32_t dtype;      /* of k and v: FPA_F16 or FPA_F32 */
    const void *k;  int64_t sk[4];
    const void *v;  int64_t sv[4];
    const float *phi; int64_t sphi[3];
    const float *psi; int64_t spsi[3];
    const int32_t *table; int64_t stable;  /* row stride of table, in elements */
    const int32_t *start;
    const int32_t *counts;                 /* or NULL */
} FpaAppendArgs;
int fpa_cache_append(const FpaAppendArgs *args, void *stream);

/* Reads the same positions back into k, v (B, H, N, D) and phi, psi (B, H, N), contiguous; zero where
 * i >= counts[b].  dtype: the pages' type, or either for FPA_E4M3.                                */
typedef struct {
    FpaPages cache;
    int64_t B, N, P;
    int32_t dtype;
    void *k, *v;
    float *phi, *psi;
    const int32_t *table; int64_t stable;
    const int32_t *start;
    const int32_t *counts;
} FpaReadArgs;
int fpa_cache_read(const FpaReadArgs *args, void *stream);

/* First Passage Attention of the last N positions of B sequences, lengths[b] positions each (the N new ones
 * among them), against their pages: query i stands at position t = lengths[b] - N + i and attends to s <= t;
 * rows with t < 0 are zero.  With prefix_length > 0 every sequence continues one prefix of that many
 * positions on the pages prefix[0 .. ceil(prefix_length / 64)): rows attend to all of it too, and to phi across
 * the border; lengths and table still count the sequence's own positions alone.
 * q: (B, H, N, D), unit d stride, 16-byte aligned rows, fp16 or fp32 (the pages' type unless that is FPA_E4M3);
 * o: likewise, any alignment.                                                                      */
typedef struct {
    FpaPages cache;
    int64_t B, N, P;
    int32_t dtype;
    const void *q;  int64_t sq[4];
    void *o;        int64_t so[4];
    const float *beta;                     /* (H,) */
    const int32_t *table; int64_t stable;
    const int32_t *lengths;
    const int32_t *prefix;                 /* or NULL */
    int64_t prefix_length;
    void *workspace;                       /* fpa_attend_workspace_bytes(), 256-byte aligned */
    int32_t *counts;                       /* fpa_attend_counts() ints of device memory, zero before the first call; every call
                                              leaves them zero.  Calls that may overlap need counts of their own,
                                              as they need workspaces of their own. */
} FpaAttendArgs;
int64_t fpa_attend_workspace_bytes(int64_t B, int64_t H, int64_t N, int64_t D, int64_t P, int64_t prefix_length, int32_t dtype,
                                   int32_t store);
int64_t fpa_attend_counts(int64_t B, int64_t H, int64_t N);
int fpa_attend(const FpaAttendArgs *args, void *stream);

/* Verifies N drafted tokens of B sequences.  target: probabilities (B, N + 1, V), draft: (B, N, V) or NULL for
 * drafts that count as certain; unit stride over V.  Draft i is accepted while
 * accept_u[b, i] * draft[b, i, x_i] < target[b, i, x_i]; a token outside 0 .. V - 1 ends the drafts.  The next token is the
 * lowest v whose running sum of weights passes sample_u[b] times their sum, the weights being
 * max(target - draft, 0) of the rejected position's row, or the target's row where that is zero, where all
 * drafts are accepted and where they end (-1 if that row has no positive finite sum).  accepted: (B,); out: (B, N + 1),
 * the accepted drafts, the next token, then -1.                                                */
typedef struct {
    int64_t B, N, V;
    int32_t dtype;      /* of target and draft: FPA_F16 or FPA_F32 */
    const void *target; int64_t st[2];     /* strides of b and position */
    const void *draft;  int64_t sd[2];
    const int64_t *tokens; int64_t sx;     /* (B, N), row stride sx */
    const float *accept_u; int64_t su;     /* (B, N), row stride su, in [0, 1) */
    const float *sample_u;                 /* (B,), in [0, 1) */
    int64_t *accepted;
    int64_t *out;                          /* contiguous */
    void *workspace;                       /* fpa_verify_workspace_bytes(), 256-byte aligned */
    int32_t *counts;                       /* B ints, as FpaAttendArgs.counts */
} FpaVerifyArgs;
int64_t fpa_verify_workspace_bytes(int64_t B, int64_t V);
int fpa_verify(const FpaVerifyArgs *args, void *stream);

/* Message of the last failed call on this host thread ("" if none). */
const char *fpa_last_error(void);

/* ABI version (bumped whenever the structs above or the buffer sizes change). */
int fpa_abi_version(void);

/* Hash of the sources the library was built from (16 hex digits; "unknown" when the build did
 * not set it).  The Python loader compares it with the sources next to it and refuses a stale
 * library.  No counterpart in the reference, which compiles its kernels at first call.  */
const char *fpa_source_hash(void);

#ifdef __cplusplus
}
#endif

#endif /* FPA_H */
