/* C-ABI of the answering end: what turns a model's last hidden states into
 * the next token ids, on one MI355X (gfx950). Library: libtoktier_head.so.
 *
 * - tk_head_norm: root-mean-square norm of x + residual with an 8-bit output;
 * - tk_head_matmul: 8-bit product with a scale for each block of 128;
 * - tk_head_sample: one token a row by temperature, top-k, top-p and min-p.
 *
 * Every pointer is a device pointer on `device`; `stream` is a hipStream_t
 * (NULL: the default stream). Calls only queue kernels: they never
 * synchronize, allocate or copy, so they can be recorded into a HIP graph.
 * Strides are in elements of the row they step over (bytes for 8-bit values
 * and scales, words for masks), and an input of one row may have any; the
 * last axis is dense. Calls return TK_OK or one of the TK_E_* codes of
 * toktier_hip.h (the values are repeated below), with a message in
 * tk_head_last_error() (per thread).
 *
 * 8-bit values are OCP e4m3 ("float8_e4m3fn"). A scale is one byte, e8m0: it
 * stands for 2^(byte - 127), and 255 for NaN. Row r of k values has
 * ceil(k / 128) scales, the last for the block that k ends in.
 */
#ifndef TOKTIER_HEAD_H
#define TOKTIER_HEAD_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* what tk_head_abi_version returns; another with any change of a struct */
#define TKH_ABI_VERSION 1
#define TKH_OK 0
#define TKH_E_INVALID_ARG (-1)
#define TKH_E_SHAPE (-2)
#define TKH_E_DEVICE (-3)
#define TKH_E_ARCH (-4)
#define TKH_E_CAPACITY (-7)
#define TKH_E_UNSUPPORTED (-9)

#define TKH_F32 0
#define TKH_BF16 1
#define TKH_F16 2

/* widest row of tk_head_norm */
#define TKH_NORM_MAX_K 65536
/* widest row of tk_head_sample: its masses, 2^40 at most, sum below 2^64 */
#define TKH_SAMPLE_MAX_VOCAB 16777215

/* Sizes whose kernels would pass a launch's 2^32 - 1 threads are refused with
 * TKH_E_SHAPE: 2^26 rows for a norm of up to 512 values, fewer for wider ones
 * (2^22 for the widest); n over 2^30 - 64, or c of over 2^23 pieces of 128 x
 * 128; 2^22 rows to sample from, fewer of long ones (2^12 of the widest). */

/* y = (x + residual) * rsqrt(mean((x + residual)^2) + eps) * weight in
 * 32 bits (of h scaled by a power of two where its squares are beyond them:
 * a finite row has a finite norm), then for each block of 128 the least power of two s with
 * amax <= 448 s (1 for a block of zeros), q = e4m3(y / s). Values that are
 * not finite become NaN and do not count for amax. residual_out (optional;
 * may be residual itself) receives x + residual in x's type. The pad of a
 * q row, up to a multiple of 128, is written as zeros. */
typedef struct tkh_norm {
    const void* x;          /* [rows, k] of dtype */
    const void* residual;   /* [rows, k] of dtype, or NULL */
    const void* weight;     /* [k] of weight_dtype */
    void* q;                /* [rows, q_stride], 16-byte aligned */
    void* scale;            /* [rows, ceil(k / 128)] */
    void* residual_out;     /* [rows, k] of dtype, or NULL */
    int64_t rows, k;
    int64_t x_stride, residual_stride, q_stride, scale_stride, out_stride;
    float eps;
    int32_t dtype;          /* TKH_* */
    int32_t weight_dtype;   /* dtype or TKH_F32 */
    int32_t device;
} tkh_norm;

/* c[i, j] = sum over blocks b of 2^(ea[i,b] + ew[j,b]) * sum over k in b of
 * a[i,k] w[j,k], summed in the matrix unit and rounded once to out_dtype
 * (TKH_BF16 or TKH_F16). The unit adds the products of 8 neighbours along k
 * to each other, each cut to a multiple of 2^-13 of the power of two that the
 * exponents of the largest one's factors make, and these sums in 32 bits. A
 * sum is thus off by less than 7 * 2^-13 of the largest product of each 8,
 * added up: where products of very unequal size stand side by side, by up to
 * 2^-10 of the sum of |a w|, and where the large ones cancel, by all that is
 * left. On normally distributed rows of 4096 it is 2^-21 of that sum (root
 * mean square), 2^-17.7 at most with a channel in 97 twelve times as large.
 * Rows of a and w are 16-byte aligned (base,
 * and stride where there are several) and read in whole 16-byte pieces; what
 * lies beyond k does not count. */
typedef struct tkh_matmul {
    const void* a;          /* [m, k] e4m3 */
    const void* a_scale;    /* [m, ceil(k / 128)] e8m0 */
    const void* w;          /* [n, k] e4m3 */
    const void* w_scale;    /* [n, ceil(k / 128)] e8m0 */
    void* c;                /* [m, n] of out_dtype */
    int64_t m, n, k;
    int64_t a_stride, a_scale_stride, w_stride, w_scale_stride, c_stride;
    int32_t out_dtype;      /* TKH_BF16 or TKH_F16 */
    int32_t device;
} tkh_matmul;

/* One token a row. With x the row's logits in 32 bits (NaN, -inf and tokens
 * whose `allowed` bit is 0 left out), m their largest and s = log2(e) / T in
 * 32 bits, token i has the mass q_i = floor(2^40 * 2^((x_i - m) * s)), a
 * whole number, so that no sum depends on its order. In the order of falling
 * x, equal ones by rising index: the first top_k tokens stay (0: all), of
 * these each with less than ceil(top_p * (their mass)) before it (top_p >= 1:
 * all; the first always), and of these those of at least min_p times the
 * largest's weight. With K the mass that stays, the token is the first by
 * index at which the running mass passes floor(u * K), u in [0, 1).
 * T <= 0 (or NaN) takes the largest logit, the lowest index of equal ones.
 * logprob is ln(q_id / K). A row that leaves nothing out of which to draw
 * gets id -1 and logprob -inf. Each parameter is a device array of one value
 * a row, or NULL and the value beside it for every row. */
typedef struct tkh_sample {
    const void* logits;         /* [rows, vocab] of dtype */
    const float* u;             /* [rows] */
    const float* temperature;   /* [rows] or NULL */
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const uint32_t* allowed;    /* [rows, ceil(vocab / 32)] bits, or NULL */
    int32_t* ids;               /* [rows] */
    float* logprob;             /* [rows] or NULL */
    void* workspace;            /* tk_head_sample_workspace bytes */
    uint64_t workspace_size;
    int64_t rows, vocab;
    int64_t logits_stride, allowed_stride;  /* allowed_stride 0: one mask */
    float temperature_value;
    int32_t top_k_value;
    float top_p_value;
    float min_p_value;
    int32_t dtype;              /* TKH_* */
    int32_t device;
} tkh_sample;

int tk_head_norm(const tkh_norm* args, void* stream);
int tk_head_matmul(const tkh_matmul* args, void* stream);
int tk_head_sample(const tkh_sample* args, void* stream);

/* Bytes of workspace tk_head_sample needs for these sizes (0 if none);
 * 16-byte aligned; its contents need not be kept between calls. */
uint64_t tk_head_sample_workspace(int64_t rows, int64_t vocab, int32_t dtype);

const char* tk_head_last_error(void);

/* TKH_ABI_VERSION of the library, and the digest of the sources and flags
 * that it was built from. */
int tk_head_abi_version(void);
const char* tk_head_sources(void);

#ifdef __cplusplus
}
#endif
#endif
