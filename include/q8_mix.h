/* q8_mix.h: what stands between the Q8_0 products of a layer, on activations in HBM: the short
 * convolution and the gated delta rule of a DeltaNet layer (between the quartet QKV/GATE/BETA/ALPHA and
 * W_OUT, src/apl/qwen35.apl:92-98), and the head norms, the rotation, the paged key-value cache and the
 * attention over it of an attention layer (between Q/K/V and W_O, qwen35.apl:116-121).
 *
 * Additions, like every _dev entry point of q8_rt.h: device pointers, enqueued on the runtime's stream
 * in call order, no wait; each may be recorded into a graph (rt_graph_begin). Everything the host must
 * know lies in the structures; token counts, positions and pages are device data, so that a recorded
 * decode step goes on as the caller's arrays change. A violation that the host can see prints the
 * reason and aborts; what it cannot see (starts, positions, pages) never makes a kernel read or write
 * outside the arrays described here.
 *
 * Alignment: every float or cache address is 16-byte aligned and every stride a multiple of 4 floats,
 * except where said. Activations, norms, states and gates are F32. An array that a call writes must
 * not overlap one that it reads (from its first element to its last, whatever lies between its rows), but for
 * a state (s_out may be s_in) and a rotation in place.
 *
 * The workspace (the delta rule's for runs of tokens, the attention's) grows to what a call needs, or to twice what it
 * was, not while a graph is recorded: run a call with the same n, t and longest (and cache, heads, window and sinks) once before. All
 * of a runtime's calls share it, in the order of its stream; one that was replaced is freed by rt_fini. */
#ifndef Q8_MIX_H
#define Q8_MIX_H

#include "q8_rt.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The new tokens of a call, sequence by sequence: rows start[s] .. start[s + 1] - 1 of every
 * token-major array are sequence s's, in order. start ascends from 0 or more to t or less; a sequence
 * may have none. Rows that no sequence has are left as they were. */
#define RT_TOKENS_MAX ((1L << 23) - 1)
#define RT_HEADS_MAX 4096L
struct rt_seqs {
    long n;           /* sequences, 1 to 65535 */
    long t;           /* rows of the token-major arrays, 1 to RT_TOKENS_MAX */
    long longest;     /* the most tokens that one sequence has, 1 to t, as far as the caller knows: it
                       * chooses kernels and grids. Sequences with more are computed all the same, slower */
    const int *start; /* device [n + 1] */
    const int *past;  /* device [n]: sequence s's tokens are at positions past[s], past[s] + 1, ...
                       * (rt_rope_kv_dev, rt_kv_read_dev, rt_attn_kv_dev, rt_attn_window_dev; else unused) */
};

/* y[i] = SiLU(sum_j w[c][j] u[i - taps + 1 + j]) per channel c and token i of a sequence, u the
 * sequence's x behind the taps - 1 inputs that s_in[s] holds (oldest first); s_out[s] = its last
 * taps - 1 inputs, for the next call. x [t] rows x_ld floats apart, w [ch][taps], s_in and s_out
 * [n][taps - 1][ch], y [t] rows y_ld apart. taps 2 to 8; ch % 4 == 0. */
void rt_conv_silu_dev(struct rt *R, const struct rt_seqs *s, const float *x, long x_ld, long ch, const float *w, long taps, const float *s_in,
                      float *s_out, float *y, long y_ld);

/* The gated delta rule. Per token and value head h, on the state S [k_dim][v_dim] of the sequence's
 * head, with key head h / (v_heads / k_heads), or h % k_heads when tiled:
 *
 *   alpha = exp(decay[h] * softplus(a[h] + dt[h]))       beta = 1 / (1 + exp(-b[h]))
 *   S <- alpha S,  d = beta (v - S^T k),  S <- S + k d^T,  o = scale * S^T q
 *
 * q and k divided by sqrt(their sum of squares + eps) first when eps >= 0. With z, the output's
 * RMS norm over the head and its gate: o <- nw * o / sqrt(nw_eps + mean(o^2)) * SiLU(z).
 * Every sequence goes from s_in[s] to s_out[s], [n][v_heads][k_dim][v_dim] (one without tokens: a copy).
 * One token, or the few of a speculative check, run token by token; longer runs in chunks of tokens on
 * the matrix cores, in F32.
 * k_dim 32, 64, 96, 128, 192 or 256; v_dim a multiple of 16, 16 to 512; v_heads a multiple of k_heads;
 * n * v_heads * v_dim / 16 below 2^24. */
struct rt_delta {
    long k_heads, v_heads, k_dim, v_dim;
    long tiled;
    const float *q, *k, *v; /* [t] rows q_ld, k_ld, v_ld floats apart, heads side by side */
    long q_ld, k_ld, v_ld;
    const float *a, *b; /* [t] rows a_ld, b_ld floats apart (any alignment), v_heads each */
    long a_ld, b_ld;
    const float *decay, *dt; /* [v_heads] (any alignment); decay <= 0 in a model */
    float eps, scale;
    const float *s_in;
    float *s_out;
    const float *z; /* [t] rows z_ld apart, as o; NULL: no norm and gate */
    long z_ld;
    const float *nw; /* [v_dim], with z */
    float nw_eps;
    float *o; /* [t] rows o_ld apart, v_heads * v_dim each */
    long o_ld;
};
void rt_delta_rule_dev(struct rt *R, const struct rt_seqs *s, const struct rt_delta *a);

/* A paged key-value cache: k and v [pages][heads][page][dim]. Position p of sequence s lies in page
 * table[s * table_ld + p / page], row p % page.
 *
 * RT_Q8 holds a row (a position's head) as dim int8 values q and one F32 scale d, of which an element is q * d: k and v are the
 * values [pages][heads][page][dim] with the scales [pages][heads][page] right behind them (4-byte aligned, whatever page is). A scale
 * is 0 or more and finite; a row whose scale is NaN reads as NaN. Each row has a scale of its own, so that appending changes no row
 * that is there: a cache is the same however its tokens came, one by one or as a prompt, drafts taken back or not. */
#define RT_F32 0
#define RT_F16 1
#define RT_BF16 2
#define RT_Q8 8
struct rt_kv {
    void *k, *v;
    long type;        /* RT_F32, RT_F16, RT_BF16 or RT_Q8 */
    long dim;         /* a head's size: a multiple of 32, 32 to 256 */
    long heads;       /* key-value heads */
    long page, pages; /* positions a page (1 or more), pages in the cache: pages * heads * page < 2^31 */
    const int *table; /* device [n][table_ld]: entries that no position uses may be anything */
    long table_ld;    /* pages a sequence may have */
};
/* the bytes of such a cache's k, and of its v (the addresses are not looked at) */
long rt_kv_bytes(const struct rt_kv *kv);

/* Queries and keys to the cache and the attention: each head of q and k through its RMS norm (q_norm,
 * k_norm [dim]; NULL: none), then its first rot elements turned by the token's position p: pair i by
 * the angle p * freq[i], pair i being elements i and i + rot / 2, or 2 i and 2 i + 1 with pairs. q goes to
 * out in F32; k and v are rounded to the cache's type (to nearest, ties to even) into their position's row. In 8 bits
 * d = max|x| / 127 over the row and q = x / d rounded so; a row with an element that is not finite gets NaN for d, and so reads as
 * NaN, and one whose d would be below 2^-126 gets zeros.
 * A position before 0, behind the table's last page, or in a page that the cache does not have is not
 * stored. freq is F64, and so is the angle: positions in the millions turn exactly.
 * out may be q (the same strides). */
struct rt_rope {
    const float *q; /* [t] rows q_ld apart, head h at q_hd * h */
    long q_ld, q_hd, q_heads;
    const float *k, *v; /* the same, kv->heads each */
    long k_ld, k_hd, v_ld, v_hd;
    const float *q_norm, *k_norm;
    float eps;
    long rot;   /* even, 0 to dim */
    long pairs;
    const double *freq; /* device [rot / 2] (8-byte aligned): radians a position */
    float *out;
    long out_ld, out_hd;
};
void rt_rope_kv_dev(struct rt *R, const struct rt_seqs *s, const struct rt_kv *kv, const struct rt_rope *a);

/* Rows of the cache: K and V of the positions past[s], past[s] + 1, ... as rows start[s] .. of k and v (either may be NULL:
 * not read), head h at k_hd * h, from any type of cache to F32, F16 or BF16 (8-bit values q * d rounded to F32, then to the rows'
 * type). Strides in elements, multiples of 8 for 16-bit rows; k's rows, from the first to the last, lie apart from v's. A position before 0, behind the table's last page, or in a page that the
 * cache does not have reads as NaN. */
struct rt_kv_rows {
    long type; /* RT_F32, RT_F16 or RT_BF16 */
    void *k;
    long k_ld, k_hd;
    void *v;
    long v_ld, v_hd;
};
void rt_kv_read_dev(struct rt *R, const struct rt_seqs *s, const struct rt_kv *kv, const struct rt_kv_rows *a);

/* o = softmax(scale q K^T) V over the cache: the token at position p sees positions 0 .. p of its sequence
 * (its own and earlier new ones included: append them first), query head h the key-value head
 * h / (q_heads / heads). Times 1 / (1 + exp(-gate)), where given. For a few new tokens on a cache of any
 * length the positions are split over the GPU and joined; a prompt's tokens go 16 rows (token, head) at a time, 64 over
 * RT_Q8. There a query, times scale, is held in 24 bits of its row's largest element, and in steps of 1.2e-37 where that is below 1e-30; a
 * position whose weight is far below its row's largest, or whose value is near F32's smallest, may be off by 2^-118 (1 + |value|);
 * everything else is as exact as F32 sums.
 * A token that sees nothing (a position before 0) gives zeros; one that would have to see a position behind
 * the table's last page, or in a page that the cache does not have, gives NaN. */
struct rt_attn {
    const float *q; /* [t] rows q_ld apart, head h at q_hd * h */
    long q_ld, q_hd, q_heads;
    float scale;
    const float *gate; /* the same shape; NULL: none */
    long gate_ld, gate_hd;
    float *o; /* [t] rows o_ld apart, q_heads * dim each */
    long o_ld;
};
void rt_attn_kv_dev(struct rt *R, const struct rt_seqs *s, const struct rt_kv *kv, const struct rt_attn *a);

/* The same through a sliding window: the token at position p sees the positions j <= p with j > p - window, and those with
 * j < sinks, which stay visible. window 1 or more, sinks 0 or more; the time goes by what is seen. Pages of which no new token sees
 * anything may be gone: the table's entries for them may be anything, and so may what lies at positions that no new token sees.
 * (Over F16 and BF16 caches a prompt's rows that see infinities or NaN are computed apart, one by one, and slowly: 50 times where
 * all do.) */
void rt_attn_window_dev(struct rt *R, const struct rt_seqs *s, const struct rt_kv *kv, const struct rt_attn *a, long window, long sinks);

#ifdef __cplusplus
}
#endif

#endif
