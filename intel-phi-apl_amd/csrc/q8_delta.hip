/* q8_delta.hip: the gated delta rule (include/q8_mix.h), and the norm and gate of its output. */
#include "q8_mix.h"

namespace {

/* The two gates of a token's head. softplus as max(x, 0) + log1p(exp(-|x|)): no overflow. */
__device__ __forceinline__ float decay_of(float a, float dt, float rate)
{
    const float x = a + dt;
    return expf(rate * (fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x)))));
}

/* Token by token. A wave owns 16 columns of a head's state: lane 16 c + g holds rows g*KR .. g*KR + KR - 1
 * of columns 4 c .. 4 c + 3, so a column's dot products go over a row of 16 lanes. Both products with
 * the state are taken before it changes, in one reduction:
 *
 *   S' = alpha S + k d^T,  d = beta (v - alpha S^T k),  S'^T q = alpha S^T q + (q.k) d
 *
 * and so are |q|^2, |k|^2 and q.k, whose scales are applied to the results. Bound by HBM (the state, read
 * and written once) on many sequences, by latency on one. */
template <int KR>
__global__ __launch_bounds__(64) void delta_step_k(rt_seqs b, rt_delta a)
{
    const int lane = threadIdx.x, g = lane & 15, c = 4 * (lane >> 4);
    const long s = blockIdx.z, h = blockIdx.y, col = 16 * (long)blockIdx.x + c;
    const long kh = a.tiled ? h % a.k_heads : h / (a.v_heads / a.k_heads);
    long first, last;
    q8_rows_of(b, s, first, last);
    const long base = ((s * a.v_heads + h) * a.k_dim + g * KR) * a.v_dim + col;
    float4 st[KR];
#pragma unroll
    for (int r = 0; r < KR; r++)
        st[r] = *(const float4 *)(a.s_in + base + r * a.v_dim);
    const float rate = a.decay[h], dt = a.dt[h];
    for (long i = first; i < last; i++) {
        float q[KR], k[KR];
#pragma unroll
        for (int r = 0; r < KR; r += 2) {
            *(float2 *)(q + r) = *(const float2 *)(a.q + i * a.q_ld + kh * a.k_dim + g * KR + r);
            *(float2 *)(k + r) = *(const float2 *)(a.k + i * a.k_ld + kh * a.k_dim + g * KR + r);
        }
        const float4 v = *(const float4 *)(a.v + i * a.v_ld + h * a.v_dim + col);
        const float alpha = decay_of(a.a[i * a.a_ld + h], dt, rate), beta = q8_sigmoid(a.b[i * a.b_ld + h]);
        float qq = 0.0f, kk = 0.0f, qk = 0.0f;
        float4 sq = {0.0f, 0.0f, 0.0f, 0.0f}, sk = sq;
#pragma unroll
        for (int r = 0; r < KR; r++) {
            qq = fmaf(q[r], q[r], qq);
            kk = fmaf(k[r], k[r], kk);
            qk = fmaf(q[r], k[r], qk);
            sq = float4{fmaf(st[r].x, q[r], sq.x), fmaf(st[r].y, q[r], sq.y), fmaf(st[r].z, q[r], sq.z), fmaf(st[r].w, q[r], sq.w)};
            sk = float4{fmaf(st[r].x, k[r], sk.x), fmaf(st[r].y, k[r], sk.y), fmaf(st[r].z, k[r], sk.z), fmaf(st[r].w, k[r], sk.w)};
        }
        qk = q8_row_sum(qk);
        sq = float4{q8_row_sum(sq.x), q8_row_sum(sq.y), q8_row_sum(sq.z), q8_row_sum(sq.w)};
        sk = float4{q8_row_sum(sk.x), q8_row_sum(sk.y), q8_row_sum(sk.z), q8_row_sum(sk.w)};
        float rq = 1.0f, rk = 1.0f;
        if (a.eps >= 0.0f) {
            rq = 1.0f / sqrtf(q8_row_sum(qq) + a.eps);
            rk = 1.0f / sqrtf(q8_row_sum(kk) + a.eps);
        }
        const float ak = alpha * rk;
        const float4 d = {beta * (v.x - ak * sk.x), beta * (v.y - ak * sk.y), beta * (v.z - ak * sk.z), beta * (v.w - ak * sk.w)};
        const float oq = a.scale * rq, od = oq * (rk * qk), oa = oq * alpha;
        if (g == 0)
            *(float4 *)(a.o + i * a.o_ld + h * a.v_dim + col) =
                float4{fmaf(oa, sq.x, od * d.x), fmaf(oa, sq.y, od * d.y), fmaf(oa, sq.z, od * d.z), fmaf(oa, sq.w, od * d.w)};
#pragma unroll
        for (int r = 0; r < KR; r++) {
            const float kr = rk * k[r];
            st[r] = float4{fmaf(kr, d.x, alpha * st[r].x), fmaf(kr, d.y, alpha * st[r].y), fmaf(kr, d.z, alpha * st[r].z), fmaf(kr, d.w, alpha * st[r].w)};
        }
    }
#pragma unroll
    for (int r = 0; r < KR; r++)
        *(float4 *)(a.s_out + base + r * a.v_dim) = st[r];
}

/* o <- nw * o / sqrt(eps + mean(o^2)) * SiLU(z), a wave a head of a token */
__global__ __launch_bounds__(256) void gated_norm_k(rt_seqs b, rt_delta a)
{
    const long i = blockIdx.x, h = 4 * (long)blockIdx.y + (threadIdx.x >> 6);
    if (q8_sequence_of(b, i) < 0 || h >= a.v_heads)
        return;
    const int lane = threadIdx.x & 63;
    float *o = a.o + i * a.o_ld + h * a.v_dim;
    const float *z = a.z + i * a.z_ld + h * a.v_dim;
    float sum = 0.0f;
    for (long c = lane; c < a.v_dim; c += 64)
        sum = fmaf(o[c], o[c], sum);
    const float r = 1.0f / sqrtf(a.nw_eps + q8_wave_sum(sum) / (float)a.v_dim);
    for (long c = lane; c < a.v_dim; c += 64)
        o[c] = a.nw[c] * (o[c] * r) * (z[c] * q8_sigmoid(z[c]));
}

} /* namespace */

void q8_launch_delta(q8_stream_t s, const rt_seqs &b, const rt_delta &a)
{
    const dim3 grid((unsigned)(a.v_dim / 16), (unsigned)a.v_heads, (unsigned)b.n);
    switch (a.k_dim) {
#define STEP(K)                                                                                                                                            \
    case K:                                                                                                                                                \
        delta_step_k<K / 16><<<grid, 64, 0, (hipStream_t)s>>>(b, a);                                                                                       \
        break;
        STEP(32)
        STEP(64)
        STEP(96)
        STEP(128)
        STEP(192)
        STEP(256)
#undef STEP
    }
    if (a.z)
        gated_norm_k<<<dim3((unsigned)b.t, (unsigned)((a.v_heads + 3) / 4)), 256, 0, (hipStream_t)s>>>(b, a);
}
