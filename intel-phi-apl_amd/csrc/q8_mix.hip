/* q8_mix.hip: the small operators of include/q8_mix.h, one pass over their data each: the short
 * convolution with SiLU, and the head norms with the rotation and the way into the paged cache. */
#include "q8_mix.h"

namespace {

/* ---- the short convolution
 *
 * A thread owns 4 neighbouring channels of one sequence and CONV_RUN tokens: it holds the run's rows and
 * the TAPS - 1 before them in registers, all loaded before any arithmetic, so each x is read from HBM once
 * (the rows at a run's start once more, from L2) and a workgroup's loads are whole lines. The first run of a
 * sequence takes those rows from the state and is also the one that writes the new state, after it has
 * read the old one, so that the state may be updated in place: no other thread touches its channels. */
constexpr int CONV_RUN = 8;
static_assert(CONV_RUN >= 7, "only a sequence's first run reads the state: taps - 1 <= CONV_RUN");

template <int TAPS>
__global__ __launch_bounds__(256) void conv_k(rt_seqs b, const float *__restrict__ x, long x_ld, long ch, const float *__restrict__ w, const float *s_in,
                                              float *s_out, float *__restrict__ y, long y_ld)
{
    const long c = 4 * ((long)blockIdx.x * 256 + threadIdx.x), s = blockIdx.y;
    if (c >= ch)
        return;
    long first, last;
    q8_rows_of(b, s, first, last);
    const long n = last - first;
    float wt[4 * TAPS];
#pragma unroll
    for (int i = 0; i < TAPS; i++)
        *(float4 *)(wt + 4 * i) = *(const float4 *)(w + c * TAPS + 4 * i);
    for (long r = blockIdx.z; r == 0 || r * CONV_RUN < n; r += gridDim.z) {
        const long i0 = r * CONV_RUN;
        float4 u[CONV_RUN + TAPS - 1];
#pragma unroll
        for (int j = 0; j < CONV_RUN + TAPS - 1; j++) {
            const long i = i0 + j - (TAPS - 1); /* this input's place in the sequence; before it, the state's */
            u[j] = float4{0.0f, 0.0f, 0.0f, 0.0f};
            if (i < 0)
                u[j] = *(const float4 *)(s_in + (s * (TAPS - 1) + i + TAPS - 1) * ch + c);
            else if (i < n)
                u[j] = *(const float4 *)(x + (first + i) * x_ld + c);
        }
        if (r == 0) {
            float4 keep[TAPS - 1];
#pragma unroll
            for (int j = 0; j < TAPS - 1; j++) {
                const long i = n - (TAPS - 1) + j;
                keep[j] = i < 0 ? *(const float4 *)(s_in + (s * (TAPS - 1) + i + TAPS - 1) * ch + c) : *(const float4 *)(x + (first + i) * x_ld + c);
            }
#pragma unroll
            for (int j = 0; j < TAPS - 1; j++)
                *(float4 *)(s_out + (s * (TAPS - 1) + j) * ch + c) = keep[j];
        }
#pragma unroll
        for (int j = 0; j < CONV_RUN; j++) {
            if (i0 + j >= n)
                break;
            float4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < TAPS; k++) {
                v.x = fmaf(wt[k], u[j + k].x, v.x);
                v.y = fmaf(wt[TAPS + k], u[j + k].y, v.y);
                v.z = fmaf(wt[2 * TAPS + k], u[j + k].z, v.z);
                v.w = fmaf(wt[3 * TAPS + k], u[j + k].w, v.w);
            }
            v = float4{v.x * q8_sigmoid(v.x), v.y * q8_sigmoid(v.y), v.z * q8_sigmoid(v.z), v.w * q8_sigmoid(v.w)};
            *(float4 *)(y + (first + i0 + j) * y_ld + c) = v;
        }
    }
}

/* ---- the rotation
 *
 * The angle a = p * freq and its rest after whole quarter turns are F64 (the quarter turn as two F64
 * parts), so that far positions lose nothing; the sine and cosine of the rest, at most pi/4, are Taylor
 * polynomials in F32 (next terms r^11 / 11! and r^12 / 12!: below 2e-9 and 2e-10). */
__device__ __forceinline__ void turn(long p, double freq, float &co, float &si)
{
    const double a = (double)p * freq, q = rint(a * 0.63661977236758134308);
    const double rest = fma(-q, 6.123233995736766036e-17, fma(-q, 1.5707963267948966192, a));
    const float r = (float)rest, z = r * r;
    const float s = fmaf(r * z, fmaf(z, fmaf(z, fmaf(z, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), r);
    const float c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
    const int k = (int)(q - 4.0 * floor(0.25 * q)); /* the quarter, 0 to 3 */
    co = (k & 1) ? s : c;
    si = (k & 1) ? c : s;
    co = (k == 1 || k == 2) ? -co : co;
    si = (k >= 2) ? -si : si;
}

template <int TYPE>
__device__ __forceinline__ void store4(void *cache, long at, float4 v)
{
    if constexpr (TYPE == RT_F32) {
        *(float4 *)((float *)cache + at) = v;
    } else if constexpr (TYPE == RT_F16) {
        typedef _Float16 h4 __attribute__((ext_vector_type(4)));
        *(h4 *)((_Float16 *)cache + at) = h4{(_Float16)v.x, (_Float16)v.y, (_Float16)v.z, (_Float16)v.w};
    } else {
        typedef __bf16 b4 __attribute__((ext_vector_type(4)));
        *(b4 *)((__bf16 *)cache + at) = b4{(__bf16)v.x, (__bf16)v.y, (__bf16)v.z, (__bf16)v.w};
    }
}

/* Query, key and value heads of a token alike: LANES lanes (a power of two, 8 to 64) hold a head, 4
 * elements a lane; the norm's sum goes over them, and halves that turn together trade places through
 * LDS. Bound by latency on a few tokens, by HBM on a prompt. */
constexpr int ROPE_WAVES = 4;

template <int TYPE>
__global__ __launch_bounds__(64 * ROPE_WAVES) void rope_k(rt_seqs b, rt_kv kv, rt_rope a, int lanes)
{
    __shared__ __align__(16) float row[64 * ROPE_WAVES * 4];
    const long i = blockIdx.x, s = q8_sequence_of(b, i);
    if (s < 0)
        return;
    const int at = 4 * ((int)threadIdx.x & (lanes - 1));
    const long h = ((long)blockIdx.y * 64 * ROPE_WAVES + threadIdx.x) / lanes, nq = a.q_heads, nk = kv.heads;
    const int kind = h < nq ? 0 : h < nq + nk ? 1 : h < nq + 2 * nk ? 2 : 3;
    const long hh = kind == 0 ? h : kind == 1 ? h - nq : h - nq - nk;
    const bool live = kind < 3 && at < kv.dim;
    const long p = (long)b.past[s] + (i - b.start[s]);
    const float *src = kind == 0 ? a.q + i * a.q_ld + hh * a.q_hd : kind == 1 ? a.k + i * a.k_ld + hh * a.k_hd : a.v + i * a.v_ld + hh * a.v_hd;
    const float *nw = kind == 0 ? a.q_norm : a.k_norm;
    float4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (live)
        v = *(const float4 *)(src + at);
    float sum = fmaf(v.w, v.w, fmaf(v.z, v.z, fmaf(v.y, v.y, v.x * v.x)));
    for (int o = lanes >> 1; o >= 1; o >>= 1)
        sum += __shfl_xor(sum, o, 64);
    if (live && kind < 2 && nw) {
        const float r = 1.0f / sqrtf(a.eps + sum / (float)kv.dim);
        const float4 g = *(const float4 *)(nw + at);
        v = float4{g.x * (v.x * r), g.y * (v.y * r), g.z * (v.z * r), g.w * (v.w * r)};
    }
    float *mine = row + 4 * ((int)threadIdx.x & ~(lanes - 1));
    if (!a.pairs)
        *(float4 *)(mine + at) = v;
    __syncthreads();
    if (live && kind < 2 && at < a.rot) {
        float *e = &v.x;
        const int half = (int)a.rot / 2;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int d = at + k;
            float co, si;
            if (a.pairs) {
                if ((k & 1) || d >= a.rot)
                    continue;
                turn(p, a.freq[d / 2], co, si);
                const float u = e[k], w = e[k + 1];
                e[k] = u * co - w * si;
                e[k + 1] = w * co + u * si;
            } else if (d < a.rot) {
                turn(p, a.freq[d < half ? d : d - half], co, si);
                e[k] = d < half ? e[k] * co - mine[d + half] * si : e[k] * co + mine[d - half] * si;
            }
        }
    }
    if (!live)
        return;
    if (kind == 0) {
        *(float4 *)(a.out + i * a.out_ld + hh * a.out_hd + at) = v;
        return;
    }
    if (p < 0 || p / kv.page >= kv.table_ld)
        return;
    const long page = kv.table[s * kv.table_ld + p / kv.page];
    if (page < 0 || page >= kv.pages)
        return;
    store4<TYPE>(kind == 1 ? kv.k : kv.v, ((page * nk + hh) * kv.page + p % kv.page) * kv.dim + at, v);
}

} /* namespace */

void q8_launch_conv(q8_stream_t s, const rt_seqs &b, const float *x, long x_ld, long ch, const float *w, long taps, const float *s_in, float *s_out,
                    float *y, long y_ld)
{
    /* a sequence's runs over as many workgroups as the longest needs, but no more than four times what all
     * tokens need in all: with many sequences of mixed lengths a longer one's workgroups take several runs */
    const long runs = (b.longest + CONV_RUN - 1) / CONV_RUN, most = 4 * (b.t / CONV_RUN + b.n) / b.n, parts = runs < most ? runs : most;
    const dim3 grid((unsigned)((ch / 4 + 255) / 256), (unsigned)b.n, (unsigned)(parts < 65535 ? parts : 65535));
    switch (taps) {
#define CONV(T)                                                                                                                                            \
    case T:                                                                                                                                                \
        conv_k<T><<<grid, 256, 0, (hipStream_t)s>>>(b, x, x_ld, ch, w, s_in, s_out, y, y_ld);                                                              \
        break;
        CONV(2)
        CONV(3)
        CONV(4)
        CONV(5)
        CONV(6)
        CONV(7)
        CONV(8)
#undef CONV
    }
}

void q8_launch_rope(q8_stream_t s, const rt_seqs &b, const rt_kv &kv, const rt_rope &a)
{
    int lanes = 8;
    while (lanes * 4 < kv.dim)
        lanes *= 2;
    const long heads = a.q_heads + 2 * kv.heads, per = 64 * ROPE_WAVES / lanes;
    const dim3 grid((unsigned)b.t, (unsigned)((heads + per - 1) / per));
    if (kv.type == RT_F32)
        rope_k<RT_F32><<<grid, 64 * ROPE_WAVES, 0, (hipStream_t)s>>>(b, kv, a, lanes);
    else if (kv.type == RT_F16)
        rope_k<RT_F16><<<grid, 64 * ROPE_WAVES, 0, (hipStream_t)s>>>(b, kv, a, lanes);
    else
        rope_k<RT_BF16><<<grid, 64 * ROPE_WAVES, 0, (hipStream_t)s>>>(b, kv, a, lanes);
}
