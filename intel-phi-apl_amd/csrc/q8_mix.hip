/* q8_mix.hip: the small operators of include/q8_mix.h, one pass over their data each: the short
 * convolution with SiLU, and the head norms with the rotation and the way into the paged cache. */
#include "q8_mix.h"

namespace {

/* ---- the short convolution
 *
 * A thread owns 4 neighbouring channels of one sequence and RUN tokens: it holds the run's rows and the TAPS - 1
 * before them in registers, all loaded before any arithmetic, so each x is read from HBM once (the rows at a run's
 * start once more, from L2) and a workgroup's loads are whole lines. Every load is unconditional: rows that there are not
 * are ones that there are, and their results are not stored. A sequence's first workgroup, the only one to read its
 * state, writes the new one at its end, so that the state may be updated in place. Bound by HBM on prompts (3996 tokens
 * of 8192 channels 52 us, 5.0 TB/s), by latency on single tokens, for which RUN is 1. */
template <int TAPS, int RUN>
__global__ __launch_bounds__(256) void conv_k(rt_seqs b, const float *__restrict__ x, long x_ld, long ch, const float *__restrict__ w, const float *s_in,
                                              float *s_out, float *__restrict__ y, long y_ld)
{
    const long c = 4 * ((long)blockIdx.x * 256 + threadIdx.x), s = blockIdx.y;
    if (c >= ch)
        return;
    float wt[4 * TAPS];
#pragma unroll
    for (int i = 0; i < TAPS; i++)
        *(float4 *)(wt + 4 * i) = *(const float4 *)(w + c * TAPS + 4 * i);
    long first, last;
    q8_rows_of(b, s, first, last);
    const long n = last - first;
    const float *xs = x + first * x_ld + c, *old = s_in + s * (TAPS - 1) * ch + c;
    /* input i of the sequence, those before 0 from the state (the nearest that there is) */
    const auto input = [&](long i) {
        const long k = i < n ? i : n - 1;
        return *(const float4 *)(k < 0 ? old + (k + TAPS - 1 > 0 ? k + TAPS - 1 : 0) * ch : xs + k * x_ld);
    };
    for (long r = blockIdx.z; r * RUN < n; r += gridDim.z) {
        const long i0 = r * RUN;
        float4 u[RUN + TAPS - 1];
#pragma unroll
        for (int j = 0; j < RUN + TAPS - 1; j++)
            u[j] = input(i0 + j - (TAPS - 1));
#pragma unroll
        for (int j = 0; j < RUN; j++) {
            float4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < TAPS; k++) {
                v.x = fmaf(wt[k], u[j + k].x, v.x);
                v.y = fmaf(wt[TAPS + k], u[j + k].y, v.y);
                v.z = fmaf(wt[2 * TAPS + k], u[j + k].z, v.z);
                v.w = fmaf(wt[3 * TAPS + k], u[j + k].w, v.w);
            }
            v = float4{v.x * q8_sigmoid(v.x), v.y * q8_sigmoid(v.y), v.z * q8_sigmoid(v.z), v.w * q8_sigmoid(v.w)};
            if (i0 + j < n)
                *(float4 *)(y + (first + i0 + j) * y_ld + c) = v;
        }
    }
    if (blockIdx.z == 0) {
        float4 keep[TAPS - 1];
#pragma unroll
        for (int j = 0; j < TAPS - 1; j++)
            keep[j] = input(n - (TAPS - 1) + j);
#pragma unroll
        for (int j = 0; j < TAPS - 1; j++)
            *(float4 *)(s_out + (s * (TAPS - 1) + j) * ch + c) = keep[j];
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
    } else if constexpr (TYPE == RT_BF16) {
        typedef __bf16 b4 __attribute__((ext_vector_type(4)));
        *(b4 *)((__bf16 *)cache + at) = b4{(__bf16)v.x, (__bf16)v.y, (__bf16)v.z, (__bf16)v.w};
    }
}

/* A row of 8 bits: d = max|x| / 127 over the lanes that hold it, x as rint(x / d), which is within 127 (max / d is off by
 * less than a step of 127). A row with an element that is not finite gets NaN for d, so that it reads as NaN, and one whose d has no
 * full precision (below 2^-126) zeros. The scales lie behind all rows. The quotients are F32's own, so that a row's bits are those of
 * the definition (reciprocals: 2 us of 61 in a prompt of 3936 tokens, 24 heads of 256). */
__device__ __forceinline__ void store_q8(const rt_kv &kv, void *cache, long row, int at, int lanes, bool live, float4 x)
{
    const auto bits = [](float v) { return __builtin_bit_cast(uint32_t, fabsf(v)); };
    const uint32_t a = bits(x.x) > bits(x.y) ? bits(x.x) : bits(x.y), b = bits(x.z) > bits(x.w) ? bits(x.z) : bits(x.w);
    uint32_t most = live ? a > b ? a : b : 0;
    for (int o = lanes >> 1; o >= 1; o >>= 1) {
        const uint32_t other = __shfl_xor(most, o, 64);
        most = most > other ? most : other;
    }
    if (!live || row < 0)
        return;
    const float d = most < 0x7f800000u ? __builtin_bit_cast(float, most) / 127.0f : NAN;
    const bool plain = d >= 0x1p-126f;
    const auto byte = [&](float v) { return plain ? (uint32_t)(int)rintf(v / d) & 0xffu : 0u; };
    *(uint32_t *)((char *)cache + row * kv.dim + at) = byte(x.x) | byte(x.y) << 8 | byte(x.z) << 16 | byte(x.w) << 24;
    if (at == 0)
        ((float *)((char *)cache + kv.pages * kv.heads * kv.page * kv.dim))[row] = d < 0x1p-126f ? 0.0f : d;
}

/* Query, key and value heads of a token alike: LANES lanes (a power of two, 8 to 64) hold a head, 4 elements a lane, of
 * RUN tokens one after the other; the norm's sum goes over the lanes. A workgroup computes its tokens' cosines and
 * sines once, a thread one pair, and leaves them in LDS with the heads, whose halves turn together. Bound by latency on
 * a few tokens (RUN 1), by HBM on a prompt. */
constexpr int ROPE_WAVES = 4, ROPE_THREADS = 64 * ROPE_WAVES;

template <int TYPE, int RUN>
__global__ __launch_bounds__(ROPE_THREADS) void rope_k(rt_seqs b, rt_kv kv, rt_rope a, int lanes)
{
    __shared__ __align__(16) float row[RUN][ROPE_THREADS * 4];
    __shared__ float2 angle[RUN][128];
    const int tid = threadIdx.x, at = 4 * (tid & (lanes - 1)), half = (int)a.rot / 2;
    const long i0 = (long)blockIdx.x * RUN, h = ((long)blockIdx.y * ROPE_THREADS + tid) / lanes, nq = a.q_heads, nk = kv.heads;
    const int kind = h < nq ? 0 : h < nq + nk ? 1 : h < nq + 2 * nk ? 2 : 3;
    const long hh = kind == 0 ? h : kind == 1 ? h - nq : kind == 2 ? h - nq - nk : 0;
    const bool live = kind < 3 && at < kv.dim;
    const float *src = kind == 0 ? a.q + hh * a.q_hd : kind == 1 ? a.k + hh * a.k_hd : a.v + hh * a.v_hd, *nw = kind == 0 ? a.q_norm : a.k_norm;
    const long ld = kind == 0 ? a.q_ld : kind == 1 ? a.k_ld : a.v_ld;
    float4 v[RUN], norm = {1.0f, 1.0f, 1.0f, 1.0f};
#pragma unroll
    for (int k = 0; k < RUN; k++)
        v[k] = *(const float4 *)(src + (i0 + k < b.t ? i0 + k : i0) * ld + (live ? at : 0));
    if (kind < 2 && nw)
        norm = *(const float4 *)(nw + (live ? at : 0));
    long s[RUN], p[RUN];
#pragma unroll
    for (int k = 0; k < RUN; k++) {
        s[k] = i0 + k < b.t ? q8_sequence_of(b, i0 + k) : -1;
        p[k] = s[k] < 0 ? 0 : (long)b.past[s[k]] + (i0 + k - b.start[s[k]]);
    }
    for (int j = tid; j < RUN * half; j += ROPE_THREADS) {
        long pos = p[0];
        int pair = j;
#pragma unroll
        for (int k = 1; k < RUN; k++)
            if (j >= k * half)
                pos = p[k], pair = j - k * half;
        float2 cs;
        turn(pos, a.freq[pair], cs.x, cs.y);
        angle[0][(j - pair) / (half > 0 ? half : 1) * 128 + pair] = cs;
    }
#pragma unroll
    for (int k = 0; k < RUN; k++) {
        if (!live)
            v[k] = float4{0.0f, 0.0f, 0.0f, 0.0f};
        float sum = fmaf(v[k].w, v[k].w, fmaf(v[k].z, v[k].z, fmaf(v[k].y, v[k].y, v[k].x * v[k].x)));
        for (int o = lanes >> 1; o >= 1; o >>= 1)
            sum += __shfl_xor(sum, o, 64);
        if (kind < 2 && nw) {
            const float r = 1.0f / sqrtf(a.eps + sum / (float)kv.dim);
            v[k] = float4{norm.x * (v[k].x * r), norm.y * (v[k].y * r), norm.z * (v[k].z * r), norm.w * (v[k].w * r)};
        }
        *(float4 *)&row[k][4 * tid] = v[k];
    }
    __syncthreads();
    if (TYPE != RT_Q8 && !live)
        return;
    const int mine = 4 * (tid & ~(lanes - 1));
#pragma unroll
    for (int k = 0; k < RUN; k++) {
        if (s[k] < 0)
            continue;
        float4 x = v[k];
        if (kind < 2 && at < a.rot) {
            float *e = &x.x;
#pragma unroll
            for (int n = 0; n < 4; n++) {
                const int d = at + n;
                if (a.pairs) {
                    if ((n & 1) || d >= a.rot)
                        continue;
                    const float2 cs = angle[k][d / 2];
                    const float y = e[n], z = e[n + 1];
                    e[n] = y * cs.x - z * cs.y;
                    e[n + 1] = z * cs.x + y * cs.y;
                } else if (d < a.rot) {
                    const float2 cs = angle[k][d < half ? d : d - half];
                    const float other = row[k][mine + (d < half ? d + half : d - half)];
                    e[n] = d < half ? e[n] * cs.x - other * cs.y : e[n] * cs.x + other * cs.y;
                }
            }
        }
        if (kind == 0 && live) {
            *(float4 *)(a.out + (i0 + k) * a.out_ld + hh * a.out_hd + at) = x;
            continue;
        }
        const uint32_t pos = (uint32_t)p[k], slot = pos / (uint32_t)kv.page; /* p is below 2^32 */
        const long page = p[k] >= 0 && slot < kv.table_ld ? kv.table[s[k] * kv.table_ld + slot] : -1;
        const bool there = page >= 0 && page < kv.pages;
        const long to = (page * nk + hh) * kv.page + (pos - slot * (uint32_t)kv.page);
        if constexpr (TYPE == RT_Q8)
            store_q8(kv, kind == 1 ? kv.k : kv.v, there ? to : -1, at, lanes, live && kind > 0, x);
        else if (there)
            store4<TYPE>(kind == 1 ? kv.k : kv.v, to * kv.dim + at, x);
    }
}

template <int RUN>
void launch_rope(hipStream_t s, dim3 grid, const rt_seqs &b, const rt_kv &kv, const rt_rope &a, int lanes)
{
    if (kv.type == RT_F32)
        rope_k<RT_F32, RUN><<<grid, ROPE_THREADS, 0, s>>>(b, kv, a, lanes);
    else if (kv.type == RT_F16)
        rope_k<RT_F16, RUN><<<grid, ROPE_THREADS, 0, s>>>(b, kv, a, lanes);
    else if (kv.type == RT_BF16)
        rope_k<RT_BF16, RUN><<<grid, ROPE_THREADS, 0, s>>>(b, kv, a, lanes);
    else
        rope_k<RT_Q8, RUN><<<grid, ROPE_THREADS, 0, s>>>(b, kv, a, lanes);
}

template <int TAPS>
void launch_conv(hipStream_t st, const rt_seqs &b, const float *x, long x_ld, long ch, const float *w, const float *s_in, float *s_out, float *y, long y_ld)
{
    constexpr int RUN = 8; /* at least taps - 1: only a sequence's first run reads the state */
    const unsigned blocks = (unsigned)((ch / 4 + 255) / 256);
    if (b.longest == 1) {
        conv_k<TAPS, 1><<<dim3(blocks, (unsigned)b.n), 256, 0, st>>>(b, x, x_ld, ch, w, s_in, s_out, y, y_ld);
        return;
    }
    /* a sequence's runs over as many workgroups as the longest needs, but no more than four times what all
     * tokens need in all: with many sequences of mixed lengths a longer one's workgroups take several runs */
    const long runs = (b.longest + RUN - 1) / RUN, most = 4 * (b.t / RUN + b.n) / b.n, parts = runs < most ? runs : most;
    conv_k<TAPS, RUN><<<dim3(blocks, (unsigned)b.n, (unsigned)(parts < 65535 ? parts : 65535)), 256, 0, st>>>(b, x, x_ld, ch, w, s_in, s_out, y, y_ld);
}

} /* namespace */

void q8_launch_conv(q8_stream_t s, const rt_seqs &b, const float *x, long x_ld, long ch, const float *w, long taps, const float *s_in, float *s_out,
                    float *y, long y_ld)
{
    switch (taps) {
#define CONV(T)                                                                                                                                            \
    case T:                                                                                                                                                \
        launch_conv<T>((hipStream_t)s, b, x, x_ld, ch, w, s_in, s_out, y, y_ld);                                                                           \
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
    const long heads = a.q_heads + 2 * kv.heads, per = ROPE_THREADS / lanes, groups = (heads + per - 1) / per;
    /* two tokens a workgroup where that still gives every compute unit eight of them (5027 tokens, 24 heads of 256: 57 us, 4.0
     * TB/s; four 66, eight 82) */
    if (b.t * groups >= 4096)
        launch_rope<2>((hipStream_t)s, dim3((unsigned)((b.t + 1) / 2), (unsigned)groups), b, kv, a, lanes);
    else
        launch_rope<1>((hipStream_t)s, dim3((unsigned)b.t, (unsigned)groups), b, kv, a, lanes);
}
