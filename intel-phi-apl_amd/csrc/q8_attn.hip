/* q8_attn.hip: attention of new tokens over the paged key-value cache (include/q8_mix.h). */
#include "q8_mix.h"

namespace {

template <int TYPE>
__device__ __forceinline__ float cached(const void *cache, long at)
{
    if constexpr (TYPE == RT_F32)
        return ((const float *)cache)[at];
    else if constexpr (TYPE == RT_F16)
        return (float)((const _Float16 *)cache)[at];
    else
        return __builtin_bit_cast(float, (uint32_t)((const uint16_t *)cache)[at] << 16);
}

/* A wave a query head of a token, position by position, with the running maximum and sum of the softmax;
 * lane l holds elements l, l + 64, ... of the head. */
template <int TYPE>
__global__ __launch_bounds__(64) void attn_k(rt_seqs b, rt_kv kv, rt_attn a)
{
    const long i = blockIdx.x, h = blockIdx.y, s = q8_sequence_of(b, i);
    if (s < 0)
        return;
    const int lane = threadIdx.x;
    const long last = (long)b.past[s] + (i - b.start[s]), kh = h / (a.q_heads / kv.heads);
    float q[4], o[4] = {};
#pragma unroll
    for (int e = 0; e < 4; e++)
        q[e] = lane + 64 * e < kv.dim ? a.scale * a.q[i * a.q_ld + h * a.q_hd + lane + 64 * e] : 0.0f;
    float m = -INFINITY, l = 0.0f;
    for (long p = 0; p <= last; p++) {
        const long page = p / kv.page < kv.table_ld ? (long)kv.table[s * kv.table_ld + p / kv.page] : -1;
        const bool there = page >= 0 && page < kv.pages;
        const long at = ((there ? page : 0) * kv.heads + kh) * kv.page * kv.dim + (there ? p % kv.page : 0) * kv.dim;
        float x = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (lane + 64 * e < kv.dim)
                x = fmaf(q[e], cached<TYPE>(kv.k, at + lane + 64 * e), x);
        x = there ? q8_wave_sum(x) : NAN;
        const float mn = fmaxf(m, x), ref = mn == -INFINITY ? 0.0f : mn, f = expf(m - ref), w = expf(x - ref);
        l = fmaf(l, f, w);
        m = mn;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (lane + 64 * e < kv.dim)
                o[e] = fmaf(w, cached<TYPE>(kv.v, at + lane + 64 * e), o[e] * f);
        if (!there)
            break; /* NaN from here on */
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (lane + 64 * e < kv.dim) {
            float v = last < 0 ? 0.0f : o[e] / l;
            if (a.gate)
                v *= q8_sigmoid(a.gate[i * a.gate_ld + h * a.gate_hd + lane + 64 * e]);
            a.o[i * a.o_ld + h * kv.dim + lane + 64 * e] = v;
        }
}

} /* namespace */

void q8_launch_attn(q8_stream_t s, const rt_seqs &b, const rt_kv &kv, const rt_attn &a)
{
    const dim3 grid((unsigned)b.t, (unsigned)a.q_heads);
    if (kv.type == RT_F32)
        attn_k<RT_F32><<<grid, 64, 0, (hipStream_t)s>>>(b, kv, a);
    else if (kv.type == RT_F16)
        attn_k<RT_F16><<<grid, 64, 0, (hipStream_t)s>>>(b, kv, a);
    else
        attn_k<RT_BF16><<<grid, 64, 0, (hipStream_t)s>>>(b, kv, a);
}
