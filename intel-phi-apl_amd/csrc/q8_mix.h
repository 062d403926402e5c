/* q8_mix.h: the launchers of the operators of include/q8_mix.h, and what their kernels share. */
#ifndef Q8_MIX_DEVICE_H
#define Q8_MIX_DEVICE_H

#include "../../include/q8_mix.h"
#include "q8_device.h"

void q8_launch_conv(q8_stream_t s, const rt_seqs &b, const float *x, long x_ld, long ch, const float *w, long taps, const float *s_in, float *s_out,
                    float *y, long y_ld);
void q8_launch_rope(q8_stream_t s, const rt_seqs &b, const rt_kv &kv, const rt_rope &a);
/* prep: q8_delta_prep_floats floats of workspace (none: may be NULL) */
long q8_delta_prep_floats(const rt_seqs &b, const rt_delta &a);
void q8_launch_delta(q8_stream_t s, const rt_seqs &b, const rt_delta &a, float *prep);
/* part: q8_attn_part_floats floats of workspace (none: may be NULL) */
long q8_attn_part_floats(const rt_seqs &b, const rt_kv &kv, const rt_attn &a);
void q8_launch_attn(q8_stream_t s, const rt_seqs &b, const rt_kv &kv, const rt_attn &a, float *part);

#if defined(__HIPCC__)

/* Sequence s's rows [first, last) of the token-major arrays: inside [0, t) whatever start holds */
__device__ __forceinline__ void q8_rows_of(const rt_seqs &b, long s, long &first, long &last)
{
    const long t = b.t, f = b.start[s], l = b.start[s + 1];
    first = f < 0 ? 0 : f > t ? t : f;
    last = l < first ? first : l > t ? t : l;
}

/* The sequence that has row i, or -1: the starts at or before i counted 64 at a time by the wave (all
 * of whose active lanes ask for the same row) */
__device__ __forceinline__ long q8_sequence_of(const rt_seqs &b, long i)
{
    const int lane = threadIdx.x & 63;
    long c = 0;
    for (long s = 0; s <= b.n; s += 64) {
        const bool at = s + lane <= b.n && (long)b.start[s + lane <= b.n ? s + lane : 0] <= i;
        const unsigned long long m = __ballot(at);
        c += __popcll(m);
        if (m != ~0ull)
            break;
    }
    if (c < 1 || c > b.n)
        return -1;
    const long s = c - 1;
    return (long)b.start[s] <= i && i < (long)b.start[s + 1] ? s : -1;
}

/* 1 / (1 + exp(-x)) without an overflow on either side */
__device__ __forceinline__ float q8_sigmoid(float x)
{
    const float e = expf(-fabsf(x));
    return (x >= 0.0f ? 1.0f : e) / (1.0f + e);
}

#endif
#endif
