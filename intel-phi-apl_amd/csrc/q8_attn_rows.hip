/* q8_attn_rows.hip: attention of prompts through a window over a 16-bit cache (include/q8_mix.h). */
#include "q8_attn.h"

namespace {

/* As the 8-bit cache's prompts: 64 query rows a workgroup, 16 a wave, which share a tile of positions in LDS, the keys as they
 * lie and the values transposed, the next tile's loads under way in registers. The products are those of the 16-bit caches: the
 * queries as LIMBS 16-bit values each, in registers. The weights are three bf16 limbs here, which hold any F32 weight, so that none
 * is too small; a BF16 value is their operand as it is, an F16 one is the sum of two (its upper 8 bits, and the 3 that
 * are left, which the third limb need not meet: 2^-24 of the product).
 *
 * A wave of 256 elements has 64 registers of output and 96 of queries. With tiles of 32 positions the rest of a tile fits beside
 * them for two waves a SIMD, one of which multiplies while the other waits or is in its softmax: prompts of 4001 tokens and
 * less through 512 positions, 8 heads on 2 of 256, BF16, 142 us, 204 with 64 positions and one wave; 394 with 16 rows a workgroup. With
 * nothing spilled, that is: who waits for a reload waits for the next tile's loads, which were issued before it (45 registers: 193 us). Heads of up to 128 have room for 64 positions. The limbs' products go to one sum, as
 * three would be 16 registers more; two LDS buffers with one barrier a tile measured the same, and so did layouts with a fifth of
 * the bank conflicts (which are a third of LDS's time).
 *
 * Infinities and NaN in a key or a value make a product with a limb or a weight of 0 NaN where the definition has none. So a
 * wave whose sums are not all finite at the end computes its rows again, one by one and in F32, without what a row does not
 * see (50 times slower, where all do). Positions that none of the workgroup's rows sees are 0 in LDS, whatever lies there. */

template <int D, int TYPE>
__device__ __forceinline__ float element(const void *cache, uint64_t row, int d)
{
    return half_of<TYPE>::back(((const uint16_t *)cache)[row * D + d]);
}

/* Row `i` of the wave's again: its maximum and sum, and element lane + 64 n of its output in o[n] */
template <int D, int TYPE>
__device__ __forceinline__ void slowly(const rt_kv &kv, const rt_attn &a, const plan &p, const share &u, uint32_t head_rows, int i, float &m, float &l, float (&o)[(D + 63) / 64])
{
    constexpr int SUB = q8_attn_rows_tile(D), POS = 16 * SUB;
    const int lane = threadIdx.x & 63, j = __shfl(u.j, i, 64), head = __shfl(u.h, i, 64), lim = __shfl(u.lim, i, 64), low = __shfl(u.low, i, 64);
    const float *q = a.q + (long)(u.q.first + j) * a.q_ld + head * a.q_hd;
    m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int n = 0; n < (D + 63) / 64; n++)
        o[n] = 0.0f;
    const int stop = (u.t1 + SUB - 1) / SUB;
    for (int first = u.t0 / SUB; first < stop; first += 64 / POS) {
        const int tile = first + lane / POS, pos = place_of<true>(u, tile, SUB) * POS + lane % POS;
        const bool seen = tile < stop && pos <= lim && !passed<true>(p, pos, low);
        const int entry = seen ? u.table[p.page.of(pos)] : 0;
        const bool there = (uint32_t)entry < (uint32_t)kv.pages;
        const uint32_t row = (seen && there ? (uint32_t)entry * (uint32_t)(kv.heads * kv.page) + ((uint32_t)pos - p.page.of(pos) * (uint32_t)kv.page) : 0) + head_rows;
        float s = 0.0f;
        for (int d = 0; d < D; d++)
            s = fmaf(q[d] * p.qscale, element<D, TYPE>(kv.k, row, d), s);
        s = !seen ? -INFINITY : there ? s : NAN;
        float top = s;
        for (int k = 32; k >= 1; k >>= 1)
            top = fmaxf(top, __shfl_xor(top, k, 64));
        const float raised = fmaxf(m, top), ref = raised == -INFINITY ? 0.0f : raised, f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - raised);
        const float weight = seen ? __builtin_amdgcn_exp2f(s - ref) : 0.0f;
        m = raised;
        float sum = weight;
        for (int k = 32; k >= 1; k >>= 1)
            sum += __shfl_xor(sum, k, 64);
        l = fmaf(l, f, sum);
#pragma unroll
        for (int n = 0; n < (D + 63) / 64; n++)
            o[n] *= f;
        for (int k = 0; k < 64; k++) {
            const float w = __shfl(weight, k, 64);
            const uint32_t at = (uint32_t)__shfl((int)row, k, 64);
            if (w != 0.0f) /* a NaN is not 0 */
#pragma unroll
                for (int n = 0; n < (D + 63) / 64; n++)
                    if (lane + 64 * n < D)
                        o[n] = fmaf(w, element<D, TYPE>(kv.v, at, lane + 64 * n), o[n]);
        }
    }
}

template <int D, int TYPE>
__global__ __launch_bounds__(64 * WAVES, 2) void attn_rows_k(rt_seqs b, rt_kv kv, rt_attn a, plan p, order places)
{
    typedef half_of<TYPE> H;
    constexpr int SUB = q8_attn_rows_tile(D), POS = 16 * SUB, LIMBS = H::LIMBS, NK = D / 32, VE = D / 16, PIECES = D / 8, NP = (POS * PIECES + 255) / 256, FOURTH = 17 * D / 16 + 1, EACH = D > 128 ? 4 : D > 64 ? 2 : 1;
    constexpr int PARTS = TYPE == RT_F16 ? 2 : 1; /* bf16 values that a value is the sum of */
    struct shared {
        uint8_t k[POS][2 * D + 16];
        v4i v[PARTS][SUB == 4 ? 8 * D : 4 * FOURTH];
    };
    __shared__ __align__(16) shared sh;
    /* Positions 8 n .. 8 n + 7 of element d, so that neither 16 lanes' reads (of d, d + 1, ..) nor their writes (of d, d + 4, ..) meet in a
     * bank. With 4 pieces an element: every fourth element's in a row, 16 bytes between each 4, which takes no register for
     * the next elements' places. */
    const auto value = [&](int part, int d, int n) __attribute__((always_inline)) -> v4i & {
        return sh.v[part][SUB == 4 ? 8 * d + ((n + spread(d)) & 7) : (d & 3) * FOURTH + 4 * (d >> 2) + (d >> 4) + n];
    };
    const int tid = threadIdx.x, lane = tid & 63, wave = first_lane(tid >> 6), c = lane & 15, g = lane >> 4;
    const int group = p.heads;
    int number, head;
    if (!place_in(places, (int)blockIdx.x, number, head))
        return;
    const uint32_t head_rows = (uint32_t)head * (uint32_t)kv.page;
    share u;
    if (!share_of<true, ROWS>(b, kv, p, group, number, head, u))
        return;
    const int stop = (u.t1 + SUB - 1) / SUB;
    int tile = u.t0 / SUB;
    const int least = window_from(p, u.q, first_lane((int)p.group.of(u.z * ROWS))); /* the first that any row's window has */
    const auto here = [&](int t) __attribute__((always_inline)) { /* the lane's position of tile t, or the last that there is */
        const int i = place_of<true>(u, t, SUB) * POS + lane;
        return u.end < 0 ? 0 : i < u.end ? i : u.end;
    };
    int entry = u.table[p.page.of(here(tile))]; /* (the table reaches them all) */
    v4i kx[NP];
    uint32_t vx[4 * SUB][EACH > 2 ? 2 : 1];
    bool none = false, gone = false; /* the lane's position of the tile has no row; no row of the workgroup sees it */
    const auto load = [&](int t) __attribute__((always_inline)) {
        const uint32_t pos = (uint32_t)here(t);
        none = (uint32_t)entry >= (uint32_t)kv.pages;
        gone = passed<true>(p, (int)pos, least);
        const uint32_t place = (none ? 0 : (uint32_t)entry * (uint32_t)(kv.heads * kv.page) + (pos - p.page.of(pos) * (uint32_t)kv.page)) + head_rows; /* below 2^31 */
        entry = u.table[p.page.of(here(t + 1))];
        uint32_t rows[NP];
#pragma unroll
        for (int i = 0; i < NP; i++)
            rows[i] = (uint32_t)__shfl((int)place, (tid + 256 * i) / PIECES, 64);
#pragma unroll
        for (int i = 0; i < 4 * SUB; i++) {
            /* positions 16 n + 4 g + r: g the wave's number, i = 4 n + r */
            const char *v = (const char *)kv.v + (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)place, i / 4 * 16 + 4 * wave + i % 4) * (2 * D);
            const uint32_t off = lane * EACH < D ? lane * EACH * 2 : 0;
            if constexpr (EACH == 4) {
                const uint2 w = *(const uint2 *)(v + off);
                vx[i][0] = w.x, vx[i][1] = w.y;
            } else {
                vx[i][0] = EACH == 2 ? *(const uint32_t *)(v + off) : *(const uint16_t *)(v + off);
            }
        }
#pragma unroll
        for (int i = 0; i < NP; i++)
            kx[i] = *(const v4i *)((const char *)kv.k + (uint64_t)rows[i] * (2 * D) + (tid + 256 * i) % PIECES * 16);
    };
    unsigned long long missing = 0; /* the tile's positions that have no row */
    const auto store = [&]() __attribute__((always_inline)) {
        missing = __ballot(none && !gone);
        if (__ballot(gone))
#pragma unroll
            for (int i = 0; i < 4 * SUB; i++)
                if (__builtin_amdgcn_readlane(gone ? 1 : 0, i / 4 * 16 + 4 * wave + i % 4))
#pragma unroll
                    for (int e = 0; e < (EACH > 2 ? 2 : 1); e++)
                        vx[i][e] = 0;
#pragma unroll
        for (int i = 0; i < NP; i++)
            if (POS * PIECES % 256 == 0 || tid + 256 * i < POS * PIECES)
                *(v4i *)&sh.k[(tid + 256 * i) / PIECES][(tid + 256 * i) % PIECES * 16] = kx[i];
        if (D % (64 * EACH) == 0 || lane * EACH < D)
#pragma unroll
            for (int e = 0; e < EACH; e++)
#pragma unroll
                for (int k = 0; k < SUB / 2; k++) {
                    v4i w[PARTS];
#pragma unroll
                    for (int r = 0; r < 8; r += 2) {
                        const uint32_t x = vx[8 * k + r][e / 2], y = vx[8 * k + r + 1][e / 2];
                        if constexpr (TYPE == RT_BF16) {
                            w[0][r / 2] = (int)__builtin_amdgcn_perm(y, x, e & 1 ? 0x07060302u : 0x05040100u);
                        } else {
                            const float f = H::back((uint16_t)(x >> (16 * (e & 1)))), h = H::back((uint16_t)(y >> (16 * (e & 1))));
                            w[0][r / 2] = (int)pack_hi(f, h); /* the upper 8 bits */
                            w[PARTS - 1][r / 2] = (int)pack_hi(f - __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, f) & 0xffff0000u),
                                                              h - __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, h) & 0xffff0000u));
                        }
                    }
#pragma unroll
                    for (int n = 0; n < PARTS; n++)
                        value(n, lane * EACH + e, 4 * k + wave) = w[n];
                }
    };
    if (tile < stop)
        load(tile);
    /* the wave's queries as limbs: elements 32 i + 8 g .. of row c */
    v4i query[NK][LIMBS];
    float back = 1.0f; /* (F16) the power of two that the row is smaller by than its limbs */
    {
        const float *q = a.q + (u.live ? (long)(u.q.first + u.j) * a.q_ld + u.h * a.q_hd : 0) + 8 * g;
        v4f x[NK][2];
#pragma unroll
        for (int i = 0; i < NK; i++)
            x[i][0] = *(const v4f *)(q + 32 * i), x[i][1] = *(const v4f *)(q + 32 * i + 4);
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < NK; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                x[i][e / 4][e % 4] = u.live ? x[i][e / 4][e % 4] * p.qscale : 0.0f;
                most = fmaxf(most, fabsf(x[i][e / 4][e % 4]));
            }
        int up = 0;
        if (TYPE == RT_F16) {
            most = group_max(most);
            up = most > 0.0f && most < INFINITY ? 14 - __builtin_amdgcn_frexp_expf(most) : 0;
            up = up > 120 ? 120 : up < -120 ? -120 : up;
            back = ldexpf(1.0f, -up);
        }
#pragma unroll
        for (int i = 0; i < NK; i++) {
            float y[8];
            uint4 w[LIMBS];
#pragma unroll
            for (int e = 0; e < 8; e++)
                y[e] = TYPE == RT_F16 ? ldexpf(x[i][e / 4][e % 4], up) : x[i][e / 4][e % 4];
            limbs_of<TYPE>(y, w);
#pragma unroll
            for (int n = 0; n < LIMBS; n++)
                query[i][n] = __builtin_bit_cast(v4i, w[n]);
        }
    }
    v4f acc[VE];
#pragma unroll
    for (int i = 0; i < VE; i++)
        acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    const bool some = u.row < u.q.n * group; /* the wave has rows */
    for (; tile < stop; tile++) {
        __syncthreads(); /* the tile before has been read */
        store();
        __syncthreads();
        const unsigned long long lost = missing;
        if (tile + 1 < stop)
            load(tile + 1);
        const int base = place_of<true>(u, tile, SUB) * POS;
        /* none of the wave's rows sees any of it */
        if (!some || base > u.last || (base + POS <= u.lo0 && base >= p.sinks))
            continue;
        const bool whole = all_seen<true>(p, u, base, POS); /* every row sees every position of the tile */
        float x[4 * SUB], top = -INFINITY;
        const auto key = [&](int n, int i) __attribute__((always_inline)) { return *(const uint4 *)&sh.k[16 * n + c][64 * i + 16 * g]; };
        uint4 kk[2][SUB]; /* the next 32 elements' operands are read under these ones' products */
        v4f s[SUB];
#pragma unroll
        for (int n = 0; n < SUB; n++) {
            kk[0][n] = key(n, 0);
            s[n] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        }
#pragma unroll
        for (int i = 0; i < NK; i++) {
            if (i + 1 < NK)
#pragma unroll
                for (int n = 0; n < SUB; n++)
                    kk[(i + 1) & 1][n] = key(n, i + 1);
#pragma unroll
            for (int e = LIMBS - 1; e >= 0; e--) /* the smallest first */
#pragma unroll
                for (int n = 0; n < SUB; n++)
                    s[n] = H::mfma(kk[i & 1][n], __builtin_bit_cast(uint4, query[i][e]), s[n]);
        }
#pragma unroll
        for (int n = 0; n < SUB; n++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                x[4 * n + r] = s[n][r] * back;
        if (lost)
#pragma unroll
            for (int r = 0; r < 4 * SUB; r++)
                x[r] = (uint32_t)(lost >> (r / 8 * 32)) >> 4 * g & 1u << (r / 4 % 2 * 16 + r % 4) ? NAN : x[r];
        if (!whole)
#pragma unroll
            for (int r = 0; r < 4 * SUB; r++) {
                const int i = base + r / 4 * 16 + 4 * g + r % 4;
                x[r] = i > u.lim || passed<true>(p, i, u.low) ? -INFINITY : x[r];
            }
#pragma unroll
        for (int r = 0; r < 4 * SUB; r++)
            top = fmaxf(top, x[r]);
        const float ref = reference(top, SLACK, m, l, acc);
#pragma unroll
        for (int r = 0; r < 4 * SUB; r++) {
            x[r] = __builtin_amdgcn_exp2f(x[r] - ref);
            l += x[r];
        }
#pragma unroll
        for (int k = 0; k < SUB / 2; k++) {
            v4i w[3];
            limbs8(x + 8 * k, w);
#pragma unroll
            for (int e = 0; e < VE; e += 2) {
                v4i v[PARTS][2];
#pragma unroll
                for (int n = 0; n < PARTS; n++)
#pragma unroll
                    for (int f = 0; f < 2; f++)
                        v[n][f] = value(n, 16 * (e + f) + c, 4 * k + g);
#pragma unroll
                for (int n = 0; n < PARTS; n++)
#pragma unroll
                    for (int i = 0; i < 3 - n; i++)
#pragma unroll
                        for (int f = 0; f < 2; f++)
                            acc[e + f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, v[n][f]), __builtin_bit_cast(b8, w[i]), acc[e + f], 0, 0, 0);
            }
        }
    }
    l = group_sum(l);
    float odd = l * 0.0f;
#pragma unroll
    for (int e = 0; e < VE; e++)
#pragma unroll
        for (int r = 0; r < 4; r++)
            odd = fmaf(acc[e][r], 0.0f, odd);
    const long slot0 = ((long)head * p.slots + number) * ROWS + (u.row - u.z * ROWS), sums = kv.heads * p.slots * ROWS * D;
    if (__ballot(u.live && odd != 0.0f)) { /* something is infinite or NaN */
        for (int i = 0; i < 16 && u.row + i < u.q.n * group; i++) {
            float o[(D + 63) / 64];
            slowly<D, TYPE>(kv, a, p, u, head_rows, i, m, l, o);
            const int j = __shfl(u.j, i, 64), h = __shfl(u.h, i, 64);
            const long token = u.q.first + j, pos = (long)u.q.past + j;
            l = pos >= p.cap ? NAN : l;
#pragma unroll
            for (int n = 0; n < (D + 63) / 64; n++) {
                const int d = lane + 64 * n;
                if (d >= D)
                    continue;
                if (u.q.chunks > 1)
                    p.part[(slot0 + i) * D + d] = o[n];
                else
                    a.o[token * a.o_ld + (long)h * D + d] = pos < 0 ? 0.0f : o[n] / l * (a.gate ? q8_sigmoid(a.gate[token * a.gate_ld + h * a.gate_hd + d]) : 1.0f);
            }
            if (u.q.chunks > 1 && lane == 0)
                *(float2 *)(p.part + sums + (slot0 + i) * 2) = float2{m, l};
        }
        return;
    }
    if (!u.live)
        return;
    const long pos = (long)u.q.past + u.j;
    const float sum = pos >= p.cap ? NAN : l; /* a position that the table does not reach */
    if (u.q.chunks > 1) {
#pragma unroll
        for (int e = 0; e < VE; e++)
            *(v4f *)(p.part + (slot0 + c) * D + 16 * e + 4 * g) = acc[e];
        if (g == 0)
            *(float2 *)(p.part + sums + (slot0 + c) * 2) = float2{m, sum};
        return;
    }
    const float r = 1.0f / sum;
    const long token = u.q.first + u.j;
    float *o = a.o + token * a.o_ld + (long)u.h * D + 4 * g;
    const float *gate = a.gate ? a.gate + token * a.gate_ld + u.h * a.gate_hd + 4 * g : nullptr;
    v4f gx[VE]; /* all gates under way at once, not one after the other */
    if (gate)
#pragma unroll
        for (int e = 0; e < VE; e++)
            gx[e] = *(const v4f *)(gate + 16 * e);
#pragma unroll
    for (int e = 0; e < VE; e++) {
        v4f v;
#pragma unroll
        for (int n = 0; n < 4; n++)
            v[n] = pos < 0 ? 0.0f : acc[e][n] * r * (gate ? gate_weight(gx[e][n]) : 1.0f);
        *(v4f *)(o + 16 * e) = v;
    }
}

} /* namespace */

void q8_launch_attn_rows(q8_stream_t stream, long blocks, const rt_seqs &b, const rt_kv &kv, const rt_attn &a, const q8_attn_plan &p)
{
    const order places = order_of(blocks, kv.heads);
    const unsigned all = 8u * (unsigned)places.count;
    switch (kv.dim) {
#define DIM(D)                                                                                                                                             \
    case D:                                                                                                                                                \
        kv.type == RT_F16 ? attn_rows_k<D, RT_F16><<<all, 64 * WAVES, 0, (hipStream_t)stream>>>(b, kv, a, p, places)                                       \
                          : attn_rows_k<D, RT_BF16><<<all, 64 * WAVES, 0, (hipStream_t)stream>>>(b, kv, a, p, places);                                     \
        break;
        DIM(32)
        DIM(64)
        DIM(96)
        DIM(128)
        DIM(160)
        DIM(192)
        DIM(224)
        DIM(256)
#undef DIM
    }
}
