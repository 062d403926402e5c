/* q8_attn.hip: attention of new tokens over the paged key-value cache of 32 or 16 bits, and the join of every type's parts
 * (include/q8_mix.h). */
#include "q8_attn.h"

namespace {

/* An F32 cache, 16 positions a tile, on v_mfma_f32_16x16x4_f32: position 4 g + r in the second product's step r. */
template <int D, bool WINDOW>
__global__ __launch_bounds__(64 * WAVES, D > 128 ? 1 : 2) void attn_f32_k(rt_seqs b, rt_kv kv, rt_attn a, plan p)
{
    constexpr int NK = D / 16, VE = D / 16, VEC = pieces(VE, 4), NV = VE / VEC;
    __shared__ __align__(16) char lds[joint_bytes<D>()];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const int group = p.heads;
    const uint32_t head_rows = (uint32_t)(blockIdx.y * kv.page);
    /* with starts that overlap there may be more chunks than slots: those are left out */
    for (int number = (int)blockIdx.x; p.target == 0 || number < p.slots; number += (int)gridDim.x) {
        share u;
        if (!share_of<WINDOW>(b, kv, p, group, number, (int)blockIdx.y, u))
            return;
        v4f acc[VE];
#pragma unroll
        for (int i = 0; i < VE; i++)
            acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        float m = -INFINITY, l = 0.0f;
        const auto here = [&](int tile) {
            const int i = place_of<WINDOW>(u, tile, 1) * 16 + c;
            return i < u.last ? i : u.last;
        };
        const auto load_k = [&](uint32_t (*kw)[4], int row) {
            const char *at = address(kv.k, row, head_rows, D * 4) + g * 16;
#pragma unroll
            for (int i = 0; i < NK; i++)
                load_words<4>(kw[i], at + i * 64);
        };
        uint32_t kw[NK][4], vw[4][NV][VEC];
        int tile = u.t0 + wave;
        const int stop = u.t1, now = entry_of(kv, p, u.table, here(tile));
        int entry = entry_of(kv, p, u.table, here(tile + WAVES));
        float4 qv[NK]; /* under way with the table's entries; the keys need those */
        const float *query = a.q + (u.live ? (long)(u.q.first + u.j) * a.q_ld + u.h * a.q_hd : 0) + g * 4;
#pragma unroll
        for (int i = 0; i < NK; i++)
            qv[i] = *(const float4 *)(query + i * 16);
        int row_now = row_of(kv, p, here(tile), now);
        load_k(kw, row_now);
#pragma unroll
        for (int i = 0; i < NK; i++)
            qv[i] = u.live ? float4{qv[i].x * p.qscale, qv[i].y * p.qscale, qv[i].z * p.qscale, qv[i].w * p.qscale} : float4{0.0f, 0.0f, 0.0f, 0.0f};
        for (; tile < stop; tile += WAVES) {
            int rows[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                rows[r] = __shfl(row_now, 4 * g + r, 64);
                const char *at = address(kv.v, rows[r], head_rows, D * 4) + c * VEC * 4;
#pragma unroll
                for (int i = 0; i < NV; i++)
                    stream_words<VEC>(vw[r][i], at + i * 16 * VEC * 4);
            }
            v4f s[2] = {v4f{0.0f, 0.0f, 0.0f, 0.0f}, v4f{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
            for (int i = 0; i < NK; i++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    s[e & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, kw[i][e]), (&qv[i].x)[e], s[e & 1], 0, 0, 0);
            if (tile + WAVES < stop) {
                row_now = row_of(kv, p, here(tile + WAVES), entry);
                entry = entry_of(kv, p, u.table, here(tile + 2 * WAVES));
                load_k(kw, row_now);
            }
            float x[4];
            const int base = place_of<WINDOW>(u, tile, 1) * 16;
            const bool whole = all_seen<WINDOW>(p, u, base, 16); /* every row sees every position of the tile */
#pragma unroll
            for (int r = 0; r < 4; r++) {
                x[r] = rows[r] < 0 ? NAN : s[0][r] + s[1][r];
                if (!whole && (base + 4 * g + r > u.lim || passed<WINDOW>(p, base + 4 * g + r, u.low)))
                    x[r] = -INFINITY;
            }
            const float ref = reference(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), SLACK, m, l, acc);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                x[r] = __builtin_amdgcn_exp2f(x[r] - ref);
                l += x[r];
            }
            /* a weight of 0 times an infinite or NaN value would be NaN: values that no row of the tile sees are 0, and
             * those that some do not see are looked at */
            bool apart = false;
            if (!whole) {
                float odd = 0.0f; /* NaN: one is infinite or NaN */
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int i = 0; i < NV; i++)
#pragma unroll
                        for (int e = 0; e < VEC; e++) {
                            vw[r][i][e] = base + 4 * g + r > u.last || passed<WINDOW>(p, base + 4 * g + r, u.lo0) ? 0 : vw[r][i][e];
                            odd = fmaf(__builtin_bit_cast(float, vw[r][i][e]), 0.0f, odd);
                        }
                apart = u.j0 < u.j1 && __ballot(odd != 0.0f);
            }
            if (!apart) {
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int i = 0; i < NV; i++)
#pragma unroll
                        for (int e = 0; e < VEC; e++)
                            acc[i * VEC + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, vw[r][i][e]), x[r], acc[i * VEC + e], 0, 0, 0);
            } else {
                /* each token's rows are computed apart, without the values that it does not see */
                for (int jj = u.j0; jj <= u.j1; jj++) {
                    const long upto = (long)u.q.past + jj < u.last ? (long)u.q.past + jj : u.last;
                    const int from = WINDOW ? window_from(p, u.q, jj) : 0;
#pragma unroll
                    for (int i = 0; i < NV; i++)
#pragma unroll
                        for (int e = 0; e < VEC; e++) {
                            v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                            for (int r = 0; r < 4; r++)
                                o = __builtin_amdgcn_mfma_f32_16x16x4f32(base + 4 * g + r <= upto && !passed<WINDOW>(p, base + 4 * g + r, from) ? __builtin_bit_cast(float, vw[r][i][e]) : 0.0f,
                                                                         x[r], o, 0, 0, 0);
                            if (u.j == jj)
                                acc[i * VEC + e] += o;
                        }
                }
            }
        }
        finish<D, VEC>(lds, kv, a, p, u, number, m, l, acc);
    }
}

/* A 16-bit cache, 32 or 64 positions a tile, on v_mfma_f32_16x16x32: the cache's values are its
 * operands as they are, and the F32 queries and weights are cut into LIMBS 16-bit values each, every one the
 * rest of those before rounded to nearest: in F16 two of them are off by at most 2^-23 of the value, in BF16 three by 2^-26, at
 * 2/16 and 3/16 of the time of F32 products.
 *
 * F16 has few exponents: its smallest step is 2^-24. A row of queries is scaled by the power of two that brings its
 * largest to 2^14 (and its scores back), so an element is off by up to 2^-39 of the row's largest. The weights are taken
 * 2^LIFT times as large (the sum that divides them is, too), up to 2^15: those from LEAST up are off by 2^-20 of themselves
 * at most, the others by more, and below 2^-25 they would be lost. They are a row's output where its largest weights' values
 * are near 0, as a sequence's first position's often are. So in a tile with a weight below LEAST each row's are scaled until
 * the largest is at 2^14 to 2^15, the sums with them. Where that leaves one below LEAST, too (20 powers of two between two
 * positions of a tile, as beside such a first position itself), what the limbs leave of it is taken again 2^38 times as large,
 * and again, until it is below 2^-22 of the weight. The sums wait in LDS meanwhile. 8 sequences of 4000 to 20000 positions, 32
 * heads of 128: 81 us, 93 where a first position of 18 nats above the rest makes every tile scale; a prompt of 2048 351
 * and 459.
 * The queries' limbs stay in LDS for the four waves. The second product's first operand is V transposed: of a
 * lane's 8 rows, the same element of two at a time by v_perm_b32. */
/* An infinite key is one in its product with the first limb; the others would make NaN of it (they
 * may be 0, or of the other sign), so where there may be one they get it as 0, and NaN, too. A value's weights are all
 * taken with this, and what it leaves out with 1 (where the weight is not 0): their first limb may be 0, too */
template <int TYPE>
__device__ __forceinline__ uint4 finite_only(uint4 x)
{
    constexpr uint32_t TOP = half_of<TYPE>::INF;
    const auto one = [](uint32_t w) { return ((w & TOP) == TOP ? 0u : w & 0xffffu) | ((w >> 16 & TOP) == TOP ? 0u : w & 0xffff0000u); };
    return uint4{one(x.x), one(x.y), one(x.z), one(x.w)};
}

__device__ __forceinline__ uint4 without(uint4 x, uint4 y) { return uint4{x.x ^ y.x, x.y ^ y.y, x.z ^ y.z, x.w ^ y.w}; }

typedef unsigned short u2 __attribute__((ext_vector_type(2)));
/* the larger magnitudes of two pairs of 16-bit values, as their bits: an infinity or NaN stays the largest */
__device__ __forceinline__ uint32_t larger(uint32_t x, uint32_t y)
{
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u2, x), __builtin_bit_cast(u2, y & 0x7fff7fffu)));
}

/* 16s of positions a tile: a tile's keys (and values) are 64 registers a lane from heads of 128 up, which then are one wave
 * a SIMD; smaller heads have two waves, which hold more in flight between them (64 elements, F16, 16 sequences of 500
 * to 9000: 43 us; with 64 positions a tile, which spills there, 62) */
constexpr int sixteens(long d) { return d == 128 ? 4 : 2; }
constexpr bool alone(long d) { return d >= 128; }

template <int D, int TYPE, bool WINDOW>
__global__ __launch_bounds__(64 * WAVES, alone(D) ? 1 : 2) void attn_half_k(rt_seqs b, rt_kv kv, rt_attn a, plan p)
{
    typedef half_of<TYPE> H;
    constexpr int LIMBS = H::LIMBS, NK = D / 32, VE = D / 16, VEC = pieces(VE, 8), NV = VE / VEC, VW = VEC / 2, SUB = sixteens(D), POS = 16 * SUB;
    static_assert(WAVES == 4);
    constexpr int KEPT = NK * LIMBS * 1024 + WAVES * 16 * 4, QUERIES = KEPT + (TYPE == RT_F16 ? WAVES * 64 * 4 * (VE * 4 + 4 * SUB) : 0);
    __shared__ __align__(16) char lds[joint_bytes<D>() > QUERIES ? joint_bytes<D>() : QUERIES];
    uint4(*sq)[LIMBS][64] = (uint4(*)[LIMBS][64])lds; /* until the waves join */
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    /* (F16) the lane's output and weights, while a tile's are on another scale */
    v4f *kept_acc = (v4f *)(lds + KEPT) + wave * 64 * VE + lane;
    float *kept = (float *)(lds + KEPT + WAVES * 64 * 16 * VE) + wave * 64 * 4 * SUB + lane;
    const int group = p.heads;
    const uint32_t head_rows = (uint32_t)(blockIdx.y * kv.page);
    for (int number = (int)blockIdx.x; p.target == 0 || number < p.slots; number += (int)gridDim.x) {
        share u;
        if (!share_of<WINDOW>(b, kv, p, group, number, (int)blockIdx.y, u))
            return;
        const int stop = (u.t1 + SUB - 1) / SUB; /* tiles: a chunk is a whole number of them, but for the last */
        int tile = u.t0 / SUB + wave, row[SUB], entry[SUB];
        const auto here = [&](int i) { return i < u.last ? i : u.last; };
        uint4 kx[SUB][NK];
        const auto load_k = [&]() {
#pragma unroll
            for (int n = 0; n < SUB; n++) {
                const char *at = address(kv.k, row[n], head_rows, D * 2) + g * 16;
#pragma unroll
                for (int i = 0; i < NK; i++)
                    kx[n][i] = *(const uint4 *)(at + i * 64);
            }
        };
        const auto load_entries = [&](int t) {
#pragma unroll
            for (int n = 0; n < SUB; n++)
                entry[n] = entry_of(kv, p, u.table, here(place_of<WINDOW>(u, t, SUB) * POS + 16 * n + c));
        };
        const auto rows_next = [&](int t) {
#pragma unroll
            for (int n = 0; n < SUB; n++)
                row[n] = row_of(kv, p, here(place_of<WINDOW>(u, t, SUB) * POS + 16 * n + c), entry[n]);
            load_entries(t + WAVES);
        };
        /* the table's entries, the queries, and with the entries the keys; wave w has the queries' columns 32 i, i = w,
         * w + WAVES, ..., and makes their limbs, for all waves */
        load_entries(tile);
        constexpr int NQ = (NK + WAVES - 1) / WAVES;
        const float *query = a.q + (u.live ? (long)(u.q.first + u.j) * a.q_ld + u.h * a.q_hd : 0) + g * 8;
        float4 qv[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            const int i = wave + n * WAVES < NK ? wave + n * WAVES : 0;
            qv[n][0] = *(const float4 *)(query + i * 32), qv[n][1] = *(const float4 *)(query + i * 32 + 4);
        }
        rows_next(tile);
        load_k();
        float back = 1.0f;
        int up = 0;
        if (TYPE == RT_F16) {
            float(*smost)[16] = (float(*)[16])(lds + NK * LIMBS * 1024); /* behind the limbs */
            float most = 0.0f;
#pragma unroll
            for (int n = 0; n < NQ; n++)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    most = fmaxf(most, fabsf((&qv[n][0].x)[e]));
            most = group_max(most * fabsf(p.qscale));
            if (g == 0)
                smost[wave][c] = most;
            __syncthreads();
            most = fmaxf(fmaxf(smost[0][c], smost[1][c]), fmaxf(smost[2][c], smost[3][c]));
            up = most > 0.0f && most < INFINITY ? 14 - __builtin_amdgcn_frexp_expf(most) : 0;
            up = up > 120 ? 120 : up < -120 ? -120 : up;
            back = ldexpf(1.0f, -up);
        }
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            const int i = wave + n * WAVES;
            float x[8];
            uint4 w[LIMBS];
#pragma unroll
            for (int e = 0; e < 8; e++)
                x[e] = u.live ? ldexpf((&qv[n][0].x)[e] * p.qscale, up) : 0.0f;
            limbs_of<TYPE>(x, w);
            if (i < NK)
#pragma unroll
                for (int l = 0; l < LIMBS; l++)
                    sq[i][l][lane] = w[l];
        }
        __syncthreads();
        v4f acc[VE];
#pragma unroll
        for (int i = 0; i < VE; i++)
            acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        float m = -INFINITY, l = 0.0f;
        for (; tile < stop; tile += WAVES) {
            int rows[4 * SUB]; /* rows 4 g + r of each 16 */
            uint32_t vw[NV][4 * SUB][VW];
#pragma unroll
            for (int r = 0; r < 4 * SUB; r++) {
                rows[r] = __shfl(row[r / 4], 4 * g + r % 4, 64);
                const char *at = address(kv.v, rows[r], head_rows, D * 2) + c * VEC * 2;
#pragma unroll
                for (int i = 0; i < NV; i++)
                    stream_words<VW>(vw[i][r], at + i * 16 * VEC * 2);
            }
            v4f s[SUB];
#pragma unroll
            for (int n = 0; n < SUB; n++)
                s[n] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            /* the scheduler is held to one step's limbs ahead: left free it reads them all before the first
             * product, and spills */
            __builtin_amdgcn_sched_barrier(0);
            uint4 qw[2][LIMBS];
#pragma unroll
            for (int n = 0; n < LIMBS; n++)
                qw[0][n] = sq[0][n][lane];
#pragma unroll
            for (int i = 0; i < NK; i++) {
#pragma unroll
                for (int n = 0; n < LIMBS && i + 1 < NK; n++)
                    qw[(i + 1) & 1][n] = sq[i + 1][n][lane];
#pragma unroll
                for (int n = 0; n < LIMBS; n++)
#pragma unroll
                    for (int k = 0; k < SUB; k++)
                        s[k] = H::mfma(kx[k][i], qw[i & 1][n], s[k]);
                __builtin_amdgcn_sched_barrier(0);
            }
            v4f odd = s[0] * 0.0f; /* NaN: a score is infinite or NaN */
#pragma unroll
            for (int n = 1; n < SUB; n++)
                odd += s[n] * 0.0f;
            if (__ballot(odd[0] + odd[1] + odd[2] + odd[3] != 0.0f)) {
#pragma unroll
                for (int n = 0; n < SUB; n++)
                    s[n] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < NK; i++) {
#pragma unroll
                    for (int n = 0; n < LIMBS; n++) {
                        const uint4 w = sq[i][n][lane];
#pragma unroll
                        for (int k = 0; k < SUB; k++)
                            s[k] = H::mfma(n ? finite_only<TYPE>(kx[k][i]) : kx[k][i], w, s[k]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (tile + WAVES < stop) {
                rows_next(tile + WAVES);
                load_k();
            }
            const int base = place_of<WINDOW>(u, tile, SUB) * POS;
            const auto place = [&](int r) { return base + r / 4 * 16 + 4 * g + r % 4; }; /* the lane's positions */
            float x[4 * SUB];
            const bool whole = all_seen<WINDOW>(p, u, base, POS); /* every row sees every position of the tile */
            float top = -INFINITY;
#pragma unroll
            for (int r = 0; r < 4 * SUB; r++) {
                x[r] = rows[r] < 0 ? NAN : back * s[r / 4][r % 4];
                if (!whole && (place(r) > u.lim || passed<WINDOW>(p, place(r), u.low)))
                    x[r] = -INFINITY;
                top = fmaxf(top, x[r]);
            }
            const float ref = reference(top, H::SLACK, m, l, acc) - H::LIFT;
            const auto limb = [](uint4 w, int e) { return H::back((uint16_t)((&w.x)[e / 2] >> (e & 1 ? 16 : 0))); };
            uint32_t least = ~0u; /* the smallest weight's bits but 0's, less 1 */
#pragma unroll
            for (int r = 0; r < 4 * SUB; r++) {
                x[r] = __builtin_amdgcn_exp2f(x[r] - ref);
                l += x[r];
                const uint32_t bits = __builtin_bit_cast(uint32_t, x[r]) - 1;
                least = least < bits ? least : bits;
            }
            constexpr uint32_t LEAST = __builtin_bit_cast(uint32_t, H::LEAST) - 1;
            const bool small = TYPE == RT_F16 && __ballot(least < LEAST);
            bool apart = false; /* the output is in LDS, and the tile's own in acc */
            float down = 1.0f;
            if (TYPE == RT_F16 && small) {
                float most = x[0];
#pragma unroll
                for (int r = 1; r < 4 * SUB; r++)
                    most = fmaxf(most, x[r]);
                most = group_max(most);
                int lift = most > 0.0f ? 15 - __builtin_amdgcn_frexp_expf(most) : 0;
                lift = lift < 140 ? lift : 140;
                down = ldexpf(1.0f, -lift);
                least = ~0u;
#pragma unroll
                for (int r = 0; r < 4 * SUB; r++) {
                    x[r] = ldexpf(x[r], lift);
                    const uint32_t bits = __builtin_bit_cast(uint32_t, x[r]) - 1;
                    least = least < bits ? least : bits;
                }
                apart = __ballot(least < LEAST || lift > 40);
                if (apart) {
#pragma unroll
                    for (int r = 0; r < 4 * SUB; r++)
                        kept[64 * r] = x[r];
#pragma unroll
                    for (int i = 0; i < VE; i++) {
                        kept_acc[64 * i] = acc[i];
                        acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
                    }
                } else {
                    const float up = ldexpf(1.0f, lift); /* outputs are below 2^(15 + 16 + 31): no overflow */
#pragma unroll
                    for (int i = 0; i < VE; i++)
                        acc[i] *= up;
                }
            }
            uint4 w[SUB / 2][LIMBS];
#pragma unroll
            for (int k = 0; k < SUB / 2; k++)
                limbs_of<TYPE>(x + 8 * k, w[k]);
            const auto turned = [](const uint32_t(*v)[VW], int e) {
                const uint32_t pick = e & 1 ? 0x07060302u : 0x05040100u;
                return uint4{__builtin_amdgcn_perm(v[1][e / 2], v[0][e / 2], pick), __builtin_amdgcn_perm(v[3][e / 2], v[2][e / 2], pick),
                             __builtin_amdgcn_perm(v[5][e / 2], v[4][e / 2], pick), __builtin_amdgcn_perm(v[7][e / 2], v[6][e / 2], pick)};
            };
            /* values that no row of the tile sees are 0: 0 times an infinite or NaN one would be NaN */
            uint32_t size = 0;
#pragma unroll
            for (int r = 0; r < 4 * SUB; r++) {
                const bool hide = !whole && (place(r) > u.last || passed<WINDOW>(p, place(r), u.lo0));
#pragma unroll
                for (int i = 0; i < NV; i++)
#pragma unroll
                    for (int e = 0; e < VW; e++) {
                        vw[i][r][e] = hide ? 0 : vw[i][r][e];
                        size = larger(size, vw[i][r][e]);
                    }
            }
            const bool odd_values = __ballot((size & 0xffffu) >= H::INF || size >> 16 >= H::INF);
            if (!odd_values) {
#pragma unroll
                for (int i = 0; i < NV; i++)
#pragma unroll
                    for (int e = 0; e < VEC; e++) {
#pragma unroll
                        for (int k = 0; k < SUB / 2; k++) {
                            const uint4 v = turned(vw[i] + 8 * k, e);
#pragma unroll
                            for (int n = 0; n < LIMBS; n++)
                                acc[i * VEC + e] = H::mfma(v, w[k][n], acc[i * VEC + e]);
                        }
                        if (e & 1)
                            __builtin_amdgcn_sched_barrier(0);
                    }
            }
            if (!odd_values && !apart) {
                if (TYPE == RT_F16 && small)
#pragma unroll
                    for (int i = 0; i < VE; i++)
                        acc[i] *= down;
                continue;
            }
            for (int pass = 0;; pass++) {
                if (odd_values || pass > 0) {
                    /* with values that are not finite each token's rows are computed apart, without the values that it does not see.
                     * The values are loaded again, so that the fast path keeps its registers */
                    uint4 seen[SUB / 2]; /* F16: 1 where there is a weight */
                    if constexpr (TYPE == RT_F16)
#pragma unroll
                        for (int k = 0; k < SUB / 2; k++) {
                            uint32_t one[8];
#pragma unroll
                            for (int e = 0; e < 8; e++) {
                                const float at = apart ? kept[64 * (8 * k + e)] : limb(w[k][0], e);
                                one[e] = H::round(at > 0.0f ? 1.0f : at);
                            }
                            seen[k] = uint4{one[0] | one[1] << 16, one[2] | one[3] << 16, one[4] | one[5] << 16, one[6] | one[7] << 16};
                        }
                    for (int jj = odd_values ? u.j0 : u.j1; jj <= u.j1; jj++) {
                        const long upto = (long)u.q.past + jj < u.last ? (long)u.q.past + jj : u.last;
                        const int from = !WINDOW ? 0 : odd_values ? window_from(p, u.q, jj) : u.lo0;
#pragma unroll
                        for (int k = 0; k < SUB / 2; k++)
#pragma unroll
                            for (int i = 0; i < NV; i++) {
                                uint32_t again[8][VW];
#pragma unroll
                                for (int r = 0; r < 8; r++) {
                                    load_words<VW>(again[r], address(kv.v, rows[8 * k + r], head_rows, D * 2) + (i * 16 + c) * VEC * 2);
                                    const bool hide = place(8 * k + r) > upto || passed<WINDOW>(p, place(8 * k + r), from);
#pragma unroll
                                    for (int e = 0; e < VW; e++)
                                        again[r][e] = hide ? 0 : again[r][e];
                                }
#pragma unroll
                                for (int e = 0; e < VEC; e++) {
                                    const uint4 v = turned(again, e), part = finite_only<TYPE>(v);
                                    v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                                    for (int n = 0; n < LIMBS; n++)
                                        o = H::mfma(TYPE == RT_F16 || n ? part : v, w[k][n], o);
                                    if (TYPE == RT_F16 && pass == 0)
                                        o = H::mfma(without(v, part), seen[k], o);
                                    if (!odd_values || u.j == jj)
                                        acc[i * VEC + e] += o;
                                    __builtin_amdgcn_sched_barrier(0);
                                }
                                asm volatile("" ::: "memory"); /* the loads stay in the loop, and out of registers */
                            }
                    }
                }
                if (TYPE != RT_F16)
                    break;
                if (!apart) {
#pragma unroll
                    for (int i = 0; i < VE; i++)
                        acc[i] *= down;
                    break;
                }
                bool more = false; /* the limbs leave something of a weight that counts */
#pragma unroll
                for (int k = 0; k < SUB / 2; k++) {
                    float next[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float had = kept[64 * (8 * k + e)];
                        float left = had;
#pragma unroll
                        for (int n = 0; n < LIMBS; n++)
                            left -= limb(w[k][n], e);
                        const bool counts = fabsf(left) > 0x1p-22f * fabsf(had);
                        more |= counts;
                        next[e] = counts ? left * 0x1p38f : 0.0f;
                        kept[64 * (8 * k + e)] = next[e];
                    }
                    limbs_of<TYPE>(next, w[k]);
                }
                const bool done = pass == 5 || !__ballot(more);
#pragma unroll
                for (int i = 0; i < VE; i++) {
                    const v4f sum = kept_acc[64 * i] + acc[i] * down;
                    kept_acc[64 * i] = sum;
                    acc[i] = done ? sum : v4f{0.0f, 0.0f, 0.0f, 0.0f};
                }
                if (done)
                    break;
                down *= 0x1p-38f;
            }
        }
        finish<D, VEC>(lds, kv, a, p, u, number, m, l, acc);
    }
}

/* A query row's chunks joined, 64 elements of it a workgroup, 16 threads an element: each takes every 16th chunk,
 * loading its elements and its maximum and sum at once, with a running maximum of its own; then the 16 are scaled
 * to the largest and added in one order. Bound by the latency of its few dependent loads. */
__global__ __launch_bounds__(256) void attn_join_k(rt_seqs b, rt_kv kv, rt_attn a, plan p)
{
    __shared__ __align__(16) float4 so[16][16];
    __shared__ float sm[16], sl[16];
    const int at = threadIdx.x & 15, turn = threadIdx.x >> 4;
    const long D = kv.dim, d = 64 * (long)blockIdx.z + 4 * at, dd = d < D ? d : 0;
    const float4 gate = gate_of(a, blockIdx.x, blockIdx.y, dd);
    const long i = blockIdx.x, h = blockIdx.y;
    int s, before, chunk;
    seq_plan q;
    if (!locate<true>(b, p, p.heads, -1, i, s, q, before, chunk) || q.chunks == 1)
        return;
    const int kh = (int)p.group.of((uint32_t)h), row = (int)(i - q.first) * p.heads + (int)h - kh * p.heads, rows = 1 << p.shift,
              z = q.rows - 1 - (row >> p.shift), r = row & (rows - 1);
    if ((long)before + (long)(z + 1) * q.chunks > p.slots)
        return;
    const long slot = (long)kh * p.slots + before + z * q.chunks;
    const float *ml = p.part + kv.heads * p.slots * rows * D + (slot * rows + r) * 2, *part = p.part + (slot * rows + r) * D + dd;
    float4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    for (int k0 = turn; k0 < q.chunks; k0 += 64) {
        float2 x[4];
        float4 w[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int at_chunk = k0 + 16 * k < q.chunks ? k0 + 16 * k : k0;
            x[k] = *(const float2 *)(ml + (long)at_chunk * (2 * rows));
            w[k] = *(const float4 *)(part + (long)at_chunk * rows * D);
        }
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (k0 + 16 * k < q.chunks) {
                /* a chunk whose maximum is -infinity holds zeros, or NaN: taken as it is */
                const float top = fmaxf(m, x[k].x), f = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - top),
                            e = x[k].x == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(x[k].x - top);
                v = float4{fmaf(w[k].x, e, v.x * f), fmaf(w[k].y, e, v.y * f), fmaf(w[k].z, e, v.z * f), fmaf(w[k].w, e, v.w * f)};
                l = fmaf(x[k].y, e, l * f);
                m = top;
            }
    }
    so[turn][at] = v;
    if (at == 0)
        sm[turn] = m, sl[turn] = l;
    __syncthreads();
    if (turn == 0 && d < D) {
        float top = sm[0], sum = 0.0f;
        for (int k = 1; k < 16; k++)
            top = fmaxf(top, sm[k]);
        v = float4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int k = 0; k < 16; k++) {
            const float f = sm[k] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(sm[k] - top);
            const float4 x = so[k][at];
            v = float4{fmaf(x.x, f, v.x), fmaf(x.y, f, v.y), fmaf(x.z, f, v.z), fmaf(x.w, f, v.w)};
            sum = fmaf(sl[k], f, sum);
        }
        store_row(a, D, i, h, d, v, sum, (long)q.past + (i - q.first) < 0, gate);
    }
}

/* The same for prompts: a workgroup a chunk, as the chunks were computed, each with its part of the row tile's rows, so that a launch
 * of many row tiles of which few or none were cut is few workgroups (8192 tokens of 16 heads of 256, none cut: 486 us with a
 * workgroup for each token, head and 64 elements). 4 elements of a row a thread, 4 chunks' loads at once, one behind the other: few
 * rows on a long history, a row tile of hundreds of chunks, wait for them (8 tokens of 8 heads of 128 on one at 100000 positions: 81 us of
 * 103; 3 tokens, which the other join has, 23 in all). */
__global__ __launch_bounds__(256) void attn_join_rows_k(rt_seqs b, rt_kv kv, rt_attn a, plan p)
{
    int s, before, chunk, number = (int)blockIdx.x;
    seq_plan q;
    if (!locate<true>(b, p, p.heads, number, 0, s, q, before, chunk) || q.chunks == 1)
        return;
    const int at = number - before, z = at / q.chunks, part = at - z * q.chunks, rows = 1 << p.shift, first = (q.rows - 1 - z) << p.shift;
    if ((long)before + (long)(z + 1) * q.chunks > p.slots)
        return;
    const int D = (int)kv.dim, per = 256 / (D / 4), mine = (int)threadIdx.x / (D / 4), d = 4 * ((int)threadIdx.x - mine * (D / 4));
    const int live = q.n * p.heads - first < rows ? q.n * p.heads - first : rows, r1 = (int)((long)live * (part + 1) / q.chunks);
    const long slot = (long)blockIdx.y * p.slots + before + z * q.chunks;
    if (mine >= per)
        return;
    for (int r = (int)((long)live * part / q.chunks) + mine; r < r1; r += per) {
        const float *ml = p.part + kv.heads * p.slots * rows * D + (slot * rows + r) * 2, *v = p.part + (slot * rows + r) * D + d;
        const int j = (int)p.group.of(first + r), h = (int)blockIdx.y * p.heads + (first + r - j * p.heads);
        const float4 gate = gate_of(a, q.first + j, h, d);
        float4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
        float m = -INFINITY, l = 0.0f;
        for (int k0 = 0; k0 < q.chunks; k0 += 4) {
            float2 x[4];
            float4 w[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const long i = k0 + k < q.chunks ? k0 + k : k0;
                x[k] = *(const float2 *)(ml + i * (2 * rows));
                w[k] = *(const float4 *)(v + i * rows * D);
            }
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (k0 + k < q.chunks) {
                    /* a chunk whose maximum is -infinity holds zeros, or NaN: taken as it is */
                    const float top = fmaxf(m, x[k].x), f = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - top),
                                e = x[k].x == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(x[k].x - top);
                    sum = float4{fmaf(w[k].x, e, sum.x * f), fmaf(w[k].y, e, sum.y * f), fmaf(w[k].z, e, sum.z * f), fmaf(w[k].w, e, sum.w * f)};
                    l = fmaf(x[k].y, e, l * f);
                    m = top;
                }
        }
        store_row(a, D, q.first + j, h, d, sum, l, (long)q.past + j < 0, gate);
    }
}

template <int TYPE, bool WINDOW>
void launch(hipStream_t s, dim3 grid, const rt_seqs &b, const rt_kv &kv, const rt_attn &a, const plan &p)
{
    switch (kv.dim) {
#define DIM(D)                                                                                                                                             \
    case D:                                                                                                                                                \
        if constexpr (TYPE == RT_F32)                                                                                                                      \
            attn_f32_k<D, WINDOW><<<grid, 64 * WAVES, 0, s>>>(b, kv, a, p);                                                                                \
        else                                                                                                                                               \
            attn_half_k<D, TYPE, WINDOW><<<grid, 64 * WAVES, 0, s>>>(b, kv, a, p);                                                                         \
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

/* Row tiles of a call at most, and the chunks (a key-value head) to spread them over: so many that with each
 * row tile's last one, which is smaller, they fill the workgroups that run at once (one or two a compute unit) a
 * whole number of times, at least half of them whole. Runs of tokens (16 a sequence on average) whose row tiles fill them
 * as they are get as few as that: only a much longer one is cut (512 tokens of 32 heads of 128 74 us, 128 with the others'
 * count; 256 single tokens of 100 to 8000 positions 859 us with theirs and 891 with this). None (0) when the row tiles
 * alone are more than SLOTS */
constexpr long SLOTS = 4096;

int tile_of(const rt_kv &kv, int shift) { return kv.type == RT_F32 ? 1 : kv.type == RT_Q8 ? 4 : shift == 6 ? q8_attn_rows_tile(kv.dim) : sixteens(kv.dim); }

/* The positions that the table reaches */
long reach_of(const rt_kv &kv)
{
    const long most = (1L << 31) - 4096;
    return kv.table_ld > most / kv.page ? most : kv.table_ld * kv.page;
}

/* A window that holds all positions is none */
bool cuts(const rt_kv &kv, long window, long sinks) { return window > 0 && window < reach_of(kv) && sinks < reach_of(kv); }

/* Row tiles of 64 (as a shift), where a kernel has them, from 64 rows of the longest sequence and 32 of each on (and as far as their
 * workgroups are one launch) */
int shift_of(const rt_seqs &b, const rt_kv &kv, const rt_attn &a, bool window)
{
    const long group = a.q_heads / kv.heads;
    const bool some = kv.type == RT_Q8 || (window && kv.type != RT_F32), many = b.longest * group >= 64 && b.t * group >= 32 * b.n;
    return some && many && ((b.t * group >> 6) + b.n) * kv.heads < 1L << 23 ? 6 : 4;
}

/* The plan's target, and once (0: chunks of the target's size) */
void plan_chunks(const rt_seqs &b, const rt_kv &kv, const rt_attn &a, long window, long sinks, long &tiles, long &target, long &rounds)
{
    rounds = 0;
    const int shift = shift_of(b, kv, a, cuts(kv, window, sinks));
    tiles = (b.t * (a.q_heads / kv.heads) >> shift) + b.n;
    const bool single = kv.type == RT_F32 ? kv.dim > 128 : kv.type == RT_Q8 ? shift == 4 && q8_attn8_alone(kv.dim) : shift == 4 && alone(kv.dim);
    const long once = ((single ? 256 : 512) + kv.heads - 1) / kv.heads;
    const long most = reach_of(kv), seen = cuts(kv, window, sinks) && window + sinks + 16 < most ? window + sinks + 16 : most;
    if (tiles * kv.heads > SLOTS || seen <= 16 * WAVES * tile_of(kv, shift))
        target = 0;
    else if (b.t >= 16 * b.n && tiles >= once)
        target = once;
    else {
        target = (2 * tiles + once - 1) / once * once - tiles;
        if (shift == 4 && b.n > 1 && (kv.type == RT_Q8 || cuts(kv, window, sinks))) {
            /* (few row tiles fill one round evenly; every workgroup of a launch costs, also one without a chunk) */
            if (tiles <= once) {
                rounds = once;
                target = (4 * tiles <= once ? 1 : 2) * once - tiles;
            }
        }
    }
}

} /* namespace */

long q8_attn_part_floats(const rt_seqs &b, const rt_kv &kv, const rt_attn &a, long window, long sinks)
{
    long tiles, target, rounds;
    plan_chunks(b, kv, a, window, sinks, tiles, target, rounds);
    return target ? (kv.heads * (target + tiles) * (kv.dim + 2) << shift_of(b, kv, a, cuts(kv, window, sinks))) + 4 : 0;
}

void q8_launch_attn(q8_stream_t stream, const rt_seqs &b, const rt_kv &kv, const rt_attn &a, long window, long sinks, float *part)
{
    plan p;
    long tiles, target, rounds;
    plan_chunks(b, kv, a, window, sinks, tiles, target, rounds);
    p.once = (int)rounds;
    p.target = (int)target;
    p.shift = shift_of(b, kv, a, cuts(kv, window, sinks));
    p.tile = tile_of(kv, p.shift);
    p.least = WAVES * p.tile;
    const auto by = [](long d) {
        int up = 0;
        while ((1L << up) < d)
            up++;
        return q8_divisor{(uint32_t)((((__uint128_t)1 << (31 + up)) + d - 1) / d), 31 + up};
    };
    p.heads = (int)(a.q_heads / kv.heads);
    p.page = by(kv.page), p.group = by(p.heads);
    p.share = target ? 1.00001f / (float)target : 0.0f;
    p.cap = (int)reach_of(kv);
    p.window = cuts(kv, window, sinks) ? (int)window : 0;
    p.sinks = p.window ? (int)sinks : 0;
    p.slots = (int)(target + (target ? tiles : 0));
    p.part = part;
    p.size = (int *)(part + (kv.heads * p.slots * (kv.dim + 2) << p.shift)); /* behind the parts */
    p.qscale = (float)((double)a.scale * 1.4426950408889634074);
    const hipStream_t s = (hipStream_t)stream;
    const long n = p.target ? p.slots : p.shift == 6 || tiles < 1L << 20 ? tiles : 1L << 20;
    const dim3 grid((unsigned)n, (unsigned)kv.heads);
    if (kv.type == RT_Q8)
        q8_launch_attn8(stream, n, b, kv, a, p);
    else if (p.shift == 6)
        q8_launch_attn_rows(stream, n, b, kv, a, p);
    else if (kv.type == RT_F32)
        p.window ? launch<RT_F32, true>(s, grid, b, kv, a, p) : launch<RT_F32, false>(s, grid, b, kv, a, p);
    else if (kv.type == RT_F16)
        p.window ? launch<RT_F16, true>(s, grid, b, kv, a, p) : launch<RT_F16, false>(s, grid, b, kv, a, p);
    else
        p.window ? launch<RT_BF16, true>(s, grid, b, kv, a, p) : launch<RT_BF16, false>(s, grid, b, kv, a, p);
    if (p.target && (kv.type == RT_Q8 || p.window) && b.t * p.heads >= 32 * b.n)
        attn_join_rows_k<<<grid, 256, 0, s>>>(b, kv, a, p);
    else if (p.target)
        attn_join_k<<<dim3((unsigned)b.t, (unsigned)a.q_heads, (unsigned)((kv.dim + 63) / 64)), 256, 0, s>>>(b, kv, a, p);
}
