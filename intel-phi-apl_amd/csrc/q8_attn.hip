/* q8_attn.hip: attention of new tokens over the paged key-value cache (include/q8_mix.h). */
#include "q8_mix.h"

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int WAVES = 4;
constexpr int LEAST = WAVES; /* tiles a chunk at least: one a wave */

/* p / page for p < 2^31: (p * mul) >> shift with shift = 31 + ceil(log2 page), mul = ceil(2^shift / page): exact, as
 * the excess mul * page - 2^shift is below page <= 2^(shift - 31) */
struct paging {
    uint32_t mul;
    int shift;
};

/* What a launch shares: row tiles are 16 query rows (token, head of the group) of one key-value head and
 * sequence; a sequence's positions, in tiles of 16, are cut into chunks of one size for the whole batch. */
struct plan {
    paging pg;
    int group;     /* query heads a key-value head */
    long cap;      /* positions that the table reaches */
    long target;   /* chunks (a key-value head) to spread all tiles over; 0: one a row tile */
    long slots;    /* partial results a key-value head */
    float *part;   /* [heads][slots][16][dim], then [heads][slots][16][2]: maximum and sum */
    float qscale;  /* scale * log2 e: scores are in powers of two */
};

struct seq_plan {
    long first, n;      /* its rows of the token-major arrays */
    long past, tiles;   /* position tiles of all it sees, within the table */
    long rows, chunks;  /* row tiles, and chunks of each */
};

__device__ __forceinline__ seq_plan plan_of(const rt_seqs &b, const plan &p, long s, long chunk)
{
    seq_plan q;
    long last;
    q8_rows_of(b, s, q.first, last);
    q.n = last - q.first;
    q.past = b.past[s];
    const long len = q.past + q.n;
    q.tiles = len <= 0 ? 0 : ((len < p.cap ? len : p.cap) + 15) / 16;
    q.rows = (q.n * p.group + 15) / 16;
    q.chunks = chunk > 0 && q.tiles > chunk ? (q.tiles + chunk - 1) / chunk : 1;
    return q;
}

__device__ __forceinline__ long wave_sum(long v)
{
    for (int o = 32; o >= 1; o >>= 1)
        v += __shfl_xor(v, o, 64);
    return v;
}

/* tiles a chunk: every sequence's tiles over the target, the same for each of them, so that workgroups
 * read the same amounts whatever the lengths (a share of each sequence's own length left the short ones'
 * workgroups waiting for the longest) */
__device__ __forceinline__ long chunk_of(const rt_seqs &b, const plan &p)
{
    if (p.target <= 0)
        return 0;
    long all = 0;
    for (long s = threadIdx.x & 63; s < b.n; s += 64) {
        const seq_plan q = plan_of(b, p, s, 0);
        all += q.rows * q.tiles;
    }
    if (b.n > 1)
        all = wave_sum(all);
    else
        all = __shfl(all, 0, 64);
    const long c = (all + p.target - 1) / p.target;
    return c < LEAST ? LEAST : c;
}

/* The sequence whose row tiles' chunks hold number i of all, -1 behind the last; before = the chunks of
 * those before it */
__device__ __forceinline__ long sequence_of_chunk(const rt_seqs &b, const plan &p, long chunk, long i, long &before)
{
    const int lane = threadIdx.x & 63;
    before = 0;
    for (long s0 = 0; s0 < b.n; s0 += 64) {
        long c = 0;
        if (s0 + lane < b.n) {
            const seq_plan q = plan_of(b, p, s0 + lane, chunk);
            c = q.rows * q.chunks;
        }
        long upto = c;
        if (b.n > 1)
            for (int o = 1; o < 64; o <<= 1) {
                const long u = __shfl_up(upto, o, 64);
                upto += lane >= o ? u : 0;
            }
        const unsigned long long m = __ballot(i < before + upto);
        if (m) {
            const int at = __ffsll((long long)m) - 1;
            before += __shfl(upto - c, at, 64);
            return s0 + at;
        }
        before += __shfl(upto, 63, 64);
    }
    return -1;
}

template <int TYPE>
struct elem {
    static constexpr int bytes = TYPE == RT_F32 ? 4 : 2;
};

/* element e of 32-bit words w, in F32 (exact) */
template <int TYPE>
__device__ __forceinline__ float element(const uint32_t *w, int e)
{
    if constexpr (TYPE == RT_F32)
        return __builtin_bit_cast(float, w[e]);
    else if constexpr (TYPE == RT_F16)
        return (float)__builtin_bit_cast(_Float16, (uint16_t)(w[e / 2] >> (16 * (e & 1))));
    else
        return __builtin_bit_cast(float, e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
}

template <int WORDS>
__device__ __forceinline__ void load_words(uint32_t *w, const char *p)
{
    if constexpr (WORDS == 4)
        *(uint4 *)w = *(const uint4 *)p;
    else if constexpr (WORDS == 2)
        *(uint2 *)w = *(const uint2 *)p;
    else
        *w = *(const uint32_t *)p;
}

/* the largest of a value's copies in lanes l, l ^ 16, l ^ 32, l ^ 48, and their sum */
__device__ __forceinline__ float group_max(float v)
{
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float group_sum(float v)
{
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

/* o's final form: the gate, and what a row that sees nothing gives */
__device__ __forceinline__ void store_row(const rt_attn &a, long dim, long token, long head, long at, float4 v, float l, bool empty)
{
    v = empty ? float4{0.0f, 0.0f, 0.0f, 0.0f} : float4{v.x / l, v.y / l, v.z / l, v.w / l};
    if (a.gate) {
        const float4 g = *(const float4 *)(a.gate + token * a.gate_ld + head * a.gate_hd + at);
        v = float4{v.x * q8_sigmoid(g.x), v.y * q8_sigmoid(g.y), v.z * q8_sigmoid(g.z), v.w * q8_sigmoid(g.w)};
    }
    *(float4 *)(a.o + token * a.o_ld + head * dim + at) = v;
}

/* A workgroup takes a chunk of positions for a row tile; its waves take the chunk's position tiles in
 * turn, and join at the end through LDS.
 *
 * Per tile of 16 positions a wave computes S^T = K Q^T (v_mfma_f32_16x16x4_f32: K's rows are the
 * positions), so that lane 16 g + c has the scores of query row c at positions 4 g .. 4 g + 3, which is how the
 * next product wants its second operand: O^T += V^T P^T takes them as they are, position 4 g + r in its step
 * r. So nothing passes through LDS, and the cache's rows go from memory to the matrix cores in the registers that
 * they were loaded into: lane 16 g + c loads K's row c, 16 bytes of each 64 from byte 16 g on, and V's rows 4 g ..
 * 4 g + 3, elements c * VEC .. of each 16 * VEC. The products are F32 whatever the cache's type.
 *
 * The softmax's maximum is a running one that is raised only when a score passes it by more than SLACK (a
 * power of two: the exponentials stay below 2^SLACK): then the sums and outputs are scaled, which a tile
 * rarely needs after the first. Each lane sums its own positions; the four lanes of a row add up at the end. */
constexpr float SLACK = 8.0f;

template <int D, int TYPE>
__global__ __launch_bounds__(64 * WAVES, D *elem<TYPE>::bytes > 512 ? 1 : 2) void attn_tile_k(rt_seqs b, rt_kv kv, rt_attn a, plan p)
{
    constexpr int SIZE = elem<TYPE>::bytes, E = 16 / SIZE, NK = D / (4 * E);
    constexpr int VE = D / 16, VEC = VE % E == 0 ? E : VE % (E / 2) == 0 ? E / 2 : 2, NV = VE / VEC, VW = VEC * SIZE / 4;
    constexpr int LD = D + 4; /* rows of the waves' outputs in LDS, off each other's banks */
    __shared__ __align__(16) float so[WAVES][16][LD];
    __shared__ float sm[WAVES][16], sl[WAVES][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, g = lane >> 4;
    const long kh = blockIdx.y, chunk = chunk_of(b, p);
    const long head_rows = kh * kv.page, page_rows = kv.heads * kv.page;
    /* with starts that overlap there may be more chunks than slots: those are left out */
    for (long number = blockIdx.x; p.target == 0 || number < p.slots; number += gridDim.x) {
        long before;
        const long s = sequence_of_chunk(b, p, chunk, number, before);
        if (s < 0)
            return;
        const seq_plan q = plan_of(b, p, s, chunk);
        const long z = (number - before) / q.chunks, part = (number - before) % q.chunks;
        const int32_t *table = kv.table + s * kv.table_ld;
        /* this lane's query row: token j of the sequence, head h; it sees positions up to lim */
        const long row = z * 16 + c, j = row / p.group, h = kh * p.group + row % p.group;
        const bool live = j < q.n;
        const long seen = q.past + j;
        const int lim = !live || seen < 0 ? -1 : (int)(seen < p.cap ? seen : p.cap - 1);
        const long j0 = z * 16 / p.group, j1 = (z * 16 + 15) / p.group < q.n ? (z * 16 + 15) / p.group : q.n - 1; /* the row tile's tokens */
        const long end = q.past + j1 < p.cap ? q.past + j1 : p.cap - 1;
        const int last = (int)(end < -1 ? -1 : end); /* the last position that any row sees */
        const int least = (int)(q.past + j0 < -1 ? -1 : q.past + j0 > last ? last : q.past + j0); /* every row sees up to here */
        const long t0 = part * chunk, t1 = last < 0 ? 0 : last / 16 + 1;
        const int stop = (int)(q.chunks > 1 && t0 + chunk < t1 ? t0 + chunk : t1);

        float qv[NK * E];
#pragma unroll
        for (int i = 0; i < NK; i++)
#pragma unroll
            for (int e = 0; e < E; e += 4) {
                float4 v = {0.0f, 0.0f, 0.0f, 0.0f};
                if (live)
                    v = *(const float4 *)(a.q + (q.first + j) * a.q_ld + h * a.q_hd + (i * 4 + g) * E + e);
                qv[i * E + e] = v.x * p.qscale, qv[i * E + e + 1] = v.y * p.qscale, qv[i * E + e + 2] = v.z * p.qscale, qv[i * E + e + 3] = v.w * p.qscale;
            }
        v4f acc[VE];
#pragma unroll
        for (int i = 0; i < VE; i++)
            acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        float m = -INFINITY, l = 0.0f;

        /* a position's row in the cache's k and v, counted from the head's first page, or -1 where there is
         * none; entry: its page from the table, loaded a tile ahead */
        const auto entry_of = [&](int pos) {
            const uint32_t pg = (uint32_t)(((uint64_t)(uint32_t)pos * p.pg.mul) >> p.pg.shift);
            return (long)pg < kv.table_ld ? table[pg] : -1;
        };
        const auto row_of = [&](int pos, int entry) {
            const uint32_t pg = (uint32_t)(((uint64_t)(uint32_t)pos * p.pg.mul) >> p.pg.shift);
            return entry >= 0 && entry < kv.pages ? (int)(entry * page_rows + (pos - (long)pg * kv.page)) : -1;
        };
        const auto at = [&](const void *cache, int r) { return (const char *)cache + (size_t)((r < 0 ? 0 : r) + head_rows) * (D * SIZE); };
        const auto here = [&](int tile) { return tile * 16 + c < last ? tile * 16 + c : last; };

        uint32_t kw[NK][4], vw[4][NV][VW];
        int tile = (int)t0 + wave, row_now = -1, entry = -1;
        if (tile < stop) {
            row_now = row_of(here(tile), entry_of(here(tile)));
            entry = entry_of(here(tile + WAVES));
#pragma unroll
            for (int i = 0; i < NK; i++)
                load_words<4>(kw[i], at(kv.k, row_now) + (i * 4 + g) * 16);
        }
        for (; tile < stop; tile += WAVES) {
            int rows[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                rows[r] = __shfl(row_now, 4 * g + r, 64);
#pragma unroll
                for (int i = 0; i < NV; i++)
                    load_words<VW>(vw[r][i], at(kv.v, rows[r]) + (i * 16 + c) * VEC * SIZE);
            }
            v4f s2[2] = {v4f{0.0f, 0.0f, 0.0f, 0.0f}, v4f{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
            for (int i = 0; i < NK; i++)
#pragma unroll
                for (int e = 0; e < E; e++)
                    s2[e & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(element<TYPE>(kw[i], e), qv[i * E + e], s2[e & 1], 0, 0, 0);
            if (tile + WAVES < stop) {
                row_now = row_of(here(tile + WAVES), entry);
                entry = entry_of(here(tile + 2 * WAVES));
#pragma unroll
                for (int i = 0; i < NK; i++)
                    load_words<4>(kw[i], at(kv.k, row_now) + (i * 4 + g) * 16);
            }
            float x[4];
            const bool whole = tile * 16 + 15 <= least; /* every row sees every position of the tile */
#pragma unroll
            for (int r = 0; r < 4; r++) {
                x[r] = rows[r] < 0 ? NAN : s2[0][r] + s2[1][r];
                if (!whole && tile * 16 + 4 * g + r > lim)
                    x[r] = -INFINITY;
            }
            const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
            if (__ballot(top > m + SLACK)) {
                const float raised = fmaxf(m, group_max(top)), f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - raised);
                m = raised;
                l *= f;
#pragma unroll
                for (int i = 0; i < VE; i++)
                    acc[i] *= f;
            }
            const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                x[r] = __builtin_amdgcn_exp2f(x[r] - ref);
                l += x[r];
            }
            if (whole) {
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int i = 0; i < NV; i++)
#pragma unroll
                        for (int e = 0; e < VEC; e++)
                            acc[i * VEC + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(element<TYPE>(vw[r][i], e), x[r], acc[i * VEC + e], 0, 0, 0);
            } else {
                /* positions that some of the rows do not see: 0 times an infinite or NaN value would be NaN,
                 * so each token's rows are computed apart, without the values behind it */
                for (long jj = j0; jj <= j1; jj++) {
                    const long upto = q.past + jj;
#pragma unroll
                    for (int i = 0; i < NV; i++)
#pragma unroll
                        for (int e = 0; e < VEC; e++) {
                            v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                const bool sees = tile * 16 + 4 * g + r <= upto && tile * 16 + 4 * g + r <= last;
                                o = __builtin_amdgcn_mfma_f32_16x16x4f32(sees ? element<TYPE>(vw[r][i], e) : 0.0f, x[r], o, 0, 0, 0);
                            }
                            if (j == jj)
                                acc[i * VEC + e] += o;
                        }
                }
            }
        }

        /* the waves' results, scaled to the largest of their maxima, added in the waves' order */
        l = group_sum(l);
        if (g == 0)
            sm[wave][c] = m, sl[wave][c] = l;
        __syncthreads();
        float top = sm[0][c];
#pragma unroll
        for (int w = 1; w < WAVES; w++)
            top = fmaxf(top, sm[w][c]);
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int e = 0; e < VEC; e += 2)
                    *(float2 *)&so[wave][c][(i * 16 + 4 * g + r) * VEC + e] = float2{acc[i * VEC + e][r] * f, acc[i * VEC + e + 1][r] * f};
        __syncthreads();
        const long left = q.n * p.group - z * 16;
        const int rows_here = (int)(left < 16 ? left : 16);
        for (int i = tid; i < rows_here * (D / 4); i += 64 * WAVES) {
            const int r = i / (D / 4), d = 4 * (i % (D / 4));
            float t = sm[0][r], sum = 0.0f;
            for (int w = 1; w < WAVES; w++)
                t = fmaxf(t, sm[w][r]);
            float4 v = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int w = 0; w < WAVES; w++) {
                const float4 u = *(const float4 *)&so[w][r][d];
                v = float4{v.x + u.x, v.y + u.y, v.z + u.z, v.w + u.w};
                sum += sl[w][r] * (sm[w][r] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(sm[w][r] - t));
            }
            const long jr = (z * 16 + r) / p.group, hr = kh * p.group + (z * 16 + r) % p.group, pos = q.past + jr;
            if (pos >= p.cap)
                sum = NAN; /* a position that the table does not reach */
            if (q.chunks == 1) {
                store_row(a, D, q.first + jr, hr, d, v, sum, pos < 0);
            } else {
                const long slot = kh * p.slots + number;
                *(float4 *)(p.part + (slot * 16 + r) * D + d) = v;
                if (d == 0)
                    *(float2 *)(p.part + kv.heads * p.slots * 16 * D + (slot * 16 + r) * 2) = float2{t, sum};
            }
        }
        __syncthreads();
    }
}

/* A query row's chunks joined: each scaled to the largest maximum, added wave by wave and then over the
 * waves, in one order. */
__global__ __launch_bounds__(64 * WAVES) void attn_join_k(rt_seqs b, rt_kv kv, rt_attn a, plan p)
{
    __shared__ __align__(16) float4 so[WAVES][64];
    const long i = blockIdx.x, h = blockIdx.y, s = q8_sequence_of(b, i);
    if (s < 0)
        return;
    const long chunk = chunk_of(b, p);
    const seq_plan q = plan_of(b, p, s, chunk);
    if (q.chunks == 1)
        return;
    long before = 0;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (long k = lane; k < s; k += 64) {
        const seq_plan o = plan_of(b, p, k, chunk);
        before += o.rows * o.chunks;
    }
    before = wave_sum(before);
    const long kh = h / p.group, row = (i - q.first) * p.group + h % p.group, z = row / 16, r = row % 16;
    if (before + (z + 1) * q.chunks > p.slots)
        return;
    const long slot = kh * p.slots + before + z * q.chunks, D = kv.dim;
    const float *ml = p.part + kv.heads * p.slots * 16 * D;
    float top = -INFINITY;
    for (long k = lane; k < q.chunks; k += 64)
        top = fmaxf(top, ml[((slot + k) * 16 + r) * 2]);
    for (int o = 32; o >= 1; o >>= 1)
        top = fmaxf(top, __shfl_xor(top, o, 64));
    float sum = 0.0f;
    for (long k = lane; k < q.chunks; k += 64) {
        const float2 v = *(const float2 *)(ml + ((slot + k) * 16 + r) * 2);
        sum += v.y * (v.x == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(v.x - top));
    }
    sum = q8_wave_sum(sum);
    float4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (4 * lane < D)
#pragma unroll 4
        for (long k = wave; k < q.chunks; k += WAVES) {
            const float x = ml[((slot + k) * 16 + r) * 2], f = x == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(x - top);
            const float4 u = *(const float4 *)(p.part + ((slot + k) * 16 + r) * D + 4 * lane);
            v = float4{fmaf(u.x, f, v.x), fmaf(u.y, f, v.y), fmaf(u.z, f, v.z), fmaf(u.w, f, v.w)};
        }
    so[wave][lane] = v;
    __syncthreads();
    if (wave == 0 && 4 * lane < D) {
        for (int w = 1; w < WAVES; w++) {
            const float4 u = so[w][lane];
            v = float4{v.x + u.x, v.y + u.y, v.z + u.z, v.w + u.w};
        }
        store_row(a, D, i, h, 4 * lane, v, sum, false);
    }
}

template <int TYPE>
void launch(hipStream_t s, dim3 grid, const rt_seqs &b, const rt_kv &kv, const rt_attn &a, const plan &p)
{
    switch (kv.dim) {
#define DIM(D)                                                                                                                                             \
    case D:                                                                                                                                                \
        attn_tile_k<D, TYPE><<<grid, 64 * WAVES, 0, s>>>(b, kv, a, p);                                                                                     \
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

/* Enough chunks for two workgroups a compute unit twice over, so that the last ones to end leave few idle */
constexpr long CHUNKS = 1024, SLOTS = 4096;

/* Row tiles of a call at most, and the chunks to spread them over: none when there are as many row tiles as chunks
 * would fill SLOTS with, else at least as many as row tiles */
void plan_chunks(const rt_seqs &b, const rt_kv &kv, const rt_attn &a, long &tiles, long &target)
{
    tiles = b.t * (a.q_heads / kv.heads) / 16 + b.n;
    const long want = (CHUNKS + kv.heads - 1) / kv.heads;
    target = tiles * kv.heads > SLOTS || kv.table_ld * kv.page <= 16 * LEAST ? 0 : tiles > want ? tiles : want;
}

} /* namespace */

long q8_attn_part_floats(const rt_seqs &b, const rt_kv &kv, const rt_attn &a)
{
    long tiles, target;
    plan_chunks(b, kv, a, tiles, target);
    return target ? kv.heads * (target + tiles) * 16 * (kv.dim + 2) : 0;
}

void q8_launch_attn(q8_stream_t stream, const rt_seqs &b, const rt_kv &kv, const rt_attn &a, float *part)
{
    plan p;
    long tiles;
    plan_chunks(b, kv, a, tiles, p.target);
    int up = 0;
    while ((1L << up) < kv.page)
        up++;
    p.pg.shift = 31 + up;
    p.pg.mul = (uint32_t)((((__uint128_t)1 << p.pg.shift) + kv.page - 1) / kv.page);
    p.group = (int)(a.q_heads / kv.heads);
    const long reach = (1L << 31) - 4096;
    p.cap = kv.table_ld > reach / kv.page ? reach : kv.table_ld * kv.page;
    p.slots = p.target + tiles;
    p.part = part;
    p.qscale = (float)((double)a.scale * 1.4426950408889634074);
    const hipStream_t s = (hipStream_t)stream;
    const long n = p.target ? p.slots : tiles < 1L << 20 ? tiles : 1L << 20;
    const dim3 grid((unsigned)n, (unsigned)kv.heads);
    if (kv.type == RT_F32)
        launch<RT_F32>(s, grid, b, kv, a, p);
    else if (kv.type == RT_F16)
        launch<RT_F16>(s, grid, b, kv, a, p);
    else
        launch<RT_BF16>(s, grid, b, kv, a, p);
    if (p.target)
        attn_join_k<<<dim3((unsigned)b.t, (unsigned)a.q_heads), 64 * WAVES, 0, s>>>(b, kv, a, p);
}
