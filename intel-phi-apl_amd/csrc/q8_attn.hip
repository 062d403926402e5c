/* q8_attn.hip: attention of new tokens over the paged key-value cache (include/q8_mix.h). */
#include "q8_mix.h"

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

constexpr int WAVES = 4;

/* x / d for x < 2^31: (x * mul) >> shift with shift = 31 + ceil(log2 d), mul = ceil(2^shift / d): exact, as the
 * excess mul * d - 2^shift is below d <= 2^(shift - 31) */
struct divisor {
    uint32_t mul;
    int shift;
    __device__ __forceinline__ uint32_t of(uint32_t x) const { return (uint32_t)(((uint64_t)x * mul) >> shift); }
};

/* What a launch shares: row tiles are 16 query rows (token, head of the group) of one key-value head and
 * sequence; a sequence's positions, in tiles of 16, are cut into chunks of one size for the whole batch. */
struct plan {
    divisor page, group; /* by the positions of a page, by the query heads of a key-value head */
    int heads;    /* query heads of a key-value head */
    int cap;      /* positions that the table reaches */
    int tile;     /* 16s of positions that a wave takes at once (a power of two): chunks are whole numbers of them */
    int least;    /* 16s a chunk at least: one tile of each wave */
    int target;   /* chunks (a key-value head) to spread all tiles over; 0: one a row tile */
    int slots;    /* partial results a key-value head */
    float share;  /* 1 / target, and a little: rounded sums must not make a chunk too small */
    float qscale; /* scale * log2 e: scores are in powers of two */
    float *part;  /* [heads][slots][16][dim], then [heads][slots][16][2]: maximum and sum */
};

struct seq_plan {
    int first, n;     /* its rows of the token-major arrays */
    int past, tiles;  /* position tiles of all it sees, within the table */
    int rows, chunks; /* row tiles, and chunks of each */
};

__device__ __forceinline__ seq_plan plan_of(const rt_seqs &b, const plan &p, int group, int s)
{
    seq_plan q;
    long first, last;
    q8_rows_of(b, s, first, last);
    q.first = (int)first;
    q.n = (int)(last - first);
    q.past = b.past[s];
    const long len = (long)q.past + q.n;
    q.tiles = len <= 0 ? 0 : (int)((len < p.cap ? len : p.cap) + 15) / 16;
    q.rows = (int)(((uint32_t)q.n * (uint32_t)group + 15) / 16);
    q.chunks = 1;
    return q;
}

__device__ __forceinline__ int first_lane(int v) { return __builtin_amdgcn_readfirstlane(v); }

/* tiles a chunk, from all sequences' (row tiles x position tiles): the target's share, the same for each sequence, so
 * that workgroups read the same amounts whatever the lengths (a share of each one's own length left the short ones'
 * waiting for the longest). Rounded up, by floats: any size will do that every workgroup finds alike and that leaves no
 * more chunks than slots. 0: a row tile is one chunk. */
__device__ __forceinline__ int chunk_from(const plan &p, float all)
{
    const float c = all * p.share + 1.0f;
    const int n = c < 1e8f ? ((int)c + p.tile - 1) & ~(p.tile - 1) : 0;
    return n == 0 || n > p.least ? n : p.least;
}
/* ceil(tiles / chunk), which is at most a few thousand */
__device__ __forceinline__ int chunks_of(int tiles, int chunk)
{
    if (chunk == 0 || tiles <= chunk)
        return 1;
    int n = (int)((float)tiles * __builtin_amdgcn_rcpf((float)chunk));
    n -= (long)n * chunk >= tiles ? 1 : 0;
    n += (long)n * chunk < tiles ? 1 : 0;
    n += (long)n * chunk < tiles ? 1 : 0;
    return n;
}

/* the sums of a value over the lanes up to each: by 1, 2, 4 and 8 within each 16, then the 16s' last to the next */
#define UPTO(v, ctrl, rows) (v) += __builtin_amdgcn_update_dpp(0, (v), ctrl, rows, 0xf, false)
__device__ __forceinline__ int wave_upto(int v)
{
    UPTO(v, 0x111, 0xf);
    UPTO(v, 0x112, 0xf);
    UPTO(v, 0x114, 0xf);
    UPTO(v, 0x118, 0xf);
    UPTO(v, 0x142, 0xa); /* row_bcast:15 into rows 1 and 3 */
    UPTO(v, 0x143, 0xc); /* row_bcast:31 into rows 2 and 3 */
    return v;
}
#undef UPTO

/* The sequence that holds chunk `number` of all row tiles' (or, with number < 0, row `token`), its plan, and the
 * chunks of the sequences before it; false: there is none. A lane a sequence, 64 at a time. */
__device__ __forceinline__ bool locate(const rt_seqs &b, const plan &p, int group, int number, long token, int &s, seq_plan &q, int &before, int &chunk)
{
    before = 0;
    if (b.n == 1) {
        s = 0;
        q = plan_of(b, p, group, 0);
        chunk = p.target > 0 ? chunk_from(p, (float)q.rows * (float)q.tiles) : 0;
        q.chunks = chunks_of(q.tiles, chunk);
        return number >= 0 ? number < q.rows * q.chunks : token >= q.first && token < q.first + q.n;
    }
    const int lane = threadIdx.x & 63, n = (int)b.n;
    const seq_plan none = {0, 0, 0, 0, 0, 1};
    seq_plan at = lane < n ? plan_of(b, p, group, lane) : none;
    chunk = 0;
    if (p.target > 0) {
        float all = (float)at.rows * (float)at.tiles;
        for (int s0 = 64; s0 < n; s0 += 64)
            if (s0 + lane < n) {
                const seq_plan o = plan_of(b, p, group, s0 + lane);
                all += (float)o.rows * (float)o.tiles;
            }
        chunk = first_lane(chunk_from(p, q8_wave_sum_dpp(all)));
    }
    for (int s0 = 0; s0 < n; s0 += 64) {
        if (s0 > 0)
            at = s0 + lane < n ? plan_of(b, p, group, s0 + lane) : none;
        at.chunks = chunks_of(at.tiles, chunk);
        const int mine = at.rows * at.chunks, upto = wave_upto(mine);
        const unsigned long long m = __ballot(number >= 0 ? number < before + upto : token >= at.first && token < at.first + at.n);
        if (m) {
            const int l = __ffsll((long long)m) - 1;
            const auto from = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
            s = s0 + l;
            before += from(upto - mine);
            q = seq_plan{from(at.first), from(at.n), from(at.past), from(at.tiles), from(at.rows), from(at.chunks)};
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
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

/* The same for values, which a row tile reads once, in whole lines an instruction: not kept in the caches (32 sequences of
 * 100 to 16384 positions 220 us, 234 without; a prompt's row tiles read them again each). A key row's line is read by two
 * instructions, and has to be. */
template <int WORDS>
__device__ __forceinline__ void stream_words(uint32_t *w, const char *p)
{
    typedef uint32_t words __attribute__((ext_vector_type(WORDS)));
    const words x = __builtin_nontemporal_load((const words *)p);
#pragma unroll
    for (int i = 0; i < WORDS; i++)
        w[i] = x[i];
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
__device__ __forceinline__ float4 gate_of(const rt_attn &a, long token, long head, long at)
{
    return a.gate ? *(const float4 *)(a.gate + token * a.gate_ld + head * a.gate_hd + at) : float4{0.0f, 0.0f, 0.0f, 0.0f};
}
__device__ __forceinline__ void store_row(const rt_attn &a, long dim, long token, long head, long at, float4 v, float l, bool empty, float4 g)
{
    v = empty ? float4{0.0f, 0.0f, 0.0f, 0.0f} : float4{v.x / l, v.y / l, v.z / l, v.w / l};
    if (a.gate) {
        v = float4{v.x * q8_sigmoid(g.x), v.y * q8_sigmoid(g.y), v.z * q8_sigmoid(g.z), v.w * q8_sigmoid(g.w)};
    }
    *(float4 *)(a.o + token * a.o_ld + head * dim + at) = v;
}

/* A workgroup takes a chunk of positions for a row tile (16 query rows); its waves take the chunk's position tiles
 * in turn, and join at the end through LDS.
 *
 * A wave computes S^T = K Q^T, K's rows being the positions, so that lane 16 g + c has the scores of query
 * row c at positions 4 g .. 4 g + 3 of 16. The next product, O^T += V^T P^T, takes them as its second operand as
 * they lie, if its first has V's rows in the same order. So the cache's rows go from memory to the matrix cores in
 * the registers that they were loaded into: lane 16 g + c loads K's row c, 16 bytes of each 64 from byte 16 g on,
 * and V's rows 4 g .. 4 g + 3, VEC elements of each 16 * VEC from c * VEC on. The output's element (i * 16 + 4 g + r)
 * * VEC + e of query row c is acc[i * VEC + e][r].
 *
 * The softmax's maximum is a running one that is raised only when a score passes it by more than SLACK (a
 * power of two: the exponentials stay below 2^SLACK; an F16 cache has less, for its weights' range): then the sums and outputs are scaled, which a tile
 * rarely needs after the first. Each lane sums its own positions; the four lanes of a row add up at the end. */
constexpr float SLACK = 8.0f;

/* A workgroup's share: chunk `part` of sequence s's row tile z, and what its lane has of it */
struct share {
    seq_plan q;
    const int32_t *table;
    int z, j0, j1;   /* the row tile, and its tokens */
    int j, h;        /* the lane's query row: token and head */
    bool live;       /* there is one */
    int lim;         /* the last position that the lane's row sees, -1 none */
    int last, least; /* the last that any row of the tile sees, and the last that all do */
    int t0, t1;      /* the chunk's position tiles, 16 each */
};

__device__ __forceinline__ bool share_of(const rt_seqs &b, const rt_kv &kv, const plan &p, int group, int number, share &u)
{
    int before, s, chunk;
    if (!locate(b, p, group, number, 0, s, u.q, before, chunk))
        return false;
    const seq_plan &q = u.q;
    number -= before;
    int z = number;
    if (q.chunks > 1) {
        z = (int)((float)number * __builtin_amdgcn_rcpf((float)q.chunks)); /* below 2^14: one off at most */
        z -= z * q.chunks > number ? 1 : 0;
        z += (z + 1) * q.chunks <= number ? 1 : 0;
    }
    z = first_lane(z);
    const int part = number - z * q.chunks;
    u.z = q.rows - 1 - z; /* those that see most first (8192 tokens of 16 heads of 256 3114 us, 3403 last) */
    const int row = u.z * 16 + (int)(threadIdx.x & 15);
    u.table = kv.table + s * kv.table_ld;
    u.j = (int)p.group.of(row);
    u.h = (int)blockIdx.y * group + (row - u.j * group);
    u.live = u.j < q.n;
    const auto sees = [&](int j) { /* the last position that token j sees, within the table */
        const long pos = (long)q.past + j;
        return pos < 0 ? -1 : pos < p.cap ? (int)pos : p.cap - 1;
    };
    u.lim = u.live ? sees(u.j) : -1;
    u.j0 = first_lane((int)p.group.of(u.z * 16));
    u.j1 = first_lane((int)p.group.of(u.z * 16 + 15));
    u.j1 = u.j1 < q.n ? u.j1 : q.n - 1;
    u.last = sees(u.j1);
    u.least = sees(u.j0);
    u.t0 = part * chunk;
    u.t1 = u.last < 0 ? 0 : u.last / 16 + 1;
    if (q.chunks > 1 && u.t0 + chunk < u.t1)
        u.t1 = u.t0 + chunk;
    return true;
}

/* A position's page from the table, and its row in the cache's k and v counted from the head's first page
 * (-1: it has none) */
__device__ __forceinline__ int entry_of(const rt_kv &kv, const plan &p, const int32_t *table, int pos)
{
    const uint32_t pg = p.page.of(pos);
    return (long)pg < kv.table_ld ? table[pg] : -1;
}
__device__ __forceinline__ int row_of(const rt_kv &kv, const plan &p, int pos, int entry)
{
    const uint32_t pg = p.page.of(pos);
    return entry >= 0 && entry < kv.pages ? entry * (int)(kv.heads * kv.page) + (pos - (int)(pg * (uint32_t)kv.page)) : -1;
}
__device__ __forceinline__ const char *address(const void *cache, int row, uint32_t head_rows, int bytes)
{
    return (const char *)cache + (uint64_t)((uint32_t)(row < 0 ? 0 : row) + head_rows) * (uint32_t)bytes;
}

/* The running maximum raised where a lane's largest score passes it by slack, and the reference that
 * the exponents are taken from */
template <int VE>
__device__ __forceinline__ float reference(float top, float slack, float &m, float &l, v4f (&acc)[VE])
{
    if (__ballot(top > m + slack)) {
        const float raised = fmaxf(m, group_max(top)), f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - raised);
        m = raised;
        l *= f;
#pragma unroll
        for (int i = 0; i < VE; i++)
            acc[i] *= f;
    }
    return m == -INFINITY ? 0.0f : m;
}

/* The waves' results, scaled to the largest of their maxima and added in the waves' order: the output, or
 * the chunk's part of it */
template <int D>
constexpr int joint_bytes() { return WAVES * 16 * (D + 4 + 2) * 4; }

template <int D, int VEC>
__device__ __forceinline__ void finish(char *lds, const rt_kv &kv, const rt_attn &a, const plan &p, const share &u, int number, float m, float l, const v4f (&acc)[D / 16])
{
    constexpr int LD = D + 4; /* rows off each other's banks */
    float(*so)[16][LD] = (float(*)[16][LD])lds;
    float(*sm)[16] = (float(*)[16])(lds + WAVES * 16 * LD * 4), (*sl)[16] = sm + WAVES;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, g = lane >> 4;
    const int kh = (int)blockIdx.y;
    l = group_sum(l);
    __syncthreads();
    if (g == 0)
        sm[wave][c] = m, sl[wave][c] = l;
    __syncthreads();
    float top = sm[0][c];
#pragma unroll
    for (int w = 1; w < WAVES; w++)
        top = fmaxf(top, sm[w][c]);
    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
    const int group = p.heads, left = u.q.n * group - u.z * 16, rows = left < 16 ? left : 16;
    if (c < rows)
#pragma unroll
        for (int i = 0; i < D / 16 / VEC; i++)
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int e = 0; e < VEC; e += 2)
                    *(float2 *)&so[wave][c][(i * 16 + 4 * g + r) * VEC + e] = float2{acc[i * VEC + e][r] * f, acc[i * VEC + e + 1][r] * f};
    __syncthreads();
    for (int i = tid; i < rows * (D / 4); i += 64 * WAVES) {
        const int r = i / (D / 4), d = 4 * (i % (D / 4));
        float t = sm[0][r], sum = 0.0f;
        for (int w = 1; w < WAVES; w++)
            t = fmaxf(t, sm[w][r]);
        float4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int w = 0; w < WAVES; w++) {
            const float4 x = *(const float4 *)&so[w][r][d];
            v = float4{v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w};
            sum += sl[w][r] * (sm[w][r] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(sm[w][r] - t));
        }
        const int jr = (int)p.group.of(u.z * 16 + r), hr = kh * group + (u.z * 16 + r - jr * group);
        const long pos = (long)u.q.past + jr;
        if (pos >= p.cap)
            sum = NAN; /* a position that the table does not reach */
        if (u.q.chunks == 1) {
            store_row(a, D, u.q.first + jr, hr, d, v, sum, pos < 0, gate_of(a, u.q.first + jr, hr, d));
        } else {
            const long slot = (long)kh * p.slots + number;
            *(float4 *)(p.part + (slot * 16 + r) * D + d) = v;
            if (d == 0)
                *(float2 *)(p.part + kv.heads * p.slots * 16 * D + (slot * 16 + r) * 2) = float2{t, sum};
        }
    }
    __syncthreads();
}

/* The most elements (at most full) that a lane's VE elements of a V row divide into */
constexpr int pieces(int ve, int full) { return ve % full == 0 ? full : ve % (full / 2) == 0 ? full / 2 : 2; }

/* An F32 cache, 16 positions a tile, on v_mfma_f32_16x16x4_f32: position 4 g + r in the second product's step r. */
template <int D>
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
        if (!share_of(b, kv, p, group, number, u))
            return;
        v4f acc[VE];
#pragma unroll
        for (int i = 0; i < VE; i++)
            acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        float m = -INFINITY, l = 0.0f;
        const auto here = [&](int tile) { return tile * 16 + c < u.last ? tile * 16 + c : u.last; };
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
            const bool whole = tile * 16 + 15 <= u.least; /* every row sees every position of the tile */
#pragma unroll
            for (int r = 0; r < 4; r++) {
                x[r] = rows[r] < 0 ? NAN : s[0][r] + s[1][r];
                if (!whole && tile * 16 + 4 * g + r > u.lim)
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
                            vw[r][i][e] = tile * 16 + 4 * g + r > u.last ? 0 : vw[r][i][e];
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
                /* each token's rows are computed apart, without the values behind it */
                for (int jj = u.j0; jj <= u.j1; jj++) {
                    const long upto = (long)u.q.past + jj < u.last ? (long)u.q.past + jj : u.last;
#pragma unroll
                    for (int i = 0; i < NV; i++)
#pragma unroll
                        for (int e = 0; e < VEC; e++) {
                            v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                            for (int r = 0; r < 4; r++)
                                o = __builtin_amdgcn_mfma_f32_16x16x4f32(tile * 16 + 4 * g + r <= upto ? __builtin_bit_cast(float, vw[r][i][e]) : 0.0f, x[r], o, 0, 0, 0);
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
template <int TYPE>
struct half_of;
template <>
struct half_of<RT_F16> {
    static constexpr int LIMBS = 2;
    static constexpr float SLACK = 1.0f, LIFT = 15.0f - SLACK, LEAST = 0x1p-5f;
    static constexpr uint32_t INF = 0x7c00;
    static __device__ __forceinline__ uint16_t round(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
    static __device__ __forceinline__ float back(uint16_t x) { return (float)__builtin_bit_cast(_Float16, x); }
    static __device__ __forceinline__ v4f mfma(uint4 x, uint4 y, v4f z) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, x), __builtin_bit_cast(h8, y), z, 0, 0, 0); }
};
template <>
struct half_of<RT_BF16> {
    static constexpr int LIMBS = 3;
    static constexpr float SLACK = ::SLACK, LIFT = 0.0f, LEAST = 0.0f;
    static constexpr uint32_t INF = 0x7f80;
    static __device__ __forceinline__ uint16_t round(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
    static __device__ __forceinline__ float back(uint16_t x) { return __builtin_bit_cast(float, (uint32_t)x << 16); }
    static __device__ __forceinline__ v4f mfma(uint4 x, uint4 y, v4f z) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, x), __builtin_bit_cast(b8, y), z, 0, 0, 0); }
};

/* 8 F32 values as LIMBS operands */
template <int TYPE>
__device__ __forceinline__ void limbs_of(const float *x, uint4 *out)
{
    typedef half_of<TYPE> H;
    float rest[8];
#pragma unroll
    for (int e = 0; e < 8; e++)
        rest[e] = x[e];
#pragma unroll
    for (int n = 0; n < H::LIMBS; n++) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const uint16_t lo = H::round(rest[e]), hi = H::round(rest[e + 1]);
            w[e / 2] = lo | (uint32_t)hi << 16;
            rest[e] -= H::back(lo);
            rest[e + 1] -= H::back(hi);
        }
        out[n] = uint4{w[0], w[1], w[2], w[3]};
    }
}

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

template <int D, int TYPE>
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
        if (!share_of(b, kv, p, group, number, u))
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
                entry[n] = entry_of(kv, p, u.table, here(t * POS + 16 * n + c));
        };
        const auto rows_next = [&](int t) {
#pragma unroll
            for (int n = 0; n < SUB; n++)
                row[n] = row_of(kv, p, here(t * POS + 16 * n + c), entry[n]);
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
            const auto place = [&](int r) { return tile * POS + r / 4 * 16 + 4 * g + r % 4; }; /* the lane's positions */
            float x[4 * SUB];
            const bool whole = tile * POS + POS - 1 <= u.least; /* every row sees every position of the tile */
            float top = -INFINITY;
#pragma unroll
            for (int r = 0; r < 4 * SUB; r++) {
                x[r] = rows[r] < 0 ? NAN : back * s[r / 4][r % 4];
                if (!whole && place(r) > u.lim)
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
                const bool hide = !whole && place(r) > u.last;
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
                    /* with values that are not finite each token's rows are computed apart, without the values behind it.
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
#pragma unroll
                        for (int k = 0; k < SUB / 2; k++)
#pragma unroll
                            for (int i = 0; i < NV; i++) {
                                uint32_t again[8][VW];
#pragma unroll
                                for (int r = 0; r < 8; r++) {
                                    load_words<VW>(again[r], address(kv.v, rows[8 * k + r], head_rows, D * 2) + (i * 16 + c) * VEC * 2);
                                    const bool hide = place(8 * k + r) > upto;
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
    if (!locate(b, p, p.heads, -1, i, s, q, before, chunk) || q.chunks == 1)
        return;
    const int kh = (int)p.group.of((uint32_t)h), row = (int)(i - q.first) * p.heads + (int)h - kh * p.heads, z = q.rows - 1 - row / 16, r = row % 16;
    if ((long)before + (long)(z + 1) * q.chunks > p.slots)
        return;
    const long slot = (long)kh * p.slots + before + z * q.chunks;
    const float *ml = p.part + kv.heads * p.slots * 16 * D + (slot * 16 + r) * 2, *part = p.part + (slot * 16 + r) * D + dd;
    float4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    for (int k0 = turn; k0 < q.chunks; k0 += 64) {
        float2 x[4];
        float4 w[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int at_chunk = k0 + 16 * k < q.chunks ? k0 + 16 * k : k0;
            x[k] = *(const float2 *)(ml + (long)at_chunk * 32);
            w[k] = *(const float4 *)(part + (long)at_chunk * 16 * D);
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

template <int TYPE>
void launch(hipStream_t s, dim3 grid, const rt_seqs &b, const rt_kv &kv, const rt_attn &a, const plan &p)
{
    switch (kv.dim) {
#define DIM(D)                                                                                                                                             \
    case D:                                                                                                                                                \
        if constexpr (TYPE == RT_F32)                                                                                                                      \
            attn_f32_k<D><<<grid, 64 * WAVES, 0, s>>>(b, kv, a, p);                                                                                        \
        else                                                                                                                                               \
            attn_half_k<D, TYPE><<<grid, 64 * WAVES, 0, s>>>(b, kv, a, p);                                                                                 \
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

int tile_of(const rt_kv &kv) { return kv.type == RT_F32 ? 1 : sixteens(kv.dim); }

void plan_chunks(const rt_seqs &b, const rt_kv &kv, const rt_attn &a, long &tiles, long &target)
{
    tiles = b.t * (a.q_heads / kv.heads) / 16 + b.n;
    const bool single = kv.type == RT_F32 ? kv.dim > 128 : alone(kv.dim);
    const long once = ((single ? 256 : 512) + kv.heads - 1) / kv.heads;
    if (tiles * kv.heads > SLOTS || kv.table_ld * kv.page <= 16 * WAVES * tile_of(kv))
        target = 0;
    else if (b.t >= 16 * b.n && tiles >= once)
        target = once;
    else
        target = (2 * tiles + once - 1) / once * once - tiles;
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
    long tiles, target;
    plan_chunks(b, kv, a, tiles, target);
    p.target = (int)target;
    p.tile = tile_of(kv);
    p.least = WAVES * p.tile;
    const auto by = [](long d) {
        int up = 0;
        while ((1L << up) < d)
            up++;
        return divisor{(uint32_t)((((__uint128_t)1 << (31 + up)) + d - 1) / d), 31 + up};
    };
    p.heads = (int)(a.q_heads / kv.heads);
    p.page = by(kv.page), p.group = by(p.heads);
    p.share = target ? 1.00001f / (float)target : 0.0f;
    const long reach = (1L << 31) - 4096;
    p.cap = (int)(kv.table_ld > reach / kv.page ? reach : kv.table_ld * kv.page);
    p.slots = (int)(target + (target ? tiles : 0));
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
        attn_join_k<<<dim3((unsigned)b.t, (unsigned)a.q_heads, (unsigned)((kv.dim + 63) / 64)), 256, 0, s>>>(b, kv, a, p);
}
