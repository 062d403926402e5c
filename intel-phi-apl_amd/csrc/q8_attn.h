/* q8_attn.h: what the kernels of the attention over the paged cache share: the plan of a launch, a workgroup's share of it,
 * the way from positions to rows, and the waves' joint result. */
#ifndef Q8_ATTN_H
#define Q8_ATTN_H

#include "q8_mix.h"
#include "q8_bf16.h"

/* x / d for x < 2^31: (x * mul) >> shift with shift = 31 + ceil(log2 d), mul = ceil(2^shift / d): exact, as the
 * excess mul * d - 2^shift is below d <= 2^(shift - 31) */
struct q8_divisor {
    uint32_t mul;
    int shift;
    __device__ __forceinline__ uint32_t of(uint32_t x) const { return (uint32_t)(((uint64_t)x * mul) >> shift); }
};

/* What a launch shares: row tiles are 16 or 64 query rows (token, head of the group) of one key-value head and
 * sequence; the positions that one sees, in tiles of 16, are cut into chunks of one size for the whole batch. */
struct q8_attn_plan {
    q8_divisor page, group; /* by the positions of a page, by the query heads of a key-value head */
    int heads;    /* query heads of a key-value head */
    int shift;    /* a row tile has 1 << shift rows */
    int cap;      /* positions that the table reaches */
    int tile;     /* 16s of positions that a wave takes at once (a power of two): chunks are whole numbers of them */
    int least;    /* 16s a chunk at least: one tile of each wave */
    int target;   /* chunks (a key-value head) to spread all tiles over; 0: one a row tile */
    int slots;    /* partial results a key-value head, a row tile's each */
    float share;  /* 1 / target, and a little: rounded sums must not make a chunk too small */
    int once;     /* the workgroups (a key-value head) that run at once, where the chunks' size is chosen by rounds of them; or 0 */
    int *size;    /* then the size that was chosen, for the join */
    float qscale; /* scale * log2 e: scores are in powers of two */
    int window;   /* positions that a token sees, itself and those before it; 0: all */
    int sinks;    /* with a window, the first positions, which every later token sees, too */
    float *part;  /* [heads][slots][rows][dim], then [heads][slots][rows][2]: maximum and sum */
};

/* the 8-bit cache's kernel on `blocks` x heads workgroups */
void q8_launch_attn8(q8_stream_t stream, long blocks, const rt_seqs &b, const rt_kv &kv, const rt_attn &a, const q8_attn_plan &p);
/* the 16-bit caches' through a window, of many rows (p.shift 6) */
void q8_launch_attn_rows(q8_stream_t stream, long blocks, const rt_seqs &b, const rt_kv &kv, const rt_attn &a, const q8_attn_plan &p);
/* 16s of positions that it takes at once */
constexpr int q8_attn_rows_tile(long dim) { return dim > 128 ? 2 : 4; }
/* whether a compute unit holds one of its workgroups, not two */
constexpr bool q8_attn8_alone(long dim) { return dim > 128; }

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

constexpr int WAVES = 4;

typedef q8_attn_plan plan;

struct seq_plan {
    int first, n;     /* its rows of the token-major arrays */
    int past, tiles;  /* position tiles of all that a row tile of it sees at most, within the table */
    int rows, chunks; /* row tiles, and chunks of each */
};

/* With a window, the position tiles that a row tile sees at most: the sinks' tiles, and those from the first token's first
 * position, rounded down to a wave's tile, to the last of as many tokens as it may have rows */
__host__ __device__ __forceinline__ int window_tiles(const plan &p)
{
    return (p.sinks + 16 * p.tile - 1) / (16 * p.tile) * p.tile + (p.window + 15) / 16 + (1 << p.shift) / 16 + p.tile + 1;
}

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
    if (p.window > 0) {
        const int most = window_tiles(p);
        q.tiles = q.tiles < most ? q.tiles : most;
    }
    q.rows = (int)(((uint32_t)q.n * (uint32_t)group + (1u << p.shift) - 1) >> p.shift);
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

/* The size of chunks of which the rounds of workgroups take least: of some sizes that make one or two rounds, the one with the
 * smallest rounds x (size + FIXED), FIXED being what a workgroup takes besides, in tiles. A batch's last, partial round
 * costs a whole one: of 32 sequences of 1028 positions and 4 heads the other calls' chunks (chunk_from), a third of a sequence,
 * take two rounds (45.5 us with the join), halves one (39.7); 32 of 100 to 16384 positions 131, 111 with these. A single sequence's
 * fill a round as they are, and its call is latency alone, which eight sizes add a microsecond to. `chunks`: how many chunks
 * there are of a size. */
constexpr float FIXED = 10.0f;
template <class F>
__device__ __forceinline__ int chunk_of_rounds(const plan &p, float all, F chunks)
{
    constexpr float size[] = {2.0f, 1.5f, 1.25f, 1.125f, 1.0f, 0.75f, 0.625f, 0.55f};
    const float even = all * __builtin_amdgcn_rcpf((float)p.once) * 1.00001f + 1.0f, turn = __builtin_amdgcn_rcpf((float)p.once);
    float least = INFINITY;
    int best = p.least;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        int c = ((int)(even * size[i]) + p.tile) / p.tile * p.tile;
        c = c > p.least ? c : p.least;
        const int count = chunks(c);
        const float cost = ceilf((float)count * turn - 0.001f) * ((float)c + FIXED);
        const bool better = i == 0 || (count <= p.slots && cost < least);
        best = better ? c : best;
        least = better ? cost : least;
    }
    return best;
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
 * chunks of the sequences before it; false: there is none. A lane a sequence, 64 at a time. JOIN: after the launch of the chunks. */
template <bool JOIN = false>
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
    if (JOIN && p.once) {
        chunk = *p.size;
    } else if (p.target > 0) {
        float all = (float)at.rows * (float)at.tiles;
        for (int s0 = 64; s0 < n; s0 += 64)
            if (s0 + lane < n) {
                const seq_plan o = plan_of(b, p, group, s0 + lane);
                all += (float)o.rows * (float)o.tiles;
            }
        all = q8_wave_sum_dpp(all);
        chunk = first_lane(p.once && n <= 64 && all < 1e8f ? chunk_of_rounds(p, all, [&](int c) { return (int)q8_wave_sum_dpp((float)(at.rows * chunks_of(at.tiles, c))); })
                                                           : chunk_from(p, all));
        if (!JOIN && p.once && number == 0 && threadIdx.x == 0)
            *p.size = chunk; /* each head's first workgroup the same */
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
    int z, row;      /* the row tile, and the wave's first row: all waves have the same 16, or each its own 16 of 64 */
    int j0, j1;      /* the tokens of the wave's rows */
    int j, h;        /* the lane's query row: token and head */
    bool live;       /* there is one */
    int lim;         /* the last position that the lane's row sees, -1 none */
    int end;         /* the last that any row of the tile sees */
    int last, least; /* the last that any of the wave's rows sees, and the last that all do */
    int t0, t1;      /* the chunk's position tiles, 16 each */
    /* with a window the tiles are counted without those that the row tile does not see: from tile `sunk` on, a tile is `skip`
     * further on */
    int sunk, skip;
    int low;         /* the first position, but for the sinks, that the lane's row sees; lo0 and lo1: the wave's first and last row's */
    int lo0, lo1;
};

/* The first position of token j's window, or behind the table */
__device__ __forceinline__ int window_from(const plan &p, const seq_plan &q, int j)
{
    const long pos = (long)q.past + j - (p.window - 1);
    return pos < 0 ? 0 : pos < p.cap ? (int)pos : p.cap;
}
/* Whether a row whose window begins at low has position i before it, and not as a sink */
template <bool WINDOW>
__device__ __forceinline__ bool passed(const plan &p, int i, int low)
{
    return WINDOW && i < low && i >= p.sinks;
}
/* Whether all of the wave's rows see the positions [i, i + n), so that no mask is needed */
template <bool WINDOW>
__device__ __forceinline__ bool all_seen(const plan &p, const share &u, int i, int n)
{
    return i + n - 1 <= u.least && (!WINDOW || i >= u.lo1 || i + n <= p.sinks);
}
/* The place of the row tile's tile t, in tiles of 16 * sub positions */
template <bool WINDOW>
__device__ __forceinline__ int place_of(const share &u, int t, int sub)
{
    return WINDOW && t * sub >= u.sunk ? t + u.skip / sub : t;
}

template <bool WINDOW, int ROWS = 16>
__device__ __forceinline__ bool share_of(const rt_seqs &b, const rt_kv &kv, const plan &p, int group, int number, int kv_head, share &u)
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
    constexpr int WAVE = 16; /* rows of a wave */
    u.row = u.z * ROWS + (ROWS == 16 ? 0 : first_lane((int)threadIdx.x / 64 * WAVE));
    const int row = u.row + (int)(threadIdx.x & (WAVE - 1));
    u.table = kv.table + s * kv.table_ld;
    u.j = (int)p.group.of(row);
    u.h = kv_head * group + (row - u.j * group);
    u.live = u.j < q.n;
    const auto sees = [&](int j) { /* the last position that token j sees, within the table */
        const long pos = (long)q.past + j;
        return pos < 0 ? -1 : pos < p.cap ? (int)pos : p.cap - 1;
    };
    u.lim = u.live ? sees(u.j) : -1;
    const auto token = [&](int i) {
        const int j = first_lane((int)p.group.of(i));
        return j < q.n ? j : q.n - 1;
    };
    u.j0 = token(u.row);
    u.j1 = token(u.row + WAVE - 1);
    u.last = sees(u.j1);
    u.least = sees(u.j0);
    u.end = ROWS == 16 ? u.last : sees(token(u.z * ROWS + ROWS - 1));
    u.t0 = part * chunk;
    u.t1 = u.end < 0 ? 0 : u.end / 16 + 1;
    if constexpr (WINDOW) {
        u.low = u.live ? window_from(p, q, u.j) : 0;
        u.lo0 = window_from(p, q, u.j0);
        u.lo1 = window_from(p, q, u.j1);
        const int low = ROWS == 16 ? u.lo0 : window_from(p, q, token(u.z * ROWS));
        const int first = low / (16 * p.tile) * p.tile, some = (p.sinks + 16 * p.tile - 1) / (16 * p.tile) * p.tile;
        u.sunk = some < first ? some : first;
        u.skip = first - u.sunk;
        u.t1 = u.t1 > first ? u.t1 - u.skip : u.t1 < u.sunk ? u.t1 : u.sunk;
    }
    if (q.chunks > 1 && u.t0 + chunk < u.t1)
        u.t1 = u.t0 + chunk;
    if constexpr (ROWS != 16) { /* a wave's, not a lane's: in scalar registers */
        for (int *v : {&u.last, &u.least, &u.end, &u.t0, &u.t1})
            *v = first_lane(*v);
        if constexpr (WINDOW)
            for (int *v : {&u.lo0, &u.lo1, &u.sunk, &u.skip})
                *v = first_lane(*v);
    }
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

template <int D, int VEC, int VE = D / 16>
__device__ __forceinline__ void finish(char *lds, const rt_kv &kv, const rt_attn &a, const plan &p, const share &u, int number, float m, float l, const v4f (&acc)[VE])
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
        for (int i = 0; i < VE / VEC; i++)
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int e = 0; e < VEC; e += 2)
                    if (VE * 16 == D || (i * 16 + 4 * g + r) * VEC < D)
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

/* ---- what the kernels of prompts share: 64 query rows a workgroup on tiles of 64 positions in LDS */
constexpr int ROWS = 64;

/* A value's row in LDS (one element, 64 positions) is 8 pieces of 16 bytes, of which piece n lies at (n + spread) & 7 */
__device__ __forceinline__ int spread(int d) { return (d >> 2) + 2 * (d & 3); }

/* Which row tile (and chunk) of which key-value head a workgroup takes. Workgroups go to the 8 XCDs in turn, each with an L2 of its
 * own, so a head's go to as few XCDs as there are for it, and an XCD's go through a head's row tiles in order: what they read together is
 * a part of one head's cache. (A prompt of 2048 tokens 114 us, 152 in the grid's order. Left out: the second 32 of an XCD's, which share
 * the compute units with the first, from the shortest row tiles on: 850 tokens 59 us, 60 as it is; 1400 through a window of 1024 96, 95 as
 * it is.) */
struct order {
    int blocks, heads; /* row tiles or chunks a head; heads */
    int each, count;   /* XCDs a head (0: several heads an XCD); workgroups an XCD */
};
order order_of(long blocks, long heads)
{
    order q = {(int)blocks, (int)heads, 0, 0};
    if (heads < 8 && 8 % heads == 0)
        q.each = (int)(8 / heads);
    q.count = (int)(q.each ? (blocks + q.each - 1) / q.each : (heads * blocks + 7) / 8);
    return q;
}
__device__ __forceinline__ bool place_in(const order &q, int block, int &number, int &head)
{
    const int xcd = block & 7;
    const int at = block >> 3;
    if (q.each) {
        head = xcd / q.each;
        number = at * q.each + xcd % q.each;
    } else {
        const int i = at * 8 + xcd; /* with a multiple of 8 heads each XCD has heads of its own */
        if (q.heads % 8 == 0) {
            head = at / q.blocks * 8 + xcd;
            number = at % q.blocks;
        } else {
            head = i / q.blocks;
            number = i % q.blocks;
        }
    }
    return head < q.heads && number < q.blocks;
}

/* 1 / (1 + exp(-x)): the exponent in two parts, a reciprocal off by a step. An exponential below 2^-126 is 0, and so it is from |x| =
 * 104 on, infinity among them, where neither part could be made of x itself; NaN stays NaN */
__device__ __forceinline__ float gate_weight(float x)
{
    const float y = fabsf(x) > 104.0f ? -104.0f : -fabsf(x), t = y * 1.44269504f, r = fmaf(y, 1.92596300e-8f, fmaf(y, 1.44269504f, -t)), e = __builtin_amdgcn_exp2f(t);
    const float f = fmaf(e * r, 0.693147181f, e);
    return (x >= 0.0f ? 1.0f : f) * __builtin_amdgcn_rcpf(1.0f + f);
}

/* 8 finite F32 values as three bf16 limbs, 8 bits each: exact */
__device__ __forceinline__ void limbs8(const float *x, v4i (&w)[3])
{
    float mid[8], lo[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        mid[e] = x[e] - __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x[e]) & 0xffff0000u);
        lo[e] = mid[e] - __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, mid[e]) & 0xffff0000u);
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
        w[0][e] = (int)pack_hi(x[2 * e], x[2 * e + 1]);
        w[1][e] = (int)pack_hi(mid[2 * e], mid[2 * e + 1]);
        w[2][e] = (int)pack_hi(lo[2 * e], lo[2 * e + 1]);
    }
}

} /* namespace */

#endif
