/* q8_attn8.hip: attention of new tokens over the paged key-value cache of 8 bits, and reading a cache back (include/q8_mix.h). */
#include "q8_attn.h"

namespace {

/* A row of the cache is d * q, q in -127 .. 127 and d the F32 scale of that position and head. So
 *
 *   score = scale d_k (query . q_k)          o = sum_j (p_j d_v) q_v / sum_j p_j
 *
 * Keys are the integer instruction's operand as they lie (v_mfma_i32_16x16x64_i8): a query row is rounded to 24 bits of its
 * largest element, X = rint(query * FULL / most), and cut into three balanced bytes; the three integer sums are exact (below
 * 2^23 each), and joined in F32. An element is off by 2^-24 of its row's largest.
 *
 * Values have to meet weights of any size: where a large weight's value is 0 in an element, the small ones are its output. So
 * the weights p_j d_v are cut into three bf16 limbs that hold all 24 bits at their own exponents, and a value is made bf16
 * (exact, 8 bits) on the way. Integers are always finite: a scale that is not finite makes its score or its row's
 * weights NaN, and where it is masked the weight is 0 by choice, not by product.
 *
 * A wave takes 64 positions at a time, one a lane for the page table and the scales, which go through LDS to where the
 * products have them. Otherwise as the 16-bit caches' kernel: scores S^T = K Q^T leave lane 16 g + c with positions
 * 16 n + 4 g + r of query row c, which is how the second product's operand has them. Bound by HBM on long histories (32 sequences of
 * 100 to 16384 positions, 4 heads of 256: 107 us, 5.3 TB/s; 4 tokens at 131072 positions 49, 5.5 TB/s), by the latency of its dependent loads
 * on short ones. The first values under way with the first keys measured 4 us slower on the former: the keys come later. */
constexpr int SUB = 4, POS = 64;
constexpr float FULL = 8355584.0f; /* 127 * 2^16 + 127 * 2^8: three balanced bytes hold 127 more, and the quotient's rounding adds 1 at most */

/* 4 floats as FULL's integers, their three balanced bytes gathered by byte: w[n] is byte n of the four */
__device__ __forceinline__ void bytes_of(float4 x, float up, uint32_t (&w)[3])
{
    uint32_t y[4];
#pragma unroll
    for (int e = 0; e < 4; e++)
        y[e] = (uint32_t)((int)__builtin_rintf((&x.x)[e] * up) + 0x808080);
    const uint32_t a = __builtin_amdgcn_perm(y[1], y[0], 0x05010400u), b = __builtin_amdgcn_perm(y[3], y[2], 0x05010400u); /* bytes 0 0 1 1 */
    w[0] = __builtin_amdgcn_perm(b, a, 0x05040100u) ^ 0x80808080u;
    w[1] = __builtin_amdgcn_perm(b, a, 0x07060302u) ^ 0x80808080u;
    w[2] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(y[3], y[2], 0x0c0c0602u), __builtin_amdgcn_perm(y[1], y[0], 0x0c0c0602u), 0x05040100u) ^ 0x80808080u;
}

/* The lane's scores from the three sums: exact integers, two roundings */
__device__ __forceinline__ float joined(int l0, int l1, int l2) { return fmaf((float)l2, 65536.0f, (float)((l1 << 8) + l0)); }

/* Elements of a V row that a lane has: the largest of 4, 8 and 16 that 16 lanes cover the row with; with heads that are no
 * power of two the last lanes have none */
constexpr int each(int d) { return d <= 64 ? 4 : d <= 128 ? 8 : 16; }

template <int D, bool WINDOW>
__global__ __launch_bounds__(64 * WAVES, q8_attn8_alone(D) ? 1 : 2) void attn8_k(rt_seqs b, rt_kv kv, rt_attn a, plan p)
{
    constexpr int NK = (D + 63) / 64, VE = each(D), VW = VE / 4;
    struct shared {
        uint4 query[NK][3][64];
        float most[WAVES][16];
        int row[WAVES][64];
        float dk[WAVES][64], dv[WAVES][64];
    };
    constexpr int NEED = sizeof(shared);
    __shared__ __align__(16) char lds[joint_bytes<D>() > NEED ? joint_bytes<D>() : NEED];
    shared &sh = *(shared *)lds;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const int group = p.heads;
    const uint32_t head_rows = (uint32_t)(blockIdx.y * kv.page);
    const size_t all_rows = (size_t)(kv.pages * kv.heads * kv.page);
    const float *const scale_k = (const float *)((const char *)kv.k + all_rows * D), *const scale_v = (const float *)((const char *)kv.v + all_rows * D);
    for (int number = (int)blockIdx.x; p.target == 0 || number < p.slots; number += (int)gridDim.x) {
        share u;
        if (!share_of<WINDOW>(b, kv, p, group, number, (int)blockIdx.y, u))
            return;
        const int stop = (u.t1 + SUB - 1) / SUB;
        int tile = u.t0 / SUB + wave;
        const auto here = [&](int t) { /* the lane's position of tile t, or the last that there is */
            const int i = place_of<WINDOW>(u, t, SUB) * POS + lane;
            return u.last < 0 ? 0 : i < u.last ? i : u.last;
        };
        uint4 kx[SUB][NK];
        float dk, dv; /* of the lane's position of the tile whose keys kx has */
        int entry;
        bool none; /* the position has no row */
        /* rows of tile t from its entries, by way of LDS to the lanes that load them, and the next entries */
        const auto load_keys = [&](int t) __attribute__((always_inline)) {
            const uint32_t pos = (uint32_t)here(t);
            none = (uint32_t)entry >= (uint32_t)kv.pages;
            const uint32_t row = none ? 0 : (uint32_t)entry * (uint32_t)(kv.heads * kv.page) + (pos - p.page.of(pos) * (uint32_t)kv.page);
            sh.row[wave][lane] = (int)row;
            dk = scale_k[row + head_rows], dv = scale_v[row + head_rows];
            entry = u.table[p.page.of(here(t + WAVES))];
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int n = 0; n < SUB; n++) {
                const char *k = address(kv.k, sh.row[wave][16 * n + c], head_rows, D);
#pragma unroll
                for (int i = 0; i < NK; i++)
                    kx[n][i] = *(const uint4 *)(k + (64 * i + 16 * g < D ? 64 * i + 16 * g : 0));
            }
        };
        uint32_t vw[4 * SUB][VW]; /* rows 16 n + 4 g + r */
        const auto load_values = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int n = 0; n < SUB; n++) {
                const int4 rows = *(const int4 *)&sh.row[wave][16 * n + 4 * g];
#pragma unroll
                for (int r = 0; r < 4; r++)
                    stream_words<VW>(vw[4 * n + r], address(kv.v, (&rows.x)[r], head_rows, D) + (c * VE < D ? c * VE : 0));
            }
        };
        entry = u.table[p.page.of(here(tile))]; /* (the table reaches them all) */
        /* wave w has the queries' columns 64 i, i = w, w + WAVES, ..., and makes their bytes for all waves */
        static_assert(NK <= WAVES);
        const float *query = a.q + (u.live ? (long)(u.q.first + u.j) * a.q_ld + u.h * a.q_hd : 0);
        const bool mine = wave < NK && 64 * wave + 16 * g < D;
        float4 qv[4];
        uint32_t most = 0; /* of the magnitudes' bits: an infinity or NaN stays the largest */
#pragma unroll
        for (int e = 0; e < 4; e++)
            qv[e] = *(const float4 *)(query + (mine ? 64 * wave + 16 * g : 0) + 4 * e);
        load_keys(tile);
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                float &x = (&qv[e].x)[k];
                x = mine && u.live ? x * p.qscale : 0.0f;
                const uint32_t bits = __builtin_bit_cast(uint32_t, fabsf(x));
                most = most > bits ? most : bits;
            }
        {
            const uint32_t o = __shfl_xor(most, 16, 64);
            most = most > o ? most : o;
            const uint32_t o2 = __shfl_xor(most, 32, 64);
            most = most > o2 ? most : o2;
        }
        if (g == 0)
            sh.most[wave][c] = __builtin_bit_cast(float, most);
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const uint32_t o = __builtin_bit_cast(uint32_t, sh.most[w][c]);
            most = most > o ? most : o;
        }
        const float top_query = fmaxf(__builtin_bit_cast(float, most), 1e-30f); /* smaller rows: in steps of 1e-37 */
        const float up = FULL / top_query, back = most < 0x7f800000u ? top_query / FULL : NAN;
        if (wave < NK) {
            uint32_t w[4][3];
#pragma unroll
            for (int e = 0; e < 4; e++)
                bytes_of(qv[e], up, w[e]);
#pragma unroll
            for (int n = 0; n < 3; n++)
                sh.query[wave][n][lane] = uint4{w[0][n], w[1][n], w[2][n], w[3][n]};
        }
        __syncthreads();
        v4f acc[VE];
#pragma unroll
        for (int i = 0; i < VE; i++)
            acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        float m = -INFINITY, l = 0.0f;
        for (; tile < stop; tile += WAVES) {
            sh.dk[wave][lane] = none ? NAN : dk;
            sh.dv[wave][lane] = dv;
            __builtin_amdgcn_wave_barrier();
            load_values();
            v4i s[SUB][3];
#pragma unroll
            for (int n = 0; n < SUB; n++)
#pragma unroll
                for (int e = 0; e < 3; e++)
                    s[n][e] = v4i{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < NK; i++)
#pragma unroll
                for (int e = 0; e < 3; e++) {
                    const v4i w = __builtin_bit_cast(v4i, sh.query[i][e][lane]);
#pragma unroll
                    for (int n = 0; n < SUB; n++)
                        s[n][e] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(v4i, kx[n][i]), w, s[n][e], 0, 0, 0);
                }
            if (tile + WAVES < stop)
                load_keys(tile + WAVES);
            const int base = place_of<WINDOW>(u, tile, SUB) * POS;
            const bool whole = all_seen<WINDOW>(p, u, base, POS); /* every row sees every position of the tile */
            const auto hidden = [&](int r) {
                const int i = base + r / 4 * 16 + 4 * g + r % 4;
                return i > u.lim || passed<WINDOW>(p, i, u.low);
            };
            float x[4 * SUB], top = -INFINITY;
#pragma unroll
            for (int n = 0; n < SUB; n++) {
                const float4 d = *(const float4 *)&sh.dk[wave][16 * n + 4 * g];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float &y = x[4 * n + r];
                    y = joined(s[n][0][r], s[n][1][r], s[n][2][r]) * (back * (&d.x)[r]);
                    if (!whole && hidden(4 * n + r))
                        y = -INFINITY;
                    top = fmaxf(top, y);
                }
            }
            /* the weights stay at most 1: times a scale they do not overflow */
            const float ref = reference(top, SLACK, m, l, acc) + SLACK;
            uint4 w[SUB / 2][3];
#pragma unroll
            for (int n = 0; n < SUB; n++) {
                const float4 d = *(const float4 *)&sh.dv[wave][16 * n + 4 * g];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float &y = x[4 * n + r];
                    const float weight = __builtin_amdgcn_exp2f(y - ref);
                    l += weight;
                    y = !whole && hidden(4 * n + r) ? 0.0f : weight * (&d.x)[r];
                }
            }
#pragma unroll
            for (int k = 0; k < SUB / 2; k++)
                xsplit8(float4{x[8 * k], x[8 * k + 1], x[8 * k + 2], x[8 * k + 3]}, float4{x[8 * k + 4], x[8 * k + 5], x[8 * k + 6], x[8 * k + 7]}, w[k][0], w[k][1],
                        w[k][2]);
#pragma unroll
            for (int e = 0; e < VE; e++) {
#pragma unroll
                for (int k = 0; k < SUB / 2; k++) {
                    uint32_t v[4];
#pragma unroll
                    for (int r = 0; r < 8; r += 2)
                        v[r / 2] = pack_hi((float)(int8_t)(vw[8 * k + r][e / 4] >> (8 * (e % 4))), (float)(int8_t)(vw[8 * k + r + 1][e / 4] >> (8 * (e % 4))));
#pragma unroll
                    for (int n = 0; n < 3; n++)
                        acc[e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, uint4{v[0], v[1], v[2], v[3]}), __builtin_bit_cast(b8, w[k][n]), acc[e], 0, 0, 0);
                }
                if (e & 1)
                    __builtin_amdgcn_sched_barrier(0);
            }
        }
        finish<D, VE, VE>(lds, kv, a, p, u, number, m, l, acc);
    }
}

/* ---- prompts
 *
 * 64 query rows a workgroup, 16 a wave, which share a tile of 64 positions in LDS: the keys as they lie, the values as bf16 and
 * transposed, in the order in which the second product's operand has the positions. So a key or value is loaded, and a value
 * converted, once for 64 rows and not for 16. The next tile's loads are under way in registers while the products of this one
 * run, and two workgroups share a compute unit, so that one's softmax and staging go under the other's matrix instructions.
 *
 * Heads of 256, 16 on 4: a prompt of 2048 115 us (16 rows a workgroup, as single tokens go: 299, the join's 95 among them); 8192
 * tokens through 1024 positions 358 (1075). A wave's tile is 144 matrix instructions, 2304 cycles, and some 575 others (queries and gates
 * among them), 2300, of 5100 that it takes of its SIMD: between two matrix instructions two others go unnoticed, the third costs,
 * so the issue of both bounds it. Tried and not faster: 32 rows a wave on the 32x32 instructions, one wave a SIMD (213 and 530); tiles of 32 positions in double buffers with one
 * barrier and the next scores beside this softmax (115 and 379); 128 rows a workgroup (141 and 356).
 *
 * LDS: the keys' rows are 16 bytes apart, which keeps 8 neighbouring rows off each other's banks; a value's row (one element, 64
 * positions) is 8 pieces of 16 bytes, of which piece n lies at (n + spread) & 7, so that neither 8 elements' pieces read together nor 8 lanes'
 * written together meet. */
template <int D, bool WINDOW>
__global__ __launch_bounds__(64 * WAVES, 2) void attn8_rows_k(rt_seqs b, rt_kv kv, rt_attn a, plan p, order places)
{
    constexpr int NK = (D + 63) / 64, VE = D / 16, PIECES = D / 16, NP = (POS * PIECES + 255) / 256, EACH = each(D) / 4;
    struct shared {
        uint8_t k[POS][D + 16];
        v4i v[D][8];
        float scale[2][POS]; /* of the keys, of the values */
    };
    __shared__ __align__(16) shared sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = first_lane(tid >> 6), c = lane & 15, g = lane >> 4;
    const int group = p.heads;
    int number, head;
    if (!place_in(places, (int)blockIdx.x, number, head))
        return;
    const uint32_t head_rows = (uint32_t)head * (uint32_t)kv.page;
    const size_t all_rows = (size_t)(kv.pages * kv.heads * kv.page);
    const float *const scales = (const float *)((const char *)(wave == 0 ? kv.k : kv.v) + all_rows * D);
    share u;
    if (!share_of<WINDOW, ROWS>(b, kv, p, group, number, head, u))
        return;
    const int stop = (u.t1 + SUB - 1) / SUB;
    int tile = u.t0 / SUB;
    const auto here = [&](int t) __attribute__((always_inline)) { /* the lane's position of tile t, or the last that there is */
        const int i = place_of<WINDOW>(u, t, SUB) * POS + lane;
        return u.end < 0 ? 0 : i < u.end ? i : u.end;
    };
    int entry = u.table[p.page.of(here(tile))]; /* (the table reaches them all) */
    v4i kx[NP];
    uint32_t vx[16];
    float scale = 0.0f;
    bool none = false; /* the lane's position has no row */
    const auto load = [&](int t) __attribute__((always_inline)) {
        const uint32_t pos = (uint32_t)here(t), page_rows = (uint32_t)(kv.heads * kv.page);
        none = (uint32_t)entry >= (uint32_t)kv.pages;
        const uint32_t place = (none ? 0 : (uint32_t)entry * page_rows + (pos - p.page.of(pos) * (uint32_t)kv.page)) + head_rows; /* below 2^31 */
        entry = u.table[p.page.of(here(t + 1))];
        uint32_t rows[NP];
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int piece = tid + 256 * i, n = piece / PIECES < POS ? piece / PIECES : 0;
            rows[i] = (uint32_t)__shfl((int)place, n, 64);
        }
        scale = scales[place];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            /* positions 16 n + 4 g + r: g the wave's number, i = 4 n + r */
            const char *v = (const char *)kv.v + (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)place, i / 4 * 16 + 4 * wave + i % 4) * D;
            const uint32_t off = lane * EACH < D ? lane * EACH : 0;
            vx[i] = EACH == 4 ? *(const uint32_t *)(v + off) : EACH == 2 ? *(const uint16_t *)(v + off) : *(const uint8_t *)(v + off);
        }
#pragma unroll
        for (int i = 0; i < NP; i++)
            kx[i] = *(const v4i *)((const char *)kv.k + (uint64_t)rows[i] * D + (tid + 256 * i) % PIECES * 16);
    };
    const auto store = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int piece = tid + 256 * i;
            if (POS * PIECES % 256 == 0 || piece < POS * PIECES)
                *(v4i *)&sh.k[piece / PIECES][piece % PIECES * 16] = kx[i];
        }
        if (D % (64 * EACH) == 0 || lane * EACH < D)
#pragma unroll
            for (int e = 0; e < EACH; e++)
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    v4i w;
#pragma unroll
                    for (int r = 0; r < 8; r += 2)
                        w[r / 2] = (int)pack_hi((float)(int8_t)(vx[8 * k + r] >> (8 * e)), (float)(int8_t)(vx[8 * k + r + 1] >> (8 * e)));
                    const int d = lane * EACH + e;
                    sh.v[d][(4 * k + wave + spread(d)) & 7] = w;
                }
        if (wave < 2)
            sh.scale[wave][lane] = none && wave == 0 ? NAN : scale;
    };
    if (tile < stop)
        load(tile);
    /* the wave's queries as balanced bytes: elements 64 i + 16 g .. of row c */
    v4i query[NK][3];
    float back;
    {
        const float *q = a.q + (u.live ? (long)(u.q.first + u.j) * a.q_ld + u.h * a.q_hd : 0);
        v4f x[NK][4];
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < NK; i++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                x[i][e] = *(const v4f *)(q + (64 * i + 16 * g < D ? 64 * i + 16 * g : 0) + 4 * e);
#pragma unroll
        for (int i = 0; i < NK; i++)
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    x[i][e][k] = 64 * i + 16 * g < D && u.live ? x[i][e][k] * p.qscale : 0.0f;
                    const uint32_t bits = __builtin_bit_cast(uint32_t, fabsf(x[i][e][k]));
                    most = most > bits ? most : bits;
                }
        const uint32_t o = __shfl_xor(most, 16, 64);
        most = most > o ? most : o;
        const uint32_t o2 = __shfl_xor(most, 32, 64);
        most = most > o2 ? most : o2;
        const float top = fmaxf(__builtin_bit_cast(float, most), 1e-30f), up = FULL / top;
        back = most < 0x7f800000u ? top / FULL : NAN;
#pragma unroll
        for (int i = 0; i < NK; i++) {
            uint32_t w[4][3];
#pragma unroll
            for (int e = 0; e < 4; e++)
                bytes_of(float4{x[i][e][0], x[i][e][1], x[i][e][2], x[i][e][3]}, up, w[e]);
#pragma unroll
            for (int n = 0; n < 3; n++)
                query[i][n] = v4i{(int)w[0][n], (int)w[1][n], (int)w[2][n], (int)w[3][n]};
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
        if (tile + 1 < stop)
            load(tile + 1);
        const int base = place_of<WINDOW>(u, tile, SUB) * POS;
        /* none of the wave's rows sees any of it */
        if (!some || base > u.last || (WINDOW && base + POS <= u.lo0 && base >= p.sinks))
            continue;
        const bool whole = all_seen<WINDOW>(p, u, base, POS); /* every row sees every position of the tile */
        const auto hidden = [&](int r) __attribute__((always_inline)) {
            const int i = base + r / 4 * 16 + 4 * g + r % 4;
            return i > u.lim || passed<WINDOW>(p, i, u.low);
        };
        float x[4 * SUB], top = -INFINITY;
        const auto key = [&](int n, int i) __attribute__((always_inline)) { return *(const v4i *)&sh.k[16 * n + c][64 * i + 16 * g < D ? 64 * i + 16 * g : 0]; };
        v4i kk[2][NK]; /* the operands of the next 16 positions are read under this one's products */
#pragma unroll
        for (int i = 0; i < NK; i++)
            kk[0][i] = key(0, i);
#pragma unroll
        for (int n = 0; n < SUB; n++) {
            if (n + 1 < SUB)
#pragma unroll
                for (int i = 0; i < NK; i++)
                    kk[(n + 1) & 1][i] = key(n + 1, i);
            const v4f d = *(const v4f *)&sh.scale[0][16 * n + 4 * g] * back; /* first: the sums times a large scale may overflow */
            v4i s[3] = {v4i{0, 0, 0, 0}, v4i{0, 0, 0, 0}, v4i{0, 0, 0, 0}};
#pragma unroll
            for (int i = 0; i < NK; i++)
#pragma unroll
                for (int e = 0; e < 3; e++)
                    s[e] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kk[n & 1][i], query[i][e], s[e], 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; r++)
                x[4 * n + r] = joined(s[0][r], s[1][r], s[2][r]) * d[r];
        }
        if (!whole)
#pragma unroll
            for (int r = 0; r < 4 * SUB; r++)
                x[r] = hidden(r) ? -INFINITY : x[r];
#pragma unroll
        for (int r = 0; r < 4 * SUB; r++)
            top = fmaxf(top, x[r]);
        const float ref = reference(top, SLACK, m, l, acc) + SLACK;
#pragma unroll
        for (int n = 0; n < SUB; n++) {
            const v4f d = *(const v4f *)&sh.scale[1][16 * n + 4 * g];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float weight = __builtin_amdgcn_exp2f(x[4 * n + r] - ref);
                l += weight;
                x[4 * n + r] = weight * d[r];
            }
        }
        if (!whole)
#pragma unroll
            for (int r = 0; r < 4 * SUB; r++)
                x[r] = hidden(r) ? 0.0f : x[r]; /* whatever the scale is */
        const auto value = [&](int k, int e) __attribute__((always_inline)) { return sh.v[16 * e + c][(4 * k + g + 4 * e + spread(c)) & 7]; };
#pragma unroll
        for (int k = 0; k < SUB / 2; k++) {
            v4i w[3], v[2][2];
            v[0][0] = value(k, 0), v[0][1] = value(k, VE > 1 ? 1 : 0);
            limbs8(x + 8 * k, w);
#pragma unroll
            for (int e = 0; e < VE; e += 2) {
                if (e + 2 < VE)
                    v[(e / 2 + 1) & 1][0] = value(k, e + 2), v[(e / 2 + 1) & 1][1] = value(k, e + 3);
#pragma unroll
                for (int n = 0; n < 3; n++)
#pragma unroll
                    for (int f = 0; f < 2; f++)
                        acc[e + f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, v[e / 2 & 1][f]), __builtin_bit_cast(b8, w[n]), acc[e + f], 0, 0, 0);
            }
        }
    }
    l = group_sum(l);
    if (!u.live)
        return;
    const long pos = (long)u.q.past + u.j, slot = ((long)head * p.slots + number) * ROWS + (u.row - u.z * ROWS + c);
    const float sum = pos >= p.cap ? NAN : l; /* a position that the table does not reach */
    if (u.q.chunks > 1) {
#pragma unroll
        for (int e = 0; e < VE; e++)
            *(v4f *)(p.part + slot * D + 16 * e + 4 * g) = acc[e];
        if (g == 0)
            *(float2 *)(p.part + kv.heads * p.slots * ROWS * D + slot * 2) = float2{m, sum};
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

/* ---- reading a cache back
 *
 * A thread has 8 neighbouring elements of a row, of RUN tokens one behind the other, whose places and values are all under way at
 * once; one rounding to F32 (of 8 bits) and one to the rows' type. Bound by HBM on long ranges (32767 positions of 4 heads of 256 to
 * BF16 49 us, 4.1 TB/s; a token a workgroup 64, two 56, eight 54), by latency (starts, positions, table, values) on short ones, for
 * which RUN is 1. */
template <int TYPE>
struct eight { /* 8 elements as they lie in the cache */
    v4i w[TYPE == RT_F32 ? 2 : 1];
    float d;
};
template <int TYPE>
__device__ __forceinline__ eight<TYPE> load8(const void *cache, size_t row, long at, long dim, size_t all_rows)
{
    eight<TYPE> x;
    if constexpr (TYPE == RT_F32) {
        x.w[0] = *(const v4i *)((const float *)cache + row * dim + at);
        x.w[1] = *(const v4i *)((const float *)cache + row * dim + at + 4);
    } else if constexpr (TYPE == RT_Q8) {
        const int2 q = *(const int2 *)((const char *)cache + row * dim + at);
        x.w[0][0] = q.x, x.w[0][1] = q.y;
        x.d = ((const float *)((const char *)cache + all_rows * dim))[row];
    } else {
        x.w[0] = *(const v4i *)((const uint16_t *)cache + row * dim + at);
    }
    return x;
}
template <int TYPE>
__device__ __forceinline__ void values8(const eight<TYPE> &x, float (&v)[8])
{
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
#pragma unroll
    for (int e = 0; e < 8; e++) {
        if constexpr (TYPE == RT_F32) {
            const int word = x.w[e / 4][e % 4];
            v[e] = __builtin_bit_cast(float, word);
        } else if constexpr (TYPE == RT_Q8) {
            const int word = x.w[0][e / 4];
            v[e] = (float)(int8_t)(word >> (8 * (e % 4))) * x.d;
        } else
            v[e] = TYPE == RT_F16 ? (float)__builtin_bit_cast(h8, x.w[0])[e] : (float)__builtin_bit_cast(b8, x.w[0])[e];
    }
}

template <int TYPE, int RUN>
__global__ __launch_bounds__(256) void read_k(rt_seqs b, rt_kv kv, rt_kv_rows a)
{
    const long i0 = (long)blockIdx.x * RUN;
    const int d = (int)kv.dim, per = d / 8, n = 2 * (int)kv.heads * per;
    const size_t all_rows = (size_t)(kv.pages * kv.heads * kv.page);
    long place[RUN]; /* of the token's first head in the cache; -1: it has none, -2: no sequence has the token */
#pragma unroll
    for (int k = 0; k < RUN; k++) {
        const long s = i0 + k < b.t ? q8_sequence_of(b, i0 + k) : -1;
        const long pos = s < 0 ? -1 : (long)b.past[s] + (i0 + k - b.start[s]), slot = (uint32_t)pos / (uint32_t)kv.page; /* below 2^32 */
        const long entry = pos >= 0 && slot < kv.table_ld ? kv.table[s * kv.table_ld + slot] : -1;
        place[k] = s < 0 ? -2 : entry >= 0 && entry < kv.pages ? entry * kv.heads * kv.page + (pos - slot * kv.page) : -1;
    }
    for (int k = (int)threadIdx.x; k < n; k += 256) {
        const int which = k >= n / 2, h = (k - which * (n / 2)) / per, at = 8 * ((k - which * (n / 2)) % per);
        void *out = which ? a.v : a.k;
        if (!out)
            continue;
        eight<TYPE> x[RUN];
#pragma unroll
        for (int r = 0; r < RUN; r++)
            x[r] = load8<TYPE>(which ? kv.v : kv.k, (size_t)((place[r] < 0 ? 0 : place[r]) + h * kv.page), at, d, all_rows);
#pragma unroll
        for (int r = 0; r < RUN; r++) {
            if (place[r] == -2)
                continue;
            float v[8];
            values8<TYPE>(x[r], v);
            if (place[r] < 0)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    v[e] = NAN;
            const long to = (i0 + r) * (which ? a.v_ld : a.k_ld) + h * (which ? a.v_hd : a.k_hd) + at;
            if (a.type == RT_F32) {
                *(v4f *)((float *)out + to) = v4f{v[0], v[1], v[2], v[3]}, *(v4f *)((float *)out + to + 4) = v4f{v[4], v[5], v[6], v[7]};
            } else if (a.type == RT_F16) {
                typedef _Float16 h8 __attribute__((ext_vector_type(8)));
                *(h8 *)((_Float16 *)out + to) = h8{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3], (_Float16)v[4], (_Float16)v[5], (_Float16)v[6], (_Float16)v[7]};
            } else {
                *(b8 *)((__bf16 *)out + to) = b8{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3], (__bf16)v[4], (__bf16)v[5], (__bf16)v[6], (__bf16)v[7]};
            }
        }
    }
}

template <int TYPE>
void launch_read(hipStream_t s, const rt_seqs &b, const rt_kv &kv, const rt_kv_rows &a)
{
    if (b.t >= 4096)
        read_k<TYPE, 4><<<(unsigned)((b.t + 3) / 4), 256, 0, s>>>(b, kv, a);
    else
        read_k<TYPE, 1><<<(unsigned)b.t, 256, 0, s>>>(b, kv, a);
}

} /* namespace */

void q8_launch_attn8(q8_stream_t stream, long blocks, const rt_seqs &b, const rt_kv &kv, const rt_attn &a, const q8_attn_plan &p)
{
    const dim3 grid((unsigned)blocks, (unsigned)kv.heads);
    const order places = order_of(blocks, kv.heads);
    const unsigned all = 8u * (unsigned)places.count;
    switch (kv.dim) {
#define DIM(D)                                                                                                                                             \
    case D:                                                                                                                                                \
        if (p.shift == 6)                                                                                                                                  \
            p.window ? attn8_rows_k<D, true><<<all, 64 * WAVES, 0, (hipStream_t)stream>>>(b, kv, a, p, places)                                             \
                     : attn8_rows_k<D, false><<<all, 64 * WAVES, 0, (hipStream_t)stream>>>(b, kv, a, p, places);                                           \
        else if (p.window)                                                                                                                                 \
            attn8_k<D, true><<<grid, 64 * WAVES, 0, (hipStream_t)stream>>>(b, kv, a, p);                                                                   \
        else                                                                                                                                               \
            attn8_k<D, false><<<grid, 64 * WAVES, 0, (hipStream_t)stream>>>(b, kv, a, p);                                                                  \
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

void q8_launch_kv_read(q8_stream_t stream, const rt_seqs &b, const rt_kv &kv, const rt_kv_rows &a)
{
    const hipStream_t s = (hipStream_t)stream;
    if (kv.type == RT_F32)
        launch_read<RT_F32>(s, b, kv, a);
    else if (kv.type == RT_F16)
        launch_read<RT_F16>(s, b, kv, a);
    else if (kv.type == RT_BF16)
        launch_read<RT_BF16>(s, b, kv, a);
    else
        launch_read<RT_Q8>(s, b, kv, a);
}
