/* q8_delta.hip: the gated delta rule (include/q8_mix.h), and the norm and gate of its output. */
#include "q8_mix.h"

namespace {

/* The two gates of a token's head. softplus as max(x, 0) + log1p(exp(-|x|)): no overflow. */
__device__ __forceinline__ float decay_of(float a, float dt, float rate)
{
    const float x = a + dt;
    return expf(rate * (fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x)))));
}

/* Token by token. A wave owns 16 columns of a head's state: lane 16 c + g holds rows g*KR .. g*KR + KR - 1
 * of columns 4 c .. 4 c + 3, so a column's dot products go over a row of 16 lanes. Both products with
 * the state are taken before it changes, in one reduction:
 *
 *   S' = alpha S + k d^T,  d = beta (v - alpha S^T k),  S'^T q = alpha S^T q + (q.k) d
 *
 * and so are |q|^2, |k|^2 and q.k, whose scales are applied to the results. Bound by HBM (the state, read
 * and written once) on many sequences, by latency on one. */
template <int KR>
__global__ __launch_bounds__(64) void delta_step_k(rt_seqs b, rt_delta a, int most)
{
    const int lane = threadIdx.x, g = lane & 15, c = 4 * (lane >> 4);
    const long s = blockIdx.z, h = blockIdx.y, col = 16 * (long)blockIdx.x + c;
    const long kh = a.tiled ? h % a.k_heads : h / (a.v_heads / a.k_heads);
    long first, last;
    q8_rows_of(b, s, first, last);
    if (last - first > most)
        return; /* in chunks */
    const long base = ((s * a.v_heads + h) * a.k_dim + g * KR) * a.v_dim + col;
    float4 st[KR];
#pragma unroll
    for (int r = 0; r < KR; r++)
        st[r] = *(const float4 *)(a.s_in + base + r * a.v_dim);
    const float rate = a.decay[h], dt = a.dt[h];
    for (long i = first; i < last; i++) {
        float q[KR], k[KR];
#pragma unroll
        for (int r = 0; r < KR; r += 2) {
            *(float2 *)(q + r) = *(const float2 *)(a.q + i * a.q_ld + kh * a.k_dim + g * KR + r);
            *(float2 *)(k + r) = *(const float2 *)(a.k + i * a.k_ld + kh * a.k_dim + g * KR + r);
        }
        const float4 v = *(const float4 *)(a.v + i * a.v_ld + h * a.v_dim + col);
        const float alpha = decay_of(a.a[i * a.a_ld + h], dt, rate), beta = q8_sigmoid(a.b[i * a.b_ld + h]);
        float qq = 0.0f, kk = 0.0f, qk = 0.0f;
        float4 sq = {0.0f, 0.0f, 0.0f, 0.0f}, sk = sq;
#pragma unroll
        for (int r = 0; r < KR; r++) {
            qq = fmaf(q[r], q[r], qq);
            kk = fmaf(k[r], k[r], kk);
            qk = fmaf(q[r], k[r], qk);
            sq = float4{fmaf(st[r].x, q[r], sq.x), fmaf(st[r].y, q[r], sq.y), fmaf(st[r].z, q[r], sq.z), fmaf(st[r].w, q[r], sq.w)};
            sk = float4{fmaf(st[r].x, k[r], sk.x), fmaf(st[r].y, k[r], sk.y), fmaf(st[r].z, k[r], sk.z), fmaf(st[r].w, k[r], sk.w)};
        }
        qk = q8_row_sum(qk);
        sq = float4{q8_row_sum(sq.x), q8_row_sum(sq.y), q8_row_sum(sq.z), q8_row_sum(sq.w)};
        sk = float4{q8_row_sum(sk.x), q8_row_sum(sk.y), q8_row_sum(sk.z), q8_row_sum(sk.w)};
        float rq = 1.0f, rk = 1.0f;
        if (a.eps >= 0.0f) {
            rq = 1.0f / sqrtf(q8_row_sum(qq) + a.eps);
            rk = 1.0f / sqrtf(q8_row_sum(kk) + a.eps);
        }
        const float ak = alpha * rk;
        const float4 d = {beta * (v.x - ak * sk.x), beta * (v.y - ak * sk.y), beta * (v.z - ak * sk.z), beta * (v.w - ak * sk.w)};
        const float oq = a.scale * rq, od = oq * (rk * qk), oa = oq * alpha;
        if (g == 0)
            *(float4 *)(a.o + i * a.o_ld + h * a.v_dim + col) =
                float4{fmaf(oa, sq.x, od * d.x), fmaf(oa, sq.y, od * d.y), fmaf(oa, sq.z, od * d.z), fmaf(oa, sq.w, od * d.w)};
#pragma unroll
        for (int r = 0; r < KR; r++) {
            const float kr = rk * k[r];
            st[r] = float4{fmaf(kr, d.x, alpha * st[r].x), fmaf(kr, d.y, alpha * st[r].y), fmaf(kr, d.z, alpha * st[r].z), fmaf(kr, d.w, alpha * st[r].w)};
        }
    }
#pragma unroll
    for (int r = 0; r < KR; r++)
        *(float4 *)(a.s_out + base + r * a.v_dim) = st[r];
}

/* ---- longer sequences, CHUNK tokens at a time
 *
 * With the decays' products D_ij = alpha_{j+1} ... alpha_i (j <= i) and gamma_i = alpha_1 ... alpha_i inside a
 * chunk that starts from the state S0, the tokens' updates d_i solve a unit triangular system:
 *
 *   (I + A) d = beta (V - gamma K S0),        A_ij = beta_i (k_i . k_j) D_ij for j < i
 *   O = scale (gamma Q S0 + (Q K^T * D) d),   S = gamma_C S0 + K^T (D_C d)
 *
 * delta_prep_k computes what does not depend on the state, for all chunks at once: T = (I + A)^-1 diag(beta) and
 * P = scale Q K^T * D, and the rows' factors. delta_chunk_k goes from chunk to chunk, 16 columns of the state a
 * workgroup. All products are F32 (v_mfma_f32_16x16x4_f32): on these operands 16-bit limbs would need six
 * products each. The decays are multiplied, not taken as differences of summed logarithms: a long chunk's
 * sum would lose what a small decay after a large one is, and a decay of 0 would make NaN of it.
 *
 * The operands' order is the matrix instruction's: a result's lane 16 g + c has rows 4 g + r of column c, and as the second
 * operand of the next product, step r, that is row 4 g + r again. So results pass between the waves through LDS
 * as they lie, 16 bytes a lane, and a first operand's lane takes row c, columns 4 g .. 4 g + 3 of 16 with one load. */
constexpr int CHUNK = 64, TILES = CHUNK / 16, PAIRS = TILES * (TILES + 1) / 2;
/* a chunk's part of a head: tiles (i, j), j <= i, of T and of P, 256 floats each in a first operand's order, and
 * gamma rk, scale gamma rq and D_C rk of its tokens, gamma_C, and whether anything of it is not finite (a wave each) */
constexpr int PREP = 2 * PAIRS * 256 + 4 * CHUNK;
constexpr int PREP_BYTES = 4 * PREP;

typedef float v4f __attribute__((ext_vector_type(4)));

__device__ __forceinline__ v4f mfma4(float4 x, float4 y, v4f z)
{
    z = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x, y.x, z, 0, 0, 0);
    z = __builtin_amdgcn_mfma_f32_16x16x4f32(x.y, y.y, z, 0, 0, 0);
    z = __builtin_amdgcn_mfma_f32_16x16x4f32(x.z, y.z, z, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(x.w, y.w, z, 0, 0, 0);
}
__device__ __forceinline__ float4 as4(v4f x) { return float4{x[0], x[1], x[2], x[3]}; }
__device__ __forceinline__ float dot4(float4 x, float4 y) { return fmaf(x.w, y.w, fmaf(x.z, y.z, fmaf(x.y, y.y, x.x * y.x))); }
__device__ __forceinline__ float group_sum(float v)
{
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}
__device__ __forceinline__ bool finite4(float4 x) { return (x.x * 0.0f + x.y * 0.0f) + (x.z * 0.0f + x.w * 0.0f) == 0.0f; }

/* The chunks of a call are numbered by slots: sequence s has first / CHUNK + s and on, which are its own (the starts
 * ascend). A launch takes slots [from, from + count). */
__device__ __forceinline__ long slot_of(long first, long s) { return first / CHUNK + s; }

/* The sequence that slot i may belong to: the last whose slots begin at or before it */
__device__ __forceinline__ long sequence_of_slot(const rt_seqs &b, long i)
{
    const int lane = threadIdx.x & 63;
    long c = 0;
    for (long s0 = 0; s0 < b.n; s0 += 64) {
        const long s = s0 + lane;
        long first = 0, last;
        if (s < b.n)
            q8_rows_of(b, s, first, last);
        const unsigned long long m = __ballot(s < b.n && slot_of(first, s) <= i);
        c += __popcll(m);
        if (m != ~0ull)
            break;
    }
    return c - 1;
}

/* A workgroup a chunk and key head; wave w has key rows 16 w .. of K K^T and query rows 16 (3 - w) .. of Q K^T, five
 * tiles of 16 x 16 each, which the key head's value heads share. Bound by the matrix products and, for each value
 * head, the latency of the inverse: 16 x 16 on the diagonal by substitution, a column a lane, then by diagonals
 * T_ij = -T_ii sum_k A_ik T_kj. */
template <int DK>
__global__ __launch_bounds__(256) void delta_prep_k(rt_seqs b, rt_delta a, int most, long from, float *out)
{
    constexpr int NT = DK / 16, LK = DK + 4, LT = CHUNK + 4;
    constexpr int KEYS = CHUNK * LK, MATRIX = CHUNK * LT;
    __shared__ __align__(16) float lds[KEYS > 3 * MATRIX ? KEYS : 3 * MATRIX];
    float(*sk)[LK] = (float(*)[LK])lds;
    float(*sd)[LT] = (float(*)[LT])lds, (*sa)[LT] = sd + CHUNK, (*st)[LT] = sa + CHUNK;
    __shared__ __align__(16) float sbeta[CHUNK], srk[CHUNK], srq[CHUNK];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    const long slot = from + blockIdx.x, kh = blockIdx.y, s = sequence_of_slot(b, slot);
    if (s < 0)
        return;
    long first, last;
    q8_rows_of(b, s, first, last);
    const long at = first + (slot - slot_of(first, s)) * CHUNK;
    if (last - first <= most || at < first || at >= last)
        return; /* (before first: with starts that do not ascend) */
    const int n = (int)(last - at < CHUNK ? last - at : CHUNK);
    const int kr = 16 * wave + c, qr = 16 * (3 - wave) + c;

    float4 qv[NT], kv[NT];
    float kk = 0.0f, qq = 0.0f;
#pragma unroll
    for (int t = 0; t < NT; t++) {
        kv[t] = qv[t] = float4{0.0f, 0.0f, 0.0f, 0.0f};
        if (kr < n)
            kv[t] = *(const float4 *)(a.k + (at + kr) * a.k_ld + kh * DK + 16 * t + 4 * g);
        if (qr < n)
            qv[t] = *(const float4 *)(a.q + (at + qr) * a.q_ld + kh * DK + 16 * t + 4 * g);
    }
#pragma unroll
    for (int t = 0; t < NT; t++) {
        *(float4 *)&sk[kr][16 * t + 4 * g] = kv[t];
        kk += dot4(kv[t], kv[t]);
        qq += dot4(qv[t], qv[t]);
    }
    kk = group_sum(kk), qq = group_sum(qq);
    if (g == 0) {
        srk[kr] = a.eps >= 0.0f && kr < n ? 1.0f / sqrtf(kk + a.eps) : 1.0f;
        srq[qr] = a.scale * (a.eps >= 0.0f && qr < n ? 1.0f / sqrtf(qq + a.eps) : 1.0f);
    }
    __syncthreads();
    v4f kt[TILES], qt[TILES];
#pragma unroll
    for (int j = 0; j < TILES; j++) {
        kt[j] = qt[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        if (j <= wave)
#pragma unroll
            for (int t = 0; t < NT; t++)
                kt[j] = mfma4(kv[t], *(const float4 *)&sk[16 * j + c][16 * t + 4 * g], kt[j]);
        if (j <= 3 - wave)
#pragma unroll
            for (int t = 0; t < NT; t++)
                qt[j] = mfma4(qv[t], *(const float4 *)&sk[16 * j + c][16 * t + 4 * g], qt[j]);
    }

    __syncthreads(); /* the keys' place is the matrices' now */

    const int heads = (int)(a.v_heads / a.k_heads);
    for (int hn = 0; hn < heads; hn++) {
        const long h = a.tiled ? kh + hn * a.k_heads : kh * heads + hn;
        float *mine = out + ((long)blockIdx.x * a.v_heads + h) * PREP, *factor = mine + 2 * PAIRS * 256;
        /* lane i of every wave: token i's gates */
        const float alpha = lane < n ? decay_of(a.a[(at + lane) * a.a_ld + h], a.dt[h], a.decay[h]) : 1.0f;
        if (wave == 0)
            sbeta[lane] = lane < n ? q8_sigmoid(a.b[(at + lane) * a.b_ld + h]) : 0.0f;
        {
            /* the decays between tokens: lane j has column j and goes down to the wave's rows */
            float d = 1.0f;
            for (int i = 0; i < 16 * wave; i++) {
                const float x = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, alpha), i));
                d = i <= lane ? 1.0f : d * x;
            }
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int i = 16 * wave + r;
                const float x = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, alpha), i));
                d = i <= lane ? 1.0f : d * x;
                sd[i][lane] = i >= lane ? d : 0.0f;
            }
        }
        __syncthreads();
        const float first_alpha = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, alpha), 0));
        const float gamma = sd[lane][0] * first_alpha; /* of token `lane` */
        if (wave == 0)
            factor[lane] = gamma * srk[lane];
        else if (wave == 1)
            factor[CHUNK + lane] = gamma * srq[lane];
        else if (wave == 2)
            factor[2 * CHUNK + lane] = sd[CHUNK - 1][lane] * srk[lane];
        else if (lane == CHUNK - 1)
            factor[3 * CHUNK] = gamma;
        /* A, and P, which takes the decays' place */
        const float4 bk = *(const float4 *)&sbeta[16 * wave + 4 * g] * *(const float4 *)&srk[16 * wave + 4 * g], qf = *(const float4 *)&srq[16 * (3 - wave) + 4 * g];
        const float *bf = &bk.x, *qs = &qf.x;
        float pr[TILES][4];
#pragma unroll
        for (int j = 0; j < TILES; j++) {
            const float rk = srk[16 * j + c];
            if (j <= wave)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int i = 16 * wave + 4 * g + r;
                    sa[i][16 * j + c] = i > 16 * j + c ? bf[r] * rk * kt[j][r] * sd[i][16 * j + c] : 0.0f;
                }
            if (j <= 3 - wave)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int i = 16 * (3 - wave) + 4 * g + r;
                    pr[j][r] = i >= 16 * j + c ? qs[r] * rk * qt[j][r] * sd[i][16 * j + c] : 0.0f;
                }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < TILES; j++)
            if (j <= 3 - wave)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    sd[16 * (3 - wave) + 4 * g + r][16 * j + c] = pr[j][r];
        {
            /* the diagonal's inverses: column c of block `wave` */
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                float4 row[4];
#pragma unroll
                for (int k = 0; k < i; k += 4)
                    row[k / 4] = *(const float4 *)&sa[16 * wave + i][16 * wave + k];
                float u[2] = {i == c ? 1.0f : 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < i; k++)
                    u[k & 1] = fmaf(-(&row[k / 4].x)[k & 3], x[k], u[k & 1]);
                x[i] = u[0] + u[1];
                if (g == 0)
                    st[16 * wave + i][16 * wave + c] = x[i];
            }
        }
        __syncthreads();
#pragma unroll
        for (int d = 1; d < TILES; d++) {
            if (wave < TILES - d) {
                const int i = wave + d, j = wave;
                v4f m = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < d; k++)
                    m = mfma4(*(const float4 *)&sa[16 * i + c][16 * (j + k) + 4 * g],
                              float4{st[16 * (j + k) + 4 * g][16 * j + c], st[16 * (j + k) + 4 * g + 1][16 * j + c], st[16 * (j + k) + 4 * g + 2][16 * j + c],
                                     st[16 * (j + k) + 4 * g + 3][16 * j + c]},
                              m);
                m = mfma4(*(const float4 *)&st[16 * i + c][16 * i + 4 * g], as4(m), v4f{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                for (int r = 0; r < 4; r++)
                    st[16 * i + 4 * g + r][16 * j + c] = -m[r];
            }
            __syncthreads();
        }
        bool finite = true;
        int pair = 0;
#pragma unroll
        for (int i = 0; i < TILES; i++)
#pragma unroll
            for (int j = 0; j <= i; j++, pair++)
                if (pair % 4 == wave) {
                    const float4 t = *(const float4 *)&st[16 * i + c][16 * j + 4 * g] * *(const float4 *)&sbeta[16 * j + 4 * g];
                    const float4 p = *(const float4 *)&sd[16 * i + c][16 * j + 4 * g];
                    finite = finite && finite4(t) && finite4(p);
                    *(float4 *)(mine + pair * 256 + lane * 4) = t;
                    *(float4 *)(mine + (PAIRS + pair) * 256 + lane * 4) = p;
                }
        const bool odd = __ballot(!finite) != 0;
        if (lane == 0)
            factor[3 * CHUNK + 4 + wave] = odd ? 1.0f : 0.0f;
        __syncthreads();
    }
}

/* A workgroup 16 columns of a sequence's head. Its waves' halves share a SIMD each: wave w < 4 has the keys of
 * tokens 16 w .. 16 w + 15 of a chunk and T's rows for them, wave 4 + w the queries of tokens 16 (3 - w) .. and P's
 * rows, so that each SIMD has the same number of matrix instructions (116 a chunk at k_dim 128), and wave v the state's
 * rows 16 v .., 16 (v + 8) ... The state stays in LDS from chunk to chunk. A chunk, with a barrier behind each
 * line (the second half's work stands in brackets):
 *
 *   R = V - gamma K S0
 *   d = T R, D_C d                                 [gamma Q S0]
 *   S = gamma_C S0 + K^T (D_C d)                   [the same, and O = gamma Q S0 + P d]
 *
 * What a wave needs of the next chunk is loaded as soon as this one's has been used. The workgroups of a head are
 * on one XCD, whose L2 then has K, Q, T and P for all of them.
 *
 * A chunk with anything that is not finite goes token by token: in the products 0 times a later token's NaN
 * would reach earlier ones. */
constexpr int CHUNK_THREADS = 512;

template <int DK>
__global__ __launch_bounds__(CHUNK_THREADS) void delta_chunk_k(rt_seqs b, rt_delta a, int most, long from, long count, const float *prep)
{
    constexpr int NT = DK / 16, LK = DK + 4;
    __shared__ __align__(16) float sk[CHUNK][LK];
    __shared__ __align__(16) float4 ss[NT][64], sr[TILES][64], sv[TILES][64], sw[TILES][64];
    __shared__ float red[5][8][16];
    __shared__ int sodd;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    const bool keys = wave < 4;
    const int tile = keys ? wave : 7 - wave;
    const int slices = (int)(a.v_dim / 16), x = (int)(blockIdx.x % 8), y = (int)(blockIdx.x / 8), slice = y % slices;
    const long unit = (long)(y / slices) * 8 + x, s = unit / a.v_heads, h = unit % a.v_heads;
    if (s >= b.n)
        return;
    const long kh = a.tiled ? h % a.k_heads : h / (a.v_heads / a.k_heads);
    long first, last;
    q8_rows_of(b, s, first, last);
    const long slot = slot_of(first, s), chunks = (last - first + CHUNK - 1) / CHUNK;
    const long c0 = from > slot ? from - slot : 0, c1 = from + count - slot < chunks ? from + count - slot : chunks;
    if (last - first <= most || c0 >= c1)
        return;
    const long col = 16 * slice + c, state = (s * a.v_heads + h) * DK * a.v_dim + col;
    const float *s_in = c0 == 0 ? a.s_in : a.s_out;
    for (int t = wave; t < NT; t += 8) {
        const float *p = s_in + state + (16 * t + 4 * g) * a.v_dim;
        ss[t][lane] = float4{p[0], p[a.v_dim], p[2 * a.v_dim], p[3 * a.v_dim]};
    }
    if (tid == 0)
        sodd = 0;

    /* the wave's rows of K or Q, of T or P, and their factors: of chunk n, whose rows behind the sequence are 0 */
    const float *rows = (keys ? a.k : a.q) + kh * DK + 4 * g, *values = a.v + h * a.v_dim + col;
    const long ld = keys ? a.k_ld : a.q_ld;
    float4 xv[NT], mv[TILES], factor, decay;
    float v[4], gamma, odd_in;
    const auto load_rows = [&](long n) {
        const long row = first + n * CHUNK + 16 * tile + c;
        const float *p = rows + (row < last ? row : first) * ld;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            xv[t] = *(const float4 *)(p + 16 * t);
            if (row >= last)
                xv[t] = float4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    };
    const auto part = [&](long n) { return prep + ((slot + n - from) * a.v_heads + h) * PREP; };
    const auto load_matrix = [&](long n) {
        const float *p = part(n) + ((keys ? 0 : PAIRS) + tile * (tile + 1) / 2) * 256 + lane * 4;
#pragma unroll
        for (int j = 0; j < TILES; j++)
            if (j <= tile)
                mv[j] = *(const float4 *)(p + j * 256);
    };
    const auto load_factors = [&](long n) {
        const float *p = part(n) + 2 * PAIRS * 256;
        factor = *(const float4 *)(p + (keys ? 0 : CHUNK) + 16 * tile + 4 * g);
        decay = *(const float4 *)(p + 2 * CHUNK + 16 * tile + 4 * g);
        gamma = p[3 * CHUNK];
        odd_in = p[3 * CHUNK + 4 + (wave & 3)];
        const long row = first + n * CHUNK + 16 * tile + 4 * g;
        if (keys)
#pragma unroll
            for (int r = 0; r < 4; r++)
                v[r] = row + r < last ? values[(row + r) * a.v_ld] : 0.0f;
    };
    load_rows(c0);
    load_factors(c0);
    load_matrix(c0);
    __syncthreads();
    for (long n = c0; n < c1; n++) {
        const long row = first + n * CHUNK + 16 * tile, next = n + 1 < c1 ? n + 1 : n;
        const auto with_state = [&]() {
            v4f z[2] = {v4f{0.0f, 0.0f, 0.0f, 0.0f}, v4f{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
            for (int t = 0; t < NT; t++)
                z[t & 1] = mfma4(xv[t], ss[t][lane], z[t & 1]);
            return z[0] + z[1];
        };
        const float end = gamma;
        float4 scaled = factor, left = decay;
        v4f mine = {0.0f, 0.0f, 0.0f, 0.0f};
        if (keys) {
#pragma unroll
            for (int t = 0; t < NT; t++)
                *(float4 *)&sk[16 * tile + c][16 * t + 4 * g] = xv[t];
            if (__ballot(odd_in != 0.0f || !finite4(float4{v[0], v[1], v[2], v[3]})) && lane == 0)
                sodd = 1;
            const v4f z = with_state();
            sr[tile][lane] = float4{fmaf(-scaled.x, z[0], v[0]), fmaf(-scaled.y, z[1], v[1]), fmaf(-scaled.z, z[2], v[2]), fmaf(-scaled.w, z[3], v[3])};
            load_rows(next);
        }
        load_factors(next);
        __syncthreads();
        if (sodd) {
            /* token by token: the thread has rows 16 t + 4 g .. + 3, t = wave, wave + 8, ..., of column c */
            const int tokens = (int)(last - (first + n * CHUNK) < CHUNK ? last - (first + n * CHUNK) : CHUNK);
            for (int j = 0; j < tokens; j++) {
                const long i = first + n * CHUNK + j;
                float sum[5] = {};
                for (int t = wave; t < NT; t += 8) {
                    const float4 kj = *(const float4 *)(a.k + i * a.k_ld + kh * DK + 16 * t + 4 * g), qj = *(const float4 *)(a.q + i * a.q_ld + kh * DK + 16 * t + 4 * g);
                    sum[0] += dot4(kj, ss[t][lane]), sum[1] += dot4(qj, ss[t][lane]);
                    sum[2] += dot4(kj, kj), sum[3] += dot4(qj, qj), sum[4] += dot4(qj, kj);
                }
                for (int k = 0; k < 5; k++) {
                    sum[k] = group_sum(sum[k]);
                    if (g == 0)
                        red[k][wave][c] = sum[k];
                }
                __syncthreads();
                for (int k = 0; k < 5; k++) {
                    sum[k] = 0.0f;
                    for (int w = 0; w < 8; w++)
                        sum[k] += red[k][w][c];
                }
                const float alpha = decay_of(a.a[i * a.a_ld + h], a.dt[h], a.decay[h]), beta = q8_sigmoid(a.b[i * a.b_ld + h]);
                const float rk = a.eps >= 0.0f ? 1.0f / sqrtf(sum[2] + a.eps) : 1.0f, rq = a.scale * (a.eps >= 0.0f ? 1.0f / sqrtf(sum[3] + a.eps) : 1.0f);
                const float d = beta * (a.v[i * a.v_ld + h * a.v_dim + col] - alpha * rk * sum[0]);
                if (tid < 16)
                    a.o[i * a.o_ld + h * a.v_dim + col] = fmaf(rq * alpha, sum[1], rq * (rk * sum[4]) * d);
                for (int t = wave; t < NT; t += 8) {
                    const float4 kj = *(const float4 *)(a.k + i * a.k_ld + kh * DK + 16 * t + 4 * g), o = ss[t][lane];
                    ss[t][lane] = float4{fmaf(rk * kj.x, d, alpha * o.x), fmaf(rk * kj.y, d, alpha * o.y), fmaf(rk * kj.z, d, alpha * o.z), fmaf(rk * kj.w, d, alpha * o.w)};
                }
                __syncthreads();
            }
            if (tid == 0)
                sodd = 0;
            if (!keys)
                load_rows(next);
            load_matrix(next);
            __syncthreads();
            continue;
        }
        if (keys) {
#pragma unroll
            for (int j = 0; j < TILES; j++)
                if (j <= tile)
                    mine = mfma4(mv[j], sr[j][lane], mine);
            sv[tile][lane] = as4(mine);
            sw[tile][lane] = as4(mine) * left;
            load_matrix(next);
        } else {
            mine = with_state();
            mine = v4f{scaled.x * mine[0], scaled.y * mine[1], scaled.z * mine[2], scaled.w * mine[3]};
            load_rows(next);
        }
        __syncthreads();
#pragma unroll
        for (int t0 = 0; t0 < NT; t0 += 8) {
            const int t = t0 + wave;
            if (t < NT) {
                const float4 o = ss[t][lane];
                v4f z[2] = {v4f{end * o.x, end * o.y, end * o.z, end * o.w}, v4f{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
                for (int j = 0; j < TILES; j++)
                    z[j & 1] = mfma4(float4{sk[16 * j + 4 * g][16 * t + c], sk[16 * j + 4 * g + 1][16 * t + c], sk[16 * j + 4 * g + 2][16 * t + c],
                                            sk[16 * j + 4 * g + 3][16 * t + c]},
                                     sw[j][lane], z[j & 1]);
                ss[t][lane] = as4(z[0] + z[1]);
            }
        }
        if (!keys) {
#pragma unroll
            for (int j = 0; j < TILES; j++)
                if (j <= tile)
                    mine = mfma4(mv[j], sv[j][lane], mine);
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (row + 4 * g + r < last)
                    a.o[(row + 4 * g + r) * a.o_ld + h * a.v_dim + col] = mine[r];
            load_matrix(next);
        }
        __syncthreads();
    }
    for (int t = wave; t < NT; t += 8) {
        float *p = a.s_out + state + (16 * t + 4 * g) * a.v_dim;
        const float4 z = ss[t][lane];
        p[0] = z.x, p[a.v_dim] = z.y, p[2 * a.v_dim] = z.z, p[3 * a.v_dim] = z.w;
    }
}

/* o <- nw * o / sqrt(eps + mean(o^2)) * SiLU(z), a wave a head of a token */
__global__ __launch_bounds__(256) void gated_norm_k(rt_seqs b, rt_delta a)
{
    const long i = blockIdx.x, h = 4 * (long)blockIdx.y + (threadIdx.x >> 6);
    if (q8_sequence_of(b, i) < 0 || h >= a.v_heads)
        return;
    const int lane = threadIdx.x & 63;
    float *o = a.o + i * a.o_ld + h * a.v_dim;
    const float *z = a.z + i * a.z_ld + h * a.v_dim;
    float sum = 0.0f;
    for (long c = lane; c < a.v_dim; c += 64)
        sum = fmaf(o[c], o[c], sum);
    const float r = 1.0f / sqrtf(a.nw_eps + q8_wave_sum(sum) / (float)a.v_dim);
    for (long c = lane; c < a.v_dim; c += 64)
        o[c] = a.nw[c] * (o[c] * r) * (z[c] * q8_sigmoid(z[c]));
}

} /* namespace */

/* Sequences of more tokens than this go in chunks */
constexpr int SHORT = 16;
/* The chunks' parts of all heads that a launch makes and takes, in bytes: longer calls alternate */
constexpr long PREP_MAX = 256L << 20;

static long slots_of(const rt_seqs &b) { return b.t / CHUNK + b.n; }
static long slots_a_launch(const rt_delta &a)
{
    const long n = PREP_MAX / (PREP_BYTES * a.v_heads);
    return n < 1 ? 1 : n;
}

long q8_delta_prep_floats(const rt_seqs &b, const rt_delta &a)
{
    const long all = slots_of(b), most = slots_a_launch(a);
    return b.longest > SHORT ? (all < most ? all : most) * a.v_heads * PREP : 0;
}

template <int DK>
static void launch_delta(hipStream_t s, const rt_seqs &b, const rt_delta &a, float *prep)
{
    const bool chunked = b.longest > SHORT;
    const dim3 grid((unsigned)(a.v_dim / 16), (unsigned)a.v_heads, (unsigned)b.n);
    delta_step_k<DK / 16><<<grid, 64, 0, s>>>(b, a, chunked ? SHORT : 0x7fffffff);
    if (!chunked)
        return;
    const long all = slots_of(b), most = slots_a_launch(a), units = (b.n * a.v_heads + 7) / 8 * 8;
    for (long from = 0; from < all; from += most) {
        const long count = all - from < most ? all - from : most;
        delta_prep_k<DK><<<dim3((unsigned)count, (unsigned)a.k_heads), 256, 0, s>>>(b, a, SHORT, from, prep);
        delta_chunk_k<DK><<<dim3((unsigned)(units * (a.v_dim / 16))), CHUNK_THREADS, 0, s>>>(b, a, SHORT, from, count, prep);
    }
}

void q8_launch_delta(q8_stream_t stream, const rt_seqs &b, const rt_delta &a, float *prep)
{
    const hipStream_t s = (hipStream_t)stream;
    switch (a.k_dim) {
#define KDIM(K)                                                                                                                                            \
    case K:                                                                                                                                                \
        launch_delta<K>(s, b, a, prep);                                                                                                                    \
        break;
        KDIM(32)
        KDIM(64)
        KDIM(96)
        KDIM(128)
        KDIM(192)
        KDIM(256)
#undef KDIM
    }
    if (a.z)
        gated_norm_k<<<dim3((unsigned)b.t, (unsigned)((a.v_heads + 3) / 4)), 256, 0, s>>>(b, a);
}
