/* q8_delta.hip: the gated delta rule (include/q8_mix.h), and the norm and gate of its output. */
#include "q8_mix.h"

namespace {

/* The decay of a token's head. softplus as max(x, 0) + log1p(exp(-|x|)): no overflow. A decay near 1 rounded to F32 is off by
 * up to 2^-25, which is far more of 1 - decay: under a gate that stays as it is that error has one sign, and the
 * state, which remembers 1 / (1 - decay) tokens, would be off by it so many times. So it goes with what it is apart from
 * 1, which keeps its own 24 bits (8192 tokens at 1 - decay = 3e-4: the state is off by 2e-6, without it by 1.7e-4). */
struct decay {
    float all, rest; /* rest: all - 1 where all is near 1, else all again */
    __device__ __forceinline__ bool near() const { return rest != all; }
};
__device__ __forceinline__ decay decay_of(float a, float dt, float rate)
{
    const float x = a + dt, e = rate * (fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x))));
    if (fabsf(e) < 0.6875f) {
        /* e^x - 1 by its series: the next term is below 1e-8 of it */
        float y = fmaf(e, 1.0f / 362880, 1.0f / 40320);
        y = fmaf(e, fmaf(e, fmaf(e, y, 1.0f / 5040), 1.0f / 720), 1.0f / 120);
        y = fmaf(e, fmaf(e, fmaf(e, y, 1.0f / 24), 1.0f / 6), 0.5f);
        y = fmaf(e * e, y, e);
        return decay{1.0f + y, y};
    }
    const float all = expf(e);
    return decay{all, all};
}

__device__ __forceinline__ float dot4(float4 x, float4 y) { return fmaf(x.w, y.w, fmaf(x.z, y.z, fmaf(x.y, y.y, x.x * y.x))); }
/* nw * (o * r) * SiLU(z) */
__device__ __forceinline__ float4 gated(float4 o, float r, float4 w, float4 z)
{
    return float4{w.x * (o.x * r) * (z.x * q8_sigmoid(z.x)), w.y * (o.y * r) * (z.y * q8_sigmoid(z.y)), w.z * (o.z * r) * (z.z * q8_sigmoid(z.z)),
                  w.w * (o.w * r) * (z.w * q8_sigmoid(z.w))};
}

/* the sum over each group of G lanes (4, 8 or 16, aligned), in every lane of it */
template <int G>
__device__ __forceinline__ float lanes_sum(float v)
{
    v += Q8_DPP(v, 0xb1);
    v += Q8_DPP(v, 0x4e);
    if (G >= 8)
        v += Q8_DPP(v, 0x141);
    if (G >= 16)
        v += Q8_DPP(v, 0x140);
    return v;
}

/* Token by token. A wave owns COLS columns of a head's state, 4 a lane: lane RG c + g has rows g*KR .. g*KR + KR - 1 of
 * columns 4 c .. 4 c + 3, so a column's dot products go over RG neighbouring lanes. Both products with the state
 * are taken before it changes, in one reduction:
 *
 *   S' = alpha S + k d^T,  d = beta (v - alpha S^T k),  S'^T q = alpha S^T q + (q.k) d
 *
 * and so are |q|^2, |k|^2 and q.k, whose scales are applied to the results. The gates of 64 tokens are computed at
 * once, a lane a token. The next token's rows are loaded while this one's are used, and the state before anything is
 * known of the tokens. With the output's norm the head's waves are one workgroup (NORM), whose sums of
 * squares meet in LDS, and each lane gates one column; else each wave is a workgroup.
 * Bound by HBM (the state, read and written once) on many sequences, by latency on one. 32 columns a wave read whole
 * 128-byte lines (64 sequences of 32 heads of 128 x 128: 52 us, 5.3 TB/s; with 16 columns 76) and their stores
 * pass the caches, which would only lose other data to them (57 us otherwise); 16 columns have half the arithmetic a
 * token and lane, and twice the waves, where there are few. */
constexpr int STEP_WAVES = 8; /* of a workgroup, at most */
typedef float v4f __attribute__((ext_vector_type(4)));

template <int DK, int COLS, bool NORM>
__global__ __launch_bounds__(NORM ? 64 * STEP_WAVES : 64) void delta_step_k(rt_seqs b, rt_delta a, int most)
{
    constexpr int RG = 256 / COLS, KR = DK / RG, W = KR % 4 == 0 ? 4 : 2;
    __shared__ float squares[2][STEP_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, g = lane % RG;
    const long s = blockIdx.z, h = blockIdx.y, own = COLS * ((long)blockIdx.x * waves + wave) + 4 * (lane / RG), col = own < a.v_dim ? own : 0;
    const bool live = own < a.v_dim;
    const long kh = a.tiled ? h % a.k_heads : h / (a.v_heads / a.k_heads);
    const long base = ((s * a.v_heads + h) * DK + g * KR) * a.v_dim + col;
    float4 st[KR];
#pragma unroll
    for (int r = 0; r < KR; r++)
        st[r] = *(const float4 *)(a.s_in + base + r * a.v_dim);
    long first, last;
    q8_rows_of(b, s, first, last);
    if (last - first > most)
        return; /* in chunks */
    float q[KR], k[KR], qn[KR], kn[KR], z = 0.0f, zn = 0.0f;
    float4 v, vn;
    const auto load = [&](long i) {
        const float *qp = a.q + i * a.q_ld + kh * DK + g * KR, *kp = a.k + i * a.k_ld + kh * DK + g * KR;
#pragma unroll
        for (int r = 0; r < KR; r += W)
            if constexpr (W == 4)
                *(float4 *)(qn + r) = *(const float4 *)(qp + r), *(float4 *)(kn + r) = *(const float4 *)(kp + r);
            else
                *(float2 *)(qn + r) = *(const float2 *)(qp + r), *(float2 *)(kn + r) = *(const float2 *)(kp + r);
        vn = *(const float4 *)(a.v + i * a.v_ld + h * a.v_dim + col);
        if (NORM)
            zn = a.z[i * a.z_ld + h * a.v_dim + col + (g & 3)];
    };
    const float rate = a.decay[h], dt = a.dt[h];
    float ga = 0.0f, gb = 0.0f;
    if (first < last) {
        const long i = first + lane < last ? first + lane : first;
        ga = a.a[i * a.a_ld + h], gb = a.b[i * a.b_ld + h];
        load(first);
    }
    const float w = NORM ? a.nw[col + (g & 3)] : 0.0f;
    for (long i0 = first; i0 < last; i0 += 64) {
        if (i0 > first) {
            const long i = i0 + lane < last ? i0 + lane : i0;
            ga = a.a[i * a.a_ld + h], gb = a.b[i * a.b_ld + h];
        }
        const decay gate = decay_of(ga, dt, rate);
        const int alphas = __builtin_bit_cast(int, gate.all), rests = __builtin_bit_cast(int, gate.rest), betas = __builtin_bit_cast(int, q8_sigmoid(gb));
        const int count = (int)(last - i0 < 64 ? last - i0 : 64);
        for (int j = 0; j < count; j++) {
            const long i = i0 + j;
#pragma unroll
            for (int r = 0; r < KR; r++)
                q[r] = qn[r], k[r] = kn[r];
            v = vn, z = zn;
            load(i + 1 < last ? i + 1 : i);
            float rest = __builtin_bit_cast(float, __builtin_amdgcn_readlane(rests, j));
            const float alpha = __builtin_bit_cast(float, __builtin_amdgcn_readlane(alphas, j)), beta = __builtin_bit_cast(float, __builtin_amdgcn_readlane(betas, j));
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
            float rq = 1.0f, rk = 1.0f;
            if (a.eps >= 0.0f) {
                rq = rsqrtf(lanes_sum<RG>(qq) + a.eps);
                rk = rsqrtf(lanes_sum<RG>(kk) + a.eps);
            }
            qk = lanes_sum<RG>(qk);
            sk = float4{lanes_sum<RG>(sk.x), lanes_sum<RG>(sk.y), lanes_sum<RG>(sk.z), lanes_sum<RG>(sk.w)};
            sq = float4{lanes_sum<RG>(sq.x), lanes_sum<RG>(sq.y), lanes_sum<RG>(sq.z), lanes_sum<RG>(sq.w)};
            const float ak = alpha * rk;
            const float4 d = {beta * (v.x - ak * sk.x), beta * (v.y - ak * sk.y), beta * (v.z - ak * sk.z), beta * (v.w - ak * sk.w)};
            const float oq = a.scale * rq, od = oq * (rk * qk), oa = oq * alpha;
            const float4 o = {fmaf(oa, sq.x, od * d.x), fmaf(oa, sq.y, od * d.y), fmaf(oa, sq.z, od * d.z), fmaf(oa, sq.w, od * d.w)};
            if (NORM) {
                float sum = live ? dot4(o, o) : 0.0f;
#pragma unroll
                for (int m = RG; m < 64; m *= 2)
                    sum += __shfl_xor(sum, m, 64);
                if (lane == 0)
                    squares[j & 1][wave] = sum;
            }
            if (!decay{alpha, rest}.near()) {
#pragma unroll
                for (int r = 0; r < KR; r++)
                    st[r] *= alpha;
                rest = 0.0f;
            }
#pragma unroll
            for (int r = 0; r < KR; r++) {
                const float kr = rk * k[r];
                st[r] = float4{fmaf(kr, d.x, fmaf(rest, st[r].x, st[r].x)), fmaf(kr, d.y, fmaf(rest, st[r].y, st[r].y)), fmaf(kr, d.z, fmaf(rest, st[r].z, st[r].z)),
                               fmaf(kr, d.w, fmaf(rest, st[r].w, st[r].w))};
            }
            float *to = a.o + i * a.o_ld + h * a.v_dim + col;
            if (NORM) {
                __syncthreads();
                float sum = 0.0f;
                for (int n = 0; n < waves; n++)
                    sum += squares[j & 1][n];
                const float mine = (g & 2) ? (g & 1 ? o.w : o.z) : (g & 1 ? o.y : o.x);
                if (g < 4 && live)
                    to[g] = w * (mine * rsqrtf(a.nw_eps + sum / (float)a.v_dim)) * (z * q8_sigmoid(z));
            } else if (g == 0 && live) {
                *(float4 *)to = o;
            }
        }
    }
    if (live)
#pragma unroll
        for (int r = 0; r < KR; r++) {
            if (COLS == 32)
                __builtin_nontemporal_store(v4f{st[r].x, st[r].y, st[r].z, st[r].w}, (v4f *)(a.s_out + base + r * a.v_dim));
            else
                *(float4 *)(a.s_out + base + r * a.v_dim) = st[r];
        }
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
 * gamma rk, scale gamma rq and D_C rk of its tokens, gamma_C as 1 or 0 and the rest, and whether anything of it is not
 * finite (a wave each) */
constexpr int PREP = 2 * PAIRS * 256 + 4 * CHUNK;
/* a chunk's part in floats: its value heads', then each key head's rows of K and of Q as first operands lie, 256 floats
 * a tile of 16 rows and 16 columns. There consecutive lanes load consecutive 16 bytes; from the rows themselves each lane's
 * are in another row, and the vector cache takes a cycle for every lane. */
__host__ __device__ __forceinline__ long part_of(const rt_delta &a) { return a.v_heads * PREP + a.k_heads * 2 * CHUNK * a.k_dim; }
template <int DK>
__device__ __forceinline__ long rows_at(const rt_delta &a, long kh, int q, int tile) { return a.v_heads * PREP + ((kh * 2 + q) * TILES + tile) * 16 * DK; }

__device__ __forceinline__ v4f mfma4(float4 x, float4 y, v4f z)
{
    z = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x, y.x, z, 0, 0, 0);
    z = __builtin_amdgcn_mfma_f32_16x16x4f32(x.y, y.y, z, 0, 0, 0);
    z = __builtin_amdgcn_mfma_f32_16x16x4f32(x.z, y.z, z, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(x.w, y.w, z, 0, 0, 0);
}
__device__ __forceinline__ float4 as4(v4f x) { return float4{x[0], x[1], x[2], x[3]}; }
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

/* A product of decays as an unevaluated sum of two floats. gamma_C, which a state is multiplied by chunk after chunk, is
 * computed in these, and taken like a token's decay; the others reach a state once a token */
struct pair {
    float hi, lo;
};
__device__ __forceinline__ pair operator*(pair x, pair y)
{
    const float p = x.hi * y.hi;
    return pair{p, fmaf(x.hi, y.hi, -p) + fmaf(x.hi, y.lo, x.lo * y.hi)};
}

/* A workgroup a chunk and key head; wave w has key rows 16 w .. of K K^T and query rows 16 (3 - w) .. of Q K^T, five
 * tiles of 16 x 16 each, which the key head's value heads share. The inverse of each value head is 16 x 16 on the
 * diagonal by substitution, a column a lane, then by diagonals T_ij = -T_ii sum_k A_ik T_kj. Bound by HBM (8192 tokens of 16
 * and 32 heads of 128: 136 MB read and 222 written in 109 us, 3.3 TB/s; its matrix instructions take 20 us). */
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

    const int heads = (int)(a.v_heads / a.k_heads);
    const auto head = [&](int hn) { return a.tiled ? kh + hn * a.k_heads : kh * heads + hn; };
    float ga, gb, rate, dt; /* the next value head's gates of token `lane` */
    const auto load_gates = [&](int hn) {
        const long h = head(hn), i = at + (lane < n ? lane : 0);
        ga = a.a[i * a.a_ld + h], gb = a.b[i * a.b_ld + h], rate = a.decay[h], dt = a.dt[h];
    };
    float4 qv[NT], kv[NT];
    float kk = 0.0f, qq = 0.0f;
    const float *kp = a.k + (at + (kr < n ? kr : 0)) * a.k_ld + kh * DK + 4 * g, *qp = a.q + (at + (qr < n ? qr : 0)) * a.q_ld + kh * DK + 4 * g;
#pragma unroll
    for (int t = 0; t < NT; t++) {
        kv[t] = *(const float4 *)(kp + 16 * t);
        qv[t] = *(const float4 *)(qp + 16 * t);
    }
    load_gates(0);
    float *part = out + blockIdx.x * part_of(a);
#pragma unroll
    for (int t = 0; t < NT; t++) {
        kv[t] = kr < n ? kv[t] : float4{0.0f, 0.0f, 0.0f, 0.0f};
        qv[t] = qr < n ? qv[t] : float4{0.0f, 0.0f, 0.0f, 0.0f};
        *(float4 *)&sk[kr][16 * t + 4 * g] = kv[t];
        *(float4 *)(part + rows_at<DK>(a, kh, 0, wave) + t * 256 + lane * 4) = kv[t];
        *(float4 *)(part + rows_at<DK>(a, kh, 1, 3 - wave) + t * 256 + lane * 4) = qv[t];
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

    for (int hn = 0; hn < heads; hn++) {
        const long h = head(hn);
        float *mine = part + h * PREP, *factor = mine + 2 * PAIRS * 256;
        /* lane i of every wave: token i's gates */
        const decay gate = lane < n ? decay_of(ga, dt, rate) : decay{1.0f, 0.0f};
        const float alpha = gate.all;
        if (wave == 0)
            sbeta[lane] = lane < n ? q8_sigmoid(gb) : 0.0f;
        load_gates(hn + 1 < heads ? hn + 1 : hn);
        if (wave == 0) {
            /* gamma_C, with its rest: over each 16 lanes from the back, then the four first ones' */
#define LANE(v, old, ctrl) __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(old, __builtin_bit_cast(int, v), ctrl, 0xf, 0xf, false))
#define BEHIND(ctrl) all = all * pair{LANE(all.hi, 0x3f800000, ctrl), LANE(all.lo, 0, ctrl)}
            pair all = gate.near() ? pair{alpha, gate.rest - (alpha - 1.0f)} : pair{alpha, 0.0f};
            BEHIND(0x101);
            BEHIND(0x102);
            BEHIND(0x104);
            BEHIND(0x108);
#undef BEHIND
#undef LANE
            const auto of_lane = [&](int i) {
                return pair{__builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, all.hi), i)),
                            __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, all.lo), i))};
            };
            const pair whole = (of_lane(0) * of_lane(16)) * (of_lane(32) * of_lane(48));
            const bool near = whole.hi > 0.5f && whole.hi < 2.0f;
            if (lane == 0)
                *(float2 *)(factor + 3 * CHUNK) = float2{near ? 1.0f : 0.0f, near ? (whole.hi - 1.0f) + whole.lo : whole.hi + whole.lo};
        }
        {
            /* the decays between tokens, lane j with column j: up to the end of its own 16 rows by a scan from the
             * back, then by whole 16s, then down the wave's rows */
            const auto from = [](float v, int i) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), i)); };
            float rest = alpha; /* alpha_j .. of its 16, to the last */
#define BACK(ctrl) rest *= __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0x3f800000, __builtin_bit_cast(int, rest), ctrl, 0xf, 0xf, false))
            BACK(0x101); /* row_shl:1: from the lane behind, 1 beyond the row */
            BACK(0x102);
            BACK(0x104);
            BACK(0x108);
#undef BACK
            const float own = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0x3f800000, __builtin_bit_cast(int, rest), 0x101, 0xf, 0xf, false));
            float d = lane < 16 * wave ? own : 1.0f;
            for (int k = 1; k < wave; k++)
                d *= (lane >> 4) < k ? from(rest, 16 * k) : 1.0f;
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int i = 16 * wave + r;
                d = i <= lane ? 1.0f : d * from(alpha, i);
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
        /* A, and P, which takes the decays' place */
        const float4 bk = *(const float4 *)&sbeta[16 * wave + 4 * g] * *(const float4 *)&srk[16 * wave + 4 * g], qf = *(const float4 *)&srq[16 * (3 - wave) + 4 * g];
        const float *bf = &bk.x, *qs = &qf.x;
        float pr[TILES][4];
#pragma unroll
        for (int j = 0; j < TILES; j++) {
            const float rk = srk[16 * j + c];
            if (j <= wave) {
                float d[4];
#pragma unroll
                for (int r = 0; r < 4; r++)
                    d[r] = sd[16 * wave + 4 * g + r][16 * j + c];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float x = bf[r] * rk * kt[j][r] * d[r];
                    sa[16 * wave + 4 * g + r][16 * j + c] = 16 * wave + 4 * g + r > 16 * j + c ? x : 0.0f;
                }
            }
            if (j <= 3 - wave) {
                float d[4]; /* 0 behind the diagonal */
#pragma unroll
                for (int r = 0; r < 4; r++)
                    d[r] = sd[16 * (3 - wave) + 4 * g + r][16 * j + c];
#pragma unroll
                for (int r = 0; r < 4; r++)
                    pr[j][r] = qs[r] * rk * qt[j][r] * d[r];
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
        float4 check = {0.0f, 0.0f, 0.0f, 0.0f}; /* 0, or NaN */
#pragma unroll
        for (int k = 0; k < 3; k++) {
            const int pair = wave + 4 * k, i = pair < 1 ? 0 : pair < 3 ? 1 : pair < 6 ? 2 : 3, j = pair - i * (i + 1) / 2;
            if (pair < PAIRS) {
                const float4 t = *(const float4 *)&st[16 * i + c][16 * j + 4 * g] * *(const float4 *)&sbeta[16 * j + 4 * g];
                const float4 p = *(const float4 *)&sd[16 * i + c][16 * j + 4 * g];
                check = float4{fmaf(t.x, 0.0f, check.x), fmaf(t.y, 0.0f, check.y), fmaf(t.z, 0.0f, check.z), fmaf(t.w, 0.0f, check.w)};
                check = float4{fmaf(p.x, 0.0f, check.x), fmaf(p.y, 0.0f, check.y), fmaf(p.z, 0.0f, check.z), fmaf(p.w, 0.0f, check.w)};
                *(float4 *)(mine + pair * 256 + lane * 4) = t;
                *(float4 *)(mine + (PAIRS + pair) * 256 + lane * 4) = p;
            }
        }
        const bool odd = __ballot(!finite4(check)) != 0;
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
 *   R = V - gamma K S0                             [Q S0, half of it; O = Z + P d of the chunk before]
 *   d = T R, D_C d                                 [the other half: Z = gamma Q S0]
 *   S = gamma_C S0 + K^T (D_C d)                   [the same]
 *
 * What a wave needs of the next chunk is loaded as soon as this one's has been used. The workgroups of a head are
 * on one XCD, whose L2 then has K, Q, T and P for all of them. A chunk takes 2.7 us (8192 tokens of 32 heads, a workgroup a
 * compute unit), 1.5 of them the matrix instructions' own; the rest is what the three barriers leave waiting, which a
 * second workgroup on the compute unit, where the call has as many, fills in part.
 *
 * A chunk with anything that is not finite goes token by token: in the products 0 times a later token's NaN
 * would reach earlier ones. So do the chunks behind it: a way back into the loop would hold its registers meanwhile, and
 * there would be no second workgroup (16 heads of 1003, 963 and 692 tokens 72 us, 84 that way). A token there takes
 * 2.5 us (8192 tokens of which the first holds a NaN 20 ms). */
constexpr int CHUNK_THREADS = 512;
/* a launch has fewer than 2^32 threads along x: this many workgroups (whole eighths, for the XCDs), the others along y */
constexpr unsigned CHUNK_GRID = 1u << 22;

template <int DK>
struct chunk_lds {
    float sk[DK][CHUNK + 4];                                          /* the chunk's keys, transposed */
    float4 ss[DK / 16][64], sr[TILES][64], sv[TILES][64], sw[TILES][64]; /* S0, R, d, D_C d as results lie */
    float red[5][8][16];
    int odd;
};

/* A workgroup's unit: columns col - c .. + 15 of head h of sequence s, chunks [c0, c1) of it */
struct chunk_unit {
    long first, last, slot, h, kh, col, c0, c1;
    int slice, slices;
};

/* A chunk token by token, on the state in LDS: the thread has rows 16 t + 4 g .. + 3, t = wave, wave + 8, ..., of
 * column c */
template <int DK>
__device__ __forceinline__ void odd_chunk(const rt_delta &a, const chunk_unit &u, chunk_lds<DK> &m, long n)
{
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    const long from = u.first + n * CHUNK, to = from + CHUNK < u.last ? from + CHUNK : u.last;
    for (long i = from; i < to; i++) {
        const float *kp = a.k + i * a.k_ld + u.kh * DK + 4 * g, *qp = a.q + i * a.q_ld + u.kh * DK + 4 * g;
        float sum[5] = {};
        for (int t = wave; t < DK / 16; t += 8) {
            const float4 kj = *(const float4 *)(kp + 16 * t), qj = *(const float4 *)(qp + 16 * t);
            sum[0] += dot4(kj, m.ss[t][lane]), sum[1] += dot4(qj, m.ss[t][lane]);
            sum[2] += dot4(kj, kj), sum[3] += dot4(qj, qj), sum[4] += dot4(qj, kj);
        }
#pragma unroll
        for (int k = 0; k < 5; k++) {
            sum[k] = group_sum(sum[k]);
            if (g == 0)
                m.red[k][wave][c] = sum[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 5; k++) {
            sum[k] = 0.0f;
            for (int w = 0; w < 8; w++)
                sum[k] += m.red[k][w][c];
        }
        const decay gate = decay_of(a.a[i * a.a_ld + u.h], a.dt[u.h], a.decay[u.h]);
        const float alpha = gate.all, rest = gate.rest, keep = gate.near() ? 1.0f : 0.0f, beta = q8_sigmoid(a.b[i * a.b_ld + u.h]);
        const float rk = a.eps >= 0.0f ? 1.0f / sqrtf(sum[2] + a.eps) : 1.0f, rq = a.scale * (a.eps >= 0.0f ? 1.0f / sqrtf(sum[3] + a.eps) : 1.0f);
        const float d = beta * (a.v[i * a.v_ld + u.h * a.v_dim + u.col] - alpha * rk * sum[0]);
        if (tid < 16)
            a.o[i * a.o_ld + u.h * a.v_dim + u.col] = fmaf(rq * alpha, sum[1], rq * (rk * sum[4]) * d);
        for (int t = wave; t < DK / 16; t += 8) {
            const float4 kj = *(const float4 *)(kp + 16 * t), o = m.ss[t][lane];
            m.ss[t][lane] = float4{fmaf(rk * kj.x, d, fmaf(rest, o.x, keep * o.x)), fmaf(rk * kj.y, d, fmaf(rest, o.y, keep * o.y)),
                                   fmaf(rk * kj.z, d, fmaf(rest, o.z, keep * o.z)), fmaf(rk * kj.w, d, fmaf(rest, o.w, keep * o.w))};
        }
        __syncthreads();
    }
}

/* The chunks, as one half of the waves sees them: up to the last, or to one that is not finite, whose number it returns.
 * Every load of the next chunk is unconditional (rows of V behind the sequence's end are the chunk's first one again,
 * whose products go nowhere; those of K and Q are 0), and the halves have loops of their own: under a branch the
 * compiler no longer knows how many loads are in flight, and waits for those of the next chunk with this one's. */
template <int DK, bool KEYS>
__device__ __forceinline__ long chunk_loop(const rt_delta &a, const chunk_unit &u, chunk_lds<DK> &m, const float *prep)
{
    constexpr int NT = DK / 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const int tile = KEYS ? wave : 7 - wave;
    const long part = part_of(a);
    const float *rows = prep + u.slot * part + rows_at<DK>(a, u.kh, KEYS ? 0 : 1, tile) + lane * 4, *values = a.v + u.first * a.v_ld + u.h * a.v_dim + u.col;
    const float *matrix = prep + u.slot * part + u.h * PREP + ((KEYS ? 0 : PAIRS) + tile * (tile + 1) / 2) * 256 + lane * 4;
    const float *factors = prep + u.slot * part + u.h * PREP + 2 * PAIRS * 256;
    const long count = u.last - u.first;
    float4 xv[NT], mv[TILES], scale, left;
    float v[4], odd;
    float2 gamma;
    const auto load_rows = [&](long n) {
#pragma unroll
        for (int t = 0; t < NT; t++)
            xv[t] = *(const float4 *)(rows + n * part + t * 256);
        scale = *(const float4 *)(factors + n * part + (KEYS ? 0 : CHUNK) + 16 * tile + 4 * g);
        if constexpr (KEYS) {
            odd = factors[n * part + 3 * CHUNK + 4 + wave];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const long k = n * CHUNK + 16 * tile + 4 * g + r;
                v[r] = values[(k < count ? k : n * CHUNK) * a.v_ld];
            }
        }
    };
    const auto load_matrix = [&](long n) {
#pragma unroll
        for (int j = 0; j < TILES; j++)
            mv[j] = *(const float4 *)(matrix + n * part + (j < tile ? j : tile) * 256);
        if constexpr (KEYS)
            left = *(const float4 *)(factors + n * part + 2 * CHUNK + 16 * tile + 4 * g);
    };
    /* Into the XCD's L2, two chunks ahead: the head's workgroups there take a share of the chunk's lines each (128
     * bytes: its keys, its queries, its part of prep), and the last wave the rows of V that are its own. Loads that
     * find their lines there come back within a line of the chunk; from HBM they did not (8192 tokens, one workgroup a compute
     * unit: a quarter slower). */
    float ahead = 0.0f;
    const auto fetch = [&](long n) {
        constexpr int ROWS = 2 * CHUNK * DK / 32, SHARED = ROWS + PREP / 32;
        const long rest = count - n * CHUNK;
        const int l = u.slice + u.slices * ((wave - 4) * 64 + lane);
        const float *chunk = prep + (u.slot + n) * part, *p = nullptr;
        if (wave == 7)
            p = values + (n * CHUNK + (lane < rest ? lane : 0)) * a.v_ld - c;
        else if (l < SHARED)
            p = chunk + (l < ROWS ? rows_at<DK>(a, u.kh, 0, 0) + l * 32 : u.h * PREP + (l - ROWS) * 32);
        if (p)
            ahead = *p;
    };
    if constexpr (KEYS)
        __builtin_amdgcn_s_setprio(1); /* the chain from state to state is theirs */
    /* The queries' last product, of a chunk's P with its D, and the rows of O, are done a chunk later, while the keys have
     * their longest part: D stays in LDS until then. As the chunk's last part every wave waited for it. */
    v4f under_way = {0.0f, 0.0f, 0.0f, 0.0f};
    const auto finish = [&](long n) {
#pragma unroll
        for (int j = 0; j < TILES; j++)
            if (j <= tile)
                under_way = mfma4(mv[j], m.sv[j][lane], under_way);
        const int here = (int)(count - n * CHUNK < CHUNK ? count - n * CHUNK : CHUNK) - 16 * tile - 4 * g;
        float *o = a.o + (u.first + n * CHUNK + 16 * tile + 4 * g) * a.o_ld + u.h * a.v_dim + u.col;
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (r < here)
                o[r * a.o_ld] = under_way[r];
    };
    load_rows(u.c0);
    if constexpr (KEYS)
        load_matrix(u.c0);
    gamma = *(const float2 *)(factors + u.c0 * part + 3 * CHUNK);
    __syncthreads();
    bool whole = true; /* left at the loop's end only: a way out from its middle would let the compiler count fewer loads in flight */
    long n = u.c0;
    for (; n < u.c1 && whole; n++) {
        const long next = n + 1 < u.c1 ? n + 1 : n;
        v4f z = {0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (KEYS) {
            const int here = (int)(count - n * CHUNK < CHUNK ? count - n * CHUNK : CHUNK) - 16 * tile - 4 * g; /* rows from 4 g on that there are */
            v4f y[2] = {z, z};
#pragma unroll
            for (int t = 0; t < NT; t++) {
                y[t & 1] = mfma4(xv[t], m.ss[t][lane], y[t & 1]);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    m.sk[16 * t + 4 * g + e][16 * tile + c] = (&xv[t].x)[e];
            }
            y[0] += y[1];
            if (__ballot(odd != 0.0f || !finite4(float4{v[0], v[1], v[2], v[3]})) && lane == 0)
                m.odd = 1;
            m.sr[tile][lane] = float4{here > 0 ? fmaf(-scale.x, y[0][0], v[0]) : 0.0f, here > 1 ? fmaf(-scale.y, y[0][1], v[1]) : 0.0f,
                                      here > 2 ? fmaf(-scale.z, y[0][2], v[2]) : 0.0f, here > 3 ? fmaf(-scale.w, y[0][3], v[3]) : 0.0f};
            load_rows(next);
        } else {
            asm volatile("" : : "v"(ahead));
            fetch(n + 2 < u.c1 ? n + 2 : n);
#pragma unroll
            for (int t = 0; t < NT / 2; t++)
                z = mfma4(xv[t], m.ss[t][lane], z);
            if (n > u.c0)
                finish(n - 1);
            load_matrix(n);
        }
        __syncthreads();
        whole = __builtin_amdgcn_readfirstlane(m.odd) == 0;
        if constexpr (KEYS) {
#pragma unroll
            for (int j = 0; j < TILES; j++)
                if (j <= tile)
                    z = mfma4(mv[j], m.sr[j][lane], z);
            m.sv[tile][lane] = as4(z);
            m.sw[tile][lane] = as4(z) * left;
            load_matrix(next);
        } else {
#pragma unroll
            for (int t = NT / 2; t < NT; t++)
                z = mfma4(xv[t], m.ss[t][lane], z);
            under_way = v4f{scale.x * z[0], scale.y * z[1], scale.z * z[2], scale.w * z[3]};
            load_rows(next);
        }
        __syncthreads();
#pragma unroll
        for (int t0 = 0; t0 < NT; t0 += 8) {
            const int t = t0 + wave;
            if (t < NT) {
                const float4 o = m.ss[t][lane];
                v4f s[2] = {v4f{gamma.x * o.x, gamma.x * o.y, gamma.x * o.z, gamma.x * o.w}, v4f{gamma.y * o.x, gamma.y * o.y, gamma.y * o.z, gamma.y * o.w}};
#pragma unroll
                for (int j = 0; j < TILES; j++)
                    s[j & 1] = mfma4(*(const float4 *)&m.sk[16 * t + c][16 * j + 4 * g], m.sw[j][lane], s[j & 1]);
                if (whole)
                    m.ss[t][lane] = as4(s[0] + s[1]);
            }
        }
        gamma = *(const float2 *)(factors + next * part + 3 * CHUNK);
        __syncthreads();
    }
    if (!whole)
        return n - 1;
    if constexpr (!KEYS)
        finish(n - 1);
    return n;
}

/* WAVES: of a SIMD, 4 for two workgroups a compute unit, for which k_dim 128 has a few registers too many (smaller ones have
 * room as they are, larger ones none in LDS): 8 times 512 tokens of 32 heads, 8 workgroups a compute unit, 177 us, 200 with one
 * at a time; 8192 tokens, one workgroup, 380 and 354 */
template <int DK, int WAVES>
__global__ __launch_bounds__(CHUNK_THREADS, WAVES) void delta_chunk_k(rt_seqs b, rt_delta a, int most, long from, long count, const float *prep)
{
    __shared__ __align__(16) chunk_lds<DK> m;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    const int index = (int)(blockIdx.x + blockIdx.y * CHUNK_GRID), slices = (int)(a.v_dim / 16), x = index % 8, y = index / 8, slice = y % slices;
    const long unit = (long)(y / slices) * 8 + x, s = unit / a.v_heads;
    if (s >= b.n)
        return;
    chunk_unit u;
    u.h = unit % a.v_heads;
    u.kh = a.tiled ? u.h % a.k_heads : u.h / (a.v_heads / a.k_heads);
    q8_rows_of(b, s, u.first, u.last);
    const long slot = slot_of(u.first, s), chunks = (u.last - u.first + CHUNK - 1) / CHUNK;
    u.slot = slot - from; /* of chunk 0, in this launch's parts */
    u.c0 = from > slot ? from - slot : 0;
    u.c1 = from + count - slot < chunks ? from + count - slot : chunks;
    if (u.last - u.first <= most || u.c0 >= u.c1)
        return;
    u.col = 16 * slice + c;
    u.slice = slice, u.slices = slices;
    const long state = (s * a.v_heads + u.h) * DK * a.v_dim + u.col;
    const float *s_in = u.c0 == 0 ? a.s_in : a.s_out;
    for (int t = wave; t < DK / 16; t += 8) {
        const float *p = s_in + state + (16 * t + 4 * g) * a.v_dim;
        m.ss[t][lane] = float4{p[0], p[a.v_dim], p[2 * a.v_dim], p[3 * a.v_dim]};
    }
    if (tid == 0)
        m.odd = 0;
    for (long n = wave < 4 ? chunk_loop<DK, true>(a, u, m, prep) : chunk_loop<DK, false>(a, u, m, prep); n < u.c1; n++)
        odd_chunk(a, u, m, n);
    for (int t = wave; t < DK / 16; t += 8) {
        float *p = a.s_out + state + (16 * t + 4 * g) * a.v_dim;
        const float4 z = m.ss[t][lane];
        p[0] = z.x, p[a.v_dim] = z.y, p[2 * a.v_dim] = z.z, p[3 * a.v_dim] = z.w;
    }
}

/* o <- nw * o / sqrt(eps + mean(o^2)) * SiLU(z), the rows from the first sequence's first to the last one's last. LANES
 * lanes (a power of two) hold a head, 4 elements each, NV times, of NORM_RUN rows one after the other, all loaded
 * first. Bound by HBM: o and z once, o once (8192 rows of 32 heads of 128: 66 us, 6.1 TB/s). */
constexpr int NORM_RUN = 4;

template <int NV>
__global__ __launch_bounds__(256) void gated_norm_k(rt_seqs b, rt_delta a, int lanes)
{
    const int per = 256 / lanes, at = 4 * ((int)threadIdx.x & (lanes - 1));
    const long i0 = (long)blockIdx.x * NORM_RUN, own = (long)blockIdx.y * per + (int)threadIdx.x / lanes, h = own < a.v_heads ? own : 0;
    float4 o[NORM_RUN][NV], z[NORM_RUN][NV], w[NV];
#pragma unroll
    for (int k = 0; k < NORM_RUN; k++) {
        const long row = i0 + k < b.t ? i0 + k : i0;
#pragma unroll
        for (int n = 0; n < NV; n++) {
            const long c = h * a.v_dim + (at + 256 * n < a.v_dim ? at + 256 * n : 0);
            o[k][n] = *(const float4 *)(a.o + row * a.o_ld + c);
            z[k][n] = *(const float4 *)(a.z + row * a.z_ld + c);
        }
    }
#pragma unroll
    for (int n = 0; n < NV; n++)
        w[n] = *(const float4 *)(a.nw + (at + 256 * n < a.v_dim ? at + 256 * n : 0));
    const long first = b.start[0], last = b.start[b.n];
#pragma unroll
    for (int k = 0; k < NORM_RUN; k++) {
        float sum = 0.0f;
#pragma unroll
        for (int n = 0; n < NV; n++)
            sum += at + 256 * n < a.v_dim ? dot4(o[k][n], o[k][n]) : 0.0f;
        for (int m = lanes >> 1; m >= 1; m >>= 1)
            sum += __shfl_xor(sum, m, 64);
        const float r = 1.0f / sqrtf(a.nw_eps + sum / (float)a.v_dim);
        const long row = i0 + k;
        if (row < b.t && row >= first && row < last && own < a.v_heads)
#pragma unroll
            for (int n = 0; n < NV; n++)
                if (at + 256 * n < a.v_dim)
                    *(float4 *)(a.o + row * a.o_ld + h * a.v_dim + at + 256 * n) = gated(o[k][n], r, w[n], z[k][n]);
    }
}

} /* namespace */

/* Sequences of more tokens than this go in chunks (heads of 128 x 128, 32 of them, no norm; us token by token and in chunks: one
 * sequence of 24 tokens 21 / 27, of 32 26 / 27, of 48 38 / 27; 4 of 32 32 / 41, of 48 45 / 42; 16 of 32 79 / 94, of 48 114 / 95) */
constexpr int SHORT = 32;
/* The chunks' parts of all heads that a launch makes and takes, in bytes: longer calls alternate */
constexpr long PREP_MAX = 256L << 20;

static long slots_of(const rt_seqs &b) { return b.t / CHUNK + b.n; }
static long slots_a_launch(const rt_delta &a)
{
    const long n = PREP_MAX / (4 * part_of(a));
    return n < 1 ? 1 : n;
}

long q8_delta_prep_floats(const rt_seqs &b, const rt_delta &a)
{
    const long all = slots_of(b), most = slots_a_launch(a);
    return b.longest > SHORT ? (all < most ? all : most) * part_of(a) : 0;
}

/* true where the output's norm and gate were done with it */
template <int DK>
static bool launch_delta(hipStream_t s, const rt_seqs &b, const rt_delta &a, float *prep)
{
    const bool chunked = b.longest > SHORT;
    const int limit = chunked ? SHORT : 0x7fffffff;
    const auto waves = [&](int cols) { return (unsigned)((a.v_dim + cols - 1) / cols); };
    /* 16 columns a wave for several tokens, or as long as that gives no more waves than the GPU has places for two of
     * each SIMD */
    const bool few = b.longest > 1 || b.n * a.v_heads * waves(16) <= 2048;
    /* the norm in the same launch: for single tokens always (one sequence of 32 heads: 7.9 us, 7.7 to 9.9 as two launches),
     * for several where there is a head for every compute unit: with fewer, a head's waves share one, and a launch more costs
     * less (the same sequence, 8 tokens: 21 us and 14) */
    const bool normed = a.z && !chunked && waves(32) <= STEP_WAVES && (b.longest == 1 || b.n * a.v_heads >= 256);
    if (normed && few && waves(16) <= STEP_WAVES)
        delta_step_k<DK, 16, true><<<dim3(1, (unsigned)a.v_heads, (unsigned)b.n), 64 * waves(16), 0, s>>>(b, a, limit);
    else if (normed)
        delta_step_k<DK, 32, true><<<dim3(1, (unsigned)a.v_heads, (unsigned)b.n), 64 * waves(32), 0, s>>>(b, a, limit);
    else if (few)
        delta_step_k<DK, 16, false><<<dim3(waves(16), (unsigned)a.v_heads, (unsigned)b.n), 64, 0, s>>>(b, a, limit);
    else
        delta_step_k<DK, 32, false><<<dim3(waves(32), (unsigned)a.v_heads, (unsigned)b.n), 64, 0, s>>>(b, a, limit);
    if (!chunked)
        return normed;
    const long all = slots_of(b), most = slots_a_launch(a), units = (b.n * a.v_heads + 7) / 8 * 8;
    for (long from = 0; from < all; from += most) {
        const long count = all - from < most ? all - from : most;
        delta_prep_k<DK><<<dim3((unsigned)count, (unsigned)a.k_heads), 256, 0, s>>>(b, a, SHORT, from, prep);
        const long groups = units * (a.v_dim / 16);
        const dim3 grid((unsigned)(groups < CHUNK_GRID ? groups : CHUNK_GRID), (unsigned)((groups + CHUNK_GRID - 1) / CHUNK_GRID));
        if (DK == 128 && groups > 256)
            delta_chunk_k<DK, DK == 128 ? 4 : 2><<<grid, CHUNK_THREADS, 0, s>>>(b, a, SHORT, from, count, prep);
        else
            delta_chunk_k<DK, 2><<<grid, CHUNK_THREADS, 0, s>>>(b, a, SHORT, from, count, prep);
    }
    return false;
}

void q8_launch_delta(q8_stream_t stream, const rt_seqs &b, const rt_delta &a, float *prep)
{
    const hipStream_t s = (hipStream_t)stream;
    bool normed = false;
    switch (a.k_dim) {
#define KDIM(K)                                                                                                                                            \
    case K:                                                                                                                                                \
        normed = launch_delta<K>(s, b, a, prep);                                                                                                                  \
        break;
        KDIM(32)
        KDIM(64)
        KDIM(96)
        KDIM(128)
        KDIM(192)
        KDIM(256)
#undef KDIM
    }
    if (a.z && !normed) {
        int lanes = 4;
        while (lanes < 64 && 4 * lanes < a.v_dim)
            lanes *= 2;
        const dim3 grid((unsigned)((b.t + NORM_RUN - 1) / NORM_RUN), (unsigned)((a.v_heads * lanes + 255) / 256));
        if (a.v_dim > 256)
            gated_norm_k<2><<<grid, 256, 0, s>>>(b, a, lanes);
        else
            gated_norm_k<1><<<grid, 256, 0, s>>>(b, a, lanes);
    }
}
