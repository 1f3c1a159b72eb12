// Backward pass of the attention with a bucketed relative position bias.  With P from the saved row maxima and sums and dO the gradient of O:
//
//   delta_i = dO_i . O_i,   dP = dO V^T,   dS = P (dP - delta),   dQ = scale dS K,   dK = scale dS^T Q,   dV = P^T dO,
//   dtable[c, h] = sum over batch rows and pairs (i, j) with bucket c of dS
//
// Two kernels, each owning what it sums, so nothing is added by atomics and the bits do not depend on the run:
//   dq:  a wave owns 32 query rows and walks the keys (scores transposed as in the forward pass; also delta and the bias gradient);
//   dkv: a wave owns 32 keys and walks the query rows of every query head of its key head (scores untransposed, a lane owns one key).
// With few such workgroups the 4 waves of one share 32 rows (keys) and take a part of the other axis each; their sums are joined in LDS
// in wave order (attention_narrow in vita_attention.h).  Where 32 keys are all that the rows have, delta is sum P dP.
// Each forms S and dP again: 7 products of Sq x Sk x D against 5 for one kernel that would have to add dQ or dK, dV across workgroups.
// In both the second operand of the next product is the score tile's own registers (vita_attention.h), so P and dS never touch LDS.
//
// Measured: bf16, 2 x 4095 tokens, 16 heads of 128, causal: dq 317 us (206 GFLOP, 0.65 PFLOP/s), dkv 531 us (275 GFLOP, 0.52 PFLOP/s: its
// accumulators and k, v fragments leave one wave a SIMD, and the LDS serves 44 KB a wave and 32 x 32 scores, 1400 cycles of a CU for 4 waves
// against 1024 of the matrix units); fp32, 16 x 1000 of 8 heads of 64: both 1200 us (115 GFLOP, 96 TFLOP/s, 0.63 of a large product's).
//
// Bias gradient: a tile's dS is summed along its diagonals (one distance each) through 4 KB of LDS a wave, lane t taking diagonal t in
// row order; tiles wholly outside the radius add to one of two scalars a lane.  A workgroup writes one row of sums by distance, and a
// second launch adds the rows and gathers distances into buckets, both in index order.
//
// bf16 calls round P and dS to bf16 for the products that consume them; delta, statistics and sums are fp32.
#include "vita_attention.h"

namespace vita {
namespace {

constexpr int kDiag = 33;                                            // row stride of a wave's score tile in LDS
__host__ __device__ inline int dist_slots(int R) { return 2 * R + 1 + 124; }      // distances of a tile that touches the radius: -R - 62 .. R + 62

// what a wave's lanes wrote to LDS is read by its other lanes: LDS operations of a wave are served in order, the compiler must keep them so
__device__ __forceinline__ void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <class T, int DP, int NQ, int NK, int KT>
__global__ __launch_bounds__(64 * NQ * NK, (sizeof(T) == 4 && DP >= 64) || (NK > 1 && DP >= 96) ? 1 : 2) void attention_dq_kernel(AttnParams p) {
    constexpr int NW = NQ * NK, NT = 64 * NW, KS = lds_stride<T, DP>(), NC = DP / 16, ND = DP / 32;
    // the next tile is fetched while this one is multiplied; one-wave workgroups mostly have one tile, and 128 long fp32 rows do not fit registers
    constexpr bool AHEAD = NW > 1 && !(NK > 1 && sizeof(T) == 4 && DP > 96);
    constexpr bool EXACT = sizeof(T) == 2 && NQ == 1;      // few rows or keys: roundings do not average out, and there is time to multiply them too
    static_assert(NK == 1 || KT == NK * 32, "a wave has one block of 32 keys of a tile");
    // a row's dS has to sum to zero (not in bf16 of 128, which has no registers for it); what it does sum to is delta's rounding, which the far keys' bias gradient (P of it a row) and the
    // dkv kernel's delta are rid of afterwards (96 x 52 x 239 keys, 3 heads, radius 16: the table's gradient 1.8e-6 -> 0.4e-6 off).
    // dq and the near diagonals keep it, for that would take a product more: fp32 rows whose only two keys lie in different tiles come out
    // up to 1.1e-6 off, three keys 0.9e-6 (formed from P dP 0.3e-6)
    constexpr bool FIX = (sizeof(T) == 4 || DP < 128) && NW > 1;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    T* kt = reinterpret_cast<T*>(smem);
    T* vt = kt + KT * KS;
    float* bias = reinterpret_cast<float*>(vt + KT * KS);
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wq = wave / NK, wk = wave % NK;

    int bh, id;
    if (!pair_order(blockIdx.x, p.B * p.H, p.tiles, p.causal, bh, id)) return;
    const int qt = p.causal ? p.tiles - 1 - id : id;
    const int h = bh % p.H, b = bh / p.H, kvh = h / p.G;

    const int first_row = (qt * NQ + wq) * 32, row = first_row + col;
    const bool valid = row < p.Sq;
    const int qi = min(row, p.Sq - 1), qpos = p.Sk - p.Sq + qi;
    const int pos_lo = p.Sk - p.Sq + min(first_row, p.Sq - 1), pos_hi = p.Sk - p.Sq + min(first_row + 31, p.Sq - 1);
    const int wg_hi = p.Sk - p.Sq + min((qt + 1) * NQ * 32 - 1, p.Sq - 1);

    const int64_t rec = ((int64_t)b * p.H + h) * p.Sq + qi;
    Frag<T> q[NC], g[NC];
    float delta = 0.f;
    {
        const T* qs = at<T>(p.q, b, qi, h);
        const T* gs = at<T>(p.dout, b, qi, h);
        [[maybe_unused]] const T* os = at<T>(p.o, b, qi, h);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = c * 16 + half * 8;
            const bool in = valid && d < p.D;
            q[c] = in ? load8(qs + d) : zero8<T>();
            g[c] = in ? load8(gs + d) : zero8<T>();
            if constexpr (NW > 1) {
                const Frag<T> o = in ? load8(os + d) : zero8<T>();
#pragma unroll
                for (int j = 0; j < 8; ++j) delta = fmaf((float)g[c].v[j], (float)o.v[j], delta);
            }
            if constexpr (NW > 1 && sizeof(T) == 2) {                 // what o lost when it was rounded
                const Frag<T> rest = in ? load8(reinterpret_cast<const T*>(p.stats + rec * p.stats_row + 4) + d) : zero8<T>();
#pragma unroll
                for (int j = 0; j < 8; ++j) delta = fmaf((float)g[c].v[j], (float)rest.v[j], delta);
            }
        }
    }
    if constexpr (NW > 1) {
        delta += __shfl_xor(delta, 32, 64);
    }
    const float2 st = *reinterpret_cast<const float2*>(p.stats + rec * p.stats_row);
    [[maybe_unused]] const float top = st.x, inv = valid ? st.y : 0.f, dinv = delta * inv;      // dS = 2^(s - top) (dP inv - delta inv)

    const bool has_bias = p.table != nullptr, want = p.want_dtable != 0;
    const int R = p.R, nb = 2 * R + 1;
    float* diag = bias + (has_bias ? ((nb + 3) & ~3) : 0) + wave * (want ? 32 * kDiag + ((dist_slots(R) + 3) & ~3) : 0);
    float* dist = diag + 32 * kDiag;
    float far_lo = 0.f, far_hi = 0.f, left = 0.f, p_lo = 0.f, p_hi = 0.f;      // left: what the row's dS sums to; p: sums of P / inv over far keys
    if (has_bias) load_bias<T>(p, bias, h, 1, tid, NT);
    if (want)
        for (int i = lane; i < dist_slots(R); i += 64) dist[i] = 0.f;

    f32x16 dq[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) dq[d][r] = 0.f;

    const int limit = p.causal ? min(p.Sk, wg_hi + 1) : p.Sk;
    const int t1 = limit > 0 ? (limit + KT - 1) / KT : 0;
    KeyMask mask;
    mask.init(p, b);
    uint64_t m0 = 0, m1 = 0;
    auto next = [&](int t) {
        for (; t < t1; ++t) {
            mask.tile<KT>(t, m0, m1);
            if ((m0 | m1) != 0) break;               // tiles of 128 keys: two words
        }
        return t;
    };
    Stage<T, DP, KT, NT> sk, sv;
    sk.init(p.k.ss, tid);
    sv.init(p.v.ss, tid);
    const T* kbase = at<T>(p.k, b, 0, kvh);
    const T* vbase = at<T>(p.v, b, 0, kvh);
    auto fetch = [&](int t) {
        sk.load(kbase + (int64_t)t * KT * p.k.ss, m0, m1, p.D, tid);
        sv.load(vbase + (int64_t)t * KT * p.v.ss, m0, m1, p.D, tid);
    };
    int t = next(0);
    if (AHEAD && t < t1) fetch(t);
    [[maybe_unused]] bool first = true;
    while (t < t1) {
        const uint64_t c0 = m0, c1 = m1;
        __syncthreads();
        if (!AHEAD) fetch(t);
        sk.store(kt, tid);
        sv.store(vt, tid);
        __syncthreads();
        const int tn = next(t + 1);
        if (AHEAD && tn < t1) fetch(tn);
        // all the keys that these rows have lie in this tile's first 32 (bf16: one-wave kernels only, its long one has no registers to spare)
        const bool single = NW == 1 || (FIX && first && tn >= t1 && (c0 >> 32) == 0 && c1 == 0);
        first = false;
#pragma unroll
        for (int j = 0; j < KT / 32 / NK; ++j) {
            const int n = NK > 1 ? wk : j, key0 = t * KT + n * 32;
            const uint32_t bits = (uint32_t)((n < 2 ? c0 : c1) >> ((n & 1) * 32));
            if (bits == 0 || first_row >= p.Sq || (p.causal && key0 > pos_hi)) continue;      // (a wave behind the last row has nothing)
            f32x16 s, dp;
#pragma unroll
            for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = 0.f; }
            pipelined<T, NC, 2>([&](int c, int j) { return row_frag<T, DP>(j == 0 ? kt : vt, n * 32 + col, c * 2 + half); },
                                [&](int c, int j, const Frag<T>& a) { mma(j == 0 ? s : dp, a, j == 0 ? q[c] : g[c]); });
            const int dmax = key0 + 31 - pos_lo, dmin = key0 - pos_hi;
            const bool far = dmax <= -R || dmin >= R, full = bits == 0xffffffffu && !(p.causal && key0 + 31 > pos_lo);
            const float add = has_bias ? bias[dmax <= -R ? 0 : 2 * R] : 0.f;
            float psum = 0.f, ssum = 0.f;
            if (single) {
                // delta = sum P dP from the same P and dP, so that dS sums to zero over the row as it has to
                // (dO . O, rounded by itself, left dq and dk of 3 causal keys 1.3e-6 off where P and dP put them 0.2e-6)
                const uint32_t mine = bits >> (half * 4);
                const int see = p.causal ? qpos - key0 - half * 4 : 1 << 30;
                delta = 0.f;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int k = acc_row(r, 0);
                    const float bv = has_bias ? bias[max(-R, min(R, key0 + half * 4 + k - qpos)) + R] : 0.f;
                    const float v = __builtin_amdgcn_exp2f(fmaf(s[r], p.scale_log2, bv) - top) * inv;
                    const bool on = ((mine >> k) & 1) != 0 && k <= see;
                    s[r] = on ? v : 0.f;
                    dp[r] = on ? dp[r] : 0.f;
                    delta = fmaf(s[r], dp[r], delta);
                }
                delta += __shfl_xor(delta, 32, 64);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] *= dp[r] - delta;
            } else if (full && (!has_bias || (far && __builtin_fabsf(add) < kFoldBias))) {
                const float shift = add - top;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float e = __builtin_amdgcn_exp2f(fmaf(s[r], p.scale_log2, shift));
                    s[r] = e * fmaf(dp[r], inv, -dinv);
                    if constexpr (FIX) psum += e;
                }
            } else {
                const uint32_t mine = bits >> (half * 4);
                const int see = p.causal ? qpos - key0 - half * 4 : 1 << 30;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int k = acc_row(r, 0);
                    const float bv = has_bias ? bias[max(-R, min(R, key0 + half * 4 + k - qpos)) + R] : 0.f;
                    const bool on = ((mine >> k) & 1) != 0 && k <= see;
                    const float e = __builtin_amdgcn_exp2f(fmaf(s[r], p.scale_log2, bv) - top);
                    s[r] = on ? e * fmaf(dp[r], inv, -dinv) : 0.f;
                    if constexpr (FIX) psum += on ? e : 0.f;
                }
            }
            if (FIX || (want && far)) {
#pragma unroll
                for (int r = 0; r < 16; ++r) ssum += s[r];
                if constexpr (FIX) left += ssum;
            }
            {
                const Frag<T> df[2] = {pack8<T>(s, 0), pack8<T>(s, 1)};
                Frag<T> rest[2];
                if constexpr (EXACT) { rest[0] = pack8_rest(s, 0, df[0]); rest[1] = pack8_rest(s, 1, df[1]); }
                pipelined<T, 2, ND>([&](int c, int d) { return col_frag<T, DP>(kt, n * 32 + c * 16, d * 32, lane); },
                                    [&](int c, int d, const Frag<T>& a) {
                                        mma(dq[d], a, df[c]);
                                        if constexpr (EXACT) mma(dq[d], a, rest[c]);
                                    });
            }
            if (want) {
                if (far) {
                    if (dmax <= -R) { far_lo += ssum; p_lo += psum; }
                    else { far_hi += ssum; p_hi += psum; }
                } else {
                    // rows are queries here: lane t sums the elements (i, i + t - 31)
#pragma unroll
                    for (int r = 0; r < 16; ++r) diag[col * kDiag + acc_row(r, half)] = valid ? s[r] : 0.f;
                    wave_lds_order();
                    float a = 0.f;
                    const int off = lane - 31;
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const int j = i + off;
                        const float v = diag[i * kDiag + (j & 31)];
                        a += (j & ~31) == 0 ? v : 0.f;
                    }
                    wave_lds_order();
                    if (lane < 63) dist[key0 - (p.Sk - p.Sq + first_row) + off + R + 62] += a;
                }
            }
        }
        t = tn;
    }
    if constexpr (FIX) {
        left += __shfl_xor(left, 32, 64);
        if constexpr (NK > 1) {
            float* red = reinterpret_cast<float*>(smem);              // (NK, 32)
            __syncthreads();
            if (half == 0) red[wk * 32 + col] = left;
            __syncthreads();
            left = 0.f;
#pragma unroll
            for (int w = 0; w < NK; ++w) left += red[w * 32 + col];
        }
        far_lo -= p_lo * inv * left;
        far_hi -= p_hi * inv * left;
    }
    if (valid && half == 0 && wk == 0) p.delta[rec] = delta + left;
    if constexpr (NK > 1) {
        // the waves' sums are added in wave order
        static_assert(NK * DP * 32 * 4 <= 2 * KT * KS * (int)sizeof(T), "the join must fit the tiles' room");
        __syncthreads();
        float* buf = reinterpret_cast<float*>(smem);                  // (NK, DP, 32)
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) buf[(wk * DP + d * 32 + acc_row(r, half)) * 32 + col] = dq[d][r];
        __syncthreads();
        if (valid) {
            T* dst = at_mut<T>(p.dq, b, qi, h);
            for (int c = (wave * 2 + half) * 4; c < p.D; c += NK * 8) {
                float a[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    a[j] = 0.f;
#pragma unroll
                    for (int w = 0; w < NK; ++w) a[j] += buf[(w * DP + c + j) * 32 + col];
                }
                store4<T>(dst + c, a[0] * p.scale, a[1] * p.scale, a[2] * p.scale, a[3] * p.scale);
            }
        }
    } else if (valid) {
        T* dst = at_mut<T>(p.dq, b, qi, h);
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int c = d * 32 + acc_row(r, half);
                if (c < p.D) store4<T>(dst + c, dq[d][r] * p.scale, dq[d][r + 1] * p.scale, dq[d][r + 2] * p.scale, dq[d][r + 3] * p.scale);
            }
    }
    if (want) {
        far_lo = wave_sum(valid ? far_lo : 0.f);
        far_hi = wave_sum(valid ? far_hi : 0.f);
        wave_lds_order();
        if (lane == 0) {
            dist[R + 62 - R] += far_lo;       // distances -R and below, R and above
            dist[R + 62 + R] += far_hi;
        }
        __syncthreads();
        const int stride = 32 * kDiag + ((dist_slots(R) + 3) & ~3);
        const float* all = dist - wave * stride;
        float* out = p.dist_part + ((int64_t)(b * p.tiles + qt) * p.H + h) * nb;
        float lo = 0.f, hi = 0.f;                 // what lies beyond the radius belongs to its ends: 62 slots on either side
        if (wave == 0) {
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                lo += lane < 62 ? all[w * stride + lane] : 0.f;
                hi += lane < 62 ? all[w * stride + 2 * R + 63 + lane] : 0.f;
            }
            lo = wave_sum(lo);
            hi = wave_sum(hi);
        }
        for (int i = tid; i < nb; i += NT) {
            float a = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) a += all[w * stride + i + 62];
            if (i == 0) a += R > 0 ? lo : lo + hi;
            if (i != 2 * R || R == 0) out[i] = a;
        }
        if (tid == 0 && R > 0) {
            float a = hi;
#pragma unroll
            for (int w = 0; w < NW; ++w) a += all[w * stride + 2 * R + 62];
            out[2 * R] = a;
        }
    }
}

template <class T, int DP, int NB, int NR, int QT>
__global__ __launch_bounds__(64 * NB * NR, DP >= 64 ? 1 : 2) void attention_dkv_kernel(AttnParams p) {
    constexpr int NW = NB * NR, NT = 64 * NW, KS = lds_stride<T, DP>(), NC = DP / 16, ND = DP / 32;
    // the next tile is fetched while this one is multiplied; one-wave workgroups mostly have one tile, and 128 long fp32 rows do not fit registers
    constexpr bool AHEAD = NW > 1 && !(NR > 1 && sizeof(T) == 4 && DP > 64);
    constexpr bool EXACT = sizeof(T) == 2 && NW == 1;      // few keys: their roundings do not average out, and there is time to multiply them too
    constexpr int NBUF = NR > 1 ? 1 : 2, BUF = 2 * QT * KS;          // tiles in LDS; q and dO rows of a tile
    static_assert(NR == 1 || QT == NR * 32, "a wave has one block of 32 rows of a tile");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    T* tiles = reinterpret_cast<T*>(smem);
    float* stats = reinterpret_cast<float*>(tiles + NBUF * BUF);     // (NBUF, 3, QT): maximum, reciprocal sum, delta of the tiles' rows
    float* biases = stats + NBUF * 3 * QT;                                  // (2, 2 R + 1): of the current and the next query head
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    int bh, kt;
    if (!pair_order(blockIdx.x, p.B * p.Hk, p.tiles, p.causal, bh, kt)) return;
    const int kvh = bh % p.Hk, b = bh / p.Hk;
    const int wb = wave / NR, wr = wave % NR;
    const int key0 = (kt * NB + wb) * 32, key = key0 + col;
    const bool valid = key < p.Sk && (p.pad == nullptr || p.pad[(int64_t)b * p.ld_pad + key] == 0);
    const int wg_key0 = kt * NB * 32;

    Frag<T> k[NC], v[NC];
    {
        const T* ks = at<T>(p.k, b, min(key, p.Sk - 1), kvh);
        const T* vs = at<T>(p.v, b, min(key, p.Sk - 1), kvh);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = c * 16 + half * 8;
            k[c] = valid && d < p.D ? load8(ks + d) : zero8<T>();
            v[c] = valid && d < p.D ? load8(vs + d) : zero8<T>();
        }
    }
    f32x16 dk[ND], dv[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) { dk[d][r] = 0.f; dv[d][r] = 0.f; }

    const bool has_bias = p.table != nullptr, alive = __ballot(valid) != 0, whole = __ballot(valid) == ~uint64_t(0);
    const int R = p.R, back = p.Sk - p.Sq;
    // causal: query i sees the workgroup's first key from i = wg_key0 - back on
    const int q_first = p.causal ? max(0, wg_key0 - back) / QT : 0, q_tiles = (p.Sq + QT - 1) / QT;
    const int per = max(0, q_tiles - q_first);
    const int any = __syncthreads_or(alive);
    const int total = any ? per * p.G : 0;

    Stage<T, DP, QT, NT> sq, sg;
    sq.init(p.q.ss, tid);
    sg.init(p.dout.ss, tid);
    float2 st = make_float2(0.f, 0.f);
    float st_d = 0.f;
    auto fetch = [&](int i) {
        const int gi = i / per, h = kvh * p.G + gi, row0 = (q_first + i - gi * per) * QT;
        const int left = p.Sq - row0;
        const uint64_t m0 = left >= 64 ? ~uint64_t(0) : (uint64_t(1) << left) - 1;
        const uint64_t m1 = left >= 128 ? ~uint64_t(0) : (left > 64 ? (uint64_t(1) << (left - 64)) - 1 : 0);
        sq.load(at<T>(p.q, b, row0, h), m0, m1, p.D, tid);
        sg.load(at<T>(p.dout, b, row0, h), m0, m1, p.D, tid);
        if (tid < QT) {
            const int64_t rec = ((int64_t)b * p.H + h) * p.Sq + row0 + tid;
            // rows behind the last: 2^(anything - inf) = 0, whatever the bias
            st = tid < left ? *reinterpret_cast<const float2*>(p.stats + rec * p.stats_row) : make_float2(kInf, 0.f);
            st_d = tid < left ? p.delta[rec] : 0.f;
        }
    };
    // fp32 sums over many rows go to the output in parts of 512 rows (read back and added: 1 / 16 of a part's traffic), so that their
    // rounding does not grow with the sequence and the heads of a group: 4 heads x 4095 rows come out 0.6e-6 off, half of what one chain leaves
    constexpr int PART = 512 / QT;
    bool parted = false;
    auto store = [&](bool last) {
        if (key < p.Sk) {
            T* kd = at_mut<T>(p.dk, b, key, kvh);
            T* vd = at_mut<T>(p.dv, b, key, kvh);
            const float scale = last ? p.scale : 1.f;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const int c = d * 32 + acc_row(r, half);
                    if (c < p.D) {
                        float k4[4], v4[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            k4[j] = dk[d][r + j];
                            v4[j] = dv[d][r + j];
                            if constexpr (sizeof(T) == 4) {
                                if (parted) {
                                    k4[j] += kd[c + j];
                                    v4[j] += vd[c + j];
                                }
                            }
                        }
                        store4<T>(kd + c, k4[0] * scale, k4[1] * scale, k4[2] * scale, k4[3] * scale);
                        store4<T>(vd + c, v4[0], v4[1], v4[2], v4[3]);
                    }
                }
        }
        if (!last) {
            parted = true;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) { dk[d][r] = 0.f; dv[d][r] = 0.f; }
        }
    };
    // two tiles in LDS: tile i + 1 is written while others may still read tile i, one barrier a tile (one tile: two barriers)
    int have = -1;
    auto put = [&](int i) {
        T* t = tiles + i % NBUF * BUF;
        float* stat = stats + i % NBUF * 3 * QT;
        sq.store(t, tid);
        sg.store(t + QT * KS, tid);
        if (tid < QT) {
            stat[tid] = st.x;
            stat[QT + tid] = st.y;
            stat[2 * QT + tid] = st_d;
        }
        const int gi = i / per;
        if (has_bias && gi != have) {
            load_bias<T>(p, biases + (gi & 1) * (2 * R + 1), kvh * p.G + gi, 1, tid, NT);
            have = gi;
        }
    };
    if (total > 0) {
        fetch(0);
        put(0);
    }
    __syncthreads();
    auto part = [&](int i, int end) {
        for (; i < end; ++i) {
            const int gi = i / per, row0 = (q_first + i - gi * per) * QT;
            const T* qs = tiles + i % NBUF * BUF;
            const T* gs = qs + QT * KS;
            const float* stat = stats + i % NBUF * 3 * QT;
            const float* bias = biases + (gi & 1) * (2 * R + 1);
            if (AHEAD && i + 1 < total) fetch(i + 1);
#pragma unroll
            for (int j = 0; j < QT / 32 / NR; ++j) {
                const int n = NR > 1 ? wr : j;
                const int pos0 = back + row0 + n * 32;                     // position of the tile's first query
                if (!alive || row0 + n * 32 >= p.Sq || (p.causal && pos0 + 31 < key0)) continue;
                f32x16 s, dp;
#pragma unroll
                for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = 0.f; }
                {
                    Pipe<T, NC, 2, sizeof(T) == 2 ? 2 : 1> pipe;
                    auto read = [&](int c, int j) { return row_frag<T, DP>(j == 0 ? qs : gs, n * 32 + col, c * 2 + half); };
                    pipe.start(read);
                    pipe.run(read, [&](int c, int j, const Frag<T>& a) { mma(j == 0 ? s : dp, a, j == 0 ? k[c] : v[c]); });
                }
                // the transposed fragments of the first steps are on their way while the probabilities are formed
                Pipe<T, 4, ND, sizeof(T) == 2 ? 2 : 1> pipe;
                auto read = [&](int i, int d) { return col_frag<T, DP>((i & 1) == 0 ? gs : qs, n * 32 + (i >> 1) * 16, d * 32, lane); };
                pipe.start(read);
                const int dmax = key0 + 31 - pos0, dmin = key0 - pos0 - 31;
                const bool far = dmax <= -R || dmin >= R;
                const float add = has_bias ? bias[dmax <= -R ? 0 : 2 * R] : 0.f;
                if (whole && (!has_bias || (far && __builtin_fabsf(add) < kFoldBias)) && !(p.causal && key0 + 31 > pos0)) {
#pragma unroll
                    for (int r = 0; r < 16; r += 4) {
                        const f32x4 m4 = *reinterpret_cast<const f32x4*>(stat + n * 32 + acc_row(r, half));
                        const f32x4 i4 = *reinterpret_cast<const f32x4*>(stat + QT + n * 32 + acc_row(r, half));
                        const f32x4 d4 = *reinterpret_cast<const f32x4*>(stat + 2 * QT + n * 32 + acc_row(r, half));
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            s[r + j] = __builtin_amdgcn_exp2f(fmaf(s[r + j], p.scale_log2, add - m4[j])) * i4[j];
                            dp[r + j] = s[r + j] * (dp[r + j] - d4[j]);
                        }
                    }
                } else {
                    const int see = p.causal ? key - pos0 - half * 4 : -(1 << 30);       // rows from `see` on see this key
#pragma unroll
                    for (int r = 0; r < 16; r += 4) {
                        const f32x4 m4 = *reinterpret_cast<const f32x4*>(stat + n * 32 + acc_row(r, half));
                        const f32x4 i4 = *reinterpret_cast<const f32x4*>(stat + QT + n * 32 + acc_row(r, half));
                        const f32x4 d4 = *reinterpret_cast<const f32x4*>(stat + 2 * QT + n * 32 + acc_row(r, half));
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float bv = has_bias ? bias[max(-R, min(R, key - pos0 - acc_row(r + j, half))) + R] : 0.f;
                            // (rows without keys and behind the last: their distance's bias may be infinite or NaN)
                            const bool on = valid && acc_row(r + j, 0) >= see && i4[j] != 0.f;
                            const float pr = __builtin_amdgcn_exp2f(fmaf(s[r + j], p.scale_log2, bv) - m4[j]) * i4[j];
                            s[r + j] = on ? pr : 0.f;
                            dp[r + j] = on ? pr * (dp[r + j] - d4[j]) : 0.f;
                        }
                    }
                }
                const Frag<T> pf[2] = {pack8<T>(s, 0), pack8<T>(s, 1)}, df[2] = {pack8<T>(dp, 0), pack8<T>(dp, 1)};
                Frag<T> rest[4];
                if constexpr (EXACT) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) { rest[2 * c] = pack8_rest(s, c, pf[c]); rest[2 * c + 1] = pack8_rest(dp, c, df[c]); }
                }
                pipe.run(read, [&](int i, int d, const Frag<T>& a) {
                    f32x16& to = (i & 1) == 0 ? dv[d] : dk[d];
                    mma(to, a, (i & 1) == 0 ? pf[i >> 1] : df[i >> 1]);
                    if constexpr (EXACT) mma(to, a, rest[i]);
                });
            }
            if (i + 1 < total) {
                if (!AHEAD) fetch(i + 1);
                if (NBUF == 1) __syncthreads();
                put(i + 1);
            }
            __syncthreads();
        }
    };
    if constexpr (sizeof(T) == 4 && NR == 1) {
        for (int i = 0; i < total;) {
            const int end = min(total, i + PART);
            part(i, end);
            i = end;
            if (i < total) store(false);
        }
    } else part(0, total);
    if constexpr (NR == 1) {
        store(true);
    } else {
        // the waves' sums are added in wave order, dk's and then dv's
        static_assert(NR * DP * 32 * 4 <= BUF * (int)sizeof(T), "the join must fit the tiles' room");
        float* buf = reinterpret_cast<float*>(smem);                  // (NR, DP, 32)
        for (int which = 0; which < 2; ++which) {
            __syncthreads();
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) buf[(wr * DP + d * 32 + acc_row(r, half)) * 32 + col] = which == 0 ? dk[d][r] : dv[d][r];
            __syncthreads();
            if (key < p.Sk) {
                T* dst = at_mut<T>(which == 0 ? p.dk : p.dv, b, key, kvh);
                const float scale = which == 0 ? p.scale : 1.f;
                for (int c = (wr * 2 + half) * 4; c < p.D; c += NR * 8) {
                    float a[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        a[j] = 0.f;
#pragma unroll
                        for (int w = 0; w < NR; ++w) a[j] += buf[(w * DP + c + j) * 32 + col];
                    }
                    store4<T>(dst + c, a[0] * scale, a[1] * scale, a[2] * scale, a[3] * scale);
                }
            }
        }
    }
}

// the sums by distance of every (batch row, query tile), added in index order in kSeg segments ...
constexpr int kSeg = 32;
__global__ __launch_bounds__(256) void attention_dist_kernel(const float* part, float* seg, int parts, int H, int nb) {
    const int64_t n = (int64_t)H * nb, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int per = (parts + kSeg - 1) / kSeg, s0 = blockIdx.y * per, s1 = min(parts, s0 + per);
    float a = 0.f;
    for (int s = s0; s < s1; s += 8) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = s + j < s1 ? part[(s + j) * n + i] : 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) a += v[j];
    }
    seg[blockIdx.y * n + i] = a;
}
// ... then the segments (four groups of them a workgroup), and distances into buckets: 32 lanes a bucket, each adding every 32nd distance
template <class T>
__global__ __launch_bounds__(1024) void attention_bucket_kernel(const float* seg, const int32_t* buckets, int segs, int H, int nb, int NB, T* dtable) {
    extern __shared__ float sum[];                                     // (4, nb) sums, then (nb) bucket ids
    int* ids = reinterpret_cast<int*>(sum + 4 * nb);
    const int h = blockIdx.x, group = threadIdx.x >> 8, per = (segs + 3) / 4, s0 = group * per, s1 = min(segs, s0 + per);
    for (int i = threadIdx.x & 255; i < nb; i += 256) {
        const float* src = seg + (int64_t)h * nb + i;
        float a = 0.f;
        for (int s = s0; s < s1; s += 8) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = s + j < s1 ? src[(int64_t)(s + j) * H * nb] : 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) a += v[j];
        }
        sum[group * nb + i] = a;
        if (group == 0) ids[i] = buckets[i];
    }
    __syncthreads();
    const int l = threadIdx.x & 31;
    for (int c = threadIdx.x >> 5; c < NB; c += 32) {
        float a = 0.f;
        for (int i = l; i < nb; i += 32)
            if (ids[i] == c) a += (sum[i] + sum[nb + i]) + (sum[2 * nb + i] + sum[3 * nb + i]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) a += __shfl_xor(a, o, 64);
        if (l == 0) dtable[(int64_t)c * H + h] = (T)a;
    }
}

template <class T>
__global__ __launch_bounds__(256) void attention_zero_kernel(T* p, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = (T)0.f;
}

// queries or keys are none: every gradient is zero
template <class T>
__global__ __launch_bounds__(256) void attention_zero_rows_kernel(AttnTensor t, int S, int H, int D, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int d = (int)(i % D);
    const int64_t r = i / D, tok = r / H;
    const int h = (int)(r % H), b = (int)(tok / S);
    at_mut<T>(t, b, tok - (int64_t)b * S, h)[d] = (T)0.f;
}

// LDS of a dq workgroup beside its tiles: the bias by distance, and each wave's score tile and sums by distance
size_t dq_bias_bytes(bool table, bool want, int R, int waves) {
    return (table ? (size_t)((2 * R + 1 + 3) & ~3) * 4 : 0) + (want ? (size_t)waves * (32 * kDiag + ((dist_slots(R) + 3) & ~3)) * 4 : 0);
}

// q: query rows of a workgroup by 32, qk: waves that share them, a part of the keys each; k, kr: the same of keys and query rows
struct BPlan { int q, qk, k, kr, qtiles, ktiles; };
BPlan plan(const vita_attention_args* a) {
    BPlan f{};
    const int64_t qwide = (int64_t)(a->Sq + 127) / 128 * a->H * a->B, kwide = (int64_t)(a->Sk + 127) / 128 * a->Hk * a->B;
    const int64_t rows = (int64_t)a->Sq * (a->H / a->Hk);
    // (fp32 heads above 96 with the bias gradient of a radius from 244 on do not fit that form)
    const bool fits = tiles128_bytes(a->dtype, a->D, 2) + dq_bias_bytes(a->table != nullptr, a->dtable != nullptr, a->radius, 4) <= kLds;
    f.q = (a->Sk <= 32 ? a->Sq <= 32 : fits && (a->Sq <= 32 || attention_narrow(a, qwide))) ? 1 : 4;
    f.qk = f.q == 1 && a->Sk > 32 ? 4 : 1;
    f.k = a->Sk <= 32 || (rows > 32 && attention_narrow(a, kwide)) ? 1 : 4;
    f.kr = f.k == 1 && rows > 32 ? 4 : 1;
    f.qtiles = (a->Sq + 32 * f.q - 1) / (32 * f.q);
    f.ktiles = (a->Sk + 32 * f.k - 1) / (32 * f.k);
    return f;
}
size_t carve(const vita_attention_args* a, void* ws, float** delta, float** part, float** seg) {
    const BPlan f = plan(a);
    Carver c(ws);
    *delta = c.take((size_t)a->B * a->H * a->Sq);
    *part = *seg = nullptr;
    if (a->dtable != nullptr) {
        const size_t n = (size_t)a->H * (2 * a->radius + 1);
        *part = c.take((size_t)a->B * f.qtiles * n);
        *seg = c.take(kSeg * n);
    }
    return c.off;
}

template <class T, int DP, int NQ, int NK, int KT>
int launch_dq(const AttnParams& p, int64_t blocks, hipStream_t s) {
    constexpr int NW = NQ * NK;
    const size_t lds = (size_t)2 * KT * lds_stride<T, DP>() * sizeof(T) + dq_bias_bytes(p.table != nullptr, p.want_dtable != 0, p.R, NW);
    auto kernel = attention_dq_kernel<T, DP, NQ, NK, KT>;
    VITA_REQUIRE(lds <= kLds, "vita_attention_bwd: %zu bytes of LDS", lds);
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(64 * NW), lds, s, p);
    VITA_CHECK_HIP(hipGetLastError());
    return VITA_OK;
}
template <class T, int DP, int NB, int NR, int QT>
int launch_dkv(const AttnParams& p, int64_t blocks, hipStream_t s) {
    constexpr int NW = NB * NR, tiles = NR > 1 ? 1 : 2;
    const size_t lds = (size_t)2 * tiles * QT * lds_stride<T, DP>() * sizeof(T) + 3 * tiles * QT * 4 + (p.table != nullptr ? (size_t)(2 * p.R + 1) * 8 : 0);
    VITA_REQUIRE(lds <= kLds, "vita_attention_bwd: %zu bytes of LDS", lds);
    auto kernel = attention_dkv_kernel<T, DP, NB, NR, QT>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(64 * NW), lds, s, p);
    VITA_CHECK_HIP(hipGetLastError());
    return VITA_OK;
}
template <class T, int DP>
int launch_dp(const vita_attention_args* a, AttnParams p, const BPlan& f, hipStream_t s) {
    constexpr int T4 = sizeof(T) == 2 ? 64 : 32;
    constexpr int TQ = sizeof(T) == 2 && DP < 128 ? 64 : 32;      // dq at 128: with tiles of 64 keys the prefetch does not fit two waves a SIMD
    const int64_t qgrid = pair_grid((int64_t)a->H * a->B, f.qtiles), kgrid = pair_grid((int64_t)a->Hk * a->B, f.ktiles);
    p.tiles = f.qtiles;
    if (f.q == 4) VITA_TRY((launch_dq<T, DP, 4, 1, TQ>(p, qgrid, s)));
    else if (f.qk == 4) VITA_TRY((launch_dq<T, DP, 1, 4, 128>(p, qgrid, s)));
    else VITA_TRY((launch_dq<T, DP, 1, 1, 32>(p, qgrid, s)));
    p.tiles = f.ktiles;
    if (f.k == 4) return launch_dkv<T, DP, 4, 1, T4>(p, kgrid, s);
    if (f.kr == 4) return launch_dkv<T, DP, 1, 4, 128>(p, kgrid, s);
    return launch_dkv<T, DP, 1, 1, 32>(p, kgrid, s);
}
template <class T>
int run(const vita_attention_args* a, AttnParams& p, float* seg, hipStream_t s) {
    const int64_t nt = (int64_t)a->num_buckets * a->H;
    if (a->Sq == 0 || a->Sk == 0) {
        auto zero = [&](const AttnTensor& t, int S, int H) -> int {
            const int64_t n = (int64_t)a->B * S * H * a->D;
            if (n == 0) return VITA_OK;
            hipLaunchKernelGGL(attention_zero_rows_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, t, S, H, a->D, n);
            VITA_CHECK_HIP(hipGetLastError());
            return VITA_OK;
        };
        VITA_TRY(zero(p.dq, a->Sq, a->H));
        VITA_TRY(zero(p.dk, a->Sk, a->Hk));
        VITA_TRY(zero(p.dv, a->Sk, a->Hk));
        if (a->dtable != nullptr) {
            hipLaunchKernelGGL(attention_zero_kernel<T>, dim3((unsigned)((nt + 255) / 256)), dim3(256), 0, s, (T*)a->dtable, nt);
            VITA_CHECK_HIP(hipGetLastError());
        }
        return VITA_OK;
    }
    const BPlan f = plan(a);
    if (a->D <= 32) VITA_TRY((launch_dp<T, 32>(a, p, f, s)));
    else if (a->D <= 64) VITA_TRY((launch_dp<T, 64>(a, p, f, s)));
    else if (a->D <= 96) VITA_TRY((launch_dp<T, 96>(a, p, f, s)));
    else VITA_TRY((launch_dp<T, 128>(a, p, f, s)));
    if (a->dtable != nullptr) {
        const int nb = 2 * a->radius + 1, parts = a->B * f.qtiles;
        const int64_t n = (int64_t)a->H * nb;
        const bool two = parts > 8 * kSeg;                                 // few parts: the bucket kernel adds them itself
        if (two) {
            hipLaunchKernelGGL(attention_dist_kernel, dim3((unsigned)((n + 255) / 256), kSeg), dim3(256), 0, s, p.dist_part, seg, parts, a->H, nb);
            VITA_CHECK_HIP(hipGetLastError());
        }
        hipLaunchKernelGGL(attention_bucket_kernel<T>, dim3((unsigned)a->H), dim3(1024), (size_t)nb * 20, s, two ? seg : p.dist_part, a->buckets,
                           two ? kSeg : parts, a->H, nb, a->num_buckets, (T*)a->dtable);
        VITA_CHECK_HIP(hipGetLastError());
    }
    return VITA_OK;
}

}  // namespace
}  // namespace vita

using namespace vita;

extern "C" {

size_t vita_attention_bwd_workspace_bytes(const vita_attention_args* a) {
    if (!attention_sizes_ok(a) || a->Sk == 0) return 0;
    float *d, *p, *s;
    return carve(a, nullptr, &d, &p, &s);
}

int vita_attention_bwd(const vita_attention_args* a, void* workspace, size_t workspace_bytes, vita_stream_t stream) {
    const char* who = "vita_attention_bwd";
    VITA_TRY(attention_check(a, true, who));
    if (a->B == 0 && a->dtable == nullptr) return VITA_OK;
    VITA_REQUIRE(a->B > 0, "%s: an empty batch has no bias gradient to write", who);
    VITA_TRY(check_ws(workspace, workspace_bytes, vita_attention_bwd_workspace_bytes(a), who));
    VITA_REQUIRE(((int64_t)a->B * a->H + 8) * ((a->Sq > a->Sk ? a->Sq : a->Sk) / 32 + 1) < (int64_t(1) << 31), "%s: too many rows", who);
    AttnParams p{};
    attention_fill(a, p);
    auto t = [](const void* q, int64_t b, int64_t s, int64_t h) { return AttnTensor{(char*)const_cast<void*>(q), b, s, h}; };
    p.dout = t(a->dout, a->dout_sb, a->dout_ss, a->dout_sh); p.dq = t(a->dq, a->dq_sb, a->dq_ss, a->dq_sh);
    p.dk = t(a->dk, a->dk_sb, a->dk_ss, a->dk_sh); p.dv = t(a->dv, a->dv_sb, a->dv_ss, a->dv_sh);
    p.want_dtable = a->dtable != nullptr;
    float* seg = nullptr;
    if (a->Sq > 0 && a->Sk > 0) carve(a, workspace, &p.delta, &p.dist_part, &seg);
    return a->dtype == VITA_DT_F32 ? run<float>(a, p, seg, (hipStream_t)stream) : run<bf16>(a, p, seg, (hipStream_t)stream);
}

}  // extern "C"
