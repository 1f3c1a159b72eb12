// Softmax attention with a bucketed relative position bias, forward: one pass over the keys with the running maximum and sum of every
// query row, scores and probabilities never in memory.
//
//   s2 = (scale q.k + bias) log2 e;   m' = max(m, max s2);   l' = l 2^(m - m') + sum 2^(s2 - m');   O' = O 2^(m - m') + 2^(s2 - m') V
//
// Workgroups: NQ waves of 32 query rows each (long sequences: 4, tiny ones: 1), or one 32-row tile whose keys are dealt to NK = 4
// waves and joined in LDS at the end (few rows over a long cache: bound by reading k and v, so a tile of 128 keys is in flight while
// the previous one is multiplied).  With few rows the key axis is also split over workgroups, whose (O, m, l) a second launch joins in
// split order.  Query heads that share a key head share a row tile there (row = query * G + head), so the cache is read once.
// Tiles whose keys are all padded, or all ahead of a causal row, are skipped without being read.
//
// Measured: bf16, 2 x 4095 tokens, 16 heads of 128, causal 205 us (137 GFLOP, 0.67 PFLOP/s: the matrix unit is busy half of the time, the
// exponentials of a wave run beside the products of its SIMD's other one); fp32, 16 x 1000 of 8 heads of 64 291 us (113 TFLOP/s, 0.74 of
// a large product's); one new token, 32 over 8 heads of 128, 25 rows of up to 4097 bf16 keys: 46 us for 210 MB (4.6 TB/s) and 4 us for the join.
// P is rounded to bf16 for the second product of bf16 calls (the matrix unit's operand type); sums, maxima and O stay fp32.  EXACT: what
// the rounding lost is multiplied too, and O's own rounding is kept beside the row statistics: the backward pass's sum dO . O needs O
// nearer than bf16 where a row has few keys (dq, dk and the bias gradient came out 1.5 - 1.8 times as far off as their own rounding puts
// them, with it 1.4).  The few-row kernels always do it (they wait for memory), the long one in training only and for the first 256 keys
// that a row meets: among more keys the roundings average out (2 x 4095 rows, 16 heads of 128, causal: 205 us without, 223 with, 247 for
// all keys).
#include "vita_attention.h"

namespace vita {
namespace {

constexpr int kExactTiles = 4;      // ... of 64 keys

template <class T, int DP, int NQ, int NK, int KW, bool EXACT>
__global__ __launch_bounds__(64 * NQ * NK, sizeof(T) == 4 && DP >= 96 ? 1 : 2) void attention_fwd_kernel(AttnParams p) {
    constexpr int NT = 64 * NQ * NK, KT = KW * NK, KS = lds_stride<T, DP>(), NC = DP / 16, ND = DP / 32, NS = KW / 32;
    constexpr bool AHEAD = NQ * NK > 1;      // the next tile is fetched while this one is multiplied; one-wave workgroups mostly have one tile
    extern __shared__ __attribute__((aligned(16))) char smem[];
    T* kt = reinterpret_cast<T*>(smem);
    T* vt = kt + KT * KS;
    float* ml = reinterpret_cast<float*>(vt + KT * KS);        // NK > 1: (NK, 32, 2)
    float* bias = ml + (NK > 1 ? NK * 64 : 0);
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wq = NK > 1 ? 0 : wave, wk = NK > 1 ? wave : 0;

    const int groups = p.H / p.pack;
    int pair, id;
    if (!pair_order(blockIdx.x, p.B * groups, p.tiles * p.splits, p.causal, pair, id)) return;
    const int split = id % p.splits, qt = p.causal ? p.tiles - 1 - id / p.splits : id / p.splits;       // the rows with the most keys first
    const int hy = pair % groups, b = pair / groups;
    const int rows = p.Sq * p.pack, head0 = hy * p.pack, kvh = head0 / p.G;

    const int row = (qt * NQ + wq) * 32 + col;
    const bool valid = row < rows;
    const int qi = min(row, rows - 1) / p.pack, g = min(row, rows - 1) - qi * p.pack;
    const int qpos = p.Sk - p.Sq + qi;
    // positions of the wave's first and last valid row, and of the workgroup's last
    const int first_row = (qt * NQ + wq) * 32;
    const int pos_lo = p.Sk - p.Sq + min(first_row, rows - 1) / p.pack, pos_hi = p.Sk - p.Sq + min(first_row + 31, rows - 1) / p.pack;
    const int wg_hi = p.Sk - p.Sq + min((qt + 1) * NQ * 32 - 1, rows - 1) / p.pack;

    Frag<T> q[NC];
    {
        const T* src = at<T>(p.q, b, qi, head0 + g);
#pragma unroll
        for (int c = 0; c < NC; ++c) q[c] = valid && c * 16 + half * 8 < p.D ? load8(src + c * 16 + half * 8) : zero8<T>();
    }
    const bool has_bias = p.table != nullptr;
    const int R = p.R, nb = 2 * R + 1;
    if (has_bias) load_bias<T>(p, bias, head0, p.pack, tid, NT);
    const float* my_bias = bias + g * nb;

    f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
    float m = -kInf, l = 0.f;

    const int limit = p.causal ? min(p.Sk, wg_hi + 1) : p.Sk;                  // keys that some row of the workgroup sees
    const int ntile = limit > 0 ? (limit + KT - 1) / KT : 0;
    const int t0 = split * p.tiles_per_split, t1 = min(ntile, t0 + p.tiles_per_split);
    KeyMask mask;
    mask.init(p, b);
    uint64_t m0 = 0, m1 = 0;
    auto next = [&](int t) {       // the first tile from t on that has a key
        for (; t < t1; ++t) {
            mask.tile<KT>(t, m0, m1);
            if ((m0 | m1) != 0) break;
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

    int t = next(t0);
    if (AHEAD && t < t1) fetch(t);
    [[maybe_unused]] int seen = 0;
    while (t < t1) {
        const uint64_t c0 = m0, c1 = m1;
        __syncthreads();           // the previous tile has been read by every wave
        if (!AHEAD) fetch(t);
        sk.store(kt, tid);
        sv.store(vt, tid);
        __syncthreads();
        const int tn = next(t + 1);
        if (AHEAD && tn < t1) fetch(tn);

        const int key0 = t * KT + wk * KW;
        const uint64_t bits = NK == 1 ? c0 : ((wk * KW < 64 ? c0 : c1) >> (wk * KW & 63)) & (KW == 64 ? ~uint64_t(0) : 0xffffffffu);
        if (bits != 0 && first_row < rows && !(p.causal && key0 > pos_hi)) {
            f32x16 s[NS];
#pragma unroll
            for (int n = 0; n < NS; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[n][r] = 0.f;
            pipelined<T, NC, NS>([&](int c, int n) { return row_frag<T, DP>(kt, wk * KW + n * 32 + col, c * 2 + half); },
                                 [&](int c, int n, const Frag<T>& a) { mma(s[n], a, q[c]); });
            const bool full = (KW == 64 ? bits == ~uint64_t(0) : (uint32_t)bits == 0xffffffffu) && !(p.causal && key0 + KW - 1 > pos_lo);
            const int far_lo = key0 + KW - 1 - pos_lo, far_hi = key0 - pos_hi;           // largest and smallest distance of the wave's tile
            // a tile that every row sees whole, its bias one number: the scale goes into the exponent's multiply-add
            float mul = p.scale_log2, add = 0.f;
            bool fold = full && p.scale_log2 > 0.f;
            if (has_bias && fold) {
                add = my_bias[far_lo <= -R ? 0 : 2 * R];
                fold = (far_lo <= -R || far_hi >= R) && __ballot(__builtin_fabsf(add) < kFoldBias) == ~uint64_t(0);
                if (!fold) add = 0.f;
            }
            if (!fold) {
                const uint64_t mine = bits >> (half * 4);
                const int see = p.causal ? qpos - key0 - half * 4 : 1 << 30;
#pragma unroll
                for (int n = 0; n < NS; ++n)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int k = n * 32 + acc_row(r, 0);
                        const float bv = has_bias ? my_bias[max(-R, min(R, key0 + half * 4 + k - qpos)) + R] : 0.f;
                        const float v = fmaf(s[n][r], mul, bv);
                        s[n][r] = ((mine >> k) & 1) != 0 && k <= see ? v : -kInf;
                    }
                mul = 1.f;
            }
            float top = s[0][0];
#pragma unroll
            for (int n = 0; n < NS; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) top = fmaxf(top, s[n][r]);
            top = fmaf(max_halves(top), mul, add);
            // the running maximum moves when a score passes it by 2^8: what is summed stays far inside fp32's range, and O is rarely rescaled
            if (__ballot(top > m + 8.f) != 0) {
                const float to = fmaxf(top, m);
                const float f = to == -kInf ? 0.f : __builtin_amdgcn_exp2f(m - to);
                l *= f;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[d][r] *= f;
                m = to;
            }
            const float shift = add - (m == -kInf ? 0.f : m);
            // fp32: a tile's product is summed by itself and then added, so that O's rounding grows with the number of tiles, not of key pairs:
            // dO . O, which the backward pass takes from every dS of a row, would carry it into the bias gradient's sums over all rows
            // (5 x 1954 rows and keys, 2 heads of 128: the table's gradient 1.4e-6 off, the chained plain form's 0.5e-6)
            f32x16 own[sizeof(T) == 4 ? ND : 1];
            f32x16* to = o;
            if constexpr (sizeof(T) == 4) {
                to = own;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) own[d][r] = 0.f;
            }
            // probabilities of 16 keys at a time, so that a step's exponentials run beside the previous step's products
            Frag<T> pf, rest;
            const bool near = NQ == 1 || seen++ < kExactTiles;
            pipelined<T, 2 * NS, ND>(
                [&](int i, int d) { return col_frag<T, DP>(vt, wk * KW + i * 16, d * 32, lane); },
                [&](int i, int d, const Frag<T>& a) {
                    if (d == 0) {
                        f32x16& sn = s[i >> 1];
                        float sum = 0.f;
#pragma unroll
                        for (int r = (i & 1) * 8; r < (i & 1) * 8 + 8; ++r) {
                            sn[r] = __builtin_amdgcn_exp2f(fmaf(sn[r], mul, shift));
                            sum += sn[r];
                        }
                        l += sum;
                        pf = pack8<T>(sn, i & 1);
                        if constexpr (EXACT)
                            if (near) rest = pack8_rest(sn, i & 1, pf);
                    }
                    mma(to[d], a, pf);
                    if constexpr (EXACT)
                        if (near) mma(to[d], a, rest);
                });
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[d][r] += own[d][r];
            }
        }
        t = tn;
    }
    l += __shfl_xor(l, 32, 64);

    const int64_t rec = ((int64_t)b * p.H + head0 + g) * p.Sq + qi;
    if constexpr (NK == 1) {                                    // (the keys are never split here)
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        if (valid) {
            T* dst = at_mut<T>(p.o, b, qi, head0 + g);
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const int c = d * 32 + acc_row(r, half);
                    if (c < p.D) {
                        const float v0 = o[d][r] * inv, v1 = o[d][r + 1] * inv, v2 = o[d][r + 2] * inv, v3 = o[d][r + 3] * inv;
                        store4<T>(dst + c, v0, v1, v2, v3);
                        if (sizeof(T) == 2 && p.stats != nullptr) store_rest4(p.stats + rec * p.stats_row, c, v0, v1, v2, v3);
                    }
                }
            if (half == 0 && p.stats != nullptr) store_stats<T>(p.stats + rec * p.stats_row, m == -kInf ? 0.f : m, inv);
        }
    } else {
        const int64_t nrec = (int64_t)p.B * p.H * p.Sq;
        // join the waves: every wave scales its O to the common maximum, the four are added in wave order
        if (half == 0) {
            ml[(wk * 32 + col) * 2] = m;
            ml[(wk * 32 + col) * 2 + 1] = l;
        }
        __syncthreads();
        float top = -kInf, total = 0.f;
#pragma unroll
        for (int w = 0; w < NK; ++w) top = fmaxf(top, ml[(w * 32 + col) * 2]);
        const float safe = top == -kInf ? 0.f : top;
#pragma unroll
        for (int w = 0; w < NK; ++w) total = fmaf(ml[(w * 32 + col) * 2 + 1], __builtin_amdgcn_exp2f(ml[(w * 32 + col) * 2] - safe), total);
        const float f = __builtin_amdgcn_exp2f(m - safe);
        float* buf = reinterpret_cast<float*>(smem);            // (NK, DP, 32): the tiles' room, which every wave has left
        static_assert(NK * DP * 32 * 4 <= 2 * KT * KS * (int)sizeof(T), "the join must fit the tiles' room");
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) buf[(wk * DP + d * 32 + acc_row(r, half)) * 32 + col] = o[d][r] * f;
        __syncthreads();
        const float scale = p.splits > 1 ? 1.f : (total == 0.f ? 0.f : 1.0f / total);
        if (valid) {
            T* dst = at_mut<T>(p.o, b, qi, head0 + g);
            float* part = p.splits > 1 ? p.part_o + (split * nrec + rec) * p.D : nullptr;
            for (int c = (wave * 2 + half) * 4; c < p.D; c += NK * 8) {
                float a[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    a[j] = buf[(c + j) * 32 + col];
#pragma unroll
                    for (int w = 1; w < NK; ++w) a[j] += buf[(w * DP + c + j) * 32 + col];
                    a[j] *= scale;
                }
                if (part != nullptr) {
                    store4<float>(part + c, a[0], a[1], a[2], a[3]);
                } else {
                    store4<T>(dst + c, a[0], a[1], a[2], a[3]);
                    if (sizeof(T) == 2 && p.stats != nullptr) store_rest4(p.stats + rec * p.stats_row, c, a[0], a[1], a[2], a[3]);
                }
            }
            if (wave == 0 && half == 0) {
                if (part != nullptr) {
                    p.part_ml[(split * nrec + rec) * 2] = top;
                    p.part_ml[(split * nrec + rec) * 2 + 1] = total;
                } else if (p.stats != nullptr) {
                    store_stats<T>(p.stats + rec * p.stats_row, safe, scale);
                }
            }
        }
    }
}

// the splits of a row, added in split order; D / 4 lanes a row
template <class T>
__global__ __launch_bounds__(256) void attention_join_kernel(AttnParams p) {
    const int per = p.D >> 2;
    const int64_t nrec = (int64_t)p.B * p.H * p.Sq, i = (int64_t)blockIdx.x * 256 + threadIdx.x, rec = i / per;
    if (rec >= nrec) return;
    const int c = (int)(i - rec * per) * 4;
    float top = -kInf;
    for (int s = 0; s < p.splits; ++s) top = fmaxf(top, p.part_ml[(s * nrec + rec) * 2]);
    const float safe = top == -kInf ? 0.f : top;
    float total = 0.f;
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < p.splits; ++s) {
        const float f = __builtin_amdgcn_exp2f(p.part_ml[(s * nrec + rec) * 2] - safe);
        total = fmaf(p.part_ml[(s * nrec + rec) * 2 + 1], f, total);
        const f32x4 v = *reinterpret_cast<const f32x4*>(p.part_o + (s * nrec + rec) * p.D + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = fmaf(v[j], f, a[j]);
    }
    const float inv = total == 0.f ? 0.f : 1.0f / total;
    const int64_t bh = rec / p.Sq;
    const int qi = (int)(rec - bh * p.Sq), b = (int)(bh / p.H), h = (int)(bh - (int64_t)b * p.H);
    store4<T>(at_mut<T>(p.o, b, qi, h) + c, a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv);
    if (p.stats != nullptr) {
        float* row = p.stats + rec * p.stats_row;
        if (sizeof(T) == 2) store_rest4(row, c, a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv);
        if (c == 0) store_stats<T>(row, safe, inv);
    }
}

// LDS of the form whose 4 waves share out the keys, with the bias of `pack` heads
size_t keys4_bytes(int dtype, int D, int pack, int R) { return tiles128_bytes(dtype, D, 2) + 4 * 64 * 4 + (size_t)pack * (2 * R + 1) * 4; }

enum { FWD_ROWS4 = 0, FWD_ROWS1 = 1, FWD_KEYS4 = 2 };
struct Plan { int mode, pack, rows, tiles, splits, tiles_per_split; int64_t blocks; };

Plan plan(const vita_attention_args* a) {
    Plan f{};
    const int G = a->H / a->Hk;
    // few rows of a head over many keys: the key axis is what there is to share out
    const bool few = (int64_t)a->Sq * G <= 64 && a->Sk > 128;
    const bool narrow = a->Sk > 128 && attention_narrow(a, (int64_t)(a->Sq + 127) / 128 * a->H * a->B);
    f.mode = few || narrow ? FWD_KEYS4 : (a->Sq <= 32 ? FWD_ROWS1 : FWD_ROWS4);
    // as many heads to a row tile as leave their biases room beside the tiles (fp32 heads of 128, a radius of 1024: 3)
    f.pack = few ? G : 1;
    if (a->table != nullptr)
        while (f.pack > 1 && (G % f.pack != 0 || keys4_bytes(a->dtype, a->D, f.pack, a->radius) > kLds)) --f.pack;
    f.rows = a->Sq * f.pack;
    const int per = f.mode == FWD_ROWS4 ? 128 : 32;
    f.tiles = (f.rows + per - 1) / per;
    f.splits = 1;
    const int64_t base = (int64_t)f.tiles * (a->H / f.pack) * a->B;
    const int ktiles = (a->Sk + 127) / 128;
    f.tiles_per_split = 1 << 30;
    if (few && base < 512 && ktiles > 1) {
        int64_t want = (768 + base - 1) / base;
        if (want > ktiles) want = ktiles;
        f.tiles_per_split = (int)((ktiles + want - 1) / want);
        f.splits = (ktiles + f.tiles_per_split - 1) / f.tiles_per_split;
    }
    f.blocks = pair_grid((int64_t)(a->H / f.pack) * a->B, f.tiles * f.splits);
    return f;
}

template <class T, int DP, int NQ, int NK, int KW, bool EXACT>
int launch(const AttnParams& p, int64_t blocks, hipStream_t s) {
    const size_t lds = (size_t)2 * KW * NK * lds_stride<T, DP>() * sizeof(T) + (NK > 1 ? NK * 64 * 4 : 0) +
                       (p.table != nullptr ? (size_t)p.pack * (2 * p.R + 1) * 4 : 0);
    VITA_REQUIRE(lds <= kLds, "vita_attention: %zu bytes of LDS", lds);
    auto kernel = attention_fwd_kernel<T, DP, NQ, NK, KW, EXACT>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(64 * NQ * NK), lds, s, p);
    VITA_CHECK_HIP(hipGetLastError());
    return VITA_OK;
}
template <class T, int DP>
int launch_mode(const AttnParams& p, const Plan& f, hipStream_t s) {
    constexpr bool BF = sizeof(T) == 2;
    if (f.mode == FWD_ROWS4) {
        if constexpr (BF)
            if (p.stats != nullptr) return launch<T, DP, 4, 1, 64, true>(p, f.blocks, s);
        return launch<T, DP, 4, 1, BF ? 64 : 32, false>(p, f.blocks, s);
    }
    if (f.mode == FWD_ROWS1) return launch<T, DP, 1, 1, 32, BF>(p, f.blocks, s);
    return launch<T, DP, 1, 4, 32, BF>(p, f.blocks, s);
}
template <class T>
int launch_type(const AttnParams& p, const Plan& f, hipStream_t s) {
    if (p.D <= 32) VITA_TRY((launch_mode<T, 32>(p, f, s)));
    else if (p.D <= 64) VITA_TRY((launch_mode<T, 64>(p, f, s)));
    else if (p.D <= 96) VITA_TRY((launch_mode<T, 96>(p, f, s)));
    else VITA_TRY((launch_mode<T, 128>(p, f, s)));
    if (f.splits > 1) {
        const int64_t n = (int64_t)p.B * p.H * p.Sq * (p.D / 4);
        hipLaunchKernelGGL(attention_join_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, p);
        VITA_CHECK_HIP(hipGetLastError());
    }
    return VITA_OK;
}

}  // namespace

bool attention_sizes_ok(const vita_attention_args* a) {
    return a != nullptr && a->B > 0 && a->Sq > 0 && a->Sk >= 0 && a->Sq <= (1 << 28) && a->Sk <= (1 << 28) && a->Hk >= 1 && a->H >= a->Hk &&
           a->H % a->Hk == 0 && (int64_t)a->Sq * (a->H / a->Hk) <= (1 << 28) && a->D >= 8 && a->D <= 128 && a->D % 8 == 0 &&
           ((a->table == nullptr && a->dtable == nullptr) || (a->radius >= 0 && a->radius <= kMaxRadius));
}

int attention_check(const vita_attention_args* a, bool bwd, const char* who) {
    VITA_REQUIRE(a != nullptr, "%s: null args", who);
    VITA_REQUIRE(a->dtype == VITA_DT_F32 || a->dtype == VITA_DT_BF16, "%s: unknown dtype %d", who, a->dtype);
    VITA_REQUIRE(a->B >= 0 && a->Sq >= 0 && a->Sk >= 0 && a->H >= 1 && a->Hk >= 1, "%s: bad shape B=%d Sq=%d Sk=%d H=%d Hk=%d", who, a->B, a->Sq, a->Sk,
                 a->H, a->Hk);
    VITA_REQUIRE(a->H % a->Hk == 0, "%s: %d query heads over %d key heads", who, a->H, a->Hk);
    VITA_REQUIRE(a->D >= 8 && a->D <= 128 && a->D % 8 == 0, "%s: head dimension %d (a multiple of 8, 8..128)", who, a->D);
    VITA_REQUIRE(a->Sq <= (1 << 28) && a->Sk <= (1 << 28) && (int64_t)a->Sq * (a->H / a->Hk) <= (1 << 28), "%s: sequence too long", who);
    VITA_REQUIRE(a->scale == a->scale && a->scale > -kInf && a->scale < kInf, "%s: bad scale", who);
    const int es = a->dtype == VITA_DT_F32 ? 4 : 2, vec = 16 / es;
    auto ok = [&](const void* q, int64_t b, int64_t t, int64_t h) {
        return q != nullptr && (reinterpret_cast<uintptr_t>(q) & 15u) == 0 && b % vec == 0 && t % vec == 0 && h % vec == 0;
    };
    VITA_REQUIRE((a->B == 0 || a->Sq == 0 || (ok(a->q, a->q_sb, a->q_ss, a->q_sh) && ok(a->o, a->o_sb, a->o_ss, a->o_sh))) &&
                     (a->B == 0 || a->Sk == 0 || (ok(a->k, a->k_sb, a->k_ss, a->k_sh) && ok(a->v, a->v_sb, a->v_ss, a->v_sh))),
                 "%s: q, k, v and o must be non-null, 16-byte aligned, with strides that are multiples of 16 bytes", who);
    VITA_REQUIRE((int64_t)a->k_ss < (1 << 23) && a->v_ss < (1 << 23) && a->q_ss < (1 << 23) && (!bwd || a->dout_ss < (1 << 23)) && a->k_ss >= 0 && a->v_ss >= 0 &&
                     a->q_ss >= 0 && (!bwd || a->dout_ss >= 0),
                 "%s: token strides must be below 2^23 elements", who);
    VITA_REQUIRE((reinterpret_cast<uintptr_t>(a->stats) & 15u) == 0, "%s: misaligned stats", who);
    VITA_REQUIRE(a->key_pad == nullptr || a->ld_pad == 0 || a->ld_pad >= a->Sk, "%s: bad ld_pad", who);
    if (a->table != nullptr) {
        VITA_REQUIRE(a->buckets != nullptr && a->radius >= 0 && a->radius <= kMaxRadius && a->num_buckets >= 1, "%s: bias with radius %d, %d buckets", who,
                     a->radius, a->num_buckets);
        VITA_REQUIRE((reinterpret_cast<uintptr_t>(a->table) & (es - 1)) == 0, "%s: misaligned bias table", who);
    }
    if (bwd) {
        VITA_REQUIRE(a->stats != nullptr && ok(a->dout, a->dout_sb, a->dout_ss, a->dout_sh) && ok(a->dq, a->dq_sb, a->dq_ss, a->dq_sh) &&
                         ok(a->dk, a->dk_sb, a->dk_ss, a->dk_sh) && ok(a->dv, a->dv_sb, a->dv_ss, a->dv_sh),
                     "%s: stats, dout, dq, dk and dv must be non-null, 16-byte aligned, with strides that are multiples of 16 bytes", who);
        VITA_REQUIRE(a->dtable == nullptr || a->table != nullptr, "%s: dtable without a table", who);
    }
    return VITA_OK;
}

void attention_fill(const vita_attention_args* a, AttnParams& p) {
    auto t = [](const void* q, int64_t b, int64_t s, int64_t h) { return AttnTensor{(char*)const_cast<void*>(q), b, s, h}; };
    p.q = t(a->q, a->q_sb, a->q_ss, a->q_sh); p.k = t(a->k, a->k_sb, a->k_ss, a->k_sh);
    p.v = t(a->v, a->v_sb, a->v_ss, a->v_sh); p.o = t(a->o, a->o_sb, a->o_ss, a->o_sh);
    p.stats = a->stats; p.stats_row = stats_row(a->dtype == VITA_DT_BF16, a->D); p.pad = a->key_pad; p.ld_pad = a->ld_pad;
    p.table = a->table; p.buckets = a->buckets; p.R = a->table != nullptr ? a->radius : 0; p.NB = a->num_buckets;
    p.B = a->B; p.H = a->H; p.Hk = a->Hk; p.G = a->H / a->Hk; p.Sq = a->Sq; p.Sk = a->Sk; p.D = a->D; p.causal = a->causal != 0;
    p.scale = a->scale; p.scale_log2 = a->scale * kLog2e;
    p.pack = 1; p.splits = 1;
}

}  // namespace vita

using namespace vita;

extern "C" {

int32_t vita_attention_stats_row(int32_t dtype, int32_t D) { return stats_row(dtype == VITA_DT_BF16, D); }

size_t vita_attention_workspace_bytes(const vita_attention_args* a) {
    if (!attention_sizes_ok(a)) return 0;
    const Plan f = plan(a);
    if (f.splits == 1) return 0;
    Carver c(nullptr);
    const size_t n = (size_t)f.splits * a->B * a->H * a->Sq;
    c.take(n * a->D);
    c.take(n * 2);
    return c.off;
}

int vita_attention(const vita_attention_args* a, void* workspace, size_t workspace_bytes, vita_stream_t stream) {
    const char* who = "vita_attention";
    VITA_TRY(attention_check(a, false, who));
    if (a->B == 0 || a->Sq == 0) return VITA_OK;
    VITA_TRY(check_ws(workspace, workspace_bytes, vita_attention_workspace_bytes(a), who));
    const Plan f = plan(a);
    VITA_REQUIRE(f.blocks < (int64_t(1) << 31) && (int64_t)a->B * a->H * a->Sq * (a->D / 4) < (int64_t(1) << 38), "%s: too many rows", who);
    AttnParams p{};
    attention_fill(a, p);
    p.pack = f.pack; p.tiles = f.tiles; p.splits = f.splits; p.tiles_per_split = f.tiles_per_split;
    if (f.splits > 1) {
        Carver c(workspace);
        const size_t n = (size_t)f.splits * a->B * a->H * a->Sq;
        p.part_o = c.take(n * a->D);
        p.part_ml = c.take(n * 2);
    }
    return a->dtype == VITA_DT_F32 ? launch_type<float>(p, f, (hipStream_t)stream) : launch_type<bf16>(p, f, (hipStream_t)stream);
}

}  // extern "C"
