// Norms of queries and keys over a head with the rotation in the same pass, forward and backward (the transformer blocks'
// attention: flare/models/attention.py:38-48, pos_embed.py:74-125).  Per row x of D elements (one head of one token):
//
//     n = (x - mean) * r, r = 1 / sqrt(var + eps)      VITA_NORM_LAYER        n = x * r, r = 1 / sqrt(mean(x^2) + eps)   VITA_NORM_RMS
//     t = n * weight + bias;     y[2i] = t[2i] c_i - t[2i+1] s_i,  y[2i+1] = t[2i+1] c_i + t[2i] s_i      (c, s: the row's position)
// backward, with d = the rotation's transpose applied to dy and e = d * weight:
//     dx = r * (e - mean(e) [LAYER] - n * mean(e * n)),   dweight = sum over rows of d * n,   dbias = sum over rows of d
//
// Bound by memory: forward reads and writes a row once, backward reads x and dy and writes dx; the statistics are formed again in
// the backward pass (a row sits in one group of lanes' registers), nothing is kept between the passes.  Everything is fp32 between
// the load and the one rounding at the store.
//
// A row belongs to a group of LPR lanes (a power of two), 16 bytes a lane, so a wave's loads are contiguous when the heads of a token
// are.  A lane keeps its columns' weight and bias in registers over the rows that its group walks.  The weight gradients: a lane sums
// its columns over its rows, a workgroup joins its groups through LDS and writes one partial row, a second launch adds the partial
// rows in index order: no atomics, the same bits every time.
//
// 2 x 8191 tokens, 32 + 8 heads of 128, bf16: forward 82 us (335 MB, 4.1 TB/s), backward 126 us (503 MB,
// 4.0 TB/s) and 5 us for the weights' partial rows; a copy of that size reaches 4.7 TB/s.  128 x 17 tokens of 16 heads of 64: launches.
#include "vita_host.h"

namespace vita {
namespace {

constexpr int RNT = 256;
// rows a group has in flight: enough to cover the latency at 4 workgroups a CU (backward: 2 leave room for those 4)
constexpr int rows_in_flight(bool bwd) { return bwd ? 2 : 4; }
constexpr int kMaxBlocks = 1024;       // backward: workgroups (4 a CU, shared out by the sides' rows), and partial rows of the weight gradients

template <class T> struct Vec;
template <> struct Vec<float> { static constexpr int N = 4; };
template <> struct Vec<__bf16> { static constexpr int N = 8; };

struct Side {
    const char* x; int64_t x_sb, x_ss, x_sh;
    char* y; int64_t y_sb, y_ss, y_sh;            // forward: the result; backward: dx
    const char* dy; int64_t dy_sb, dy_ss, dy_sh;
    const float* weight; const float* bias;
    float* partial;                               // backward: (blocks, 2, D)
    int H; unsigned rows;                         // rows = B * S * H < 2^31
    int blocks;
};
struct Params {
    Side side[2];
    int S, D, rope_heads;
    float eps;
    const float* rope; int64_t rope_rows;
    const int64_t* positions; int64_t ld_positions;
};

// a lane's columns of a row as they lie in memory; `wide` turns them into fp32 where they are used, so that the loads of several rows
// are in flight together at their own size
template <class T, int N> struct Raw { T v[N] __attribute__((aligned(16))); };
template <class T, int N, bool ALIGNED>
__device__ __forceinline__ void load_row(const char* base, int64_t off, int c0, int D, Raw<T, N>& r) {
    const T* p = reinterpret_cast<const T*>(base) + off + c0;
    if constexpr (ALIGNED) {
        const uint4 u = c0 < D ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
        r = __builtin_bit_cast(Raw<T , N>, u);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) r.v[j] = c0 + j < D ? p[j] : (T)0.f;
    }
}
template <class T, int N>
__device__ __forceinline__ void wide(const Raw<T, N>& r, float (&v)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (float)r.v[j];
}

template <class T, int N, bool ALIGNED>
__device__ __forceinline__ void store_row(char* base, int64_t off, int c0, int D, const float (&v)[N]) {
    T* p = reinterpret_cast<T*>(base) + off + c0;
    if constexpr (ALIGNED) {
        typedef T vec __attribute__((ext_vector_type(N)));
        if (c0 < D) {
            vec u;
#pragma unroll
            for (int j = 0; j < N; ++j) u[j] = (T)v[j];
            *reinterpret_cast<vec*>(p) = u;
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (c0 + j < D) p[j] = (T)v[j];
    }
}

template <int LPR>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// cos / sin of the lane's N / 2 pairs.  A position outside the table never leaves it: its row becomes NaN.
template <int N>
__device__ __forceinline__ void load_turn(const Params& p, int b, int s, int h, int c0, float2 (&t)[N / 2]) {
    const int64_t pos = p.positions != nullptr ? p.positions[(int64_t)b * p.ld_positions + s] : (int64_t)s;
    const bool in = pos >= 0 && pos < p.rope_rows;
    const int half = p.D >> 1;
    const float* src = p.rope + (((in ? pos : 0) * p.rope_heads + (p.rope_heads > 1 ? h : 0)) * half + (c0 >> 1)) * 2;
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
        const float2 v = c0 + 2 * j < p.D ? *reinterpret_cast<const float2*>(src + 2 * j) : make_float2(1.f, 0.f);
        t[j] = in ? v : make_float2(__builtin_nanf(""), __builtin_nanf(""));
    }
}

// n = normalised x (zero beyond D), r
template <int N, int LPR, bool LAYER>
__device__ __forceinline__ void normalise(float (&x)[N], int c0, int D, float eps, float& r) {
    const float inv = 1.0f / (float)D;
    if constexpr (LAYER) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < N; ++j) s += x[j];
        const float mean = group_sum<LPR>(s) * inv;
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = c0 + j < D ? x[j] - mean : 0.f;
    }
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) q = fmaf(x[j], x[j], q);
    r = 1.0f / sqrtf(fmaf(group_sum<LPR>(q), inv, eps));
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] *= r;
}

template <class T, int LPR, bool LAYER, bool ALIGNED, bool BWD>
__global__ __launch_bounds__(RNT) void norm_rope_kernel(Params p) {
    constexpr int N = Vec<T>::N, GPB = RNT / LPR, U = rows_in_flight(BWD);
    const bool second = (int)blockIdx.x >= p.side[0].blocks;
    const Side& sd = p.side[second];
    const int block = (int)blockIdx.x - (second ? p.side[0].blocks : 0);
    const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR, c0 = lane * N, D = p.D;

    float w[N], bias[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        w[j] = c0 + j < D ? (sd.weight != nullptr ? sd.weight[c0 + j] : 1.f) : 0.f;
        bias[j] = c0 + j < D && sd.bias != nullptr ? sd.bias[c0 + j] : 0.f;
    }
    float dw[N] = {}, db[N] = {};

    // U rows of a group at a time: their loads are in flight together, and where they are heads of one token under one table (H a
    // multiple of U) the token's place and its cos / sin are formed once
    const bool share = sd.H % U == 0, one_turn = share && p.rope_heads == 1;
    const uint64_t stride = (uint64_t)sd.blocks * GPB * U;
    for (uint64_t row0 = ((uint64_t)block * GPB + group) * U; row0 < sd.rows; row0 += stride) {
        Raw<T, N> xr[U], gr[BWD ? U : 1];
        float2 turn[U][N / 2];
        int b[U], s[U], h[U];
        const int n = sd.rows - (unsigned)row0 < U ? (int)(sd.rows - (unsigned)row0) : U;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u > 0 && share) {
                b[u] = b[0];
                s[u] = s[0];
                h[u] = h[0] + u;
            } else {
                const unsigned row = (unsigned)row0 + (u < n ? u : 0), tok = row / (unsigned)sd.H;
                h[u] = (int)(row - tok * sd.H);
                b[u] = (int)(tok / (unsigned)p.S);
                s[u] = (int)(tok - (unsigned)b[u] * p.S);
            }
            load_row<T, N, ALIGNED>(sd.x, (int64_t)b[u] * sd.x_sb + (int64_t)s[u] * sd.x_ss + (int64_t)h[u] * sd.x_sh, c0, D, xr[u]);
            if constexpr (BWD)
                load_row<T, N, ALIGNED>(sd.dy, (int64_t)b[u] * sd.dy_sb + (int64_t)s[u] * sd.dy_ss + (int64_t)h[u] * sd.dy_sh, c0, D, gr[u]);
            if (u == 0 || !one_turn) load_turn<N>(p, b[u], s[u], h[u], c0, turn[u]);
            else {
#pragma unroll
                for (int j = 0; j < N / 2; ++j) turn[u][j] = turn[0][j];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u >= n) break;
            float x[N], r;
            wide<T, N>(xr[u], x);
            normalise<N, LPR, LAYER>(x, c0, D, p.eps, r);
            const int64_t to = (int64_t)b[u] * sd.y_sb + (int64_t)s[u] * sd.y_ss + (int64_t)h[u] * sd.y_sh;
            float out[N];
            if constexpr (!BWD) {
#pragma unroll
                for (int j = 0; j < N / 2; ++j) {
                    const float c = turn[u][j].x, sn = turn[u][j].y;
                    const float t0 = fmaf(x[2 * j], w[2 * j], bias[2 * j]), t1 = fmaf(x[2 * j + 1], w[2 * j + 1], bias[2 * j + 1]);
                    out[2 * j] = fmaf(t0, c, -(t1 * sn));
                    out[2 * j + 1] = fmaf(t1, c, t0 * sn);
                }
            } else {
                float g[N], e_sum = 0.f, en_sum = 0.f;
                wide<T, N>(gr[u], g);
#pragma unroll
                for (int j = 0; j < N / 2; ++j) {
                    const float c = turn[u][j].x, sn = turn[u][j].y;
                    out[2 * j] = fmaf(g[2 * j], c, g[2 * j + 1] * sn);
                    out[2 * j + 1] = fmaf(g[2 * j + 1], c, -(g[2 * j] * sn));
                }
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    dw[j] = fmaf(out[j], x[j], dw[j]);
                    db[j] += out[j];
                    out[j] *= w[j];
                    e_sum += out[j];
                    en_sum = fmaf(out[j], x[j], en_sum);
                }
                const float inv = 1.0f / (float)D;
                const float en = group_sum<LPR>(en_sum) * inv;
                const float em = LAYER ? group_sum<LPR>(e_sum) * inv : 0.f;
#pragma unroll
                for (int j = 0; j < N; ++j) out[j] = r * (out[j] - em - x[j] * en);
            }
            store_row<T, N, ALIGNED>(sd.y, to, c0, D, out);
        }
    }
    if constexpr (BWD) {
        if (sd.partial == nullptr) return;
        __shared__ float part[GPB][2][LPR * N + 1];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            part[group][0][c0 + j] = dw[j];
            part[group][1][c0 + j] = db[j];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * D; i += RNT) {
            const int which = i >= D, col = i - which * D;
            float a = 0.f;
            for (int g = 0; g < GPB; ++g) a += part[g][which][col];
            sd.partial[((int64_t)block * 2 + which) * D + col] = a;
        }
    }
}

// the partial rows of a side, added in index order: 64 segments of rows a workgroup, 16 columns each, then the segments
struct ReduceSide { const float* partial; float* dweight; float* dbias; int blocks; };
__global__ __launch_bounds__(1024) void norm_rope_reduce_kernel(ReduceSide q, ReduceSide k, int D) {
    const ReduceSide& s = blockIdx.y ? k : q;
    __shared__ float part[64][17];
    const int col = blockIdx.x * 16 + (threadIdx.x & 15), seg = threadIdx.x >> 4;
    const int per = (s.blocks + 63) / 64, r0 = seg * per, r1 = min(s.blocks, r0 + per);
    float a = 0.f;
    if (col < 2 * D) {
        const float* src = s.partial + col;
        for (int r = r0; r < r1; r += 8) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = r + j < r1 ? src[(int64_t)(r + j) * 2 * D] : 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) a += v[j];
        }
    }
    part[seg][threadIdx.x & 15] = a;
    __syncthreads();
    if (seg == 0 && col < 2 * D) {
        float t = 0.f;
#pragma unroll
        for (int g = 0; g < 64; ++g) t += part[g][threadIdx.x & 15];
        if (col < D) {
            if (s.dweight != nullptr) s.dweight[col] = t;
        } else if (s.dbias != nullptr) {
            s.dbias[col - D] = t;
        }
    }
}

template <class T, int LPR, bool BWD>
void launch_lpr(const Params& p, bool layer, bool aligned, unsigned grid, hipStream_t s) {
    if (layer) {
        if (aligned) hipLaunchKernelGGL((norm_rope_kernel<T, LPR, true, true, BWD>), dim3(grid), dim3(RNT), 0, s, p);
        else hipLaunchKernelGGL((norm_rope_kernel<T, LPR, true, false, BWD>), dim3(grid), dim3(RNT), 0, s, p);
    } else {
        if (aligned) hipLaunchKernelGGL((norm_rope_kernel<T, LPR, false, true, BWD>), dim3(grid), dim3(RNT), 0, s, p);
        else hipLaunchKernelGGL((norm_rope_kernel<T, LPR, false, false, BWD>), dim3(grid), dim3(RNT), 0, s, p);
    }
}
template <class T, bool BWD>
void launch_t(const Params& p, int lpr, bool layer, bool aligned, unsigned grid, hipStream_t s) {
    switch (lpr) {
        case 2: launch_lpr<T, 2, BWD>(p, layer, aligned, grid, s); break;
        case 4: launch_lpr<T, 4, BWD>(p, layer, aligned, grid, s); break;
        case 8: launch_lpr<T, 8, BWD>(p, layer, aligned, grid, s); break;
        case 16: launch_lpr<T, 16, BWD>(p, layer, aligned, grid, s); break;
        case 32: launch_lpr<T, 32, BWD>(p, layer, aligned, grid, s); break;
        default: launch_lpr<T, 64, BWD>(p, layer, aligned, grid, s); break;
    }
}

int group_lanes(int dtype, int D) {
    const int vec = dtype == VITA_DT_F32 ? 4 : 8;
    int lpr = 2;
    while (lpr * vec < D) lpr *= 2;
    return lpr;
}

int side_blocks(const vita_norm_rope_args* a, int H, bool bwd) {
    const int gpb = RNT / group_lanes(a->dtype, a->D);
    const int64_t rows = (int64_t)a->B * a->S * H;
    const int64_t per = (int64_t)rows_in_flight(bwd) * gpb, want = (rows + per - 1) / per;
    if (!bwd) return (int)(want < 1 ? 1 : want);
    const int64_t most = kMaxBlocks * (int64_t)H / (a->q.H + a->k.H);
    return (int)(want < 1 || most < 1 ? 1 : (want > most ? most : want));
}

int check(const vita_norm_rope_args* a, bool bwd, const char* who) {
    VITA_REQUIRE(a != nullptr, "%s: null args", who);
    VITA_REQUIRE(a->dtype == VITA_DT_F32 || a->dtype == VITA_DT_BF16, "%s: unknown dtype %d", who, a->dtype);
    VITA_REQUIRE(a->norm == VITA_NORM_LAYER || a->norm == VITA_NORM_RMS, "%s: unknown norm %d", who, a->norm);
    VITA_REQUIRE(a->B >= 0 && a->S >= 0 && a->D >= 2 && a->D <= 256 && a->D % 2 == 0, "%s: bad shape B=%d S=%d D=%d (D even, 2..256)", who, a->B, a->S,
                 a->D);
    VITA_REQUIRE(a->q.H >= 1 && a->k.H >= 1, "%s: bad head counts %d / %d", who, a->q.H, a->k.H);
    VITA_REQUIRE((int64_t)a->B * a->S * (a->q.H > a->k.H ? a->q.H : a->k.H) < (int64_t(1) << 31), "%s: more than 2^31 rows (B * S * heads)", who);
    VITA_REQUIRE(a->rope != nullptr && a->rope_rows >= 1, "%s: no rotation table", who);
    VITA_REQUIRE((reinterpret_cast<uintptr_t>(a->rope) & 7u) == 0, "%s: the rotation table must be 8-byte aligned", who);
    VITA_REQUIRE(a->rope_heads == 1 || (a->rope_heads == a->q.H && a->rope_heads == a->k.H),
                 "%s: the rotation table has %d heads; 1 (shared) or the head count of both queries (%d) and keys (%d)", who, a->rope_heads, a->q.H, a->k.H);
    VITA_REQUIRE(a->positions != nullptr || a->S <= a->rope_rows, "%s: %d tokens, the rotation table has %lld positions", who, a->S,
                 (long long)a->rope_rows);
    VITA_REQUIRE(a->positions == nullptr || a->ld_positions == 0 || a->ld_positions >= a->S, "%s: bad ld_positions", who);
    const int es = a->dtype == VITA_DT_F32 ? 4 : 2;
    for (const vita_norm_rope_side* s : {&a->q, &a->k}) {
        VITA_REQUIRE(s->x != nullptr && s->y != nullptr && (!bwd || s->dy != nullptr), "%s: null tensor", who);
        for (const void* ptr : {s->x, (const void*)s->y, s->dy})
            VITA_REQUIRE((reinterpret_cast<uintptr_t>(ptr) & (es - 1)) == 0, "%s: misaligned tensor", who);
    }
    return VITA_OK;
}

bool side_aligned(const vita_norm_rope_args* a, const vita_norm_rope_side* s, bool bwd) {
    const int vec = a->dtype == VITA_DT_F32 ? 4 : 8;
    auto ok = [&](const void* q, int64_t b, int64_t t, int64_t h) {
        return (reinterpret_cast<uintptr_t>(q) & 15u) == 0 && b % vec == 0 && t % vec == 0 && h % vec == 0;
    };
    return a->D % vec == 0 && ok(s->x, s->x_sb, s->x_ss, s->x_sh) && ok(s->y, s->y_sb, s->y_ss, s->y_sh) &&
           (!bwd || ok(s->dy, s->dy_sb, s->dy_ss, s->dy_sh));
}

int run(const vita_norm_rope_args* a, bool bwd, void* ws, hipStream_t s) {
    Params p{};
    p.S = a->S; p.D = a->D; p.rope_heads = a->rope_heads; p.eps = a->eps; p.rope = a->rope; p.rope_rows = a->rope_rows;
    p.positions = a->positions; p.ld_positions = a->ld_positions;
    Carver c(ws);
    const vita_norm_rope_side* in[2] = {&a->q, &a->k};
    bool aligned = true, any = false;
    ReduceSide red[2] = {};
    for (int i = 0; i < 2; ++i) {
        Side& o = p.side[i];
        const vita_norm_rope_side& t = *in[i];
        o.x = (const char*)t.x; o.x_sb = t.x_sb; o.x_ss = t.x_ss; o.x_sh = t.x_sh;
        o.y = (char*)t.y; o.y_sb = t.y_sb; o.y_ss = t.y_ss; o.y_sh = t.y_sh;
        o.dy = (const char*)t.dy; o.dy_sb = t.dy_sb; o.dy_ss = t.dy_ss; o.dy_sh = t.dy_sh;
        o.weight = t.weight; o.bias = t.bias; o.H = t.H; o.rows = (unsigned)((int64_t)a->B * a->S * t.H);
        o.blocks = side_blocks(a, t.H, bwd);
        aligned = aligned && side_aligned(a, &t, bwd);
        if (bwd) {
            float* part = c.take((size_t)o.blocks * 2 * a->D);
            if (t.dweight != nullptr || t.dbias != nullptr) { o.partial = part; any = true; }
            red[i] = ReduceSide{part, t.dweight, t.dbias, o.partial != nullptr ? o.blocks : 0};
        }
    }
    const unsigned grid = (unsigned)(p.side[0].blocks + p.side[1].blocks);
    const int lpr = group_lanes(a->dtype, a->D);
    const bool layer = a->norm == VITA_NORM_LAYER;
    if (a->dtype == VITA_DT_F32) {
        if (bwd) launch_t<float, true>(p, lpr, layer, aligned, grid, s);
        else launch_t<float, false>(p, lpr, layer, aligned, grid, s);
    } else {
        if (bwd) launch_t<__bf16, true>(p, lpr, layer, aligned, grid, s);
        else launch_t<__bf16, false>(p, lpr, layer, aligned, grid, s);
    }
    VITA_CHECK_HIP(hipGetLastError());
    if (any) {
        hipLaunchKernelGGL(norm_rope_reduce_kernel, dim3((2 * a->D + 15) / 16, 2), dim3(1024), 0, s, red[0], red[1], a->D);
        VITA_CHECK_HIP(hipGetLastError());
    }
    return VITA_OK;
}

}  // namespace
}  // namespace vita

using namespace vita;

extern "C" {

int vita_qk_norm_rope(const vita_norm_rope_args* a, vita_stream_t stream) {
    VITA_TRY(check(a, false, "vita_qk_norm_rope"));
    if (a->B == 0 || a->S == 0) return VITA_OK;
    return run(a, false, nullptr, (hipStream_t)stream);
}

size_t vita_qk_norm_rope_bwd_workspace_bytes(const vita_norm_rope_args* a) {
    if (a == nullptr || a->B <= 0 || a->S <= 0 || a->D < 2 || a->D > 256 || a->q.H < 1 || a->k.H < 1) return 0;
    Carver c(nullptr);
    c.take((size_t)side_blocks(a, a->q.H, true) * 2 * a->D);
    c.take((size_t)side_blocks(a, a->k.H, true) * 2 * a->D);
    return c.off;
}

int vita_qk_norm_rope_bwd(const vita_norm_rope_args* a, void* workspace, size_t workspace_bytes, vita_stream_t stream) {
    const char* who = "vita_qk_norm_rope_bwd";
    VITA_TRY(check(a, true, who));
    VITA_REQUIRE(a->B > 0 && a->S > 0, "%s: no rows", who);
    VITA_TRY(check_ws(workspace, workspace_bytes, vita_qk_norm_rope_bwd_workspace_bytes(a), who));
    return run(a, true, workspace, (hipStream_t)stream);
}

}  // extern "C"
