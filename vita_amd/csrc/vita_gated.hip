// The gated feed-forward product h = act(x Wg^T + bg) * (x Wu^T + bu) and its backward pass (see include/vita_hip.h).
//
// bf16 products that fill the chip run on the 256 x 256 tile of vita_gemm_bf16_wide.h: a tile's columns are 128 features' gate and up
// projections, a wave's two column blocks the same 32 features, so both are in one lane's registers and the epilogue writes h alone.
// Backward: the same product again with another epilogue (reads dh, writes dz = [dg | du] in bf16 and fp32 partial sums for db), then
// dx = dz W and dw = dz^T x on the operands as they lie.  Forming z again trades time for memory: 8191 x 2048 x 8192 takes 647 us for it
// where z in fp32, written and read once, would move 1.07 GB (228 us at a copy's rate), but nothing is kept between the passes (z is 8 M F
// bytes, 0.54 GB there, four times h; in bf16 it would round the slopes' arguments).  dz is rounded to bf16 because the matrix unit takes
// bf16 operands; db is summed before that rounding.
// Up to 64 bf16 rows: a kernel of its own, bound by reading the weights once.
// Everything else goes over z (M, 2F) in fp32 with the library's GEMMs and one elementwise pass: fp32 (where the product runs at a
// sixteenth of the rate and saving z is the cheap choice) and small bf16 calls.
//
// Measured, median (best) of ten: bf16 8191 x 2048 x 8192 577 (533) us forward, 647 (600) dz, 511 (467) dx, 559 (511) dw (550 GFLOP each,
// 0.85 - 1.08 PFLOP/s); fp32 2176 x 512 x 2048 116 us z (79 TFLOP/s), 11 us h, 20 us dz, 5 us db, 6 + 107 + 7 us dx, 94 + 8 us dw; few
// rows 25 x 2048 x 8192 bf16 18 us (67 MB, 3.7 TB/s).
#include <type_traits>

#include "vita_gemm_bf16_wide.h"

namespace vita {
namespace {

template <class T>
__global__ __launch_bounds__(256) void gated_product_kernel(const float* z, int64_t ldz, T* h, int64_t ldh, int M, int F, int act) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int n4 = F / 4;
    const int64_t row = i / n4;
    if (row >= M) return;
    const int c = (int)(i - row * n4) * 4;
    const f32x4 g = *reinterpret_cast<const f32x4*>(z + row * ldz + c), u = *reinterpret_cast<const f32x4*>(z + row * ldz + F + c);
    T* o = h + row * ldh + c;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (T)(apply_act(g[j], act) * u[j]);
}

// dz and the partial sums of db (lo: also what the rounding of dz lost, M rows further on): a workgroup has 256 features and kDzRows rows, a thread 4 features of every 4th row; 16-byte accesses
constexpr int kDzRows = 32;
template <class T>
__global__ __launch_bounds__(256) void gated_dz_kernel(const float* z, int64_t ldz, const T* dh, int64_t ld_dh, T* dz, int64_t ld_dz, float* db_part, int M,
                                                       int F, int act, int64_t segs, bool lo) {
    typedef T vec4 __attribute__((ext_vector_type(4)));
    __shared__ float part[4][2][256];
    const int lane = threadIdx.x & 63, y = threadIdx.x >> 6, blocks = (F + 255) / 256;
    const int64_t seg = blockIdx.x / blocks;
    const int c = (int)(blockIdx.x - seg * blocks) * 256 + lane * 4;
    const int64_t r0 = seg * kDzRows, r1 = min((int64_t)M, r0 + kDzRows);
    f32x4 sg = {0.f, 0.f, 0.f, 0.f}, su = sg;
    if (c < F)
        for (int64_t r = r0 + y; r < r1; r += 4) {
            const f32x4 g = *reinterpret_cast<const f32x4*>(z + r * ldz + c), u = *reinterpret_cast<const f32x4*>(z + r * ldz + F + c);
            const vec4 d = *reinterpret_cast<const vec4*>(dh + r * ld_dh + c);
            vec4 og, ou, lg, lu;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float dg = (float)d[j] * u[j] * act_grad(g[j], act), du = (float)d[j] * apply_act(g[j], act);
                og[j] = (T)dg;
                ou[j] = (T)du;
                lg[j] = (T)(dg - (float)og[j]);
                lu[j] = (T)(du - (float)ou[j]);
                sg[j] += dg;
                su[j] += du;
            }
            *reinterpret_cast<vec4*>(dz + r * ld_dz + c) = og;
            *reinterpret_cast<vec4*>(dz + r * ld_dz + F + c) = ou;
            if (lo) {
                *reinterpret_cast<vec4*>(dz + (M + r) * ld_dz + c) = lg;
                *reinterpret_cast<vec4*>(dz + (M + r) * ld_dz + F + c) = lu;
            }
        }
    if (db_part == nullptr) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        part[y][0][lane * 4 + j] = sg[j];
        part[y][1][lane * 4 + j] = su[j];
    }
    __syncthreads();
    const int f = (int)(blockIdx.x - seg * blocks) * 256 + threadIdx.x;
    if (f < F)
#pragma unroll
        for (int k = 0; k < 2; ++k)
            db_part[seg * 2 * F + k * F + f] = (part[0][k][threadIdx.x] + part[1][k][threadIdx.x]) + (part[2][k][threadIdx.x] + part[3][k][threadIdx.x]);
}

// (rows, cols) -> (cols, rows) of 16-bit elements
__global__ __launch_bounds__(256) void transpose16_kernel(const uint16_t* src, int64_t ld, uint16_t* dst, int64_t ldd, int rows, int cols) {
    __shared__ uint16_t t[64][66];
    const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64, x = threadIdx.x & 63, y = threadIdx.x >> 6;
    for (int j = y; j < 64; j += 4)
        if (r0 + j < rows && c0 + x < cols) t[j][x] = src[(int64_t)(r0 + j) * ld + c0 + x];
    __syncthreads();
    for (int j = y; j < 64; j += 4)
        if (c0 + j < cols && r0 + x < rows) dst[(int64_t)(c0 + j) * ldd + r0 + x] = t[x][j];
}
// the sum of `parts` fp32 matrices, one below the other
__global__ __launch_bounds__(256) void to_bf16_kernel(const float* src, bf16* dst, int64_t ldd, int rows, int cols, int parts) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)rows * cols) return;
    const int64_t r = i / cols, n = (int64_t)rows * cols;
    float v = src[i];
    for (int k = 1; k < parts; ++k) v += src[k * n + i];
    dst[r * ldd + (i - r * cols)] = (bf16)v;
}

// ---- the wide bf16 products ------------------------------------------------------------------------------------------------------
// a (2 M, K) matrix whose halves both are x
__global__ __launch_bounds__(256) void rows_twice_kernel(const bf16* x, int64_t ldx, bf16* dst, int M, int K) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, n8 = K / 8, r = i / n8;
    if (r >= M) return;
    const int64_t c = (i - r * n8) * 8;
    const bf16x8 v = *reinterpret_cast<const bf16x8*>(x + r * ldx + c);
    *reinterpret_cast<bf16x8*>(dst + r * K + c) = v;
    *reinterpret_cast<bf16x8*>(dst + (M + r) * K + c) = v;
}

struct WideOut {
    const float* bias;
    bf16* c; int64_t ldc;                 // h, or C
    const bf16* dh; int64_t ld_dh;        // dz
    bf16* dz; int64_t ld_dz;
    float* db_part;                       // (tiles_m, 2 F)
};
enum { WIDE_H = 0, WIDE_DZ = 1, WIDE_C = 2 };

// act(z), and its slope where SLOPE, on the hardware's exp2 and reciprocal (one unit in the last place each; the results are rounded to
// bf16, and the sums for db are within 1e-6 of 64 bits).  The library's forms divide and range-reduce: they cost the dz product's epilogue
// a seventh of the kernel.
template <int ACT, bool SLOPE>
__device__ __forceinline__ void wide_act(float z, float& a, float& slope) {
    if constexpr (ACT == VITA_ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f));      // z -> -inf: rcp(inf) = 0
        a = z * s;
        if constexpr (SLOPE) slope = fmaf(a, 1.0f - s, s);
    } else if constexpr (ACT == VITA_ACT_GELU_TANH && SLOPE) {
        // 0.5 (1 + tanh(u)) = s with s = 1 / (1 + exp(-2 u)); a = z s; a' = s + 2 z s (1 - s) u'
        const float c0 = -2.8853900817779268f * 0.7978845608028654f, c1 = c0 * 0.044715f, z2 = z * z;
        const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * fmaf(z2, c1, c0)));
        a = z * s;
        slope = fmaf(a * (1.0f - s), fmaf(z2, 2.0f * 0.7978845608028654f * 3.0f * 0.044715f, 2.0f * 0.7978845608028654f), s);
    } else {
        a = apply_act_t<ACT>(z);
        if constexpr (SLOPE) slope = act_grad(z, ACT);
    }
}

// EPI WIDE_H: h (M, F) of a gated product; WIDE_DZ: dz (M, 2F) of a gated product; WIDE_C: plain C (M, N)
template <bool ACOL, bool BCOL, int EPI, int ACT>
__global__ __launch_bounds__(WNT, 2) void wide_gemm_kernel(WideGemm g, WideOut o) {
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    constexpr bool GATED = EPI != WIDE_C;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 2, wn = wave & 3, col = lane & 31, half = lane >> 5;
    int tm, tn;
    wide_place(g, blockIdx.x, gridDim.x, tm, tn);
    const int m0 = tm * WBM, n0 = tn * (GATED ? WBN / 2 : WBN);
    f32x16 acc[4][2];
    wide_tile<ACOL, BCOL, GATED>(g, lds, m0, n0, acc);

    // through LDS, so that the global stores are whole 16-byte pieces of rows
    if constexpr (!GATED) {
        bf16* t = reinterpret_cast<bf16*>(lds);
        constexpr int LD = WBN;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    t[(wm * 128 + i * 32 + (r >> 2) * 8 + half * 4 + (r & 3)) * LD + wn * 64 + j * 32 + col] = (bf16)acc[i][j][r];
        __syncthreads();
        for (int i = tid; i < WBM * (WBN / 8); i += WNT) {
            const int row = i / (WBN / 8), c = (i - row * (WBN / 8)) * 8;
            if (m0 + row < g.M && n0 + c < g.N)
                *reinterpret_cast<uint4*>(o.c + (int64_t)(m0 + row) * o.ldc + n0 + c) = *reinterpret_cast<const uint4*>(t + row * LD + c);
        }
        return;
    }
    const int f = n0 + wn * 32 + col;
    float bg = 0.f, bu = 0.f;
    if (o.bias != nullptr && f < g.F) {
        bg = o.bias[f];
        bu = o.bias[g.F + f];
    }
    constexpr int LD = WBN / 2;
    bf16* t = reinterpret_cast<bf16*>(lds);               // (256, 128): h, or dh and then dg
    bf16* tu = t + WBM * LD;                              // (256, 128): du
    if constexpr (EPI == WIDE_DZ) {
        for (int i = tid; i < WBM * (LD / 8); i += WNT) {
            const int row = i / (LD / 8), c = (i - row * (LD / 8)) * 8;
            const bool in = m0 + row < g.M && n0 + c < g.F;
            *reinterpret_cast<uint4*>(t + row * LD + c) = in ? *reinterpret_cast<const uint4*>(o.dh + (int64_t)(m0 + row) * o.ld_dh + n0 + c) : make_uint4(0, 0, 0, 0);
        }
        __syncthreads();
    }
    float sg = 0.f, su = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int at = (wm * 128 + i * 32 + (r >> 2) * 8 + half * 4 + (r & 3)) * LD + wn * 32 + col;
            const float zg = acc[i][0][r] + bg, zu = acc[i][1][r] + bu;
            float a, slope;
            wide_act<ACT, EPI == WIDE_DZ>(zg, a, slope);
            if constexpr (EPI == WIDE_H) {
                t[at] = (bf16)(a * zu);
            } else {
                const float d = (float)t[at];
                const float dg = d * zu * slope, du = d * a;
                t[at] = (bf16)dg;
                tu[at] = (bf16)du;
                sg += dg;
                su += du;
            }
        }
    __syncthreads();
    for (int i = tid; i < WBM * (LD / 8); i += WNT) {
        const int row = i / (LD / 8), c = (i - row * (LD / 8)) * 8;
        if (m0 + row < g.M && n0 + c < g.F) {
            if constexpr (EPI == WIDE_H) {
                *reinterpret_cast<uint4*>(o.c + (int64_t)(m0 + row) * o.ldc + n0 + c) = *reinterpret_cast<const uint4*>(t + row * LD + c);
            } else {
                bf16* dst = o.dz + (int64_t)(m0 + row) * o.ld_dz + n0 + c;
                *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(t + row * LD + c);
                *reinterpret_cast<uint4*>(dst + g.F) = *reinterpret_cast<const uint4*>(tu + row * LD + c);
            }
        }
    }
    if constexpr (EPI == WIDE_DZ) {
        if (o.db_part != nullptr) {                       // the halves, then the two waves of a column block, in that order
            __syncthreads();
            float* part = reinterpret_cast<float*>(lds);  // (2, 4, 2, 32)
            sg += __shfl_xor(sg, 32, 64);
            su += __shfl_xor(su, 32, 64);
            if (half == 0) {
                part[((wm * 4 + wn) * 2 + 0) * 32 + col] = sg;
                part[((wm * 4 + wn) * 2 + 1) * 32 + col] = su;
            }
            __syncthreads();
            if (wm == 0 && half == 0 && f < g.F) {
                float* dst = o.db_part + (int64_t)tm * 2 * g.F + f;
                dst[0] = part[(wn * 2 + 0) * 32 + col] + part[((4 + wn) * 2 + 0) * 32 + col];
                dst[g.F] = part[(wn * 2 + 1) * 32 + col] + part[((4 + wn) * 2 + 1) * 32 + col];
            }
        }
    }
}

template <bool ACOL, bool BCOL, int EPI, int ACT = VITA_ACT_NONE>
int launch_wide(const bf16* A, int64_t lda, const bf16* B, int64_t ldb, int M, int N, int K, int F, const WideOut& o, hipStream_t s) {
    WideGemm g{{A, lda}, {B, ldb}, M, N, K, (M + WBM - 1) / WBM, 0, F};
    g.tiles_n = EPI == WIDE_C ? (N + WBN - 1) / WBN : (F + WBN / 2 - 1) / (WBN / 2);
    hipLaunchKernelGGL((wide_gemm_kernel<ACOL, BCOL, EPI, ACT>), dim3((unsigned)(g.tiles_m * g.tiles_n)), dim3(WNT), wide_stages(ACOL, BCOL) * WSTAGE, s, g, o);
    VITA_CHECK_HIP(hipGetLastError());
    return VITA_OK;
}
template <class Go>
int by_act(int act, Go go) {
    switch (act) {
        case VITA_ACT_RELU: return go(std::integral_constant<int, VITA_ACT_RELU>{});
        case VITA_ACT_GELU_ERF: return go(std::integral_constant<int, VITA_ACT_GELU_ERF>{});
        case VITA_ACT_GELU_TANH: return go(std::integral_constant<int, VITA_ACT_GELU_TANH>{});
        case VITA_ACT_SILU: return go(std::integral_constant<int, VITA_ACT_SILU>{});
        default: return go(std::integral_constant<int, VITA_ACT_MISH>{});
    }
}
template <int EPI>
int launch_wide_gated(const vita_gated_args* a, const WideOut& o, hipStream_t s) {
    auto go = [&](auto act) {
        return launch_wide<false, false, EPI, decltype(act)::value>((const bf16*)a->x, a->ldx, (const bf16*)a->w, a->ldw, a->M, 2 * a->F, a->K, a->F, o, s);
    };
    return by_act(a->act, go);
}
// whether a C of M x N has enough 256 x 256 tiles to keep the 256 CUs busy
bool wide_fills(int64_t M, int64_t N) {
    const int64_t t = ((M + WBM - 1) / WBM) * ((N + WBN - 1) / WBN);
    return t >= 192 && t < (int64_t(1) << 31);
}

// ---- few rows, bf16 ---------------------------------------------------------------------------------------------------------------
// h of up to 64 rows: bound by reading the weights once.  A workgroup has 16 features (their 16 gate and 16 up rows of W), its 8 waves an
// eighth of k each; a wave's fragments of v_mfma_f32_16x16x32_bf16 come straight from memory, 64 bytes of a row to a load (32 x 32 tiles
// would take 32: 18.6 against 18.2 us for 25 x 2048 x 8192, 67 MB of weights, 3.7 TB/s), those of U steps in flight together, x from the caches;
// the waves' sums meet in LDS in wave order.  RB: blocks of 16 rows.
template <int ACT, int RB>
__global__ __launch_bounds__(512, 4) void gated_few_rows_kernel(const bf16* x, int64_t ldx, const bf16* w, int64_t ldw, const float* bias, bf16* h, int64_t ldh,
                                                                int M, int F, int K) {
    constexpr int U = RB <= 2 ? 4 : 2;
    __shared__ float part[8][2][4 * 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, quad = lane >> 4;
    const int f = blockIdx.x * 16 + col;
    const bool in = f < F;
    const bf16* wg = w + (int64_t)(in ? f : 0) * ldw + quad * 8;
    const bf16* wu = w + ((int64_t)(in ? f : 0) + F) * ldw + quad * 8;
    const bf16* xr[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) xr[b] = x + (int64_t)min(b * 16 + col, M - 1) * ldx + quad * 8;
    f32x4 g[RB], u[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) { g[b][r] = 0.f; u[b][r] = 0.f; }
    const bf16x8 zero = {};
    const int steps = (K + 31) / 32, per = (steps + 7) / 8, s0 = wave * per, s1 = min(steps, s0 + per);
    for (int s = s0; s < s1; s += U) {
        bf16x8 a[U][RB], bg[U], bu[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int k = (s + j) * 32;
            const bool ok = s + j < s1 && k + quad * 8 < K;
            bg[j] = ok ? *reinterpret_cast<const bf16x8*>(wg + k) : zero;
            bu[j] = ok ? *reinterpret_cast<const bf16x8*>(wu + k) : zero;
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int k = (s + j) * 32;
            const bool ok = s + j < s1 && k + quad * 8 < K;
#pragma unroll
            for (int b = 0; b < RB; ++b) a[j][b] = ok ? *reinterpret_cast<const bf16x8*>(xr[b] + k) : zero;
        }
#pragma unroll
        for (int j = 0; j < U; ++j)
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                g[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[j][b], bg[j], g[b], 0, 0, 0);
                u[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[j][b], bu[j], u[b], 0, 0, 0);
            }
    }
    const float b0 = bias != nullptr && in ? bias[f] : 0.f, b1 = bias != nullptr && in ? bias[F + f] : 0.f;
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        if (b > 0) __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            part[wave][0][r * 64 + lane] = g[b][r];
            part[wave][1][r * 64 + lane] = u[b][r];
        }
        __syncthreads();
        if (wave < 4) {                                    // a wave finishes one of the 4 accumulator rows
            const int row = b * 16 + quad * 4 + wave;
            float zg = b0, zu = b1;
#pragma unroll
            for (int v = 0; v < 8; ++v) {
                zg += part[v][0][wave * 64 + lane];
                zu += part[v][1][wave * 64 + lane];
            }
            float act, slope;
            wide_act<ACT, false>(zg, act, slope);
            if (in && row < M) h[(int64_t)row * ldh + f] = (bf16)(act * zu);
        }
    }
}
constexpr int kFewRows = 64;
int launch_few_rows(const vita_gated_args* a, hipStream_t s) {
    auto go = [&](auto act) -> int {
        constexpr int ACT = decltype(act)::value;
        const dim3 grid((a->F + 15) / 16);
        auto launch = [&](auto rb) {
            hipLaunchKernelGGL((gated_few_rows_kernel<ACT, decltype(rb)::value>), grid, dim3(512), 0, s, (const bf16*)a->x, a->ldx, (const bf16*)a->w, a->ldw, a->b,
                               (bf16*)a->h, a->ldh, a->M, a->F, a->K);
        };
        if (a->M <= 16) launch(std::integral_constant<int, 1>{});
        else if (a->M <= 32) launch(std::integral_constant<int, 2>{});
        else launch(std::integral_constant<int, 4>{});
        VITA_CHECK_HIP(hipGetLastError());
        return VITA_OK;
    };
    return by_act(a->act, go);
}

int check(const vita_gated_args* a, bool bwd, const char* who) {
    VITA_REQUIRE(a != nullptr, "%s: null args", who);
    VITA_REQUIRE(a->dtype == VITA_DT_F32 || a->dtype == VITA_DT_BF16, "%s: unknown dtype %d", who, a->dtype);
    VITA_REQUIRE(a->act >= VITA_ACT_RELU && a->act <= VITA_ACT_MISH, "%s: unknown activation %d", who, a->act);
    VITA_REQUIRE(a->M >= 0 && a->F >= 8 && a->K >= 8 && a->F % 8 == 0 && a->K % 8 == 0 && a->F <= (1 << 20) && a->K <= (1 << 20) && a->M <= (1 << 28),
                 "%s: bad shape M=%d F=%d K=%d (F and K multiples of 8, at most 2^20)",
                 who, a->M, a->F, a->K);
    const int vec = a->dtype == VITA_DT_F32 ? 4 : 8;
    auto ok = [&](const void* p, int64_t ld, int64_t n) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % vec == 0 && ld >= n; };
    VITA_REQUIRE(ok(a->w, a->ldw, a->K) && (a->M == 0 || ok(a->x, a->ldx, a->K)), "%s: x and w need 16-byte aligned rows of at least K elements", who);
    VITA_REQUIRE(a->b == nullptr || (reinterpret_cast<uintptr_t>(a->b) & 15u) == 0, "%s: b must be 16-byte aligned", who);
    VITA_REQUIRE(a->z == nullptr || ((reinterpret_cast<uintptr_t>(a->z) & 15u) == 0 && a->ldz % 4 == 0 && a->ldz >= 2 * (int64_t)a->F), "%s: bad z", who);
    if (!bwd) {
        VITA_REQUIRE(a->M == 0 || ok(a->h, a->ldh, a->F), "%s: h needs 16-byte aligned rows of at least F elements", who);
    } else {
        VITA_REQUIRE(a->M == 0 || ok(a->dh, a->ld_dh, a->F), "%s: dh needs 16-byte aligned rows of at least F elements", who);
        VITA_REQUIRE(a->dx == nullptr || ok(a->dx, a->ld_dx, a->K), "%s: dx needs 16-byte aligned rows of at least K elements", who);
        VITA_REQUIRE(a->dw == nullptr || ok(a->dw, a->ld_dw, a->K), "%s: dw needs 16-byte aligned rows of at least K elements", who);
        VITA_REQUIRE(a->db == nullptr || (reinterpret_cast<uintptr_t>(a->db) & 3u) == 0, "%s: misaligned db", who);
    }
    return VITA_OK;
}

// bf16 products whose z is not given and whose tiles fill the chip
bool wide_product(const vita_gated_args* a) { return a->dtype == VITA_DT_BF16 && a->z == nullptr && wide_fills(a->M, 2 * (int64_t)a->F); }

// a forward call that the few-row kernel takes (z wanted: the general path, which writes it)
bool few_rows(const vita_gated_args* a) { return a->dtype == VITA_DT_BF16 && a->z == nullptr && a->M <= kFewRows; }

// bf16 gradients of few rows: dz goes into dx and dw as two bf16 numbers, a second set of M rows, for with few terms its rounding does
// not average out (2 x 48 x 88: dx and dw 1.64 times as far off as their own rounding puts them, 1 x 400 x 6784 1.55, many rows 1.41, both
// parts 1.0).  Such products wait for the weights, the added rows cost little; more rows would double the products.
int dz_parts(const vita_gated_args* a) { return a->dtype == VITA_DT_BF16 && a->M <= kFewRows && !wide_product(a) ? 2 : 1; }

struct Ws { float* sk; float* z; void* dz; float* dx32; void* xx; float* dw32; void* wt; float* db_part; float* cs; size_t bytes; };
Ws carve(const vita_gated_args* a, bool bwd, void* ws) {
    Carver c(ws);
    Ws r{};
    const size_t M = a->M, F2 = 2 * (size_t)a->F, K = a->K;
    const bool wide = wide_product(a);
    if (!bwd && few_rows(a)) return r;
    if (bwd || !wide) r.sk = c.take(kSplitkBytes / 4);
    if (a->z == nullptr && !wide) r.z = c.take(M * F2);
    if (bwd) {
        const size_t es = a->dtype == VITA_DT_F32 ? 4 : 2, parts = dz_parts(a);
        r.dz = c.take((M * F2 * parts * es + 3) / 4);
        if (a->dtype == VITA_DT_BF16 && a->dw != nullptr && !wide_fills(F2, K)) r.dw32 = c.take(F2 * K);
        if (a->dtype == VITA_DT_BF16 && a->dx != nullptr && (parts == 2 || !wide_fills(M, K))) r.wt = c.take((F2 * K * es + 3) / 4);
        if (parts == 2 && a->dx != nullptr) r.dx32 = c.take(parts * M * K);
        if (parts == 2 && a->dw != nullptr) r.xx = c.take((parts * M * K * es + 3) / 4);
        // fp32 dx: W transposed once lets the product take the row-operand GEMM (2176 x 512 x 4096: 162 us on W as it lies), from as many
        // rows as the training step does so; the transpose wants W without gaps
        if (a->dtype == VITA_DT_F32 && a->dx != nullptr && a->M >= kWtMinRows && a->ldw == a->K) r.wt = c.take(F2 * K);
        const size_t segs = (M + kDzRows - 1) / kDzRows;
        r.db_part = c.take(segs * F2);
        r.cs = c.take((size_t)vita_colsum_partials_count((int32_t)F2));
    }
    r.bytes = c.off;
    return r;
}

// Parts of dx's long reduction (2 F): the product's 64 x 128 tiles go over the 256 CUs in whole rounds, so S parts take
// ceil(tiles S / 256) / S rounds, and each part costs the sum of partial results about 2 % of one.  2176 x 512 x 4096: 136 tiles, 1 part
// 141 us, 5 parts 115 us.
int dx_splits(int M, int K, int F2) {
    const long tiles = (long)((M + 63) / 64) * ((K + 127) / 128);
    int best = 1;
    double cost = 1e30;
    for (int S = 1; S <= 8 && F2 / S >= 512; ++S) {
        const double c = (double)((tiles * S + 255) / 256) / S + 0.02 * S;
        if (c < cost) { cost = c; best = S; }
    }
    return best;
}

// z = x w^T + b (fp32)
int preact(const vita_gated_args* a, float* z, int64_t ldz, const Ws& ws, hipStream_t s) {
    if (a->dtype == VITA_DT_F32) {
        SplitkScope sk(ws.sk, kSplitkBytes);
        return gemm_f32(lin((const float*)a->x, a->ldx, (const float*)a->w, a->ldw, a->b, z, ldz, a->M, 2 * a->F, a->K, VITA_ACT_NONE), s);
    }
    vita_linear_args l{};
    l.X = (const float*)a->x; l.ldx = a->ldx; l.W = (const float*)a->w; l.ldw = a->ldw; l.bias = a->b; l.Y = z; l.ldy = ldz;
    l.M = a->M; l.N = 2 * a->F; l.K = a->K;
    return gemm_bf16_dma(l, nullptr, 0, s);
}

int run_bwd(const vita_gated_args* a, void* workspace, hipStream_t s) {
    const Ws ws = carve(a, true, workspace);
    const int M = a->M, F = a->F, F2 = 2 * a->F, K = a->K, parts = dz_parts(a);
    const float* z = a->z;
    int64_t ldz = a->ldz;
    const bool wide = wide_product(a);
    if (z == nullptr && !wide) {
        VITA_TRY(preact(a, ws.z, F2, ws, s));
        z = ws.z;
        ldz = F2;
    }
    float* part = a->db != nullptr ? ws.db_part : nullptr;
    int segs = (M + kDzRows - 1) / kDzRows;
    const int64_t blocks = (int64_t)segs * ((F + 255) / 256);
    VITA_REQUIRE(blocks < (int64_t(1) << 31), "vita_gated_linear_bwd: too many elements");
    const dim3 grid((unsigned)blocks);
    if (wide) {
        WideOut o{};
        o.bias = a->b; o.dh = (const bf16*)a->dh; o.ld_dh = a->ld_dh; o.dz = (bf16*)ws.dz; o.ld_dz = F2; o.db_part = part;
        VITA_TRY(launch_wide_gated<WIDE_DZ>(a, o, s));
        segs = (M + WBM - 1) / WBM;
    } else if (a->dtype == VITA_DT_F32)
        hipLaunchKernelGGL(gated_dz_kernel<float>, grid, dim3(256), 0, s, z, ldz, (const float*)a->dh, a->ld_dh, (float*)ws.dz, F2, part, M, F, a->act, (int64_t)segs, false);
    else
        hipLaunchKernelGGL(gated_dz_kernel<bf16>, grid, dim3(256), 0, s, z, ldz, (const bf16*)a->dh, a->ld_dh, (bf16*)ws.dz, F2, part, M, F, a->act, (int64_t)segs, parts == 2);
    VITA_CHECK_HIP(hipGetLastError());
    if (a->db != nullptr) VITA_TRY(vita_colsum_f32(part, F2, segs, F2, ws.cs, a->db, 0, s));
    SplitkScope sk(ws.sk, kSplitkBytes);
    if (a->dtype == VITA_DT_F32) {
        if (a->dx != nullptr && ws.wt != nullptr) {
            VITA_TRY(launch_transpose_f32((const float*)a->w, F2, K, (float*)ws.wt, s));
            VITA_TRY(gemm_f32_rows_split(lin((const float*)ws.dz, F2, (const float*)ws.wt, F2, nullptr, (float*)a->dx, a->ld_dx, M, K, F2, VITA_ACT_NONE),
                                         dx_splits(M, K, F2), s));
        } else if (a->dx != nullptr) {
            VITA_TRY(gemm_f32(dgrad((const float*)ws.dz, F2, (const float*)a->w, a->ldw, (float*)a->dx, a->ld_dx, M, K, F2), s));
        }
        if (a->dw != nullptr) VITA_TRY(gemm_f32(wgrad((const float*)ws.dz, F2, (const float*)a->x, a->ldx, (float*)a->dw, a->ld_dw, M, K, F2), s));
        return VITA_OK;
    }
    if (a->dx != nullptr && parts == 1 && wide_fills(M, K)) {
        WideOut o{};
        o.c = (bf16*)a->dx; o.ldc = a->ld_dx;
        VITA_TRY((launch_wide<false, true, WIDE_C>((const bf16*)ws.dz, F2, (const bf16*)a->w, a->ldw, M, K, F2, 0, o, s)));
    } else if (a->dx != nullptr) {
        hipLaunchKernelGGL(transpose16_kernel, dim3((K + 63) / 64, (F2 + 63) / 64), dim3(256), 0, s, (const uint16_t*)a->w, a->ldw, (uint16_t*)ws.wt, (int64_t)F2, F2, K);
        VITA_CHECK_HIP(hipGetLastError());
        vita_linear_args l{};
        l.X = (const float*)ws.dz; l.ldx = F2; l.W = (const float*)ws.wt; l.ldw = F2; l.M = parts * M; l.N = K; l.K = F2; l.ldy = K;
        if (parts == 1) {
            VITA_TRY(gemm_bf16_dma(l, (uint16_t*)a->dx, a->ld_dx, s));
        } else {
            l.Y = ws.dx32;
            VITA_TRY(gemm_bf16_dma(l, nullptr, 0, s));
            hipLaunchKernelGGL(to_bf16_kernel, dim3((unsigned)(((int64_t)M * K + 255) / 256)), dim3(256), 0, s, ws.dx32, (bf16*)a->dx, a->ld_dx, M, K, parts);
            VITA_CHECK_HIP(hipGetLastError());
        }
    }
    const bf16* x = (const bf16*)a->x;
    int64_t ldx = a->ldx;
    if (a->dw != nullptr && parts == 2) {
        hipLaunchKernelGGL(rows_twice_kernel, dim3((unsigned)(((int64_t)M * (K / 8) + 255) / 256)), dim3(256), 0, s, x, ldx, (bf16*)ws.xx, M, K);
        VITA_CHECK_HIP(hipGetLastError());
        x = (const bf16*)ws.xx;
        ldx = K;
    }
    if (a->dw != nullptr && wide_fills(F2, K)) {
        WideOut o{};
        o.c = (bf16*)a->dw; o.ldc = a->ld_dw;
        VITA_TRY((launch_wide<true, true, WIDE_C>((const bf16*)ws.dz, F2, x, ldx, F2, K, parts * M, 0, o, s)));
    } else if (a->dw != nullptr) {
        vita_linear_args l{};
        l.Y = ws.dw32; l.ldy = K; l.M = F2; l.N = K; l.K = parts * M; l.splitk_ws = ws.sk; l.splitk_ws_bytes = kSplitkBytes;
        VITA_TRY(gemm_bf16_wgrad_tn((const uint16_t*)ws.dz, F2, (const uint16_t*)x, ldx, l, s));
        const int64_t n = (int64_t)F2 * K;
        hipLaunchKernelGGL(to_bf16_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, ws.dw32, (bf16*)a->dw, a->ld_dw, F2, K, 1);
        VITA_CHECK_HIP(hipGetLastError());
    }
    return VITA_OK;
}

}  // namespace
}  // namespace vita

using namespace vita;

extern "C" {

size_t vita_gated_linear_workspace_bytes(const vita_gated_args* a) {
    if (a == nullptr || a->M <= 0 || a->F <= 0 || a->K <= 0) return 0;
    return carve(a, false, nullptr).bytes;
}
int vita_gated_linear(const vita_gated_args* a, void* workspace, size_t workspace_bytes, vita_stream_t stream) {
    const char* who = "vita_gated_linear";
    VITA_TRY(check(a, false, who));
    if (a->M == 0) return VITA_OK;
    VITA_TRY(check_ws(workspace, workspace_bytes, vita_gated_linear_workspace_bytes(a), who));
    hipStream_t s = (hipStream_t)stream;
    if (few_rows(a)) return launch_few_rows(a, s);
    if (wide_product(a)) {
        WideOut o{};
        o.bias = a->b; o.c = (bf16*)a->h; o.ldc = a->ldh;
        return launch_wide_gated<WIDE_H>(a, o, s);
    }
    const Ws ws = carve(a, false, workspace);
    float* z = a->z != nullptr ? a->z : ws.z;
    const int64_t ldz = a->z != nullptr ? a->ldz : 2 * (int64_t)a->F;
    VITA_TRY(preact(a, z, ldz, ws, s));
    const int64_t n = (int64_t)a->M * (a->F / 4);
    if (a->dtype == VITA_DT_F32)
        hipLaunchKernelGGL(gated_product_kernel<float>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, z, ldz, (float*)a->h, a->ldh, a->M, a->F, a->act);
    else
        hipLaunchKernelGGL(gated_product_kernel<bf16>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, z, ldz, (bf16*)a->h, a->ldh, a->M, a->F, a->act);
    VITA_CHECK_HIP(hipGetLastError());
    return VITA_OK;
}
size_t vita_gated_linear_bwd_workspace_bytes(const vita_gated_args* a) {
    if (a == nullptr || a->M <= 0 || a->F <= 0 || a->K <= 0) return 0;
    return carve(a, true, nullptr).bytes;
}
int vita_gated_linear_bwd(const vita_gated_args* a, void* workspace, size_t workspace_bytes, vita_stream_t stream) {
    const char* who = "vita_gated_linear_bwd";
    VITA_TRY(check(a, true, who));
    VITA_REQUIRE(a->M > 0, "%s: no rows", who);
    VITA_TRY(check_ws(workspace, workspace_bytes, vita_gated_linear_bwd_workspace_bytes(a), who));
    return run_bwd(a, workspace, (hipStream_t)stream);
}

}  // extern "C"
