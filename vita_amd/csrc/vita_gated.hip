// The gated feed-forward product h = act(x Wg^T + bg) * (x Wu^T + bu) and its backward pass (see include/vita_hip.h).
//
// First form: one product for both projections into a pre-activation matrix z (M, 2F) with the library's GEMMs, then one elementwise
// pass.  Backward: z (saved, or formed again), one pass for dz and the bias gradient's partial sums, then dx = dz W and dw = dz^T x.
#include "vita_host.h"

namespace vita {
namespace {

typedef __bf16 bf16;

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

constexpr int kDzRows = 64;      // rows of one partial sum of the bias gradient
template <class T>
__global__ __launch_bounds__(256) void gated_dz_kernel(const float* z, int64_t ldz, const T* dh, int64_t ld_dh, T* dz, int64_t ld_dz, float* db_part, int M,
                                                       int F, int act) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= F) return;
    const int r0 = blockIdx.y * kDzRows, r1 = min(M, r0 + kDzRows);
    float sg = 0.f, su = 0.f;
    for (int r = r0; r < r1; ++r) {
        const float g = z[(int64_t)r * ldz + c], u = z[(int64_t)r * ldz + F + c], d = (float)dh[(int64_t)r * ld_dh + c];
        const float dg = d * u * act_grad(g, act), du = d * apply_act(g, act);
        dz[(int64_t)r * ld_dz + c] = (T)dg;
        dz[(int64_t)r * ld_dz + F + c] = (T)du;
        sg += dg;
        su += du;
    }
    if (db_part != nullptr) {
        db_part[(int64_t)blockIdx.y * 2 * F + c] = sg;
        db_part[(int64_t)blockIdx.y * 2 * F + F + c] = su;
    }
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
__global__ __launch_bounds__(256) void to_bf16_kernel(const float* src, bf16* dst, int64_t ldd, int rows, int cols) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)rows * cols) return;
    const int64_t r = i / cols;
    dst[r * ldd + (i - r * cols)] = (bf16)src[i];
}

int check(const vita_gated_args* a, bool bwd, const char* who) {
    VITA_REQUIRE(a != nullptr, "%s: null args", who);
    VITA_REQUIRE(a->dtype == VITA_DT_F32 || a->dtype == VITA_DT_BF16, "%s: unknown dtype %d", who, a->dtype);
    VITA_REQUIRE(a->act >= VITA_ACT_RELU && a->act <= VITA_ACT_MISH, "%s: unknown activation %d", who, a->act);
    VITA_REQUIRE(a->M >= 0 && a->F >= 8 && a->K >= 8 && a->F % 8 == 0 && a->K % 8 == 0 && a->F <= (1 << 28), "%s: bad shape M=%d F=%d K=%d (F and K multiples of 8)",
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

struct Ws { float* sk; float* z; void* dz; float* dw32; void* wt; float* db_part; float* cs; size_t bytes; };
Ws carve(const vita_gated_args* a, bool bwd, void* ws) {
    Carver c(ws);
    Ws r{};
    const size_t M = a->M, F2 = 2 * (size_t)a->F, K = a->K;
    r.sk = c.take(kSplitkBytes / 4);
    if (a->z == nullptr) r.z = c.take(M * F2);
    if (bwd) {
        const size_t es = a->dtype == VITA_DT_F32 ? 4 : 2;
        r.dz = c.take((M * F2 * es + 3) / 4);
        if (a->dtype == VITA_DT_BF16) r.dw32 = c.take(F2 * K);
        r.wt = c.take((F2 * K * es + 3) / 4);
        const size_t segs = (M + kDzRows - 1) / kDzRows;
        r.db_part = c.take(segs * F2);
        r.cs = c.take((size_t)vita_colsum_partials_count((int32_t)F2));
    }
    r.bytes = c.off;
    return r;
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
    const int M = a->M, F = a->F, F2 = 2 * a->F, K = a->K;
    const float* z = a->z;
    int64_t ldz = a->ldz;
    if (z == nullptr) {
        VITA_TRY(preact(a, ws.z, F2, ws, s));
        z = ws.z;
        ldz = F2;
    }
    const int segs = (M + kDzRows - 1) / kDzRows;
    const dim3 grid((F + 255) / 256, segs);
    float* part = a->db != nullptr ? ws.db_part : nullptr;
    if (a->dtype == VITA_DT_F32)
        hipLaunchKernelGGL(gated_dz_kernel<float>, grid, dim3(256), 0, s, z, ldz, (const float*)a->dh, a->ld_dh, (float*)ws.dz, F2, part, M, F, a->act);
    else
        hipLaunchKernelGGL(gated_dz_kernel<bf16>, grid, dim3(256), 0, s, z, ldz, (const bf16*)a->dh, a->ld_dh, (bf16*)ws.dz, F2, part, M, F, a->act);
    VITA_CHECK_HIP(hipGetLastError());
    if (a->db != nullptr) VITA_TRY(vita_colsum_f32(part, F2, segs, F2, ws.cs, a->db, 0, s));
    SplitkScope sk(ws.sk, kSplitkBytes);
    if (a->dtype == VITA_DT_F32) {
        if (a->dx != nullptr) VITA_TRY(gemm_f32(dgrad((const float*)ws.dz, F2, (const float*)a->w, a->ldw, (float*)a->dx, a->ld_dx, M, K, F2), s));
        if (a->dw != nullptr) VITA_TRY(gemm_f32(wgrad((const float*)ws.dz, F2, (const float*)a->x, a->ldx, (float*)a->dw, a->ld_dw, M, K, F2), s));
        return VITA_OK;
    }
    if (a->dx != nullptr) {
        hipLaunchKernelGGL(transpose16_kernel, dim3((K + 63) / 64, (F2 + 63) / 64), dim3(256), 0, s, (const uint16_t*)a->w, a->ldw, (uint16_t*)ws.wt, (int64_t)F2, F2, K);
        VITA_CHECK_HIP(hipGetLastError());
        vita_linear_args l{};
        l.X = (const float*)ws.dz; l.ldx = F2; l.W = (const float*)ws.wt; l.ldw = F2; l.M = M; l.N = K; l.K = F2; l.ldy = K;
        VITA_TRY(gemm_bf16_dma(l, (uint16_t*)a->dx, a->ld_dx, s));
    }
    if (a->dw != nullptr) {
        vita_linear_args l{};
        l.Y = ws.dw32; l.ldy = K; l.M = F2; l.N = K; l.K = M; l.splitk_ws = ws.sk; l.splitk_ws_bytes = kSplitkBytes;
        VITA_TRY(gemm_bf16_wgrad_tn((const uint16_t*)ws.dz, F2, (const uint16_t*)a->x, a->ldx, l, s));
        const int64_t n = (int64_t)F2 * K;
        hipLaunchKernelGGL(to_bf16_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, ws.dw32, (bf16*)a->dw, a->ld_dw, F2, K);
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
