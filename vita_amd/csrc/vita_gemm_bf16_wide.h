// bf16 GEMM tile for products that fill the chip: 256 x 256 of C per workgroup, 8 waves as 2 x 4, each 128 x 64 (4 x 2 accumulators of
// v_mfma_f32_32x32x16_bf16), k in tiles of 32 through 4 or 5 LDS stages of 32 KB.  Used by the gated feed-forward product and its
// backward pass (vita_gated.hip), which give it three pairs of operand layouts:
//     C[m][n] = sum_k A(m, k) B(n, k);   a ROW operand has k contiguous (X, dY; weights as they lie in nn.Linear), a COL operand has its
//     own index contiguous, k across rows (the weight in dX = dY W, both operands of dW = dY^T X).
// Tiles go from memory to LDS directly (global_load_lds, 16 bytes a lane, swizzled on the source address): a ROW tile as [256][32], its
// 16-byte pieces XORed with (row / 4) % 4, a COL tile as [32][256], XORed so that the four rows of a transposed read lie in different
// banks; both are read without bank conflicts (counted: 0).  COL fragments come out through the transposed LDS read.
// One wait and one barrier a k-tile: when tile t is multiplied, t + 1 has landed or is about to, and the requests run 3 (two COL
// operands: 4) tiles ahead: what bounds the loop is the latency of lines that no workgroup of the XCD has touched yet, and the clock that
// the power limit leaves (1.8 - 2.1 GHz in a run of such products).  A wave's k-step is 8 MFMAs (256 cycles) on 6 KB of LDS reads.
// Measured, 550 GFLOP each, median (best) of ten: X W^T 8191 x 16384 x 2048 with the activation's epilogue 577 (533) us, dY W 511 (467) us
// (1.08 PFLOP/s), dY^T X 16384 x 2048 x 8191 559 (511) us; the best with k tiles of 64 in two stages: 547 / 495 / 590 us, with 4 stages of
// COL tiles 550 us; 5 stages of ROW tiles were slower.
#pragma once
#include <type_traits>

#include "vita_host.h"

namespace vita {

typedef __bf16 bf16;

struct WideOperand { const bf16* p; int64_t ld; };
struct WideGemm {
    WideOperand a, b;
    int M, N, K;          // C is M x N
    int tiles_m, tiles_n;
    int F;                // gated: N = 2 F, tile column block j of a wave is the gate (0) or the up projection (1) of the same 32 features
};

constexpr int WNT = 512, WBM = 256, WBN = 256, WBK = 32;
constexpr int WDMA = WBK / 16;                                              // DMA instructions a wave, operand and tile
constexpr int WHALF = WBM * WBK * 2, WSTAGE = 2 * WHALF;   // bytes
constexpr int wide_stages(bool acol, bool bcol) { return acol && bcol ? 5 : 4; }

static __device__ __attribute__((aligned(16))) uint32_t g_wide_zero[4] = {0, 0, 0, 0};

typedef unsigned wide_u2 __attribute__((ext_vector_type(2)));
struct WideFrag { wide_u2 lo, hi; };

__device__ __forceinline__ int wide_row_swz(int r) { return (r >> 2) & 3; }
__device__ __forceinline__ int wide_col_swz(int r) { return ((r & 3) << 2) | ((r >> 2) & 3); }

// where each lane's 16-byte pieces of an operand's tiles come from
template <bool COL, bool GATED>
struct WideSource {
    const char* p[WDMA];
    int64_t step;         // bytes from tile to tile
    int kk[WDMA];          // k of the piece within a tile
    __device__ __forceinline__ void init(const WideOperand& o, int first, int n, int F, int wave, int lane) {
#pragma unroll
        for (int j = 0; j < WDMA; ++j) {
            const bf16* src;
            bool in;
            if constexpr (COL) {
                const int r = (j * 8 + wave) * 2 + (lane >> 5), pos = lane & 31;
                const int c = first + ((pos & 16) | ((pos & 15) ^ wide_col_swz(r))) * 8;
                kk[j] = r;
                in = c < n;
                src = o.p + (int64_t)r * o.ld + c;
                step = (int64_t)WBK * o.ld * 2;
            } else {
                constexpr int PC = WBK / 8;          // 16-byte pieces of a row
                const int r = (j * 8 + wave) * (64 / PC) + lane / PC, pos = lane % PC;
                kk[j] = (pos ^ wide_row_swz(r)) * 8;
                int row = first + r;
                in = row < n;
                if constexpr (GATED) {      // 64 tile rows a wave: 32 gate rows, then the same features' 32 up rows
                    const int f = first + (r >> 6) * 32 + (r & 31);
                    in = f < F;
                    row = f + ((r >> 5) & 1) * F;
                }
                src = o.p + (int64_t)row * o.ld + kk[j];
                step = WBK * 2;
            }
            p[j] = reinterpret_cast<const char*>(src);
            if (!in) kk[j] = 1 << 30;        // never inside k
        }
    }
};

// 64 lanes' 16 bytes to 1 KB of LDS from byte address `lds` (uniform).  Written out because behind the builtin the compiler lets no LDS
// read pass: it waited for the tile just requested before the first read of the tile that is there (656 against 563 us for 8191 x 16384
// x 2048).  It has no register result; the kernel's own wait and barrier order it with the reads.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void wide_dma(const char* src, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src) : "memory", "m0");
}
#pragma clang diagnostic pop

// `left`: k rows from the tile's first to K (<= 0: behind the end).  What is outside A or B comes from the zero piece.
template <bool COL, bool GATED>
__device__ __forceinline__ void wide_issue(WideSource<COL, GATED>& s, int j, const char* zero, unsigned lds, int left, int wave) {
    wide_dma(s.kk[j] < left ? s.p[j] : zero, lds + (unsigned)(j * 8 + wave) * 1024);
    s.p[j] += s.step;
}

// Fragments of one 16-deep step.  ROW: 16-byte LDS reads.  COL: transposed reads, issued and waited for in one asm block (a read in
// flight must not share a register with anything the compiler believes free).
template <int N>
__device__ __forceinline__ void wide_read_row(const char* tile, int addr, WideFrag (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = __builtin_bit_cast(WideFrag, *reinterpret_cast<const f32x4*>(tile + addr + i * 32 * WBK * 2));
}
#define VITA_TR "ds_read_b64_tr_b16 "
template <int OFF>
__device__ __forceinline__ void wide_read_col(const unsigned (&a)[4][2], WideFrag (&f)[4]) {
    asm volatile(VITA_TR "%0, %8 offset:%16\n\t" VITA_TR "%1, %9 offset:%16\n\t" VITA_TR "%2, %10 offset:%16\n\t" VITA_TR "%3, %11 offset:%16\n\t"
                 VITA_TR "%4, %12 offset:%16\n\t" VITA_TR "%5, %13 offset:%16\n\t" VITA_TR "%6, %14 offset:%16\n\t" VITA_TR "%7, %15 offset:%16\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(f[0].lo), "=&v"(f[0].hi), "=&v"(f[1].lo), "=&v"(f[1].hi), "=&v"(f[2].lo), "=&v"(f[2].hi), "=&v"(f[3].lo), "=&v"(f[3].hi)
                 : "v"(a[0][0]), "v"(a[0][1]), "v"(a[1][0]), "v"(a[1][1]), "v"(a[2][0]), "v"(a[2][1]), "v"(a[3][0]), "v"(a[3][1]), "n"(OFF)
                 : "memory");
}
template <int OFF>
__device__ __forceinline__ void wide_read_col(const unsigned (&a)[2][2], WideFrag (&f)[2]) {
    asm volatile(VITA_TR "%0, %4 offset:%8\n\t" VITA_TR "%1, %5 offset:%8\n\t" VITA_TR "%2, %6 offset:%8\n\t" VITA_TR "%3, %7 offset:%8\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(f[0].lo), "=&v"(f[0].hi), "=&v"(f[1].lo), "=&v"(f[1].hi)
                 : "v"(a[0][0]), "v"(a[0][1]), "v"(a[1][0]), "v"(a[1][1]), "n"(OFF)
                 : "memory");
}
#undef VITA_TR

// the tile's position: contiguous ranges of tiles an XCD, in bands of 8 tile rows (neighbours share operands in its L2)
__device__ __forceinline__ void wide_place(const WideGemm& g, int id, int n, int& tm, int& tn) {
    const int per = n >> 3, rem = n & 7, x = id & 7;
    id = x * per + min(x, rem) + (id >> 3);
    const int band = id / (8 * g.tiles_n), rows = min(8, g.tiles_m - band * 8), in = id - band * 8 * g.tiles_n;
    tm = band * 8 + in % rows;
    tn = in / rows;
}

// accumulates the tile; on return every wave has left the LDS stages
template <bool ACOL, bool BCOL, bool GATED>
__device__ __forceinline__ void wide_tile(const WideGemm& g, char* lds, int m0, int n0, f32x16 (&acc)[4][2]) {
    constexpr int NS = wide_stages(ACOL, BCOL);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 2, wn = wave & 3;
    WideSource<ACOL, false> sa;
    WideSource<BCOL, GATED> sb;
    sa.init(g.a, m0, g.M, 0, wave, lane);
    sb.init(g.b, n0, g.N, g.F, wave, lane);
    const int nk = (g.K + WBK - 1) / WBK;
    const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds);
    const char* zero = reinterpret_cast<const char*>(g_wide_zero);
    auto issue = [&](int kt, unsigned stage, int j) {      // a pair of requests of tile kt; behind the last tile zero pieces
        wide_issue(sa, j, zero, lds0 + stage, g.K - kt * WBK, wave);
        wide_issue(sb, j, zero, lds0 + stage + WHALF, g.K - kt * WBK, wave);
    };
#pragma unroll
    for (int t = 0; t < NS - 1; ++t)
#pragma unroll
        for (int j = 0; j < WDMA; ++j) issue(t, t * WSTAGE, j);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    // fragment addresses within a stage
    const int fr = lane & 31, half = lane >> 5;
    int ra[2], rb[2];                           // ROW: by k-step
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
        const int r = wm * 128 + fr, q = wn * 64 + fr;
        ra[ks] = r * WBK * 2 + ((ks * 2 + half) ^ wide_row_swz(r)) * 16;
        rb[ks] = WHALF + q * WBK * 2 + ((ks * 2 + half) ^ wide_row_swz(q)) * 16;
    }
    unsigned ca[4][2], cb[2][2];                        // COL: by 32-column block and half of the 8-deep operand
    const unsigned base = lds0;
    const int grp = lane >> 4, q4 = (lane & 15) >> 2, pp = lane & 3;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int row = 8 * (grp >> 1) + 4 * h + q4, f = wide_col_swz(row);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = wm * 16 + i * 4 + (grp & 1) * 2 + (pp >> 1);
            ca[i][h] = base + 512 * row + ((c & 16) | ((c & 15) ^ f)) * 16 + 8 * (pp & 1);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int c = wn * 8 + j * 4 + (grp & 1) * 2 + (pp >> 1);
            cb[j][h] = base + WHALF + 512 * row + ((c & 16) | ((c & 15) ^ f)) * 16 + 8 * (pp & 1);
        }
    }

    unsigned here = 0, there = (NS - 1) * WSTAGE;      // stages of tiles kt and kt + NS - 1
    for (int kt = 0; kt < nk; ++kt) {
        // this wave's pieces of tile kt have landed; behind the barrier everyone's have, and everyone has left tile kt - 1, whose stage
        // is filled next
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 2) * 2 * WDMA) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const char* st = lds + here;
        unsigned xa[4][2], xb[2][2];
        if constexpr (ACOL) {
#pragma unroll
            for (int i = 0; i < 4; ++i) { xa[i][0] = ca[i][0] + here; xa[i][1] = ca[i][1] + here; }
        }
        if constexpr (BCOL) {
#pragma unroll
            for (int j = 0; j < 2; ++j) { xb[j][0] = cb[j][0] + here; xb[j][1] = cb[j][1] + here; }
        }
        WideFrag a[2][4], b[2][2];
        auto read = [&](auto step, bool row) {          // ROW fragments are requested in front of the previous step's products, COL ones
            constexpr int ks = decltype(step)::value;   // (waited for where they are read) behind them
            if constexpr (ks < 2) {
                if constexpr (!ACOL) { if (row) wide_read_row<4>(st, ra[ks], a[ks & 1]); }
                else { if (!row) wide_read_col<ks * 16 * 512>(xa, a[ks & 1]); }
                if constexpr (!BCOL) { if (row) wide_read_row<2>(st, rb[ks], b[ks & 1]); }
                else { if (!row) wide_read_col<ks * 16 * 512>(xb, b[ks & 1]); }
            }
        };
        auto products = [&](int ks, int i0, int i1) {
#pragma unroll
            for (int i = i0; i < i1; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a[ks & 1][i]), __builtin_bit_cast(bf16x8, b[ks & 1][j]), acc[i][j], 0, 0, 0);
        };
        // a later tile's requests go between the products, a pair a step: all of them at once would fill the memory pipe's queue and
        // hold the wave (behind the last tile they fetch zero pieces, so that the wait's count holds)
        auto step = [&](auto next) {
            constexpr int ks = decltype(next)::value - 1;
            read(next, true);
            products(ks, 0, 2);
            __builtin_amdgcn_sched_barrier(0);
            issue(kt + NS - 1, there, ks);
            __builtin_amdgcn_sched_barrier(0);
            products(ks, 2, 4);
            __builtin_amdgcn_sched_barrier(0);
            read(next, false);
            __builtin_amdgcn_sched_barrier(0);
        };
        read(std::integral_constant<int, 0>{}, true);
        read(std::integral_constant<int, 0>{}, false);
        step(std::integral_constant<int, 1>{});
        step(std::integral_constant<int, 2>{});
        there = here;
        here = here == (NS - 1) * WSTAGE ? 0 : here + WSTAGE;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // the last requests must not land in what the epilogue writes
    __syncthreads();
}

}  // namespace vita
