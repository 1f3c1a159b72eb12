// Device code shared by the attention kernels (vita_attention_fwd.hip, vita_attention_bwd.hip).
//
// One fragment format for both types: a lane of a 32 x 32 MFMA holds 8 elements of its row (A) or column (B) of a 16-deep step, element
// j of half-wave h standing for depth 8 h + j.  bf16: one v_mfma_f32_32x32x16_bf16; fp32: eight v_mfma_f32_32x32x2_f32, the j-th
// multiplying element j of both halves.  A and B only have to agree on what depth an element stands for, which is what lets a product's
// OUTPUT be the next product's B operand without leaving its registers: accumulator register r of half h is row
// 8 (r / 4) + 4 h + r % 4, so registers 0 .. 7 are a 16-deep B fragment over those rows, and the A fragment is read in the same order.
// The scores are therefore formed transposed (rows = keys, columns = queries): a lane owns one query, the softmax statistics are
// per-lane scalars joined by one exchange between the half-waves, and P^T feeds O^T = V^T P^T directly.
#pragma once
#include "vita_host.h"

namespace vita {

typedef __bf16 bf16;
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short attn_s16x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_inff(), kMaxFloat = 3.402823466e+38f;
constexpr float kFoldBias = 1e6f;      // a tile's single bias joins the exponent's shift only below this: a larger one has to absorb the score first
constexpr int kMaxRadius = 1024;

struct AttnTensor { char* p; int64_t sb, ss, sh; };      // strides in elements

struct AttnParams {
    AttnTensor q, k, v, o, dout, dq, dk, dv;
    float* stats;                    // (B, H, Sq, stats_row): maximum of a row's scores times log2 e (0: no key), reciprocal of the sum of
                                     // 2^(score - maximum) (0: no key); bf16: two zeros, then D bf16, what o lost when it was rounded
    int stats_row;
    float* delta;                    // backward: (B, H, Sq) in the workspace
    const uint8_t* pad; int64_t ld_pad;
    const void* table; const int32_t* buckets; int R, NB;
    int B, H, Hk, G, Sq, Sk, D, causal;
    float scale, scale_log2;
    int pack;                        // forward: query heads of one key head that share a row tile (1 or G)
    int tiles, splits, tiles_per_split;
    float* part_o; float* part_ml;   // forward, splits > 1
    float* dist_part;                // backward: (B * q tiles, H, 2 R + 1)
    int want_dtable;
};

template <class T> struct Frag;
template <> struct Frag<float> { float v[8]; };
template <> struct Frag<bf16> { bf16x8 v; };

__device__ __forceinline__ void mma(f32x16& acc, const Frag<float>& a, const Frag<float>& b) {
#pragma unroll
    for (int j = 0; j < 8; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[j], b.v[j], acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16& acc, const Frag<bf16>& a, const Frag<bf16>& b) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, acc, 0, 0, 0);
}

__device__ __forceinline__ int acc_row(int r, int half) { return (r >> 2) * 8 + half * 4 + (r & 3); }

// A tile in LDS: rows of DP elements and a padding.  The 16-byte reads of 16 consecutive rows meet 16 different groups of 4 banks where
// the stride is an odd number of 16 bytes.  The transposed reads of bf16 take 4 rows x 64 bytes at a time, which share no more than two
// to a bank where the stride is 48, 80, 176 or 208 bytes beyond a multiple of 256.  (XORed pieces in place of padding free both of
// conflicts, but want an address register for every piece: the dq kernel spilled and went from 340 to 374 us, 2 x 4096 x 16 heads of 128.)
constexpr int lds_stride_of(int element, int DP) { return DP + (element == 2 && DP % 64 == 0 ? 24 : 16 / element); }
template <class T, int DP> constexpr int lds_stride() { return lds_stride_of((int)sizeof(T), DP); }
constexpr size_t kLds = 160 * 1024;                                                     // of a workgroup
// bytes of `tiles` tiles of 128 rows of D elements, as the kernels whose waves share out an axis keep them
inline size_t tiles128_bytes(int dtype, int D, int tiles) {
    const int es = dtype == VITA_DT_F32 ? 4 : 2;
    return (size_t)tiles * 128 * lds_stride_of(es, (D + 31) / 32 * 32) * es;
}
// the 16-byte piece `piece` of a row
template <class T, int DP>
__device__ __forceinline__ int lds_at(int row, int piece) { return row * lds_stride<T, DP>() + piece * (16 / (int)sizeof(T)); }

template <class T>
__device__ __forceinline__ Frag<T> load8(const T* p) {      // 16-byte aligned
    Frag<T> f;
    if constexpr (sizeof(T) == 2) {
        f.v = *reinterpret_cast<const bf16x8*>(p);
    } else {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) { f.v[j] = a[j]; f.v[4 + j] = b[j]; }
    }
    return f;
}
// 8 elements from column 8 c of a tile's row
template <class T, int DP>
__device__ __forceinline__ Frag<T> row_frag(const T* tile, int row, int c) {
    return load8(tile + row * lds_stride<T, DP>() + c * 8);
}
template <class T>
__device__ __forceinline__ Frag<T> zero8() {
    Frag<T> f;
    if constexpr (sizeof(T) == 2) f.v = bf16x8{};
    else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f.v[j] = 0.f;
    }
    return f;
}

// fragment whose depth is the transpose of the tile: row = column col0 + lane % 32 of the tile, depth = the tile's rows row0 ..
// row0 + 15 in accumulator order.  bf16: the hardware's transposed read (a group of 16 lanes gives 4 rows x 16 columns, lane i
// getting column i); fp32: 8 reads of 32 neighbouring columns.
template <class T, int DP>
__device__ __forceinline__ Frag<T> col_frag(const T* tile, int row0, int col0, int lane) {
    constexpr int KS = lds_stride<T, DP>();
    Frag<T> f;
    if constexpr (sizeof(T) == 2) {
        const int g = lane >> 4, q = (lane & 15) >> 2, c = lane & 3;
        const T* a = tile + (row0 + (g >> 1) * 4 + q) * KS + col0 + (g & 1) * 16 + c * 4;
        typedef __attribute__((address_space(3))) attn_s16x4* lds_ptr;
        struct { attn_s16x4 lo, hi; } t;
        t.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)a);
        t.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(a + 8 * KS));
        f.v = __builtin_bit_cast(bf16x8, t);
    } else {
        const T* a = tile + (row0 + (lane >> 5) * 4) * KS + col0 + (lane & 31);
#pragma unroll
        for (int j = 0; j < 8; ++j) f.v[j] = a[((j >> 2) * 8 + (j & 3)) * KS];
    }
    return f;
}

// Products of one tile in steps, fragments requested DEPTH steps ahead: a step is long enough to cover the LDS reads together with the
// SIMD's other wave (one fp32 fragment feeds 512 cycles of MFMA, one bf16 fragment 32, so a bf16 step takes N of them; DEPTH 2 where a
// wave has its SIMD to itself), and the scheduler may not move reads over a step's border.  read(i, j): the A fragment of column block j
// at step i;  use(i, j, a): multiplies it.  start() may stand well in front of run().
template <class T, int STEPS, int N, int DEPTH>
struct Pipe {
    static constexpr int W = sizeof(T) == 2 ? N : 1, TOTAL = STEPS * N / W;
    Frag<T> a[DEPTH + 1][W];
    template <class Read>
    __device__ __forceinline__ void request(int i, Read read) {
        if (i < TOTAL) {
#pragma unroll
            for (int j = 0; j < W; ++j) a[i % (DEPTH + 1)][j] = read(i * W / N, i * W % N + j);
        }
    }
    template <class Read>
    __device__ __forceinline__ void start(Read read) {
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) request(i, read);
        __builtin_amdgcn_sched_barrier(0);
    }
    template <class Read, class Use>
    __device__ __forceinline__ void run(Read read, Use use) {
#pragma unroll
        for (int i = 0; i < TOTAL; ++i) {
            request(i + DEPTH, read);
#pragma unroll
            for (int j = 0; j < W; ++j) use(i * W / N, i * W % N + j, a[i % (DEPTH + 1)][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};
template <class T, int STEPS, int N, class Read, class Use>
__device__ __forceinline__ void pipelined(Read read, Use use) {
    Pipe<T, STEPS, N, 1> pipe;
#pragma unroll
    for (int j = 0; j < pipe.W; ++j) pipe.a[0][j] = read(0, j);
    pipe.run(read, use);
}

template <class T>
__device__ __forceinline__ Frag<T> pack8(const f32x16& s, int chunk) {
    Frag<T> f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f.v[j] = (T)s[chunk * 8 + j];
    return f;
}
// ... and what that rounding lost
template <class T>
__device__ __forceinline__ Frag<T> pack8_rest(const f32x16& s, int chunk, const Frag<T>& hi) {
    Frag<T> f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f.v[j] = (T)(s[chunk * 8 + j] - (float)hi.v[j]);
    return f;
}

// rows of a tile: global -> registers -> LDS, 16 bytes a thread.  A thread's place in the tile never changes, so a whole tile is fetched
// from one uniform base with constant 32-bit offsets: no vector arithmetic (a token stride is below 2^23 elements).  Tiles with missing
// rows (bit clear) or columns (from D on) take the slow form, which makes those zero.
template <class T, int DP, int ROWS, int NT>
struct Stage {
    static constexpr int NV = DP * (int)sizeof(T) / 16, E = 16 / (int)sizeof(T), NLD = ROWS * NV / NT;
    static constexpr bool REGULAR = NT % NV == 0;                    // every load of a thread is in the same column
    static_assert(ROWS * NV % NT == 0 && NLD >= 1, "tile and workgroup do not match");
    uint4 r[NLD];
    uint32_t off[REGULAR ? 1 : NLD];
    uint32_t step;                                                   // bytes between a thread's rows (REGULAR)
    int64_t tile_bytes;
    __device__ __forceinline__ void init(int64_t stride, int tid) {
        const uint32_t sb = (uint32_t)(stride * (int64_t)sizeof(T));
#pragma unroll
        for (int j = 0; j < (REGULAR ? 1 : NLD); ++j) {
            const int i = j * NT + tid, row = i / NV, vec = i - row * NV;
            off[j] = (uint32_t)row * sb + (uint32_t)vec * 16;
        }
        step = REGULAR ? (uint32_t)(NT / NV) * sb : 0;
        tile_bytes = (int64_t)ROWS * sb;
    }
    __device__ __forceinline__ void load(const T* base, uint64_t m0, uint64_t m1, int D, int tid) {
        const char* c = reinterpret_cast<const char*>(base);
        const bool all = ROWS == 32 ? (uint32_t)m0 == 0xffffffffu : (m0 == ~uint64_t(0) && (ROWS <= 64 || m1 == ~uint64_t(0)));
        if (all && D == DP) {
#pragma unroll
            for (int j = 0; j < NLD; ++j) r[j] = *reinterpret_cast<const uint4*>(c + (REGULAR ? (int64_t)(j * step) : 0) + off[REGULAR ? 0 : j]);
        } else {
#pragma unroll
            for (int j = 0; j < NLD; ++j) {
                const int i = j * NT + tid, row = i / NV, vec = i - row * NV;
                const bool in = ((ROWS <= 64 || row < 64 ? m0 >> (row & 63) : m1 >> (row & 63)) & 1) != 0 && vec * E < D;
                r[j] = in ? *reinterpret_cast<const uint4*>(c + (REGULAR ? (int64_t)(j * step) : 0) + off[REGULAR ? 0 : j]) : make_uint4(0, 0, 0, 0);
            }
        }
    }
    __device__ __forceinline__ void store(T* tile, int tid) const {
#pragma unroll
        for (int j = 0; j < NLD; ++j) {
            const int i = j * NT + tid, row = i / NV, vec = i - row * NV;
            *reinterpret_cast<uint4*>(tile + lds_at<T, DP>(row, vec)) = r[j];
        }
    }
};

// the larger of the two half-waves' values, in both.  (The compiler's builtin for this exchange loses its second result where both
// operands are one value, so it is written out; the s_nop covers the wait between a vector write and the exchange.)
__device__ __forceinline__ float max_halves(float v) {
    float lo = v, hi = v;
    asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(lo), "+v"(hi));
    return fmaxf(lo, hi);
}

// which keys exist, 64 to a word; a wave holds the words of 4096 keys, one a lane
struct KeyMask {
    const uint8_t* pad;      // this batch row's bytes, or null
    int Sk, base;            // base: first word held
    uint64_t w;
    __device__ __forceinline__ void init(const AttnParams& p, int b) {
        pad = p.pad != nullptr ? p.pad + (int64_t)b * p.ld_pad : nullptr;
        Sk = p.Sk;
        base = -(1 << 28);
    }
    __device__ __forceinline__ void fill(int first) {
        base = first;
        const int64_t k0 = ((int64_t)first + (threadIdx.x & 63)) * 64;
        const int64_t left = (int64_t)Sk - k0;
        const int n = left >= 64 ? 64 : (left > 0 ? (int)left : 0);
        uint64_t m = n == 64 ? ~uint64_t(0) : (uint64_t(1) << n) - 1;
        if (pad != nullptr) {
            uint64_t here = 0;
            if (n == 64) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    uint32_t v;
                    __builtin_memcpy(&v, pad + k0 + 4 * j, 4);
                    const uint32_t t = ((((v & 0x7f7f7f7fu) + 0x7f7f7f7fu) | v) & 0x80808080u) >> 7;      // 1 in each byte that is not 0
                    here |= (uint64_t)((t * 0x01020408u) >> 24 & 15u) << (4 * j);
                }
            } else {
                for (int j = 0; j < n; ++j) here |= (uint64_t)(pad[k0 + j] != 0) << j;
            }
            m &= ~here;
        }
        w = m;
    }
    // word i of the row (uniform i); 0 behind the last key
    __device__ __forceinline__ uint64_t word(int i) {
        if (i < base || i >= base + 64) fill(i);
        const int l = i - base;
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)w, l), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(w >> 32), l);
        return (uint64_t)hi << 32 | lo;
    }
    // bits of the KT keys of tile t
    template <int KT>
    __device__ __forceinline__ void tile(int t, uint64_t& m0, uint64_t& m1) {
        m1 = 0;
        if constexpr (KT == 32) m0 = (word(t >> 1) >> ((t & 1) * 32)) & 0xffffffffu;
        else if constexpr (KT == 64) m0 = word(t);
        else { m0 = word(2 * t); m1 = word(2 * t + 1); }
    }
};

// the bias of every distance -R .. R of `heads` heads from `head0`, times log2 e
template <class T>
__device__ __forceinline__ void load_bias(const AttnParams& p, float* bias, int head0, int heads, int tid, int nt) {
    const int n = 2 * p.R + 1;
    for (int i = tid; i < n * heads; i += nt) {
        const int g = i / n, id = p.buckets[i - g * n];
        const bool in = id >= 0 && id < p.NB;
        const float v = (float)reinterpret_cast<const T*>(p.table)[(int64_t)(in ? id : 0) * p.H + head0 + g];
        // the type's lowest value, used as a mask, stays finite: a row whose every key has it averages them, as the formula does
        bias[i] = in ? (__builtin_fabsf(v) < kInf ? fmaxf(-kMaxFloat, fminf(kMaxFloat, v * kLog2e)) : v) : __builtin_nanf("");
    }
}

// Workgroup ids go round the 8 XCDs.  The tiles of one (batch row, head) pair stay on one XCD, whose L2 then holds what they share, and
// neighbouring pairs are on different ones, so that batch rows of unequal length load all XCDs alike.  Within an XCD pair after pair, or
// (causal: tiles cost from one to all of the keys) tile after tile, the costliest of every pair first: 32 pairs of 4095 tokens end
// within 1 % of an even share that way, 47 % over it pair after pair.  The grid is rounded up to whole groups of 8 pairs; false = nothing
// to do.
__host__ __device__ inline int64_t pair_grid(int64_t pairs, int tiles) { return (pairs + 7) / 8 * 8 * tiles; }
__device__ __forceinline__ bool pair_order(int id, int pairs, int tiles, int by_tile, int& pair, int& tile) {
    const int i = id >> 3, per = (pairs + 7) >> 3;
    tile = by_tile ? i / per : i % tiles;
    pair = (by_tile ? i - tile * per : i / tiles) * 8 + (id & 7);
    return pair < pairs;
}

// Whether workgroups of 32 rows whose 4 waves share out the other axis run instead of workgroups of 4 x 32 rows, of which there would be
// `wide`.  Each tile is then read for a quarter of the rows, but where the wide ones leave CUs without work, or give the CU with the
// longest rows twice the mean, all share it.  Forward / backward, 8 heads, wide -> narrow: 1 x 512 tokens of 64 (32 workgroups) fp32
// 46 / 147 -> 20 / 54 us; 1 x 1000 of 128 (64) fp32 155 / 519 -> 60 / 203, bf16 29 / 102 -> 22 / 64; 2 x 2048 of 64 causal (256) fp32
// 168 / 578 -> 105 / 386; all rows alike (1 x 4095 of 64, 256) 334 / 1186 -> 333 / 1321; one tile long (32 x 100 causal, 256) 19 / 53 ->
// 19 / 89; of 128 causal (2 x 2000 x 16 heads, 512) 340 / 1127 -> 447 / 1640.  (The second clause's edges lie somewhere between these
// points: 100 and 512 tokens, heads of 64 and 128, 256 and 512 workgroups.)
inline bool attention_narrow(const vita_attention_args* a, int64_t wide) {
    if (a->dtype == VITA_DT_F32 && a->D > 96 && a->radius > 240) return false;                // its tiles and the bias gradient's rows fill the LDS
    // (bf16 tiles are short of delivery sooner: 4 x 1000 padded tokens of 64, 256: 28 / 84 -> 36 / 111)
    const bool uneven = a->dtype == VITA_DT_F32 && (a->causal || a->key_pad != nullptr);
    return wide < 256 || (wide < 512 && uneven && a->D <= 64 && a->Sq >= 512 && a->Sk >= 512);
}

template <class T> __device__ __forceinline__ const T* at(const AttnTensor& t, int b, int64_t s, int h) {
    return reinterpret_cast<const T*>(t.p) + b * t.sb + s * t.ss + h * t.sh;
}
template <class T> __device__ __forceinline__ T* at_mut(const AttnTensor& t, int b, int64_t s, int h) {
    return reinterpret_cast<T*>(t.p) + b * t.sb + s * t.ss + h * t.sh;
}
__host__ __device__ constexpr int stats_row(bool bf, int D) { return bf ? 4 + D / 2 : 2; }
// 4 consecutive columns of a result row, and of its stats row where the backward pass will want them
template <class T>
__device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
    if constexpr (sizeof(T) == 2) {
        bf16x4 v = {(bf16)a, (bf16)b, (bf16)c, (bf16)d};
        *reinterpret_cast<bf16x4*>(p) = v;
    } else {
        *reinterpret_cast<f32x4*>(p) = f32x4{a, b, c, d};
    }
}

// what bf16 leaves of 4 numbers, in bf16 again
__device__ __forceinline__ void store_rest4(float* stats, int c, float a, float b, float d, float e) {
    store4<bf16>(reinterpret_cast<bf16*>(stats + 4) + c, a - (float)(bf16)a, b - (float)(bf16)b, d - (float)(bf16)d, e - (float)(bf16)e);
}
template <class T>
__device__ __forceinline__ void store_stats(float* stats, float m, float r) {
    if constexpr (sizeof(T) == 2) *reinterpret_cast<f32x4*>(stats) = f32x4{m, r, 0.f, 0.f};
    else *reinterpret_cast<float2*>(stats) = make_float2(m, r);
}

int attention_check(const vita_attention_args* a, bool bwd, const char* who);
bool attention_sizes_ok(const vita_attention_args* a);      // whether a size query's sizes are ones that a call would take
void attention_fill(const vita_attention_args* a, AttnParams& p);

}  // namespace vita
