// tq_gemm_block.hip -- FP8 (e4m3) products with a scale for each block of 128:
//
//   y[m, n] = sum_b sa[b, m] sw[n / 128, b] sum_{k in b} qa[m, k] qw[n, k]  (+ bias[n])
//
// The FP8 matrix cores drop low bits of small products inside their sums (1.3e-5 of a 128-long
// sum on normal data, whatever the instruction shape, and no scale outside can bring them back), so
// codes are widened to f16, in which e4m3 is exact, and run on the f16 matrix cores with
// f32 sums: 1e-7.
#include "tq_gemm_tile.h"
#include "tq_rowfmt.h"

namespace tq {
namespace {

constexpr int kBlk = 128;
constexpr int kQuantBlock = 256;

template <int kType>
struct Act;
template <>
struct Act<TQ_DT_F32> {
    typedef float type;
};
template <>
struct Act<TQ_DT_BF16> {
    typedef __bf16 type;
};
template <>
struct Act<TQ_DT_F16> {
    typedef _Float16 type;
};

// 16 lanes, 8 columns each, for a row's 128; 16 such groups to a block, adjacent 128s of a row first.
template <int kType, bool kVec>
__global__ __launch_bounds__(kQuantBlock) void k_quant_g128(const void* x, int m, int k, uint8_t* __restrict__ q,
                                                            float* __restrict__ s) {
    typedef typename Act<kType>::type T;
    const int l = threadIdx.x & 15, blocks = (k + kBlk - 1) / kBlk;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 4);
    if (i >= static_cast<int64_t>(m) * blocks) return;
    const int row = static_cast<int>(i / blocks), b = static_cast<int>(i - static_cast<int64_t>(row) * blocks);
    const int k0 = b * kBlk + 8 * l;
    const T* p = static_cast<const T*>(x) + static_cast<int64_t>(row) * k + k0;
    float v[8];
    if constexpr (kVec) {  // k % 8 == 0, 16-byte aligned
        typedef T V __attribute__((ext_vector_type(8), aligned(16)));
        V u{};
        if (k0 < k) u = *reinterpret_cast<const V*>(p);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = static_cast<float>(u[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = k0 + e < k ? static_cast<float>(p[e]) : 0.0f;
    }
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (k0 + e < k) top = fmaxf(top, fabsf(v[e]));
    const float sc = row_scale<FmtFp8>(absmax_finish(group_max<16>(top)));
    const FmtFp8::Row coder(sc);
    *reinterpret_cast<uint2*>(q + (static_cast<int64_t>(row) * blocks + b) * kBlk + 8 * l) =
        make_uint2(coder.code4(f32x4{v[0], v[1], v[2], v[3]}), coder.code4(f32x4{v[4], v[5], v[6], v[7]}));
    if (l == 0) s[static_cast<int64_t>(b) * m + row] = sc;
}

// One 128 x 128 block of a weight to a thread block: thread t holds column t % 128 of rows
// t / 128 + 2 i (a weight is coded once, when a model is converted).
__global__ __launch_bounds__(kQuantBlock) void k_quant_block(const float* __restrict__ w, int n, int k,
                                                             uint8_t* __restrict__ q, float* __restrict__ s) {
    __shared__ float red[4];
    const int blocks = (k + kBlk - 1) / kBlk;
    const int nb = blockIdx.x / blocks, b = blockIdx.x - nb * blocks;
    const int col = b * kBlk + (threadIdx.x & 127), r0 = nb * kBlk + (threadIdx.x >> 7);
    const bool in = col < k;
    float v[64], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 64; ++i) {
        const int r = r0 + 2 * i;
        v[i] = in && r < n ? w[static_cast<int64_t>(r) * k + col] : 0.0f;
        if (in && r < n) top = fmaxf(top, fabsf(v[i]));
    }
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float sc = row_scale<FmtFp8>(absmax_finish(top));
    const FmtFp8::Row coder(sc);
    if (threadIdx.x == 0) s[blockIdx.x] = sc;
#pragma unroll
    for (int i = 0; i < 64; ++i) {
        const int r = r0 + 2 * i;
        if (in && r < n) q[static_cast<int64_t>(r) * k + col] = coder.code1(v[i]);
    }
}

__global__ __launch_bounds__(kQuantBlock) void k_dequant_block(const uint8_t* __restrict__ q, const float* __restrict__ s,
                                                               int64_t total, int k, float* __restrict__ w) {
    // (as many turns as it takes: weights may have more codes than a launch has threads)
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kQuantBlock + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * kQuantBlock) {
        const int row = static_cast<int>(i / k), col = static_cast<int>(i - static_cast<int64_t>(row) * k);
        w[i] = FmtFp8::value1(q[i], s[static_cast<int64_t>(row / kBlk) * ((k + kBlk - 1) / kBlk) + col / kBlk]);
    }
}

// ------------------------------------------------------------------ many tokens
// Block: 128 (m) x 128 (n), four waves of 64 x 64.  K in stages of one scale block, 128 codes, through two
// LDS buffers filled by direct global -> LDS loads (16-byte chunks XOR-swizzled by row, so that fragment
// reads do not conflict); codes stay bytes in LDS and become f16 after the fragment read: half the LDS of f16, whose
// fragments alone would fill it (128 bytes a cycle at 64 x 64 a wave).  A lane reads 16 adjacent codes of its row,
// two steps of v_mfma_f32_32x32x16_f16 (the order of k within a chunk is the same for both operands).  A stage's
// sums start from zero and join the totals times sa sw: W is the matrix cores' row operand, so a lane's sums share
// one token, and the factor is one number for each 32 tokens.
// The activations' codes are padded to whole stages with zeros; weight chunks past K re-read their row's first one,
// which meets those zeros.  Direct loads take K % 16 == 0 and 16-byte aligned weights.
// M=2047, N=4104, K=4000: 72 us and 5 for the joins, 0.93 PFLOP/s; 128 x 256 tiles, a block a CU, take 158.  A stage's 8
// conversions and 16 matrix instructions a wave fill the SIMD's issue; the two blocks of a CU cover each other's barriers.
constexpr int kTN = 2, kBM = 128, kBN = 64 * kTN, kBK = 128;

__device__ __forceinline__ int blk_swz(int row) { return (row >> 1) & 7; }

__device__ __forceinline__ tile_f16x8 widen8(int a, int b) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 x = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false));
    const h2 y = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true));
    const h2 z = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false));
    const h2 w = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true));
    return tile_f16x8{x.x, x.y, y.x, y.y, z.x, z.y, w.x, w.y};
}

struct BlockArgs {
    const uint8_t* a;  // [m, lda]
    const float* sa;   // [lda / 128, m]
    const uint8_t* w;  // [n, k]
    const float* sw;   // [n / 128, lda / 128]
    const float* bias;
    int m, n, k, lda, tiles_m, tiles_n;
    int full, split;  // tiles [0, full) have a block each, the others `split` blocks, each a share of K
    bool vec;         // n % 4 == 0, y and bias 16-byte aligned
    float* y;
    float* part;      // split > 1: sums of tile full + i's share s at [i * split + s][kBM][kBN]
};

// Tile L of the order in which n runs fastest within groups of eight row tiles.
__device__ __forceinline__ void block_tile(const BlockArgs& p, int L, int& tm, int& tn) {
    const int group = L / (8 * p.tiles_n), rows = min(8, p.tiles_m - group * 8), in = L - group * 8 * p.tiles_n;
    tm = group * 8 + in % rows;
    tn = in / rows;
}

// Bytes k0 .. k0 + 15 of a row of k >= 16, zeros past it: 16 bytes that end where the row does, shifted into place.
__device__ __forceinline__ u32x4 row_tail(const uint8_t* row, int k0, int k) {
    const int back = min(max(k0 + 16 - k, 0), 16);
    const u32x4 v = *reinterpret_cast<const u32x4_a1*>(row + k0 - max(k0 + 16 - k, 0));
    const int s = 8 * (back & 7);
    uint64_t lo = v.x | static_cast<uint64_t>(v.y) << 32, hi = v.z | static_cast<uint64_t>(v.w) << 32;
    lo = back >= 8 ? hi : lo;
    hi = back >= 8 ? 0 : hi;
    const uint64_t carry = s ? hi << (64 - s) : 0;
    lo = (lo >> s) | carry;
    hi >>= s;
    if (back == 16) lo = hi = 0;
    return u32x4{static_cast<uint32_t>(lo), static_cast<uint32_t>(lo >> 32), static_cast<uint32_t>(hi),
                 static_cast<uint32_t>(hi >> 32)};
}

// kAligned: as above; else the weights come through registers, 16 bytes at any address, and go to LDS behind the stage's
// products (M=2047, N=4104, the call of three launches: 88 us at K=4000, 102 at K=4001, 204 on the smaller tiles).
template <bool kAligned>
__global__ __launch_bounds__(256, 2) void k_gemm_block_dma(BlockArgs p) {
    constexpr int kWBytes = kBN * kBK, kStage = kWBytes + kBM * kBK;
    constexpr int kWDma = kBN / 32, kADma = kBM / 32;  // 16-byte loads of a lane for each stage (8 rows a wave and load)
    constexpr int kEpi = 32 * kTN + 4;                 // f32 row of the epilogue, padded
    __shared__ __attribute__((aligned(1024))) int8_t lds[2 * kStage];
    static_assert(4 * 32 * kEpi * 4 <= 2 * kStage, "the epilogue fits");
    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 31, lh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave & 1, wn = wave >> 1;
    // each XCD (consecutive blocks go to different ones) has a contiguous run of tiles, so that blocks
    // sharing an L2 share operand rows
    int L = blockIdx.x, share = 0;
    if (L < p.full) {
        const int q8 = p.full >> 3, r8 = p.full & 7, xcd = L & 7;
        L = xcd * q8 + min(xcd, r8) + (L >> 3);
    } else {
        share = (L - p.full) % p.split;
        L = p.full + (L - p.full) / p.split;
    }
    const bool whole = L < p.full || p.split == 1;
    int tm, tn;
    block_tile(p, L, tm, tn);
    const int m0 = tm * kBM, n0 = tn * kBN;

    // load t of a lane: row 8 slot + lane / 8 of its operand, global chunk (lane % 8) ^ swz in LDS chunk lane % 8
    const int8_t* src[kWDma + kADma];
    int chunk[2];  // the lane's column of codes in loads of even and odd slots
    uint32_t dst[kWDma + kADma];
#pragma unroll
    for (int t = 0; t < kWDma + kADma; ++t) {
        const bool isw = t < kWDma;
        const int slot = isw ? kWDma * wave + t : kADma * wave + t - kWDma;
        const int row = slot * 8 + (lane >> 3);
        const int koff = ((lane & 7) ^ blk_swz(row)) * 16;
        if (t < 2) chunk[t] = koff;
        src[t] = isw ? reinterpret_cast<const int8_t*>(p.w) + static_cast<int64_t>(min(n0 + row, p.n - 1)) * p.k + koff
                     : reinterpret_cast<const int8_t*>(p.a) + static_cast<int64_t>(min(m0 + row, p.m - 1)) * p.lda + koff;
        dst[t] = lds_addr(lds) + (isw ? 0 : kWBytes) + slot * 1024;
    }
    static_assert(kWDma % 2 == 0, "swizzles alternate between even and odd slots");
    u32x4 held[kAligned ? 1 : kWDma];
    auto load_stage = [&](int k0, int buf) {
        const uint32_t to = buf * kStage;
        if constexpr (!kAligned) {
#pragma unroll
            for (int t = 0; t < kWDma; ++t) {
                if (k0 + kBK <= p.k)
                    held[t] = *reinterpret_cast<const u32x4_a1*>(src[t] + k0);
                else
                    held[t] = row_tail(reinterpret_cast<const uint8_t*>(src[t]) - chunk[t & 1], k0 + chunk[t & 1], p.k);
            }
#pragma unroll
            for (int t = kWDma; t < kWDma + kADma; ++t) lds_dma16(src[t] + k0, dst[t] + to);
        } else if (k0 + kBK <= p.k) {
#pragma unroll
            for (int t = 0; t < kWDma + kADma; ++t) lds_dma16(src[t] + k0, dst[t] + to);
        } else {
#pragma unroll
            for (int t = 0; t < kWDma; ++t)
                lds_dma16(src[t] + (k0 + chunk[t & 1] < p.k ? k0 : -chunk[t & 1]), dst[t] + to);
#pragma unroll
            for (int t = kWDma; t < kWDma + kADma; ++t) lds_dma16(src[t] + k0, dst[t] + to);
        }
    };

    auto store_stage = [&](int buf) {
        if constexpr (!kAligned) {
#pragma unroll
            for (int t = 0; t < kWDma; ++t)
                *reinterpret_cast<u32x4*>(lds + buf * kStage + (kWDma * wave + t) * 1024 + 16 * lane) = held[t];
        }
    };

    f32x16 tot[kTN][2];
#pragma unroll
    for (int i = 0; i < kTN; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) tot[i][j] = f32x16{};
    const int stages = p.lda / kBK;
    const int s_begin = whole ? 0 : static_cast<int>(static_cast<int64_t>(share) * stages / p.split);
    const int s_end = whole ? stages : static_cast<int>(static_cast<int64_t>(share + 1) * stages / p.split);
    const float* sa = p.sa + m0 + wm * 64;
    int col[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) col[j] = min(32 * j + lr, p.m - 1 - m0 - wm * 64);  // (may be negative: rows past m)
    const float* sw = p.sw + static_cast<int64_t>(min(n0 + wn * 32 * kTN, p.n - 1) >> 7) * stages;
    float fa[2], fw;
    auto load_scales = [&](int s) {
#pragma unroll
        for (int j = 0; j < 2; ++j) fa[j] = sa[static_cast<int64_t>(s) * p.m + col[j]];
        fw = sw[s];
    };
    load_scales(s_begin);
    load_stage(s_begin * kBK, s_begin & 1);
    store_stage(s_begin & 1);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    // fragments: the next 32 codes' are read while these run, a stage's first ones while the sums of the one
    // before join the totals
    i32x4 w[2][kTN], x[2][2];
    auto read = [&](const int8_t* st, int c) {
        const int ch = 2 * c + lh;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int row = wm * 64 + 32 * j + lr;
            x[c & 1][j] = *reinterpret_cast<const i32x4*>(st + kWBytes + row * kBK + ((ch ^ blk_swz(row)) << 4));
        }
#pragma unroll
        for (int i = 0; i < kTN; ++i) {
            const int row = wn * 32 * kTN + 32 * i + lr;
            w[c & 1][i] = *reinterpret_cast<const i32x4*>(st + row * kBK + ((ch ^ blk_swz(row)) << 4));
        }
    };
    read(lds + (s_begin & 1) * kStage, 0);
    for (int s = s_begin; s < s_end; ++s) {
        const int8_t* st = lds + (s & 1) * kStage;
        float f[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) f[j] = fa[j] * fw;
        if (s + 1 < s_end) {
            load_stage((s + 1) * kBK, (s + 1) & 1);
            load_scales(s + 1);
        }
        f32x16 acc[kTN][2];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if (c < 3) read(st, c + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                tile_f16x8 xf[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) xf[j] = widen8(x[c & 1][j][2 * half], x[c & 1][j][2 * half + 1]);
#pragma unroll
                for (int i = 0; i < kTN; ++i) {
                    const tile_f16x8 wf = widen8(w[c & 1][i][2 * half], w[c & 1][i][2 * half + 1]);
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(wf, xf[j], c + half ? acc[i][j] : f32x16{}, 0, 0, 0);
                }
            }
        }
        if (s + 1 < s_end) store_stage((s + 1) & 1);
        // the next stage has landed and every wave is past its reads of this one
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        read(lds + ((s + 1) & 1) * kStage, 0);  // (after the last stage: read and not used)
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < kTN; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) tot[i][j][e] = fmaf(acc[i][j][e], f[j], tot[i][j][e]);
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");

    // lane holds y[m = 32 j + lr][n = 32 i + 8 (e / 4) + 4 lh + e % 4] of the wave's tile: 32 rows at a time through
    // LDS, out again as runs of n
    float* ep = reinterpret_cast<float*>(lds) + wave * (32 * kEpi);
    const int nb = n0 + wn * 32 * kTN;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int i = 0; i < kTN; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<f32x4*>(ep + lr * kEpi + 32 * i + 8 * g + 4 * lh) =
                    f32x4{tot[i][j][4 * g], tot[i][j][4 * g + 1], tot[i][j][4 * g + 2], tot[i][j][4 * g + 3]};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const int mb = m0 + wm * 64 + 32 * j;
        if (!whole) {
            float* o = p.part + (static_cast<int64_t>(L - p.full) * p.split + share) * (kBM * kBN) +
                       (wm * 64 + 32 * j) * kBN + wn * 32 * kTN;
            constexpr int kLanes = 8 * kTN;
#pragma unroll 4
            for (int r = lane / kLanes; r < 32; r += 64 / kLanes)
                *reinterpret_cast<f32x4*>(o + r * kBN + 4 * (lane % kLanes)) =
                    *reinterpret_cast<const f32x4*>(ep + r * kEpi + 4 * (lane % kLanes));
        } else if (p.vec) {
            constexpr int kLanes = 8 * kTN;  // of a row, four n each
            const int c4 = 4 * (lane % kLanes), nn = nb + c4;
            f32x4 b = f32x4{0.f, 0.f, 0.f, 0.f};
            if (p.bias && nn < p.n) b = *reinterpret_cast<const f32x4*>(p.bias + nn);
#pragma unroll 4
            for (int r = lane / kLanes; r < 32; r += 64 / kLanes) {
                const f32x4 v = *reinterpret_cast<const f32x4*>(ep + r * kEpi + c4) + b;
                if (nn < p.n && mb + r < p.m)
                    __builtin_nontemporal_store(v, reinterpret_cast<f32x4*>(p.y + static_cast<int64_t>(mb + r) * p.n + nn));
            }
        } else {
            for (int i = lane; i < 32 * 32 * kTN; i += 64) {
                const int r = i / (32 * kTN), c = i % (32 * kTN), nn = nb + c;
                if (nn < p.n && mb + r < p.m)
                    p.y[static_cast<int64_t>(mb + r) * p.n + nn] = ep[r * kEpi + c] + (p.bias ? p.bias[nn] : 0.f);
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// ------------------------------------------------------------------ few tokens
// Up to 16 kNT tokens: a block a CU, with 16 weight rows after 16, sixteen waves that take K in blocks of 128 by
// turns, two at a time in flight and the next two, of these or of the block's next rows, behind them.  Lane (r, q) =
// (l % 16, l / 16) has the codes 16 q .. and 64 + 16 q .. of its row and of its token (64-byte runs of a row in each
// load), four steps of v_mfma_f32_16x16x32_f16 (8 codes of each, in the same order); a block's sums join the total
// times sa sw, and the waves' totals meet in LDS.  The activations' codes lie in LDS: coded there by each block from x
// (kFromX: for a token or few, the launch that codes them costs more), copied (kFromCodes), or, where they do not fit,
// read as they are needed (kFromMemory).
// One token, N=14336, K=4096: 16 us, 3.7 TB/s; the loads alone, without a product, take 14.9 (their 64-byte runs; whole
// 128-byte lines or non-temporal loads are no faster), waves of eight with four blocks in flight each 16.4.
enum { kFromX, kFromCodes, kFromMemory };
constexpr int kSkinnyWaves = 16, kSkinnyThreads = 64 * kSkinnyWaves, kSkinnyU = 2;

// Codes that a block keeps in LDS, beside 32 KB of partial sums; and those that each block makes itself.
constexpr int kSkinnyCodes = 24576, kSkinnyFused = 16384;

struct SkinnyArgs {
    const void* x;     // activations (kFromX)
    const uint8_t* a;  // codes [m, lda] and scales [lda / 128, m] (else)
    const float* sa;
    const uint8_t* w;
    const float* sw;
    const float* bias;
    int m, n, k, lda;
    float* y;
};

template <int kType, int kFrom, int kNT>
__global__ __launch_bounds__(kSkinnyThreads, 4) void k_gemm_block_skinny(SkinnyArgs p) {
    typedef typename Act<kType>::type T;
    constexpr int kParts = kNT == 1 ? 2 : 1;
    __shared__ f32x4 part[kParts][kSkinnyWaves][kNT][64];
    extern __shared__ __attribute__((aligned(16))) uint8_t codes[];  // [m][lda], then scales [lda / 128][m]
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int blocks = p.lda / kBlk, tiles = static_cast<int>((static_cast<int64_t>(p.n) + 15) / 16);
    constexpr int kTurn = kSkinnyWaves * kSkinnyU;
    const int whole = p.k / kBlk;  // blocks of 128; a partial last one comes apart
    u32x4 cur[kSkinnyU][2], nxt[kSkinnyU][2];
    float cur_s[kSkinnyU], nxt_s[kSkinnyU];
    auto load = [&](u32x4 (&w)[kSkinnyU][2], float (&sc)[kSkinnyU], int tile, int c0) {
        const uint8_t* wr = p.w + min(static_cast<int64_t>(tile) * 16 + r, static_cast<int64_t>(p.n - 1)) * p.k + 16 * q;
        const float* sw = p.sw + (tile >> 3) * static_cast<int64_t>(blocks);
#pragma unroll
        for (int u = 0; u < kSkinnyU; ++u) {  // past the last: the last one again, not used
            const int c = min(c0 + kSkinnyWaves * u, whole - 1);
            const uint8_t* at = wr + static_cast<int64_t>(c) * kBlk;
#pragma unroll
            for (int i = 0; i < 2; ++i) w[u][i] = *reinterpret_cast<const u32x4_a1*>(at + 64 * i);
            sc[u] = sw[c];
        }
    };
    if (whole) load(cur, cur_s, blockIdx.x, wave);
    float* scales = reinterpret_cast<float*>(codes + p.m * p.lda);
    if constexpr (kFrom == kFromCodes) {
        for (int i = tid; i < p.m * p.lda / 16; i += kSkinnyThreads)
            reinterpret_cast<u32x4*>(codes)[i] = reinterpret_cast<const u32x4*>(p.a)[i];
        for (int i = tid; i < p.m * blocks; i += kSkinnyThreads) scales[i] = p.sa[i];
        __syncthreads();
    }
    if constexpr (kFrom == kFromX) {
        // 16 lanes, 8 columns each, for a row's 128
        for (int i = tid >> 4; i < p.m * blocks; i += kSkinnyThreads / 16) {
            const int row = i / blocks, b = i - row * blocks, k0 = b * kBlk + 8 * (tid & 15);
            const T* src = static_cast<const T*>(p.x) + static_cast<int64_t>(row) * p.k + k0;
            float v[8], top = -INFINITY;
            if (p.k % 8 == 0 && (reinterpret_cast<uintptr_t>(p.x) & 15) == 0) {  // uniform
                typedef T V __attribute__((ext_vector_type(8), aligned(16)));
                V t{};
                if (k0 < p.k) t = *reinterpret_cast<const V*>(src);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = static_cast<float>(t[e]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = k0 + e < p.k ? static_cast<float>(src[e]) : 0.0f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (k0 + e < p.k) top = fmaxf(top, fabsf(v[e]));
            const float sc = row_scale<FmtFp8>(absmax_finish(group_max<16>(top)));
            const FmtFp8::Row coder(sc);
            *reinterpret_cast<uint2*>(codes + row * p.lda + k0) =
                make_uint2(coder.code4(f32x4{v[0], v[1], v[2], v[3]}), coder.code4(f32x4{v[4], v[5], v[6], v[7]}));
            if ((tid & 15) == 0) scales[b * p.m + row] = sc;
        }
        __syncthreads();
    }
    // the block's tiles one after the other: the next weights, of this tile or of the next one, are in flight
    int buf = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, buf ^= kParts - 1) {
        const int64_t n0 = static_cast<int64_t>(tile) * 16;
        f32x4 tot[kNT];
#pragma unroll
        for (int t = 0; t < kNT; ++t) tot[t] = f32x4{};
        // the sums of block c, whose weight codes are in w, into the totals
        auto add = [&](const u32x4 (&w)[2], float fw, int c) {
            tile_f16x8 wf[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                wf[i] = widen8(static_cast<int>(w[i >> 1][2 * (i & 1)]), static_cast<int>(w[i >> 1][2 * (i & 1) + 1]));
#pragma unroll
            for (int t = 0; t < kNT; ++t) {
                const int row = 16 * t + r;
                u32x4 x[2] = {};
                float fa = 0.f;
                if (row < p.m) {
                    if constexpr (kFrom == kFromMemory) {
                        const uint8_t* at = p.a + static_cast<int64_t>(row) * p.lda + c * kBlk + 16 * q;
                        x[0] = *reinterpret_cast<const u32x4*>(at);
                        x[1] = *reinterpret_cast<const u32x4*>(at + 64);
                        fa = p.sa[static_cast<int64_t>(c) * p.m + row];
                    } else {
                        const uint8_t* at = codes + row * p.lda + c * kBlk + 16 * q;
                        x[0] = *reinterpret_cast<const u32x4*>(at);
                        x[1] = *reinterpret_cast<const u32x4*>(at + 64);
                        fa = scales[c * p.m + row];
                    }
                }
                f32x4 d{};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    d = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        wf[i], widen8(static_cast<int>(x[i >> 1][2 * (i & 1)]), static_cast<int>(x[i >> 1][2 * (i & 1) + 1])), d,
                        0, 0, 0);
                const float f = fa * fw;
#pragma unroll
                for (int e = 0; e < 4; ++e) tot[t][e] = fmaf(d[e], f, tot[t][e]);
            }
        };
        for (int c0 = wave; c0 < whole + wave; c0 += kTurn) {  // as many turns for every wave
            const bool more = c0 - wave + kTurn < whole;
            const int next = more ? tile : min(tile + static_cast<int>(gridDim.x), tiles - 1);
            load(nxt, nxt_s, next, more ? c0 + kTurn : wave);  // (after the last tile: read and not used)
#pragma unroll
            for (int u = 0; u < kSkinnyU; ++u) {
                if (c0 + kSkinnyWaves * u < whole) add(cur[u], cur_s[u], c0 + kSkinnyWaves * u);  // uniform
                __builtin_amdgcn_sched_barrier(0);  // (both blocks' fragments at once would not fit)
            }
#pragma unroll
            for (int u = 0; u < kSkinnyU; ++u) {
                cur[u][0] = nxt[u][0];
                cur[u][1] = nxt[u][1];
                cur_s[u] = nxt_s[u];
            }
        }
        if (whole < blocks && wave == whole % kSkinnyWaves) {  // the partial last block, zeros past K
            const uint8_t* row = p.w + min(n0 + r, static_cast<int64_t>(p.n - 1)) * p.k;
            u32x4 w[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) w[i] = row_tail(row, whole * kBlk + 16 * q + 64 * i, p.k);
            add(w, p.sw[(tile >> 3) * static_cast<int64_t>(blocks) + whole], whole);
        }
#pragma unroll
        for (int t = 0; t < kNT; ++t) part[buf][wave][t][lane] = tot[t];
        __syncthreads();  // (of two parts the other one is read before the barrier after this one)
        // thread: weight row i % 16, token i / 16
        for (int i = tid; i < 256 * kNT; i += kSkinnyThreads) {
            const int row = i & 15, token = i >> 4, src = (row >> 2) * 16 + (token & 15), e = row & 3;
            const int64_t nn = n0 + row;
            if (token >= p.m || nn >= p.n) continue;
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < kSkinnyWaves; ++w) v += part[buf][w][token >> 4][src][e];
            p.y[static_cast<int64_t>(token) * p.n + nn] = v + (p.bias ? p.bias[nn] : 0.f);
        }
        if (kParts == 1) __syncthreads();
    }
}

// Adds the shares of the split tiles in order: four n of a row to a thread.
__global__ __launch_bounds__(256) void k_gemm_block_join(BlockArgs p) {
    const int per = kBM * kBN / 4 / 256;
    const int tile = blockIdx.x / per, i = (blockIdx.x - tile * per) * 256 + threadIdx.x;
    const int r = i / (kBN / 4), c = i % (kBN / 4) * 4;
    int tm, tn;
    block_tile(p, p.full + tile, tm, tn);
    const int mm = tm * kBM + r, nn = tn * kBN + c;
    if (mm >= p.m || nn >= p.n) return;
    const float* o = p.part + static_cast<int64_t>(tile) * p.split * (kBM * kBN) + r * kBN + c;
    f32x4 v = *reinterpret_cast<const f32x4*>(o);
    for (int s = 1; s < p.split; ++s) v += *reinterpret_cast<const f32x4*>(o + static_cast<int64_t>(s) * (kBM * kBN));
    float* y = p.y + static_cast<int64_t>(mm) * p.n + nn;
    if (p.vec) {
        if (p.bias) v += *reinterpret_cast<const f32x4*>(p.bias + nn);
        *reinterpret_cast<f32x4*>(y) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (nn + e < p.n) y[e] = v[e] + (p.bias ? p.bias[nn + e] : 0.f);
    }
}

// The tiles of 128 x 128 fill the chip's slots (two blocks a CU) in whole rounds; those of the last, partial round are
// cut along K into as many shares as there are slots for them, of four stages at least (M=2047, N=4104, K=4000:
// 528 tiles, 16 of them in a second round: 104 us whole, 79 us with these in 8 shares).
struct BlockPlan {
    int full, left, split;
    int64_t part_bytes;
};
BlockPlan block_plan(int64_t m, int64_t n, int64_t k) {
    const int64_t slots = 2 * device_cu_count(), stages = (k + kBK - 1) / kBK;
    const int64_t tiles = ((m + kBM - 1) / kBM) * ((n + 127) / 128);
    BlockPlan b{};
    b.left = static_cast<int>(tiles % slots);
    b.full = static_cast<int>(tiles - b.left);
    b.split = 1;
    if (b.left) {
        b.split = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({slots / b.left, stages / 4, 8})));
    }
    if (b.split == 1) {
        b.full = static_cast<int>(tiles);
        b.left = 0;
    }
    b.part_bytes = b.split > 1 ? static_cast<int64_t>(b.left) * b.split * (kBM * 128 * 4) : 0;
    return b;
}
// From 64 tokens on (N=14336, K=4096: 31.5 us against the smaller tiles' 32.3, with 96 tokens 33.8 against 45); a stage
// of K at least.
bool block_dma(int64_t m, int64_t k) { return k >= kBK && m >= 64; }

bool block_fits(int64_t m, int64_t n, int64_t k) { return tile_fits(m, n, k); }

int check_sizes(const char* what, int64_t m, int64_t n, int64_t k) {
    TQ_REQUIRE(m >= 0 && n >= 0 && k >= 0, "%s: negative shape", what);
    TQ_REQUIRE(block_fits(m, n, k), "%s: M=%lld, N=%lld, K=%lld are past the kernels' 32-bit indexes", what, (long long)m,
               (long long)n, (long long)k);
    return TQ_OK;
}

struct BlockLayout {
    int64_t sa, part;
};
BlockLayout block_layout(int64_t m, int64_t k) {
    const int64_t blocks = (k + kBlk - 1) / kBlk;
    const int64_t sa = (m * blocks * kBlk + 255) / 256 * 256;
    return BlockLayout{sa, sa + (4 * m * blocks + 255) / 256 * 256};
}

// Up to 16 tokens (N=14336, K=4096, us: 17 for one, 23 for 8 and 25.5 for 16, against 25.5 to 26 of the tile kernel), and
// up to 32 where a block has one tile and K is short (N=K=4096: 13.7 against 17.3; N=14336: 34 against 26; N=4096, K=14336:
// 29.6 against 28.6).
bool block_skinny(int64_t m, int64_t n, int64_t k) {
    return k >= kBlk && (m <= 16 || (m <= 32 && k <= 4096 && (n + 15) / 16 <= device_cu_count()));
}
// Codes made by each block: N=14336, K=4096 17.0 us for one token against 19.1, for four 19.0 against 19.2.
bool block_fused(int64_t m, int64_t n, int64_t k) {
    return block_skinny(m, n, k) && m * ((k + kBlk - 1) / kBlk * kBlk) <= kSkinnyFused;
}

template <int kType, int kFrom>
int launch_skinny(const SkinnyArgs& p, hipStream_t st, const char* what) {
    // as many blocks as the chip holds at once (one a CU), each with as many tiles as the others
    const int64_t tiles = (static_cast<int64_t>(p.n) + 15) / 16, fit = device_cu_count();
    const unsigned grid = static_cast<unsigned>((tiles + (tiles + fit - 1) / fit - 1) / ((tiles + fit - 1) / fit));
    const unsigned lds = kFrom == kFromMemory ? 0 : static_cast<unsigned>(p.m * p.lda + 4 * p.m * (p.lda / kBlk));
    clear_error();
    if (p.m <= 16)
        k_gemm_block_skinny<kType, kFrom, 1><<<grid, kSkinnyThreads, lds, st>>>(p);
    else
        k_gemm_block_skinny<kType, kFrom, 2><<<grid, kSkinnyThreads, lds, st>>>(p);
    return check_launch(what);
}

SkinnyArgs skinny_args(const uint8_t* qw, const float* sw, const float* bias, int64_t m, int64_t n, int64_t k, float* y) {
    SkinnyArgs p{};
    p.w = qw;
    p.sw = sw;
    p.bias = bias;
    p.m = static_cast<int>(m);
    p.n = static_cast<int>(n);
    p.k = static_cast<int>(k);
    p.lda = static_cast<int>((k + kBlk - 1) / kBlk * kBlk);
    p.y = y;
    return p;
}

int gemm_block(const uint8_t* qa, const float* sa, const uint8_t* qw, const float* sw, const float* bias, int64_t m,
               int64_t n, int64_t k, void* ws, int64_t ws_bytes, float* y, hipStream_t st, const char* what) {
    int rc = check_sizes(what, m, n, k);
    if (rc != TQ_OK) return rc;
    if (m == 0 || n == 0) return TQ_OK;
    TQ_REQUIRE(y && (k == 0 || (qa && sa && qw && sw)), "%s: null pointer", what);
    TQ_REQUIRE(aligned(qa, 16) && aligned(sa, 4) && aligned(sw, 4) && aligned(y, 4) && aligned(bias, 4),
               "%s: misaligned pointer", what);
    if (block_skinny(m, n, k)) {
        SkinnyArgs p = skinny_args(qw, sw, bias, m, n, k, y);
        p.a = qa;
        p.sa = sa;
        return m * p.lda <= kSkinnyCodes ? launch_skinny<TQ_DT_F32, kFromCodes>(p, st, what)
                                         : launch_skinny<TQ_DT_F32, kFromMemory>(p, st, what);
    }
    if (block_dma(m, k)) {
        const BlockPlan plan = block_plan(m, n, k);
        TQ_REQUIRE(plan.part_bytes == 0 || (ws && aligned(ws, 256) && ws_bytes >= plan.part_bytes),
                   "%s: workspace of %lld bytes (256-byte aligned), %lld needed", what, (long long)ws_bytes,
                   (long long)plan.part_bytes);
        BlockArgs b{};
        b.a = qa;
        b.sa = sa;
        b.w = qw;
        b.sw = sw;
        b.bias = bias;
        b.m = static_cast<int>(m);
        b.n = static_cast<int>(n);
        b.k = static_cast<int>(k);
        b.lda = static_cast<int>((k + kBlk - 1) / kBlk * kBlk);
        b.tiles_m = static_cast<int>((m + kBM - 1) / kBM);
        b.tiles_n = static_cast<int>((n + 127) / 128);
        b.full = plan.full;
        b.split = plan.split;
        b.vec = n % 4 == 0 && aligned(y, 16) && aligned(bias, 16);
        b.y = y;
        b.part = static_cast<float*>(ws);
        TQ_REQUIRE(plan.full <= kMaxBlocks - plan.left * plan.split, "%s: M=%lld, N=%lld are more than %lld blocks", what, (long long)m,
                   (long long)n, (long long)kMaxBlocks);
        clear_error();
        const unsigned grid = static_cast<unsigned>(plan.full + plan.left * plan.split);
        if (k % 16 == 0 && aligned(qw, 16))
            k_gemm_block_dma<true><<<grid, 256, 0, st>>>(b);
        else
            k_gemm_block_dma<false><<<grid, 256, 0, st>>>(b);
        rc = check_launch(what);
        if (rc != TQ_OK || plan.split == 1) return rc;
        k_gemm_block_join<<<plan.left * (kBM * kBN / 4 / 256), 256, 0, st>>>(b);
        return check_launch(what);
    }
    const TilePlan plan = tile_plan<GemmF8Block>(m, n, k, nullptr, true);
    TQ_REQUIRE(plan.part_bytes == 0 || (ws && aligned(ws, 256) && ws_bytes >= plan.part_bytes),
               "%s: workspace of %lld bytes (256-byte aligned), %lld needed", what, (long long)ws_bytes,
               (long long)plan.part_bytes);
    TQ_REQUIRE(static_cast<int64_t>(plan.tiles_m) * plan.tiles_n * plan.split <= kMaxBlocks, "%s: M=%lld, N=%lld are more than %lld blocks",
               what, (long long)m, (long long)n, (long long)kMaxBlocks);
    TileArgs p{};
    p.a = qa;
    p.w = qw;
    p.sa = sa;
    p.sw = sw;
    p.bias = bias;
    p.m = static_cast<int>(m);
    p.n = static_cast<int>(n);
    p.k = static_cast<int>(k);
    p.lda = static_cast<int>((k + kBlk - 1) / kBlk * kBlk);
    p.y = y;
    p.part = ws;
    clear_error();
    return launch_tile<GemmF8Block>(plan, p, st, what);
}

int quantize_g128(const void* x, int dtype, int64_t m, int64_t k, uint8_t* q, float* s, hipStream_t st, const char* what) {
    TQ_REQUIRE(dtype == TQ_DT_F32 || dtype == TQ_DT_BF16 || dtype == TQ_DT_F16, "%s: dtype %d is not f32, bf16 or f16", what,
               dtype);
    int rc = check_sizes(what, m, 1, k);
    if (rc != TQ_OK) return rc;
    if (m == 0 || k == 0) return TQ_OK;
    const int64_t size = dtype == TQ_DT_F32 ? 4 : 2;
    TQ_REQUIRE(x && q && s, "%s: null pointer", what);
    TQ_REQUIRE(aligned(x, size) && aligned(q, 16) && aligned(s, 4), "%s: misaligned pointer", what);
    const int64_t groups = m * ((k + kBlk - 1) / kBlk);
    TQ_REQUIRE((groups + 15) / 16 <= kMaxBlocks, "%s: M=%lld, K=%lld are more than %lld blocks", what, (long long)m, (long long)k,
               (long long)kMaxBlocks);
    const unsigned grid = static_cast<unsigned>((groups + 15) / 16);
    const bool vec = k % 8 == 0 && aligned(x, 16);
    const int mi = static_cast<int>(m), ki = static_cast<int>(k);
    clear_error();
#define TQ_QUANT(T)                                                                \
    if (vec)                                                                       \
        k_quant_g128<T, true><<<grid, kQuantBlock, 0, st>>>(x, mi, ki, q, s);      \
    else                                                                           \
        k_quant_g128<T, false><<<grid, kQuantBlock, 0, st>>>(x, mi, ki, q, s)
    if (dtype == TQ_DT_F32) {
        TQ_QUANT(TQ_DT_F32);
    } else if (dtype == TQ_DT_BF16) {
        TQ_QUANT(TQ_DT_BF16);
    } else {
        TQ_QUANT(TQ_DT_F16);
    }
#undef TQ_QUANT
    return check_launch(what);
}

}  // namespace
}  // namespace tq

using namespace tq;

extern "C" {

int tq_quantize_fp8_block(const float* w, int64_t n, int64_t k, uint8_t* q, float* s, tq_stream_t stream) {
    static const char* what = "tq_quantize_fp8_block";
    const int rc = check_sizes(what, 1, n, k);
    if (rc != TQ_OK || n == 0 || k == 0) return rc;
    TQ_REQUIRE(w && q && s, "%s: null pointer", what);
    TQ_REQUIRE(aligned(w, 4) && aligned(s, 4), "%s: misaligned pointer", what);
    const int64_t blocks = ((n + kBlk - 1) / kBlk) * ((k + kBlk - 1) / kBlk);
    TQ_REQUIRE(blocks <= kMaxBlocks, "%s: N=%lld, K=%lld are more than %lld blocks", what, (long long)n, (long long)k,
               (long long)kMaxBlocks);
    clear_error();
    k_quant_block<<<static_cast<unsigned>(blocks), kQuantBlock, 0, as_hip(stream)>>>(w, static_cast<int>(n),
                                                                                     static_cast<int>(k), q, s);
    return check_launch(what);
}

int tq_dequantize_fp8_block(const uint8_t* q, const float* s, int64_t n, int64_t k, float* w_hat, tq_stream_t stream) {
    static const char* what = "tq_dequantize_fp8_block";
    const int rc = check_sizes(what, 1, n, k);
    if (rc != TQ_OK || n == 0 || k == 0) return rc;
    TQ_REQUIRE(q && s && w_hat, "%s: null pointer", what);
    TQ_REQUIRE(aligned(s, 4) && aligned(w_hat, 4), "%s: misaligned pointer", what);
    const int64_t grid = std::min((n * k + kQuantBlock - 1) / kQuantBlock, kMaxBlocks);
    clear_error();
    k_dequant_block<<<static_cast<unsigned>(grid), kQuantBlock, 0, as_hip(stream)>>>(q, s, n * k, static_cast<int>(k), w_hat);
    return check_launch(what);
}

int tq_quantize_fp8_g128(const void* x, int dtype, int64_t m, int64_t k, uint8_t* q, float* s, tq_stream_t stream) {
    return quantize_g128(x, dtype, m, k, q, s, as_hip(stream), "tq_quantize_fp8_g128");
}

int64_t tq_gemm_fp8_block_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    if (m < 0 || n < 0 || k < 0 || !block_fits(m, n, k)) return -1;
    if (m == 0 || n == 0) return 0;
    return block_dma(m, k) ? block_plan(m, n, k).part_bytes : tile_plan<GemmF8Block>(m, n, k, nullptr, true).part_bytes;
}

int tq_gemm_fp8_block(const uint8_t* qa, const float* sa, const uint8_t* qw, const float* sw, const float* bias,
                      int64_t m, int64_t n, int64_t k, void* workspace, int64_t workspace_bytes, float* y,
                      tq_stream_t stream) {
    return gemm_block(qa, sa, qw, sw, bias, m, n, k, workspace, workspace_bytes, y, as_hip(stream), "tq_gemm_fp8_block");
}

int64_t tq_linear_fp8_block_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    const int64_t part = tq_gemm_fp8_block_workspace_bytes(m, n, k);
    return part < 0 ? -1 : m == 0 || n == 0 ? 0 : block_layout(m, k).part + part;
}

int tq_linear_fp8_block(const void* x, int dtype, int64_t m, const uint8_t* qw, const float* sw, const float* bias,
                        int64_t n, int64_t k, void* workspace, int64_t workspace_bytes, float* y, tq_stream_t stream) {
    static const char* what = "tq_linear_fp8_block";
    int rc = check_sizes(what, m, n, k);
    if (rc != TQ_OK || m == 0 || n == 0) return rc;
    TQ_REQUIRE(y && (k == 0 || (x && qw && sw)), "%s: null pointer", what);
    TQ_REQUIRE(aligned(sw, 4) && aligned(y, 4) && aligned(bias, 4), "%s: misaligned pointer", what);
    const int64_t need = tq_linear_fp8_block_workspace_bytes(m, n, k);
    TQ_REQUIRE(need == 0 || (workspace && aligned(workspace, 256) && workspace_bytes >= need),
               "%s: workspace of %lld bytes (256-byte aligned), %lld needed", what, (long long)workspace_bytes,
               (long long)need);
    if (block_fused(m, n, k)) {
        TQ_REQUIRE(aligned(x, dtype == TQ_DT_F32 ? 4 : 2) && (dtype == TQ_DT_F32 || dtype == TQ_DT_BF16 || dtype == TQ_DT_F16),
                   "%s: dtype %d, or x not aligned to its elements", what, dtype);
        SkinnyArgs p = skinny_args(qw, sw, bias, m, n, k, y);
        p.x = x;
        return dtype == TQ_DT_F32    ? launch_skinny<TQ_DT_F32, kFromX>(p, as_hip(stream), what)
               : dtype == TQ_DT_BF16 ? launch_skinny<TQ_DT_BF16, kFromX>(p, as_hip(stream), what)
                                     : launch_skinny<TQ_DT_F16, kFromX>(p, as_hip(stream), what);
    }
    const BlockLayout lay = block_layout(m, k);
    uint8_t* q = static_cast<uint8_t*>(workspace);
    float* s = reinterpret_cast<float*>(q + lay.sa);
    if ((rc = quantize_g128(x, dtype, m, k, q, s, as_hip(stream), what)) != TQ_OK) return rc;
    return gemm_block(q, s, qw, sw, bias, m, n, k, q + lay.part, need - lay.part, y, as_hip(stream), what);
}

}  // extern "C"
