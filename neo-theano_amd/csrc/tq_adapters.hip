// tq_adapters.hip -- low-rank adapters of many requests beside one projection.
//
//   t[i]   = A_a x_i                       (A_a [parts * rank, K], a = index[i])
//   out[i] = y[i] + s_a B_a t[i]           (B_a [N, rank]; output slice p uses ranks p of t)
//
// Both products run on v_mfma_f32_16x16x32 with the weights as the first operand (16 ranks, or 16
// outputs) and 16 tokens as the second, so that a lane's four sums are neighbours in t and in y.  A tile of tokens
// may hold several adapters: the distinct ones are taken one after the other (or by blocks of their own), each
// with all 16 tokens, and a token keeps the sums of its own adapter.  What a token does not use cannot reach
// it, since a token is a column of its own.  Sums are f32 and the operands exact: f32 values are three bf16
// planes of 8 bits each, f16 values two, 16-bit values that meet their own type one.
//
// The first product is bound by reading x (prompts) or A (a token for each adapter) once; K is split over the
// waves of a block and over blocks, whose sums the second product adds as it loads t.  The second is bound by reading y
// and writing out.
#include <algorithm>

#include "tq_internal.h"

namespace tq {
namespace {

constexpr int kBlock = 256, kWaves = 4;
constexpr int kMaxRank = 256, kMaxParts = 16, kKUnit = 64;
constexpr int kRowsOutputs = 64;  // of a wave's step where there are many rows
constexpr int64_t kMaxRows = 1 << 30;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// The planes that x of type kX and weights of type kW (TQ_DT_*) meet as; t, which is f32, is kX = TQ_DT_F32.
template <int kX, int kW>
struct Planes {
    static constexpr bool kNative = kX == kW;  // products of 16-bit values of one type are exact in f32
    static constexpr bool kF16 = kNative && kW == TQ_DT_F16;
    static constexpr int kOfX = kNative ? 1 : kX == TQ_DT_F32 ? 3 : kX == TQ_DT_F16 ? 2 : 1;
    static constexpr int kOfW = kNative ? 1 : kW == TQ_DT_F16 ? 2 : 1;
};

template <bool kF16>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (kF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Eight f32 values as kN bf16 planes by cutting 8 bits off at a time: exact for three planes (24 bits), and for
// two where the values have 16 bits (f16 has 11).  Cut and not rounded, so that the largest values stay finite.
template <int kN>
__device__ __forceinline__ void cut8(const float (&v)[8], u32x4 (&out)[kN]) {
    uint32_t rest[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) rest[i] = __float_as_uint(v[i]);
#pragma unroll
    for (int p = 0; p < kN; ++p) {
#pragma unroll
        for (int i = 0; i < 4; ++i) out[p][i] = __builtin_amdgcn_perm(rest[2 * i + 1], rest[2 * i], 0x07060302);
        if (p + 1 < kN) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                rest[i] = __float_as_uint(__uint_as_float(rest[i]) - __uint_as_float(rest[i] & 0xFFFF0000u));
        }
    }
}

template <int kN>
__device__ __forceinline__ void planes_of_16(u32x4 raw, u32x4 (&out)[kN]) {
    if constexpr (kN == 1) {
        out[0] = raw;
    } else {  // f16
        const f16x8 h = __builtin_bit_cast(f16x8, raw);
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(h[i]);
        cut8<kN>(v, out);
    }
}

// Elements k .. k + 7 of a row of x of `n`, zeros from n on (n is not 0).
template <int kX, bool kVec, int kN>
__device__ __forceinline__ void load_x(const void* row, int k, int n, u32x4 (&out)[kN]) {
    if constexpr (kX == TQ_DT_F32) {
        const float* p = static_cast<const float*>(row);
        float v[8];
        if constexpr (kVec) {  // rows 16-byte aligned, n a multiple of 8
            const int at = min(k, n - 8);
            const f32x4 lo = *reinterpret_cast<const f32x4*>(p + at), hi = *reinterpret_cast<const f32x4*>(p + at + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = k < n ? lo[i] : 0.f;
                v[4 + i] = k < n ? hi[i] : 0.f;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = p[min(k + i, n - 1)];
                v[i] = k + i < n ? x : 0.f;
            }
        }
        cut8<kN>(v, out);
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(row);
        u32x4 raw;
        if constexpr (kVec) {
            raw = *reinterpret_cast<const u32x4*>(p + min(k, n - 8));
            if (k >= n) raw = u32x4{0, 0, 0, 0};
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t lo = p[min(k + 2 * i, n - 1)], hi = p[min(k + 2 * i + 1, n - 1)];
                raw[i] = (k + 2 * i < n ? lo : 0) | (k + 2 * i + 1 < n ? hi << 16 : 0);
            }
        }
        planes_of_16<kN>(raw, out);
    }
}

// c + w x by all pairs of planes but those under 2^-24 of the product.
template <bool kF16, int kNW, int kNX>
__device__ __forceinline__ f32x4 products(const u32x4 (&w)[kNW], const u32x4 (&x)[kNX], f32x4 c) {
#pragma unroll
    for (int p = kNW + kNX - 2; p >= 0; --p)
#pragma unroll
        for (int i = 0; i < kNW; ++i)
            if (p - i >= 0 && p - i < kNX && p <= 2) c = mfma<kF16>(w[i], x[p - i], c);
    return c;
}

// The adapters of 16 kT tokens: mine[s] that of token 16 s + lane % 16 (-1: none).  next() names a distinct one
// after the other, in the order of their first tokens; -1 behind the last.
template <int kT>
struct Distinct {
    int mine[kT];
    uint32_t left[kT];
    __device__ __forceinline__ Distinct(const int32_t* index, int count, int first, int m, int lane) {
#pragma unroll
        for (int s = 0; s < kT; ++s) {
            const int tok = first + 16 * s + (lane & 15);
            const int a = tok < m ? index[tok] : -1;
            mine[s] = static_cast<uint32_t>(a) < static_cast<uint32_t>(count) ? a : -1;
        }
        restart();
    }
    __device__ __forceinline__ void restart() {
#pragma unroll
        for (int s = 0; s < kT; ++s) left[s] = static_cast<uint32_t>(__ballot(mine[s] >= 0)) & 0xFFFFu;
    }
    __device__ __forceinline__ int next() {
        int who = -1;
#pragma unroll
        for (int s = kT - 1; s >= 0; --s)
            if (left[s]) who = __builtin_amdgcn_readlane(mine[s], __ffs(left[s]) - 1);
        if (who >= 0) {
#pragma unroll
            for (int s = 0; s < kT; ++s) left[s] &= ~static_cast<uint32_t>(__ballot(mine[s] == who));
        }
        return who;
    }
};

struct AdaptArg {
    const void* x;
    const int32_t* index;
    const uint16_t* a;
    const uint16_t* b;
    const float* scales;
    float* t;  // [splits, m, parts * rank]
    const float* y;
    float* out;
    int m, k, k_row, n, count, parts, rank;
    int splits, k_per;        // K of a block of the first product
    int slots, groups;        // first product: blocks for a tile's distinct adapters, and for its ranks
    int ranges, per, tiles;   // second product: ranges of `per` 16-output tiles, and 16 kT-token tiles
};

// Block (token tile, rank group, slot, split): 16 kT tokens, 16 kR ranks, every slots-th distinct adapter.  The
// waves take 64 of K in turn; a lane holds 16 neighbours of K (two steps of the matrix instruction, whose order of K is
// free), so that a rank's 128 bytes and a token's 128 or 256 are read whole.
template <int kX, int kW, int kT, int kR, bool kVec>
__global__ __launch_bounds__(kBlock) void k_adapt_low(AdaptArg a) {
    typedef Planes<kX, kW> P;
    __shared__ f32x4 part[kWaves][kT * kR][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quad = lane >> 4;
    int id = blockIdx.x;
    const int split = id % a.splits;
    id /= a.splits;
    const int slot = id % a.slots;
    id /= a.slots;
    const int group = id % a.groups, first = id / a.groups * 16 * kT;
    const int ranks = a.parts * a.rank, end = min((split + 1) * a.k_per, a.k_row);
    Distinct<kT> set(a.index, a.count, first, a.m, lane);
    int u = 0;
    for (int who; (who = set.next()) >= 0; ++u) {
        if (u % a.slots != slot) continue;
        const char* xs[kT];
#pragma unroll
        for (int s = 0; s < kT; ++s) {
            // tokens of other adapters read a line that is read anyway
            const uint64_t on = __ballot(set.mine[s] == who) & 0xFFFF;
            const int tok = first + 16 * s + (set.mine[s] == who ? col : on ? __ffsll(static_cast<unsigned long long>(on)) - 1 : 0);
            xs[s] = static_cast<const char*>(a.x) + static_cast<int64_t>(min(tok, a.m - 1)) * a.k * (kX == TQ_DT_F32 ? 4 : 2);
        }
        const uint16_t* ws[kR];
#pragma unroll
        for (int r = 0; r < kR; ++r) {
            const int rank = min((group * kR + r) * 16, ranks - 16) + col;
            ws[r] = a.a + (static_cast<int64_t>(who) * ranks + rank) * a.k_row + 16 * quad;
        }
        f32x4 acc[kT][kR];
#pragma unroll
        for (int s = 0; s < kT; ++s)
#pragma unroll
            for (int r = 0; r < kR; ++r) acc[s][r] = f32x4{0, 0, 0, 0};
        for (int k = split * a.k_per + kKUnit * wave; k < end; k += kKUnit * kWaves) {
            u32x4 raw[kR][2];
#pragma unroll
            for (int r = 0; r < kR; ++r)
#pragma unroll
                for (int h = 0; h < 2; ++h) raw[r][h] = *reinterpret_cast<const u32x4*>(ws[r] + k + 8 * h);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                u32x4 xp[kT][P::kOfX];
#pragma unroll
                for (int s = 0; s < kT; ++s) load_x<kX, kVec>(xs[s], k + 16 * quad + 8 * h, a.k, xp[s]);
#pragma unroll
                for (int r = 0; r < kR; ++r) {
                    u32x4 wp[P::kOfW];
                    planes_of_16(raw[r][h], wp);
#pragma unroll
                    for (int s = 0; s < kT; ++s) acc[s][r] = products<P::kF16>(wp, xp[s], acc[s][r]);
                }
            }
        }
#pragma unroll
        for (int s = 0; s < kT; ++s)
#pragma unroll
            for (int r = 0; r < kR; ++r) part[wave][s * kR + r][lane] = acc[s][r];
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kT * kR; ++j) {
            const int s = j / kR, rank = (group * kR + j % kR) * 16;
            if (j % kWaves != wave || rank >= ranks || set.mine[s] != who) continue;
            const f32x4 v = (part[0][j][lane] + part[1][j][lane]) + (part[2][j][lane] + part[3][j][lane]);
            const int64_t row = static_cast<int64_t>(split) * a.m + first + 16 * s + col;
            *reinterpret_cast<f32x4*>(a.t + row * ranks + rank + 4 * quad) = v;
        }
        __syncthreads();
    }
}

// Planes of s_a t for the 16 kT tokens of a wave: the second operand of the second product, kept in registers.
template <int kW, int kT, int kS>
__device__ __forceinline__ void load_t(const AdaptArg& a, const Distinct<kT>& set, int first, int p,
                                       u32x4 (&tp)[kT][kS][Planes<TQ_DT_F32, kW>::kOfX]) {
    const int col = threadIdx.x & 15, quad = (threadIdx.x & 63) >> 4, ranks = a.parts * a.rank;
#pragma unroll
    for (int s = 0; s < kT; ++s) {
        const int tok = min(first + 16 * s + col, a.m - 1);
        const float scale = set.mine[s] < 0 ? 0.f : a.scales ? a.scales[set.mine[s]] : 1.f;
#pragma unroll
        for (int h = 0; h < kS; ++h) {
            const int rank = 32 * h + 8 * quad;
            f32x4 lo{0, 0, 0, 0}, hi{0, 0, 0, 0};
            if (rank < a.rank && set.mine[s] >= 0) {
                const float* src = a.t + static_cast<int64_t>(tok) * ranks + p * a.rank + rank;
                for (int i = 0; i < a.splits; ++i, src += static_cast<int64_t>(a.m) * ranks) {
                    lo += *reinterpret_cast<const f32x4*>(src);
                    hi += *reinterpret_cast<const f32x4*>(src + 4);
                }
            }
            float v[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = lo[i] * scale;
                v[4 + i] = hi[i] * scale;
            }
            cut8(v, tp[s][h]);
        }
    }
}

// What the wave's lanes wrote to LDS before is there for all of them (LDS serves a wave in order; the compiler has to
// keep that order, too).
__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Ranks of adapter `who` for output `row` of b: the first operand of the second product.
template <int kS>
__device__ __forceinline__ void load_b(const AdaptArg& a, int who, int64_t row, u32x4 (&raw)[kS]) {
    const int quad = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int h = 0; h < kS; ++h) {
        raw[h] = u32x4{0, 0, 0, 0};
        if (who >= 0 && 32 * h + 8 * quad < a.rank)
            raw[h] = *reinterpret_cast<const u32x4*>(a.b + (static_cast<int64_t>(who) * a.n + row) * a.rank + 32 * h + 8 * quad);
    }
}

template <int kW, int kS>
__device__ __forceinline__ f32x4 up_sums(const u32x4 (&raw)[kS], const u32x4 (&tp)[kS][Planes<TQ_DT_F32, kW>::kOfX]) {
    typedef Planes<TQ_DT_F32, kW> P;
    f32x4 v{0, 0, 0, 0};
#pragma unroll
    for (int h = 0; h < kS; ++h) {
        u32x4 wp[P::kOfW];
        planes_of_16(raw[h], wp);
        v = products<false>(wp, tp[h], v);
    }
    return v;
}

// Few rows, and rows that no 16-byte access reaches.  Wave (token tile, part, range of outputs): outputs go by in tiles
// of 16, 4 outputs of a token to a lane; up to kU distinct adapters' weights are loaded together, those of the
// next tile before this one's sums.
template <int kW, int kT, int kS, int kU, bool kVec>
__global__ __launch_bounds__(kBlock) void k_adapt_up(AdaptArg a) {
    const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    int id = blockIdx.x * kWaves + (threadIdx.x >> 6);
    const int tile = id % a.tiles;
    id /= a.tiles;
    const int p = id % a.parts, range = id / a.parts;
    if (range >= a.ranges) return;
    const int first = tile * 16 * kT, np = a.n / a.parts, begin = range * a.per * 16, end = min(begin + a.per * 16, np);
    Distinct<kT> set(a.index, a.count, first, a.m, lane);
    int64_t at[kT];
#pragma unroll
    for (int s = 0; s < kT; ++s)
        at[s] = static_cast<int64_t>(min(first + 16 * s + col, a.m - 1)) * a.n + static_cast<int64_t>(p) * np + 4 * quad;
    auto row_of_b = [&](int n0) { return static_cast<int64_t>(p) * np + min(n0 + col, np - 1); };
    f32x4 y[kT];
    u32x4 raw[kU][kS];
    int names[kU];
    auto load = [&](int n0) {  // the tile's y, and its first kU adapters
#pragma unroll
        for (int s = 0; s < kT; ++s) {
            if constexpr (kVec) {
                y[s] = *reinterpret_cast<const f32x4*>(a.y + at[s] + min(n0, np - 4 - 4 * quad));
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) y[s][i] = a.y[at[s] - 4 * quad + min(n0 + 4 * quad + i, np - 1)];
            }
        }
        set.restart();
#pragma unroll
        for (int i = 0; i < kU; ++i) {
            names[i] = set.next();
            load_b(a, names[i], row_of_b(n0), raw[i]);
        }
    };
    load(begin);
    u32x4 tp[kT][kS][Planes<TQ_DT_F32, kW>::kOfX];
    load_t<kW>(a, set, first, p, tp);
    for (int n0 = begin; n0 < end; n0 += 16) {
        f32x4 d[kT];
#pragma unroll
        for (int s = 0; s < kT; ++s) d[s] = f32x4{-0.f, -0.f, -0.f, -0.f};  // what leaves y as it is
        while (true) {
#pragma unroll
            for (int i = 0; i < kU; ++i) {
                if (names[i] < 0) break;
#pragma unroll
                for (int s = 0; s < kT; ++s) {
                    const bool mine = set.mine[s] == names[i];
                    if (!__ballot(mine)) continue;
                    const f32x4 v = up_sums<kW>(raw[i], tp[s]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) d[s][e] = mine ? v[e] : d[s][e];
                }
            }
            names[0] = set.next();
            if (names[0] < 0) break;
#pragma unroll
            for (int i = 1; i < kU; ++i) names[i] = set.next();
#pragma unroll
            for (int i = 0; i < kU; ++i) load_b(a, names[i], row_of_b(n0), raw[i]);
        }
#pragma unroll
        for (int s = 0; s < kT; ++s) d[s] += y[s];
        if (n0 + 16 < end) load(n0 + 16);
#pragma unroll
        for (int s = 0; s < kT; ++s) {
            if (first + 16 * s + col >= a.m) continue;
            if constexpr (kVec) {
                if (n0 + 4 * quad < np) *reinterpret_cast<f32x4*>(a.out + at[s] + n0) = d[s];
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n0 + 4 * quad + i < np) a.out[at[s] + n0 + i] = d[s][i];
            }
        }
    }
}

// Many rows.  Block (token tile, part, range of outputs), whose waves take 64 outputs each of 256 side by side: 16 kT tokens of a
// wave.  The sums go through LDS (a wave's own part, no barrier) so that y is read and out written in runs of 256 bytes of a
// row: the 64 bytes that a tile of the matrix instruction holds of one took 127 us where this takes 81 (4093 rows of 14336), with
// stores that keep out of the caches (kStream: 106 us without), which then hold y and b.  y is on its way a step ahead.
template <int kW, int kT, int kS, bool kStream>
__global__ __launch_bounds__(kBlock) void k_adapt_up_rows(AdaptArg a) {
    constexpr int kRows = 16 * kT, kY = kRows / 4, kStep = kRowsOutputs * kWaves;
    __shared__ float sums[kWaves][kRows][kRowsOutputs + 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quad = lane >> 4;
    int id = blockIdx.x;
    const int range = id % a.ranges;
    id /= a.ranges;
    const int p = id % a.parts, first = id / a.parts * kRows, np = a.n / a.parts;
    const int begin = range * a.per * kStep, end = min(begin + a.per * kStep, np);
    Distinct<kT> set(a.index, a.count, first, a.m, lane);
    u32x4 tp[kT][kS][Planes<TQ_DT_F32, kW>::kOfX];
    load_t<kW>(a, set, first, p, tp);
    // rows without an adapter: nothing is ever added
#pragma unroll
    for (int i = 0; i < kY; ++i) *reinterpret_cast<f32x4*>(&sums[wave][4 * i + quad][4 * col]) = f32x4{-0.f, -0.f, -0.f, -0.f};
    auto place = [&](int i, int n) { return static_cast<int64_t>(min(first + 4 * i + quad, a.m - 1)) * a.n + static_cast<int64_t>(p) * np + n; };
    auto load_y = [&](int n0, f32x4 (&y)[kY]) {
        const int n = min(n0 + wave * kRowsOutputs + 4 * col, np - 4);
#pragma unroll
        for (int i = 0; i < kY; ++i) y[i] = *reinterpret_cast<const f32x4*>(a.y + place(i, n));
    };
    constexpr int kN = kRowsOutputs / 16;
    u32x4 raw[kN][kS];
    auto weights = [&](int who, int n0) {
#pragma unroll
        for (int j = 0; j < kN; ++j)
            load_b(a, who, static_cast<int64_t>(p) * np + min(n0 + wave * kRowsOutputs + 16 * j + col, np - 1), raw[j]);
    };
    auto multiply = [&](int who) {
#pragma unroll
        for (int s = 0; s < kT; ++s) {
            const bool mine = set.mine[s] == who;
            if (!__ballot(mine)) continue;
#pragma unroll
            for (int j = 0; j < kN; ++j) {
                const f32x4 v = up_sums<kW>(raw[j], tp[s]);
                if (mine) *reinterpret_cast<f32x4*>(&sums[wave][16 * s + col][16 * j + 4 * quad]) = v;
            }
        }
    };
    auto step = [&](int n0, const f32x4 (&now)[kY], f32x4 (&next)[kY]) {
        set.restart();
        int who = set.next();
        weights(who, n0);
        load_y(n0 + kStep, next);
        while (who >= 0) {
            multiply(who);
            if ((who = set.next()) >= 0) weights(who, n0);
        }
        wave_order();
        const int n = n0 + wave * kRowsOutputs + 4 * col;
#pragma unroll
        for (int i = 0; i < kY; ++i) {
            const f32x4 v = now[i] + *reinterpret_cast<const f32x4*>(&sums[wave][4 * i + quad][4 * col]);
            if (first + 4 * i + quad >= a.m || n >= end) continue;
            f32x4* to = reinterpret_cast<f32x4*>(a.out + place(i, n));
            if constexpr (kStream) __builtin_nontemporal_store(v, to);
            else *to = v;
        }
        wave_order();
    };
    f32x4 y[2][kY];
    load_y(begin, y[0]);
    for (int n0 = begin; n0 < end; n0 += 2 * kStep) {
        step(n0, y[0], y[1]);
        if (n0 + kStep < end) step(n0 + kStep, y[1], y[0]);
    }
}

// How a call is cut.
struct Cut {
    bool few;
    int low_tokens, low_ranks, slots, groups, splits, k_per;
};

// Up to this many rows tiles are of 16 tokens and a tile's distinct adapters have blocks of their own.
constexpr int kFewRows = 256;

Cut cut_of(const tq_adapters* a, int64_t m) {
    Cut c;
    const int64_t k_row = (a->k + kKUnit - 1) / kKUnit * kKUnit, rank_tiles = a->parts * a->rank / 16;
    c.few = m <= kFewRows;
    c.low_tokens = c.few ? 16 : 32;
    c.low_ranks = rank_tiles == 1 ? 1 : rank_tiles == 2 ? 2 : 4;
    c.slots = c.few ? static_cast<int>(std::min<int64_t>({16, m, a->count})) : 1;
    c.groups = static_cast<int>((rank_tiles + c.low_ranks - 1) / c.low_ranks);
    const int64_t units = (k_row + kKUnit * kWaves - 1) / (kKUnit * kWaves);
    const int64_t blocks = (m + c.low_tokens - 1) / c.low_tokens * c.slots * c.groups;
    // two blocks for each CU, four where there are many rows (4093 rows, rank 64: 38 us with one, 32 with two, 28 with four)
    const int64_t splits = std::max<int64_t>(1, std::min(units, (c.few ? 2 : 4) * device_cu_count() / std::max<int64_t>(1, blocks)));
    const int64_t per = (units + splits - 1) / splits;
    c.k_per = static_cast<int>(per * kKUnit * kWaves);
    c.splits = static_cast<int>((units + per - 1) / per);
    return c;
}

int check_adapters(const char* what, const tq_adapters* a, int64_t m) {
    TQ_REQUIRE(a, "%s: null adapters", what);
    TQ_REQUIRE(a->dtype == TQ_DT_F16 || a->dtype == TQ_DT_BF16, "%s: adapters are f16 or bf16, not dtype %d", what, a->dtype);
    TQ_REQUIRE(a->count >= 1 && a->count <= 1 << 20, "%s: %lld adapters, 1 to 2^20", what, (long long)a->count);
    TQ_REQUIRE(a->parts >= 1 && a->parts <= kMaxParts, "%s: parts=%lld is not in 1..16", what, (long long)a->parts);
    TQ_REQUIRE(a->rank >= 16 && a->rank <= kMaxRank && a->rank % 16 == 0, "%s: rank=%lld is not a multiple of 16 up to 256", what,
               (long long)a->rank);
    TQ_REQUIRE(a->k >= 1 && a->k <= 1 << 24 && a->n >= 1 && a->n <= 1 << 24 && a->n % a->parts == 0,
               "%s: K=%lld, N=%lld in %lld parts", what, (long long)a->k, (long long)a->n, (long long)a->parts);
    TQ_REQUIRE(a->a && a->b && aligned(a->a, 16) && aligned(a->b, 16) && aligned(a->scales, 4), "%s: null or unaligned weights",
               what);
    TQ_REQUIRE(m >= 0 && m <= kMaxRows, "%s: m=%lld", what, (long long)m);
    return TQ_OK;
}

template <int kX, int kW, int kT, int kR>
void launch_low(const AdaptArg& a, bool vec, int64_t blocks, hipStream_t st) {
    if (vec)
        k_adapt_low<kX, kW, kT, kR, true><<<static_cast<int>(blocks), kBlock, 0, st>>>(a);
    else
        k_adapt_low<kX, kW, kT, kR, false><<<static_cast<int>(blocks), kBlock, 0, st>>>(a);
}

template <int kX, int kW, int kT>
void launch_low_ranks(const AdaptArg& a, int ranks, bool vec, int64_t blocks, hipStream_t st) {
    if (ranks == 1) launch_low<kX, kW, kT, 1>(a, vec, blocks, st);
    else if (ranks == 2) launch_low<kX, kW, kT, 2>(a, vec, blocks, st);
    else launch_low<kX, kW, kT, 4>(a, vec, blocks, st);
}

template <int kX, int kW>
void launch_low_tokens(const AdaptArg& a, const Cut& c, bool vec, int64_t blocks, hipStream_t st) {
    if (c.few) launch_low_ranks<kX, kW, 1>(a, c.low_ranks, vec, blocks, st);
    else launch_low_ranks<kX, kW, 2>(a, c.low_ranks, vec, blocks, st);
}

int64_t blocks_of(const AdaptArg& a, int waves) {
    return (static_cast<int64_t>(a.tiles) * a.parts * a.ranges + waves - 1) / waves;
}

// Tiles of 16 kT tokens, a wave each, ranges so that there are about sixteen waves for each CU.
template <int kW, int kT, int kS, int kU>
int launch_up(AdaptArg a, bool vec, hipStream_t st, const char* what) {
    const int64_t n_tiles = (a.n / a.parts + 15) / 16;
    a.tiles = (a.m + 16 * kT - 1) / (16 * kT);
    const int64_t all = a.tiles * a.parts * n_tiles;
    a.per = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(32, all / (16 * device_cu_count()))));
    a.ranges = static_cast<int>((n_tiles + a.per - 1) / a.per);
    const int64_t blocks = blocks_of(a, kWaves);
    TQ_REQUIRE(blocks <= kMaxBlocks, "%s: %d tokens are more than %lld blocks", what, a.m, (long long)kMaxBlocks);
    if (vec)
        k_adapt_up<kW, kT, kS, kU, true><<<static_cast<int>(blocks), kBlock, 0, st>>>(a);
    else
        k_adapt_up<kW, kT, kS, kU, false><<<static_cast<int>(blocks), kBlock, 0, st>>>(a);
    return check_launch(what);
}

// Blocks of 16 kT tokens; ranges by what the fullest CU gets: its blocks' steps of 16 output tiles, and about 9 tiles'
// time for a block's start (4093 rows of 14336, rank 64: 80, 81 and 86 us with one, two and four blocks for each CU).
template <int kW, int kT, int kS>
int launch_up_rows(AdaptArg a, hipStream_t st, const char* what) {
    const int64_t np = a.n / a.parts, steps = (np + kRowsOutputs * kWaves - 1) / (kRowsOutputs * kWaves);
    a.tiles = (a.m + 16 * kT - 1) / (16 * kT);
    const int64_t every = static_cast<int64_t>(a.tiles) * a.parts, cus = device_cu_count();
    int64_t best = 0;
    for (int64_t r = 1; r <= steps && r <= 64; ++r) {
        const int64_t per = (steps + r - 1) / r, blocks = every * ((steps + per - 1) / per);
        const int64_t cost = (blocks + cus - 1) / cus * (16 * per + 9);
        if (best == 0 || cost < best) {
            best = cost;
            a.per = static_cast<int>(per);
        }
    }
    a.ranges = static_cast<int>((steps + a.per - 1) / a.per);
    const int64_t blocks = blocks_of(a, 1);
    TQ_REQUIRE(blocks <= kMaxBlocks, "%s: %d tokens are more than %lld blocks", what, a.m, (long long)kMaxBlocks);
    // outputs that the L2 caches (4 MB for each XCD) would not hold anyway
    if (static_cast<int64_t>(a.m) * a.n * 4 >= int64_t(32) << 20)
        k_adapt_up_rows<kW, kT, kS, true><<<static_cast<int>(blocks), kBlock, 0, st>>>(a);
    else
        k_adapt_up_rows<kW, kT, kS, false><<<static_cast<int>(blocks), kBlock, 0, st>>>(a);
    return check_launch(what);
}

template <int kW>
int launch_typed(const AdaptArg& a, const Cut& c, int dtype, bool vec_x, bool vec_y, int64_t low, hipStream_t st, const char* what) {
    clear_error();
    if (dtype == TQ_DT_F32) launch_low_tokens<TQ_DT_F32, kW>(a, c, vec_x, low, st);
    else if (dtype == TQ_DT_BF16) launch_low_tokens<TQ_DT_BF16, kW>(a, c, vec_x, low, st);
    else launch_low_tokens<TQ_DT_F16, kW>(a, c, vec_x, low, st);
    const int rc = check_launch(what);
    if (rc != TQ_OK) return rc;
    if (!c.few && vec_y) {
        if (a.rank > 128) return launch_up_rows<kW, 1, 8>(a, st, what);
        if (a.rank > 64) return launch_up_rows<kW, 1, 4>(a, st, what);
        if (a.rank > 32) return launch_up_rows<kW, 2, 2>(a, st, what);
        return launch_up_rows<kW, 2, 1>(a, st, what);
    }
    if (a.rank > 128) return launch_up<kW, 1, 8, 1>(a, vec_y, st, what);
    if (a.rank > 64) return launch_up<kW, 1, 4, 2>(a, vec_y, st, what);
    if (a.rank > 32) return launch_up<kW, 1, 2, 4>(a, vec_y, st, what);
    return launch_up<kW, 1, 1, 4>(a, vec_y, st, what);
}

}  // namespace
}  // namespace tq

extern "C" {

int64_t tq_adapters_workspace_bytes(const tq_adapters* adapters, int64_t m) {
    using namespace tq;
    if (check_adapters("tq_adapters_add", adapters, m) != TQ_OK) return -1;
    return m == 0 ? 0 : cut_of(adapters, m).splits * m * adapters->parts * adapters->rank * 4;
}

int tq_adapters_add(const tq_adapters* adapters, const void* x, int dtype, int64_t m, const int32_t* index, const float* y,
                    float* out, void* workspace, int64_t workspace_bytes, tq_stream_t stream) {
    using namespace tq;
    static const char* what = "tq_adapters_add";
    const int rc = check_adapters(what, adapters, m);
    if (rc != TQ_OK) return rc;
    TQ_REQUIRE(dtype == TQ_DT_F32 || dtype == TQ_DT_BF16 || dtype == TQ_DT_F16, "%s: dtype %d is not f32, bf16 or f16", what, dtype);
    if (m == 0) return TQ_OK;
    const int size = dtype == TQ_DT_F32 ? 4 : 2;
    TQ_REQUIRE(x && index && y && out, "%s: null x, index, y or out", what);
    TQ_REQUIRE(aligned(x, size) && aligned(index, 4) && aligned(y, 4) && aligned(out, 4), "%s: a pointer is not aligned to its elements",
               what);
    const int64_t need = tq_adapters_workspace_bytes(adapters, m);
    TQ_REQUIRE(workspace && workspace_bytes >= need && aligned(workspace, 16), "%s: workspace of %lld bytes, 16-byte aligned, needed",
               what, (long long)need);
    const Cut c = cut_of(adapters, m);
    AdaptArg a{};
    a.x = x;
    a.index = index;
    a.a = static_cast<const uint16_t*>(adapters->a);
    a.b = static_cast<const uint16_t*>(adapters->b);
    a.scales = adapters->scales;
    a.t = static_cast<float*>(workspace);
    a.y = y;
    a.out = out;
    a.m = static_cast<int>(m);
    a.k = static_cast<int>(adapters->k);
    a.k_row = static_cast<int>((adapters->k + kKUnit - 1) / kKUnit * kKUnit);
    a.n = static_cast<int>(adapters->n);
    a.count = static_cast<int>(adapters->count);
    a.parts = static_cast<int>(adapters->parts);
    a.rank = static_cast<int>(adapters->rank);
    a.splits = c.splits;
    a.k_per = c.k_per;
    a.slots = c.slots;
    a.groups = c.groups;
    const int64_t low = (m + c.low_tokens - 1) / c.low_tokens * c.slots * c.groups * c.splits;
    TQ_REQUIRE(low <= kMaxBlocks, "%s: %lld tokens are more than %lld blocks", what, (long long)m, (long long)kMaxBlocks);
    const bool vec_x = aligned(x, 16) && adapters->k % 8 == 0;
    const bool vec_y = aligned(y, 16) && aligned(out, 16) && adapters->n / adapters->parts % 4 == 0;
    return adapters->dtype == TQ_DT_F16 ? launch_typed<TQ_DT_F16>(a, c, dtype, vec_x, vec_y, low, as_hip(stream), what)
                                        : launch_typed<TQ_DT_BF16>(a, c, dtype, vec_x, vec_y, low, as_hip(stream), what);
}

}  // extern "C"
