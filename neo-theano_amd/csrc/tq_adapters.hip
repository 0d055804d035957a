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
// and writing out.  4093 rows of six adapters' runs, rank 64, 4096 to 14336: 24 + 107 us by a trace of the dispatches, the second 4.4 TB/s, where a
// large copy gets 4.7; 64 rows of 48 adapters of rank 16: 5.6 + 10 us; a row alone, both in one launch: 7 us.
#include <algorithm>

#include "tq_internal.h"

namespace tq {
namespace {

constexpr int kBlock = 256, kWaves = 4, kOnceBlock = 512;
constexpr int kMaxRank = 256, kMaxParts = 16, kKUnit = 64;
constexpr int kMaxShares = 8;  // shares of K that the second product adds
constexpr int kStep = 256;  // outputs of a block's step where there are many rows
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

// Eight neighbours of a row of x as they are loaded: f32, or 16-bit values (in both words of `v`, the second unused).
template <int kX>
struct Raw8 {
    f32x4 v[kX == TQ_DT_F32 ? 2 : 1];
};

// Vectors wherever they lie.
typedef f32x4 f32x4_a4 __attribute__((aligned(4)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));

// Elements k .. k + 7 of a row of n > 0; what lies past it is any element of the row, see planes_of.
template <int kX, bool kVec>
__device__ __forceinline__ Raw8<kX> fetch(const void* row, int k, int n) {
    Raw8<kX> r;
    if constexpr (kX == TQ_DT_F32) {
        const float* p = static_cast<const float*>(row);
        if constexpr (kVec) {  // rows 16-byte aligned, n a multiple of 8
            const int at = min(k, n - 8);
            r.v[0] = *reinterpret_cast<const f32x4*>(p + at);
            r.v[1] = *reinterpret_cast<const f32x4*>(p + at + 4);
        } else if (k + 8 <= n) {
            r.v[0] = *reinterpret_cast<const f32x4_a4*>(p + k);
            r.v[1] = *reinterpret_cast<const f32x4_a4*>(p + k + 4);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) r.v[i / 4][i % 4] = p[min(k + i, n - 1)];
        }
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(row);
        if constexpr (kVec) {
            r.v[0] = *reinterpret_cast<const f32x4*>(p + min(k, n - 8));
        } else if (k + 8 <= n) {
            r.v[0] = __builtin_bit_cast(f32x4, static_cast<u32x4>(*reinterpret_cast<const u32x4_a2*>(p + k)));
        } else {
            u32x4 raw;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                raw[i] = p[min(k + 2 * i, n - 1)] | static_cast<uint32_t>(p[min(k + 2 * i + 1, n - 1)]) << 16;
            r.v[0] = __builtin_bit_cast(f32x4, raw);
        }
    }
    return r;
}

// Their planes, zeros for elements from n on.
template <int kX, bool kVec, int kN>
__device__ __forceinline__ void planes_of(const Raw8<kX>& r, int k, int n, u32x4 (&out)[kN]) {
    if constexpr (kX == TQ_DT_F32) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (kVec ? k : k + i) < n ? r.v[i / 4][i % 4] : 0.f;
        cut8<kN>(v, out);
    } else {
        u32x4 raw = __builtin_bit_cast(u32x4, r.v[0]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (kVec) raw[i] = k < n ? raw[i] : 0;
            else raw[i] &= (k + 2 * i < n ? 0xFFFFu : 0) | (k + 2 * i + 1 < n ? 0xFFFF0000u : 0);
        }
        planes_of_16<kN>(raw, out);
    }
}

// c + w x by all pairs of planes, which are the whole product (planes are cut, so a low one may be 2^-7 of what is above it, the
// third 2^-15: of f16 weights and f32 values the lowest pair is up to 2^-22 of the product), the least first.
template <bool kF16, int kNW, int kNX>
__device__ __forceinline__ f32x4 products(const u32x4 (&w)[kNW], const u32x4 (&x)[kNX], f32x4 c) {
#pragma unroll
    for (int p = kNW + kNX - 2; p >= 0; --p)
#pragma unroll
        for (int i = 0; i < kNW; ++i)
            if (p - i >= 0 && p - i < kNX) c = mfma<kF16>(w[i], x[p - i], c);
    return c;
}

// The adapters of 16 kT tokens: mine[s] that of token 16 s + lane % 16 (-1: none).  next() names a distinct one
// after the other, in the order of their first tokens; -1 behind the last.
template <int kT>
struct Distinct {
    int mine[kT];
    uint32_t firsts[kT], left[kT];  // bits of the tokens that are their adapter's first
    __device__ __forceinline__ Distinct(const int32_t* index, int count, int first, int m, int lane) {
        const int col = lane & 15;
#pragma unroll
        for (int s = 0; s < kT; ++s) {
            const int tok = first + 16 * s + col;
            const int a = tok < m ? index[tok] : -1;
            mine[s] = static_cast<uint32_t>(a) < static_cast<uint32_t>(count) ? a : -1;
        }
#pragma unroll
        for (int s = 0; s < kT; ++s) {
            bool again = mine[s] < 0;
#pragma unroll
            for (int t = 0; t <= s; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) again |= (t < s || i < col) && mine[s] == readlane(mine[t], i);
            firsts[s] = static_cast<uint32_t>(__ballot(!again)) & 0xFFFFu;
        }
        restart();
    }
    __device__ __forceinline__ void restart() {
#pragma unroll
        for (int s = 0; s < kT; ++s) left[s] = firsts[s];
    }
    __device__ __forceinline__ int all() const {
        int n = 0;
#pragma unroll
        for (int s = 0; s < kT; ++s) n += __popc(firsts[s]);
        return n;
    }
    __device__ __forceinline__ int next() {
        int who = -1;
        bool done = false;
#pragma unroll
        for (int s = 0; s < kT; ++s) {
            const bool here = !done && left[s] != 0;
            if (here) {
                who = readlane(mine[s], __ffs(left[s]) - 1);
                left[s] &= left[s] - 1;
            }
            done |= here;
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
    int32_t* shares;  // of K, [low tiles]
    float* t;         // [shares, m, parts * rank]
    const float* y;
    float* out;
    int m, k, k_row, n, np, count, parts, rank;  // np: outputs of a part
    int low_shift, gang_shift, turns;            // first product: tiles of 1 << low_shift tokens, 1 << gang_shift blocks for each, k_row
                                                 // in turns of a block's waves
    int per;                                     // second product: turns (steps) of a block
};

// Adds to acc the products of 16 kT tokens from `first` on with 16 kR ranks of adapter `who` from rank0 on (ranks past the last: the
// last 16 again), over every step-th 64 columns from k to `end`.  A load takes a tile of 16 ranks x 32 columns, 1 KB in one run (of
// rows 8 KB apart a block got 20 GB/s), and 64 or 128 bytes of a token.  kAtOnce 1: the next 64 columns are on their way while these are multiplied; more: so many are loaded together
// (for a block with little to do beside it).
template <int kX, int kW, int kT, int kR, bool kVec, int kAtOnce>
__device__ __forceinline__ void low_products(const AdaptArg& a, const Distinct<kT>& set, int who, int first, int rank0, int k, int end, int step,
                                             f32x4 (&acc)[kT][kR]) {
    typedef Planes<kX, kW> P;
    const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4, ranks = a.parts * a.rank;
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
        const int rank = min(rank0 + 16 * r, ranks - 16);
        ws[r] = a.a + (static_cast<int64_t>(who) * ranks + rank) * a.k_row + 32 * col + 8 * quad;
    }
    struct Loads {
        Raw8<kX> x[kT][2];
        u32x4 w[kR][2];
    };
    auto load = [&](int k) {
        Loads l;
        k = min(k, a.k_row - kKUnit);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int r = 0; r < kR; ++r) l.w[r][h] = *reinterpret_cast<const u32x4*>(ws[r] + 16 * k + 512 * h);
#pragma unroll
            for (int s = 0; s < kT; ++s) l.x[s][h] = fetch<kX, kVec>(xs[s], k + 32 * h + 8 * quad, a.k);
        }
        return l;
    };
    auto multiply = [&](int k, const Loads& l) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            u32x4 xp[kT][P::kOfX];
#pragma unroll
            for (int s = 0; s < kT; ++s) planes_of<kX, kVec>(l.x[s][h], k + 32 * h + 8 * quad, a.k, xp[s]);
#pragma unroll
            for (int r = 0; r < kR; ++r) {
                u32x4 wp[P::kOfW];
                planes_of_16(l.w[r][h], wp);
#pragma unroll
                for (int s = 0; s < kT; ++s) acc[s][r] = products<P::kF16>(wp, xp[s], acc[s][r]);
            }
        }
    };
    if constexpr (kAtOnce > 1) {
        for (; k < end; k += step * kAtOnce) {
            Loads some[kAtOnce];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) some[i] = load(k + i * step);
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
                if (k + i * step < end) multiply(k + i * step, some[i]);
        }
        return;
    }
    if (k >= end) return;
    Loads now = load(k);
    for (; k + step < end; k += step) {
        const Loads next = load(k + step);
        multiply(k, now);
        now = next;
    }
    multiply(k, now);
}

// Grid (token tile and one of its gang, rank group): 16 kT tokens, 16 kR ranks.  The tile's distinct adapters, which only the
// device knows, and as many shares of K as then keep the gang busy are its blocks' units of work.  The waves take
// 64 of K in turn.
template <int kX, int kW, int kT, int kR, bool kVec>
__global__ __launch_bounds__(kBlock) void k_adapt_low(AdaptArg a) {
    __shared__ f32x4 part[kWaves][kT * kR][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quad = lane >> 4;
    // a gang's blocks are neighbours: they read neighbouring columns of the same rows
    const int gang = 1 << a.gang_shift, tile = blockIdx.x >> a.gang_shift, mate = blockIdx.x & (gang - 1), group = blockIdx.y;
    const int first = tile * 16 * kT, ranks = a.parts * a.rank;
    Distinct<kT> set(a.index, a.count, first, a.m, lane);
    const int adapters = set.all();
    int bits = 0;  // the shares of K are a power of two
    while (2 << bits <= min(kMaxShares, a.turns) && adapters << (bits + 1) <= gang) ++bits;
    const int per = (a.turns + (1 << bits) - 1) >> bits;
    if (mate == 0 && group == 0 && threadIdx.x == 0) a.shares[tile] = 1 << bits;
    int who = -1, named = 0;  // the adapter that next() gave `named`-th
    for (int unit = mate; unit < adapters << bits; unit += gang) {
        const int share = unit & ((1 << bits) - 1), k_begin = min(share * per, a.turns) * kKUnit * kWaves,
                  end = min(k_begin + per * kKUnit * kWaves, a.k_row);
        for (; named <= unit >> bits; ++named) who = set.next();
        f32x4 acc[kT][kR] = {};
        low_products<kX, kW, kT, kR, kVec, 1>(a, set, who, first, group * kR * 16, k_begin + kKUnit * wave, end, kKUnit * kWaves, acc);
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
            const int64_t row = static_cast<int64_t>(share) * a.m + first + 16 * s + col;
            *reinterpret_cast<f32x4*>(a.t + row * ranks + rank + 4 * quad) = v;
        }
        __syncthreads();
    }
}

// s_a t of kRows tokens from `first` on, part p's ranks, summed over the shares of K once for the block: lds[token][rank].
template <int kRows, int kS, int kRow>
__device__ __forceinline__ void sum_t(const AdaptArg& a, int first, int p, float (&lds)[kRows][kRow]) {
    const int64_t ranks = a.parts * a.rank;
#pragma unroll
    for (int i = threadIdx.x; i < kRows * 8 * kS; i += kBlock) {
        const int row = i / (8 * kS), rank = 4 * (i % (8 * kS)), tok = first + row;
        if (rank >= a.rank) continue;
        const int who = tok < a.m ? a.index[tok] : -1;
        f32x4 v{0, 0, 0, 0};
        if (static_cast<uint32_t>(who) < static_cast<uint32_t>(a.count)) {
            const float* src = a.t + tok * ranks + p * a.rank + rank;
            const float scale = a.scales ? a.scales[who] : 1.f;
            const int shares = a.shares[tok >> a.low_shift];
            f32x4 x[kMaxShares];  // all on their way at once; those past the last are the first again, and left out
#pragma unroll
            for (int k = 0; k < kMaxShares; ++k)
                x[k] = *reinterpret_cast<const f32x4*>(src + (k < shares ? static_cast<int64_t>(k) * a.m * ranks : 0));
#pragma unroll
            for (int k = 0; k < kMaxShares; ++k)
                if (k < shares) v += x[k];
            v *= scale;
        }
        *reinterpret_cast<f32x4*>(&lds[row][rank]) = v;
    }
}

// Planes of it for the 16 kT tokens of a wave: the second operand of the second product, kept in registers.
template <int kT, int kS, int kRow, int kN>
__device__ __forceinline__ void planes_of_t(const AdaptArg& a, const float (&lds)[16 * kT][kRow], u32x4 (&tp)[kT][kS][kN]) {
    const int col = threadIdx.x & 15, quad = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int s = 0; s < kT; ++s)
#pragma unroll
        for (int h = 0; h < kS; ++h) {
            const int rank = 32 * h + 8 * quad;
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = rank < a.rank ? lds[16 * s + col][rank + i] : 0.f;
            cut8(v, tp[s][h]);
        }
}

// Ranks of adapter `who` for output `row` of b: the first operand of the second product.  Lanes behind the last rank
// take other ranks of the row, which meet zeros of t.
template <int kS>
__device__ __forceinline__ void load_b(const AdaptArg& a, int who, int64_t row, u32x4 (&raw)[kS]) {
    const int quad = (threadIdx.x & 63) >> 4;
    const uint16_t* from = a.b + (static_cast<int64_t>(who) * a.n + row) * a.rank;
#pragma unroll
    for (int h = 0; h < kS; ++h) raw[h] = *reinterpret_cast<const u32x4*>(from + min(32 * h + 8 * quad, a.rank - 8));
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

// Tiles of 16 outputs of part p for the 16 tokens from `first` on, 4 outputs of a token to a lane: up to kU distinct adapters'
// weights are loaded together, those of the next tile before this one's sums.
template <int kW, int kS, int kU, bool kVec>
struct UpTiles {
    const AdaptArg& a;
    Distinct<1> set;
    const int64_t at;  // y and out
    const int first, p;
    f32x4 y;
    u32x4 raw[kU][kS];
    int names[kU];

    __device__ __forceinline__ UpTiles(const AdaptArg& arg, const Distinct<1>& tokens, int first_token, int part)
        : a(arg), set(tokens), at(static_cast<int64_t>(min(first_token + col(), arg.m - 1)) * arg.n + static_cast<int64_t>(part) * arg.np + 4 * quad()),
          first(first_token), p(part) {}
    static __device__ __forceinline__ int col() { return threadIdx.x & 15; }
    static __device__ __forceinline__ int quad() { return (threadIdx.x & 63) >> 4; }

    __device__ __forceinline__ void weights(int n0) {  // of the next kU adapters
#pragma unroll
        for (int i = 0; i < kU; ++i) {
            names[i] = set.next();
            if (names[i] >= 0) load_b(a, names[i], static_cast<int64_t>(p) * a.np + min(n0 + col(), a.np - 1), raw[i]);
        }
    }
    __device__ __forceinline__ void load(int n0) {
        if constexpr (kVec) {
            y = *reinterpret_cast<const f32x4*>(a.y + at + min(n0, a.np - 4 - 4 * quad()));
        } else if (n0 + 4 * quad() + 4 <= a.np) {
            y = *reinterpret_cast<const f32x4_a4*>(a.y + at + n0);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = a.y[at - 4 * quad() + min(n0 + 4 * quad() + i, a.np - 1)];
        }
        set.restart();
        weights(n0);
    }
    // The tiles from `begin`, which load() has, to `end`, every turn-th output.
    __device__ __forceinline__ void run(int begin, int end, int turn, const u32x4 (&tp)[kS][Planes<TQ_DT_F32, kW>::kOfX]) {
        for (int n0 = begin; n0 < end; n0 += turn) {
            f32x4 d{-0.f, -0.f, -0.f, -0.f};  // what leaves y as it is
            while (names[0] >= 0) {
#pragma unroll
                for (int i = 0; i < kU; ++i) {
                    if (names[i] < 0) break;
                    const f32x4 v = up_sums<kW>(raw[i], tp);
#pragma unroll
                    for (int e = 0; e < 4; ++e) d[e] = set.mine[0] == names[i] ? v[e] : d[e];
                }
                weights(n0);
            }
            d += y;
            if (n0 + turn < end) load(n0 + turn);
            if (first + col() >= a.m) continue;
            if constexpr (kVec) {
                if (n0 + 4 * quad() < a.np) *reinterpret_cast<f32x4*>(a.out + at + n0) = d;
            } else if (n0 + 4 * quad() + 4 <= a.np) {
                *reinterpret_cast<f32x4_a4*>(a.out + at + n0) = d;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n0 + 4 * quad() + i < a.np) a.out[at + n0 + i] = d[i];
            }
        }
    }
};

// Few rows, and rows that no 16-byte access reaches.  Grid (token tile, part, range of outputs): a block's waves take tiles of 16
// outputs in turn.
template <int kW, int kS, int kU, bool kVec>
__global__ __launch_bounds__(kBlock) void k_adapt_up(AdaptArg a) {
    __shared__ float t[16][32 * kS + 4];
    const int wave = threadIdx.x >> 6, p = blockIdx.y, first = blockIdx.x * 16, from = blockIdx.z * a.per * kWaves * 16;
    const int begin = from + 16 * wave, end = min(from + a.per * kWaves * 16, a.np);
    UpTiles<kW, kS, kU, kVec> tiles(a, Distinct<1>(a.index, a.count, first, a.m, threadIdx.x & 63), first, p);
    tiles.load(begin < end ? begin : from);  // (a wave may have no tile: the block's first)
    sum_t<16, kS>(a, first, p, t);
    __syncthreads();
    u32x4 tp[1][kS][Planes<TQ_DT_F32, kW>::kOfX];
    planes_of_t(a, t, tp);
    tiles.run(begin, end, 16 * kWaves, tp[0]);
}

// A token or a few, of few adapters and low ranks: both products in one launch, without a workspace.  Grid (range of outputs, part): every block
// forms t of its part by itself, its waves 64 columns of K in turn, and then its outputs.  For the GPU that is about what
// two launches are, for the host a launch and a buffer less; figures at in_one_launch.
template <int kX, int kW, int kR, bool kVecX, bool kVecY>
__global__ __launch_bounds__(kOnceBlock) void k_adapt_once(AdaptArg a) {
    constexpr int kOnceWaves = kOnceBlock / 64;
    __shared__ f32x4 part[kOnceWaves][kR][64];
    __shared__ float t[16][32 + 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quad = lane >> 4, p = blockIdx.y;
    const int from = blockIdx.x * kOnceWaves * 16, begin = from + 16 * wave, end = min(from + kOnceWaves * 16, a.np);
    Distinct<1> set(a.index, a.count, 0, a.m, lane);
    UpTiles<kW, 1, 4, kVecY> tiles(a, set, 0, p);
    tiles.load(begin < end ? begin : from);
    for (int who; (who = set.next()) >= 0;) {
        f32x4 acc[1][kR] = {};
        low_products<kX, kW, 1, kR, kVecX, kR == 1 ? 4 : 2>(a, set, who, 0, p * a.rank, kKUnit * wave, a.k_row, kKUnit * kOnceWaves, acc);
#pragma unroll
        for (int r = 0; r < kR; ++r) part[wave][r][lane] = acc[0][r];
        __syncthreads();
        if (wave < kR && set.mine[0] == who) {
            f32x4 v = part[0][wave][lane];
#pragma unroll
            for (int w = 1; w < kOnceWaves; ++w) v += part[w][wave][lane];
            *reinterpret_cast<f32x4*>(&t[col][16 * wave + 4 * quad]) = v * (a.scales ? a.scales[who] : 1.f);
        }
        __syncthreads();
    }
    u32x4 tp[1][1][Planes<TQ_DT_F32, kW>::kOfX];
    planes_of_t(a, t, tp);  // (of tokens without an adapter: anything, and left out)
    tiles.run(begin, end, kOnceWaves * 16, tp[0]);
}

// Many rows.  Grid (range of outputs, part, token tile): 16 kT tokens and 256 outputs a step, 64 for each wave.  The
// sums go through LDS, so that y is read and out written in runs of 1 KB of a row: both products of 4093 rows, rank 64, 4096 to
// 14336, replayed: 126 us, 190 with k_adapt_up, which touches 64 bytes of a row at a time.  kStream: loads and stores that are not kept in the
// caches, which b needs (134 us without).
template <int kW, int kT, int kS, bool kStream>
__global__ __launch_bounds__(kBlock) void k_adapt_up_rows(AdaptArg a) {
    constexpr int kRows = 16 * kT, kY = kRows / kWaves, kN = kStep / 16 / kWaves;
    __shared__ float sums[kRows][kStep + 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quad = lane >> 4;
    const int range = blockIdx.x, p = blockIdx.y, first = blockIdx.z * kRows, np = a.np;
    const int begin = range * a.per * kStep, end = min(begin + a.per * kStep, np);
    Distinct<kT> set(a.index, a.count, first, a.m, lane);
    sum_t<kRows, kS>(a, first, p, sums);
    __syncthreads();
    u32x4 tp[kT][kS][Planes<TQ_DT_F32, kW>::kOfX];
    planes_of_t(a, sums, tp);
    __syncthreads();
    // rows without an adapter: nothing is ever added
#pragma unroll
    for (int i = 0; i < kY; ++i) *reinterpret_cast<f32x4*>(&sums[kWaves * i + wave][4 * lane]) = f32x4{-0.f, -0.f, -0.f, -0.f};
    __syncthreads();
    const int64_t at = static_cast<int64_t>(first + wave) * a.n + static_cast<int64_t>(p) * np;
    for (int n0 = begin; n0 < end; n0 += kStep) {
        const int n = n0 + 4 * lane;
        f32x4 y[kY];
        auto weights = [&](int who, u32x4 (&raw)[kN][kS]) {
#pragma unroll
            for (int j = 0; j < kN; ++j)
                load_b(a, who, static_cast<int64_t>(p) * np + min(n0 + (wave * kN + j) * 16 + col, np - 1), raw[j]);
        };
        auto multiply = [&](int who, const u32x4 (&raw)[kN][kS]) {
#pragma unroll
            for (int s = 0; s < kT; ++s) {
                const bool mine = set.mine[s] == who;
                if (!__ballot(mine)) continue;
#pragma unroll
                for (int j = 0; j < kN; ++j) {
                    const f32x4 v = up_sums<kW>(raw[j], tp[s]);
                    if (mine) *reinterpret_cast<f32x4*>(&sums[16 * s + col][(wave * kN + j) * 16 + 4 * quad]) = v;
                }
            }
        };
        set.restart();
        u32x4 raw[2][kN][kS];
        int who = set.next();
        if (who >= 0) weights(who, raw[0]);  // before y: loads come back in order, and the sums wait for these alone
#pragma unroll
        for (int i = 0; i < kY; ++i) {
            const int64_t row = min(first + wave + kWaves * i, a.m - 1);
            const f32x4* from = reinterpret_cast<const f32x4*>(a.y + row * a.n + static_cast<int64_t>(p) * np + min(n, np - 4));
            y[i] = kStream ? __builtin_nontemporal_load(from) : *from;
        }
        while (who >= 0) {  // the next adapter's weights are on their way while these are multiplied
            const int then = set.next();
            if (then >= 0) weights(then, raw[1]);
            multiply(who, raw[0]);
            if (then < 0) break;
            if ((who = set.next()) >= 0) weights(who, raw[0]);
            multiply(then, raw[1]);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kY; ++i) {
            if (first + wave + kWaves * i >= a.m || n >= end) continue;
            const f32x4 v = y[i] + *reinterpret_cast<const f32x4*>(&sums[kWaves * i + wave][4 * lane]);
            f32x4* to = reinterpret_cast<f32x4*>(a.out + at + static_cast<int64_t>(kWaves) * i * a.n + n);
            if constexpr (kStream) __builtin_nontemporal_store(v, to);
            else *to = v;
        }
        __syncthreads();
    }
}

// Eight elements of a tile a lane: a [groups, rank, K] to tiles of 16 x 32, zeros past rank and K.
__global__ __launch_bounds__(kBlock) void k_tile(const uint16_t* a, int64_t units, int rank, int k, int rank_tiles, int k_tiles, u32x4* out) {
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; u < units; u += static_cast<int64_t>(gridDim.x) * kBlock) {
        const int64_t tile = u / 64, row_tile = tile / k_tiles, group = row_tile / rank_tiles;
        const int r = static_cast<int>(row_tile - group * rank_tiles) * 16 + (u % 64) / 4,
                  k0 = static_cast<int>(tile - row_tile * k_tiles) * 32 + (u % 4) * 8;
        u32x4 v{};
        if (r < rank) {
            const uint16_t* row = a + (group * rank + r) * k;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (k0 + i < k) v[i / 2] |= static_cast<uint32_t>(row[k0 + i]) << (16 * (i & 1));
        }
        out[u] = v;
    }
}

// How the first product is cut.
struct Cut {
    bool few;
    int tokens, ranks, gang_shift, groups;
    int64_t tiles;
};

// The first product's tiles are of 16 tokens, or of 32 where it is long: from 3 2^28 products on (rows x ranks x K; f32, six
// adapters' runs, 16 / 32: 4096 rows, rank 64, K 1408 20.1 / 28.3 us, rank 48, K 4096 29.0 / 28.9, rank 192, K 4096 86 / 69; 1024 rows,
// rank 192, K 4096 31.8 / 29.4; 512 rows, rank 192, K 12288 41 / 44; 2048 rows, rank 256, K 12288 197 / 136), and more than 256 rows.
constexpr int64_t kLong = int64_t(3) << 28;
constexpr int kFewRows = 256;

Cut cut_of(const tq_adapters* a, int64_t m) {
    Cut c;
    const int64_t turns = (a->k + kKUnit * kWaves - 1) / (kKUnit * kWaves), rank_tiles = a->parts * a->rank / 16;
    c.few = m <= kFewRows || m < kLong / (a->parts * a->rank * a->k);
    c.tokens = c.few ? 16 : 32;
    c.ranks = rank_tiles == 1 ? 1 : rank_tiles == 2 ? 2 : 4;
    c.groups = static_cast<int>((rank_tiles + c.ranks - 1) / c.ranks);
    c.tiles = (m + c.tokens - 1) / c.tokens;
    // about four blocks for each CU (the first product of 4093 rows, rank 64, before its weights lay in tiles: 38 us with one, 32 with two,
    // 28 with four),
    // no more than a tile can have adapters and shares
    const int64_t blocks = c.tiles * c.groups;
    const int64_t gang = std::min<int64_t>(4 * device_cu_count() / blocks,
                                           std::min<int64_t>({c.tokens, m, a->count}) * std::min<int64_t>(turns, kMaxShares));
    c.gang_shift = 0;
    while (int64_t(2) << c.gang_shift <= gang) ++c.gang_shift;
    return c;
}

// Workspace: the shares of each tile, then t of as many shares of K as a gang can take.
int64_t shares_bytes(const Cut& c) { return (c.tiles * 4 + 15) / 16 * 16; }
int64_t most_shares(const Cut& c) { return std::min<int64_t>(kMaxShares, int64_t(1) << c.gang_shift); }

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
void launch_low(const AdaptArg& a, bool vec, dim3 grid, hipStream_t st) {
    if (vec)
        k_adapt_low<kX, kW, kT, kR, true><<<grid, kBlock, 0, st>>>(a);
    else
        k_adapt_low<kX, kW, kT, kR, false><<<grid, kBlock, 0, st>>>(a);
}

template <int kX, int kW, int kT>
void launch_low_ranks(const AdaptArg& a, int ranks, bool vec, dim3 grid, hipStream_t st) {
    if (ranks == 1) launch_low<kX, kW, kT, 1>(a, vec, grid, st);
    else if (ranks == 2) launch_low<kX, kW, kT, 2>(a, vec, grid, st);
    else launch_low<kX, kW, kT, 4>(a, vec, grid, st);
}

template <int kX, int kW>
void launch_low_tokens(const AdaptArg& a, const Cut& c, bool vec, dim3 grid, hipStream_t st) {
    if (c.few) launch_low_ranks<kX, kW, 1>(a, c.ranks, vec, grid, st);
    else launch_low_ranks<kX, kW, 2>(a, c.ranks, vec, grid, st);
}

// Tiles of 16 tokens, ranges so that there are about four blocks for each CU.
template <int kW, int kS, int kU>
int launch_up(AdaptArg a, bool vec, hipStream_t st, const char* what) {
    const int64_t turns = (a.np + 16 * kWaves - 1) / (16 * kWaves), tiles = (a.m + 15) / 16;
    a.per = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(8, tiles * a.parts * turns / (4 * device_cu_count()))));
    const int64_t ranges = (turns + a.per - 1) / a.per;
    // (N is at most 2^24: up to 32768 ranges)
    const dim3 blocks(static_cast<uint32_t>(tiles), static_cast<uint32_t>(a.parts), static_cast<uint32_t>(ranges));
    if (vec)
        k_adapt_up<kW, kS, kU, true><<<blocks, kBlock, 0, st>>>(a);
    else
        k_adapt_up<kW, kS, kU, false><<<blocks, kBlock, 0, st>>>(a);
    return check_launch(what);
}

// Blocks of 16 kT tokens; ranges by what the fullest CU gets: its blocks' steps, and about one step's time for a block's
// start; a block that is alone on its CU waits for its own loads (both products, rank 64, replayed: 4093 rows, 4096 to 14336, 152, 126, 126, 139 and 131 us
// with 1, 2, 4, 7 and 14 blocks for each CU; 512 rows 30 and 24 with 1 and 2).  Of ranges that cost the same the shorter ones.
template <int kW, int kT, int kS>
int launch_up_rows(AdaptArg a, hipStream_t st, const char* what) {
    const int64_t steps = (a.np + kStep - 1) / kStep, tiles = (a.m + 16 * kT - 1) / (16 * kT), cus = device_cu_count();
    int64_t best = 0;
    for (int64_t r = 1; r <= steps && r <= 64; ++r) {
        const int64_t per = (steps + r - 1) / r, on_one = (tiles * a.parts * ((steps + per - 1) / per) + cus - 1) / cus;
        const int64_t cost = on_one * (per + 1) * (on_one == 1 ? 8 : 5);
        if (best == 0 || cost <= best) {
            best = cost;
            a.per = static_cast<int>(per);
        }
    }
    const dim3 blocks(static_cast<uint32_t>((steps + a.per - 1) / a.per), static_cast<uint32_t>(a.parts), static_cast<uint32_t>(tiles));
    // outputs that the L2 caches (4 MB for each XCD) would not hold anyway
    if (static_cast<int64_t>(a.m) * a.n * 4 >= int64_t(32) << 20)
        k_adapt_up_rows<kW, kT, kS, true><<<blocks, kBlock, 0, st>>>(a);
    else
        k_adapt_up_rows<kW, kT, kS, false><<<blocks, kBlock, 0, st>>>(a);
    return check_launch(what);
}

// Calls of one launch.  In it a block takes the adapters that its rows name one after the other, each with its own loads, sums over the
// waves and barriers, so it is for few of them (the host knows how many there can be, not how many there are) and short products.
// A call / replayed, us, rank 16, 4096 outputs, one launch against two:
//   x bf16  1 row, K 4096 6.8 / 6.5, 9.6 / 7.2; K 5120 7.9 / 7.7, 9.7 / 7.4; 2 adapters, K 1024 7.5 / 7.3, 9.6 / 7.0;
//           4, K 256 7.9 / 7.7, 9.6 / 7.2; 4, K 512 9.6 / 9.4, 9.6 / 7.2; 4, K 1024 11.1 / 11.0, 9.6 / 7.3;
//           8, K 128 10.4 / 10.2, 9.6 / 8.0; 16, K 256 20.4 / 20.3, 10.0 / 9.7
//   x f32   1 row, K 4096 8.2 / 8.0, 9.6 / 7.4; K 5120 9.8 / 9.6, 9.7 / 7.7; 2, K 1024 8.8 / 8.6, 9.6 / 7.2;
//           2, K 2048 9.4 / 9.2, 9.8 / 7.3; 4, K 256 8.9 / 8.7, 9.5 / 7.5; 16, K 256 23.2 / 23.1, 10.2 / 9.9
// (x f16 and f16 weights 6.8 / 6.6, 9.5 / 7.3 at K 4096; f32 rows of f16 weights, twice the matrix instructions, 10.2 / 10.0, 9.5 / 7.8.)
constexpr int64_t kOnceWeights = 1 << 16;  // rows x ranks x K
constexpr int64_t kOnceAdapters = 4;
bool in_one_launch(const tq_adapters* a, int64_t m) {
    const int64_t named = std::min(m, a->count);
    return m <= 16 && a->rank <= 32 && named <= kOnceAdapters && std::max(m, named * named) * a->rank * a->k <= kOnceWeights;
}

template <int kX, int kW, int kR>
void launch_once_vec(const AdaptArg& a, bool vec_x, bool vec_y, dim3 blocks, hipStream_t st) {
    if (vec_x && vec_y) k_adapt_once<kX, kW, kR, true, true><<<blocks, kOnceBlock, 0, st>>>(a);
    else if (vec_x) k_adapt_once<kX, kW, kR, true, false><<<blocks, kOnceBlock, 0, st>>>(a);
    else if (vec_y) k_adapt_once<kX, kW, kR, false, true><<<blocks, kOnceBlock, 0, st>>>(a);
    else k_adapt_once<kX, kW, kR, false, false><<<blocks, kOnceBlock, 0, st>>>(a);
}

template <int kW>
int launch_once(const AdaptArg& a, int dtype, bool vec_x, bool vec_y, hipStream_t st, const char* what) {
    const dim3 blocks(static_cast<uint32_t>((a.np + kOnceBlock / 4 - 1) / (kOnceBlock / 4)), static_cast<uint32_t>(a.parts));
    clear_error();
    if (a.rank == 16) {
        if (dtype == TQ_DT_F32) launch_once_vec<TQ_DT_F32, kW, 1>(a, vec_x, vec_y, blocks, st);
        else if (dtype == TQ_DT_BF16) launch_once_vec<TQ_DT_BF16, kW, 1>(a, vec_x, vec_y, blocks, st);
        else launch_once_vec<TQ_DT_F16, kW, 1>(a, vec_x, vec_y, blocks, st);
    } else {
        if (dtype == TQ_DT_F32) launch_once_vec<TQ_DT_F32, kW, 2>(a, vec_x, vec_y, blocks, st);
        else if (dtype == TQ_DT_BF16) launch_once_vec<TQ_DT_BF16, kW, 2>(a, vec_x, vec_y, blocks, st);
        else launch_once_vec<TQ_DT_F16, kW, 2>(a, vec_x, vec_y, blocks, st);
    }
    return check_launch(what);
}

template <int kW>
int launch_typed(const AdaptArg& a, const Cut& c, int dtype, bool vec_x, bool vec_y, dim3 low, hipStream_t st, const char* what) {
    clear_error();
    if (dtype == TQ_DT_F32) launch_low_tokens<TQ_DT_F32, kW>(a, c, vec_x, low, st);
    else if (dtype == TQ_DT_BF16) launch_low_tokens<TQ_DT_BF16, kW>(a, c, vec_x, low, st);
    else launch_low_tokens<TQ_DT_F16, kW>(a, c, vec_x, low, st);
    const int rc = check_launch(what);
    if (rc != TQ_OK) return rc;
    // the form of many rows where the outputs leave the caches (rank 16, direct / rows, us: 1536 x 6144 23.2 / 26.2, 2560 x 6144 45.1 / 34.3;
    // rank 32: 1536 x 8192 27.7 / 26.9, 1024 x 14336 43.6 / 32.9), with more ranks from 3 2^19 outputs (rank 64: 256 x 4096 13.1 / 14.4,
    // 128 x 14336 18.3 / 16.5, 512 x 8192 21.9 / 18.3) or 3 2^18 on (rank 128: 128 x 4096 13.6 / 15.3, 64 x 14336 21.2 / 17.4); six runs of
    // rows, K 512, both products
    const int64_t many = a.rank > 64 ? 3 << 18 : a.rank > 32 ? 3 << 19 : 12 << 20;
    if (vec_y && static_cast<int64_t>(a.m) * a.n >= many && a.m <= 16 * 65535) {
        if (a.rank > 128) return launch_up_rows<kW, 1, 8>(a, st, what);
        if (a.rank > 64) return launch_up_rows<kW, 1, 4>(a, st, what);
        if (a.rank > 32) return launch_up_rows<kW, 2, 2>(a, st, what);
        return launch_up_rows<kW, 2, 1>(a, st, what);
    }
    if (a.rank > 128) return launch_up<kW, 8, 2>(a, vec_y, st, what);
    if (a.rank > 64) return launch_up<kW, 4, 4>(a, vec_y, st, what);
    if (a.rank > 32) return launch_up<kW, 2, 4>(a, vec_y, st, what);
    return launch_up<kW, 1, 4>(a, vec_y, st, what);
}

}  // namespace
}  // namespace tq

extern "C" {

int tq_repack_adapters_tiled(const void* a, int64_t groups, int64_t rank, int64_t k, void* tiled, tq_stream_t stream) {
    using namespace tq;
    static const char* what = "tq_repack_adapters_tiled";
    TQ_REQUIRE(groups >= 0 && groups <= int64_t(16) << 20 && rank >= 1 && rank <= kMaxRank && k >= 1 && k <= 1 << 24,
               "%s: %lld groups, rank=%lld, K=%lld", what, (long long)groups, (long long)rank, (long long)k);
    if (groups == 0) return TQ_OK;
    TQ_REQUIRE(a && tiled && aligned(a, 2) && aligned(tiled, 16), "%s: null or unaligned pointer", what);
    const int64_t rank_tiles = (rank + 15) / 16, k_tiles = (k + kKUnit - 1) / kKUnit * 2, units = groups * rank_tiles * k_tiles * 64;
    clear_error();
    k_tile<<<static_cast<int>(std::min<int64_t>((units + kBlock - 1) / kBlock, 16 * device_cu_count())), kBlock, 0, as_hip(stream)>>>(
        static_cast<const uint16_t*>(a), units, static_cast<int>(rank), static_cast<int>(k), static_cast<int>(rank_tiles),
        static_cast<int>(k_tiles), static_cast<u32x4*>(tiled));
    return check_launch(what);
}

int64_t tq_adapters_workspace_bytes(const tq_adapters* adapters, int64_t m) {
    using namespace tq;
    if (check_adapters("tq_adapters_add", adapters, m) != TQ_OK) return -1;
    if (m == 0 || in_one_launch(adapters, m)) return 0;
    const Cut c = cut_of(adapters, m);
    return shares_bytes(c) + most_shares(c) * m * adapters->parts * adapters->rank * 4;
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
    const int64_t need = tq_adapters_workspace_bytes(adapters, m), ranks = adapters->count * adapters->rank;
    const Extent to{out, m * adapters->n, 4};
    TQ_REQUIRE(out == y || !overlap(to, Extent{y, m * adapters->n, 4}), "%s: out overlaps a part of y", what);
    TQ_REQUIRE(!overlap({to}, {{x, m * adapters->k, size}, {index, m, 4}, {adapters->scales, adapters->count, 4},
                               {adapters->a, adapters->parts * ranks, (adapters->k + kKUnit - 1) / kKUnit * kKUnit * 2},
                               {adapters->b, adapters->n * ranks, 2}, {need == 0 ? nullptr : workspace, need, 1}}),
               "%s: out overlaps x, index, the adapters or the workspace", what);
    TQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 16)),
               "%s: workspace of %lld bytes, 16-byte aligned, needed", what, (long long)need);
    const Cut c = cut_of(adapters, m);
    AdaptArg a{};
    a.x = x;
    a.index = index;
    a.a = static_cast<const uint16_t*>(adapters->a);
    a.b = static_cast<const uint16_t*>(adapters->b);
    a.scales = adapters->scales;
    a.y = y;
    a.out = out;
    a.m = static_cast<int>(m);
    a.k = static_cast<int>(adapters->k);
    a.k_row = static_cast<int>((adapters->k + kKUnit - 1) / kKUnit * kKUnit);
    a.n = static_cast<int>(adapters->n);
    a.count = static_cast<int>(adapters->count);
    a.parts = static_cast<int>(adapters->parts);
    a.rank = static_cast<int>(adapters->rank);
    a.np = static_cast<int>(adapters->n / adapters->parts);
    const bool vec_x = aligned(x, 16) && adapters->k % 8 == 0;
    const bool vec_y = aligned(y, 16) && aligned(out, 16) && a.np % 4 == 0;
    if (need == 0)
        return adapters->dtype == TQ_DT_F16 ? launch_once<TQ_DT_F16>(a, dtype, vec_x, vec_y, as_hip(stream), what)
                                            : launch_once<TQ_DT_BF16>(a, dtype, vec_x, vec_y, as_hip(stream), what);
    a.shares = static_cast<int32_t*>(workspace);
    a.t = reinterpret_cast<float*>(static_cast<char*>(workspace) + shares_bytes(c));
    a.low_shift = c.tokens == 16 ? 4 : 5;
    a.turns = (a.k_row + kKUnit * kWaves - 1) / (kKUnit * kWaves);
    a.gang_shift = c.gang_shift;
    TQ_REQUIRE(c.tiles << c.gang_shift <= kMaxBlocks && (m + 15) / 16 <= kMaxBlocks, "%s: %lld tokens are more than a launch holds", what,
               (long long)m);
    const dim3 low(static_cast<uint32_t>(c.tiles << c.gang_shift), static_cast<uint32_t>(c.groups));
    return adapters->dtype == TQ_DT_F16 ? launch_typed<TQ_DT_F16>(a, c, dtype, vec_x, vec_y, low, as_hip(stream), what)
                                        : launch_typed<TQ_DT_BF16>(a, c, dtype, vec_x, vec_y, low, as_hip(stream), what);
}

}  // extern "C"
