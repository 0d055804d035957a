// tq_kv_attention.hip -- attention of new tokens over the 8-bit key/value cache.
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = 2^(scale log2(e) q . k_j - max)
//
// One pass over the cache with the running maximum and sum of the softmax.  Rows: the T new tokens x the `group`
// query heads that share a key head, 16 kNQ of them per tile.  A step of a wave is 32 keys, on the f16 matrix cores
// (v_mfma_f32_16x16x32_f16), and every operand comes into its lane straight from memory,
// without LDS or lane exchanges:
//  * S^T = K Q^T, 16 keys at a time: lane (r, g) = (l % 16, l / 16) holds key r's codes
//    D/4 g .. D/4 (g + 1) - 1 as one run of bytes; q is laid out over k the same way;
//  * the lane then holds the scores of keys 4 g + e of both 16-key halves for row r: as B operand
//    of O^T += V^T P^T its 8 k-slots are those 8 keys, so P needs no move, and V's lane loads the
//    bytes of those 8 keys at its own D/16 elements d;
//  * bytes become f16 pairs by byte permutes: INT8 as 1024 + (code + 128) (the bytes of an f16
//    with exponent 2^10) minus 1152, e4m3 by v_cvt_scalef32_pk_f16_fp8, both exact.
// The value scale sv_j goes into the exponent: with t_j = s_j + log2 sv_j and the running
// maximum of t, P_j = 2^(t_j - max) = p_j sv_j needs no normalising to fit f16's
// range whatever the scales, and the sum takes P_j / sv_j.  P has two f16 planes, 22 bits, for every type (in one, 11
// bits, 36 % of f16 outputs and 6 % of bf16 ones were not the nearest to the exact result); q, scaled by a power of
// two for each row, has two for f32 and one for 16-bit rows, which it holds exactly.
//
// Work is split along the keys by units of 128: the units of all sequences, heads and row
// tiles in one line, cut into equal shares for a grid that fits the chip at once, whatever the lengths.  A share that
// is not a whole (sequence, head, tile) leaves maximum, sum and O in the workspace, and a second launch joins them in order.
#include <algorithm>
#include <cmath>

#include "tq_kv.h"

namespace tq {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

constexpr int kAttBlock = 256, kAttWaves = kAttBlock / kWave;
constexpr int kStep = 32;                    // keys of a wave's step
constexpr int kUnit = kAttWaves * kStep;     // keys of a unit
// P = 2^(t - m): m is the running maximum less kPShift, and it and O move only once the maximum
// has passed it by more than kPShift + kPSlack, so that P stays in [0, 2^15] of f16's 2^16 (at 32 rows some
// row's maximum moves in nearly every step: rescaling O each time took as long as the softmax)
constexpr float kPShift = 8.0f, kPSlack = 7.0f;

struct AttArg {
    KvBatch b;
    const uint8_t* k;
    const float* k_scale;
    const uint8_t* v;
    const float* v_scale;
    const void* q;
    int64_t q_token, q_head;
    const int32_t* tree;
    int64_t tree_words;
    void* out;
    float* part;   // partial O, then {max, sum}; null: a block for each item, no split
    int heads, group, d, dtype, blocks;
    bool q_vec, out_vec;
    float scale2;  // scale log2(e)
    FastDiv by_group;
};

__device__ __forceinline__ void store_elem(void* p, int64_t i, int dtype, float x);

// ------------------------------------------------------------------ the line of work
// 64 sequences at a time, one in each lane: rows, keys and units, with the running totals of
// items ((head, tile) pairs) and units.
struct SeqLane {
    int first, rows, len, base;  // first row of q; new tokens; keys; place of the first new token
    int tiles, units, items;
    int items_end, units_end;    // inclusive totals within the 64
};

// inclusive sums over the lanes: within rows of 16 by shifts, then lane 15's total into the next row and lane 31's
// into the upper half
__device__ __forceinline__ int scan64(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}

// kUnit * per keys are a unit of the line.
template <int kTile>
__device__ __forceinline__ SeqLane seq_lane(const AttArg& a, int seq0, int lane, int per) {
    SeqLane s{};
    const int seq = seq0 + lane;
    bool falls = false;
    if (seq < a.b.batch) {
        int first = a.b.offsets ? a.b.offsets[seq] : seq * a.b.max_tokens;
        const int last = a.b.offsets ? a.b.offsets[seq + 1] : first + a.b.max_tokens;
        s.first = first;
        s.rows = kv_rows_fit(a.b, first, last) ? last - first : 0;
        const int length = min(max(a.b.lengths[seq], 0), 1 << 30);
        s.len = min(length, a.b.cap);
        s.base = length - s.rows;
        s.tiles = (s.rows * a.group + kTile - 1) / kTile;
        s.units = max((s.len + kUnit - 1) / kUnit, 1);
        if (per > 1) s.units = (s.units + per - 1) / per;
        s.items = s.tiles * a.heads;
        falls = last < first;
    }
    // Offsets that decrease would count rows twice, past what the host's limit on units keeps in 32 bits: none of these 64.
    if (__ballot(falls)) s.items = 0;
    if (a.b.batch == 1) {  // every lane past the first holds nothing
        s.items_end = readlane(s.items, 0);
        s.units_end = readlane(s.items * s.units, 0);
    } else {
        s.items_end = scan64(s.items);
        s.units_end = scan64(s.items * s.units);
    }
    return s;
}

// The line as the blocks share it: `units` of kUnit * per keys over `blocks`.  Where items are few, `per` is the least
// for which each unit can have a block of its own, so that no block works on two items, whose rows would be read, set up
// and written twice (trees of 48 drafts, 128 items of 4 to 16 units: 26 us with equal shares of the line, 22 so); where
// they are many, such units would leave blocks idle, and the line is cut into equal shares of single units.
struct Line {
    int per, units, blocks;
};

template <int kTile>
__device__ __forceinline__ Line share_line(const AttArg& a, SeqLane& s, int lane) {
    Line w{1, 0, a.blocks};
    s = seq_lane<kTile>(a, 0, lane, 1);
    if (!a.part) return w;
    w.units = readlane(s.units_end, 63);
    if (a.b.batch > 64) {
        int64_t units = w.units;
        for (int s0 = 64; s0 < a.b.batch; s0 += 64) units += readlane(seq_lane<kTile>(a, s0, lane, 1).units_end, 63);
        w.units = units <= INT32_MAX ? static_cast<int>(units) : 0;  // (more only where offsets decrease from one 64 to another: nothing)
        return w;
    }
    if (w.units <= a.blocks || readlane(s.items_end, 63) > a.blocks / 2) return w;
    // ends: with `per` at the longest item's units there are as many units as items
    for (w.per = (w.units + a.blocks - 1) / a.blocks;; w.per += 1 + w.per / 16) {
        const int mine = (s.units + w.per - 1) / w.per, v = s.items * mine;
        const int end = a.b.batch == 1 ? readlane(v, 0) : scan64(v), units = readlane(end, 63);
        if (units <= a.blocks) {
            s.units = mine;
            s.units_end = end;
            w.units = w.blocks = units;
            return w;
        }
    }
}

// Share i of u units over n blocks: u / n each, one more for the first u % n.
struct Shares {
    int q, r;
    __device__ Shares(int u, int n) : q(u / n), r(u - u / n * n) {}
    __device__ int begin(int i) const { return i * q + min(i, r); }
    __device__ int of(int u) const {
        const int split = r * (q + 1);
        return u < split ? u / (q + 1) : r + (u - split) / q;
    }
};

// One (sequence, head, tile) and where its units lie in the line; uniform.
struct Item {
    int first, rows, len, base, units, tile, head, unit0, seq;
    bool ok;
};

template <bool kByUnit>
__device__ __forceinline__ Item pick(const SeqLane& s, int seq0, int items0, int units0, int at) {
    const int end = kByUnit ? units0 + s.units_end : items0 + s.items_end;
    const int j = __popcll(__ballot(end <= at));
    Item it;
    it.seq = seq0 + j;
    it.first = readlane(s.first, j);
    it.rows = readlane(s.rows, j);
    it.len = readlane(s.len, j);
    it.base = readlane(s.base, j);
    it.units = readlane(s.units, j);
    const int tiles = readlane(s.tiles, j), items = readlane(s.items, j);
    const int u_start = units0 + readlane(s.units_end, j) - items * it.units;
    int i;
    if (kByUnit)
        i = (at - u_start) / it.units;
    else
        i = at - (items0 + readlane(s.items_end, j) - items);
    it.unit0 = u_start + i * it.units;
    it.head = i / tiles;
    it.tile = i - it.head * tiles;
    it.ok = true;
    return it;
}

// The item that holds unit `at` (kByUnit) or item number `at`.
template <int kTile, bool kByUnit>
__device__ __forceinline__ Item find_item(const AttArg& a, const SeqLane& s0, int at, int lane) {
    if (a.b.batch <= 64) {
        if (at >= readlane(kByUnit ? s0.units_end : s0.items_end, 63)) return Item{};
        return pick<kByUnit>(s0, 0, 0, 0, at);
    }
    int items = 0, units = 0;
    for (int seq = 0; seq < a.b.batch; seq += 64) {
        const SeqLane s = seq_lane<kTile>(a, seq, lane, 1);
        const int ni = readlane(s.items_end, 63), nu = readlane(s.units_end, 63);
        if (at < (kByUnit ? units + nu : items + ni)) return pick<kByUnit>(s, seq, items, units, at);
        items += ni;
        units += nu;
    }
    return Item{};
}

// Zeros for the rows of no sequence: those before the first one, and those whose offsets do not fit the batch.  A block looks at 64
// sequences, at its end (at the start, which the loop over the keys is scheduled with, a batch of 64 took 91 us for 79).
__device__ __forceinline__ void zero_strays(const AttArg& a, int tid) {
    if (!a.b.offsets) return;
    const int lane = tid & 63;
    const int64_t row = static_cast<int64_t>(a.heads) * a.group * a.d;
    for (int g = blockIdx.x; g <= (a.b.batch - 1) / 64; g += gridDim.x) {
        const int seq = 64 * g + lane;
        int begin = 0, end = 0;
        if (seq < a.b.batch) {
            const int first = a.b.offsets[seq], last = a.b.offsets[seq + 1];
            const bool fits = kv_rows_fit(a.b, first, last);
            begin = seq == 0 ? 0 : max(first, 0);
            end = fits ? (seq == 0 ? first : begin) : min(last, a.b.tokens);
        }
        for (uint64_t todo = __ballot(begin < end); todo; todo &= todo - 1) {  // as a rule none
            const int j = __ffsll(static_cast<unsigned long long>(todo)) - 1, r0 = readlane(begin, j), r1 = readlane(end, j);
            for (int64_t i = r0 * row + tid; i < r1 * row; i += kAttBlock) store_elem(a.out, i, a.dtype, 0.f);
        }
    }
}

// Which of the 32 keys from `key` row t of the item's new tokens sees, a bit each (keys past the
// length may be among them): one comparison, or two words of the tree, for all of them.
__device__ __forceinline__ uint32_t seen_from(const AttArg& a, const Item& it, int t, int key) {
    auto first = [](int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; };
    const int j = key - it.base;  // place among the new tokens, negative before them
    if (!a.tree) return first(t + 1 - j);
    const int32_t* row = a.tree + (it.first + static_cast<int64_t>(t)) * a.tree_words;
    const int w = j >> 5;
    const uint32_t lo = w < 0 ? ~0u : w < a.tree_words ? static_cast<uint32_t>(row[w]) : 0u;
    const uint32_t hi = w + 1 < 0 ? ~0u : w + 1 < a.tree_words ? static_cast<uint32_t>(row[w + 1]) : 0u;
    return __builtin_amdgcn_alignbit(hi, lo, j & 31) & first(it.rows - j);
}

// ------------------------------------------------------------------ arithmetic
__device__ __forceinline__ f32x4 mfma_f16(h8 a, h8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// x, as a value the compiler knows nothing of: what is computed from it is computed here, not
// before a loop and kept in registers that the loop needs
__device__ __forceinline__ int here(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// max over the lanes l, l ^ 16, l ^ 32, l ^ 48 (the four that hold a row)
template <class Op>
__device__ __forceinline__ float over_groups(float v, Op op) {
    const uint32_t u = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const uint32_t w = __float_as_uint(v);
    const auto c = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return op(__uint_as_float(c[0]), __uint_as_float(c[1]));
}

struct CodesI8 {
    static constexpr bool kNan = false;
    // bytes ready for pair(): code + 128
    __device__ static uint32_t ready(uint32_t w) { return w ^ 0x80808080u; }
    template <bool kHigh>
    __device__ static h2 pair(uint32_t w) {  // bytes 0, 1 or 2, 3
        const uint32_t u = __builtin_amdgcn_perm(0x64646464u, w, kHigh ? 0x04030402u : 0x04010400u);
        const h2 bias = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
        return __builtin_bit_cast(h2, u) + bias;
    }
};
struct CodesFp8 {
    static constexpr bool kNan = true;
    __device__ static uint32_t ready(uint32_t w) { return w; }
    template <bool kHigh>
    __device__ static h2 pair(uint32_t w) {
        return __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w), 1.0f, kHigh));
    }
};

__device__ __forceinline__ h8 join(h2 a, h2 b, h2 c, h2 d) {
    return h8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// f32 -> f16 (nearest) and, in two planes, what that leaves
template <int kPlanes>
__device__ __forceinline__ void to_planes(float x, _Float16& hi, _Float16& lo) {
    hi = static_cast<_Float16>(x);
    if constexpr (kPlanes == 2) lo = static_cast<_Float16>(x - static_cast<float>(hi));
}

// A lane's bytes of a key in V: tiles of 16 d, row r of tile t being element vpos(r, t).  One
// run of kDP / 16 bytes (kDP = 96: a run of 4 and one of 2).
template <int kDP>
__device__ __forceinline__ int vpos(int r, int t) {
    if constexpr (kDP == 96) return t < 4 ? 4 * r + t : 64 + 2 * r + (t - 4);
    return kDP / 16 * r + t;
}

template <int kDP>
struct VBytes {
    static constexpr int kWords = kDP == 128 || kDP == 96 ? 2 : 1;
    uint32_t w[kWords];
    __device__ void load(const uint8_t* row, int r) {
        if constexpr (kDP == 128) {
            const uint2 x = *reinterpret_cast<const uint2*>(row + 8 * r);
            w[0] = x.x;
            w[1] = x.y;
        } else if constexpr (kDP == 96) {
            w[0] = *reinterpret_cast<const uint32_t*>(row + 4 * r);
            w[1] = *reinterpret_cast<const uint16_t*>(row + 64 + 2 * r);
        } else if constexpr (kDP == 64) {
            w[0] = *reinterpret_cast<const uint32_t*>(row + 4 * r);
        } else {
            w[0] = *reinterpret_cast<const uint16_t*>(row + 2 * r);
        }
    }
};

template <int kDP>
struct KBytes {
    static constexpr int kWords = kDP / 16;
    uint32_t w[kWords];
    __device__ void load(const uint8_t* p) {
        if constexpr (kDP == 128 || kDP == 64) {
#pragma unroll
            for (int i = 0; i < kWords; i += 4) {
                const u32x4 x = *reinterpret_cast<const u32x4*>(p + 4 * i);
#pragma unroll
                for (int e = 0; e < 4; ++e) w[i + e] = x[e];
            }
        } else {
#pragma unroll
            for (int i = 0; i < kWords; i += 2) {
                const uint2 x = *reinterpret_cast<const uint2*>(p + 4 * i);
                w[i] = x.x;
                w[i + 1] = x.y;
            }
        }
    }
};

__device__ __forceinline__ float load_elem(const void* p, int64_t i, int dtype) {
    if (dtype == TQ_DT_F32) return static_cast<const float*>(p)[i];
    if (dtype == TQ_DT_BF16) return static_cast<float>(static_cast<const __bf16*>(p)[i]);
    return static_cast<float>(static_cast<const _Float16*>(p)[i]);
}
__device__ __forceinline__ void store_elem(void* p, int64_t i, int dtype, float x) {
    if (dtype == TQ_DT_F32)
        static_cast<float*>(p)[i] = x;
    else if (dtype == TQ_DT_BF16)
        static_cast<__bf16*>(p)[i] = static_cast<__bf16>(x);
    else
        static_cast<_Float16*>(p)[i] = static_cast<_Float16>(x);
}
// 8 adjacent elements as they lie in memory (f32: both words, else the first)
__device__ __forceinline__ void widen_8(const u32x4 (&raw)[2], int dtype, float* x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t u = raw[0][e], u1 = raw[1][e];  // (a bit cast of the vector's element itself takes element 0)
        if (dtype == TQ_DT_F32) {
            x[e] = __uint_as_float(u);
            x[4 + e] = __uint_as_float(u1);
        } else if (dtype == TQ_DT_BF16) {
            x[2 * e] = __uint_as_float(u << 16);
            x[2 * e + 1] = __uint_as_float(u & 0xFFFF0000u);
        } else {
            const h2 h = __builtin_bit_cast(h2, u);
            x[2 * e] = static_cast<float>(h.x);
            x[2 * e + 1] = static_cast<float>(h.y);
        }
    }
}
// 8 adjacent elements, 16-byte aligned
__device__ __forceinline__ void load_8(const void* p, int64_t i, int dtype, float* x) {
    u32x4 raw[2];
    if (dtype == TQ_DT_F32) {
        const u32x4* s = reinterpret_cast<const u32x4*>(static_cast<const float*>(p) + i);
        raw[0] = s[0];
        raw[1] = s[1];
    } else {
        raw[0] = raw[1] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + i);
    }
    widen_8(raw, dtype, x);
}

// 8 adjacent elements, 16-byte aligned
__device__ __forceinline__ void store_8(void* p, int64_t i, int dtype, const float (&x)[8]) {
    if (dtype == TQ_DT_F32) {
        f32x4* o = reinterpret_cast<f32x4*>(static_cast<float*>(p) + i);
        o[0] = f32x4{x[0], x[1], x[2], x[3]};
        o[1] = f32x4{x[4], x[5], x[6], x[7]};
        return;
    }
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
        w[e] = dtype == TQ_DT_BF16
                   ? __builtin_bit_cast(uint32_t, (b2{static_cast<__bf16>(x[2 * e]), static_cast<__bf16>(x[2 * e + 1])}))
                   : __builtin_bit_cast(uint32_t, (h2{static_cast<_Float16>(x[2 * e]), static_cast<_Float16>(x[2 * e + 1])}));
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + i) = u32x4{w[0], w[1], w[2], w[3]};
}

// 4 adjacent elements, aligned to their size
__device__ __forceinline__ void store_4(void* p, int64_t i, int dtype, const float (&x)[4]) {
    if (dtype == TQ_DT_F32) {
        *reinterpret_cast<f32x4*>(static_cast<float*>(p) + i) = f32x4{x[0], x[1], x[2], x[3]};
        return;
    }
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    uint32_t w[2];
#pragma unroll
    for (int e = 0; e < 2; ++e)
        w[e] = dtype == TQ_DT_BF16
                   ? __builtin_bit_cast(uint32_t, (b2{static_cast<__bf16>(x[2 * e]), static_cast<__bf16>(x[2 * e + 1])}))
                   : __builtin_bit_cast(uint32_t, (h2{static_cast<_Float16>(x[2 * e]), static_cast<_Float16>(x[2 * e + 1])}));
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) = make_uint2(w[0], w[1]);
}

// ------------------------------------------------------------------ the kernel
template <int kDP, int kNQ, class Codes, int kPlanes>
__global__ __launch_bounds__(kAttBlock, kNQ == 2 ? 1 : 2) void k_kv_attention(AttArg a) {
    constexpr int kTile = 16 * kNQ;
    constexpr int kSteps = kDP / 32;   // 32-wide d steps of S^T
    constexpr int kVT = kDP / 16;      // 16-wide d tiles of O^T
    constexpr int kORow = kDP + 4;     // padded against bank conflicts
    constexpr int kRun = kDP / 4;      // K bytes of a lane
    __shared__ float o_lds[kTile * kORow];
    __shared__ float m_lds[kAttWaves][kTile], l_lds[kAttWaves][kTile];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    SeqLane s0;
    const Line line = share_line<kTile>(a, s0, lane);
    int at = 0, end = 1;
    if (a.part) {
        const Shares sh(line.units, line.blocks);
        at = sh.begin(blockIdx.x);
        end = static_cast<int>(blockIdx.x) < line.blocks ? sh.begin(blockIdx.x + 1) : at;
    }
    bool first_share = true;
    while (at < end) {
        const Item it = a.part ? find_item<kTile, true>(a, s0, at, lane) : find_item<kTile, false>(a, s0, blockIdx.x, lane);
        if (!it.ok) break;
        const int u_first = a.part ? at - it.unit0 : 0;
        const int u_count = a.part ? min(it.units - u_first, end - at) : it.units;
        const int n_rows = it.rows * a.group;

        // what the tile's rows see: all keys before `all`, none from `lim` on
        const int t_first = static_cast<int>(a.by_group.div(it.tile * kTile));
        const int t_last = static_cast<int>(a.by_group.div(min(it.tile * kTile + kTile, n_rows) - 1));
        const int lim = a.tree ? it.len : min(it.base + t_last + 1, it.len);
        const int all = a.tree ? min(it.base, it.len) : min(it.base + t_first + 1, it.len);

        const int k_end = min((u_first + u_count) * line.per * kUnit, lim);
        const int k_begin = u_first * line.per * kUnit + wave * kStep;
        const int32_t* table = a.b.table + static_cast<int64_t>(it.seq) * a.b.table_stride;

        // Pages of the 16 keys each (a page holds whole sixteens) of the step to be loaded next: read a step before
        // they are needed, as a wave that waited for its pages had nothing under way.
        int pages[2];
        auto load_pages = [&](int key) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int kk = key + 16 * i < it.len ? key + 16 * i : 0;
                pages[i] = table[a.b.by_page.div(static_cast<uint32_t>(kk))];
            }
        };
        // Where the 16 keys from `key`, the step's i-th, lie: row of the cache's [pages, heads, page], and whether they
        // lie anywhere.
        auto place16 = [&](int key, int i, bool& ok) -> int64_t {
            ok = key < it.len && pages[i] >= 0 && pages[i] < a.b.pages;
            const int kk = ok ? key : 0, in = kk - static_cast<int>(a.b.by_page.div(static_cast<uint32_t>(kk))) * a.b.page;
            return (static_cast<int64_t>(ok ? pages[i] : 0) * a.heads + it.head) * a.b.page + in;
        };

        KBytes<kDP> kb[2];
        VBytes<kDP> vb[8];
        f32x4 ks[2], vs[2];
        bool ok_k[2], ok_v[2];
        auto load_k = [&](int key) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int64_t row = place16(key + 16 * i, i, ok_k[i]);
                kb[i].load(a.k + row * kDP + (r * kDP + kRun * g));
                ks[i] = *reinterpret_cast<const f32x4*>(a.k_scale + row + 4 * g);
            }
        };
        auto load_v = [&](int key) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int64_t row = place16(key + 16 * i, i, ok_v[i]);
                const uint8_t* p = a.v + row * kDP + 4 * g * kDP;
#pragma unroll
                for (int j = 0; j < 4; ++j) vb[4 * i + j].load(p + j * kDP, r);
                vs[i] = *reinterpret_cast<const f32x4*>(a.v_scale + row + 4 * g);
            }
        };
        // q: row r of each 16, elements kRun g + 8 s + j
        h8 q[kNQ][kPlanes][kSteps];
        float rq[kNQ];
        int t_row[kNQ];
#pragma unroll
        for (int n = 0; n < kNQ; ++n) {
            const int row = it.tile * kTile + 16 * n + r;
            const bool in = row < n_rows;
            const int rr = in ? row : n_rows - 1;
            const int t = static_cast<int>(a.by_group.div(rr));
            t_row[n] = t;
            const int64_t at_q = (it.first + static_cast<int64_t>(t)) * a.q_token +
                                 (static_cast<int64_t>(it.head) * a.group + (rr - t * a.group)) * a.q_head;
            float x[8 * kSteps];
            float top = 0.f;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const int d0 = kRun * g + 8 * s;
                if (a.q_vec) {
                    if (d0 < a.d) {
                        load_8(a.q, at_q + d0, a.dtype, x + 8 * s);
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) x[8 * s + j] = 0.f;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        x[8 * s + j] = d0 + j < a.d ? load_elem(a.q, at_q + d0 + j, a.dtype) : 0.f;
                }
            }
#pragma unroll
            for (int j = 0; j < 8 * kSteps; ++j) top = fmaxf(top, fabsf(x[j]));
            top = over_groups(top, OpMax{});
            // a power of two brings the row to [2^13, 2^14): f16 keeps all 11 bits of what counts
            const int e = top > 0.f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) - 14 : 0;
            rq[n] = a.scale2 * ldexpf(1.0f, e);
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    _Float16 hi, lo;
                    to_planes<kPlanes>(ldexpf(x[8 * s + j], -e), hi, lo);
                    q[n][0][s][j] = hi;
                    if constexpr (kPlanes == 2) q[n][1][s][j] = lo;
                }
        }

        f32x4 o[kNQ][kVT];
        float m[kNQ], l[kNQ];  // l: of this lane's keys
#pragma unroll
        for (int n = 0; n < kNQ; ++n) {
            m[n] = -INFINITY;
            l[n] = 0.f;
#pragma unroll
            for (int t = 0; t < kVT; ++t) o[n][t] = f32x4{};
        }

        if (k_begin < k_end) {
            load_pages(k_begin);
            load_k(k_begin);
            load_v(k_begin);
            load_pages(k_begin + kUnit);
        }
        for (int key = k_begin; key < k_end; key += kUnit) {
            const int next = key + kUnit < k_end ? key + kUnit : key;  // the last step again: never used
            f32x4 st[2][kNQ];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int n = 0; n < kNQ; ++n) st[i][n] = f32x4{};
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
                    const uint32_t w0 = Codes::ready(kb[i].w[2 * s]), w1 = Codes::ready(kb[i].w[2 * s + 1]);
                    const h8 kf = join(Codes::template pair<false>(w0), Codes::template pair<true>(w0),
                                       Codes::template pair<false>(w1), Codes::template pair<true>(w1));
#pragma unroll
                    for (int n = 0; n < kNQ; ++n)
#pragma unroll
                        for (int p = 0; p < kPlanes; ++p) st[i][n] = mfma_f16(kf, q[n][p][s], st[i][n]);
                }
            }
            const f32x4 ck[2] = {ks[0], ks[1]};
            const bool both = ok_k[0] && ok_k[1];
            const bool seen0 = ok_k[0], seen1 = ok_k[1];
            load_k(next);

            // log2 and reciprocal of the value scales; a scale of 0 counts as 1e-25, NaN stays
            float lsv[8], rsv[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float sv = vs[j >> 2][j & 3], c = fmaxf(sv, 1e-25f);
                lsv[j] = __builtin_amdgcn_logf(sv != sv ? sv : c);
                rsv[j] = __builtin_amdgcn_rcpf(c);
            }
            const bool slow = !both || key + kStep > all;  // uniform
            uint32_t seen[kNQ];                            // bit j: key j of the lane is seen by row n
            h8 pf[kNQ][2];
#pragma unroll
            for (int n = 0; n < kNQ; ++n) {
                float t[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) t[j] = fmaf(st[j >> 2][n][j & 3] * rq[n], ck[j >> 2][j & 3], lsv[j]);
                if (slow) {
                    const uint32_t window = seen_from(a, it, t_row[n], key);
                    uint32_t bits = 0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int i = 16 * (j >> 2) + 4 * g + (j & 3);
                        const bool see = (window >> i & 1) != 0 && key + i < it.len && (j < 4 ? seen0 : seen1);
                        t[j] = see ? t[j] : -INFINITY;
                        bits |= see ? 1u << j : 0u;
                    }
                    seen[n] = bits;
                }
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, t[j]);
                top = over_groups(top, OpMax{}) - kPShift;
                if (__ballot(top > m[n] + kPSlack)) {
                    top = top > m[n] + kPSlack ? top : m[n];  // (a row's result depends on no other row)
                    const float ref = top == -INFINITY ? 0.f : top;
                    const float alpha = exp2_hw(m[n] - ref);
                    l[n] *= alpha;
#pragma unroll
                    for (int v = 0; v < kVT; ++v) o[n][v] *= alpha;
                    m[n] = top;
                }
                const float ref = m[n] == -INFINITY ? 0.f : m[n];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float p = exp2_hw(t[j] - ref);
                    l[n] = fmaf(p, rsv[j], l[n]);
                    _Float16 hi, lo;
                    to_planes<2>(p, hi, lo);
                    pf[n][0][j] = hi;
                    pf[n][1][j] = lo;
                }
            }
            // Rows that do not see a key must not meet its codes' NaNs (0 * NaN): codes nobody sees
            // and NaN codes become 0 here, and a seen NaN code makes its element of o NaN.
            uint32_t any_nan = 0;
            if (Codes::kNan && slow) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int kk = key + 16 * (j >> 2) + 4 * g + (j & 3);
                    const bool lies = (j < 4 ? seen0 : seen1) && kk < lim;
#pragma unroll
                    for (int w = 0; w < VBytes<kDP>::kWords; ++w) {
                        const uint32_t x = lies ? vb[j].w[w] : 0u;
                        vb[j].w[w] = x;
                        any_nan |= ((x & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
                    }
                }
                if (__ballot(any_nan != 0)) {
                    const _Float16 one = static_cast<_Float16>(1.0f), zero = static_cast<_Float16>(0.0f);
#pragma unroll
                    for (int v = 0; v < kVT; ++v) {
                        h8 bad;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const uint32_t byte = vb[j].w[v >> 2] >> (8 * (v & 3)) & 0x7Fu;
                            bad[j] = byte == 0x7Fu ? one : zero;
                        }
#pragma unroll
                        for (int n = 0; n < kNQ; ++n) {
                            h8 see;
#pragma unroll
                            for (int j = 0; j < 8; ++j) see[j] = seen[n] >> j & 1 ? one : zero;
                            const f32x4 hit = mfma_f16(bad, see, f32x4{});
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[n][v][e] = hit[e] > 0.f ? NAN : o[n][v][e];
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int w = 0; w < VBytes<kDP>::kWords; ++w) {
                            const uint32_t x = vb[j].w[w];
                            const uint32_t top_bits = ((x & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
                            vb[j].w[w] = x & ~((top_bits << 1) - (top_bits >> 7));
                        }
                }
            }
            // O^T += V^T P^T, two d tiles at a time: bytes b and b + 1 of the 8 keys as pairs of keys
#pragma unroll
            for (int v = 0; v < kVT; v += 2) {
                h2 lo[4], hi[4];
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const uint32_t x = Codes::ready(vb[j].w[v >> 2]), y = Codes::ready(vb[j + 1].w[v >> 2]);
                    const uint32_t w = __builtin_amdgcn_perm(y, x, (v & 2) ? 0x07030602u : 0x05010400u);
                    lo[j >> 1] = Codes::template pair<false>(w);
                    hi[j >> 1] = Codes::template pair<true>(w);
                }
                const h8 f0 = join(lo[0], lo[1], lo[2], lo[3]), f1 = join(hi[0], hi[1], hi[2], hi[3]);
#pragma unroll
                for (int n = 0; n < kNQ; ++n)
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        o[n][v] = mfma_f16(f0, pf[n][p], o[n][v]);
                        o[n][v + 1] = mfma_f16(f1, pf[n][p], o[n][v + 1]);
                    }
            }
            load_v(next);
            load_pages(next + kUnit);
        }

        // the four waves' shares of the keys meet in LDS, in the order of the waves
        if (g == 0)
#pragma unroll
            for (int n = 0; n < kNQ; ++n) m_lds[wave][16 * n + r] = m[n];
        __syncthreads();
        float f[kNQ];
#pragma unroll
        for (int n = 0; n < kNQ; ++n) {
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kAttWaves; ++w) top = fmaxf(top, m_lds[w][16 * n + r]);
            f[n] = m[n] == -INFINITY ? 0.f : exp2_hw(m[n] - top);
            const float sum = over_groups(l[n], OpAdd{});
            if (g == 0) l_lds[wave][16 * n + r] = sum * f[n];
        }
        for (int w = 0; w < kAttWaves; ++w) {
            if (w == wave) {
#pragma unroll
                for (int n = 0; n < kNQ; ++n)
#pragma unroll
                    for (int v = 0; v < kVT; ++v)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float* p = &o_lds[(16 * n + r) * kORow + vpos<kDP>(4 * g + e, v)];
                            const float x = o[n][v][e] * f[n];
                            *p = w == 0 ? x : *p + x;
                        }
            }
            __syncthreads();
        }
        const bool whole = u_count == it.units;
        const int valid = min(kTile, n_rows - it.tile * kTile);
        if (whole) {
            for (int i = tid; i < valid * kDP; i += kAttBlock) {
                const int row = i / kDP, d = i % kDP;
                if (d >= a.d) continue;
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < kAttWaves; ++w) sum += l_lds[w][row];
                const int rr = it.tile * kTile + row, t = static_cast<int>(a.by_group.div(rr));
                const int64_t dst = ((it.first + static_cast<int64_t>(t)) * (static_cast<int64_t>(a.heads) * a.group) +
                                     static_cast<int64_t>(it.head) * a.group + (rr - t * a.group)) * a.d + d;
                store_elem(a.out, dst, a.dtype, sum == 0.f ? 0.f : o_lds[row * kORow + d] / sum);
            }
        } else {
            const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (first_share ? 0 : 1);
            float* po = a.part + slot * (kTile * kDP);
            float* pml = a.part + 2 * static_cast<int64_t>(a.blocks) * (kTile * kDP) + slot * (2 * kTile);
            for (int i = tid; i < valid * kDP; i += kAttBlock) po[i] = o_lds[i / kDP * kORow + i % kDP];
            if (tid < valid) {
                float top = -INFINITY, sum = 0.f;
#pragma unroll
                for (int w = 0; w < kAttWaves; ++w) {
                    top = fmaxf(top, m_lds[w][tid]);
                    sum += l_lds[w][tid];
                }
                pml[2 * tid] = top;
                pml[2 * tid + 1] = sum;
            }
        }
        __syncthreads();
        first_share = false;
        at += u_count;
    }
    zero_strays(a, threadIdx.x);
}

// Joins the shares of the items that several blocks worked on, in their order: kDP / 4 lanes (of a group of kG) for a
// row, four elements each.  A row has one group, or (kAll) those of the whole block, which take its shares by turns, eight
// at a time: maxima, sums and rows of O are all on their way before the first is needed (2000 rows of 8 heads in four
// shares: 13.7 us when the maxima came first).  A share whose maximum is -inf saw nothing (sum and O zero) or only NaN scores (both
// NaN): either way it is added, at weight 2^-inf = 0, which keeps the NaN.
template <int kDP, int kTile, bool kAll>
__global__ __launch_bounds__(kAttBlock) void k_kv_attention_join(AttArg a) {
    constexpr int kG = kDP <= 32 ? 8 : kDP <= 64 ? 16 : 32, kGroups = kAttBlock / kG, kParts = kAll ? kGroups : 1;
    __shared__ f32x4 x_lds[kAll ? kGroups : 1][kG];
    __shared__ float m_lds[kGroups], l_lds[kGroups];
    const int lane = threadIdx.x & 63, group = threadIdx.x / kG, d = 4 * (threadIdx.x % kG);
    const int row = kAll ? blockIdx.y : blockIdx.y * kGroups + group, part = kAll ? group : 0;
    SeqLane s0;
    const Line line = share_line<kTile>(a, s0, lane);
    const Item it = find_item<kTile, false>(a, s0, blockIdx.x, lane);
    if (!it.ok || line.units == 0) return;
    const bool mine = it.tile * kTile + row < it.rows * a.group;
    if (kAll && !mine) return;  // (the whole block)
    const Shares sh(line.units, line.blocks);
    const int b0 = sh.of(it.unit0), b1 = sh.of(it.unit0 + it.units - 1);
    if (b0 == b1) return;  // one block had it all
    const float* ml = a.part + 2 * static_cast<int64_t>(a.blocks) * (kTile * kDP);
    const int skip = sh.begin(b0) == it.unit0 ? 0 : 1, at_row = mine ? row : 0, at_d = min(d, kDP - 4);
    float top = -INFINITY, sum = 0.f;
    f32x4 x{};
    for (int b = b0 + part; b <= b1; b += 8 * kParts) {
        float m[8], l[8];
        f32x4 v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (u >= 4 && b + 4 * kParts > b1) {  // uniform without kAll; four cost less than eight
                m[u] = -INFINITY;
                l[u] = 0.f;
                v[u] = f32x4{};
                continue;
            }
            const int c = min(b + u * kParts, b1);
            const int64_t slot = static_cast<int64_t>(2 * c + (c == b0 ? skip : 0)) * kTile + at_row;
            m[u] = b + u * kParts <= b1 ? ml[2 * slot] : -INFINITY;
            l[u] = ml[2 * slot + 1];
            v[u] = *reinterpret_cast<const f32x4*>(a.part + slot * kDP + at_d);
        }
        float next = top;
#pragma unroll
        for (int u = 0; u < 8; ++u) next = fmaxf(next, m[u]);
        const float ref = next == -INFINITY ? 0.f : next, f0 = exp2_hw(top - ref);
        sum *= f0;
        x *= f0;
        top = next;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float f = exp2_hw(m[u] - ref);
            const bool there = b + u * kParts <= b1;  // (past the last share: read again, not added)
            sum = there ? fmaf(l[u], f, sum) : sum;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = there ? fmaf(v[u][e], f, x[e]) : x[e];
        }
    }
    if constexpr (kAll) {
        x_lds[group][d / 4] = x;
        if (d == 0) {
            m_lds[group] = top;
            l_lds[group] = sum;
        }
        __syncthreads();
        if (group) return;
        const float mine_top = top;
#pragma unroll
        for (int w = 1; w < kGroups; ++w) top = fmaxf(top, m_lds[w]);
        const float f0 = mine_top == -INFINITY ? 0.f : exp2_hw(mine_top - top);
        sum *= f0;
        x *= f0;
#pragma unroll
        for (int w = 1; w < kGroups; ++w) {
            const float mw = m_lds[w], f = mw == -INFINITY ? 0.f : exp2_hw(mw - top);
            sum = fmaf(l_lds[w], f, sum);
            x += x_lds[w][d / 4] * f;
        }
    }
    if (!mine || d >= a.d) return;
    const int rr = it.tile * kTile + row, t = static_cast<int>(a.by_group.div(rr));
    const int64_t dst = ((it.first + static_cast<int64_t>(t)) * (static_cast<int64_t>(a.heads) * a.group) +
                         static_cast<int64_t>(it.head) * a.group + (rr - t * a.group)) * a.d + d;
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = sum == 0.f ? 0.f : x[e] / sum;
    if (a.out_vec) {
        store_4(a.out, dst, a.dtype, y);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < a.d) store_elem(a.out, dst + e, a.dtype, y[e]);
    }
}

// ------------------------------------------------------------------ many rows
// More than 32 rows of a sequence's head: converting the codes for each 16 of them would cost more than
// the products, so four waves share the keys, 64 at a time, converted once into LDS as the very fragments
// that the matrix cores take (16 bytes a lane, read without conflicts).  Wave (wq, wk) has rows 32 wq ..
// of the tile and, with two row groups, the wk-th 32 of the 64 keys; v_mfma_f32_32x32x16_f16:
//  * S^T = K Q^T: lane (r, h) = (l % 32, l / 32) gives key r's elements 16 s + 8 h .. + 7 in step s and
//    gets the scores of keys 8 (e / 4) + 4 h + e % 4 for row r;
//  * which are, 8 at a time, the k-slots of P^T in O^T += V^T P^T; V's fragment holds the same keys at
//    element d = 32 c + 4 (r % 8) + r / 8, so that a thread that loaded 4 adjacent elements of 8 keys
//    writes them where its neighbours write the next ones, and lane (r, h) ends up with the 16
//    adjacent elements 32 c + 16 h .. of row r.
// A power of two scales each row of q, as above.  Keys with no place become zero codes with log2 sv = -inf, and only
// tiles that hold one, or that some row sees in part, pay for a mask.
template <int kDP, int kWQ, class Codes, int kPlanes>
__global__ __launch_bounds__(kAttBlock, 2) void k_kv_attention_rows(AttArg a) {
    constexpr int kTile = 32 * kWQ, kWK = kAttWaves / kWQ;
    constexpr int kKeys = 64, kSub = 2 / kWK;      // keys of a turn; 32-key halves of a wave
    constexpr int kSteps = kDP / 16, kCols = kDP / 32;
    constexpr int kKF = 2 * kSteps * 64, kVF = 4 * kCols * 64;  // 16-byte fragments of a turn
    constexpr int kRun = kDP / 4, kQuads = kDP / 4;
    constexpr int kORow = kDP + 4;
    constexpr bool kShort = kPlanes == 2 && kDP == 128;  // of registers: places are worked out again in each turn
    struct Buf {
        h8 k[kKF], v[kVF];
        float ck[kKeys], lsv[kKeys], rsv[kKeys];
        uint32_t lie[2];  // a bit for each key that has a place
        uint8_t bad[Codes::kNan ? kKeys * kQuads : 4];
        int any_bad[kAttWaves];
    };
    // the tile's rows as f32, q before the keys and o after them, in the buffers' place
    constexpr size_t kRowBytes = sizeof(float) * kTile * kORow;
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * sizeof(Buf) > kRowBytes ? 2 * sizeof(Buf) : kRowBytes];
    __shared__ float m_lds[kAttWaves][32], l_lds[kTile];
    Buf* buf = reinterpret_cast<Buf*>(lds);
    float* rows = reinterpret_cast<float*>(lds);
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wq = wave % kWQ, wk = wave / kWQ;

    SeqLane s0;
    const Line line = share_line<kTile>(a, s0, lane);
    int at = 0, end = 1;
    if (a.part) {
        const Shares sh(line.units, line.blocks);
        at = sh.begin(blockIdx.x);
        end = static_cast<int>(blockIdx.x) < line.blocks ? sh.begin(blockIdx.x + 1) : at;
    }
    bool first_share = true;
    while (at < end) {
        if (!first_share || kShort) s0 = seq_lane<kTile>(a, 0, here(lane), line.per);  // (kept, it would hold ten registers)
        const Item it = a.part ? find_item<kTile, true>(a, s0, at, lane) : find_item<kTile, false>(a, s0, blockIdx.x, lane);
        if (!it.ok) break;
        const int u_first = a.part ? at - it.unit0 : 0;
        const int u_count = a.part ? min(it.units - u_first, end - at) : it.units;
        const int n_rows = it.rows * a.group, row0 = it.tile * kTile;

        // what the block's and the wave's rows see: every key before `all`, none from `lim` on
        auto sees = [&](int row_a, int row_b, int& all, int& lim) {
            const int ta = static_cast<int>(a.by_group.div(min(row_a, n_rows - 1)));
            const int tb = static_cast<int>(a.by_group.div(min(row_b, n_rows - 1)));
            lim = a.tree ? it.len : min(it.base + tb + 1, it.len);
            all = a.tree ? it.base : it.base + ta + 1;
        };
        int all_b, lim_b, all_w, lim_w;
        sees(row0, row0 + kTile - 1, all_b, lim_b);
        sees(row0 + 32 * wq, row0 + 32 * wq + 31, all_w, lim_w);
        const bool idle = row0 + 32 * wq >= n_rows;  // a wave without rows

        const int k_begin = u_first * line.per * kUnit;
        const int k_end = min((u_first + u_count) * line.per * kUnit, lim_b);
        const int32_t* table = a.b.table + static_cast<int64_t>(it.seq) * a.b.table_stride;

        // ---- staging: raw codes of a turn in registers, then fragments in LDS
        // K: key `lane`, bytes kRun wave ..; V: keys 16 vt + 4 vh + {0..3, 8..11}, elements 4 vd ..
        const bool v_on = tid / kQuads < 8;
        uint32_t kw[kRun / 4], vw[8];
        float sk = 0.f, sv = 0.f;
        bool k_ok = false, v_ok = false;
        // page of key `lane` of the turn to be loaded next and the key's place there, read a turn before they are
        // needed (a wait for the page is a wait for all loads before it)
        const uint32_t page_rows = static_cast<uint32_t>(a.heads) * static_cast<uint32_t>(a.b.page);  // below 2^32
        const uint32_t head_row = static_cast<uint32_t>(it.head) * static_cast<uint32_t>(a.b.page);
        int page = 0;
        uint32_t in = 0;
        auto load_page = [&](int key) {
            const int lane = (kShort ? here(tid) : tid) & 63;
            const uint32_t kk = key + lane < it.len ? key + lane : 0, i = a.b.by_page.div(kk);
            in = kk - i * a.b.page + head_row;
            page = table[i];
        };
        auto place = [&](int pg, uint32_t in, bool& ok) -> int64_t {
            ok = ok && pg >= 0 && pg < a.b.pages;
            return static_cast<int64_t>(static_cast<uint64_t>(ok ? static_cast<uint32_t>(pg) : 0u) * page_rows + in);
        };
        // loads a turn's codes, and the page of the one after it
        auto load = [&](int key) {
            const int tl = kShort ? here(tid) : tid, lane = tl & 63;
            const int vd = tl % kQuads, vth = tl / kQuads, vt = vth >> 1, vh = vth & 1;
            // the first of the sixteen keys decides: a page holds whole sixteens, and keys past the length read
            // what lies there and are dropped by their scale
            const int v_page = __shfl(page, 16 * (vt & 3));
            const uint32_t v_in = __shfl(in, 16 * (vt & 3));
            k_ok = key + lane < it.len;
            const int64_t rk = place(page, in, k_ok);
            KBytes<kDP> kb;
            kb.load(a.k + rk * kDP + kRun * wave);
#pragma unroll
            for (int i = 0; i < kRun / 4; ++i) kw[i] = kb.w[i];
            if (wave == 0) {
                sk = a.k_scale[rk];
                sv = a.v_scale[rk];
            }
            if (v_on) {
                v_ok = key + 16 * vt < it.len;
                const int64_t rv = place(v_page, v_in, v_ok);
                const uint8_t* p = a.v + (rv + 4 * vh) * kDP + 4 * vd;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    vw[j] = *reinterpret_cast<const uint32_t*>(p + ((j & 3) + 8 * (j >> 2)) * kDP);
            }
            load_page(key + kKeys);
        };
        // where row `row` of the tile lies in q (token and head strides) or in the output
        auto row_at = [&](int row, int64_t token, int64_t head) {
            const int rr = row0 + row, t = static_cast<int>(a.by_group.div(rr));
            return (it.first + static_cast<int64_t>(t)) * token + (static_cast<int64_t>(it.head) * a.group + (rr - t * a.group)) * head;
        };
        const int valid = min(kTile, n_rows - row0);
        // loads in flight of a thread, of 8 elements each (f32, which is what takes two planes: two of 16 bytes)
        constexpr int kAll = (kTile * (kDP / 8) + kAttBlock - 1) / kAttBlock;
        constexpr int kAtOnce = kPlanes == 1 ? std::min(kAll, 8) : kShort ? 2 : std::min(kAll, 4);
        u32x4 raw[kAtOnce][2];
        auto q_load = [&](int i0) {
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int i = i0 + u * kAttBlock, row = i / (kDP / 8), d0 = 8 * (i % (kDP / 8));
                const int64_t at_q = row_at(min(row, valid - 1), a.q_token, a.q_head) + (d0 < a.d ? d0 : 0);
                if (kPlanes == 2) {
                    const u32x4* src = reinterpret_cast<const u32x4*>(static_cast<const float*>(a.q) + at_q);
                    raw[u][0] = src[0];
                    raw[u][1] = src[1];
                } else {
                    raw[u][0] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + at_q);
                }
            }
        };
        if (a.q_vec) q_load(here(tid));
        if (k_begin < k_end) {  // and the first turn's codes
            load_page(k_begin);
            load(k_begin);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll 1
        for (int i0 = here(tid); i0 < kTile * (kDP / 8); i0 += kAtOnce * kAttBlock) {
            if (a.q_vec && i0 >= kAttBlock) q_load(i0);
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int i = i0 + u * kAttBlock, row = i / (kDP / 8), d0 = 8 * (i % (kDP / 8));
                if (row >= kTile) continue;
                float x[8] = {};
                if (row < valid && d0 < a.d) {
                    if (a.q_vec) {
                        widen_8(raw[u], a.dtype, x);
                    } else {
                        const int64_t at_q = row_at(row, a.q_token, a.q_head) + d0;
#pragma unroll 1
                        for (int j = 0; j < 8 && d0 + j < a.d; ++j)
                            rows[row * kORow + d0 + j] = load_elem(a.q, at_q + j, a.dtype);
#pragma unroll
                        for (int j = 0; j < 8; ++j) x[j] = d0 + j < a.d ? rows[row * kORow + d0 + j] : 0.f;
                    }
                }
                f32x4* o = reinterpret_cast<f32x4*>(&rows[row * kORow + d0]);
                o[0] = f32x4{x[0], x[1], x[2], x[3]};
                o[1] = f32x4{x[4], x[5], x[6], x[7]};
            }
        }
        __syncthreads();

        // q: row r of the wave's 32, elements 16 s + 8 h + j
        const int row = 32 * wq + r;
        const int t_row = static_cast<int>(a.by_group.div(min(row0 + row, n_rows - 1)));
        h8 q[kPlanes][kSteps];
        float rq;
        {
            const float* mine = &rows[here(row) * kORow + 8 * h];
            float top = 0.f;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const f32x4 u = *reinterpret_cast<const f32x4*>(mine + 16 * s), v = *reinterpret_cast<const f32x4*>(mine + 16 * s + 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) top = fmaxf(top, fmaxf(fabsf(u[j]), fabsf(v[j])));
            }
            // the row's largest (its two lanes)
            const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            top = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
            const int e = top > 0.f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) - 14 : 0;
            rq = a.scale2 * ldexpf(1.0f, e);
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    _Float16 hi, lo;
                    to_planes<kPlanes>(ldexpf(mine[16 * s + j], -e), hi, lo);
                    q[0][s][j] = hi;
                    if constexpr (kPlanes == 2) q[1][s][j] = lo;
                }
                if (s % 2 == 1) __builtin_amdgcn_sched_barrier(0);
            }
            __syncthreads();  // the rows are read: the buffers may be filled
        }

        f32x16 o[kCols];
#pragma unroll
        for (int c = 0; c < kCols; ++c) o[c] = f32x16{};
        float m = -INFINITY, l = 0.f;

        auto store = [&](Buf& b, int key) {
            const int lane = (kShort ? here(tid) : tid) & 63;
#pragma unroll
            for (int i = 0; i < kRun / 8; ++i) {
                const int gi = wave * (kRun / 8) + i;  // elements 8 gi ..: step gi / 2, half gi % 2
                const uint32_t w0 = Codes::ready(k_ok ? kw[2 * i] : 0u), w1 = Codes::ready(k_ok ? kw[2 * i + 1] : 0u);
                b.k[((lane >> 5) * kSteps + (gi >> 1)) * 64 + (gi & 1) * 32 + (lane & 31)] =
                    join(Codes::template pair<false>(w0), Codes::template pair<true>(w0),
                         Codes::template pair<false>(w1), Codes::template pair<true>(w1));
            }
            if (wave == 0) {
                const float c = fmaxf(sv, 1e-25f);
                b.ck[lane] = k_ok ? sk : 0.f;
                b.lsv[lane] = k_ok ? __builtin_amdgcn_logf(sv != sv ? sv : c) : -INFINITY;
                b.rsv[lane] = k_ok ? __builtin_amdgcn_rcpf(c) : 0.f;
                const uint64_t lie = __ballot(k_ok);
                if (lane < 2) b.lie[lane] = static_cast<uint32_t>(lie >> (32 * lane));
            }
            uint32_t bad_here = 0;
            if (v_on) {
                const int to = kShort ? here(tid) : tid;
                const int vd = to % kQuads, vth = to / kQuads, vt = vth >> 1, vh = vth & 1;
                const int k16 = key + 16 * vt + 4 * vh;
#pragma unroll
                for (int j = 0; j < 8; ++j) vw[j] = v_ok ? vw[j] : 0u;
                if (key + kKeys > it.len) {  // uniform
#pragma unroll
                    for (int j = 0; j < 8; ++j) vw[j] = k16 + (j & 3) + 8 * (j >> 2) < it.len ? vw[j] : 0u;
                }
                if (Codes::kNan && key + kKeys > all_b) {  // rows that do not see a key must not meet its NaN
                    const int t3 = here(tid);
                    uint8_t* bad = &b.bad[(16 * (t3 / kQuads >> 1) + 4 * (t3 / kQuads & 1)) * kQuads + t3 % kQuads];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint32_t x = vw[j], top = ((x & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
                        vw[j] = x & ~((top << 1) - (top >> 7));
                        const uint32_t bits = (top >> 7 & 1) | (top >> 14 & 2) | (top >> 21 & 4) | (top >> 28 & 8);
                        bad[((j & 3) + 8 * (j >> 2)) * kQuads] = static_cast<uint8_t>(bits);
                        bad_here |= bits;
                    }
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) vw[j] = Codes::ready(vw[j]);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    h2 lo[4], hi[4];
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const uint32_t w = __builtin_amdgcn_perm(vw[j + 1], vw[j], half ? 0x07030602u : 0x05010400u);
                        lo[j >> 1] = Codes::template pair<false>(w);
                        hi[j >> 1] = Codes::template pair<true>(w);
                    }
                    // element 4 vd + i at row 8 i + vd % 8 of column block vd / 8
                    h8* f = &b.v[(vt * kCols + (vd >> 3)) * 64 + vh * 32 + (vd & 7)];
                    f[8 * (2 * half)] = join(lo[0], lo[1], lo[2], lo[3]);
                    f[8 * (2 * half + 1)] = join(hi[0], hi[1], hi[2], hi[3]);
                }
            }
            if (Codes::kNan) b.any_bad[wave] = __ballot(bad_here != 0) != 0;
        };
        if (k_begin < k_end) {
            store(buf[0], k_begin);
            __builtin_amdgcn_sched_barrier(0);
            load(k_begin + kKeys < k_end ? k_begin + kKeys : k_begin);
        }
        __syncthreads();
        int bi = 0;
        for (int key = k_begin; key < k_end; key += kKeys, bi ^= 1) {
            const Buf& b = buf[bi];
            if (!idle) {
#pragma unroll
                for (int u = 0; u < kSub; ++u) {
                    const int sub = kWK == 2 ? wk : u, k32 = key + 32 * sub;
                    if (k32 >= lim_w) continue;  // uniform: nothing that the wave's rows see
                    const int lane = (kShort ? here(tid) : tid) & 63, h = lane >> 5;
                    f32x16 st = f32x16{};
#pragma unroll
                    for (int s = 0; s < kSteps; ++s) {
                        const h8 kf = b.k[(sub * kSteps + s) * 64 + lane];
#pragma unroll
                        for (int p = 0; p < kPlanes; ++p)
                            st = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, q[p][s], st, 0, 0, 0);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    float t[16];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int k4 = 32 * sub + 8 * c + 4 * h;
                        const f32x4 ck = *reinterpret_cast<const f32x4*>(&b.ck[k4]);
                        const f32x4 ls = *reinterpret_cast<const f32x4*>(&b.lsv[k4]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) t[4 * c + e] = fmaf(st[4 * c + e] * rq, ck[e], ls[e]);
                    }
                    // (log2 sv = -inf alone would not keep a key without a place from a row of NaN scores)
                    const uint32_t lie = __builtin_amdgcn_readfirstlane(b.lie[sub]);
                    const bool slow = k32 + 32 > all_w || lie != ~0u;  // uniform
                    if (slow) {
                        const uint32_t window = (seen_from(a, it, t_row, k32) & lie) >> (4 * h);
#pragma unroll
                        for (int e = 0; e < 16; ++e) t[e] = window >> (8 * (e >> 2) + (e & 3)) & 1 ? t[e] : -INFINITY;
                    }
                    float top = t[0];
#pragma unroll
                    for (int e = 1; e < 16; ++e) top = fmaxf(top, t[e]);
                    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
                    top = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) - kPShift;
                    if (__ballot(top > m + kPSlack)) {
                        top = top > m + kPSlack ? top : m;
                        const float ref = top == -INFINITY ? 0.f : top;
                        const float alpha = exp2_hw(m - ref);
                        l *= alpha;
#pragma unroll
                        for (int c = 0; c < kCols; ++c) o[c] *= alpha;
                        m = top;
                    }
                    const float ref = m == -INFINITY ? 0.f : m;
                    h8 pf[2][2];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const f32x4 rv = *reinterpret_cast<const f32x4*>(&b.rsv[32 * sub + 8 * c + 4 * h]);
#pragma unroll
                        for (int e = 4 * c; e < 4 * c + 4; ++e) {
                            const float p = exp2_hw(t[e] - ref);
                            l = fmaf(p, rv[e & 3], l);
                            _Float16 hi, lo;
                            to_planes<2>(p, hi, lo);
                            pf[e >> 3][0][e & 7] = hi;
                            pf[e >> 3][1][e & 7] = lo;
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
                        for (int c = 0; c < kCols; ++c) {
                            const h8 vf = b.v[((2 * sub + t2) * kCols + c) * 64 + lane];
#pragma unroll
                            for (int p = 0; p < 2; ++p)
                                o[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pf[t2][p], o[c], 0, 0, 0);
                        }
                    if (Codes::kNan && key + kKeys > all_b &&
                        (b.any_bad[0] | b.any_bad[1] | b.any_bad[2] | b.any_bad[3])) {
                        const int half = here(h);
                        const uint32_t window = seen_from(a, it, t_row, k32);
                        for (int k2 = 0; k2 < 32; ++k2) {
                            if (!(window >> k2 & 1)) continue;  // (keys past the length hold no codes here)
#pragma unroll
                            for (int c = 0; c < kCols; ++c) {
                                const uint32_t w = *reinterpret_cast<const uint32_t*>(
                                    &b.bad[(32 * sub + k2) * kQuads + 8 * c + 4 * half]);
#pragma unroll
                                for (int e = 0; e < 16; ++e)  // element 16 h + 4 (e % 4) + e / 4
                                    o[c][e] = w >> (8 * (e & 3) + (e >> 2)) & 1 ? NAN : o[c][e];
                            }
                        }
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            if (key + kKeys < k_end) {
                store(buf[bi ^ 1], key + kKeys);
                load(key + 2 * kKeys < k_end ? key + 2 * kKeys : key);  // past the end: this turn again, never used
            }
            __syncthreads();
        }

        // the row's two lanes, then the two key groups
        {
            const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
            l = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
        }
        const int tid2 = here(tid), row2 = 32 * wq + (tid2 & 31), h2 = (tid2 >> 5) & 1;
        float f = 1.0f;
        if constexpr (kWK == 2) {
            if (h2 == 0) m_lds[wave][tid2 & 31] = m;
            __syncthreads();
            const float top = fmaxf(m, m_lds[wave ^ kWQ][tid2 & 31]);
            f = m == -INFINITY ? 0.f : exp2_hw(m - top);
            l *= f;
            m = top;
            if (wk == 1 && h2 == 0) l_lds[row2] = l;
        }
#pragma unroll
        for (int w = kWK - 1; w >= 0; --w) {  // (the buffers are free since the loop's last barrier)
            if (w == wk) {
#pragma unroll
                for (int c = 0; c < kCols; ++c)
#pragma unroll
                    for (int b = 0; b < 4; ++b) {  // elements 32 c + 16 h + 4 b + e / 4 ..
                        f32x4* p = reinterpret_cast<f32x4*>(&rows[row2 * kORow + 32 * c + 16 * h2 + 4 * b]);
                        f32x4 x = f32x4{o[c][b], o[c][4 + b], o[c][8 + b], o[c][12 + b]} * f;
                        if (w != kWK - 1) x += *p;
                        *p = x;
                    }
            }
            __syncthreads();
        }
        const bool whole = u_count == it.units;
        const int64_t slot = (2 * static_cast<int64_t>(blockIdx.x) + (first_share ? 0 : 1)) * kTile;
        if (kWK == 2 && wk == 0) l += l_lds[row2];
        if (wk == 0 && h2 == 0 && row2 < valid) {
            if (whole) {
                l_lds[row2] = l;
            } else {
                float* pml = a.part + 2 * static_cast<int64_t>(a.blocks) * (kTile * kDP) + 2 * (slot + row2);
                pml[0] = m;
                pml[1] = l;
            }
        }
        __syncthreads();
#pragma unroll 1
        for (int i = tid2; i < valid * (kDP / 8); i += kAttBlock) {
            const int row = i / (kDP / 8), d0 = 8 * (i % (kDP / 8));
            const f32x4* p = reinterpret_cast<const f32x4*>(&rows[row * kORow + d0]);
            if (!whole) {
                f32x4* po = reinterpret_cast<f32x4*>(a.part + (slot + row) * kDP + d0);
                po[0] = p[0];
                po[1] = p[1];
            } else if (d0 < a.d) {
                const float sum = l_lds[row];
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = sum == 0.f ? 0.f : p[j >> 2][j & 3] / sum;
                const int64_t dst = row_at(row, static_cast<int64_t>(a.heads) * a.group * a.d, a.d) + d0;
                if (a.out_vec) {
                    store_8(a.out, dst, a.dtype, x);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (d0 + j < a.d) store_elem(a.out, dst + j, a.dtype, x[j]);
                }
            }
        }
        __syncthreads();
        first_share = false;
        at += u_count;
    }
    zero_strays(a, threadIdx.x);
}

// ------------------------------------------------------------------ host
struct AttPlan {
    int tile, blocks;  // rows of a tile
    int64_t items;     // at most
    bool split;
    int64_t bytes;
};

// Rows of a tile by the most that a sequence's head can have: 16 and 32 on the kernel whose waves take
// their keys straight from memory, 64 and 128 on the one that shares converted keys (see there).
// A block for each item, and no join, where sequences are short: up to four units, of 16-row tiles (1 token, 32 on 8 heads
// of 128, bf16: 13.4 us a call for 500 keys against 17.2, 13.7 for 240 against 16.9, 64 sequences of 500 19.5 against 22.0; of
// six units 15.8 against 16.8, of eight 18.4 against 16.8) or of enough items to fill the chip (16 sequences of 200 tokens and 500
// keys, 8 heads: 38 against 44.5; one of them: 36 against 20); up to eight units of enough items for two rounds (64 such
// sequences of 1000 keys: 141 against 161), whose unequal lengths even out.  Else split along the keys over the blocks that
// the chip holds at once (two per CU, one of the 32-row tiles).
int att_plan(const char* what, const tq_kv_cache* c, const tq_kv_batch* b, int64_t group, AttPlan* p) {
    TQ_REQUIRE(b->max_tokens * group <= kKvMaxRows, "%s: %lld rows of a sequence's head", what,
               (long long)(b->max_tokens * group));
    const int64_t rows = b->max_tokens * group;
    p->tile = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
    const int64_t tile = p->tile;
    int64_t tiles = b->batch * ((rows + tile - 1) / tile);
    if (b->offsets) tiles = tiles < b->tokens * group / tile + b->batch ? tiles : b->tokens * group / tile + b->batch;
    p->items = tiles * c->heads;
    const int64_t units = (b->table_pages * c->page + kUnit - 1) / kUnit;
    TQ_REQUIRE(p->items * (units > 0 ? units : 1) < (int64_t(1) << 31), "%s: %lld heads and tiles of %lld keys", what,
               (long long)p->items, (long long)(b->table_pages * c->page));
    TQ_REQUIRE(p->items <= kMaxBlocks, "%s: %lld heads and tiles are more than %lld blocks", what, (long long)p->items,
               (long long)kMaxBlocks);
    const int64_t cus = device_cu_count(), fit = cus * (tile == 32 ? 1 : 2);
    p->split = units > (p->items >= 2 * fit ? 8 : tile == 16 || p->items >= cus ? 4 : 1);
    p->blocks = static_cast<int>(!p->split || fit < p->items * units ? (p->split ? fit : p->items) : p->items * units);
    p->bytes = p->split ? 2 * static_cast<int64_t>(p->blocks) * tile * (kv_row(c->head_dim) + 2) * 4 : 0;
    return TQ_OK;
}

template <int kDP, int kTile, class Codes, int kPlanes>
int launch_attention(const AttArg& a, const AttPlan& p, hipStream_t st) {
    clear_error();
    if constexpr (kTile <= 32)
        k_kv_attention<kDP, kTile / 16, Codes, kPlanes><<<p.blocks, kAttBlock, 0, st>>>(a);
    else
        k_kv_attention_rows<kDP, kTile / 32, Codes, kPlanes><<<p.blocks, kAttBlock, 0, st>>>(a);
    return check_launch("tq_kv_attention");
}

// a block for each row where an item has many shares
template <int kDP, int kTile>
int launch_join(const AttArg& a, const AttPlan& p, hipStream_t st) {
    constexpr int kG = kDP <= 32 ? 8 : kDP <= 64 ? 16 : 32, kRows = kAttBlock / kG;
    const int64_t rows = std::min<int64_t>(static_cast<int64_t>(a.b.max_tokens) * a.group, kTile);
    const unsigned items = static_cast<unsigned>(p.items);
    if (p.blocks >= 16 * p.items)
        k_kv_attention_join<kDP, kTile, true><<<dim3(items, static_cast<unsigned>(rows)), kAttBlock, 0, st>>>(a);
    else
        k_kv_attention_join<kDP, kTile, false>
            <<<dim3(items, static_cast<unsigned>((rows + kRows - 1) / kRows)), kAttBlock, 0, st>>>(a);
    return check_launch("tq_kv_attention");
}

template <int kDP, int kTile, class Codes>
int launch_attention_tile(const AttArg& a, const AttPlan& p, hipStream_t st) {
    const int rc = a.dtype == TQ_DT_F32 ? launch_attention<kDP, kTile, Codes, 2>(a, p, st)
                                        : launch_attention<kDP, kTile, Codes, 1>(a, p, st);
    return rc != TQ_OK || !p.split ? rc : launch_join<kDP, kTile>(a, p, st);
}

template <int kDP, class Codes>
int launch_attention_rows(const AttArg& a, const AttPlan& p, hipStream_t st) {
    switch (p.tile) {
    case 16: return launch_attention_tile<kDP, 16, Codes>(a, p, st);
    case 32: return launch_attention_tile<kDP, 32, Codes>(a, p, st);
    case 64: return launch_attention_tile<kDP, 64, Codes>(a, p, st);
    default: return launch_attention_tile<kDP, 128, Codes>(a, p, st);
    }
}

template <class Codes>
int launch_attention_dim(const AttArg& a, const AttPlan& p, hipStream_t st) {
    switch (kv_row(a.d)) {
    case 32: return launch_attention_rows<32, Codes>(a, p, st);
    case 64: return launch_attention_rows<64, Codes>(a, p, st);
    case 96: return launch_attention_rows<96, Codes>(a, p, st);
    default: return launch_attention_rows<128, Codes>(a, p, st);
    }
}

}  // namespace
}  // namespace tq

extern "C" {

int64_t tq_kv_attention_workspace_bytes(const tq_kv_cache* cache, const tq_kv_batch* batch, int64_t q_heads) {
    using namespace tq;
    if (!cache || !batch || cache->heads < 1 || cache->heads > 65535 || q_heads < 0 || q_heads > 65535 || q_heads % cache->heads ||
        cache->head_dim < 1 || cache->head_dim > kKvMaxHeadDim || cache->page < 16 || cache->page % 16 || cache->page > kKvMaxPage ||
        batch->batch < 0 || batch->batch > kKvMaxRows || batch->max_tokens < 0 || batch->max_tokens > kKvMaxRows ||
        batch->tokens < 0 || batch->tokens > kKvMaxRows || batch->table_pages < 0 || batch->table_pages > kKvMaxRows / cache->page ||
        (!batch->offsets && batch->tokens != batch->batch * batch->max_tokens))
        return -1;
    if (batch->batch == 0 || batch->tokens == 0 || batch->max_tokens == 0 || q_heads == 0) return 0;
    AttPlan p;
    return att_plan("tq_kv_attention_workspace_bytes", cache, batch, q_heads / cache->heads, &p) == TQ_OK ? p.bytes : -1;
}

int tq_kv_attention(const tq_kv_cache* cache, const tq_kv_batch* batch, const tq_heads* q, int dtype, const int32_t* tree,
                    int64_t tree_words, float scale, void* workspace, int64_t workspace_bytes, void* out,
                    tq_stream_t stream) {
    using namespace tq;
    static const char* what = "tq_kv_attention";
    AttArg a{};
    int rc = kv_check(what, cache, batch, &a.b);
    if (rc != TQ_OK) return rc;
    TQ_REQUIRE(q, "%s: null q", what);
    if ((rc = kv_check_heads(what, "q", q, q->heads, cache->head_dim, dtype)) != TQ_OK) return rc;
    TQ_REQUIRE(q->heads % cache->heads == 0, "%s: %lld query heads are no multiple of %lld key heads", what,
               (long long)q->heads, (long long)cache->heads);
    TQ_REQUIRE(!tree || (tree_words >= 1 && tree_words <= kKvMaxRows && 32 * tree_words >= batch->max_tokens),
               "%s: %lld tree words for %lld new tokens", what, (long long)tree_words, (long long)batch->max_tokens);
    TQ_REQUIRE(aligned(tree, 4), "%s: tree is not 4-byte aligned", what);
    if (batch->tokens == 0 || batch->batch == 0 || batch->max_tokens == 0 || q->heads == 0) return TQ_OK;
    TQ_REQUIRE(q->data && out, "%s: null q or out", what);
    const int64_t size = dtype == TQ_DT_F32 ? 4 : 2, group = q->heads / cache->heads;
    TQ_REQUIRE(aligned(out, size), "%s: out is not aligned to its elements", what);
    AttPlan p;
    if ((rc = att_plan(what, cache, batch, group, &p)) != TQ_OK) return rc;
    TQ_REQUIRE(p.bytes == 0 || (workspace && aligned(workspace, 256) && workspace_bytes >= p.bytes),
               "%s: workspace of %lld bytes, %lld needed (256-byte aligned)", what, (long long)workspace_bytes,
               (long long)p.bytes);
    a.k = static_cast<const uint8_t*>(cache->k);
    a.k_scale = cache->k_scale;
    a.v = static_cast<const uint8_t*>(cache->v);
    a.v_scale = cache->v_scale;
    a.q = q->data;
    a.q_token = q->token_stride;
    a.q_head = q->head_stride;
    a.tree = tree;
    a.tree_words = tree_words;
    a.out = out;
    a.part = p.split ? static_cast<float*>(workspace) : nullptr;
    a.heads = static_cast<int>(cache->heads);
    a.group = static_cast<int>(group);
    a.d = static_cast<int>(cache->head_dim);
    a.dtype = dtype;
    a.blocks = p.blocks;
    a.q_vec = aligned(q->data, 16) && cache->head_dim % 8 == 0 && q->token_stride * size % 16 == 0 &&
              q->head_stride * size % 16 == 0;
    a.out_vec = aligned(out, 16) && cache->head_dim % 8 == 0;
    a.scale2 = scale * 1.4426950408889634f;
    a.by_group = FastDiv(static_cast<uint32_t>(group));
    return cache->codes == TQ_QINT8 ? launch_attention_dim<CodesI8>(a, p, as_hip(stream))
                                    : launch_attention_dim<CodesFp8>(a, p, as_hip(stream));
}

}  // extern "C"
