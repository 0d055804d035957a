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
// maximum of t, P_j = 2^(t_j - max + 14) = p_j sv_j needs no normalising to fit f16's
// range whatever the scales, and the sum takes P_j / sv_j.  f32 rows use two f16 planes of
// q (scaled by a power of two for each row) and P, 22 bits; 16-bit rows one (11 bits: an
// eighth of a bf16 output's rounding).
//
// Work is split along the keys by units of 128: the units of all sequences, heads and row
// tiles in one line, cut into equal shares for a grid that fits the chip at once, whatever the lengths.  A share that
// is not a whole (sequence, head, tile) leaves maximum, sum and O in the workspace, and a second launch joins them in order.
#include <cmath>

#include "tq_kv.h"

namespace tq {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

constexpr int kAttBlock = 256, kAttWaves = kAttBlock / kWave;
constexpr int kStep = 32;                    // keys of a wave's step
constexpr int kUnit = kAttWaves * kStep;     // keys of a unit
constexpr float kPShift = 14.0f;             // P in [0, 2^14]: small probabilities stay normal f16 numbers

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

// ------------------------------------------------------------------ the line of work
// 64 sequences at a time, one in each lane: rows, keys and units, with the running totals of
// items ((head, tile) pairs) and units.
struct SeqLane {
    int first, rows, len, base;  // first row of q; new tokens; keys; place of the first new token
    int tiles, units, items;
    int items_end, units_end;    // inclusive totals within the 64
};

__device__ __forceinline__ int scan64(int v, int lane) {
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
        const int u = __shfl_up(v, s);
        v += lane >= s ? u : 0;
    }
    return v;
}

template <int kTile>
__device__ __forceinline__ SeqLane seq_lane(const AttArg& a, int seq0, int lane) {
    SeqLane s{};
    const int seq = seq0 + lane;
    if (seq < a.b.batch) {
        int first = a.b.offsets ? a.b.offsets[seq] : seq * a.b.max_tokens;
        const int last = a.b.offsets ? a.b.offsets[seq + 1] : first + a.b.max_tokens;
        const bool ok = first >= 0 && last <= a.b.tokens && last > first && last - first <= a.b.max_tokens;
        s.first = first;
        s.rows = ok ? last - first : 0;
        const int length = min(max(a.b.lengths[seq], 0), 1 << 30);
        s.len = min(length, a.b.cap);
        s.base = length - s.rows;
        s.tiles = (s.rows * a.group + kTile - 1) / kTile;
        s.units = max((s.len + kUnit - 1) / kUnit, 1);
        s.items = s.tiles * a.heads;
    }
    if (a.b.batch == 1) {  // every lane past the first holds nothing
        s.items_end = readlane(s.items, 0);
        s.units_end = readlane(s.items * s.units, 0);
    } else {
        s.items_end = scan64(s.items, lane);
        s.units_end = scan64(s.items * s.units, lane);
    }
    return s;
}

struct Totals {
    int items, units;
};

template <int kTile>
__device__ __forceinline__ Totals all_work(const AttArg& a, int lane) {
    Totals t{0, 0};
    for (int s0 = 0; s0 < a.b.batch; s0 += 64) {
        const SeqLane s = seq_lane<kTile>(a, s0, lane);
        t.items += readlane(s.items_end, 63);
        t.units += readlane(s.units_end, 63);
    }
    return t;
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
__device__ __forceinline__ Item pick(const SeqLane& s, int seq0, int items0, int units0, int at, int tiles_hint) {
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
        return pick<kByUnit>(s0, 0, 0, 0, at, 0);
    }
    int items = 0, units = 0;
    for (int seq = 0; seq < a.b.batch; seq += 64) {
        const SeqLane s = seq_lane<kTile>(a, seq, lane);
        const int ni = readlane(s.items_end, 63), nu = readlane(s.units_end, 63);
        if (at < (kByUnit ? units + nu : items + ni)) return pick<kByUnit>(s, seq, items, units, at, 0);
        items += ni;
        units += nu;
    }
    return Item{};
}

// ------------------------------------------------------------------ arithmetic
__device__ __forceinline__ f32x4 mfma_f16(h8 a, h8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
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
// 8 adjacent elements, 16-byte aligned
__device__ __forceinline__ void load_8(const void* p, int64_t i, int dtype, float* x) {
    if (dtype == TQ_DT_F32) {
        const f32x4* s = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i);
        const f32x4 a = s[0], b = s[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] = a[e];
            x[4 + e] = b[e];
        }
        return;
    }
    const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t u = w[e];  // (a bit cast of the vector's element itself takes element 0)
        if (dtype == TQ_DT_BF16) {
            x[2 * e] = __uint_as_float(u << 16);
            x[2 * e + 1] = __uint_as_float(u & 0xFFFF0000u);
        } else {
            const h2 h = __builtin_bit_cast(h2, u);
            x[2 * e] = static_cast<float>(h.x);
            x[2 * e + 1] = static_cast<float>(h.y);
        }
    }
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

    const SeqLane s0 = seq_lane<kTile>(a, 0, lane);
    int at, end;
    if (a.part) {
        const int units = a.b.batch <= 64 ? readlane(s0.units_end, 63) : all_work<kTile>(a, lane).units;
        const Shares sh(units, a.blocks);
        at = sh.begin(blockIdx.x);
        end = sh.begin(blockIdx.x + 1);
    } else {
        at = 0;
        end = 1;
    }
    bool first_share = true;
    while (at < end) {
        const Item it = a.part ? find_item<kTile, true>(a, s0, at, lane) : find_item<kTile, false>(a, s0, blockIdx.x, lane);
        if (!it.ok) return;
        const int u_first = a.part ? at - it.unit0 : 0;
        const int u_count = a.part ? min(it.units - u_first, end - at) : it.units;
        const int n_rows = it.rows * a.group;

        // what the tile's rows see: all keys before `all`, none from `lim` on
        const int t_first = static_cast<int>(a.by_group.div(it.tile * kTile));
        const int t_last = static_cast<int>(a.by_group.div(min(it.tile * kTile + kTile, n_rows) - 1));
        const int lim = a.tree ? it.len : min(it.base + t_last + 1, it.len);
        const int all = a.tree ? min(it.base, it.len) : min(it.base + t_first + 1, it.len);

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
        float m[kNQ], l[kNQ];  // m: the running maximum less kPShift; l: of this lane's keys
#pragma unroll
        for (int n = 0; n < kNQ; ++n) {
            m[n] = -INFINITY;
            l[n] = 0.f;
#pragma unroll
            for (int t = 0; t < kVT; ++t) o[n][t] = f32x4{};
        }

        const int k_end = min((u_first + u_count) * kUnit, lim);
        const int k_begin = u_first * kUnit + wave * kStep;
        const int32_t* table = a.b.table + static_cast<int64_t>(it.seq) * a.b.table_stride;

        // Where the 16 keys from `key` lie (a page holds whole sixteens): row of the cache's
        // [pages, heads, page], and whether they lie anywhere.
        auto place16 = [&](int key, bool& ok) -> int64_t {
            ok = key < it.len;
            const int i = static_cast<int>(a.b.by_page.div(static_cast<uint32_t>(ok ? key : 0)));
            int page = it.len > 0 ? table[i] : 0;
            if (page < 0 || page >= a.b.pages) {
                page = 0;
                ok = false;
            }
            return (static_cast<int64_t>(page) * a.heads + it.head) * a.b.page + (ok ? key - i * a.b.page : 0);
        };

        KBytes<kDP> kb[2];
        VBytes<kDP> vb[8];
        f32x4 ks[2], vs[2];
        bool ok_k[2], ok_v[2];
        auto load_k = [&](int key) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int64_t row = place16(key + 16 * i, ok_k[i]);
                kb[i].load(a.k + row * kDP + (r * kDP + kRun * g));
                ks[i] = *reinterpret_cast<const f32x4*>(a.k_scale + row + 4 * g);
            }
        };
        auto load_v = [&](int key) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int64_t row = place16(key + 16 * i, ok_v[i]);
                const uint8_t* p = a.v + row * kDP + 4 * g * kDP;
#pragma unroll
                for (int j = 0; j < 4; ++j) vb[4 * i + j].load(p + j * kDP, r);
                vs[i] = *reinterpret_cast<const f32x4*>(a.v_scale + row + 4 * g);
            }
        };
        if (k_begin < k_end) {
            load_k(k_begin);
            load_v(k_begin);
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
            h8 pf[kNQ][kPlanes];
#pragma unroll
            for (int n = 0; n < kNQ; ++n) {
                float t[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) t[j] = fmaf(st[j >> 2][n][j & 3] * rq[n], ck[j >> 2][j & 3], lsv[j]);
                if (slow) {
                    uint32_t bits = 0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int kk = key + 16 * (j >> 2) + 4 * g + (j & 3);
                        bool see;
                        if (a.tree) {
                            const int jj = kk - it.base;
                            see = kk < it.len && jj < it.rows;
                            if (see && jj >= 0 && jj < 32 * a.tree_words)
                                see = (a.tree[(it.first + static_cast<int64_t>(t_row[n])) * a.tree_words + (jj >> 5)] >>
                                       (jj & 31)) & 1;
                            else if (jj >= 0)
                                see = false;
                        } else {
                            see = kk < min(it.base + t_row[n] + 1, it.len);
                        }
                        see = see && (j < 4 ? seen0 : seen1);
                        t[j] = see ? t[j] : -INFINITY;
                        bits |= see ? 1u << j : 0u;
                    }
                    seen[n] = bits;
                }
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, t[j]);
                top = fmaxf(m[n], over_groups(top, OpMax{}) - kPShift);
                const float ref = top == -INFINITY ? 0.f : top;
                if (__ballot(top != m[n])) {
                    const float alpha = exp2_hw(m[n] - ref);
                    l[n] *= alpha;
#pragma unroll
                    for (int v = 0; v < kVT; ++v) o[n][v] *= alpha;
                    m[n] = top;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float p = exp2_hw(t[j] - ref);
                    l[n] = fmaf(p, rsv[j], l[n]);
                    _Float16 hi, lo;
                    to_planes<kPlanes>(p, hi, lo);
                    pf[n][0][j] = hi;
                    if constexpr (kPlanes == 2) pf[n][1][j] = lo;
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
                            vb[j].w[w] = x & ~((top_bits >> 7) * 0xFFu);
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
                    for (int p = 0; p < kPlanes; ++p) {
                        o[n][v] = mfma_f16(f0, pf[n][p], o[n][v]);
                        o[n][v + 1] = mfma_f16(f1, pf[n][p], o[n][v + 1]);
                    }
            }
            load_v(next);
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
}

// Joins the shares of the items that several blocks worked on: a wave for each row, 2 kDP / 128
// elements of it in each lane.
template <int kDP, int kNQ>
__global__ __launch_bounds__(kAttBlock) void k_kv_attention_join(AttArg a) {
    constexpr int kTile = 16 * kNQ, kE = (kDP + 63) / 64;
    const int lane = threadIdx.x & 63;
    const int row = blockIdx.y * kAttWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const SeqLane s0 = seq_lane<kTile>(a, 0, lane);
    const Item it = find_item<kTile, false>(a, s0, blockIdx.x, lane);
    if (!it.ok || it.tile * kTile + row >= it.rows * a.group) return;
    const int units = a.b.batch <= 64 ? readlane(s0.units_end, 63) : all_work<kTile>(a, lane).units;
    const Shares sh(units, a.blocks);
    const int b0 = sh.of(it.unit0), b1 = sh.of(it.unit0 + it.units - 1);
    if (b0 == b1) return;  // one block had it all
    const float* ml = a.part + 2 * static_cast<int64_t>(a.blocks) * (kTile * kDP);
    const int64_t skip = sh.begin(b0) == it.unit0 ? 0 : 1;
    auto slot = [&](int b) { return 2 * static_cast<int64_t>(b) + (b == b0 ? skip : 0); };
    float top = -INFINITY;
    for (int b = b0 + lane; b <= b1; b += 64) top = fmaxf(top, ml[(slot(b) * kTile + row) * 2]);
    top = wave_max(top);
    float sum = 0.f, x[kE] = {};
    for (int b = b0; b <= b1; ++b) {
        const int64_t s = slot(b);
        const float mb = ml[(s * kTile + row) * 2], lb = ml[(s * kTile + row) * 2 + 1];
        const float f = mb == -INFINITY ? 0.f : exp2_hw(mb - top);
        sum = fmaf(lb, f, sum);
        const float* po = a.part + (s * kTile + row) * kDP;
#pragma unroll
        for (int e = 0; e < kE; ++e) {
            const int d = lane + 64 * e;
            if (d < kDP) x[e] = fmaf(po[d], f, x[e]);
        }
    }
    const int rr = it.tile * kTile + row, t = static_cast<int>(a.by_group.div(rr));
    const int64_t dst = ((it.first + static_cast<int64_t>(t)) * (static_cast<int64_t>(a.heads) * a.group) +
                         static_cast<int64_t>(it.head) * a.group + (rr - t * a.group)) * a.d;
#pragma unroll
    for (int e = 0; e < kE; ++e) {
        const int d = lane + 64 * e;
        if (d < a.d) store_elem(a.out, dst + d, a.dtype, sum == 0.f ? 0.f : x[e] / sum);
    }
}

// ------------------------------------------------------------------ host
struct AttPlan {
    int nq, blocks;
    int64_t items;  // at most
    bool split;
    int64_t bytes;
};

// 16 rows per tile where no sequence has more, 32 beyond (a tile's keys are read and
// converted once for all of its rows).  Split wherever a sequence can have more than a unit
// of keys, over the blocks that the chip holds at once (two per CU, one of the 32-row tiles).
int att_plan(const char* what, const tq_kv_cache* c, const tq_kv_batch* b, int64_t group, AttPlan* p) {
    TQ_REQUIRE(b->max_tokens * group <= kKvMaxRows, "%s: %lld rows of a sequence's head", what,
               (long long)(b->max_tokens * group));
    const int64_t rows = b->max_tokens * group;
    p->nq = rows <= 16 ? 1 : 2;
    const int64_t tile = 16 * p->nq;
    int64_t tiles = b->batch * ((rows + tile - 1) / tile);
    if (b->offsets) tiles = tiles < b->tokens * group / tile + b->batch ? tiles : b->tokens * group / tile + b->batch;
    p->items = tiles * c->heads;
    const int64_t units = (b->table_pages * c->page + kUnit - 1) / kUnit;
    TQ_REQUIRE(p->items * (units > 0 ? units : 1) < (int64_t(1) << 31), "%s: %lld heads and tiles of %lld keys", what,
               (long long)p->items, (long long)(b->table_pages * c->page));
    p->split = units > 1;
    const int64_t fit = static_cast<int64_t>(device_cu_count()) * (p->nq == 2 ? 1 : 2);
    p->blocks = static_cast<int>(!p->split || fit < p->items * units ? (p->split ? fit : p->items) : p->items * units);
    p->bytes = p->split ? 2 * static_cast<int64_t>(p->blocks) * tile * (kv_row(c->head_dim) + 2) * 4 : 0;
    return TQ_OK;
}

template <int kDP, int kNQ, class Codes>
int launch_attention(const AttArg& a, const AttPlan& p, hipStream_t st) {
    clear_error();
    if (a.dtype == TQ_DT_F32)
        k_kv_attention<kDP, kNQ, Codes, 2><<<p.blocks, kAttBlock, 0, st>>>(a);
    else
        k_kv_attention<kDP, kNQ, Codes, 1><<<p.blocks, kAttBlock, 0, st>>>(a);
    const int rc = check_launch("tq_kv_attention");
    if (rc != TQ_OK || !p.split) return rc;
    const int64_t rows = static_cast<int64_t>(a.b.max_tokens) * a.group;
    const dim3 grid(static_cast<unsigned>(p.items), static_cast<unsigned>(((rows < 16 * kNQ ? rows : 16 * kNQ) + kAttWaves - 1) / kAttWaves));
    k_kv_attention_join<kDP, kNQ><<<grid, kAttBlock, 0, st>>>(a);
    return check_launch("tq_kv_attention");
}

template <int kDP, class Codes>
int launch_attention_rows(const AttArg& a, const AttPlan& p, hipStream_t st) {
    return p.nq == 1 ? launch_attention<kDP, 1, Codes>(a, p, st) : launch_attention<kDP, 2, Codes>(a, p, st);
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
    if (!cache || !batch || cache->heads < 1 || q_heads < 0 || q_heads % cache->heads || cache->page < 16 ||
        batch->batch < 0 || batch->max_tokens < 0 || batch->tokens < 0 || batch->table_pages < 0)
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
    a.scale2 = scale * 1.4426950408889634f;
    a.by_group = FastDiv(static_cast<uint32_t>(group));
    return cache->codes == TQ_QINT8 ? launch_attention_dim<CodesI8>(a, p, as_hip(stream))
                                    : launch_attention_dim<CodesFp8>(a, p, as_hip(stream));
}

}  // extern "C"
