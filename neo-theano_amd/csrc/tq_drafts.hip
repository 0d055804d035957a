// tq_drafts.hip -- which drafted tokens the target's probabilities accept, and the token that follows.
//
// Speculative sampling over trees.  At an accepted token c with target probabilities p and draft
// probabilities q, its children are tried in order.  After k children were turned down
//   left_k = max(p - a_k q, 0),   a_0 = 0, W_0 = 1,   a_{k+1} = a_k + W_k,   W_k = sum left_k,
// and child x is accepted if u q(x) W_k < p(x) - a_k q(x): the residuals max(r - q, 0) / sum of repeated
// rejection are left_k / W_k, since their clamps at zero nest.  Without q a child is a point mass: left_k is
// p without the tokens tried, W_k = 1 - their sum.  The token that follows is drawn from left at the last
// accepted token: the lowest i whose running sum exceeds final * sum left.
//
// Everything is compared and summed in f64 (the running sum is compared with a number next to a border).
// The bytes are one row of p (and of q) for a sequence; what costs is the chain of dependent loads
// (token -> its probability -> the row -> the sums -> the chosen ones), so a row is cut into shares that blocks
// sum side by side, a sum for each 256 probabilities (a wave's load), and a second launch picks one of these sums and looks into
// its 256 again.
#include <algorithm>

#include "tq_kv.h"

namespace tq {
namespace {

constexpr int kBlock = 256;
constexpr int kWalkBlock = 1024;
constexpr int kMaxShare = 8192;  // probabilities of a share
constexpr int kSegment = 256;    // of a sum: four for each lane of a wave

template <int kType>
struct Prob;
template <>
struct Prob<TQ_DT_F32> {
    typedef float type;
};
template <>
struct Prob<TQ_DT_BF16> {
    typedef __bf16 type;
};
template <>
struct Prob<TQ_DT_F16> {
    typedef _Float16 type;
};

// Where the walk over a sequence's drafts ended.
struct State {
    double a;     // share of q that is gone
    int node;     // last accepted row of the sequence; -1: the sequence has no rows
    int kept;
    int summed;   // the sums are there already
};

struct DraftArg {
    const int64_t* tokens;
    const void* target;
    const void* draft;
    int64_t target_stride, draft_stride;
    const int32_t* parents;
    const float* accept;
    const float* final;
    const int32_t* offsets;
    int batch, max_tokens, rows;
    int vocab, share, shares;  // share: probabilities of a block, shares * share >= vocab
    FastDiv by_shares;
    int32_t* path;
    int32_t* kept;
    int64_t* next;
    State* state;   // [batch]
    double* sums;   // [batch, segments], segments = shares * share / kSegment
};

struct Span {
    int first, count;
};
__device__ __forceinline__ Span span_of(const DraftArg& a, int seq) {
    const int first = a.offsets ? a.offsets[seq] : seq * a.max_tokens;
    const int last = a.offsets ? a.offsets[seq + 1] : first + a.max_tokens;
    const bool fits = first >= 0 && last <= a.rows && last > first && last - first <= a.max_tokens;
    return Span{first, fits ? last - first : 0};
}

// A probability as it counts: NaN and negative ones are 0.
template <class T>
__device__ __forceinline__ double counted(T x) {
    const float v = static_cast<float>(x);
    return static_cast<double>(v > 0.f ? v : 0.f);
}

template <class T>
__device__ __forceinline__ double at(const void* x, int64_t stride, int row, int64_t token) {
    return counted(static_cast<const T*>(x)[row * stride + token]);
}

// What is left of one token's probability, likewise: a q that is not above 0 takes nothing (the lesser of a number and NaN is
// the number), and what is not above 0 is 0.  The sums of a tree are one CU's VALU work: cutting p and q off beforehand is 3 us more
// for 128256 of them.
template <class T>
__device__ __forceinline__ double left_of(T p, T q, double a) {
    const double x = static_cast<double>(static_cast<float>(p)), y = static_cast<double>(static_cast<float>(q));
    return fmax(fmin(x - a * y, x), 0.0);
}

__device__ __forceinline__ double readlane_f64(double v, int l) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint64_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(b), l));
    const uint64_t hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(b >> 32), l));
    return __builtin_bit_cast(double, hi << 32 | lo);
}

// Walks the drafts of a sequence; whole waves, the result uniform.  path: where the accepted rows go, or null.
// mass(node, a, w): makes w the sum of what is left, called by all of the block's waves alike (only where q is there and a
// node has another child after one that was turned down); false: the walk stops there.
template <class T, class Mass>
__device__ __forceinline__ State walk(const DraftArg& a, Span s, int32_t* path, Mass mass) {
    const int lane = threadIdx.x & 63;
    State st{0.0, s.count > 0 ? 0 : -1, s.count > 0 ? 1 : 0, 1};
    if (path && lane == 0 && s.count > 0) path[0] = 0;
    double w = 1.0;
    bool pending = false;  // a child was turned down and w is not yet that of what is left
    for (int t0 = 1; t0 < s.count; t0 += 64) {
        const int t = t0 + lane;
        const bool there = t < s.count;
        const int row = s.first + (there ? t : 0);
        int parent = there ? (a.parents ? a.parents[row] : t - 1) : -1;
        if (parent >= t) parent = -1;
        const int64_t x = there ? a.tokens[row] : -1;
        const bool known = x >= 0 && x < a.vocab && parent >= 0;
        const double u = there ? static_cast<double>(a.accept[row]) : 0.0;
        const double p = known ? at<T>(a.target, a.target_stride, s.first + parent, x) : 0.0;
        const double q = !known ? 0.0 : a.draft ? at<T>(a.draft, a.draft_stride, s.first + parent, x) : 1.0;
        if (!a.parents) {  // a chain: all tests at once
            const uint64_t turned_down = __ballot(there && !(u * q < p));
            const int fine = turned_down ? __ffsll(static_cast<unsigned long long>(turned_down)) - 1 : min(64, s.count - t0);
            if (path && lane < fine) path[t] = t;
            st.kept += fine;
            st.node += fine;
            if (turned_down) {
                st.a = 1.0;
                return st;
            }
            continue;
        }
        for (int from = 0; from < 64;) {
            const uint64_t children = __ballot(there && parent == st.node && lane >= from);
            if (!children) break;
            const int l = __ffsll(static_cast<unsigned long long>(children)) - 1;
            from = l + 1;
            double px = readlane_f64(p, l);
            const double qx = readlane_f64(q, l), ux = readlane_f64(u, l);
            const int tx = t0 + l;
            bool yes;
            if (a.draft) {
                if (pending && !mass(st.node, st.a, w)) return st;
                pending = false;
                yes = ux * qx * w < px - st.a * qx;
            } else {
                // a token that a sibling was turned down with has nothing left
                const int xl = __builtin_amdgcn_readlane(static_cast<int>(x), l);  // (a known token is below 2^31)
                bool again = there && parent == st.node && lane < l && known && static_cast<int>(x) == xl;
                for (int e0 = 1; e0 < t0; e0 += 64) {
                    const int e = s.first + e0 + lane;
                    again |= a.parents[e] == st.node && e0 + lane > st.node && a.tokens[e] == xl;
                }
                if (__ballot(again)) px = 0.0;
                yes = ux * w < px;
            }
            if (yes) {
                st.node = tx;
                if (path && lane == 0) path[st.kept] = tx;
                ++st.kept;
                st.a = 0.0;
                w = 1.0;
            } else if (a.draft) {
                st.a += w;
                pending = true;
            } else {
                w -= px;
            }
        }
    }
    return st;
}

template <int kCtrl>
__device__ __forceinline__ double dpp64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, static_cast<uint64_t>(dpp_u32<kCtrl>(static_cast<uint32_t>(b >> 32))) << 32 |
                                          dpp_u32<kCtrl>(static_cast<uint32_t>(b)));
}

// Sum over a wave, the same in every lane (lane permutes of the VALU: shuffles through LDS took 11.2 us where these take 9
// for 32 rows of 128256 f32 probabilities of two models).
__device__ __forceinline__ double wave_sum64(double v) {
    v += dpp64<kDppXor1>(v);
    v += dpp64<kDppXor2>(v);
    v += dpp64<kDppHalfMirror>(v);
    v += dpp64<kDppMirror>(v);
    return (readlane_f64(v, 0) + readlane_f64(v, 16)) + (readlane_f64(v, 32) + readlane_f64(v, 48));
}

// Sums over a wave of four values: in lanes 0 to 15 that of v[0], then of v[2], v[1] and v[3] (a fifth of the instructions of four
// sums one by one: a chain over 32768 f32 probabilities of two models by one block 7.4 us, 9.0 one by one; 32 rows of 128256 by 512
// blocks 13.9 and 15.3).
__device__ __forceinline__ double wave_sums4(const double (&v)[4]) {
    auto halves = [](double x, double y) {  // x's sum over both halves in the lower one, y's in the upper
        const uint64_t a = __builtin_bit_cast(uint64_t, x), b = __builtin_bit_cast(uint64_t, y);
        const auto lo = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(a), static_cast<uint32_t>(b), false, false);
        const auto hi = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(a >> 32), static_cast<uint32_t>(b >> 32), false, false);
        return __builtin_bit_cast(double, static_cast<uint64_t>(hi[0]) << 32 | lo[0]) + __builtin_bit_cast(double, static_cast<uint64_t>(hi[1]) << 32 | lo[1]);
    };
    const uint64_t a = __builtin_bit_cast(uint64_t, halves(v[0], v[1])), b = __builtin_bit_cast(uint64_t, halves(v[2], v[3]));
    const auto lo = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(a), static_cast<uint32_t>(b), false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(a >> 32), static_cast<uint32_t>(b >> 32), false, false);
    double s = __builtin_bit_cast(double, static_cast<uint64_t>(hi[0]) << 32 | lo[0]) + __builtin_bit_cast(double, static_cast<uint64_t>(hi[1]) << 32 | lo[1]);
    s += dpp64<kDppXor1>(s);
    s += dpp64<kDppXor2>(s);
    s += dpp64<kDppHalfMirror>(s);
    return s + dpp64<kDppMirror>(s);
}

// Running sums over a wave, the lane's own among them.
__device__ __forceinline__ double wave_running(double v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double y = __shfl_up(v, d);
        if (lane >= d) v += y;
    }
    return v;
}

// Sums of f64 over a block, the same in every thread (and in every call: a fixed order).
template <int kThreads>
__device__ __forceinline__ double block_sum(double v, double* lds) {
    v = wave_sum64(v);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) s += lds[w];
    __syncthreads();
    return s;
}

template <class T>
using Four = T __attribute__((ext_vector_type(4)));
template <class T>
using FourAnywhere = T __attribute__((ext_vector_type(4), aligned(sizeof(T))));  // (one load wherever the row lies)

// Elements i .. i + 3 of a row.
template <class T>
__device__ __forceinline__ Four<T> load4(const T* row, int i) {
    return *reinterpret_cast<const FourAnywhere<T>*>(row + i);
}

// The same with zeros from `end` on.
template <class T>
__device__ __forceinline__ Four<T> load4(const T* row, int i, int end) {
    Four<T> x{};
    if (i + 4 <= end) {
        x = load4<T>(row, i);
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (i + e < end) x[e] = row[i + e];
    }
    return x;
}

// What is left of four.  q: whether y is there; gone: bits of the tokens tried.
template <class T>
__device__ __forceinline__ void left4(Four<T> x, bool q, Four<T> y, double a, uint32_t gone, double (&v)[4]) {
    if (q) {  // (uniform)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = left_of(x[e], y[e], a);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = counted(x[e]);
    }
    if (gone & 15) {  // (few)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = gone >> e & 1 ? 0.0 : v[e];
    }
}

// Sums of what is left of segments `first`, first + step, .. of those from `begin` on, by one wave: four at a time.  gone: the tokens tried,
// or null.
template <class T>
__device__ __forceinline__ void segment_sums(const T* p, const T* q, double a, const uint32_t* gone, int begin, int end, int first, int step,
                                             int segments, double* sums) {
    const int lane = threadIdx.x & 63, row = lane >> 4;
    int g = first;
    for (; g + step < segments; g += 4 * step) {
        Four<T> x[4], y[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = begin + (g + u * step) * kSegment + 4 * lane;
            x[u] = load4<T>(p, i, end);
            y[u] = q ? load4<T>(q, i, end) : Four<T>{};
        }
        double sum[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            sum[u] = 0.0;
            if (g + u * step >= segments) continue;  // (uniform)
            const int at = (g + u * step) * kSegment + 4 * lane;
            double v[4];
            left4<T>(x[u], q != nullptr, y[u], a, gone ? gone[at / 32] >> (at & 31) : 0, v);
            sum[u] = (v[0] + v[1]) + (v[2] + v[3]);
        }
        const double mine = wave_sums4(sum);
        const int seg = g + ((row & 1) * 2 + (row >> 1)) * step;
        if ((lane & 15) == 0 && seg < segments) sums[seg] = mine;
    }
    if (g < segments) {  // one is left
        const int at = g * kSegment + 4 * lane;
        double v[4];
        left4<T>(load4<T>(p, begin + at, end), q != nullptr, q ? load4<T>(q, begin + at, end) : Four<T>{}, a, gone ? gone[at / 32] >> (at & 31) : 0, v);
        const double sum = wave_sum64((v[0] + v[1]) + (v[2] + v[3]));
        if (lane == 0) sums[g] = sum;
    }
}

// Sum of what is left over the whole row, by one block; kU loads of each model in flight for each lane (a block alone at work is
// bound by their latency; without bounds to check where none is near: 8 % of 32 trees over 32768 tokens).
template <class T, int kThreads>
__device__ __forceinline__ double row_mass(const T* p, const T* q, double a, int vocab, double* lds) {
    constexpr int kU = 4, kAll = 4 * kThreads * kU;
    double s = 0.0;
    auto add = [&](const Four<T> (&x)[kU], const Four<T> (&y)[kU]) {
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            double v[4];
            left4<T>(x[u], true, y[u], a, 0, v);
            s += (v[0] + v[1]) + (v[2] + v[3]);
        }
    };
    Four<T> x[kU], y[kU];
    int i = 4 * static_cast<int>(threadIdx.x), from = 0;
    for (; q && from + kAll <= vocab; from += kAll, i += kAll) {
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            x[u] = load4<T>(p, i + 4 * kThreads * u);
            y[u] = load4<T>(q, i + 4 * kThreads * u);
        }
        add(x, y);
    }
    for (; i < vocab; i += kAll) {
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            x[u] = load4<T>(p, i + 4 * kThreads * u, vocab);
            y[u] = q ? load4<T>(q, i + 4 * kThreads * u, vocab) : Four<T>{};
        }
        add(x, y);
    }
    return block_sum<kThreads>(s, lds);
}

template <class T>
__device__ __forceinline__ const T* row_of(const void* x, int64_t stride, int row) {
    return x ? static_cast<const T*>(x) + row * stride : nullptr;
}

// The same by a block's first wave (sixteen that walk side by side take each other's cycles); the others wait for the
// node whose sum is asked for, or for the end.  sum: called by all of the block's waves.
template <class T, class Sum>
__device__ __forceinline__ State walk_by_one(const DraftArg& a, Span s, int32_t* path, State* shared, Sum sum) {
    if (threadIdx.x < 64) {
        State st = walk<T>(a, s, path, [&](int node, double share, double& w) {
            if (threadIdx.x == 0) *shared = State{share, node, 0, 0};
            __syncthreads();
            w = sum(node, share);
            return true;
        });
        if (threadIdx.x == 0) *shared = st;  // (summed: 1)
    }
    for (;;) {
        __syncthreads();
        const State st = *shared;
        if (st.summed) return st;
        sum(st.node, st.a);
    }
}

// Trees with draft probabilities, a block for each sequence: the walk needs sums on its way.  The first is there (k_left has
// summed where the walk stops without it, over all CUs); others are rare, and this block's own (128256 f32 probabilities of two
// models: 9 us, what one CU loads).
template <class T>
__global__ __launch_bounds__(kWalkBlock) void k_walk(DraftArg a) {
    __shared__ double lds[kWalkBlock / 64];
    const int seq = blockIdx.x, segments = a.shares * (a.share / kSegment);
    const Span s = span_of(a, seq);
    double first = 0.0;
    for (int i = threadIdx.x; i < segments; i += kWalkBlock) first += a.sums[static_cast<int64_t>(seq) * segments + i];
    int calls = 0;
    __shared__ State shared;
    State st = walk_by_one<T>(a, s, a.path + static_cast<int64_t>(seq) * a.max_tokens, &shared, [&](int node, double share) {
        return calls++ == 0 ? block_sum<kWalkBlock>(first, lds)
                            : row_mass<T, kWalkBlock>(row_of<T>(a.target, a.target_stride, s.first + node),
                                                      row_of<T>(a.draft, a.draft_stride, s.first + node), share, a.vocab, lds);
    });
    st.summed = calls == 0;
    if (threadIdx.x == 0) a.state[seq] = st;
}

// Bits of the tokens that were tried at the node, from `begin` on, into gone (cleared by the caller).
__device__ __forceinline__ void mark_tried(const DraftArg& a, Span s, int node, int begin, uint32_t* gone, int threads) {
    for (int t = node + 1 + threadIdx.x; t < s.count; t += threads) {
        if (a.parents ? a.parents[s.first + t] != node : t != node + 1) continue;
        const int64_t x = a.tokens[s.first + t] - begin;
        if (x >= 0 && x < a.share) atomicOr(gone + x / 32, 1u << (x & 31));
    }
}

// When k_left runs: the only time; before k_walk, up to where the walk needs a sum; after it, where it went on.
enum Stage { kOnly, kBefore, kAfter };

// Block (share, sequence): the sums of what is left of a share, where the walk ends.  Every block walks by itself (a few
// dependent loads); the first share's writes the path down.
template <class T, Stage kStage>
__global__ __launch_bounds__(kBlock) void k_left(DraftArg a) {
    __shared__ State shared;
    __shared__ uint32_t gone[kMaxShare / 32];
    const int seq = static_cast<int>(a.by_shares.div(blockIdx.x)), share = blockIdx.x - seq * a.shares, begin = share * a.share;
    const Span s = span_of(a, seq);
    if (!a.draft)
        for (int i = threadIdx.x; i < a.share / 32; i += kBlock) gone[i] = 0;
    if (threadIdx.x < 64) {
        State st;
        if constexpr (kStage == kAfter) {
            st = a.state[seq];
            if (st.summed) st.node = -1;  // nothing more to do
        } else {
            const bool write = kStage == kOnly && share == 0;
            st = walk<T>(a, s, write ? a.path + static_cast<int64_t>(seq) * a.max_tokens : nullptr,
                         [](int, double, double&) { return false; });
            if (write && threadIdx.x == 0) a.state[seq] = st;
        }
        if (threadIdx.x == 0) shared = st;
    }
    __syncthreads();
    const State st = shared;
    if (st.node < 0) return;
    if (!a.draft) {
        mark_tried(a, s, st.node, begin, gone, kBlock);
        __syncthreads();
    }
    const T* p = row_of<T>(a.target, a.target_stride, s.first + st.node);
    const T* q = st.a != 0.0 ? row_of<T>(a.draft, a.draft_stride, s.first + st.node) : nullptr;
    const int end = min(begin + a.share, a.vocab);
    double* sums = a.sums + (static_cast<int64_t>(seq) * a.shares + share) * (a.share / kSegment);
    segment_sums<T>(p, q, st.a, a.draft ? nullptr : gone, begin, end, threadIdx.x >> 6, kBlock / 64, a.share / kSegment, sums);
}

// One wave: the token inside segment `chosen`, before which the running sum is `before`.  tried: tokens of the node's children count
// as nothing.
template <class T>
__device__ __forceinline__ void look_into(const DraftArg& a, int seq, Span s, int node, const T* p, const T* q, double share_of_q, bool tried, int chosen,
                                          double before, double goal) {
    const int lane = threadIdx.x & 63;
    const int i = chosen * kSegment + 4 * lane, end = min(chosen * kSegment + kSegment, a.vocab);
    uint32_t gone = 0;
    if (tried) {
        for (int t0 = node + 1; t0 < s.count; t0 += 64) {
            const int t = t0 + lane;
            const bool child = t < s.count && (a.parents ? a.parents[s.first + t] == node : t == node + 1);
            const int64_t x = child ? a.tokens[s.first + t] - chosen * static_cast<int64_t>(kSegment) : -1;
            const int inside = x >= 0 && x < kSegment ? static_cast<int>(x) : -1;
            for (uint64_t those = __ballot(inside >= 0); those; those &= those - 1) {
                const int gone_one = readlane(inside, __ffsll(static_cast<unsigned long long>(those)) - 1);
                if (gone_one >> 2 == lane) gone |= 1u << (gone_one & 3);
            }
        }
    }
    double left[4];
    left4<T>(load4<T>(p, i, end), q != nullptr, q ? load4<T>(q, i, end) : Four<T>{}, share_of_q, gone, left);
    const double mine = (left[0] + left[1]) + (left[2] + left[3]);
    double run = before + (wave_running(mine) - mine);
    int over = -1, some = -1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        run += left[e];
        if (left[e] > 0.0) {
            some = i + e;
            if (over < 0 && run > goal) over = i + e;
        }
    }
    const uint64_t overs = __ballot(over >= 0), somes = __ballot(some >= 0);
    const int l = overs ? __ffsll(static_cast<unsigned long long>(overs)) - 1 : somes ? 63 - __clzll(static_cast<long long>(somes)) : 0;
    const int token = overs ? over : some;
    if (lane == l) a.next[seq] = token;
}

constexpr int kPickEach = 4;  // sums of a lane: 1024, of 262144 probabilities, in one round

// A block for each sequence: the segment where the running sum passes final * total, then the token in it.
template <class T>
__global__ __launch_bounds__(kBlock) void k_pick(DraftArg a) {
    __shared__ double lds[kBlock / 64];
    __shared__ double before_it;
    __shared__ int chosen_one;
    const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Span s = span_of(a, seq);
    const State st = a.state[seq];
    const int segments = a.shares * (a.share / kSegment);
    const double* sums = a.sums + static_cast<int64_t>(seq) * segments;
    double v[kPickEach];
    auto load = [&](int c0) {
#pragma unroll
        for (int e = 0; e < kPickEach; ++e) v[e] = c0 + tid * kPickEach + e < segments ? sums[c0 + tid * kPickEach + e] : 0.0;
    };
    load(0);  // (where there are no rows what lies there is not used)
    int32_t* path = a.path + static_cast<int64_t>(seq) * a.max_tokens;
    for (int i = st.kept + tid; i < a.max_tokens; i += kBlock) path[i] = -1;
    if (tid == 0) a.kept[seq] = st.kept;
    if (st.node < 0) {
        if (tid == 0) a.next[seq] = -1;
        return;
    }
    const T* p = row_of<T>(a.target, a.target_stride, s.first + st.node);
    const T* q = st.a != 0.0 ? row_of<T>(a.draft, a.draft_stride, s.first + st.node) : nullptr;
    double share_of_q = st.a, total = 0.0;
    bool tried = !a.draft;
    for (int c0 = 0; c0 < segments; c0 += kBlock * kPickEach) {
        if (c0) load(c0);
        total += (v[0] + v[1]) + (v[2] + v[3]);
    }
    total = block_sum<kBlock>(total, lds);
    // nothing left: the target's own probabilities, summed here segment by segment (on the way of no sound input)
    const bool own = !(total > 0.0);
    if (own) {
        q = nullptr;
        share_of_q = 0.0;
        tried = false;
        total = row_mass<T, kBlock>(p, nullptr, 0.0, a.vocab, lds);
        if (!(total > 0.0)) {
            if (tid == 0) a.next[seq] = -1;
            return;
        }
    }
    const double goal = static_cast<double>(a.final[seq]) * total;
    if (tid == 0) chosen_one = -1;
    double base = 0.0;
    for (int c0 = 0; c0 < segments; c0 += kBlock * kPickEach) {
        if (own) {
#pragma unroll
            for (int e = 0; e < kPickEach; ++e) {
                const int b0 = (c0 + tid * kPickEach + e) * kSegment, b1 = min(b0 + kSegment, a.vocab);
                v[e] = 0.0;
                for (int i = b0; i < b1; ++i) v[e] += counted(p[i]);
            }
        } else if (segments > kBlock * kPickEach) {
            load(c0);
        }
        const double mine = (v[0] + v[1]) + (v[2] + v[3]), run = wave_running(mine);
        if (lane == 63) lds[wave] = run;
        __syncthreads();
        double before = base + (run - mine);
        for (int w = 0; w < wave; ++w) before += lds[w];
        for (int w = 0; w < kBlock / 64; ++w) base += lds[w];
        // the first segment that passes the goal, and the last that has anything (roundings, or sums that are not finite,
        // may let none pass); a wave's first and last lane that have one put it down
        int over = -1, some = -1;
        double over_before = 0.0, some_before = 0.0;
#pragma unroll
        for (int e = 0; e < kPickEach; ++e) {
            if (v[e] > 0.0) {
                some = c0 + tid * kPickEach + e;
                some_before = before;
                if (over < 0 && before + v[e] > goal) {
                    over = some;
                    over_before = before;
                }
            }
            before += v[e];
        }
        __shared__ int firsts[kBlock / 64], lasts[kBlock / 64];
        __shared__ double first_before[kBlock / 64], last_before[kBlock / 64];
        const uint64_t overs = __ballot(over >= 0), somes = __ballot(some >= 0);
        if (lane == 0) firsts[wave] = lasts[wave] = -1;
        if (overs && lane == __ffsll(static_cast<unsigned long long>(overs)) - 1) {
            firsts[wave] = over;
            first_before[wave] = over_before;
        }
        if (somes && lane == 63 - __clzll(static_cast<long long>(somes))) {
            lasts[wave] = some;
            last_before[wave] = some_before;
        }
        __syncthreads();
        bool passed = false;
        int which = -1;
        double at_it = 0.0;
        for (int w = 0; w < kBlock / 64; ++w) {
            if (lasts[w] >= 0 && !passed) {
                which = lasts[w];
                at_it = last_before[w];
            }
            if (firsts[w] >= 0 && !passed) {
                passed = true;
                which = firsts[w];
                at_it = first_before[w];
            }
        }
        if (tid == 0 && which >= 0) {
            chosen_one = which;
            before_it = at_it;
        }
        if (passed) break;
        __syncthreads();
    }
    __syncthreads();
    if (wave != 0) return;
    const int chosen = chosen_one;
    if (chosen < 0) {
        if (lane == 0) a.next[seq] = -1;
        return;
    }
    look_into<T>(a, seq, s, st.node, p, q, share_of_q, tried, chosen, before_it, goal);
}

// Vocabularies that one block sums in about the time of a launch: all of it in one launch, a block for each sequence, without a
// workspace.  Against two launches (four for trees with draft probabilities), f32, replayed: a chain of 6 over 16000 tokens 6.5 us
// (6.9), over 32768 7.8 (6.6), over 65536 11.1 (6.7), 32 chains over 32768 9.5 (10.4), 4 drawn trees of 24 over 32768 14.0 (16.5), over
// 65536 19.1 (17.3).  A call from the host is 15.5 against 19.4 where the GPU is no longer: up to 32768 its loss is less than the host's
// gain.
constexpr int kOnceVocab = 32768;

template <class T>
__global__ __launch_bounds__(kWalkBlock) void k_verify_once(DraftArg a) {
    constexpr int kWaves = kWalkBlock / 64, kEach = kOnceVocab / kSegment / 64;
    __shared__ double lds[kWaves], sums[kOnceVocab / kSegment];
    __shared__ uint32_t gone[kOnceVocab / 32];
    __shared__ State shared;
    const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Span s = span_of(a, seq);
    if (!a.draft)
        for (int i = tid; i < kOnceVocab / 32; i += kWalkBlock) gone[i] = 0;
    for (int i = tid; i < kOnceVocab / kSegment; i += kWalkBlock) sums[i] = 0.0;
    int32_t* path = a.path + static_cast<int64_t>(seq) * a.max_tokens;
    const State st = walk_by_one<T>(a, s, path, &shared, [&](int node, double share) {
        return row_mass<T, kWalkBlock>(row_of<T>(a.target, a.target_stride, s.first + node), row_of<T>(a.draft, a.draft_stride, s.first + node),
                                       share, a.vocab, lds);
    });
    for (int i = st.kept + tid; i < a.max_tokens; i += kWalkBlock) path[i] = -1;
    if (tid == 0) a.kept[seq] = st.kept;
    if (st.node < 0) {
        if (tid == 0) a.next[seq] = -1;
        return;
    }
    __syncthreads();
    if (!a.draft) {
        mark_tried(a, s, st.node, 0, gone, kWalkBlock);
        __syncthreads();
    }
    const T* p = row_of<T>(a.target, a.target_stride, s.first + st.node);
    const T* q = st.a != 0.0 ? row_of<T>(a.draft, a.draft_stride, s.first + st.node) : nullptr;
    double share_of_q = st.a, total, run;
    bool tried = !a.draft;
    for (bool own = false;; own = true) {  // a second time where nothing is left: the target's own probabilities
        segment_sums<T>(p, q, share_of_q, tried ? gone : nullptr, 0, a.vocab, wave, kWaves, a.share / kSegment, sums);
        __syncthreads();
        double mine = 0.0;
#pragma unroll
        for (int e = 0; e < kEach; ++e) mine += sums[lane * kEach + e];
        run = wave_running(mine);
        total = readlane_f64(run, 63);
        run -= mine;
        if (total > 0.0 || own) break;
        q = nullptr;
        share_of_q = 0.0;
        tried = false;
        __syncthreads();
    }
    if (wave != 0) return;
    if (!(total > 0.0)) {
        if (lane == 0) a.next[seq] = -1;
        return;
    }
    const double goal = static_cast<double>(a.final[seq]) * total;
    // the first segment that passes the goal, or the last that has anything
    int over = -1, some = -1;
    double over_before = 0.0, some_before = 0.0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const double v = sums[lane * kEach + e];
        if (v > 0.0) {
            some = lane * kEach + e;
            some_before = run;
            if (over < 0 && run + v > goal) {
                over = some;
                over_before = run;
            }
        }
        run += v;
    }
    const uint64_t overs = __ballot(over >= 0), somes = __ballot(some >= 0);
    const int l = overs ? __ffsll(static_cast<unsigned long long>(overs)) - 1 : 63 - __clzll(static_cast<long long>(somes));
    look_into<T>(a, seq, s, st.node, p, q, share_of_q, tried, readlane(overs ? over : some, l),
                       readlane_f64(overs ? over_before : some_before, l), goal);
}

// Probabilities of a share: so that all shares are about two blocks for each CU, at least 1024 (a load for each
// lane) and at most 8192.
int share_of(int64_t vocab, int64_t batch) {
    int share = 1024;
    while (share < kMaxShare && batch * ((vocab + share - 1) / share) > 2 * device_cu_count()) share *= 2;
    return share;
}

int64_t shares_of(int64_t vocab, int64_t batch) {
    const int share = share_of(vocab, batch);
    return (vocab + share - 1) / share;
}

int check_batch(const char* what, const tq_kv_batch* b, int64_t vocab) {
    TQ_REQUIRE(b, "%s: null batch", what);
    TQ_REQUIRE(b->batch >= 0 && b->max_tokens >= 0 && b->tokens >= 0 && b->batch <= kKvMaxRows && b->max_tokens <= kKvMaxRows &&
                   b->tokens <= kKvMaxRows,
               "%s: batch of %lld sequences, %lld tokens", what, (long long)b->batch, (long long)b->tokens);
    TQ_REQUIRE(b->offsets || b->tokens == b->batch * b->max_tokens, "%s: without offsets tokens=%lld must be batch * max_tokens = %lld",
               what, (long long)b->tokens, (long long)(b->batch * b->max_tokens));
    TQ_REQUIRE(aligned(b->offsets, 4), "%s: unaligned offsets", what);
    TQ_REQUIRE(vocab >= 1 && vocab <= kKvMaxRows, "%s: vocab=%lld is not in 1..2^30", what, (long long)vocab);
    return TQ_OK;
}

template <class T>
void launch_drafts(const DraftArg& a, hipStream_t st) {
    if (a.vocab <= kOnceVocab) {
        k_verify_once<T><<<a.batch, kWalkBlock, 0, st>>>(a);
        return;
    }
    if (a.draft && a.parents) {
        k_left<T, kBefore><<<a.batch * a.shares, kBlock, 0, st>>>(a);
        k_walk<T><<<a.batch, kWalkBlock, 0, st>>>(a);
        k_left<T, kAfter><<<a.batch * a.shares, kBlock, 0, st>>>(a);
    } else {
        k_left<T, kOnly><<<a.batch * a.shares, kBlock, 0, st>>>(a);
    }
    k_pick<T><<<a.batch, kBlock, 0, st>>>(a);
}

template <class T>
int launch_typed(const DraftArg& a, hipStream_t st, const char* what) {
    clear_error();
    launch_drafts<T>(a, st);
    return check_launch(what);
}

}  // namespace
}  // namespace tq

extern "C" {

int64_t tq_verify_drafts_workspace_bytes(const tq_kv_batch* batch, int64_t vocab) {
    using namespace tq;
    if (check_batch("tq_verify_drafts", batch, vocab) != TQ_OK) return -1;
    if (vocab <= kOnceVocab) return 0;
    return (batch->batch * static_cast<int64_t>(sizeof(State)) + batch->batch * shares_of(vocab, batch->batch) * (share_of(vocab, batch->batch) / kSegment) * 8 +
            15) / 16 * 16;
}

int tq_verify_drafts(const tq_kv_batch* batch, const int64_t* tokens, const void* target, int64_t target_stride,
                     const void* draft, int64_t draft_stride, int dtype, int64_t vocab, const int32_t* parents,
                     const float* accept, const float* final, void* workspace, int64_t workspace_bytes, int32_t* path,
                     int32_t* kept, int64_t* next, tq_stream_t stream) {
    using namespace tq;
    static const char* what = "tq_verify_drafts";
    const int rc = check_batch(what, batch, vocab);
    if (rc != TQ_OK) return rc;
    TQ_REQUIRE(dtype == TQ_DT_F32 || dtype == TQ_DT_BF16 || dtype == TQ_DT_F16, "%s: dtype %d is not f32, bf16 or f16", what, dtype);
    const int size = dtype == TQ_DT_F32 ? 4 : 2;
    TQ_REQUIRE(target_stride >= 0 && (!draft || draft_stride >= 0), "%s: negative stride", what);
    if (batch->batch == 0) return TQ_OK;
    TQ_REQUIRE(kept && next && (path || batch->max_tokens == 0), "%s: null path, kept or next", what);
    TQ_REQUIRE(batch->tokens == 0 || (tokens && target && accept && final), "%s: null tokens, target, accept or final", what);
    TQ_REQUIRE(aligned(tokens, 8) && aligned(target, size) && aligned(draft, size) && aligned(parents, 4) && aligned(accept, 4) &&
                   aligned(final, 4) && aligned(path, 4) && aligned(kept, 4) && aligned(next, 8),
               "%s: a pointer is not aligned to its elements", what);
    const int64_t shares = shares_of(vocab, batch->batch);
    TQ_REQUIRE(batch->batch <= (int64_t(1) << 22) - 1 && batch->batch * shares <= kMaxBlocks,
               "%s: %lld sequences with %lld shares of %lld tokens are more than %lld blocks", what, (long long)batch->batch,
               (long long)shares, (long long)vocab, (long long)kMaxBlocks);
    const int64_t need = tq_verify_drafts_workspace_bytes(batch, vocab);
    TQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 16)), "%s: workspace of %lld bytes, 16-byte aligned, needed",
               what, (long long)need);
    const int64_t rows = batch->tokens, sequences = batch->batch;
    TQ_REQUIRE(!overlap({{path, sequences * batch->max_tokens, 4}, {kept, sequences, 4}, {next, sequences, 8}, {need == 0 ? nullptr : workspace, need, 1}},
                        {{tokens, rows, 8}, {target, rows, target_stride, vocab, size}, {draft, rows, draft_stride, vocab, size}, {parents, rows, 4},
                         {accept, rows, 4}, {final, sequences, 4}, {batch->offsets, sequences + 1, 4}}),
               "%s: path, kept, next or the workspace overlaps another of them or an input", what);
    DraftArg a{};
    a.tokens = tokens;
    a.target = target;
    a.draft = draft;
    a.target_stride = target_stride;
    a.draft_stride = draft_stride;
    a.parents = parents;
    a.accept = accept;
    a.final = final;
    a.offsets = batch->offsets;
    a.batch = static_cast<int>(batch->batch);
    a.max_tokens = static_cast<int>(batch->max_tokens);
    a.rows = static_cast<int>(batch->tokens);
    a.vocab = static_cast<int>(vocab);
    a.share = vocab <= kOnceVocab ? static_cast<int>((vocab + kSegment - 1) / kSegment * kSegment) : share_of(vocab, batch->batch);
    a.shares = static_cast<int>(shares);
    a.by_shares = FastDiv(static_cast<uint32_t>(shares));
    a.path = path;
    a.kept = kept;
    a.next = next;
    a.state = static_cast<State*>(workspace);
    a.sums = reinterpret_cast<double*>(a.state + batch->batch);
    if (dtype == TQ_DT_F32) return launch_typed<float>(a, as_hip(stream), what);
    if (dtype == TQ_DT_BF16) return launch_typed<__bf16>(a, as_hip(stream), what);
    return launch_typed<_Float16>(a, as_hip(stream), what);
}

}  // extern "C"
