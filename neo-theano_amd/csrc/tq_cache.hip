// tq_cache.hip -- rotary positions and the 8-bit key/value cache's writes and reads.
//
//   rotary:  y0 = m (x0 cos a - x1 sin a), y1 = m (x1 cos a + x0 sin a),  a = pos f_i
//   write:   s = f32(max(absmax / qmax, 1e-10)), code = q(x / s) for each token's head
//   read:    f32(code * s)
//
// All three are HBM-bound streams.  16 lanes hold a head (8 elements each), so its maximum
// is a DPP reduction within a row of lanes, and one launch does everything that a token
// needs: its cosines and sines once, in LDS, for all of its heads; q out, codes of k and v.
//
// Angles: pos * f in f64 turns, reduced to an eighth of a turn before it becomes f32 (at
// position 2^20 an f32 product is off by 0.06 radians, the f64 one by 1e-10), then the
// Taylor polynomials of sine (to x^9: 2e-9 at pi / 4) and cosine (to x^10: 1e-10).
#include <algorithm>
#include <cmath>

#include "tq_kv.h"
#include "tq_rowfmt.h"

namespace tq {
namespace {

constexpr int kGroup = 16;              // lanes of a head
constexpr int kPer = 8;                 // elements of a lane
constexpr int kRowBlock = 256;          // 16 heads at a time
constexpr int kHeadsAtOnce = kRowBlock / kGroup;
constexpr int kMaxAxes = 4;

struct HeadsArg {
    const void* data;
    int heads;
    int64_t token, head;
};

template <int kType>
struct Elem;
template <>
struct Elem<TQ_DT_F32> {
    typedef float type;
    __device__ static float to(float v) { return v; }
    __device__ static float from(float v) { return v; }
};
template <>
struct Elem<TQ_DT_BF16> {
    typedef __bf16 type;
    __device__ static float to(__bf16 v) { return static_cast<float>(v); }
    __device__ static __bf16 from(float v) { return static_cast<__bf16>(v); }
};
template <>
struct Elem<TQ_DT_F16> {
    typedef _Float16 type;
    __device__ static float to(_Float16 v) { return static_cast<float>(v); }
    __device__ static _Float16 from(float v) {
        asm("" : "+v"(v));  // (a product and its rounding to f16 would become one instruction, which skips the f32 value)
        return static_cast<_Float16>(v);
    }
};

// Element i of lane l where whole vectors are moved: 16 bytes at a time, adjacent from lane to lane (8 of a
// 16-bit type; of f32 4 at 4 l and 4 at 64 + 4 l: as 8 at 8 l each store would have filled
// every other 16 bytes, 94 against 81 us for a read of 32767 tokens, 8 heads of 128).  Element
// by element: l + 16 i.
template <int kType>
struct Lay {
    static constexpr int kRun = kType == TQ_DT_F32 ? 4 : 8, kRuns = kPer / kRun;
};
template <int kType, bool kVec>
__device__ __forceinline__ int elem(int l, int i) {
    constexpr int r = Lay<kType>::kRun;
    return kVec ? r * l + i % r + kGroup * r * (i / r) : l + kGroup * i;
}

// The elements from p[at(run)] on, for each run; zeros where that is not below d.
template <int kType, class At>
__device__ __forceinline__ void load_runs(const typename Elem<kType>::type* p, int d, At at, float (&x)[kPer]) {
    constexpr int r = Lay<kType>::kRun;
    typedef typename Elem<kType>::type T;
    typedef T V __attribute__((ext_vector_type(r), aligned(16)));
#pragma unroll
    for (int c = 0; c < Lay<kType>::kRuns; ++c) {
        V v{};
        if (at(c) < d) v = *reinterpret_cast<const V*>(p + at(c));
#pragma unroll
        for (int i = 0; i < r; ++i) x[r * c + i] = Elem<kType>::to(v[i]);
    }
}

template <int kType, bool kVec>
__device__ __forceinline__ void load_head(const typename Elem<kType>::type* p, int l, int d, float (&x)[kPer]) {
    if constexpr (kVec) {  // whole runs (d a multiple of theirs), 16-byte aligned
        load_runs<kType>(p, d, [&](int c) { return elem<kType, true>(l, c * Lay<kType>::kRun); }, x);
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) x[i] = elem<kType, false>(l, i) < d ? Elem<kType>::to(p[elem<kType, false>(l, i)]) : 0.f;
    }
}

template <int kType, bool kVec>
__device__ __forceinline__ void store_head(typename Elem<kType>::type* p, int l, int d, const float (&x)[kPer]) {
    typedef typename Elem<kType>::type T;
    if constexpr (kVec) {
        constexpr int r = Lay<kType>::kRun;
        typedef T V __attribute__((ext_vector_type(r), aligned(16)));
#pragma unroll
        for (int c = 0; c < Lay<kType>::kRuns; ++c) {
            V v;
#pragma unroll
            for (int i = 0; i < r; ++i) v[i] = Elem<kType>::from(x[r * c + i]);
            const int e = elem<kType, true>(l, r * c);
            if (e < d) *reinterpret_cast<V*>(p + e) = v;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (elem<kType, false>(l, i) < d) p[elem<kType, false>(l, i)] = Elem<kType>::from(x[i]);
    }
}

// cos and sin of `turns` turns (f64), to about an f32 ulp.
__device__ __forceinline__ void cos_sin_turns(double turns, float& c, float& s) {
    const double f = turns - rint(turns);                    // [-1/2, 1/2]
    const double quarter = rint(4.0 * f);                    // -2 .. 2
    const float x = static_cast<float>((f - 0.25 * quarter) * 6.283185307179586);
    const float x2 = x * x;
    float ps = fmaf(x2, 1.0f / 362880.0f, -1.0f / 5040.0f);
    ps = fmaf(ps, x2, 1.0f / 120.0f);
    ps = fmaf(ps, x2, -1.0f / 6.0f);
    const float sn = fmaf(ps * x2, x, x);
    float pc = fmaf(x2, -1.0f / 3628800.0f, 1.0f / 40320.0f);
    pc = fmaf(pc, x2, -1.0f / 720.0f);
    pc = fmaf(pc, x2, 1.0f / 24.0f);
    pc = fmaf(pc, x2, -0.5f);
    const float cs = fmaf(pc, x2, 1.0f);
    const int q = static_cast<int>(quarter) & 3;
    c = q == 0 ? cs : q == 1 ? -sn : q == 2 ? -cs : sn;
    s = q == 0 ? sn : q == 1 ? cs : q == 2 ? -sn : -cs;
}

struct RotaryArg {
    const double* f;
    int half;  // planes; 0: no rotation
    int pairs, inverse;
    float scale;
};

// The elements that the head at p turns against its own: the other half's, or the neighbours (which
// whole vectors hold already).
template <int kType, bool kVec>
__device__ __forceinline__ void load_others(const typename Elem<kType>::type* p, int l, int d, const RotaryArg& r,
                                            float (&y)[kPer]) {
    if constexpr (kVec) {  // half a multiple of the runs: a run's elements share their side
        load_runs<kType>(p, d,
                         [&](int c) {
                             const int e = elem<kType, true>(l, c * Lay<kType>::kRun);
                             return e < r.half ? e + r.half : e < 2 * r.half ? e - r.half : d;
                         },
                         y);
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = elem<kType, false>(l, i);
            y[i] = e >= 2 * r.half ? 0.f : Elem<kType>::to(p[r.pairs ? e ^ 1 : e < r.half ? e + r.half : e - r.half]);
        }
    }
}

// Cosine and signed sine of the lane's own elements (the same in all of the token's heads); elements
// that pass have plane -1.
template <int kType, bool kVec>
struct LaneAngles {
    float c[kPer], s[kPer];
    bool on[kPer];
    __device__ LaneAngles(int l, const RotaryArg& r, const float* cs, const float* sn) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = elem<kType, kVec>(l, i);
            on[i] = e < 2 * r.half;
            const int plane = !on[i] ? 0 : r.pairs ? e >> 1 : e < r.half ? e : e - r.half;
            const bool second = r.pairs ? (e & 1) != 0 : e >= r.half;
            c[i] = cs[plane];
            s[i] = second ? sn[plane] : -sn[plane];
        }
    }
    // x cos + (its partner) sin, elements that pass as they are
    __device__ void turn(float (&x)[kPer], const float (&y)[kPer]) const {
#pragma unroll
        for (int i = 0; i < kPer; ++i) x[i] = on[i] ? fmaf(x[i], c[i], y[i] * s[i]) : x[i];
    }
};

// row_scale in f32 for finite absmax: the f64 quotient of two f32 values rounds to f32 as the f32 division does
// (53 >= 2 24 + 2 bits), rounding keeps the order, so the floor may be applied after it, and one correction of
// absmax * (1 / qmax) is that division (checked for every f32 absmax whose scale is above the floor).
template <class Fmt>
__device__ __forceinline__ float head_scale(float absmax) {
    constexpr float b = static_cast<float>(Fmt::kQmax), r = 1.0f / b;
    const float q = absmax * r;
    return fmaxf(fmaf(fmaf(-q, b, absmax), r, q), static_cast<float>(1e-10));
}

// Codes of four finite elements for their head's own scale: the coders of tq_rowfmt.h without what only
// NaN and infinities need (|x / s| stays below 448 (1 + 2^-22), which rounds to 448, so nothing saturates).
__device__ __forceinline__ uint32_t finite4(const FmtI8::Row& r, const float* x) {
    int c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = fabsf(x[i]);
        float n = floorf(fmaf(a, r.inv, 0.5f - 0x1p-12f));
        n = fmaf(-n, r.s, a) >= r.half ? n + 1.0f : n;
        c[i] = static_cast<int>(copysignf(n, x[i]));
    }
    return pack4_i8(c[0], c[1], c[2], c[3]);
}
__device__ __forceinline__ uint32_t finite4(const FmtFp8::Row& r, const float* x) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(r.quot(x[0]), r.quot(x[1]), 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(r.quot(x[2]), r.quot(x[3]), w, true);
    return static_cast<uint32_t>(w);
}

struct OpMaxU {
    __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return max(a, b); }
};

// Which of the positions' rows turns a plane: two bits for each plane (all 0 where there is one axis).
struct AxesArg {
    uint64_t planes[2];
    int64_t stride;
    int count;
    __device__ int of(int plane) const { return static_cast<int>((plane < 32 ? planes[0] : planes[1]) >> (2 * (plane & 31))) & 3; }
};

struct RowsArg {
    HeadsArg q, k, v;
    const int64_t* positions;
    AxesArg axes;
    RotaryArg rot;
    KvBatch b;
    int d, row, n;
    void* q_out;
    void* k_out;  // rotary alone: k turned; else null and k goes to the cache
    void* k_codes;
    float* k_scale;
    void* v_codes;
    float* v_scale;
};

// Codes one head (elements in x, zeros past it) into row `at` of the cache's [pages, heads, page].  The maximum
// is taken of the bits of |x|, which order as the values do, NaN last: heads without NaN and infinities (all of the
// wave's, as a rule) take the short coder.
template <int kType, bool kVec, class Fmt>
__device__ __forceinline__ void code_head(const float (&x)[kPer], int l, int d, int row, int64_t at, void* codes0,
                                          float* scale) {
    typedef typename Fmt::code_t C;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    top = lane_group_reduce<kGroup>(top, OpMaxU{});
    float sc = head_scale<Fmt>(__uint_as_float(top));
    uint32_t c[2];
    if (!__ballot(top >= 0x7F800000u)) {
        const typename Fmt::Row coder(sc);
        c[0] = finite4(coder, x);
        c[1] = finite4(coder, x + 4);
    } else {
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (elem<kType, kVec>(l, i) < d) m = fmaxf(m, fabsf(x[i]));
        sc = row_scale<Fmt>(absmax_finish(group_max<kGroup>(m)));
        const typename Fmt::Row coder(sc);
        c[0] = coder.code4(f32x4{x[0], x[1], x[2], x[3]});
        c[1] = coder.code4(f32x4{x[4], x[5], x[6], x[7]});
    }
    C* codes = static_cast<C*>(codes0) + at * row;
    if (l == 0) scale[at] = sc;
    if constexpr (kVec) {
        const int e0 = elem<kType, true>(l, 0), e1 = elem<kType, true>(l, 4);
        if constexpr (Lay<kType>::kRuns == 1) {
            if (e0 < row) *reinterpret_cast<uint2*>(codes + e0) = make_uint2(c[0], c[1]);
        } else {
            if (e0 < row) *reinterpret_cast<uint32_t*>(codes + e0) = c[0];
            if (e1 < row) *reinterpret_cast<uint32_t*>(codes + e1) = c[1];
        }
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (elem<kType, false>(l, i) < row) codes[elem<kType, false>(l, i)] = static_cast<C>(c[i >> 2] >> (8 * (i & 3)));
    }
}

// Turns, codes and stores head h of a kind (0 q, 1 k, 2 v) of token n, whose loads are in x and y; page -1: no place.
template <int kType, bool kVec, bool kTurn, class Fmt>
__device__ __forceinline__ void finish_head(const RowsArg& a, int kind, int h, int n, int64_t page, int64_t off, int l,
                                            const LaneAngles<kType, kVec>& angles, float (&x)[kPer], float (&y)[kPer]) {
    typedef typename Elem<kType>::type T;
    const int of = kind == 0 ? a.q.heads : kind == 1 ? a.k.heads : a.v.heads;
    if (kTurn && kind < 2) {
        if (kVec && a.rot.pairs) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) y[i] = x[i ^ 1];
        }
        angles.turn(x, y);
    }
    T* out = static_cast<T*>(kind == 0 ? a.q_out : kind == 1 ? a.k_out : nullptr);
    if (out)
        store_head<kType, kVec>(out + (static_cast<int64_t>(n) * of + h) * a.d, l, a.d, x);
    else if (page >= 0)
        code_head<kType, kVec, Fmt>(x, l, a.d, a.row, (page * of + h) * a.b.page + off, kind == 1 ? a.k_codes : a.v_codes,
                                    kind == 1 ? a.k_scale : a.v_scale);
}

template <int kType, bool kVec, bool kTurn>
__device__ __forceinline__ void load_row(const RowsArg& a, int kind, int h, int n, int l, float (&x)[kPer], float (&y)[kPer]) {
    const HeadsArg& src = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
    const auto* p = static_cast<const typename Elem<kType>::type*>(src.data) + n * src.token + h * src.head;
    load_head<kType, kVec>(p, l, a.d, x);
    if (kTurn && kind < 2 && !(kVec && a.rot.pairs)) load_others<kType, kVec>(p, l, a.d, a.rot, y);
}

// Cosines and sines of plane i at `pos` into cs[i], sn[i].
__device__ __forceinline__ void plane_angle(const RotaryArg& r, int i, double pos, float* cs, float* sn) {
    float c, s;
    cos_sin_turns(pos * (r.f[i] * 0.15915494309189535), c, s);
    cs[i] = c * r.scale;
    sn[i] = (r.inverse ? -s : s) * r.scale;
}

// Few tokens: block (token, 16 heads of a kind), a group of 16 lanes for each head, whose loads are issued
// before the token's place and angles are known.
template <int kType, bool kVec, bool kTurn, class Fmt>
__global__ __launch_bounds__(kRowBlock) void k_token_rows(RowsArg a) {
    __shared__ float cs[kKvMaxHeadDim / 2], sn[kKvMaxHeadDim / 2];
    const int n = blockIdx.x, tid = threadIdx.x, l = tid % kGroup, j = tid / kGroup;
    auto shares = [](int heads) { return (heads + kHeadsAtOnce - 1) / kHeadsAtOnce; };
    const int sq = shares(a.q.heads), sk = shares(a.k.heads);
    const int y = blockIdx.y, kind = y < sq ? 0 : y < sq + sk ? 1 : 2;  // uniform
    const int h = (y - (kind == 0 ? 0 : kind == 1 ? sq : sq + sk)) * kHeadsAtOnce + j;
    const int of = kind == 0 ? a.q.heads : kind == 1 ? a.k.heads : a.v.heads;
    float x[kPer], o[kPer];
    load_row<kType, kVec, kTurn>(a, kind, min(h, of - 1), n, l, x, o);
    KvPlace place{-1, -1, false};
    if (a.b.lengths) {
        place = kv_place(a.b, n, kv_sequence(a.b, n, tid & 63));
        if (place.behind) return;  // the whole block: left as it was
    }
    if constexpr (kTurn) {
        int64_t pos = a.positions ? a.positions[n] : place.pos;  // (uniform, and the only one as a rule)
        if (a.positions && a.axes.count > 1) pos = a.positions[a.axes.of(min(tid, a.rot.half - 1)) * a.axes.stride + n];
        if (tid < a.rot.half) plane_angle(a.rot, tid, static_cast<double>(pos), cs, sn);
        __syncthreads();
    }
    if (h >= of) return;  // (whole groups)
    const LaneAngles<kType, kVec> angles(l, a.rot, cs, sn);
    const int64_t page = place.slot < 0 ? -1 : place.slot / a.b.page;
    finish_head<kType, kVec, kTurn, Fmt>(a, kind, h, n, page, place.slot - page * a.b.page, l, angles, x, o);
}

// Many tokens: block (kTB adjacent tokens, share of the steps), a group of 16 lanes for each token and each of
// 16 / kTB adjacent heads of a kind; a step is that many heads; two steps are in flight, four where nothing turns.  A lane keeps its token's
// angles in registers.  kTB = 1 reads and writes a token's heads in one run.  kAxes: positions of several axes, whose loads and lookup
// cost one axis nothing (4093 tokens, 64 heads of 128, half of them turned, one axis, replayed: 23.9 us, 24.4 by the form of several).
template <int kType, bool kVec, bool kTurn, int kTB, class Fmt, bool kAxes>
__global__ __launch_bounds__(kRowBlock) void k_rows(RowsArg a, int per_share) {
    constexpr int kHalf = kKvMaxHeadDim / 2, kHS = kHeadsAtOnce / kTB, kU = kTurn ? 2 : 4;
    __shared__ float cs[kTB][kHalf], sn[kTB][kHalf];
    __shared__ int64_t slots[kTB];
    __shared__ double at[kAxes ? kMaxAxes : 1][kTB];
    const int tid = threadIdx.x, l = tid % kGroup, j = tid / kGroup, jt = j % kTB, jh = j / kTB, n0 = blockIdx.x * kTB;
    const int n = min(n0 + jt, a.n - 1);
    if (tid < 64) {
        KvPlace p{-1, -1, false};
        const int nn = min(n0 + tid, a.n - 1);
        if (a.b.lengths) {
            const int seq = kv_sequences16(a.b, n0, a.n, tid);
            if (tid < kTB) p = kv_place(a.b, nn, seq);
        }
        if (tid < kTB) {
            slots[tid] = n0 + tid >= a.n || p.behind ? -2 : p.slot;
            at[0][tid] = static_cast<double>(a.positions ? a.positions[nn] : p.pos);
            if constexpr (kAxes)
                for (int x = 1; x < a.axes.count; ++x) at[x][tid] = static_cast<double>(a.positions[x * a.axes.stride + nn]);
        }
    }
    __syncthreads();
    if constexpr (kTurn) {
        for (int i = tid; i < kTB * a.rot.half; i += kRowBlock) {
            const int t = i / a.rot.half, plane = i - t * a.rot.half;
            plane_angle(a.rot, plane, at[kAxes ? a.axes.of(plane) : 0][t], cs[t], sn[t]);
        }
        __syncthreads();
    }
    const LaneAngles<kType, kVec> angles(l, a.rot, cs[jt], sn[jt]);
    const int64_t slot = slots[jt];
    const int64_t page = slot < 0 ? -1 : slot / a.b.page, off = slot - page * a.b.page;
    auto steps = [](int heads) { return (heads + kHS - 1) / kHS; };
    const int sq = steps(a.q.heads), sk = steps(a.k.heads), sv = steps(a.v.heads);
    const int end = min(static_cast<int>(blockIdx.y + 1) * per_share, sq + sk + sv);
    for (int s0 = blockIdx.y * per_share; s0 < end; s0 += kU) {
        float x[kU][kPer], y[kU][kPer];
        int kind[kU], h[kU], of[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int i = min(s0 + u, end - 1);
            kind[u] = i < sq ? 0 : i < sq + sk ? 1 : 2;  // uniform
            h[u] = (i - (kind[u] == 0 ? 0 : kind[u] == 1 ? sq : sq + sk)) * kHS + jh;
            of[u] = kind[u] == 0 ? a.q.heads : kind[u] == 1 ? a.k.heads : a.v.heads;
            load_row<kType, kVec, kTurn>(a, kind[u], min(h[u], of[u] - 1), n, l, x[u], y[u]);
        }
        if (slot == -2) continue;
#pragma unroll
        for (int u = 0; u < kU; ++u)
            if (s0 + u < end && h[u] < of[u])
                finish_head<kType, kVec, kTurn, Fmt>(a, kind[u], h[u], n, page, off, l, angles, x[u], y[u]);
    }
}

struct ReadArg {
    KvBatch b;
    const void* k;
    const float* k_scale;
    const void* v;
    const float* v_scale;
    int heads, d, row, n;
    void* k_out;
    void* v_out;
};

// Block (kTB adjacent tokens, share of the steps), groups and steps as in k_rows; four steps in flight.
template <int kType, bool kVec, int kTB, class Fmt>
__global__ __launch_bounds__(kRowBlock) void k_read_rows(ReadArg a, int per_share) {
    typedef typename Elem<kType>::type T;
    typedef typename Fmt::code_t C;
    constexpr int kU = 4, kHS = kHeadsAtOnce / kTB;
    __shared__ int64_t slots[kTB];
    const int tid = threadIdx.x, l = tid % kGroup, j = tid / kGroup, jt = j % kTB, jh = j / kTB, n0 = blockIdx.x * kTB;
    if (tid < 64) {
        const int seq = kv_sequences16(a.b, n0, a.n, tid);
        if (tid < kTB && n0 + tid < a.n) {
            const KvPlace p = kv_place(a.b, n0 + tid, seq);
            slots[tid] = p.behind ? -2 : p.slot;
        }
    }
    __syncthreads();
    const int n = n0 + jt;
    if (n >= a.n) return;
    const int64_t slot = slots[jt];
    if (slot == -2) return;  // left as it was
    const int64_t page = slot < 0 ? 0 : slot / a.b.page, off = slot < 0 ? 0 : slot - page * a.b.page;
    const int steps = (a.heads + kHS - 1) / kHS;  // of k, and as many of v
    const int end = min(static_cast<int>(blockIdx.y + 1) * per_share, 2 * steps);
    for (int s0 = blockIdx.y * per_share; s0 < end; s0 += kU) {
        uint32_t c[kU][kPer / 4];
        C one[kU][kPer];
        float sc[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int i = min(s0 + u, end - 1);
            const bool is_k = i < steps;
            const int h = min((is_k ? i : i - steps) * kHS + jh, a.heads - 1);
            const int64_t at = (page * a.heads + h) * a.b.page + off;
            const C* codes = static_cast<const C*>(is_k ? a.k : a.v) + at * a.row;
            sc[u] = (is_k ? a.k_scale : a.v_scale)[at];
            if constexpr (kVec) {
                if constexpr (Lay<kType>::kRuns == 1) {
                    const uint2 w = *reinterpret_cast<const uint2*>(codes + min(elem<kType, true>(l, 0), a.row - 8));
                    c[u][0] = w.x;
                    c[u][1] = w.y;
                } else {
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        c[u][e] = *reinterpret_cast<const uint32_t*>(codes + min(elem<kType, true>(l, 4 * e), a.row - 4));
                }
            } else {
#pragma unroll
                for (int e = 0; e < kPer; ++e) one[u][e] = codes[min(elem<kType, false>(l, e), a.row - 1)];
            }
        }
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const bool is_k = s0 + u < steps;
            const int h = (is_k ? s0 + u : s0 + u - steps) * kHS + jh;
            if (s0 + u >= end || h >= a.heads) continue;
            float x[kPer];
            if constexpr (kVec) {
                const f32x4 v = Fmt::value4(c[u][0], sc[u]), w = Fmt::value4(c[u][1], sc[u]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] = v[e];
                    x[4 + e] = w[e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < kPer; ++e) x[e] = Fmt::value1(one[u][e], sc[u]);
            }
#pragma unroll
            for (int e = 0; e < kPer; ++e) x[e] = slot < 0 ? 0.f : x[e];
            store_head<kType, kVec>(static_cast<T*>(is_k ? a.k_out : a.v_out) + (static_cast<int64_t>(n) * a.heads + h) * a.d, l,
                                    a.d, x);
        }
    }
}

int64_t type_size(int dtype) { return dtype == TQ_DT_F32 ? 4 : 2; }

int64_t run_of(int dtype) { return dtype == TQ_DT_F32 ? 4 : 8; }

bool vec_rows(const tq_heads* x, int64_t d, int dtype) {
    return !x || x->heads == 0 ||
           (aligned(x->data, 16) && d % run_of(dtype) == 0 && x->token_stride * type_size(dtype) % 16 == 0 &&
            x->head_stride * type_size(dtype) % 16 == 0);
}

HeadsArg heads_arg(const tq_heads* x) {
    return x ? HeadsArg{x->data, static_cast<int>(x->heads), x->token_stride, x->head_stride} : HeadsArg{};
}

int check_rotary(const char* what, const tq_rotary* r, int64_t d) {
    TQ_REQUIRE(r, "%s: null rotary", what);
    TQ_REQUIRE(r->rotary_dim >= 0 && r->rotary_dim % 2 == 0 && r->rotary_dim <= d,
               "%s: rotary_dim=%lld is not an even number up to head_dim=%lld", what, (long long)r->rotary_dim, (long long)d);
    TQ_REQUIRE(r->rotary_dim == 0 || r->frequencies, "%s: null frequencies", what);
    return TQ_OK;
}

// axes null: one axis.  Without positions every axis has the rows' places.
int check_axes(const char* what, const tq_rotary_axes* x, const tq_rotary* r, AxesArg* out) {
    *out = AxesArg{{0, 0}, 0, 1};
    if (!x) return TQ_OK;
    TQ_REQUIRE(x->axes >= 1 && x->axes <= kMaxAxes, "%s: axes=%lld is not in 1..4", what, (long long)x->axes);
    TQ_REQUIRE(r->rotary_dim <= kKvMaxHeadDim, "%s: axes are given for planes of up to 128 elements, not rotary_dim=%lld", what,
               (long long)r->rotary_dim);
    TQ_REQUIRE(x->position_stride >= 0, "%s: position_stride=%lld", what, (long long)x->position_stride);
    if (r->rotary_dim == 0) return TQ_OK;  // no plane: one axis, whose number the kernels need not look up
    *out = AxesArg{{x->planes[0], x->planes[1]}, x->position_stride, static_cast<int>(x->axes)};
    for (int64_t i = 0; i < r->rotary_dim / 2; ++i)
        TQ_REQUIRE(static_cast<int64_t>(x->planes[i / 32] >> (2 * (i % 32)) & 3) < x->axes, "%s: plane %lld is of none of the %lld axes",
                   what, (long long)i, (long long)x->axes);
    return TQ_OK;
}

RotaryArg rotary_arg(const tq_rotary* r) {
    return RotaryArg{r->frequencies, static_cast<int>(r->rotary_dim / 2), r->interleaved != 0, r->inverse != 0, r->scale};
}

template <int kType, bool kVec, bool kTurn, int kTB, class Fmt, bool kAxes = false>
void launch_many(const RowsArg& a, hipStream_t st) {
    constexpr int kHS = kHeadsAtOnce / kTB;
    auto steps = [](int heads) { return (heads + kHS - 1) / kHS; };
    const int all = steps(a.q.heads) + steps(a.k.heads) + steps(a.v.heads), groups = (a.n + kTB - 1) / kTB;
    const int want = std::max(1, std::min((8 * device_cu_count() + groups - 1) / groups, (all + 1) / 2));
    const int per = (all + want - 1) / want;
    k_rows<kType, kVec, kTurn, kTB, Fmt, kAxes><<<dim3(groups, (all + per - 1) / per), kRowBlock, 0, st>>>(a, per);
}

// Tokens to a block from 128 tokens on: 1 where heads only turn (4093 tokens, 64 heads of 128, bf16: 24 us, 26 with 4
// and 28 with 16), 16 where they are only coded, since a page's lines of codes and scales are then written by one
// block (4096 tokens, 32 heads of 80, FP8: 31 us with 1, 29 with 4, 27 with 16), 4 for both.
constexpr int kManyFrom = 128, kTurnTokens = 1, kCodeTokens = 16, kBothTokens = 4;
int tokens_to_a_block(const RowsArg& a) {
    return a.n < kManyFrom ? 1 : a.rot.half == 0 ? kCodeTokens : a.k_codes ? kBothTokens : kTurnTokens;
}
template <int kType, bool kVec, bool kTurn, class Fmt>
void launch_rows_vec(const RowsArg& a, hipStream_t st) {
    if (a.n >= kManyFrom) {
        if constexpr (!kTurn) return launch_many<kType, kVec, false, kCodeTokens, Fmt>(a, st);
        const bool axes = a.positions && a.axes.count > 1;  // (a row's place is the same on all)
        if (a.k_codes) return axes ? launch_many<kType, kVec, true, kBothTokens, Fmt, true>(a, st) : launch_many<kType, kVec, true, kBothTokens, Fmt>(a, st);
        return axes ? launch_many<kType, kVec, true, kTurnTokens, FmtI8, true>(a, st) : launch_many<kType, kVec, true, kTurnTokens, FmtI8>(a, st);
    }
    auto shares = [](int heads) { return (heads + kHeadsAtOnce - 1) / kHeadsAtOnce; };
    k_token_rows<kType, kVec, kTurn, Fmt>
        <<<dim3(a.n, shares(a.q.heads) + shares(a.k.heads) + shares(a.v.heads)), kRowBlock, 0, st>>>(a);
}

template <int kType, class Fmt>
int launch_rows(const RowsArg& a, bool vec, hipStream_t st, const char* what) {
    clear_error();
    const bool turn = a.rot.half > 0;
    if (vec && turn)
        launch_rows_vec<kType, true, true, Fmt>(a, st);
    else if (vec)
        launch_rows_vec<kType, true, false, Fmt>(a, st);
    else if (turn)
        launch_rows_vec<kType, false, true, Fmt>(a, st);
    else
        launch_rows_vec<kType, false, false, Fmt>(a, st);
    return check_launch(what);
}

template <class Fmt>
int launch_rows_typed(const RowsArg& a, int dtype, bool vec, hipStream_t st, const char* what) {
    TQ_REQUIRE(a.n <= kMaxBlocks * tokens_to_a_block(a), "%s: %d tokens, %d to a block, are more than %lld blocks", what, a.n,
               tokens_to_a_block(a), (long long)kMaxBlocks);
    if (dtype == TQ_DT_F32) return launch_rows<TQ_DT_F32, Fmt>(a, vec, st, what);
    if (dtype == TQ_DT_BF16) return launch_rows<TQ_DT_BF16, Fmt>(a, vec, st, what);
    return launch_rows<TQ_DT_F16, Fmt>(a, vec, st, what);
}

// A run of elements turns against a run: halves of whole runs.
bool vec_rotary(const RotaryArg& r, int dtype) { return r.pairs || r.half % run_of(dtype) == 0; }

int write_rows(const char* what, const tq_kv_cache* cache, const tq_kv_batch* batch, const tq_rotary* rotary,
               const tq_rotary_axes* axes, const int64_t* positions, const tq_heads* q, const tq_heads* k, const tq_heads* v,
               int dtype, void* q_out, hipStream_t st) {
    RowsArg a{};
    int rc = kv_check(what, cache, batch, &a.b);
    if (rc != TQ_OK) return rc;
    const int64_t d = cache->head_dim;
    TQ_REQUIRE(k && v, "%s: null k or v", what);
    if ((rc = kv_check_heads(what, "k", k, cache->heads, d, dtype)) != TQ_OK) return rc;
    if ((rc = kv_check_heads(what, "v", v, cache->heads, d, dtype)) != TQ_OK) return rc;
    bool vec = vec_rows(k, d, dtype) && vec_rows(v, d, dtype);
    if (rotary) {
        if ((rc = check_rotary(what, rotary, d)) != TQ_OK) return rc;
        if ((rc = check_axes(what, axes, rotary, &a.axes)) != TQ_OK) return rc;
        a.rot = rotary_arg(rotary);
        a.positions = positions;
        vec = vec && vec_rotary(a.rot, dtype);
        if (q && q->heads) {
            if ((rc = kv_check_heads(what, "q", q, q->heads, d, dtype)) != TQ_OK) return rc;
            TQ_REQUIRE(q_out || batch->tokens == 0, "%s: null q_out", what);
            a.q = heads_arg(q);
            a.q_out = q_out;
            vec = vec && vec_rows(q, d, dtype) && aligned(q_out, 16);
        }
    }
    if (batch->tokens == 0 || batch->batch == 0) return TQ_OK;
    TQ_REQUIRE(k->data && v->data && (a.q.heads == 0 || a.q.data), "%s: null data", what);
    a.k = heads_arg(k);
    a.v = heads_arg(v);
    a.d = static_cast<int>(d);
    a.row = static_cast<int>(kv_row(d));
    a.n = static_cast<int>(batch->tokens);
    a.k_codes = cache->k;
    a.k_scale = cache->k_scale;
    a.v_codes = cache->v;
    a.v_scale = cache->v_scale;
    return cache->codes == TQ_QINT8 ? launch_rows_typed<FmtI8>(a, dtype, vec, st, what)
                                    : launch_rows_typed<FmtFp8>(a, dtype, vec, st, what);
}

template <int kType, bool kVec, int kTB, class Fmt>
void launch_read_many(const ReadArg& a, hipStream_t st) {
    constexpr int kHS = kHeadsAtOnce / kTB;
    const int all = 2 * ((a.heads + kHS - 1) / kHS), groups = (a.n + kTB - 1) / kTB;
    const int want = std::max(1, std::min((8 * device_cu_count() + groups - 1) / groups, (all + 3) / 4));
    const int per = (all + want - 1) / want;
    k_read_rows<kType, kVec, kTB, Fmt><<<dim3(groups, (all + per - 1) / per), kRowBlock, 0, st>>>(a, per);
}

// four tokens to a block (32767 tokens, 8 heads of 128 to f32: 115 us with 1, 62 with 4, 75 with 16)
constexpr int kReadTokens = 4;
template <int kType, class Fmt>
int launch_read(const ReadArg& a, bool vec, hipStream_t st, const char* what) {
    clear_error();
    if (vec)
        launch_read_many<kType, true, kReadTokens, Fmt>(a, st);
    else
        launch_read_many<kType, false, kReadTokens, Fmt>(a, st);
    return check_launch(what);
}

template <class Fmt>
int launch_read_typed(const ReadArg& a, int dtype, bool vec, hipStream_t st, const char* what) {
    if (dtype == TQ_DT_F32) return launch_read<TQ_DT_F32, Fmt>(a, vec, st, what);
    if (dtype == TQ_DT_BF16) return launch_read<TQ_DT_BF16, Fmt>(a, vec, st, what);
    return launch_read<TQ_DT_F16, Fmt>(a, vec, st, what);
}

}  // namespace

int kv_check_heads(const char* what, const char* name, const tq_heads* x, int64_t heads, int64_t d, int dtype) {
    TQ_REQUIRE(dtype == TQ_DT_F32 || dtype == TQ_DT_BF16 || dtype == TQ_DT_F16,
               "%s: dtype %d is not f32, bf16 or f16", what, dtype);
    TQ_REQUIRE(x->heads == heads && heads >= 0 && heads <= 65535, "%s: %s has %lld heads, expected %lld (at most 65535)",
               what, name, (long long)x->heads, (long long)heads);
    TQ_REQUIRE(x->token_stride >= 0 && x->head_stride >= 0, "%s: %s has a negative stride", what, name);
    TQ_REQUIRE(aligned(x->data, type_size(dtype)), "%s: %s is not aligned to its elements", what, name);
    TQ_REQUIRE(d >= 1 && d <= kKvMaxHeadDim, "%s: head_dim=%lld is not in 1..128", what, (long long)d);
    return TQ_OK;
}

int kv_check(const char* what, const tq_kv_cache* c, const tq_kv_batch* b, KvBatch* out) {
    TQ_REQUIRE(c && b, "%s: null cache or batch", what);
    TQ_REQUIRE(c->codes == TQ_QINT8 || c->codes == TQ_QFP8, "%s: a cache holds INT8 or FP8 codes, not %d", what, c->codes);
    TQ_REQUIRE(c->head_dim >= 1 && c->head_dim <= kKvMaxHeadDim, "%s: head_dim=%lld is not in 1..128", what,
               (long long)c->head_dim);
    TQ_REQUIRE(c->page >= 16 && c->page % 16 == 0 && c->page <= kKvMaxPage,
               "%s: page=%lld is not a multiple of 16 up to 65536", what, (long long)c->page);
    TQ_REQUIRE(c->heads >= 1 && c->heads <= 65535 && c->pages >= 1 && c->pages <= INT32_MAX,
               "%s: cache of %lld pages, %lld heads", what, (long long)c->pages, (long long)c->heads);
    TQ_REQUIRE(c->k && c->v && c->k_scale && c->v_scale, "%s: null cache buffer", what);
    TQ_REQUIRE(aligned(c->k, 16) && aligned(c->v, 16) && aligned(c->k_scale, 16) && aligned(c->v_scale, 16),
               "%s: cache buffers are not 16-byte aligned", what);
    TQ_REQUIRE(b->batch >= 0 && b->max_tokens >= 0 && b->tokens >= 0 && b->table_pages >= 0 && b->batch <= kKvMaxRows &&
                   b->max_tokens <= kKvMaxRows && b->tokens <= kKvMaxRows,
               "%s: batch of %lld sequences, %lld tokens, %lld pages each", what, (long long)b->batch, (long long)b->tokens,
               (long long)b->table_pages);
    TQ_REQUIRE(b->table_pages <= kKvMaxRows / c->page, "%s: a table of %lld pages of %lld tokens is longer than 2^30 tokens",
               what, (long long)b->table_pages, (long long)c->page);
    TQ_REQUIRE(b->table_stride >= b->table_pages || b->batch <= 1, "%s: table_stride=%lld under %lld pages", what,
               (long long)b->table_stride, (long long)b->table_pages);
    TQ_REQUIRE(b->offsets || b->tokens == b->batch * b->max_tokens,
               "%s: without offsets tokens=%lld must be batch * max_tokens = %lld", what, (long long)b->tokens,
               (long long)(b->batch * b->max_tokens));
    TQ_REQUIRE(b->batch == 0 || (b->lengths && (b->table || b->table_pages == 0)), "%s: null lengths or table", what);
    TQ_REQUIRE(aligned(b->table, 4) && aligned(b->lengths, 4) && aligned(b->offsets, 4),
               "%s: table, lengths or offsets are not 4-byte aligned", what);
    *out = KvBatch{b->table,
                   b->table_stride,
                   b->lengths,
                   b->offsets,
                   static_cast<int>(b->batch),
                   static_cast<int>(b->max_tokens),
                   static_cast<int>(b->tokens),
                   static_cast<int>(b->table_pages),
                   static_cast<int>(c->pages),
                   static_cast<int>(c->page),
                   static_cast<int>(b->table_pages * c->page),
                   FastDiv(static_cast<uint32_t>(c->page)),
                   FastDiv(static_cast<uint32_t>(b->max_tokens > 0 ? b->max_tokens : 1))};
    return TQ_OK;
}

}  // namespace tq

namespace tq {
namespace {

int apply_rows(const char* what, const tq_rotary* rotary, const tq_rotary_axes* axes, const int64_t* positions, int64_t n,
               const tq_heads* q, const tq_heads* k, int dtype, int64_t head_dim, void* q_out, void* k_out, tq_stream_t stream) {
    int rc = check_rotary(what, rotary, head_dim);
    if (rc != TQ_OK) return rc;
    TQ_REQUIRE(n >= 0 && n <= kKvMaxRows, "%s: n=%lld", what, (long long)n);
    RowsArg a{};
    if ((rc = check_axes(what, axes, rotary, &a.axes)) != TQ_OK) return rc;
    bool vec = true;
    for (int i = 0; i < 2; ++i) {
        const tq_heads* x = i == 0 ? q : k;
        if (!x || x->heads == 0) continue;
        if ((rc = kv_check_heads(what, i == 0 ? "q" : "k", x, x->heads, head_dim, dtype)) != TQ_OK) return rc;
        void* out = i == 0 ? q_out : k_out;
        TQ_REQUIRE(n == 0 || (x->data && out), "%s: null data", what);
        TQ_REQUIRE(aligned(out, type_size(dtype)), "%s: output is not aligned to its elements", what);
        vec = vec && vec_rows(x, head_dim, dtype) && aligned(out, 16);
        (i == 0 ? a.q : a.k) = heads_arg(x);
    }
    if (n == 0 || a.q.heads + a.k.heads == 0) return TQ_OK;
    TQ_REQUIRE(positions && aligned(positions, 8), "%s: null or unaligned positions", what);
    a.positions = positions;
    a.rot = rotary_arg(rotary);
    a.d = static_cast<int>(head_dim);
    a.n = static_cast<int>(n);
    a.q_out = q_out;
    a.k_out = k_out;
    return launch_rows_typed<FmtI8>(a, dtype, vec && vec_rotary(a.rot, dtype), as_hip(stream), what);
}

}  // namespace
}  // namespace tq

extern "C" {

int tq_rotary_apply(const tq_rotary* rotary, const int64_t* positions, int64_t n, const tq_heads* q, const tq_heads* k,
                    int dtype, int64_t head_dim, void* q_out, void* k_out, tq_stream_t stream) {
    return tq::apply_rows("tq_rotary_apply", rotary, nullptr, positions, n, q, k, dtype, head_dim, q_out, k_out, stream);
}

int tq_rotary_apply_axes(const tq_rotary* rotary, const tq_rotary_axes* axes, const int64_t* positions, int64_t n,
                         const tq_heads* q, const tq_heads* k, int dtype, int64_t head_dim, void* q_out, void* k_out,
                         tq_stream_t stream) {
    TQ_REQUIRE(axes, "tq_rotary_apply_axes: null axes");
    return tq::apply_rows("tq_rotary_apply_axes", rotary, axes, positions, n, q, k, dtype, head_dim, q_out, k_out, stream);
}

int tq_kv_write(const tq_kv_cache* cache, const tq_kv_batch* batch, const tq_heads* k, const tq_heads* v, int dtype,
                tq_stream_t stream) {
    return tq::write_rows("tq_kv_write", cache, batch, nullptr, nullptr, nullptr, nullptr, k, v, dtype, nullptr, tq::as_hip(stream));
}

int tq_kv_write_rotary(const tq_kv_cache* cache, const tq_kv_batch* batch, const tq_rotary* rotary,
                       const int64_t* positions, const tq_heads* q, const tq_heads* k, const tq_heads* v, int dtype,
                       void* q_out, tq_stream_t stream) {
    TQ_REQUIRE(rotary, "tq_kv_write_rotary: null rotary");
    TQ_REQUIRE(tq::aligned(positions, 8), "tq_kv_write_rotary: unaligned positions");
    return tq::write_rows("tq_kv_write_rotary", cache, batch, rotary, nullptr, positions, q, k, v, dtype, q_out, tq::as_hip(stream));
}

int tq_kv_write_rotary_axes(const tq_kv_cache* cache, const tq_kv_batch* batch, const tq_rotary* rotary,
                            const tq_rotary_axes* axes, const int64_t* positions, const tq_heads* q, const tq_heads* k,
                            const tq_heads* v, int dtype, void* q_out, tq_stream_t stream) {
    TQ_REQUIRE(rotary && axes, "tq_kv_write_rotary_axes: null rotary or axes");
    TQ_REQUIRE(tq::aligned(positions, 8), "tq_kv_write_rotary_axes: unaligned positions");
    return tq::write_rows("tq_kv_write_rotary_axes", cache, batch, rotary, axes, positions, q, k, v, dtype, q_out, tq::as_hip(stream));
}

int tq_kv_read(const tq_kv_cache* cache, const tq_kv_batch* batch, int dtype, void* k_out, void* v_out,
               tq_stream_t stream) {
    using namespace tq;
    static const char* what = "tq_kv_read";
    ReadArg a{};
    const int rc = kv_check(what, cache, batch, &a.b);
    if (rc != TQ_OK) return rc;
    TQ_REQUIRE(dtype == TQ_DT_F32 || dtype == TQ_DT_BF16 || dtype == TQ_DT_F16, "%s: dtype %d is not f32, bf16 or f16", what,
               dtype);
    if (batch->tokens == 0 || batch->batch == 0) return TQ_OK;
    TQ_REQUIRE(batch->tokens <= kMaxBlocks * kReadTokens, "%s: %lld tokens, %d to a block, are more than %lld blocks", what,
               (long long)batch->tokens, kReadTokens, (long long)kMaxBlocks);
    TQ_REQUIRE(k_out && v_out && aligned(k_out, type_size(dtype)) && aligned(v_out, type_size(dtype)),
               "%s: null or unaligned output", what);
    a.k = cache->k;
    a.k_scale = cache->k_scale;
    a.v = cache->v;
    a.v_scale = cache->v_scale;
    a.heads = static_cast<int>(cache->heads);
    a.d = static_cast<int>(cache->head_dim);
    a.row = static_cast<int>(kv_row(cache->head_dim));
    a.n = static_cast<int>(batch->tokens);
    a.k_out = k_out;
    a.v_out = v_out;
    const bool vec = cache->head_dim % run_of(dtype) == 0 && aligned(k_out, 16) && aligned(v_out, 16);
    return cache->codes == TQ_QINT8 ? launch_read_typed<FmtI8>(a, dtype, vec, as_hip(stream), what)
                                    : launch_read_typed<FmtFp8>(a, dtype, vec, as_hip(stream), what);
}

}  // extern "C"
