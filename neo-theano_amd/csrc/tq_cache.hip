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
#include <cmath>

#include "tq_kv.h"
#include "tq_rowfmt.h"

namespace tq {
namespace {

constexpr int kGroup = 16;              // lanes of a head
constexpr int kPer = 8;                 // elements of a lane
constexpr int kRowBlock = 256;          // 16 heads at a time
constexpr int kHeadsAtOnce = kRowBlock / kGroup;

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
    __device__ static _Float16 from(float v) { return static_cast<_Float16>(v); }
};

// Element i of lane l: 8 l + i where whole vectors are moved, l + 16 i element by element.
template <bool kVec>
__device__ __forceinline__ int elem(int l, int i) {
    return kVec ? kPer * l + i : l + kGroup * i;
}

template <int kType, bool kVec>
__device__ __forceinline__ void load_head(const typename Elem<kType>::type* p, int l, int at, int d, float (&x)[kPer]) {
    typedef typename Elem<kType>::type T;
    if constexpr (kVec) {  // 8 adjacent elements from `at` (d % 8 == 0, 16-byte aligned)
        typedef T V __attribute__((ext_vector_type(kPer), aligned(16)));
        V v{};
        if (at < d) v = *reinterpret_cast<const V*>(p + at);
#pragma unroll
        for (int i = 0; i < kPer; ++i) x[i] = Elem<kType>::to(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) x[i] = elem<false>(l, i) < d ? Elem<kType>::to(p[elem<false>(l, i)]) : 0.f;
    }
}

template <int kType, bool kVec>
__device__ __forceinline__ void store_head(typename Elem<kType>::type* p, int l, int d, const float (&x)[kPer]) {
    typedef typename Elem<kType>::type T;
    if constexpr (kVec) {
        typedef T V __attribute__((ext_vector_type(kPer), aligned(16)));
        V v;
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[i] = Elem<kType>::from(x[i]);
        if (kPer * l < d) *reinterpret_cast<V*>(p + kPer * l) = v;
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (elem<false>(l, i) < d) p[elem<false>(l, i)] = Elem<kType>::from(x[i]);
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
    if constexpr (kVec) {  // half % 8 == 0: a lane's elements share their side
        const int e = kPer * l;
        load_head<kType, true>(p, l, e < r.half ? e + r.half : e < 2 * r.half ? e - r.half : d, d, y);
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = elem<false>(l, i);
            y[i] = e >= 2 * r.half ? 0.f : Elem<kType>::to(p[r.pairs ? e ^ 1 : e < r.half ? e + r.half : e - r.half]);
        }
    }
}

// Cosine and signed sine of the lane's own elements (the same in all of the token's heads); elements
// that pass have plane -1.
template <bool kVec>
struct LaneAngles {
    float c[kPer], s[kPer];
    bool on[kPer];
    __device__ LaneAngles(int l, const RotaryArg& r, const float* cs, const float* sn) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = elem<kVec>(l, i);
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

// row_scale in f32: the f64 quotient of two f32 values rounds to f32 as the f32 division does (53 >= 2 24 + 2
// bits), and rounding keeps the order, so the floor may be applied after it.  A f64 division for each head cost
// more than coding it.
template <class Fmt>
__device__ __forceinline__ float head_scale(float absmax) {
    return fmaxf(absmax / static_cast<float>(Fmt::kQmax), static_cast<float>(1e-10));
}

struct RowsArg {
    HeadsArg q, k, v;
    const int64_t* positions;
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

// Block (token, share of its heads).  The heads of q, k and v are taken one kind after the other, 16 kU at
// a time (a group of 16 lanes has kU heads, whose loads are issued together, the first ones before the
// token's place and angles are known).  blockIdx.y counts such shares, or, where the grid has one block
// for a token, it takes them all.
template <int kType, bool kVec, int kU, class Fmt>
__global__ __launch_bounds__(kRowBlock) void k_token_rows(RowsArg a) {
    typedef typename Elem<kType>::type T;
    typedef typename Fmt::code_t C;
    constexpr int kShare = kU * kHeadsAtOnce;
    __shared__ float cs[kKvMaxHeadDim / 2], sn[kKvMaxHeadDim / 2];
    const int n = blockIdx.x, tid = threadIdx.x, l = tid % kGroup, j = tid / kGroup;

    // the share: kind 0 q, 1 k, 2 v, and its first head; uniform
    auto heads_of = [&](int kind) { return kind == 0 ? a.q.heads : kind == 1 ? a.k.heads : a.v.heads; };
    int kind = 0, h0 = 0;
    auto skip_empty = [&]() {
        while (kind < 3 && h0 >= heads_of(kind)) {
            ++kind;
            h0 = 0;
        }
    };
    skip_empty();
    for (int i = 0; i < static_cast<int>(blockIdx.y); ++i) {
        h0 += kShare;
        skip_empty();
    }
    if (kind == 3) return;

    float x[kU][kPer], y[kU][kPer];
    auto load = [&]() {
        const HeadsArg& src = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
        const T* base = static_cast<const T*>(src.data) + n * src.token;
        const bool others = a.rot.half && kind < 2 && !(kVec && a.rot.pairs);
#pragma unroll
        for (int u = 0; u < kU; ++u) {  // past the last head: the last one again, not stored
            const T* p = base + min(h0 + u * kHeadsAtOnce + j, src.heads - 1) * src.head;
            load_head<kType, kVec>(p, l, kPer * l, a.d, x[u]);
            if (others) load_others<kType, kVec>(p, l, a.d, a.rot, y[u]);
        }
    };
    load();
    KvPlace place{-1, -1, false};
    if (a.b.lengths) {
        place = kv_place(a.b, n, kv_sequence(a.b, n, tid & 63));
        if (place.behind) return;  // the whole block: left as it was
    }
    if (a.rot.half) {
        const double pos = static_cast<double>(a.positions ? a.positions[n] : place.pos);
        if (tid < a.rot.half) {
            float c, s;
            cos_sin_turns(pos * (a.rot.f[tid] * 0.15915494309189535), c, s);
            cs[tid] = c * a.rot.scale;
            sn[tid] = (a.rot.inverse ? -s : s) * a.rot.scale;
        }
        __syncthreads();
    }
    const LaneAngles<kVec> angles(l, a.rot, cs, sn);
    const int64_t page = place.slot < 0 ? 0 : place.slot / a.b.page, off = place.slot - page * a.b.page;
    while (true) {
        const int of = heads_of(kind);
        if (a.rot.half && kind < 2) {
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                if (kVec && a.rot.pairs) {
#pragma unroll
                    for (int i = 0; i < kPer; ++i) y[u][i] = x[u][i ^ 1];
                }
                angles.turn(x[u], y[u]);
            }
        }
        T* out = static_cast<T*>(kind == 0 ? a.q_out : kind == 1 ? a.k_out : nullptr);
        if (out) {
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int h = h0 + u * kHeadsAtOnce + j;
                if (h < of) store_head<kType, kVec>(out + (static_cast<int64_t>(n) * of + h) * a.d, l, a.d, x[u]);
            }
        } else if (place.slot >= 0) {
            C* codes0 = static_cast<C*>(kind == 1 ? a.k_codes : a.v_codes);
            float* scale = kind == 1 ? a.k_scale : a.v_scale;
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int h = h0 + u * kHeadsAtOnce + j;
                if (h >= of) continue;
                float m = -INFINITY;
#pragma unroll
                for (int i = 0; i < kPer; ++i)
                    if (elem<kVec>(l, i) < a.d) m = fmaxf(m, fabsf(x[u][i]));
                const float sc = head_scale<Fmt>(absmax_finish(group_max<kGroup>(m)));
                const typename Fmt::Row coder(sc);
                const int64_t at = (page * of + h) * a.b.page + off;
                C* codes = codes0 + at * a.row;
                if (l == 0) scale[at] = sc;
                if constexpr (kVec) {
                    if (kPer * l < a.row)  // zeros past the head
                        *reinterpret_cast<uint2*>(codes + kPer * l) =
                            make_uint2(coder.code4(f32x4{x[u][0], x[u][1], x[u][2], x[u][3]}),
                                       coder.code4(f32x4{x[u][4], x[u][5], x[u][6], x[u][7]}));
                } else {
#pragma unroll
                    for (int i = 0; i < kPer; ++i)
                        if (elem<false>(l, i) < a.row) codes[elem<false>(l, i)] = coder.code1(x[u][i]);
                }
            }
        }
        if (gridDim.y > 1) return;
        h0 += kShare;
        skip_empty();
        if (kind == 3) return;
        load();
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

// Block: 16 adjacent tokens, a group of lanes each (so that a page's codes and scales are
// read in runs), over the heads of its share, four at a time.
template <int kType, bool kVec, class Fmt>
__global__ __launch_bounds__(kRowBlock) void k_read_rows(ReadArg a) {
    typedef typename Elem<kType>::type T;
    typedef typename Fmt::code_t C;
    constexpr int kU = 4;
    __shared__ int64_t slots[kHeadsAtOnce];
    const int tid = threadIdx.x, l = tid % kGroup, j = tid / kGroup, n0 = blockIdx.x * kHeadsAtOnce;
    if (tid < 64) {
        // lane t: the sequence of row n0 + t, all sixteen by the same loads
        int seq = 0;
        if (!a.b.offsets) {
            seq = static_cast<int>(a.b.by_tokens.div(static_cast<uint32_t>(min(n0 + tid, a.n - 1))));
        } else {
            for (int i = 0; i < a.b.batch; i += 64) {
                const int ends = i + tid < a.b.batch ? a.b.offsets[i + tid + 1] : INT32_MAX;
#pragma unroll
                for (int t = 0; t < kHeadsAtOnce; ++t) {
                    const int ended = __popcll(__ballot(ends <= n0 + t));
                    seq += tid == t ? ended : 0;
                }
            }
        }
        if (tid < kHeadsAtOnce && n0 + tid < a.n) {
            const KvPlace p = kv_place(a.b, n0 + tid, seq);
            slots[tid] = p.behind ? -2 : p.slot;
        }
    }
    __syncthreads();
    const int n = n0 + j;
    if (n >= a.n) return;
    const int64_t slot = slots[j];
    if (slot == -2) return;  // left as it was
    const int64_t page = slot < 0 ? 0 : slot / a.b.page, off = slot < 0 ? 0 : slot - page * a.b.page;
    const float zero = slot < 0 ? 0.f : 1.f;
    for (int h0 = blockIdx.y * kU; h0 < 2 * a.heads; h0 += gridDim.y * kU) {
        uint32_t c[kU][kPer / 4];
        C one[kU][kPer];
        float sc[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int h = min(h0 + u, 2 * a.heads - 1);
            const bool is_k = h < a.heads;
            const int64_t at = (page * a.heads + (is_k ? h : h - a.heads)) * a.b.page + off;
            const C* codes = static_cast<const C*>(is_k ? a.k : a.v) + at * a.row;
            sc[u] = (is_k ? a.k_scale : a.v_scale)[at];
            if constexpr (kVec) {
                const uint2 w = *reinterpret_cast<const uint2*>(codes + min(kPer * l, a.row - kPer));
                c[u][0] = w.x;
                c[u][1] = w.y;
            } else {
#pragma unroll
                for (int i = 0; i < kPer; ++i) one[u][i] = codes[min(elem<false>(l, i), a.row - 1)];
            }
        }
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int h = h0 + u;
            if (h >= 2 * a.heads) continue;
            const bool is_k = h < a.heads;
            float x[kPer];
            if constexpr (kVec) {
                const f32x4 v = Fmt::value4(c[u][0], sc[u]), w = Fmt::value4(c[u][1], sc[u]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = v[i];
                    x[4 + i] = w[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < kPer; ++i) x[i] = Fmt::value1(one[u][i], sc[u]);
            }
#pragma unroll
            for (int i = 0; i < kPer; ++i) x[i] = zero != 0.f ? x[i] : 0.f;
            store_head<kType, kVec>(static_cast<T*>(is_k ? a.k_out : a.v_out) +
                                        (static_cast<int64_t>(n) * a.heads + (is_k ? h : h - a.heads)) * a.d,
                                    l, a.d, x);
        }
    }
}

int64_t type_size(int dtype) { return dtype == TQ_DT_F32 ? 4 : 2; }

bool vec_rows(const tq_heads* x, int64_t d, int dtype) {
    return !x || x->heads == 0 ||
           (aligned(x->data, 16) && d % kPer == 0 && x->token_stride * type_size(dtype) % 16 == 0 &&
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

RotaryArg rotary_arg(const tq_rotary* r) {
    return RotaryArg{r->frequencies, static_cast<int>(r->rotary_dim / 2), r->interleaved != 0, r->inverse != 0, r->scale};
}

// One block for a token where there are tokens enough to fill the chip, else one for every 16 heads of
// a kind.
template <int kType, bool kVec, class Fmt>
void launch_rows_vec(const RowsArg& a, hipStream_t st) {
    auto shares = [](int heads) { return (heads + kHeadsAtOnce - 1) / kHeadsAtOnce; };
    if (a.n >= 4 * device_cu_count())
        k_token_rows<kType, kVec, 2, Fmt><<<dim3(a.n, 1), kRowBlock, 0, st>>>(a);
    else
        k_token_rows<kType, kVec, 1, Fmt>
            <<<dim3(a.n, shares(a.q.heads) + shares(a.k.heads) + shares(a.v.heads)), kRowBlock, 0, st>>>(a);
}

template <int kType, class Fmt>
int launch_rows(const RowsArg& a, bool vec, hipStream_t st, const char* what) {
    clear_error();
    if (vec)
        launch_rows_vec<kType, true, Fmt>(a, st);
    else
        launch_rows_vec<kType, false, Fmt>(a, st);
    return check_launch(what);
}

template <class Fmt>
int launch_rows_typed(const RowsArg& a, int dtype, bool vec, hipStream_t st, const char* what) {
    if (dtype == TQ_DT_F32) return launch_rows<TQ_DT_F32, Fmt>(a, vec, st, what);
    if (dtype == TQ_DT_BF16) return launch_rows<TQ_DT_BF16, Fmt>(a, vec, st, what);
    return launch_rows<TQ_DT_F16, Fmt>(a, vec, st, what);
}

// A lane's 8 elements turn against 8 adjacent ones: halves of whole eights.
bool vec_rotary(const RotaryArg& r) { return r.pairs || r.half % kPer == 0; }

int write_rows(const char* what, const tq_kv_cache* cache, const tq_kv_batch* batch, const tq_rotary* rotary,
               const int64_t* positions, const tq_heads* q, const tq_heads* k, const tq_heads* v, int dtype, void* q_out,
               hipStream_t st) {
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
        a.rot = rotary_arg(rotary);
        a.positions = positions;
        vec = vec && vec_rotary(a.rot);
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

template <int kType, class Fmt>
int launch_read(const ReadArg& a, bool vec, hipStream_t st, const char* what) {
    const int blocks = (a.n + kHeadsAtOnce - 1) / kHeadsAtOnce;
    // all heads in a block where there are blocks enough, else four to a block
    const dim3 grid(blocks, blocks >= 4 * device_cu_count() ? 1 : (2 * a.heads + 3) / 4);
    clear_error();
    if (vec)
        k_read_rows<kType, true, Fmt><<<grid, kRowBlock, 0, st>>>(a);
    else
        k_read_rows<kType, false, Fmt><<<grid, kRowBlock, 0, st>>>(a);
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
    TQ_REQUIRE(b->table_pages * c->page <= kKvMaxRows, "%s: a table of %lld pages of %lld tokens is longer than 2^30 tokens",
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

extern "C" {

int tq_rotary_apply(const tq_rotary* rotary, const int64_t* positions, int64_t n, const tq_heads* q, const tq_heads* k,
                    int dtype, int64_t head_dim, void* q_out, void* k_out, tq_stream_t stream) {
    using namespace tq;
    static const char* what = "tq_rotary_apply";
    int rc = check_rotary(what, rotary, head_dim);
    if (rc != TQ_OK) return rc;
    TQ_REQUIRE(n >= 0 && n <= kKvMaxRows, "%s: n=%lld", what, (long long)n);
    RowsArg a{};
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
    return launch_rows_typed<FmtI8>(a, dtype, vec && vec_rotary(a.rot), as_hip(stream), what);
}

int tq_kv_write(const tq_kv_cache* cache, const tq_kv_batch* batch, const tq_heads* k, const tq_heads* v, int dtype,
                tq_stream_t stream) {
    return tq::write_rows("tq_kv_write", cache, batch, nullptr, nullptr, nullptr, k, v, dtype, nullptr, tq::as_hip(stream));
}

int tq_kv_write_rotary(const tq_kv_cache* cache, const tq_kv_batch* batch, const tq_rotary* rotary,
                       const int64_t* positions, const tq_heads* q, const tq_heads* k, const tq_heads* v, int dtype,
                       void* q_out, tq_stream_t stream) {
    TQ_REQUIRE(rotary, "tq_kv_write_rotary: null rotary");
    TQ_REQUIRE(tq::aligned(positions, 8), "tq_kv_write_rotary: unaligned positions");
    return tq::write_rows("tq_kv_write_rotary", cache, batch, rotary, positions, q, k, v, dtype, q_out, tq::as_hip(stream));
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
    const bool vec = cache->head_dim % kPer == 0 && aligned(k_out, 16) && aligned(v_out, 16);
    return cache->codes == TQ_QINT8 ? launch_read_typed<FmtI8>(a, dtype, vec, as_hip(stream), what)
                                    : launch_read_typed<FmtFp8>(a, dtype, vec, as_hip(stream), what);
}

}  // extern "C"
