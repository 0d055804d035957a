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
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kQuantBlock + threadIdx.x;
    if (i >= total) return;
    const int row = static_cast<int>(i / k), col = static_cast<int>(i - static_cast<int64_t>(row) * k);
    w[i] = FmtFp8::value1(q[i], s[static_cast<int64_t>(row / kBlk) * ((k + kBlk - 1) / kBlk) + col / kBlk]);
}

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

int gemm_block(const uint8_t* qa, const float* sa, const uint8_t* qw, const float* sw, const float* bias, int64_t m,
               int64_t n, int64_t k, void* ws, int64_t ws_bytes, float* y, hipStream_t st, const char* what) {
    int rc = check_sizes(what, m, n, k);
    if (rc != TQ_OK) return rc;
    if (m == 0 || n == 0) return TQ_OK;
    TQ_REQUIRE(y && (k == 0 || (qa && sa && qw && sw)), "%s: null pointer", what);
    TQ_REQUIRE(aligned(qa, 16) && aligned(sa, 4) && aligned(sw, 4) && aligned(y, 4) && aligned(bias, 4),
               "%s: misaligned pointer", what);
    const TilePlan plan = tile_plan<GemmF8Block>(m, n, k, nullptr, true);
    TQ_REQUIRE(plan.part_bytes == 0 || (ws && aligned(ws, 256) && ws_bytes >= plan.part_bytes),
               "%s: workspace of %lld bytes (256-byte aligned), %lld needed", what, (long long)ws_bytes,
               (long long)plan.part_bytes);
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
    TQ_REQUIRE((groups + 15) / 16 < (int64_t(1) << 31), "%s: M=%lld, K=%lld", what, (long long)m, (long long)k);
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
    TQ_REQUIRE(blocks < (int64_t(1) << 31), "%s: N=%lld, K=%lld", what, (long long)n, (long long)k);
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
    const int64_t grid = (n * k + kQuantBlock - 1) / kQuantBlock;
    TQ_REQUIRE(grid < (int64_t(1) << 31), "%s: N=%lld, K=%lld", what, (long long)n, (long long)k);
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
    return tile_plan<GemmF8Block>(m, n, k, nullptr, true).part_bytes;
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
    const BlockLayout lay = block_layout(m, k);
    uint8_t* q = static_cast<uint8_t*>(workspace);
    float* s = reinterpret_cast<float*>(q + lay.sa);
    if ((rc = quantize_g128(x, dtype, m, k, q, s, as_hip(stream), what)) != TQ_OK) return rc;
    return gemm_block(q, s, qw, sw, bias, m, n, k, q + lay.part, need - lay.part, y, as_hip(stream), what);
}

}  // extern "C"
