// tq_kv.h -- what the cache kernels share: where a row of a call lies in its sequence
// and on which page, and the host's checks of the descriptors.
#pragma once

#include "tq_internal.h"

namespace tq {

constexpr int64_t kKvMaxHeadDim = 128;
constexpr int64_t kKvMaxPage = 1 << 16;
constexpr int64_t kKvMaxRows = 1 << 30;  // rows, heads and tokens stay 32-bit in the kernels

__host__ __device__ inline int64_t kv_row(int64_t head_dim) { return (head_dim + 31) / 32 * 32; }

// x / d and x % d for 0 <= x < 2^31 by a multiplication: m = floor((2^32 - 1) / d) gives the
// quotient or one less (the estimate falls short by x (2^32 - m d) / (d 2^32) < 1).
struct FastDiv {
    uint32_t d, m;
    FastDiv() = default;
    explicit FastDiv(uint32_t v) : d(v), m(0xFFFFFFFFu / v) {}
    __device__ __forceinline__ uint32_t div(uint32_t x) const {
        const uint32_t q = __umulhi(x, m);
        return q + (x - q * d >= d ? 1u : 0u);
    }
};

// The batch as a kernel takes it (tq_kv_batch with the cache's page size).
struct KvBatch {
    const int32_t* table;
    int64_t table_stride;
    const int32_t* lengths;
    const int32_t* offsets;
    int batch, max_tokens, tokens, table_pages, pages, page, cap;  // cap: table_pages * page
    FastDiv by_page, by_tokens;
};

// A row's place: its sequence, position there, and slot = page * page_size + offset, -1 where
// it has none.  `behind`: a row behind the last sequence.
struct KvPlace {
    int64_t slot;
    int pos;
    bool behind;
};

// Whether rows first .. last - 1 are a sequence's: some, inside the call's and no more than max_tokens.  Those of others have
// no place.
__device__ __forceinline__ bool kv_rows_fit(const KvBatch& b, int first, int last) {
    return first >= 0 && last <= b.tokens && last > first && last - first <= b.max_tokens;
}

// Sequence of row n: the number of sequences that end at or before it.  Called by whole waves
// with a uniform n.
__device__ __forceinline__ int kv_sequence(const KvBatch& b, int n, int lane) {
    if (!b.offsets) return static_cast<int>(b.by_tokens.div(static_cast<uint32_t>(n)));
    int seq = 0;
    for (int i = 0; i < b.batch; i += 64) {
        const bool ended = i + lane < b.batch && b.offsets[i + lane + 1] <= n;
        seq += __popcll(__ballot(ended));
    }
    return seq;
}

// Lane t < 16: the sequence of row n0 + t (of n), all sixteen by the same loads.  Called by one whole wave.
__device__ __forceinline__ int kv_sequences16(const KvBatch& b, int n0, int n, int lane) {
    if (!b.offsets) return static_cast<int>(b.by_tokens.div(static_cast<uint32_t>(min(n0 + lane, n - 1))));
    int seq = 0;
    for (int i = 0; i < b.batch; i += 64) {
        const int ends = i + lane < b.batch ? b.offsets[i + lane + 1] : INT32_MAX;
#pragma unroll
        for (int t = 0; t < 16; ++t) {
            const int ended = __popcll(__ballot(ends <= n0 + t));
            seq += lane == t ? ended : 0;
        }
    }
    return seq;
}

__device__ __forceinline__ KvPlace kv_place(const KvBatch& b, int n, int seq) {
    KvPlace p{-1, -1, seq >= b.batch};
    if (p.behind) return p;
    const int first = b.offsets ? b.offsets[seq] : seq * b.max_tokens;
    const int last = b.offsets ? b.offsets[seq + 1] : first + b.max_tokens;
    if (n < first || !kv_rows_fit(b, first, last)) return p;
    const int64_t pos = static_cast<int64_t>(b.lengths[seq]) - (last - n);
    if (pos < 0 || pos >= b.cap) {
        p.pos = pos < 0 ? -1 : b.cap;
        return p;
    }
    p.pos = static_cast<int>(pos);
    const int i = static_cast<int>(b.by_page.div(static_cast<uint32_t>(p.pos)));
    const int page = b.table[seq * b.table_stride + i];
    if (page >= 0 && page < b.pages) p.slot = static_cast<int64_t>(page) * b.page + (p.pos - i * b.page);
    return p;
}

// Host: fills `out` from the descriptors after checking them; `what` names the entry point.
int kv_check(const char* what, const tq_kv_cache* cache, const tq_kv_batch* batch, KvBatch* out);
int kv_check_heads(const char* what, const char* name, const tq_heads* x, int64_t heads, int64_t head_dim, int dtype);

}  // namespace tq
