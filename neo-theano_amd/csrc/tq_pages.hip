// tq_pages.hip -- what becomes of the cache's pages: tokens that stay of a verified draft, copies of
// pages, and who holds which page.
//
//   keep:  place start + i <- place start + path[i], for each kept token, head, key and value
//   copy:  page target[j] <- page source[j]
//   fork / grow / free: holders[page] = how many sequences name a page, 0 for one that is free
//
// All of it moves bytes or small integers: calls are bound by the latency of a few dependent loads
// (path -> table -> codes), or by HBM where many pages are copied.
#include <algorithm>

#include "tq_kv.h"

namespace tq {
namespace {

constexpr int kBlock = 256;
constexpr int kPoolBlock = 1024;
constexpr int kPoolSequences = 4096;  // of a call that takes pages: their counts lie in LDS

struct KeepArg {
    KvBatch b;
    const int32_t* path;
    int64_t path_stride;
    const int32_t* kept;
    int path_width, heads, row;
    FastDiv by_heads;  // 2 heads: keys and values
    int8_t* codes[2];  // k, v
    float* scales[2];
    int32_t* lengths_out;
};

// A wave for each (sequence, head, key or value).  A lane moves 16 bytes of every (64 / lanes of a row)-th
// kept row: all loads of a step are back before its stores are issued (they are the stores' data), and later
// steps read places behind the ones that earlier steps wrote (path[i] >= i, ascending), so rows move in place.
__global__ __launch_bounds__(kBlock) void k_keep(KeepArg a, int units) {
    const int lane = threadIdx.x & 63, u = blockIdx.x * (kBlock / 64) + threadIdx.x / 64;
    if (u >= units) return;
    const int seq = static_cast<int>(a.by_heads.div(static_cast<uint32_t>(u))), h = (u - seq * 2 * a.heads) >> 1, kv = u & 1;
    const int first = a.b.offsets ? a.b.offsets[seq] : seq * a.b.max_tokens;
    const int last = a.b.offsets ? a.b.offsets[seq + 1] : first + a.b.max_tokens;
    const int length = a.b.lengths[seq], kept = a.kept[seq], count = last - first;
    const int32_t* path = a.path + seq * a.path_stride;
    // a sequence whose rows do not fit or whose path does not ascend inside them stays as it is
    bool fine = kv_rows_fit(a.b, first, last) && kept >= 0 && kept <= min(count, a.path_width);
    for (int i = lane; fine && __ballot(i < kept); i += 64) {
        const int v = i < kept ? path[i] : count, before = i > 0 && i < kept ? path[i - 1] : -1;
        fine = !__ballot(i < kept && (v <= before || v >= count));
    }
    const bool tells = a.lengths_out && h == 0 && kv == 0;  // (uniform)
    if (!fine) {
        if (tells && lane == 0) a.lengths_out[seq] = length;
        return;
    }
    auto at = [&](int r) -> int64_t {  // where new token r of the sequence lies, -1: nowhere
        const int64_t pos = static_cast<int64_t>(length) - count + r;
        if (pos < 0 || pos >= a.b.cap) return -1;
        const int i = static_cast<int>(a.b.by_page.div(static_cast<uint32_t>(pos)));
        const int page = a.b.table[seq * a.b.table_stride + i];
        return page < 0 || page >= a.b.pages ? -1 : (static_cast<int64_t>(page) * a.heads + h) * a.b.page + (static_cast<int>(pos) - i * a.b.page);
    };
    const int lanes = a.row / 16, rows = 64 / lanes, j = lane / lanes, c = lane - j * lanes;
    int end = kept;  // the sequence ends before a kept row that lies nowhere, at whose place another row lies
    for (int i0 = 0; i0 < kept; i0 += rows) {
        const int i = i0 + j;
        int64_t from = -1, to = -1;  // rows of [pages, heads, page]
        if (j < rows && i < kept && path[i] != i) {
            from = at(path[i]);
            to = at(i);
        }
        const bool moves = from >= 0 && to >= 0;
        if (tells) {
            const uint64_t lost = __ballot(from < 0 && to >= 0);
            if (lost) end = min(end, i0 + (__ffsll(static_cast<unsigned long long>(lost)) - 1) / lanes);
        }
        u32x4 v{};
        float s = 0.f;
        if (moves) {
            v = *reinterpret_cast<const u32x4*>(a.codes[kv] + from * a.row + 16 * c);
            if (c == 0) s = a.scales[kv][from];
        }
        if (moves) {
            *reinterpret_cast<u32x4*>(a.codes[kv] + to * a.row + 16 * c) = v;
            if (c == 0) a.scales[kv][to] = s;
        }
    }
    if (tells && lane == 0) a.lengths_out[seq] = length - count + end;
}

// A page's codes of k, of v, its scales of k, of v, as 16-byte units one after the other.
struct CopyArg {
    const int32_t* source;
    const int32_t* target;
    u32x4* codes[2];
    u32x4* scales[2];
    int64_t code_units, scale_units;
    int chunks;  // blocks of a pair
    FastDiv by_chunks;
    int pages;
};

constexpr int kCopyUnits = 4;  // in flight for each lane

__global__ __launch_bounds__(kBlock) void k_copy_pages(CopyArg a) {
    const int pair = static_cast<int>(a.by_chunks.div(blockIdx.x)), chunk = blockIdx.x - pair * a.chunks;
    const int src = a.source[pair], dst = a.target[pair];
    if (src < 0 || src >= a.pages || dst < 0 || dst >= a.pages || src == dst) return;
    const int64_t all = 2 * (a.code_units + a.scale_units);
    u32x4 v[kCopyUnits];
    u32x4* to[kCopyUnits];
#pragma unroll
    for (int i = 0; i < kCopyUnits; ++i) {
        int64_t u = (static_cast<int64_t>(chunk) * kCopyUnits + i) * kBlock + threadIdx.x;
        to[i] = nullptr;
        if (u >= all) continue;
        const bool code = u < 2 * a.code_units;
        if (!code) u -= 2 * a.code_units;
        const int64_t n = code ? a.code_units : a.scale_units;
        const int which = u >= n;
        u32x4* base = code ? a.codes[which] : a.scales[which];
        v[i] = base[src * n + (u - which * n)];
        to[i] = base + dst * n + (u - which * n);
    }
#pragma unroll
    for (int i = 0; i < kCopyUnits; ++i)
        if (to[i]) *to[i] = v[i];
}

// ------------------------------------------------------------------ who holds a page
struct PoolArg {
    int32_t* holders;
    int pages, page;
};

struct ScanLds {
    int64_t waves[kPoolBlock / 64];
};

// Exclusive prefix sums of v over the block, the total in `total`.
__device__ __forceinline__ int64_t block_scan(int64_t v, ScanLds& lds, int64_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t x = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int64_t y = __shfl_up(static_cast<long long>(x), d);
        if (lane >= d) x += y;
    }
    if (lane == 63) lds.waves[wave] = x;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kPoolBlock / 64; ++w) {
        before += w < wave ? lds.waves[w] : 0;
        total += lds.waves[w];
    }
    __syncthreads();
    return before + x - v;
}

// prefix[i] becomes how many pages the sequences before i want (want[i] before the call), cut at the number of
// pages; returns how many all want, cut likewise.
__device__ __forceinline__ int scan_wants(int* prefix, int n, int pages, ScanLds& lds) {
    int64_t given = 0;
    for (int i0 = 0; i0 < n; i0 += kPoolBlock) {
        const int i = i0 + threadIdx.x;
        int64_t total;
        const int64_t before = block_scan(i < n ? prefix[i] : 0, lds, total);
        if (i < n) prefix[i] = static_cast<int>(min(given + before, static_cast<int64_t>(pages)));
        given += total;
    }
    __syncthreads();
    return static_cast<int>(min(given, static_cast<int64_t>(pages)));
}

constexpr int kEach = 8;  // pages of a lane: 8192 holders looked at in one round of loads

// Hands out the `total` lowest free pages: assign(rank, page), ranks ascending with pages, a lane for each of them
// (a lane that handed out those that it finds would work through neighbours one by one: 12 against 7 us for 64 pages).
// list: kPoolBlock * kEach places in LDS.  One block.
template <class Assign>
__device__ __forceinline__ void take_pages(const PoolArg& p, int total, ScanLds& lds, uint16_t* list, Assign assign) {
    int given = 0;
    for (int64_t base = 0; base < p.pages && given < total; base += kPoolBlock * kEach) {
        const int64_t mine = base + threadIdx.x * kEach;
        uint32_t free = 0;
        if (mine + kEach <= p.pages) {
            i32x4 v[kEach / 4];
#pragma unroll
            for (int i = 0; i < kEach / 4; ++i) v[i] = *reinterpret_cast<const i32x4*>(p.holders + mine + 4 * i);
#pragma unroll
            for (int i = 0; i < kEach; ++i) free |= (v[i / 4][i % 4] <= 0 ? 1u : 0u) << i;
        } else {
            for (int i = 0; i < kEach; ++i)
                if (mine + i < p.pages && p.holders[mine + i] <= 0) free |= 1u << i;
        }
        int64_t all;
        int place = static_cast<int>(block_scan(__popc(free), lds, all));
        for (; free; free &= free - 1) list[place++] = static_cast<uint16_t>(threadIdx.x * kEach + __ffs(free) - 1);
        __syncthreads();
        const int count = min(static_cast<int>(all), total - given);
        for (int i = threadIdx.x; i < count; i += kPoolBlock) {
            const int page = static_cast<int>(base) + list[i];
            atomicAdd(p.holders + page, 1);
            assign(given + i, page);
        }
        given += count;
        __syncthreads();
    }
}

// The sequence whose want a rank is: the last one with prefix <= rank (n >= 1, prefix[0] = 0).
__device__ __forceinline__ int owner(const int* prefix, int n, int rank) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (prefix[mid] <= rank) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

struct GrowArg {
    PoolArg pool;
    int32_t* table;
    int64_t stride;
    int table_pages, batch;
    const int32_t* lengths;
    const int32_t* stored;  // or null
};

// Pages that `length` tokens take, up to the table's end.
__device__ __forceinline__ int pages_of(int length, int page, int table_pages) {
    return length <= 0 ? 0 : min(static_cast<int>((static_cast<int64_t>(length) + page - 1) / page), table_pages);
}

__global__ __launch_bounds__(kPoolBlock) void k_grow(GrowArg a) {
    __shared__ int want[kPoolSequences], have[kPoolSequences];
    __shared__ uint16_t list[kPoolBlock * kEach];
    __shared__ ScanLds lds;
    const int lane = threadIdx.x & 63;
    for (int b = threadIdx.x >> 6; b < a.batch; b += kPoolBlock / 64) {
        const int need = pages_of(a.lengths[b], a.pool.page, a.table_pages);
        int end = need;  // behind the last entry that has a page
        while (end > 0) {
            const int i = end - 1 - lane;
            const uint64_t there = __ballot(i >= 0 && a.table[b * a.stride + i] >= 0);
            if (there) {
                end -= __ffsll(static_cast<unsigned long long>(there)) - 1;
                break;
            }
            end = max(end - 64, 0);
        }
        // a page that was missing when its tokens came: what lies on another one now is somebody else's
        if (a.stored) end = max(end, min(pages_of(a.stored[b], a.pool.page, a.table_pages), need));
        if (lane == 0) {
            have[b] = end;
            want[b] = need - end;
        }
    }
    __syncthreads();
    const int total = scan_wants(want, a.batch, a.pool.pages, lds);
    take_pages(a.pool, total, lds, list, [&](int rank, int page) {
        const int b = owner(want, a.batch, rank);
        a.table[b * a.stride + have[b] + (rank - want[b])] = page;
    });
}

// A wave for each sequence: the pages of its tokens that it does not have.
__global__ __launch_bounds__(kBlock) void k_lacking(GrowArg a, int32_t* lacking) {
    const int lane = threadIdx.x & 63;
    for (int b = blockIdx.x * (kBlock / 64) + (threadIdx.x >> 6); b < a.batch; b += gridDim.x * (kBlock / 64)) {
        const int need = pages_of(a.lengths[b], a.pool.page, INT32_MAX), here = min(need, a.table_pages);
        int none = need - here;  // past the table
        for (int i0 = 0; i0 < here; i0 += 64) {
            const int i = i0 + lane;
            const int page = i < here ? a.table[b * a.stride + i] : 0;
            none += __popcll(__ballot(i < here && (page < 0 || page >= a.pool.pages)));
        }
        if (lane == 0) lacking[b] = none;
    }
}

struct ForkArg {
    PoolArg pool;
    const int32_t* table;
    int64_t stride;
    int table_pages, batch, children;
    const int32_t* lengths;
    const int32_t* parents;
    int32_t* out;
    int32_t* source;
    int32_t* target;
};

// Block 0 takes a page for each child whose parent has begun one; the others share the whole pages.  Sharing
// only raises counts of pages that are held, so the free ones are the same for block 0 whenever it looks.
__global__ __launch_bounds__(kPoolBlock) void k_fork(ForkArg a) {
    __shared__ int want[kPoolSequences], begins[kPoolSequences];
    __shared__ uint16_t list[kPoolBlock * kEach];
    __shared__ ScanLds lds;
    auto begun = [&](int c, int& whole) {  // the page that child c's parent has begun, or -1
        const int p = a.parents[c];
        whole = 0;
        if (p < 0 || p >= a.batch) return -1;
        const int length = max(a.lengths[p], 0);
        whole = min(length / a.pool.page, a.table_pages);
        if (whole == a.table_pages || length % a.pool.page == 0) return -1;
        const int page = a.table[p * a.stride + whole];
        return page >= 0 && page < a.pool.pages ? page : -1;
    };
    if (blockIdx.x == 0) {
        for (int c = threadIdx.x; c < a.children; c += kPoolBlock) {
            int whole;
            const int page = begun(c, whole);
            want[c] = page >= 0;
            begins[c] = whole;
            a.source[c] = page;  // (where no page is left: -1 again below)
            a.target[c] = -1;
            if (whole < a.table_pages) a.out[static_cast<int64_t>(c) * a.table_pages + whole] = -1;
        }
        __syncthreads();  // (the writes above too: assign below writes the same places)
        const int total = scan_wants(want, a.children, a.pool.pages, lds);
        take_pages(a.pool, total, lds, list, [&](int rank, int page) {
            const int c = owner(want, a.children, rank);
            a.target[c] = page;
            a.out[static_cast<int64_t>(c) * a.table_pages + begins[c]] = page;
        });
        __syncthreads();
        for (int c = threadIdx.x; c < a.children; c += kPoolBlock)
            if (a.target[c] < 0) a.source[c] = -1;
        return;
    }
    for (int c = blockIdx.x - 1; c < a.children; c += gridDim.x - 1) {
        const int p = a.parents[c];
        const int whole = p < 0 || p >= a.batch ? 0 : min(max(a.lengths[p], 0) / a.pool.page, a.table_pages);
        for (int i = threadIdx.x; i < a.table_pages; i += kPoolBlock) {
            if (i == whole) continue;  // block 0's
            int page = -1;
            if (i < whole) {
                page = a.table[p * a.stride + i];
                if (page >= 0 && page < a.pool.pages) atomicAdd(a.pool.holders + page, 1);
            }
            a.out[static_cast<int64_t>(c) * a.table_pages + i] = page;
        }
    }
}

struct FreeArg {
    PoolArg pool;
    int32_t* table;
    int64_t stride;
    int table_pages, batch;
    const uint8_t* which;
};

__global__ __launch_bounds__(kBlock) void k_free(FreeArg a) {
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
        if (a.which && !a.which[b]) continue;
        for (int i = threadIdx.x; i < a.table_pages; i += kBlock) {
            int32_t* entry = a.table + b * a.stride + i;
            const int page = *entry;
            if (page >= 0 && page < a.pool.pages && atomicSub(a.pool.holders + page, 1) <= 0)
                atomicAdd(a.pool.holders + page, 1);  // was free already: stays at 0
            if (page >= 0) *entry = -1;
        }
    }
}

int check_pool(const char* what, const tq_page_pool* p, PoolArg* out) {
    TQ_REQUIRE(p, "%s: null pool", what);
    TQ_REQUIRE(p->pages >= 1 && p->pages <= INT32_MAX, "%s: a pool of %lld pages", what, (long long)p->pages);
    TQ_REQUIRE(p->page >= 1 && p->page <= kKvMaxPage, "%s: page=%lld is not in 1..65536", what, (long long)p->page);
    TQ_REQUIRE(p->holders && aligned(p->holders, 16), "%s: null or unaligned holders", what);
    *out = PoolArg{p->holders, static_cast<int>(p->pages), static_cast<int>(p->page)};
    return TQ_OK;
}

int check_table(const char* what, const int32_t* table, int64_t stride, int64_t table_pages, int64_t batch, int64_t most) {
    TQ_REQUIRE(batch >= 0 && batch <= most, "%s: %lld sequences, at most %lld", what, (long long)batch, (long long)most);
    TQ_REQUIRE(table_pages >= 0 && table_pages <= kKvMaxRows, "%s: table_pages=%lld", what, (long long)table_pages);
    TQ_REQUIRE(stride >= table_pages || batch <= 1, "%s: table_stride=%lld under %lld pages", what, (long long)stride,
               (long long)table_pages);
    TQ_REQUIRE(batch == 0 || table_pages == 0 || table, "%s: null table", what);
    TQ_REQUIRE(aligned(table, 4), "%s: unaligned table", what);
    return TQ_OK;
}

// Blocks for so many sequences, which they take in turn.
int blocks_for(int64_t sequences) { return static_cast<int>(std::min<int64_t>(sequences, 8 * device_cu_count())); }

int grow(const char* what, const tq_page_pool* pool, int32_t* table, int64_t table_stride, int64_t table_pages, const int32_t* lengths,
         const int32_t* stored, int64_t batch, tq_stream_t stream) {
    GrowArg a{};
    int rc = check_pool(what, pool, &a.pool);
    if (rc != TQ_OK) return rc;
    if ((rc = check_table(what, table, table_stride, table_pages, batch, kPoolSequences)) != TQ_OK) return rc;
    if (batch == 0 || table_pages == 0) return TQ_OK;
    TQ_REQUIRE(lengths && aligned(lengths, 4), "%s: null or unaligned lengths", what);
    TQ_REQUIRE(!overlap({{table, batch, table_stride, table_pages, 4}, {pool->holders, pool->pages, 4}}, {{lengths, batch, 4}, {stored, batch, 4}}),
               "%s: table or holders overlaps the other or lengths", what);
    a.table = table;
    a.stride = table_stride;
    a.table_pages = static_cast<int>(table_pages);
    a.batch = static_cast<int>(batch);
    a.lengths = lengths;
    a.stored = stored;
    clear_error();
    k_grow<<<1, kPoolBlock, 0, as_hip(stream)>>>(a);
    return check_launch(what);
}

}  // namespace
}  // namespace tq

extern "C" {

int tq_kv_keep(const tq_kv_cache* cache, const tq_kv_batch* batch, const int32_t* path, int64_t path_stride, int64_t path_width,
               const int32_t* kept, int32_t* lengths_out, tq_stream_t stream) {
    using namespace tq;
    static const char* what = "tq_kv_keep";
    KeepArg a{};
    const int rc = kv_check(what, cache, batch, &a.b);
    if (rc != TQ_OK) return rc;
    TQ_REQUIRE(path_width >= 0 && path_width <= kKvMaxRows && (path_stride >= path_width || batch->batch <= 1),
               "%s: paths of %lld rows, path_stride=%lld", what, (long long)path_width, (long long)path_stride);
    if (batch->batch == 0) return TQ_OK;
    TQ_REQUIRE((path || path_width == 0) && kept, "%s: null path or kept", what);
    TQ_REQUIRE(aligned(path, 4) && aligned(kept, 4) && aligned(lengths_out, 4), "%s: unaligned path, kept or lengths", what);
    const int64_t held = cache->heads * cache->page, codes = held * kv_row(cache->head_dim);  // of a page
    TQ_REQUIRE(!overlap({{lengths_out, batch->batch, 4}},
                        {{batch->lengths, batch->batch, 4}, {kept, batch->batch, 4}, {path, batch->batch, path_stride, path_width, 4},
                         {batch->table, batch->batch, batch->table_stride, batch->table_pages, 4}, {batch->offsets, batch->batch + 1, 4},
                         {cache->k, cache->pages, codes, codes, 1}, {cache->v, cache->pages, codes, codes, 1},
                         {cache->k_scale, cache->pages, held, held, 4}, {cache->v_scale, cache->pages, held, held, 4}}),
               "%s: lengths_out overlaps the batch's lengths, table or offsets, path, kept or the cache", what);
    const int64_t units = 2 * batch->batch * cache->heads, blocks = (units + 3) / 4;
    TQ_REQUIRE(blocks <= kMaxBlocks, "%s: %lld sequences of %lld heads are more than %lld blocks", what, (long long)batch->batch,
               (long long)cache->heads, (long long)kMaxBlocks);
    a.path = path;
    a.path_stride = path_stride;
    a.path_width = static_cast<int>(path_width);
    a.kept = kept;
    a.heads = static_cast<int>(cache->heads);
    a.by_heads = FastDiv(static_cast<uint32_t>(2 * cache->heads));
    a.row = static_cast<int>(kv_row(cache->head_dim));
    a.codes[0] = static_cast<int8_t*>(cache->k);
    a.codes[1] = static_cast<int8_t*>(cache->v);
    a.scales[0] = cache->k_scale;
    a.scales[1] = cache->v_scale;
    a.lengths_out = lengths_out;
    clear_error();
    k_keep<<<static_cast<int>(blocks), kBlock, 0, as_hip(stream)>>>(a, static_cast<int>(units));
    return check_launch(what);
}

int tq_kv_copy_pages(const tq_kv_cache* cache, const int32_t* source, const int32_t* target, int64_t n, tq_stream_t stream) {
    using namespace tq;
    static const char* what = "tq_kv_copy_pages";
    const tq_kv_batch none{nullptr, 0, 0, nullptr, nullptr, 0, 0, 0};
    KvBatch unused;
    const int rc = kv_check(what, cache, &none, &unused);
    if (rc != TQ_OK) return rc;
    TQ_REQUIRE(n >= 0, "%s: n=%lld", what, (long long)n);
    if (n == 0) return TQ_OK;
    TQ_REQUIRE(source && target && aligned(source, 4) && aligned(target, 4), "%s: null or unaligned source or target", what);
    CopyArg a{};
    a.source = source;
    a.target = target;
    a.codes[0] = static_cast<u32x4*>(cache->k);
    a.codes[1] = static_cast<u32x4*>(cache->v);
    a.scales[0] = reinterpret_cast<u32x4*>(cache->k_scale);
    a.scales[1] = reinterpret_cast<u32x4*>(cache->v_scale);
    a.code_units = cache->heads * cache->page * kv_row(cache->head_dim) / 16;
    a.scale_units = cache->heads * cache->page / 4;  // page is a multiple of 16
    a.pages = static_cast<int>(cache->pages);
    const int64_t chunks = (2 * (a.code_units + a.scale_units) + kCopyUnits * kBlock - 1) / (kCopyUnits * kBlock);
    TQ_REQUIRE(chunks <= kMaxBlocks && n <= kMaxBlocks / chunks, "%s: %lld pages of %lld blocks are more than %lld blocks", what,
               (long long)n, (long long)chunks, (long long)kMaxBlocks);
    a.chunks = static_cast<int>(chunks);
    a.by_chunks = FastDiv(static_cast<uint32_t>(chunks));
    clear_error();
    k_copy_pages<<<static_cast<int>(n * chunks), kBlock, 0, as_hip(stream)>>>(a);
    return check_launch(what);
}

int tq_pages_grow(const tq_page_pool* pool, int32_t* table, int64_t table_stride, int64_t table_pages, const int32_t* lengths,
                  int64_t batch, tq_stream_t stream) {
    return tq::grow("tq_pages_grow", pool, table, table_stride, table_pages, lengths, nullptr, batch, stream);
}

int tq_pages_grow_stored(const tq_page_pool* pool, int32_t* table, int64_t table_stride, int64_t table_pages, const int32_t* lengths,
                         const int32_t* stored, int64_t batch, tq_stream_t stream) {
    static const char* what = "tq_pages_grow_stored";
    TQ_REQUIRE(batch <= 0 || table_pages == 0 || (stored && tq::aligned(stored, 4)), "%s: null or unaligned stored lengths", what);
    return tq::grow(what, pool, table, table_stride, table_pages, lengths, stored, batch, stream);
}

int tq_pages_lacking(const tq_page_pool* pool, const int32_t* table, int64_t table_stride, int64_t table_pages, const int32_t* lengths,
                     int64_t batch, int32_t* lacking, tq_stream_t stream) {
    using namespace tq;
    static const char* what = "tq_pages_lacking";
    GrowArg a{};
    int rc = check_pool(what, pool, &a.pool);
    if (rc != TQ_OK) return rc;
    if ((rc = check_table(what, table, table_stride, table_pages, batch, kKvMaxRows)) != TQ_OK) return rc;
    if (batch == 0) return TQ_OK;
    TQ_REQUIRE(lengths && aligned(lengths, 4) && lacking && aligned(lacking, 4), "%s: null or unaligned lengths or lacking", what);
    TQ_REQUIRE(!overlap({{lacking, batch, 4}}, {{table, batch, table_stride, table_pages, 4}, {lengths, batch, 4}, {pool->holders, pool->pages, 4}}),
               "%s: lacking overlaps the table, lengths or holders", what);
    a.table = const_cast<int32_t*>(table);
    a.stride = table_stride;
    a.table_pages = static_cast<int>(table_pages);
    a.batch = static_cast<int>(batch);
    a.lengths = lengths;
    clear_error();
    k_lacking<<<blocks_for((batch + kBlock / 64 - 1) / (kBlock / 64)), kBlock, 0, as_hip(stream)>>>(a, lacking);
    return check_launch(what);
}

int tq_pages_fork(const tq_page_pool* pool, const int32_t* table, int64_t table_stride, int64_t table_pages, const int32_t* lengths,
                  int64_t batch, const int32_t* parents, int64_t children, int32_t* children_table, int32_t* source,
                  int32_t* target, tq_stream_t stream) {
    using namespace tq;
    static const char* what = "tq_pages_fork";
    ForkArg a{};
    int rc = check_pool(what, pool, &a.pool);
    if (rc != TQ_OK) return rc;
    if ((rc = check_table(what, table, table_stride, table_pages, batch, kKvMaxRows)) != TQ_OK) return rc;
    TQ_REQUIRE(children >= 0 && children <= kPoolSequences, "%s: %lld children, at most %d", what, (long long)children,
               kPoolSequences);
    if (children == 0) return TQ_OK;
    TQ_REQUIRE(parents && source && target && (lengths || batch == 0) && (children_table || table_pages == 0),
               "%s: null lengths, parents, source, target or children", what);
    TQ_REQUIRE(aligned(parents, 4) && aligned(source, 4) && aligned(target, 4) && aligned(lengths, 4) && aligned(children_table, 4),
               "%s: unaligned lengths, parents, source, target or children", what);
    TQ_REQUIRE(!overlap({{children_table, children * table_pages, 4}, {source, children, 4}, {target, children, 4}, {pool->holders, pool->pages, 4}},
                        {{table, batch, table_stride, table_pages, 4}, {lengths, batch, 4}, {parents, children, 4}}),
               "%s: children, source, target or holders overlaps another of them or an input", what);
    a.table = table;
    a.stride = table_stride;
    a.table_pages = static_cast<int>(table_pages);
    a.batch = static_cast<int>(batch);
    a.children = static_cast<int>(children);
    a.lengths = lengths;
    a.parents = parents;
    a.out = children_table;
    a.source = source;
    a.target = target;
    clear_error();
    k_fork<<<1 + blocks_for(children), kPoolBlock, 0, as_hip(stream)>>>(a);
    return check_launch(what);
}

int tq_pages_free(const tq_page_pool* pool, int32_t* table, int64_t table_stride, int64_t table_pages, int64_t batch,
                  const uint8_t* sequences, tq_stream_t stream) {
    using namespace tq;
    static const char* what = "tq_pages_free";
    FreeArg a{};
    int rc = check_pool(what, pool, &a.pool);
    if (rc != TQ_OK) return rc;
    if ((rc = check_table(what, table, table_stride, table_pages, batch, kKvMaxRows)) != TQ_OK) return rc;
    if (batch == 0 || table_pages == 0) return TQ_OK;
    TQ_REQUIRE(!overlap({{table, batch, table_stride, table_pages, 4}, {pool->holders, pool->pages, 4}}, {{sequences, batch, 1}}),
               "%s: table, holders and sequences overlap", what);
    a.table = table;
    a.stride = table_stride;
    a.table_pages = static_cast<int>(table_pages);
    a.batch = static_cast<int>(batch);
    a.which = sequences;
    clear_error();
    k_free<<<blocks_for(batch), kBlock, 0, as_hip(stream)>>>(a);
    return check_launch(what);
}

}  // extern "C"
