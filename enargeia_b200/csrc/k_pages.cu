// Pages of a key/value cache: freeing, forking, growing, compacting and copying them on the device.
//
// A pool holds `pages` pages of `page_tokens` tokens in each layer.  Row r of the table
// ([rows][width]) lists the pages of sequence r in the order of its tokens, lengths[r] says how
// many tokens it holds, refs[p] how many rows hold page p; a page nobody holds is free.  All of it
// lives in device memory and every choice is made there, so a serving step that forks, grows and
// frees needs no answer from the GPU and can be captured into a graph.  All results are integers
// that do not depend on timing: a call takes the lowest free pages in the order of its list.
//
// What bounds them: the bookkeeping is a chain of dependent reads (list -> lengths -> table ->
// counts), so each call is one launch of as few steps as it can be; free and fork spread long
// tables over a cluster, whose barrier separates all checks from the first write.  Copying is HBM
// traffic: 2 * bytes moved.

#include "enx_internal.cuh"
#include "pages_want.h"

namespace enx {

namespace {

constexpr uint32_t kPgThreads = 1024;
constexpr uint32_t kPgMaxRows = 1u << 18;  // the duplicate check's bitmap: 32 KB of shared memory
constexpr uint32_t kPgCluster = 8;         // CTAs of free and fork on long tables

// status bits (include/enx.h)
constexpr int kPgNoneFree = ENX_PAGES_NONE_FREE, kPgBadList = ENX_PAGES_BAD_LIST, kPgBadPage = ENX_PAGES_BAD_PAGE;

struct PagesArgs {
    int32_t* table;
    int32_t* lengths;
    int32_t* refs;
    int32_t* status;
    uint32_t rows, width, pages, page_tokens;
};

__device__ __forceinline__ uint32_t pages_of(uint32_t tokens, uint32_t page_tokens) {
    return (tokens + page_tokens - 1) / page_tokens;
}

// Length of a listed row as the table can hold it (a corrupt negative or overlong one is cut).
__device__ __forceinline__ uint32_t row_length(const PagesArgs& a, int32_t row) {
    const int32_t l = a.lengths[row];
    return l < 0 ? 0u : min((uint32_t)l, a.width * a.page_tokens);
}

// Marks `row` in the bitmap; true if it is in range and not marked yet.
__device__ __forceinline__ bool claim_row(uint32_t* seen, int32_t row, uint32_t rows) {
    if (row < 0 || (uint32_t)row >= rows) return false;
    const uint32_t bit = 1u << (row & 31);
    return !(atomicOr(&seen[row >> 5], bit) & bit);
}

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

}  // namespace

// free: row list[i] keeps its first min(other[i], length) tokens; every page behind those loses a
// holder.  fork (FORK): row list[i], empty so far, becomes another holder of the pages of row other[i].
// Every CTA of the cluster checks the whole list, then takes a part of the rows; the lengths, which
// the checks read, change behind the cluster's barrier.
template <bool FORK>
__global__ void __launch_bounds__(kPgThreads) k_pages_rows(PagesArgs a, const int32_t* __restrict__ list,
                                                           const int32_t* __restrict__ other, uint32_t n) {
    extern __shared__ uint32_t seen[];
    __shared__ int s_bad;
    const uint32_t tid = threadIdx.x, cta = blockIdx.x, ctas = gridDim.x;
    for (uint32_t i = tid; i < (a.rows + 31) / 32; i += kPgThreads) seen[i] = 0;
    if (tid == 0) s_bad = 0;
    __syncthreads();
    for (uint32_t i = tid; i < n; i += kPgThreads) {
        const int32_t row = list[i], o = other[i];
        bool ok = claim_row(seen, row, a.rows) && o >= 0;
        if (FORK) ok = ok && (uint32_t)o < a.rows && a.lengths[row] == 0;
        if (!ok) s_bad = 1;
    }
    __syncthreads();
    if (FORK && !s_bad)  // a row is a source or a destination of one call, not both
        for (uint32_t i = tid; i < n; i += kPgThreads)
            if (seen[other[i] >> 5] >> (other[i] & 31) & 1) s_bad = 1;
    __syncthreads();
    if (s_bad) {  // the same in every CTA: no length changes before all have arrived at the barrier
        if (cta == 0 && tid == 0) atomicOr(a.status, kPgBadList);
        return;
    }
    const uint32_t lane = tid & 31, warps = ctas * (kPgThreads / 32);
    bool corrupt = false;
    for (uint32_t i = cta * (kPgThreads / 32) + (tid >> 5); i < n; i += warps) {
        const int32_t row = list[i], o = other[i];
        const uint32_t len = row_length(a, FORK ? o : row), kept = FORK ? 0 : min(len, (uint32_t)o);
        for (uint32_t k = pages_of(kept, a.page_tokens) + lane; k < pages_of(len, a.page_tokens); k += 32) {
            int32_t* e = a.table + (size_t)row * a.width + k;
            const int32_t p = FORK ? a.table[(size_t)o * a.width + k] : *e;
            *e = FORK ? p : -1;
            if (p >= 0 && (uint32_t)p < a.pages)
                atomicAdd(&a.refs[p], FORK ? 1 : -1);
            else
                corrupt = true;
        }
    }
    cluster_barrier();
    for (uint32_t i = cta * kPgThreads + tid; i < n; i += ctas * kPgThreads) {
        const int32_t row = list[i], o = other[i];
        a.lengths[row] = (int32_t)(FORK ? row_length(a, o) : min(row_length(a, row), (uint32_t)o));
    }
    if (corrupt) atomicOr(a.status, kPgBadPage);
}

namespace {

// Ranks of flagged items among kPgThreads * kPgRun of them, in the order (j, thread): shared
// memory holds a count per (j, warp), turned into exclusive prefixes by one warp.
constexpr uint32_t kPgRun = 8;

struct Ranker {
    uint32_t cnt[kPgRun * 32];
    uint32_t total;
};

// flags: bit j set when this thread's j-th item is flagged.  Returns the number flagged in the
// block; rank_of(j) below gives an item's rank.  All threads call it.
__device__ __forceinline__ uint32_t rank_items(Ranker& r, uint32_t flags) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();  // the previous round's ranks have been read
#pragma unroll
    for (uint32_t j = 0; j < kPgRun; ++j) {
        const uint32_t b = __ballot_sync(0xffffffffu, flags >> j & 1);
        if (lane == 0) r.cnt[j * 32 + warp] = __popc(b);
    }
    __syncthreads();
    if (warp == 0) {
        uint32_t v[kPgRun], sum = 0;
#pragma unroll
        for (uint32_t j = 0; j < kPgRun; ++j) {  // lane owns entries 8 lane .. 8 lane + 7
            v[j] = sum;
            sum += r.cnt[lane * kPgRun + j];
        }
        uint32_t incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
#pragma unroll
        for (uint32_t j = 0; j < kPgRun; ++j) r.cnt[lane * kPgRun + j] = v[j] + incl - sum;
        if (lane == 31) r.total = incl;
    }
    __syncthreads();
    return r.total;
}

__device__ __forceinline__ uint32_t rank_of(const Ranker& r, uint32_t flags, uint32_t j) {
    const uint32_t b = __ballot_sync(0xffffffffu, flags >> j & 1);
    return r.cnt[j * 32 + (threadIdx.x >> 5)] + __popc(b & ((1u << (threadIdx.x & 31)) - 1));
}

}  // namespace

// grow: row list[i] gets the pages that add[i] more tokens need, and the write into a partly filled
// last page that others hold as well is prepared by giving the row a copy of it.  All writers of
// such a page take copies unless nobody else holds it: then the first of them in the list keeps it.
// One CTA: the work is a few words per row, and everything hangs on the order of the list.
// Every row's chain of reads (list, length, table, count) is gone through once and kept in the workspace: each
// further step of it costs more than all the arithmetic.  A thread hands out a row's pages, a warp where there
// are more than kPgFew.  512 rows that each copy or take a page: 10 us (19 with a warp a row and the chains repeated).
// Workspace: writers[pages], first[pages], found[pages], then per row wanted (64 bits), its last page if that
// is shared and about to be written (or -1), and its length.
constexpr uint32_t kPgFew = 4;

__global__ void __launch_bounds__(kPgThreads) k_pages_grow(PagesArgs a, const int32_t* __restrict__ list,
                                                           const int32_t* __restrict__ add, uint32_t n,
                                                           int32_t* __restrict__ pairs, int32_t* __restrict__ count,
                                                           int32_t* ws) {
    extern __shared__ uint32_t seen[];
    __shared__ int s_bad, s_many;
    __shared__ unsigned long long s_sum[32], s_run;
    __shared__ Ranker ranks;
    int32_t *writers = ws, *first = ws + a.pages, *found = ws + 2 * (size_t)a.pages;
    unsigned long long* wanted = reinterpret_cast<unsigned long long*>(ws + 3 * (size_t)a.pages + (a.pages & 1));
    int32_t* last = reinterpret_cast<int32_t*>(wanted + a.rows);
    uint32_t* lens = reinterpret_cast<uint32_t*>(last + a.rows);
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, pt = a.page_tokens;
    for (uint32_t i = tid; i < (a.rows + 31) / 32; i += kPgThreads) seen[i] = 0;
    if (tid == 0) {
        s_bad = s_many = 0;
        s_run = 0;
        count[0] = count[1] = 0;
    }
    __syncthreads();
    for (uint32_t i = tid; i < n; i += kPgThreads) {
        const int32_t row = list[i], more = add[i];
        bool ok = claim_row(seen, row, a.rows) && more >= 0;
        int32_t shared = -1, len = 0;
        if (ok) {
            len = a.lengths[row];
            ok = len >= 0 && (unsigned long long)len + (uint32_t)more <= (unsigned long long)a.width * pt;
            if (ok && more && len % pt) {
                const int32_t p = a.table[(size_t)row * a.width + len / pt];
                ok = p >= 0 && (uint32_t)p < a.pages;
                if (ok && a.refs[p] > 1) {
                    shared = p;
                    writers[p] = 0;
                    first[p] = 0x7fffffff;
                }
            }
        }
        if (!ok) s_bad = 1;
        last[i] = shared;
        lens[i] = (uint32_t)len;
    }
    __syncthreads();
    if (s_bad) {
        if (tid == 0) atomicOr(a.status, kPgBadList);
        return;
    }
    for (uint32_t i = tid; i < n; i += kPgThreads) {
        const int32_t p = last[i];
        if (p >= 0) {
            atomicAdd(&writers[p], 1);
            atomicMin(&first[p], (int32_t)i);
        }
    }
    __syncthreads();
    // pages and copies wanted by the rows before each one; more pages than there are end the call
    bool enough = true;
    for (uint32_t i0 = 0; i0 < n && enough; i0 += kPgThreads) {
        const uint32_t i = i0 + tid;
        unsigned long long mine = 0;
        if (i < n) {
            const int32_t p = last[i];
            const bool copy = p >= 0 && !(__ldcg(&writers[p]) == a.refs[p] && __ldcg(&first[p]) == (int32_t)i);
            const uint32_t fresh = pages_of(lens[i] + (uint32_t)add[i], pt) - pages_of(lens[i], pt);
            if (fresh > kPgFew) s_many = 1;
            mine = want_of(copy, fresh, a.pages);
        }
        unsigned long long incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        if (lane == 31) s_sum[warp] = incl;
        __syncthreads();
        unsigned long long before = s_run;
        for (uint32_t w = 0; w < warp; ++w) before += s_sum[w];
        if (i < n) wanted[i] = before + incl - mine;
        __syncthreads();
        if (tid == kPgThreads - 1) s_run = before + incl;
        __syncthreads();
        enough = want_pages(s_run) <= a.pages;
    }
    const uint32_t total = enough ? (uint32_t)want_pages(s_run) : 0, copies = want_copies(s_run);
    // the lowest `total` free pages (a page that loses a holder to a copy keeps another one)
    uint32_t have = 0;
    for (uint32_t base = 0; enough && base < a.pages && have < total; base += kPgThreads * kPgRun) {
        uint32_t flags = 0;
#pragma unroll
        for (uint32_t j = 0; j < kPgRun; ++j) {
            const uint32_t p = base + j * kPgThreads + tid;
            if (p < a.pages && a.refs[p] == 0) flags |= 1u << j;
        }
        const uint32_t got = rank_items(ranks, flags);
#pragma unroll
        for (uint32_t j = 0; j < kPgRun; ++j) {
            const uint32_t r = have + rank_of(ranks, flags, j);
            if ((flags >> j & 1) && r < total) found[r] = (int32_t)(base + j * kPgThreads + tid);
        }
        have += got;
    }
    if (!enough || have < total) {  // not enough: nothing has changed
        if (tid == 0) atomicOr(a.status, kPgNoneFree);
        return;
    }
    __syncthreads();
    // the pages behind a row's copy: fresh ones from page `at` of the found ones on
    auto take = [&](int32_t* entries, uint32_t held, uint32_t at, uint32_t k) {
        const int32_t to = found[at + k];
        entries[held + k] = to;
        a.refs[to] = 1;
    };
    for (uint32_t i = tid; i < n; i += kPgThreads) {
        const int32_t row = list[i];
        const uint32_t old = lens[i], held = pages_of(old, pt);
        const unsigned long long at = wanted[i], next = i + 1 < n ? wanted[i + 1] : s_run;
        const uint32_t at_page = (uint32_t)want_pages(at), at_copy = want_copies(at), copy = want_copies(next) - at_copy;
        const uint32_t fresh = (uint32_t)want_pages(next) - at_page - copy;
        int32_t* entries = a.table + (size_t)row * a.width;
        if (copy) {
            const int32_t from = last[i], to = found[at_page];
            entries[old / pt] = to;
            a.refs[to] = 1;
            atomicSub(&a.refs[from], 1);
            pairs[2 * at_copy] = from;
            pairs[2 * at_copy + 1] = to;
        }
        if (fresh <= kPgFew)
            for (uint32_t k = 0; k < fresh; ++k) take(entries, held, at_page + copy, k);
        a.lengths[row] = (int32_t)(old + (uint32_t)add[i]);
    }
    if (s_many)
        for (uint32_t i = warp; i < n; i += kPgThreads / 32) {
            const unsigned long long at = wanted[i], next = i + 1 < n ? wanted[i + 1] : s_run;
            const uint32_t at_page = (uint32_t)want_pages(at), copy = want_copies(next) - want_copies(at);
            const uint32_t fresh = (uint32_t)want_pages(next) - at_page - copy;
            if (fresh > kPgFew)
                for (uint32_t k = lane; k < fresh; k += 32)
                    take(a.table + (size_t)list[i] * a.width, pages_of(lens[i], pt), at_page + copy, k);
        }
    if (tid == 0) {
        count[0] = (int32_t)copies;
        count[1] = (int32_t)total;
    }
}

// compact, step 1: where every page goes when the pages in use close up to the front.  With L
// pages in use, the i-th used page behind L moves into the i-th hole before it.
// Workspace: to[pages] (the new number of every used page), holes[pages], movers[pages], held[pages]
// (the movers' counts).  refs_out may be refs.
__global__ void __launch_bounds__(kPgThreads) k_pages_plan(PagesArgs a, int32_t* refs_out, int32_t* __restrict__ pairs,
                                                           int32_t* __restrict__ count, int32_t* ws) {
    __shared__ Ranker ranks;
    __shared__ uint32_t s_live;
    int32_t *to = ws, *holes = ws + a.pages, *movers = ws + 2 * (size_t)a.pages, *held = ws + 3 * (size_t)a.pages;
    const uint32_t tid = threadIdx.x;
    if (tid == 0) s_live = 0;
    __syncthreads();
    uint32_t live = 0;
    for (uint32_t p = tid; p < a.pages; p += kPgThreads) live += a.refs[p] > 0;
    live = __reduce_add_sync(0xffffffffu, live);
    if ((tid & 31) == 0) atomicAdd(&s_live, live);
    __syncthreads();
    const uint32_t L = s_live;
    uint32_t n_holes = 0, n_movers = 0;
    for (uint32_t base = 0; base < a.pages; base += kPgThreads * kPgRun) {
        int32_t v[kPgRun];
        uint32_t hole = 0, mover = 0;
#pragma unroll
        for (uint32_t j = 0; j < kPgRun; ++j) {
            const uint32_t p = base + j * kPgThreads + tid;
            v[j] = p < a.pages ? a.refs[p] : 0;
            if (p < L && v[j] <= 0) hole |= 1u << j;
            if (p >= L && v[j] > 0) mover |= 1u << j;
        }
#pragma unroll
        for (uint32_t j = 0; j < kPgRun; ++j) {
            const uint32_t p = base + j * kPgThreads + tid;
            if (p < a.pages) {
                to[p] = (int32_t)p;
                refs_out[p] = p < L && v[j] > 0 ? v[j] : 0;
            }
        }
        if (base < L) {  // holes only here
            const uint32_t got = rank_items(ranks, hole);
#pragma unroll
            for (uint32_t j = 0; j < kPgRun; ++j) {
                const uint32_t r = n_holes + rank_of(ranks, hole, j);
                if (hole >> j & 1) holes[r] = (int32_t)(base + j * kPgThreads + tid);
            }
            n_holes += got;
        }
        if (base + kPgThreads * kPgRun > L) {  // movers only here
            const uint32_t got = rank_items(ranks, mover);
#pragma unroll
            for (uint32_t j = 0; j < kPgRun; ++j) {
                const uint32_t r = n_movers + rank_of(ranks, mover, j);
                if (mover >> j & 1) {
                    movers[r] = (int32_t)(base + j * kPgThreads + tid);
                    held[r] = v[j];
                }
            }
            n_movers += got;
        }
    }
    __syncthreads();  // as many holes as movers: L pages are in use
    for (uint32_t r = tid; r < n_movers; r += kPgThreads) {
        to[movers[r]] = holes[r];
        refs_out[holes[r]] = held[r];
        pairs[2 * r] = movers[r];
        pairs[2 * r + 1] = holes[r];
    }
    if (tid == 0) {
        count[0] = (int32_t)n_movers;
        count[1] = (int32_t)L;
    }
}

// compact, step 2: the tables under the new numbers (table_out may be the table).  Entries behind a
// row's length, and such as name no page, become -1.
__global__ void __launch_bounds__(256) k_pages_renumber(PagesArgs a, int32_t* table_out, const int32_t* __restrict__ to) {
    const size_t total = (size_t)a.rows * a.width;
    bool corrupt = false;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (size_t)gridDim.x * blockDim.x) {
        const uint32_t row = (uint32_t)(i / a.width), k = (uint32_t)(i % a.width);
        int32_t p = -1;
        if (k < pages_of(row_length(a, (int32_t)row), a.page_tokens)) {
            p = a.table[i];
            if (p >= 0 && (uint32_t)p < a.pages) {
                p = to[p];
            } else {
                p = -1;
                corrupt = true;
            }
        }
        table_out[i] = p;
    }
    if (corrupt) atomicOr(a.status, kPgBadPage);
}

// copy: page pairs[i][0] onto page pairs[i][1] in every layer, for the first count[0] pairs.  A warp
// per (pair, layer), nine 16-byte loads in flight per lane (a page has a multiple of 4.5 KB in the usual
// shapes); more blocks than the SMs hold, so that they fill up as they empty.  HBM-bound: 526 MB (1190 pages of
// 9216 bytes in 24 layers, read and written) in 86 us, 6.1 TB/s.
__global__ void __launch_bounds__(256) k_pages_copy(uint8_t* pool, uint32_t layers, uint32_t pages, uint32_t page_bytes,
                                                    const int32_t* __restrict__ pairs, uint32_t capacity,
                                                    const int32_t* __restrict__ count, int32_t* status) {
    constexpr uint32_t kInFlight = 9;
    const uint32_t lane = threadIdx.x & 31, chunks = page_bytes / 16;
    const int32_t c = count[0];
    const size_t total = (size_t)min((uint32_t)max(c, 0), capacity) * layers;
    bool corrupt = c < 0 || (uint32_t)c > capacity;
    for (size_t i = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < total; i += (size_t)gridDim.x * 8) {
        const size_t pair = i / layers, layer = i % layers;
        const int32_t from = pairs[2 * pair], onto = pairs[2 * pair + 1];
        if (from < 0 || onto < 0 || (uint32_t)from >= pages || (uint32_t)onto >= pages) {
            corrupt = true;
            continue;
        }
        const uint4* src = reinterpret_cast<const uint4*>(pool + (layer * pages + (uint32_t)from) * page_bytes);
        uint4* dst = reinterpret_cast<uint4*>(pool + (layer * pages + (uint32_t)onto) * page_bytes);
        for (uint32_t b = lane; b < chunks; b += 32 * kInFlight) {
            uint4 v[kInFlight];
#pragma unroll
            for (uint32_t j = 0; j < kInFlight; ++j)
                if (b + 32 * j < chunks) v[j] = ld_stream(src + b + 32 * j);
#pragma unroll
            for (uint32_t j = 0; j < kInFlight; ++j)
                if (b + 32 * j < chunks) dst[b + 32 * j] = v[j];
        }
    }
    if (corrupt) atomicOr(status, kPgBadPage);
}

}  // namespace enx

using namespace enx;

// ---- entry points -------------------------------------------------------------------------------

static enx_status pages_args(PagesArgs* a, int32_t* table, int32_t* lengths, int32_t* refs, int32_t* status,
                             const enx_pages_dims* d, uint32_t n, const char* who) {
    const std::string w = who;
    if (!d || !table || !lengths || !refs || !status) return fail(ENX_ERR_INVALID, w + ": null pointer");
    if (d->rows == 0 || d->rows > kPgMaxRows) return fail(ENX_ERR_RANGE, w + ": rows must be 1 to 262144");
    if (d->width == 0 || d->pages == 0 || d->pages > (1u << 28))
        return fail(ENX_ERR_RANGE, w + ": width must be positive and pages 1 to 2^28");
    if (d->page_tokens == 0 || (uint64_t)d->width * d->page_tokens > 0x7fffffffull)
        return fail(ENX_ERR_RANGE, w + ": a row may hold 1 to 2^31 - 1 tokens");
    if (n > d->rows) return fail(ENX_ERR_RANGE, w + ": more rows listed than the table has");
    *a = PagesArgs{table, lengths, refs, status, d->rows, d->width, d->pages, d->page_tokens};
    return ENX_OK;
}

// One CTA up to this many table entries (a step of 32 per warp), a cluster of kPgCluster above it.
constexpr uint64_t kPgOneCta = 4096;

template <bool FORK>
static enx_status pages_rows(const PagesArgs& a, const int32_t* list, const int32_t* other, uint32_t n, void* stream) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at{};
    const uint32_t ctas = (uint64_t)n * a.width > kPgOneCta ? kPgCluster : 1;
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kPgThreads);
    cfg.dynamicSmemBytes = (a.rows + 31) / 32 * 4;
    cfg.stream = as_stream(stream);
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = ctas;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    ENX_CUDA(cudaLaunchKernelEx(&cfg, k_pages_rows<FORK>, a, list, other, n));
    return ENX_OK;
}

extern "C" size_t enx_pages_workspace_bytes(uint32_t rows, uint32_t pages) {
    return 4 * (size_t)pages * sizeof(int32_t) + (size_t)rows * 16 + 16;
}

extern "C" enx_status enx_pages_free(int32_t* table, int32_t* lengths, int32_t* refs, const int32_t* rows,
                                     const int32_t* keep, uint32_t n, int32_t* status, const enx_pages_dims* dims,
                                     void* stream) {
    PagesArgs a;
    ENX_TRY(pages_args(&a, table, lengths, refs, status, dims, n, "enx_pages_free"));
    if (n == 0) return ENX_OK;
    if (!rows || !keep) return fail(ENX_ERR_INVALID, "enx_pages_free: null pointer");
    return pages_rows<false>(a, rows, keep, n, stream);
}

extern "C" enx_status enx_pages_fork(int32_t* table, int32_t* lengths, int32_t* refs, const int32_t* src,
                                     const int32_t* dst, uint32_t n, int32_t* status, const enx_pages_dims* dims,
                                     void* stream) {
    PagesArgs a;
    ENX_TRY(pages_args(&a, table, lengths, refs, status, dims, n, "enx_pages_fork"));
    if (n == 0) return ENX_OK;
    if (!src || !dst) return fail(ENX_ERR_INVALID, "enx_pages_fork: null pointer");
    return pages_rows<true>(a, dst, src, n, stream);
}

extern "C" enx_status enx_pages_grow(int32_t* table, int32_t* lengths, int32_t* refs, const int32_t* rows,
                                     const int32_t* add, uint32_t n, int32_t* pairs, int32_t* count, int32_t* status,
                                     const enx_pages_dims* dims, void* workspace, void* stream) {
    PagesArgs a;
    ENX_TRY(pages_args(&a, table, lengths, refs, status, dims, n, "enx_pages_grow"));
    if (!count || !workspace || (n && (!rows || !add || !pairs)))
        return fail(ENX_ERR_INVALID, "enx_pages_grow: null pointer");
    if (reinterpret_cast<uintptr_t>(workspace) % 8) return fail(ENX_ERR_INVALID, "enx_pages_grow: workspace must be 8-byte aligned");
    k_pages_grow<<<1, kPgThreads, (a.rows + 31) / 32 * 4, as_stream(stream)>>>(a, rows, add, n, pairs, count,
                                                                              static_cast<int32_t*>(workspace));
    ENX_CUDA(cudaGetLastError());
    return ENX_OK;
}

extern "C" enx_status enx_pages_compact(const int32_t* table, const int32_t* lengths, const int32_t* refs,
                                        int32_t* table_out, int32_t* refs_out, int32_t* pairs, int32_t* count,
                                        int32_t* status, const enx_pages_dims* dims, void* workspace, void* stream) {
    PagesArgs a;
    ENX_TRY(pages_args(&a, const_cast<int32_t*>(table), const_cast<int32_t*>(lengths), const_cast<int32_t*>(refs),
                       status, dims, 0, "enx_pages_compact"));
    if (!table_out || !refs_out || !pairs || !count || !workspace)
        return fail(ENX_ERR_INVALID, "enx_pages_compact: null pointer");
    int32_t* ws = static_cast<int32_t*>(workspace);
    k_pages_plan<<<1, kPgThreads, 0, as_stream(stream)>>>(a, refs_out, pairs, count, ws);
    ENX_CUDA(cudaGetLastError());
    const uint64_t entries = (uint64_t)a.rows * a.width;
    const uint32_t blocks = (uint32_t)((entries + 255) / 256 < 148 * 8 ? (entries + 255) / 256 : 148 * 8);
    k_pages_renumber<<<blocks, 256, 0, as_stream(stream)>>>(a, table_out, ws);
    ENX_CUDA(cudaGetLastError());
    return ENX_OK;
}

extern "C" enx_status enx_pages_copy(void* pool, uint32_t layers, uint32_t pages, uint32_t page_bytes,
                                     const int32_t* pairs, uint32_t capacity, const int32_t* count, int32_t* status,
                                     void* stream) {
    if (!pool || !count || !status || (capacity && !pairs)) return fail(ENX_ERR_INVALID, "enx_pages_copy: null pointer");
    if (page_bytes == 0 || page_bytes % 16 || reinterpret_cast<uintptr_t>(pool) % 16)
        return fail(ENX_ERR_INVALID, "enx_pages_copy: pages must be a positive multiple of 16 bytes, 16-byte aligned");
    if (layers == 0 || pages == 0 || pages > (1u << 28)) return fail(ENX_ERR_RANGE, "enx_pages_copy: layers must be positive and pages 1 to 2^28");
    if (capacity == 0) return ENX_OK;
    const uint64_t warps = (uint64_t)capacity * layers, blocks = (warps + 7) / 8;
    k_pages_copy<<<(uint32_t)(blocks < 148 * 64 ? blocks : 148 * 64), 256, 0, as_stream(stream)>>>(
        static_cast<uint8_t*>(pool), layers, pages, page_bytes, pairs, capacity, count, status);
    ENX_CUDA(cudaGetLastError());
    return ENX_OK;
}
