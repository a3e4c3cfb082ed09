// Pages of a cache: copied, shared between sequences (fork), taken for new positions (extend), given back (free) and moved
// together (compact).  All of it on the device and in the stream's order, so that a captured graph may hold it.
//
// State, in buffers of the caller's: table int32 [seqs][max_pages] (the pages of a sequence in order, -1 behind them), lens
// int32 [seqs], refs int32 [n_pages] (how many sequences hold a page; 0 = free).  A sequence of n positions holds
// ceil(n / page) pages.  Free pages are always taken lowest first, in the order of the call's list, so that a call's
// result depends on nothing but its inputs.  A call that cannot be carried out (info[0]) changes nothing.
//
// The bookkeeping is one block of 1024 threads: counts and ranks are prefix sums over refs, a few microseconds for ten thousand
// pages.  The data moves in a second launch over all SMs that reads the list of (from, to) pages the first one left in
// scratch; it is bound by HBM (each page in once, out once).  8 sequences branched in 8 each, 268 MB: 48 us with all of the
// bookkeeping; a compaction of 369 MB 69 us.
#include <algorithm>

#include "paged.cuh"
#include "sync_helpers.cuh"
#include "tcgen05_helpers.cuh"

namespace rstq {

constexpr int kPlanThreads = 1024;
constexpr int kListMax = 65536;      // sequences a call names
enum { kInfoOk = 0, kInfoNoPages = 1, kInfoList = 2, kInfoWidth = 3, kInfoShared = 4 };

// scratch of the context: header, then three arrays of n_pages' most
struct PageScratch {
    int* header;     // [0] = pairs to copy
    int* from;       // pages to copy, and where to
    int* to;
    int* map;        // free pages in order (fork, extend); new numbers (compact)
};
static PageScratch page_scratch(const DeviceState& ds) {
    int* p = (int*)ds.page_scratch;
    return {p, p + 64, p + 64 + kMaxPages / 2, p + 64 + kMaxPages};
}
constexpr int64_t kPageScratchBytes = (64 + 2 * kMaxPages) * 4;

struct PageState {
    int32_t *table, *lens, *refs, *info;
    int seqs, n_pages, width, page;
};
// Positions of a sequence, whatever its word says, inside what its pages can hold.
__device__ __forceinline__ int page_len(const PageState& s, int b) {
    return (int)clamp64(s.lens[b], 0, min((int64_t)s.width * s.page, (int64_t)INT32_MAX));
}
__device__ __forceinline__ int pages_of(const PageState& s, int n) { return (int)(((int64_t)n + s.page - 1) / s.page); }

// Sums before this thread over the block, and the block's sum.  All threads call it.
__device__ __forceinline__ int block_scan(int v, int* total, int* s_warp) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
    }
    __syncthreads();                      // the last call's sums have been read
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int w = s_warp[lane];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, w, d);
            if (lane >= d) w += y;
        }
        s_warp[lane] = w;
    }
    __syncthreads();
    *total = s_warp[31];
    return x - v + (warp ? s_warp[warp - 1] : 0);
}
__device__ __forceinline__ int free4(int4 r) { return (r.x <= 0) + (r.y <= 0) + (r.z <= 0) + (r.w <= 0); }
// The counts of pages 4i .. 4i+3; pages behind the last count as held.
__device__ __forceinline__ int4 refs4(const PageState& s, int i) {
    if (4 * i + 3 < s.n_pages) return *reinterpret_cast<const int4*>(s.refs + 4 * i);
    int4 r = make_int4(1, 1, 1, 1);
    if (4 * i < s.n_pages) r.x = s.refs[4 * i];
    if (4 * i + 1 < s.n_pages) r.y = s.refs[4 * i + 1];
    if (4 * i + 2 < s.n_pages) r.z = s.refs[4 * i + 2];
    return r;
}
// Writes the first `want` free pages, in order, to `list`; returns how many pages are free.
__device__ int list_free(const PageState& s, int want, int* list, int* s_warp) {
    int free = 0;
    for (int i0 = 0; 4 * i0 < s.n_pages; i0 += kPlanThreads) {
        const int i = i0 + threadIdx.x, n = free4(refs4(s, i));
        int total;
        int at = free + block_scan(n, &total, s_warp);
        if (n && at < want) {
            const int4 r = refs4(s, i);
            const int v[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (v[j] <= 0) {
                    if (at < want) list[at] = 4 * i + j;
                    ++at;
                }
        }
        free += total;
    }
    return free;
}
__device__ __forceinline__ void say(const PageState& s, int status, int used, int copied, int what) {
    if (threadIdx.x == 0) *reinterpret_cast<int4*>(s.info) = make_int4(status, used, copied, what);
}
// The smallest index of a list at which `bad` holds, or n.  (The second barrier: whoever goes on may write *s_min.)
template <typename F>
__device__ int first_bad(int n, int* s_min, F bad) {
    if (threadIdx.x == 0) *s_min = n;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kPlanThreads)
        if (bad(i)) atomicMin(s_min, i);
    __syncthreads();
    const int first = *s_min;
    __syncthreads();
    return first;
}
__device__ __forceinline__ bool take_bit(uint32_t* bits, int i) {     // true: it was taken already
    return (atomicOr(&bits[i >> 5], 1u << (i & 31)) >> (i & 31)) & 1u;
}
// The smallest index of a list whose entry is no number below `limit`, is wrong by itself, or is there for a second time; n: none.  One look
// at the list says whether there is any, and fills the bitmap; of equal entries it takes for the second one which came later, so where it
// finds any, the places are looked at again, by the first one of each number (first: scratch of `limit` words).
template <typename F>
__device__ int first_wrong(const int32_t* list, int n, int limit, uint32_t* bits, int* s_min, int* first, F wrong) {
    auto outside = [&](int i) { return (uint32_t)list[i] >= (uint32_t)limit || wrong(i); };
    if (first_bad(n, s_min, [&](int i) { return outside(i) || take_bit(bits, list[i]); }) == n) return n;
    for (int i = threadIdx.x; i < n; i += kPlanThreads)
        if ((uint32_t)list[i] < (uint32_t)limit) first[list[i]] = n;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kPlanThreads)
        if ((uint32_t)list[i] < (uint32_t)limit) atomicMin(&first[list[i]], i);
    __syncthreads();
    return first_bad(n, s_min, [&](int i) { return outside(i) || __ldcg(&first[list[i]]) != i; });
}
__device__ __forceinline__ bool has_bit(const uint32_t* bits, int i) { return (bits[i >> 5] >> (i & 31)) & 1u; }
__device__ void clear_bits(uint32_t* bits, int n) {
    for (int i = threadIdx.x; i < (n + 31) / 32; i += kPlanThreads) bits[i] = 0;
    __syncthreads();
}

// Pages of the listed sequences given back.
__global__ void __launch_bounds__(kPlanThreads)
pages_free_kernel(const PageState s, const int32_t* __restrict__ list, const int n, const PageScratch w) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __shared__ uint32_t s_bits[kMaxSeqs / 32];
    __shared__ int s_warp[32], s_min;
    clear_bits(s_bits, s.seqs);
    const int bad = first_wrong(list, n, s.seqs, s_bits, &s_min, w.map, [](int) { return false; });
    if (bad < n) {
        const int used = s.n_pages - list_free(s, 0, nullptr, s_warp);
        say(s, kInfoList, used, 0, bad);
        return;
    }
    // a warp per sequence: its pages lose a holder, its row of the table is empty
    for (int i = threadIdx.x >> 5; i < n; i += kPlanThreads / 32) {
        const int b = list[i], np = pages_of(s, page_len(s, b));
        for (int j = threadIdx.x & 31; j < np; j += 32) {
            const int64_t e = (int64_t)b * s.width + j;
            const int pg = s.table[e];
            if ((uint32_t)pg < (uint32_t)s.n_pages) atomicSub(&s.refs[pg], 1);
            s.table[e] = -1;
        }
        __syncwarp();
        if ((threadIdx.x & 31) == 0) s.lens[b] = 0;
    }
    __syncthreads();
    say(s, kInfoOk, s.n_pages - list_free(s, 0, nullptr, s_warp), 0, 0);
}

// Room for counts[i] more positions of sequence list[i].
__global__ void __launch_bounds__(kPlanThreads)
pages_extend_kernel(const PageState s, const int32_t* __restrict__ list, const int32_t* __restrict__ counts, const int n,
                    const PageScratch w) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __shared__ uint32_t s_bits[kMaxSeqs / 32];
    __shared__ int s_warp[32], s_min;
    clear_bits(s_bits, s.seqs);
    const int64_t room = min((int64_t)s.width * s.page, (int64_t)INT32_MAX);
    int status = kInfoList;
    int bad = first_wrong(list, n, s.seqs, s_bits, &s_min, w.map, [&](int i) { return counts[i] < 0; });
    if (bad == n) {
        status = kInfoWidth;
        bad = first_bad(n, &s_min, [&](int i) { return (int64_t)page_len(s, list[i]) + counts[i] > room; });
    }
    if (bad == n) {     // a page that others hold too is not written to
        status = kInfoShared;
        bad = first_bad(n, &s_min, [&](int i) {
            const int b = list[i], len = page_len(s, b);
            if (!counts[i] || len % s.page == 0) return false;
            const int pg = s.table[(int64_t)b * s.width + len / s.page];
            return (uint32_t)pg >= (uint32_t)s.n_pages || s.refs[pg] != 1;
        });
    }
    if (bad < n) {
        const int used = s.n_pages - list_free(s, 0, nullptr, s_warp);
        say(s, status, used, 0, bad);
        return;
    }
    auto need = [&](int i) {
        const int len = page_len(s, list[i]);
        return pages_of(s, len + counts[i]) - pages_of(s, len);
    };
    int64_t want = 0;
    for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
        int total;
        block_scan(i0 + (int)threadIdx.x < n ? need(i0 + threadIdx.x) : 0, &total, s_warp);
        want += total;
    }
    const int free = list_free(s, (int)min(want, (int64_t)s.n_pages), w.map, s_warp);
    if (want > free) {
        say(s, kInfoNoPages, s.n_pages - free, 0, (int)min(want, (int64_t)INT32_MAX));
        return;
    }
    __syncthreads();
    int base = 0;
    for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
        const int i = i0 + threadIdx.x, k = i < n ? need(i) : 0;
        int total;
        const int at = base + block_scan(k, &total, s_warp);
        const int b = i < n ? list[i] : 0, len = i < n ? page_len(s, b) : 0;
        const int64_t e0 = (int64_t)b * s.width + pages_of(s, len);
        constexpr int kOwn = 2;      // pages that a thread writes itself
        for (int j = 0; j < kOwn; ++j)
            if (j < k) {
                const int pg = w.map[at + j];
                s.table[e0 + j] = pg;
                s.refs[pg] = 1;
            }
        for (uint32_t left = __ballot_sync(0xffffffffu, k > kOwn); left; left &= left - 1) {     // a warp writes the others, sequence by sequence
            const int l = __ffs((int)left) - 1, kl = __shfl_sync(0xffffffffu, k, l), al = __shfl_sync(0xffffffffu, at, l);
            const int64_t el = __shfl_sync(0xffffffffu, e0, l);
            for (int j = kOwn + (threadIdx.x & 31); j < kl; j += 32) {
                const int pg = w.map[al + j];
                s.table[el + j] = pg;
                s.refs[pg] = 1;
            }
        }
        if (i < n) s.lens[b] = len + counts[i];
        base += total;
    }
    say(s, kInfoOk, s.n_pages - free + (int)want, 0, 0);
}

// dst[i] becomes a copy of src[i]: full pages are shared, a partial last one gets a page of its own.
__global__ void __launch_bounds__(kPlanThreads)
pages_fork_kernel(const PageState s, const int32_t* __restrict__ src, const int32_t* __restrict__ dst, const int n, const PageScratch w) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __shared__ uint32_t s_bits[kMaxSeqs / 32];
    __shared__ int s_warp[32], s_min;
    if (threadIdx.x == 0) w.header[0] = 0;
    clear_bits(s_bits, s.seqs);
    int bad = first_wrong(dst, n, s.seqs, s_bits, &s_min, w.map, [&](int i) { return (uint32_t)src[i] >= (uint32_t)s.seqs || s.lens[dst[i]] != 0; });
    constexpr int LS = 8;      // lanes of a sequence: their loads are under way together, and those of many short sequences too
    if (bad == n) {   // a source is nobody's destination, and its pages are pages
        for (int i = threadIdx.x / LS; i < n; i += kPlanThreads / LS) {
            const int np = pages_of(s, page_len(s, src[i]));
            bool wrong = has_bit(s_bits, src[i]);
            for (int j = threadIdx.x % LS; j < np; j += LS) wrong |= (uint32_t)s.table[(int64_t)src[i] * s.width + j] >= (uint32_t)s.n_pages;
            if (wrong) atomicMin(&s_min, i);
        }
        __syncthreads();
        bad = s_min;
    }
    if (bad < n) {
        const int used = s.n_pages - list_free(s, 0, nullptr, s_warp);
        say(s, kInfoList, used, 0, bad);
        return;
    }
    auto partial = [&](int i) { return page_len(s, src[i]) % s.page != 0 ? 1 : 0; };
    int want = 0;
    for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
        const int i = i0 + threadIdx.x, k = i < n ? partial(i) : 0;
        int total;
        const int at = want + block_scan(k, &total, s_warp);
        if (k) w.from[at] = s.table[(int64_t)src[i] * s.width + page_len(s, src[i]) / s.page];
        want += total;
    }
    const int free = list_free(s, want, w.to, s_warp);
    if (want > free) {
        say(s, kInfoNoPages, s.n_pages - free, 0, want);
        return;
    }
    __syncthreads();
    int base = 0;
    for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
        const int i = i0 + threadIdx.x, k = i < n ? partial(i) : 0;
        int total;
        const int at = base + block_scan(k, &total, s_warp);
        if (k) {
            s.table[(int64_t)dst[i] * s.width + page_len(s, src[i]) / s.page] = w.to[at];
            s.refs[w.to[at]] = 1;
        }
        base += total;
    }
    for (int i = threadIdx.x / LS; i < n; i += kPlanThreads / LS) {
        const int len = page_len(s, src[i]), full = len / s.page;
        for (int j = threadIdx.x % LS; j < full; j += LS) {
            const int pg = s.table[(int64_t)src[i] * s.width + j];
            s.table[(int64_t)dst[i] * s.width + j] = pg;
            atomicAdd(&s.refs[pg], 1);
        }
        if (threadIdx.x % LS == 0) s.lens[dst[i]] = len;
    }
    if (threadIdx.x == 0) w.header[0] = want;
    say(s, kInfoOk, s.n_pages - free + want, want, 0);
}

// Pages held that lie behind the first `live` ones go, in order, to the free pages among those.
__global__ void __launch_bounds__(kPlanThreads)
pages_compact_kernel(const PageState s, int32_t* refs_out, const PageScratch w) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __shared__ int s_warp[32];
    const int live = s.n_pages - list_free(s, 0, nullptr, s_warp);
    int holes = 0, moves = 0;
    for (int i0 = 0; 4 * i0 < s.n_pages; i0 += kPlanThreads) {
        const int i = i0 + threadIdx.x;
        const int4 r = refs4(s, i);
        const int v[4] = {r.x, r.y, r.z, r.w};
        int h = 0, m = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int pg = 4 * i + j;
            h += pg < live && v[j] <= 0;
            m += pg >= live && pg < s.n_pages && v[j] > 0;
        }
        int th, tm;
        int ah = holes + block_scan(h, &th, s_warp), am = moves + block_scan(m, &tm, s_warp);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int pg = 4 * i + j;
            if (pg < live && v[j] <= 0) w.to[ah++] = pg;
            if (pg >= live && pg < s.n_pages) {
                if (v[j] > 0) w.from[am++] = pg;
                else w.map[pg] = pg;
            }
        }
        holes += th;
        moves += tm;
    }
    __syncthreads();
    // the counts as they become: a page that moves takes its count along (a count of a free page stays as it is)
    if (refs_out != s.refs) {
        for (int i = threadIdx.x; i < s.n_pages; i += kPlanThreads) refs_out[i] = s.refs[i];
        __syncthreads();
    }
    for (int i = threadIdx.x; i < moves; i += kPlanThreads) {
        const int a = w.from[i], b = w.to[i];
        refs_out[b] = s.refs[a];
        refs_out[a] = 0;
        w.map[a] = b;
    }
    if (threadIdx.x == 0) {
        w.header[0] = moves;
        w.header[1] = live;
    }
    say(s, kInfoOk, live, moves, 0);
}

struct CopyParams {
    uint8_t *k, *v;                 // [layers][n_pages][page_bytes]
    const int32_t *from, *to;
    const int* pairs;               // how many
    int64_t page_bytes;
    int layers, n_pages, parts;     // pieces of a page
    int* status;
    // compact: the tables as they become
    PageState s;
    int32_t* table_out;
    const int* map;
    const int* live;
};
// The copy.  A warp per block moves pieces of pages through a ring in shared memory by bulk copies, in and out, the stores some pieces behind
// the loads; its lanes look up the next 32 pieces' places together.  No register or instruction is spent on the data.  The other warps
// rewrite the table.  (In and out together, a GB of random pages of 256, 64, 8 and 2 KB: 6.1, 5.9, 5.5, 2.7 TB/s; loads and stores by
// all threads reached 5.7, 5.7, 5.4 and 3.3, and held the SMs against the launch that follows: 8 sequences branched in 8 each 62 -> 51 us.)
constexpr int kCopyPiece = 16384, kCopyStages = 6, kCopyLag = 3, kCopyBlocks = 2;      // bytes; pieces; pieces; blocks per SM
constexpr int kCopySmem = 128 + kCopyPiece * kCopyStages;
__device__ __forceinline__ int64_t quotient(int64_t a, int b) { return a >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b); }
__device__ __forceinline__ void bulk_copy_s2g(void* dst, uint32_t src, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}
__global__ void __launch_bounds__(128, kCopyBlocks)
pages_copy_kernel(const CopyParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ uint8_t s_raw0[];
    __shared__ __align__(8) uint64_t s_bar[kCopyStages];
    __shared__ int s_abort;
    const int tid = threadIdx.x, lane = tid & 31;
    const uint32_t bar = smem_u32(s_bar), ring = (smem_u32(s_raw0) + 127) & ~127u;
    if (tid == 0) {
        s_abort = 0;
        for (int i = 0; i < kCopyStages; ++i) mbar_init(bar + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (tid < 32) {
        __syncwarp();
        const int pairs = *p.pairs;
        const int64_t pieces = (int64_t)pairs * p.layers * 2 * p.parts;
        const int64_t mine = pieces > blockIdx.x ? (pieces - blockIdx.x + gridDim.x - 1) / gridDim.x : 0;
        int64_t from = 0, to = 0;       // of the lane's piece of 32: its places
        uint32_t size = 0;              // (0: it has none)
        bool ok = true;
        int64_t to_before = 0;          // the 32 before these, whose stores may be to come
        uint32_t size_before = 0;
        int64_t k = 0;
        for (; k < mine + kCopyLag && ok; ++k) {
            if ((k & 31) == 0) {
                to_before = to;
                size_before = size;
                size = 0;
                if (k + lane < mine) {
                    const int64_t i = blockIdx.x + (k + lane) * gridDim.x, page = quotient(i, p.parts);
                    const int part = (int)(i - page * p.parts), pool = (int)(page & 1);
                    const int64_t pl = page >> 1, layer = quotient(pl, pairs), pair = pl - layer * pairs;
                    const int64_t o = (int64_t)part * kCopyPiece;
                    const int a = p.from[pair], b = p.to[pair];
                    if ((uint32_t)a < (uint32_t)p.n_pages && (uint32_t)b < (uint32_t)p.n_pages) {
                        const int64_t base = (int64_t)(pool ? p.v : p.k) + layer * p.n_pages * p.page_bytes + o;
                        from = base + a * p.page_bytes;
                        to = base + b * p.page_bytes;
                        size = (uint32_t)(p.page_bytes - o < kCopyPiece ? p.page_bytes - o : kCopyPiece);
                    }
                }
            }
            const int64_t src = __shfl_sync(0xffffffffu, from, (int)(k & 31));
            const uint32_t n = __shfl_sync(0xffffffffu, size, (int)(k & 31));
            if (k < mine) {
                const int s = (int)(k % kCopyStages);
                if (lane == 0) {
                    // (of the stores so far those but the last Stages - Lag - 1 have read their stages: this one's among them)
                    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kCopyStages - kCopyLag - 1) : "memory");
                    if (n) {
                        mbar_expect_tx(bar + 8 * s, n);
                        bulk_copy_g2s(ring + s * kCopyPiece, (const void*)src, n, bar + 8 * s);
                    } else mbar_arrive(bar + 8 * s);
                }
            }
            const int64_t q = k - kCopyLag;
            if (q >= 0) {
                const bool before = (q >> 5) != (k >> 5);
                const int64_t dst = __shfl_sync(0xffffffffu, before ? to_before : to, (int)(q & 31));
                const uint32_t m = __shfl_sync(0xffffffffu, before ? size_before : size, (int)(q & 31));
                const int s = (int)(q % kCopyStages);
                ok = __all_sync(0xffffffffu, mbar_block(bar + 8 * s, (uint32_t)(q / kCopyStages) & 1u, &s_abort));
                if (ok && lane == 0) {
                    if (m) bulk_copy_s2g((void*)dst, ring + s * kCopyPiece, m);
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                }
            }
        }
        if (lane == 0) {
            asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
            if (!ok) atomicExch(p.status, 2);
        }
        if (!ok) {          // loads under way are waited for (again with a limit) before their memory is given up
            volatile int none = 0;
            const int64_t issued = k < mine ? k : mine;
            for (int s = 0; s < kCopyStages && s < issued; ++s)
                mbar_wait(bar + 8 * s, (uint32_t)((issued - 1 - s) / kCopyStages) & 1u, const_cast<volatile int*>(&none));
        }
    } else if (p.table_out) {
        const int live = *p.live;
        for (int64_t e = (int64_t)blockIdx.x * 96 + tid - 32; e < (int64_t)p.s.seqs * p.s.width; e += (int64_t)gridDim.x * 96) {
            const int b = (int)quotient(e, p.s.width), j = (int)(e - (int64_t)b * p.s.width), pg = p.s.table[e];
            const bool held = j < pages_of(p.s, page_len(p.s, b)) && pg >= live && pg < p.s.n_pages;
            p.table_out[e] = held ? p.map[pg] : pg;
        }
    }
}

// A list of pages to copy: every page in the pool, none copied to twice, none both copied and copied to.
__global__ void __launch_bounds__(kPlanThreads)
pages_list_kernel(const int32_t* __restrict__ src, const int32_t* __restrict__ dst, int32_t* info, const int n, const int n_pages,
                  const PageScratch w) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    extern __shared__ uint32_t s_map[];
    __shared__ int s_min;
    clear_bits(s_map, n_pages);
    int bad = first_wrong(dst, n, n_pages, s_map, &s_min, w.map, [&](int i) { return (uint32_t)src[i] >= (uint32_t)n_pages; });
    if (bad == n) bad = first_bad(n, &s_min, [&](int i) { return has_bit(s_map, src[i]); });
    if (threadIdx.x == 0) {
        w.header[0] = bad == n ? n : 0;
        *reinterpret_cast<int4*>(info) = bad == n ? make_int4(kInfoOk, 0, n, 0) : make_int4(kInfoList, 0, 0, bad);
    }
}

int32_t pages_configure(DeviceState& ds) {
    RSTQ_CUDA(cudaMalloc(&ds.page_scratch, (size_t)kPageScratchBytes));
    RSTQ_CUDA(cudaMemsetAsync(ds.page_scratch, 0, (size_t)kPageScratchBytes, ds.stream));
    RSTQ_CUDA(cudaFuncSetAttribute(pages_copy_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kCopySmem));
    RSTQ_CUDA(cudaFuncSetAttribute(pages_list_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kMaxPages / 8)));
    return RSTQ_OK;
}

}  // namespace rstq

using namespace rstq;

static int32_t page_state(rstq_ctx* ctx, rstq_buf* table, rstq_buf* lens, rstq_buf* refs, rstq_buf* info, int64_t seqs, int64_t n_pages,
                          int64_t max_pages, int64_t page, PageState* s) {
    RSTQ_REQUIRE(ctx && ctx->magic == kCtxMagic, RSTQ_E_INVALID, "invalid context handle");
    const int32_t rc = check_pages(seqs, page, n_pages, max_pages);
    if (rc != RSTQ_OK) return rc;
    RSTQ_REQUIRE(paged_buf(table, ctx, seqs * max_pages * 4) && paged_buf(lens, ctx, seqs * 4) && paged_buf(refs, ctx, n_pages * 4) &&
                     paged_buf(info, ctx, 16),
                 RSTQ_E_INVALID, "invalid, unaligned or too small buffer");
    RSTQ_REQUIRE(same_device(table, lens, refs, info), RSTQ_E_DEVICE, "buffers live on different devices");
    const Span written[] = {{table->ptr, seqs * max_pages * 4}, {lens->ptr, seqs * 4}, {refs->ptr, n_pages * 4}, {info->ptr, 16}}, none[] = {{nullptr, 0}};
    RSTQ_REQUIRE(apart(written, none), RSTQ_E_INVALID, "table, lens, refs and info lie over one another");
    *s = PageState{(int32_t*)table->ptr, (int32_t*)lens->ptr, (int32_t*)refs->ptr, (int32_t*)info->ptr,
                   (int)seqs, (int)n_pages, (int)max_pages, (int)page};
    return use_dev(ctx, table->dev);
}
static int32_t list_args(rstq_ctx* ctx, const PageState& s, const rstq_buf* on, rstq_buf* a, rstq_buf* b, int64_t n) {
    RSTQ_REQUIRE(n >= 0 && n <= kListMax, RSTQ_E_LIMIT, "a list of %lld (0 .. %d)", (long long)n, kListMax);
    RSTQ_REQUIRE(paged_buf(a, ctx, n * 4) && (!b || paged_buf(b, ctx, n * 4)), RSTQ_E_INVALID, "invalid, unaligned or too small list");
    RSTQ_REQUIRE(same_device(on, a, b), RSTQ_E_DEVICE, "buffers live on different devices");
    const Span written[] = {{s.table, (int64_t)s.seqs * s.width * 4}, {s.lens, s.seqs * 4ll}, {s.refs, s.n_pages * 4ll}, {s.info, 16}};
    const Span read[] = {{a->ptr, n * 4}, {b ? b->ptr : nullptr, b ? n * 4 : 0}};
    RSTQ_REQUIRE(apart(written, read), RSTQ_E_INVALID, "a list lies over what the call writes");
    return RSTQ_OK;
}
// the pools' part: layers x n_pages pages of page_bytes, K and V; `others`: the call's other arrays
template <size_t N>
static int32_t pool_args(rstq_ctx* ctx, const rstq_buf* on, rstq_buf* k, rstq_buf* v, int64_t layers, int64_t n_pages, int64_t page_bytes,
                         const Span (&others)[N], CopyParams* p) {
    RSTQ_REQUIRE(layers >= 1 && layers <= 4096 && page_bytes >= 16 && page_bytes <= (1ll << 30), RSTQ_E_SHAPE, "layers = %lld, bytes of a page = %lld",
                 (long long)layers, (long long)page_bytes);
    RSTQ_REQUIRE(page_bytes % 16 == 0, RSTQ_E_ALIGN, "%lld bytes of a page: not a multiple of 16", (long long)page_bytes);
    RSTQ_REQUIRE(paged_buf(k, ctx, layers * n_pages * page_bytes) && paged_buf(v, ctx, layers * n_pages * page_bytes), RSTQ_E_INVALID,
                 "invalid, unaligned or too small pool");
    RSTQ_REQUIRE(same_device(on, k, v), RSTQ_E_DEVICE, "buffers live on different devices");
    const Span written[] = {{k->ptr, layers * n_pages * page_bytes}, {v->ptr, layers * n_pages * page_bytes}};
    RSTQ_REQUIRE(apart(written, others), RSTQ_E_INVALID, "a pool lies over another array");
    *p = CopyParams{};
    p->k = (uint8_t*)k->ptr;
    p->v = (uint8_t*)v->ptr;
    p->page_bytes = page_bytes;
    p->layers = (int)layers;
    p->n_pages = (int)n_pages;
    p->parts = (int)((page_bytes + kCopyPiece - 1) / kCopyPiece);
    return RSTQ_OK;
}
// blocks of the copy: as many as its longest list keeps busy, and as the SMs hold at once at most
static dim3 copy_grid(const DeviceState& ds, const CopyParams& p, int64_t pairs, int64_t entries) {
    const int64_t work = std::max(pairs * p.layers * 2 * p.parts, (entries + 95) / 96);
    return dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>(work, (int64_t)kCopyBlocks * ds.sm_count)));
}

extern "C" {

int32_t rstq_pages_free(rstq_ctx* ctx, rstq_buf* table, rstq_buf* lens, rstq_buf* refs, rstq_buf* list, rstq_buf* info, int64_t n,
                        int64_t seqs, int64_t n_pages, int64_t max_pages, int64_t page) {
    PageState s;
    int32_t rc = page_state(ctx, table, lens, refs, info, seqs, n_pages, max_pages, page, &s);
    if (rc == RSTQ_OK) rc = list_args(ctx, s, table, list, nullptr, n);
    if (rc != RSTQ_OK) return rc;
    DeviceState& ds = ctx->devs[table->dev];
    RSTQ_CUDA(launch_pdl(pages_free_kernel, dim3(1), dim3(kPlanThreads), 0, ds, s, (const int32_t*)list->ptr, (int)n, page_scratch(ds)));
    ctx->launches++;
    return RSTQ_OK;
}

int32_t rstq_pages_extend(rstq_ctx* ctx, rstq_buf* table, rstq_buf* lens, rstq_buf* refs, rstq_buf* list, rstq_buf* counts,
                          rstq_buf* info, int64_t n, int64_t seqs, int64_t n_pages, int64_t max_pages, int64_t page) {
    PageState s;
    int32_t rc = page_state(ctx, table, lens, refs, info, seqs, n_pages, max_pages, page, &s);
    if (rc == RSTQ_OK) {
        RSTQ_REQUIRE(counts, RSTQ_E_INVALID, "null list");
        rc = list_args(ctx, s, table, list, counts, n);
    }
    if (rc != RSTQ_OK) return rc;
    DeviceState& ds = ctx->devs[table->dev];
    RSTQ_CUDA(launch_pdl(pages_extend_kernel, dim3(1), dim3(kPlanThreads), 0, ds, s, (const int32_t*)list->ptr,
                         (const int32_t*)counts->ptr, (int)n, page_scratch(ds)));
    ctx->launches++;
    return RSTQ_OK;
}

int32_t rstq_pages_fork(rstq_ctx* ctx, rstq_buf* kcache, rstq_buf* vcache, rstq_buf* table, rstq_buf* lens, rstq_buf* refs,
                        rstq_buf* src, rstq_buf* dst, rstq_buf* info, int64_t n, int64_t seqs, int64_t n_pages, int64_t max_pages,
                        int64_t page, int64_t layers, int64_t row_bytes) {
    PageState s;
    CopyParams p;
    int32_t rc = page_state(ctx, table, lens, refs, info, seqs, n_pages, max_pages, page, &s);
    if (rc == RSTQ_OK) {
        RSTQ_REQUIRE(dst, RSTQ_E_INVALID, "null list");
        RSTQ_REQUIRE(row_bytes >= 1 && row_bytes <= (1ll << 30), RSTQ_E_SHAPE, "row_bytes = %lld", (long long)row_bytes);
        rc = list_args(ctx, s, table, src, dst, n);
    }
    if (rc == RSTQ_OK) {
        const Span others[] = {{s.table, (int64_t)s.seqs * s.width * 4}, {s.lens, s.seqs * 4ll}, {s.refs, s.n_pages * 4ll}, {s.info, 16},
                               {src->ptr, n * 4}, {dst->ptr, n * 4}};
        rc = pool_args(ctx, table, kcache, vcache, layers, n_pages, page * row_bytes, others, &p);
    }
    if (rc != RSTQ_OK) return rc;
    DeviceState& ds = ctx->devs[table->dev];
    const PageScratch w = page_scratch(ds);
    RSTQ_CUDA(launch_pdl(pages_fork_kernel, dim3(1), dim3(kPlanThreads), 0, ds, s, (const int32_t*)src->ptr, (const int32_t*)dst->ptr,
                         (int)n, w));
    p.from = w.from;
    p.to = w.to;
    p.pairs = w.header;
    p.status = ds.status;
    RSTQ_CUDA(launch_pdl(pages_copy_kernel, copy_grid(ds, p, n, 0), dim3(128), kCopySmem, ds, p));
    ctx->launches += 2;
    return RSTQ_OK;
}

int32_t rstq_pages_compact(rstq_ctx* ctx, rstq_buf* kcache, rstq_buf* vcache, rstq_buf* table, rstq_buf* lens, rstq_buf* refs,
                           rstq_buf* table_out, rstq_buf* refs_out, rstq_buf* info, int64_t seqs, int64_t n_pages,
                           int64_t max_pages, int64_t page, int64_t layers, int64_t row_bytes) {
    PageState s;
    CopyParams p;
    int32_t rc = page_state(ctx, table, lens, refs, info, seqs, n_pages, max_pages, page, &s);
    if (rc == RSTQ_OK) {
        RSTQ_REQUIRE(row_bytes >= 1 && row_bytes <= (1ll << 30), RSTQ_E_SHAPE, "row_bytes = %lld", (long long)row_bytes);
        RSTQ_REQUIRE(paged_buf(table_out, ctx, seqs * max_pages * 4) && paged_buf(refs_out, ctx, n_pages * 4), RSTQ_E_INVALID,
                     "invalid, unaligned or too small buffer");
        RSTQ_REQUIRE(same_device(table, table_out, refs_out), RSTQ_E_DEVICE, "buffers live on different devices");
        // in place, or somewhere else
        const int64_t tb = (int64_t)s.seqs * s.width * 4, rb = s.n_pages * 4ll;
        const Span to = {table_out->ptr, tb}, ro = {refs_out->ptr, rb};
        const Span others[] = {{s.table, tb}, {s.lens, s.seqs * 4ll}, {s.refs, rb}, {s.info, 16}, to, ro};
        RSTQ_REQUIRE((to.p == s.table || apart(to, others[0])) && apart(to, others[1]) && apart(to, others[2]) && apart(to, others[3]) &&
                         apart(to, ro) && (ro.p == s.refs || apart(ro, others[2])) && apart(ro, others[0]) && apart(ro, others[1]) && apart(ro, others[3]),
                     RSTQ_E_INVALID, "table_out or refs_out lies over another array");
        rc = pool_args(ctx, table, kcache, vcache, layers, n_pages, page * row_bytes, others, &p);
    }
    if (rc != RSTQ_OK) return rc;
    DeviceState& ds = ctx->devs[table->dev];
    const PageScratch w = page_scratch(ds);
    RSTQ_CUDA(launch_pdl(pages_compact_kernel, dim3(1), dim3(kPlanThreads), 0, ds, s, (int32_t*)refs_out->ptr, w));
    p.from = w.from;
    p.to = w.to;
    p.pairs = w.header;
    p.status = ds.status;
    p.live = w.header + 1;
    p.map = w.map;
    p.s = s;
    p.table_out = (int32_t*)table_out->ptr;
    RSTQ_CUDA(launch_pdl(pages_copy_kernel, copy_grid(ds, p, n_pages / 2, seqs * max_pages), dim3(128), kCopySmem, ds, p));
    ctx->launches += 2;
    return RSTQ_OK;
}

int32_t rstq_pages_copy(rstq_ctx* ctx, rstq_buf* kcache, rstq_buf* vcache, rstq_buf* src, rstq_buf* dst, rstq_buf* info, int64_t n,
                        int64_t n_pages, int64_t layers, int64_t page_bytes) {
    RSTQ_REQUIRE(ctx && ctx->magic == kCtxMagic, RSTQ_E_INVALID, "invalid context handle");
    RSTQ_REQUIRE(n_pages >= 1 && n_pages <= kMaxPages, RSTQ_E_LIMIT, "n_pages = %lld (1 .. %lld)", (long long)n_pages, (long long)kMaxPages);
    RSTQ_REQUIRE(dst && paged_buf(info, ctx, 16), RSTQ_E_INVALID, "invalid, unaligned or too small buffer");
    CopyParams p;
    PageState s{};
    s.info = (int32_t*)info->ptr;
    int32_t rc = list_args(ctx, s, info, src, dst, n);
    if (rc == RSTQ_OK) {
        const Span others[] = {{info->ptr, 16}, {src->ptr, n * 4}, {dst->ptr, n * 4}};
        rc = pool_args(ctx, info, kcache, vcache, layers, n_pages, page_bytes, others, &p);
    }
    if (rc == RSTQ_OK) rc = use_dev(ctx, info->dev);
    if (rc != RSTQ_OK) return rc;
    DeviceState& ds = ctx->devs[info->dev];
    const PageScratch w = page_scratch(ds);
    RSTQ_CUDA(launch_pdl(pages_list_kernel, dim3(1), dim3(kPlanThreads), (size_t)((n_pages + 31) / 32 * 4), ds, (const int32_t*)src->ptr,
                         (const int32_t*)dst->ptr, (int32_t*)info->ptr, (int)n, (int)n_pages, w));
    p.from = (const int32_t*)src->ptr;
    p.to = (const int32_t*)dst->ptr;
    p.pairs = w.header;
    p.status = ds.status;
    RSTQ_CUDA(launch_pdl(pages_copy_kernel, copy_grid(ds, p, n, 0), dim3(128), kCopySmem, ds, p));
    ctx->launches += 2;
    return RSTQ_OK;
}

}  // extern "C"
