// Attention of one new token per sequence over a paged cache.
//
//   out[b, h] = sum_j p_j V[b, j] / sum_j p_j,   p_j = exp(scale q.K[b, j] - m),   j < lens[b]
//
// Bound by HBM: every cached row is read once, for all query heads of its KV head (up to 16, in f32 8; a larger group's other
// heads find the rows in L2).  64 sequences of 4100 (64 heads over 8): 175 us, 94 % of the copy rate; 16 of 4000 48 us, 83 %; 16 of 1 to 8000
// 22 us, 51 %; four in f32 of 1300 35 us, 74 %; one of 300 9 us, of 8000 18.  What is not the stream: 1.6 us until the lengths are read and the range is
// found, 3 until the first tile is there, 2 for a range's last sums, 3 and more for joining the parts of a pair.
//
// Work.  A unit is a tile of positions (64 in bf16, 32 in f32) of one sequence and KV head; the units of all sequences lie
// on one line (sequence, head, tile) and every thread block takes an equal range of it, so that lengths may be as different as they
// like and few long sequences use all SMs.  The ranges follow from the lengths alone, which are read on the device: one recorded
// launch serves every step.  A (sequence, head) pair that lies in one range is finished there; the parts of one that spans
// several are left in slots, announced at the end of each range (an arrival counter), and the block that comes last joins them in the
// order of the ranges, so the result does not depend on who came last.  Nobody waits for another block.
//
// Block.  A thread brings K and V by TMA, a box per page (its rows 128 bytes wide, swizzled), through a ring of 80 KB in two blocks
// per SM, and the queries of each part ahead of it; the pages are looked up a part (512 positions) ahead.  Four warps take a quarter of
// each tile's positions and keep a softmax of their own (running maximum, sum, weighted V), joined at the end of a range's
// part.  V's rows behind the end are zeroed in shared memory before they are used and their scores masked, so what stale pages
// hold never reaches a result.
//   bf16: m16n8k16 MMAs, positions (of V: head_dim) in the 16 rows, eight query heads in the columns: with the heads in the rows
//         most groups would leave more than half of them empty.  A weight enters P.V as the sum of two bf16 terms (16 bits).
//   f32:  a lane forms a quarter of a dot product in f32 FMAs for each head of the group, then owns four (two) columns of V.  (16 of
//         4000, 32 heads over 8: 91 us, 88 % of the copy rate; with a branch around each head, whose chains then came one after the other, 156.)
#include <algorithm>
#include <type_traits>

#include "paged.cuh"
#include "sync_helpers.cuh"
#include "tcgen05_helpers.cuh"

namespace rstq {

constexpr int kDecWarps = 4;                          // consumers; one more warp copies
constexpr int kDecThreads = (kDecWarps + 1) * 32;
// Blocks per SM; bytes of the ring; bytes for the queries of the parts to come.  (Above 128 columns five stages and the sums take a whole SM.)
template <int HD>
__host__ __device__ constexpr int dec_blocks() { return HD > 128 ? 1 : 2; }
template <int HD>
__host__ __device__ constexpr int dec_ring() { return (HD > 128 ? 160 : 80) * 1024; }
template <int HD>
__host__ __device__ constexpr int dec_q() { return (HD > 128 ? 16 : 7) * 1024; }
// the warps' sums, [warp][eight heads][HD + 4]: four floats of padding and a warp's stores meet no bank twice
template <int HD>
__host__ __device__ constexpr int dec_slab() { return 8 * (HD + 4); }
template <int HD>
__host__ __device__ constexpr int dec_smem() { return 1024 + dec_ring<HD>() + dec_q<HD>() + kDecWarps * dec_slab<HD>() * 4; }

struct DecodeParams {
    const void *q, *k, *v;
    void* out;
    KvPlace kv;
    int64_t ldq;
    int seqs, n_q, group, n_kv, head_dim, gz;         // gz: passes over a group of more than kPagedGroup heads
    float scale2;                                     // scale * log2(e)
    float* part;                                      // [2 * blocks] slots
    int* counters;                                    // [blocks], zero between launches
    int* status;
    int box;                                          // rows of a box: min(page, tile)
    const int64_t* start;                             // units of a head before each sequence; null: few sequences
    float* sums;                                      // [blocks][kDecWarps] x dec_sums: bf16, what warps have summed over kDecFold tiles
};
template <typename T>
__host__ __device__ constexpr int dec_tile() { return sizeof(T) == 2 ? 64 : 32; }
template <typename T, int HD>
__host__ __device__ constexpr int dec_stage() { return dec_tile<T>() * HD * (int)sizeof(T); }    // K or V of a tile
// query heads of a KV head that one pass serves: what its sums leave of the registers
template <typename T>
__host__ __device__ constexpr int dec_heads() { return sizeof(T) == 2 ? kPagedGroup : kPagedGroup / 2; }
// bf16: tiles that a warp sums up in its MMAs' registers.  An MMA's additions cut off, towards zero, so a longer sum is taken out every so often and
// added to one in memory.  (300 sequences over the same 2^20 positions, a block each: results 3.7e-3 too small without, no smaller than those of
// one sequence, which all blocks share, with it.  It costs groups of more than eight heads 2 %; every tile's sum taken out, in registers, 6 to 16.)
constexpr int kDecFold = 512;
// ... in floats: a warp's registers and maxima
template <int HD, int GH>
__host__ __device__ constexpr int dec_sums() { return 32 * (HD * GH / 32 + GH / 4); }
// a slot, in floats: the heads' weighted V, their maxima, their sums of weights
template <int HD>
__host__ __device__ constexpr int dec_slot() { return kPagedGroup * (HD + 2); }

__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ float4 lds128(uint32_t a) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// an 8 x 8 matrix of 16-bit elements, a row per four lanes, transposed
__device__ __forceinline__ uint32_t turn8x8(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.f : m; }   // nothing seen yet: exp2(-inf - 0) = 0
__device__ __forceinline__ void bar_consumers() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// What the end of a (sequence, head) costs a block, in tiles: its warps' states are joined and the next one's queries taken.  (0, 1, 2, 3:
// 16 sequences of 300 13.9, 12.9, 11.9, 12.9 us, of 4000 49.3, 48.5, 47.8, 48.9; four in f32 of 1300 35.8, 35.3, 34.9, 35.3.)
constexpr int kDecEnd = 2;
constexpr int kDecSums = 256;                         // sequences above which launch_sums adds the lengths up (1000 of 100: 115 -> 107 us)
// What a weight's second term has at least beside the rest of it: the weight times 2^-7, 2^-100 at most.  Nothing for a weight of nothing, and never
// more than a weight's own rounding to bf16: for those below 2^-93 a 128th, for one of 2^-76 the 2^-24th part.
__device__ __forceinline__ float some_rest(float w) { return fminf(w * 0.0078125f, 7.8886091e-31f); }

// Where a block's range of units lies.  Units of sequence b: for each of H heads its tiles, and kDecEnd for what the end of a part costs.  All lanes of a warp hold the same,
// but for the lengths: lane x has that of sequence first + x.
struct Walk {
    int b, h, t;          // sequence, head (pass of a head's group), tile
    int len, nt;          // positions and tiles of that sequence
    int64_t left;         // units of the range from here on
    int first, lens;
};
__device__ __forceinline__ int dec_len(const DecodeParams& p, int b) {
    int64_t r;
    return b < p.seqs ? (int)kv_length(p.kv, b, &r) : 0;
}
template <int TILE>
__device__ __forceinline__ int dec_units(int len) { return len > 0 ? (len + TILE - 1) / TILE + kDecEnd : 0; }
// to the next (sequence, head), at its first tile
template <int TILE>
__device__ __forceinline__ void dec_next(const DecodeParams& p, int H, Walk* w) {
    w->t = 0;
    if (++w->h < H) return;
    w->h = 0;
    do {
        if (++w->b >= p.seqs) {      // (cannot be, unless a length changed meanwhile)
            w->left = 0;
            return;
        }
        if (w->b >= w->first + 32) {
            w->first += 32;
            w->lens = dec_len(p, w->first + (threadIdx.x & 31));
        }
        w->len = __shfl_sync(0xffffffffu, w->lens, w->b - w->first);
        w->nt = (w->len + TILE - 1) / TILE;
    } while (w->nt == 0);
}
// past n tiles of a (sequence, head), and past its end if they are its last
template <int TILE>
__device__ __forceinline__ void dec_past(const DecodeParams& p, int H, Walk* w, int n) {
    w->t += n;
    w->left -= n;
    if (w->t < w->nt) return;
    w->left -= w->nt + kDecEnd - w->t;
    if (w->left > 0) dec_next<TILE>(p, H, w);
}
// Total units, and the place of the first one of the range that `range` gives for it.
template <int TILE, typename F>
__device__ __forceinline__ int64_t dec_find(const DecodeParams& p, int H, Walk* w, F range) {
    const int lane = threadIdx.x & 31;
    int64_t first, last;
    if (p.start) {
        const int64_t total = p.start[p.seqs] * H;
        range(total, &first, &last);
        w->left = last - first;
        if (w->left <= 0) return total;
        w->b = find_start(p.start, p.seqs, first / H);
        // (the first unit of sequence b is start[b] * H, so b is the last one with start[b] <= first / H)
        w->first = w->b & ~31;
        w->lens = dec_len(p, w->first + lane);
        w->len = __shfl_sync(0xffffffffu, w->lens, w->b - w->first);
        const int units = dec_units<TILE>(w->len);
        w->nt = units - kDecEnd;
        const int64_t in = first - p.start[w->b] * H;
        w->h = units > 0 ? (int)(in / units) : 0;
        w->t = (int)(in - (int64_t)w->h * units);
        if (units == 0 || w->h >= H) w->left = 0;      // (cannot be, unless a length changed meanwhile)
        else dec_past<TILE>(p, H, w, 0);
        return total;
    }
    const int head = dec_len(p, lane);
    int64_t total = dec_units<TILE>(head);
    for (int b0 = 32; b0 < p.seqs; b0 += 128) {
        int n[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) n[u] = dec_len(p, b0 + u * 32 + lane);
#pragma unroll
        for (int u = 0; u < 4; ++u) total += dec_units<TILE>(n[u]);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    total *= H;
    range(total, &first, &last);
    w->left = last - first;
    if (w->left <= 0) return total;
    int64_t base = 0;
    for (int b0 = 0; b0 < p.seqs; b0 += 32) {
        const int len = b0 ? dec_len(p, b0 + lane) : head;
        const int n = dec_units<TILE>(len);
        int64_t x = (int64_t)n * H;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += y;
        }
        const unsigned behind = __ballot_sync(0xffffffffu, base + x > first);
        if (behind) {
            const int src = __ffs((int)behind) - 1;
            const int64_t end = __shfl_sync(0xffffffffu, base + x, src);
            w->b = b0 + src;
            w->first = b0;
            w->lens = len;
            w->len = __shfl_sync(0xffffffffu, len, src);
            const int units = __shfl_sync(0xffffffffu, n, src);
            w->nt = units - kDecEnd;
            const int64_t in = first - (end - (int64_t)units * H);
            w->h = in >> 32 ? (int)(in / units) : (int)((uint32_t)in / (uint32_t)units);
            w->t = (int)(in - (int64_t)w->h * units);
            dec_past<TILE>(p, H, w, 0);
            return total;
        }
        base += __shfl_sync(0xffffffffu, x, 31);
    }
    w->left = 0;
    return total;
}
// GH: query heads served at once (bf16: 8 or 16; f32: what the group needs)
template <typename T, int HD, int GH>
__global__ void __launch_bounds__(kDecThreads, dec_blocks<HD>())
paged_decode_kernel(const DecodeParams p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    constexpr int TILE = dec_tile<T>(), G16 = TILE / 16, STAGE = dec_stage<T, HD>(), NST = dec_ring<HD>() / STAGE;
    constexpr int ES = (int)sizeof(T), BLKS = HD * ES / 128, BLK = TILE * 128;      // a tile's rows in pieces of 128 bytes: BLKS blocks
    constexpr bool BF = ES == 2;
    constexpr int SLOT = dec_slot<HD>(), SLAB = dec_slab<HD>(), QB = GH * HD * ES, NQ = dec_q<HD>() / QB >= 4 ? 4 : dec_q<HD>() / QB;
    constexpr int PER = dec_heads<T>();               // query heads of a pass
    static_assert(NST >= 4 && NQ >= 1 && GH <= PER, "ring");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ uint8_t s_raw0[];
    uint8_t* s_raw = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(s_raw0) + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t s_bar[2 * NST + 2 * NQ];
    __shared__ uint32_t s_seen[NST];                  // which sixteens of a stage's positions are there
    __shared__ float s_m[kDecWarps][kPagedGroup], s_l[kDecWarps][kPagedGroup];
    __shared__ int s_abort, s_last[2];
    __shared__ int4 s_open[2];                        // pairs of which the range has a part and not the whole: sequence, head, blocks
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t ring = smem_u32(s_raw), full = smem_u32(s_bar), empty = full + 8 * NST, qfull = empty + 8 * NST, qempty = qfull + 8 * NQ;
    const uint32_t s_q = ring + dec_ring<HD>();
    float* s_slab = reinterpret_cast<float*>(s_raw + dec_ring<HD>() + dec_q<HD>());
    volatile int* abort_flag = &s_abort;
    if (tid == 0) {
        s_abort = 0;
        for (int i = 0; i < NST; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, kDecWarps);
        }
        for (int i = 0; i < NQ; ++i) {
            mbar_init(qfull + 8 * i, 1);
            mbar_init(qempty + 8 * i, kDecWarps);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (tid == kDecWarps * 32) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&kmap)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&vmap)) : "memory");
    }
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const int H = p.n_kv * p.gz;
    int blocks = gridDim.x;
    int64_t r0 = 0, r1 = 0;
    Walk w;
    w.left = 0;
    const int64_t total = dec_find<TILE>(p, H, &w, [&](int64_t n, int64_t* a, int64_t* e) {
        // Ranges of two units at least: of one, every third would be the end of a pair and no tile.  (1, 2, 4: 8 sequences of 500 to 4000 of one
        // KV head 33, 24, 22 us, four f32 of 64 7.9, 6.2, 6.0, one of 300 9.2, 9.6, 11.7.)
        if (blocks > n / 2) blocks = n >= 2 ? (int)(n / 2) : n > 0;
        const int c = blockIdx.x;
        if (c < blocks) {                             // floor(c n / blocks)
            const int64_t each = n >> 32 ? n / blocks : (int64_t)((uint32_t)n / (uint32_t)blocks);
            const uint32_t rest = (uint32_t)(n - each * blocks);
            r0 = c * each + c * rest / (uint32_t)blocks;
            r1 = (c + 1) * each + (c + 1) * rest / (uint32_t)blocks;
        }
        *a = r0;
        *e = r1;
    });

    if (warp == kDecWarps) {
        // ---- copies ----
        int s = 0, sq = 0;
        uint32_t ph = 0, phq = 0;
        bool bad = false, ok = true;
        // pages of 32 sixteens of a sequence's positions, a lane each
        auto pages_of = [&](const Walk& x, int chunk) {
            const int64_t pos = ((int64_t)chunk * 32 + lane) * 16;
            return x.left > 0 && pos < x.len ? p.kv.table[(int64_t)x.b * p.kv.width + (pos >> p.kv.shift)] : 0;
        };
        int first_pages = pages_of(w, w.t * G16 >> 5);
        while (w.left > 0 && ok) {
            const int n = (int)min(w.left, (int64_t)(w.nt - w.t)), hkv = p.gz == 1 ? w.h : w.h / p.gz;
            Walk v = w;              // the part after this one
            dec_past<TILE>(p, H, &v, n);
            int chunk = w.t * G16 >> 5, pages = first_pages, more = pages_of(w, chunk + 1);
            first_pages = pages_of(v, v.t * G16 >> 5);
            {                        // the part's queries: rows of the group's heads, one behind the other
                const int g0 = (w.h - hkv * p.gz) * PER, G = min(p.group - g0, PER);
                ok = __all_sync(0xffffffffu, mbar_block(qempty + 8 * sq, phq ^ 1u, abort_flag));
                if (!ok) break;
                if (lane == 0) {
                    const uint32_t bytes = (uint32_t)(G * p.head_dim * ES);
                    mbar_expect_tx(qfull + 8 * sq, bytes);
                    bulk_copy_g2s(s_q + sq * QB, (const T*)p.q + (int64_t)w.b * p.ldq + (int64_t)(hkv * p.group + g0) * p.head_dim, bytes, qfull + 8 * sq);
                }
                if (++sq == NQ) { sq = 0; phq ^= 1u; }
            }
            for (int i = 0; i < n && ok; ++i) {
                const int pos0 = (w.t + i) * TILE, at = (w.t + i) * G16;
                if (at >> 5 != chunk) {
                    ++chunk;
                    pages = more;
                    more = pages_of(w, chunk + 1);
                }
                const int page = __shfl_sync(0xffffffffu, pages, (at & 31) + (lane & (G16 - 1)));
                const bool there = (uint32_t)page < (uint64_t)p.kv.n_pages;
                const unsigned seen = __ballot_sync(0xffffffffu, there) & ((1u << G16) - 1);
                bad |= !there;       // (0, a page, behind the end)
                const int row = there ? (page << p.kv.shift) + ((pos0 + (lane & (G16 - 1)) * 16) & ((1 << p.kv.shift) - 1)) : 0;
                // boxes that begin before the end and whose page is one
                const int per = p.box >> 4;
                unsigned boxes = 0;
#pragma unroll
                for (int g = 0; g < G16; ++g) boxes |= (g & (per - 1)) == 0 && pos0 + g * 16 < w.len ? seen & (1u << g) : 0u;
                const uint32_t bytes = (uint32_t)(__popc(boxes) * p.box * 128 * BLKS);
#pragma unroll
                for (int kv = 0; kv < 2; ++kv) {
                    if (ok) ok = __all_sync(0xffffffffu, mbar_block(empty + 8 * s, ph ^ 1u, abort_flag));
                    if (!ok) break;
                    const uint32_t bar = full + 8 * s, dst = ring + s * STAGE;
                    if (lane == 0) {
                        if (kv == 0) s_seen[s] = seen;
                        if (boxes) mbar_expect_tx(bar, bytes);
                        else mbar_arrive(bar);
                    }
#pragma unroll
                    for (int g = 0; g < G16; ++g) {
                        const int y = __shfl_sync(0xffffffffu, row, g);
                        if (lane == 0 && ((boxes >> g) & 1))
#pragma unroll
                            for (int c = 0; c < BLKS; ++c) tma_load_3d(dst + c * BLK + g * 16 * 128, kv ? &vmap : &kmap, c * (128 / ES), hkv, y, bar);
                    }
                    if (++s == NST) { s = 0; ph ^= 1u; }
                }
            }
            w = v;
        }
        if (__any_sync(0xffffffffu, bad) && lane == 0) p.status[kStatusPage] = 1;
        // sequences without a position: zeros
        for (int b = blockIdx.x; b < p.seqs; b += gridDim.x)
            if (dec_len(p, b) == 0)
                for (int e = lane * 4; e < p.n_q * p.head_dim; e += 128)
                    store4((T*)p.out + (int64_t)b * p.n_q * p.head_dim + e, make_float4(0.f, 0.f, 0.f, 0.f));
        if (!ok) {       // copies under way are waited for (again with a limit) before the block's memory is given up
            volatile int none = 0;
            for (int i = 0; i < NST; ++i) mbar_wait(full + 8 * i, ph ^ (i >= s ? 1u : 0u), const_cast<volatile int*>(&none));
            for (int i = 0; i < NQ; ++i) mbar_wait(qfull + 8 * i, phq ^ (i >= sq ? 1u : 0u), const_cast<volatile int*>(&none));
        }
        return;
    }

    // ---- consumers ----
    int s = 0, sq = 0;
    uint32_t ph = 0, phq = 0;
    bool ok = true;
    auto wait_full = [&]() {
        if (ok) ok = __all_sync(0xffffffffu, mbar_spin(full + 8 * s, ph, abort_flag));
    };
    auto release = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + 8 * s);
        if (++s == NST) { s = 0; ph ^= 1u; }
    };
    constexpr int E = HD / 16, TPH = HD / E;              // in joins a thread has E columns of one head
    const int h8 = tid / TPH, d0 = (tid % TPH) * E;
    int opened = 0;                                       // pairs of which the range has a part: at most its first and its last
    auto put = [&](int b, int pass, int h, const float (&v)[E], float sum) {
        const int hkv = p.gz == 1 ? pass : pass / p.gz, g0 = (pass - hkv * p.gz) * PER;
        const float i = sum == 0.f ? 0.f : 1.f / sum;
        T* out = (T*)p.out + ((int64_t)b * p.n_q + hkv * p.group + g0 + h) * p.head_dim + d0;
        if (h < min(p.group - g0, PER))
#pragma unroll
            for (int e = 0; e < E; e += 4)
                if (d0 + e < p.head_dim) store4(out + e, make_float4(v[e] * i, v[e + 1] * i, v[e + 2] * i, v[e + 3] * i));
    };
    while (w.left > 0) {
        const int hkv = p.gz == 1 ? w.h : w.h / p.gz, g0 = (w.h - hkv * p.gz) * PER;
        const int G = min(p.group - g0, PER);
        const int n = (int)min(w.left, (int64_t)(w.nt - w.t));
        const int len = w.len;
        const int64_t unit0 = r1 - w.left;                      // this part's first unit
        if (ok) ok = __all_sync(0xffffffffu, mbar_spin(qfull + 8 * sq, phq, abort_flag));
        const uint32_t qaddr = s_q + sq * QB;
        constexpr int NT = BF ? GH / 8 : 1, MT = HD / 16, VE = HD / 32;
        float o[BF ? MT * NT * 4 : GH * VE];
#pragma unroll
        for (int i = 0; i < (BF ? MT * NT * 4 : GH * VE); ++i) o[i] = 0.f;
        constexpr int NH = BF ? 2 * NT : GH;                    // heads whose maximum and sum a lane holds
        float m[NH], l[NH];
#pragma unroll
        for (int i = 0; i < NH; ++i) { m[i] = -INFINITY; l[i] = 0.f; }

        if constexpr (BF) {
            const int r = lane >> 2, c2 = (lane & 3) * 2;
            uint32_t qb[MT][NT][2];                             // head r of eight, dims c2 (+ 8) of sixteen
#pragma unroll
            for (int k = 0; k < MT; ++k)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int h = j * 8 + r, d = k * 16 + c2 + i * 8;
                        const uint32_t x = lds32(qaddr + (uint32_t)(min(h, G - 1) * p.head_dim + min(d, p.head_dim - 2)) * 2u);
                        qb[k][j][i] = h < G && d < p.head_dim ? x : 0u;
                    }
            __syncwarp();
            if (lane == 0) mbar_arrive(qempty + 8 * sq);
            // the weighted V so far to the sums in memory, or these to it
            float* sums = p.sums + (blockIdx.x * kDecWarps + warp) * dec_sums<HD, GH>() + lane;
            auto fold = [&](bool first, bool last) {
                constexpr int X = MT * NT * 4;
                float f[NH];
#pragma unroll
                for (int x = 0; x < NH; ++x) {
                    f[x] = first ? 0.f : ex2(sums[(X + x) * 32] - finite_max(m[x]));
                    if (!last) sums[(X + x) * 32] = m[x];
                }
#pragma unroll
                for (int x = 0; x < X; ++x) {
                    if (!first) o[x] = fmaf(sums[x * 32], f[(x >> 2) % NT * 2 + (x & 1)], o[x]);
                    if (!last) {
                        sums[x * 32] = o[x];
                        o[x] = 0.f;
                    }
                }
            };
            // rows and pieces of the four 8 x 8 matrices of a load: K as it lies, V transposed
            const int kr = lane & 15, kc = lane >> 4, vr = (lane & 7) + (lane >> 4) * 8, vc = (lane >> 3) & 1;
            for (int i = 0; i < n; ++i) {
                const int pos = (w.t + i) * TILE + warp * 16;
                wait_full();
                const bool mine = ok && pos < len && (s_seen[s] >> warp) & 1;
                float sc[NT][4];
                if (mine) {
                    const uint32_t kb = ring + s * STAGE + warp * 16 * 128;
                    float s2[NT][4];
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) sc[j][e] = s2[j][e] = 0.f;
#pragma unroll
                    for (int k = 0; k < MT; ++k) {              // (two chains of MMAs)
                        uint32_t a[4];
                        ldsm4(kb + (k >> 2) * BLK + kr * 128 + (((2 * (k & 3) + kc) ^ (kr & 7)) << 4), a);
#pragma unroll
                        for (int j = 0; j < NT; ++j) mma_bf16(k & 1 ? s2[j] : sc[j], a, qb[k][j][0], qb[k][j][1]);
                    }
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) sc[j][e] += s2[j][e];
                }
                release();
                uint32_t hi[NT][2], lo[NT][2];
                const int end = len - pos < 16 ? len - pos : 16;
                if (mine) {
                    bool grown = false;
                    float top[NH];
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            sc[j][e] = r < end ? sc[j][e] * p.scale2 : -INFINITY;
                            sc[j][2 + e] = r + 8 < end ? sc[j][2 + e] * p.scale2 : -INFINITY;
                            top[2 * j + e] = fmaxf(sc[j][e], sc[j][2 + e]);
                        }
#pragma unroll
                    for (int d = 4; d <= 16; d <<= 1)
#pragma unroll
                        for (int x = 0; x < NH; ++x) top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], d));
#pragma unroll
                    for (int x = 0; x < NH; ++x) {
                        top[x] = fmaxf(top[x], m[x]);
                        grown |= top[x] > m[x];
                    }
                    if (__any_sync(0xffffffffu, grown)) {
                        float f[NH];
#pragma unroll
                        for (int x = 0; x < NH; ++x) {
                            f[x] = ex2(m[x] - finite_max(top[x]));
                            m[x] = top[x];
                            l[x] *= f[x];
                        }
#pragma unroll
                        for (int x = 0; x < MT * NT * 4; ++x) o[x] *= f[(x >> 2) % NT * 2 + (x & 1)];
                    }
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const float m0 = finite_max(m[2 * j]), m1 = finite_max(m[2 * j + 1]);
#pragma unroll
                        for (int x = 0; x < 2; ++x) {           // positions r, r + 8
                            const float a = ex2(sc[j][2 * x] - m0), b = ex2(sc[j][2 * x + 1] - m1);
                            l[2 * j] += a;
                            l[2 * j + 1] += b;
                            // (cut, not rounded, and the rest zero with the weight alone: both terms of an infinite value have one sign)
                            const uint32_t h2 = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
                            hi[j][x] = turn8x8(h2);
                            lo[j][x] = turn8x8(bf16_pair(a - __uint_as_float(h2 << 16) + some_rest(a), b - __uint_as_float(h2 & 0xFFFF0000u) + some_rest(b)));
                        }
                    }
                }
                wait_full();
                if (mine && ok) {
                    const uint32_t vb = ring + s * STAGE + warp * 16 * 128;
                    if (end < 16) {          // V's rows behind the end: zeros, whatever was in the page
                        for (int e = end * 8 * BLKS + lane; e < 16 * 8 * BLKS; e += 32) {
                            const int x = e / (8 * BLKS), c = e - x * (8 * BLKS);
                            sts128(vb + (c >> 3) * BLK + x * 128 + ((c & 7) << 4), 0u, 0u, 0u, 0u);
                        }
                        fence_async_smem();
                        __syncwarp();
                    }
#pragma unroll
                    for (int k = 0; k < MT; ++k) {
                        uint32_t a[4];
                        ldsm4t(vb + (k >> 2) * BLK + vr * 128 + (((2 * (k & 3) + vc) ^ (vr & 7)) << 4), a);
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            float(&d)[4] = *reinterpret_cast<float(*)[4]>(&o[(k * NT + j) * 4]);
                            mma_bf16(d, a, hi[j][0], hi[j][1]);
                            mma_bf16(d, a, lo[j][0], lo[j][1]);
                        }
                    }
                }
                release();
                if ((i + 1) % kDecFold == 0) fold(i + 1 == kDecFold, false);
            }
            if (n >= kDecFold) fold(false, true);
#pragma unroll
            for (int x = 0; x < NH; ++x) {
#pragma unroll
                for (int d = 4; d <= 16; d <<= 1) l[x] += __shfl_xor_sync(0xffffffffu, l[x], d);
                if (r == 0) {
                    s_m[warp][(x >> 1) * 8 + c2 + (x & 1)] = m[x];
                    s_l[warp][(x >> 1) * 8 + c2 + (x & 1)] = l[x];
                }
            }
        } else {
            // position of the warp's eight (a quarter-warp reads rows of both halves of the swizzle), quarter of the pieces
            const int pr = ((lane >> 2) & 1) * 4 + (lane >> 3), pc = lane & 3;
            for (int i = 0; i < n; ++i) {
                const int pos = (w.t + i) * TILE + warp * 8;
                wait_full();
                const bool mine = ok && pos < len && (s_seen[s] >> (warp >> 1)) & 1;
                float pw[GH];
                if (mine) {
                    const uint32_t kb = ring + s * STAGE + warp * 8 * 128 + pr * 128;
                    float4 kk[HD / 16];
#pragma unroll
                    for (int j = 0; j < HD / 16; ++j) kk[j] = lds128(kb + (j >> 1) * BLK + (((pc + 4 * (j & 1)) ^ pr) << 4));
                    const bool in = pos + pr < len;
                    // (heads beyond the group's, of which nothing is used, are worked on too: without branches the heads' chains overlap)
                    float sc[GH];
#pragma unroll
                    for (int h = 0; h < GH; ++h) {
                        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                        for (int j = 0; j < HD / 16; ++j) {
                            const float4 x = (pc + 4 * j) * 4 < p.head_dim ? lds128(qaddr + (uint32_t)(h * p.head_dim + (pc + 4 * j) * 4) * 4u)
                                                                           : make_float4(0.f, 0.f, 0.f, 0.f);
                            a.x = fmaf(x.x, kk[j].x, a.x);
                            a.y = fmaf(x.y, kk[j].y, a.y);
                            a.z = fmaf(x.z, kk[j].z, a.z);
                            a.w = fmaf(x.w, kk[j].w, a.w);
                        }
                        sc[h] = (a.x + a.y) + (a.z + a.w);
                    }
#pragma unroll
                    for (int d = 1; d <= 2; d <<= 1)
#pragma unroll
                        for (int h = 0; h < GH; ++h) sc[h] += __shfl_xor_sync(0xffffffffu, sc[h], d);
                    float top[GH];
#pragma unroll
                    for (int h = 0; h < GH; ++h) {
                        sc[h] = in ? sc[h] * p.scale2 : -INFINITY;
                        top[h] = sc[h];
                    }
#pragma unroll
                    for (int d = 4; d <= 16; d <<= 1)
#pragma unroll
                        for (int h = 0; h < GH; ++h) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], d));
#pragma unroll
                    for (int h = 0; h < GH; ++h) {
                        const float now = fmaxf(top[h], m[h]), mf = finite_max(now), f = ex2(m[h] - mf);
                        m[h] = now;
                        pw[h] = ex2(sc[h] - mf);
                        l[h] = fmaf(l[h], f, pw[h]);
#pragma unroll
                        for (int e = 0; e < VE; ++e) o[h * VE + e] *= f;
                    }
                }
                release();
                wait_full();
                if (mine && ok) {
                    const uint32_t vb = ring + s * STAGE + warp * 8 * 128;
                    const int end = len - pos < 8 ? len - pos : 8;
                    if (end < 8) {           // V's rows behind the end: zeros, whatever was in the page
                        for (int e = end * 8 * BLKS + lane; e < 8 * 8 * BLKS; e += 32) {
                            const int x = e / (8 * BLKS), c = e - x * (8 * BLKS);
                            sts128(vb + (c >> 3) * BLK + x * 128 + ((c & 7) << 4), 0u, 0u, 0u, 0u);
                        }
                        fence_async_smem();
                        __syncwarp();
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        float vv[VE];
                        if constexpr (VE == 8) {
                            const uint32_t a = vb + (lane >> 2) * BLK + j * 128;
                            const float4 x = lds128(a + ((((lane & 3) * 2) ^ j) << 4)), y = lds128(a + ((((lane & 3) * 2 + 1) ^ j) << 4));
                            vv[0] = x.x; vv[1] = x.y; vv[2] = x.z; vv[3] = x.w;
                            vv[4] = y.x; vv[5] = y.y; vv[6] = y.z; vv[7] = y.w;
                        } else if constexpr (VE == 4) {
                            const float4 x = lds128(vb + (lane >> 3) * BLK + j * 128 + (((lane & 7) ^ j) << 4));
                            vv[0] = x.x; vv[1] = x.y; vv[2] = x.z; vv[3] = x.w;
                        } else {
                            const uint32_t a = vb + (lane >> 4) * BLK + j * 128 + ((((lane >> 1) & 7) ^ j) << 4) + (lane & 1) * 8;
                            vv[0] = __uint_as_float(lds32(a));
                            vv[1] = __uint_as_float(lds32(a + 4));
                        }
#pragma unroll
                        for (int h = 0; h < GH; ++h) {
                            const float pj = __shfl_sync(0xffffffffu, pw[h], ((j >> 2) & 1) * 4 + (j & 3) * 8);
#pragma unroll
                            for (int e = 0; e < VE; ++e) o[h * VE + e] = fmaf(pj, vv[e], o[h * VE + e]);
                        }
                    }
                }
                release();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(qempty + 8 * sq);
#pragma unroll
            for (int h = 0; h < GH; ++h) {
#pragma unroll
                for (int d = 4; d <= 16; d <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], d);
                if (lane == 0) {
                    s_m[warp][h] = m[h];
                    s_l[warp][h] = l[h];
                }
            }
        }
        if (++sq == NQ) { sq = 0; phq ^= 1u; }

        // ---- the warps' states joined, eight heads at a time: a thread has E columns of one head ----
        const bool whole = w.t == 0 && n == w.nt;
        float* slot = p.part + (2 * (int64_t)blockIdx.x + (w.t == 0 ? 1 : 0)) * SLOT;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            float* slab = s_slab + warp * SLAB;
            if constexpr (BF) {
#pragma unroll
                for (int k = 0; k < MT; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) slab[((lane & 3) * 2 + (i & 1)) * (HD + 4) + k * 16 + (lane >> 2) + (i >> 1) * 8] = o[(k * NT + j) * 4 + i];
            } else {
#pragma unroll
                for (int h = 0; h < GH; ++h)
#pragma unroll
                    for (int e = 0; e < VE; ++e) slab[h * (HD + 4) + lane * VE + e] = o[h * VE + e];
            }
            bar_consumers();
            const int h = j * 8 + h8;
            if (h8 < (GH < 8 ? GH : 8)) {
                float top = -INFINITY, sum = 0.f, a[E];
#pragma unroll
                for (int x = 0; x < kDecWarps; ++x) top = fmaxf(top, s_m[x][h]);
#pragma unroll
                for (int e = 0; e < E; ++e) a[e] = 0.f;
                const float tf = finite_max(top);
#pragma unroll
                for (int x = 0; x < kDecWarps; ++x) {
                    const float f = ex2(s_m[x][h] - tf);
                    sum = fmaf(f, s_l[x][h], sum);
#pragma unroll
                    for (int e = 0; e < E; e += 4) {
                        const float4 y = *reinterpret_cast<const float4*>(s_slab + x * SLAB + h8 * (HD + 4) + d0 + e);
                        a[e] = fmaf(f, y.x, a[e]);
                        a[e + 1] = fmaf(f, y.y, a[e + 1]);
                        a[e + 2] = fmaf(f, y.z, a[e + 2]);
                        a[e + 3] = fmaf(f, y.w, a[e + 3]);
                    }
                }
                if (whole) put(w.b, w.h, h, a, sum);
                else {
#pragma unroll
                    for (int e = 0; e < E; e += 4) store4(slot + h * HD + d0 + e, make_float4(a[e], a[e + 1], a[e + 2], a[e + 3]));
                    if (d0 == 0) {
                        slot[kPagedGroup * HD + h] = top;
                        slot[kPagedGroup * (HD + 1) + h] = sum;
                    }
                }
            }
            if (j + 1 < NT) bar_consumers();
        }
        if (!whole) {            // blocks of this pair: those of its first and last unit, and all between
            const int64_t f = unit0 - w.t, e = f + w.nt - 1;
            if (tid == 0) s_open[opened] = make_int4(w.b, w.h, (int)(((f + 1) * blocks - 1) / total), (int)(((e + 1) * blocks - 1) / total));
            ++opened;
        }
        bar_consumers();       // s_m, s_l, s_slab are the next part's
        dec_past<TILE>(p, H, &w, n);
    }
    // ---- pairs of several ranges: whoever comes last joins their parts.  Asked at the end of the range for both: a fence and an atomic
    // ---- between two parts kept the block from its tiles for 3 us (f32, under load 5).
    if (opened > 0) {
        __threadfence();
        bar_consumers();
        if (tid < opened) {
            const int c0 = s_open[tid].z, c1 = s_open[tid].w;
            s_last[tid] = atomicAdd(&p.counters[c0], 1) == c1 - c0;
        }
        bar_consumers();
        for (int x = 0; x < opened; ++x) {
            if (!s_last[x]) continue;
            const int b = s_open[x].x, pass = s_open[x].y, c0 = s_open[x].z, c1 = s_open[x].w;
            __threadfence();
            if (tid == 0) p.counters[c0] = 0;
            const int G = min(p.group - (p.gz == 1 ? 0 : pass % p.gz) * PER, PER);
#pragma unroll
            for (int j = 0; j < (BF ? GH / 8 : 1); ++j) {
                if (G <= j * 8) continue;
                constexpr int U = 4;                  // slots asked for at a time
                // eight rows of threads: those that the heads leave over share the slots, if these are many
                int heads = c1 - c0 < U ? 8 : 1;
                while (heads < 8 && heads < G - j * 8) heads *= 2;
                const int sets = 8 / heads, set = h8 / heads, h = j * 8 + h8 - set * heads;
                float top = -INFINITY, sum = 0.f, a[E];
#pragma unroll
                for (int x = 0; x < E; ++x) a[x] = 0.f;
                for (int c = h < G ? c0 + set * U : c1 + 1; c <= c1; c += sets * U) {
                    float mm[U], ll[U], vv[U][E];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const float* from = p.part + (2 * (int64_t)min(c + u, c1) + (c + u == c0 ? 1 : 0)) * SLOT;
                        mm[u] = __ldcg(from + kPagedGroup * HD + h);
                        ll[u] = __ldcg(from + kPagedGroup * (HD + 1) + h);
#pragma unroll
                        for (int x = 0; x < E; x += 4) {
                            const float4 y = __ldcg(reinterpret_cast<const float4*>(from + h * HD + d0 + x));
                            vv[u][x] = y.x; vv[u][x + 1] = y.y; vv[u][x + 2] = y.z; vv[u][x + 3] = y.w;
                        }
                    }
                    float next = top;
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (c + u <= c1) next = fmaxf(next, mm[u]);
                    const float nf = finite_max(next), g = ex2(top - nf);
                    top = next;
                    sum *= g;
#pragma unroll
                    for (int x = 0; x < E; ++x) a[x] *= g;
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (c + u <= c1) {
                            const float fu = ex2(mm[u] - nf);
                            sum = fmaf(fu, ll[u], sum);
#pragma unroll
                            for (int x = 0; x < E; ++x) a[x] = fmaf(fu, vv[u][x], a[x]);
                        }
                }
                if (sets > 1) {
                    bar_consumers();                  // (the arrays have been read by whoever used them before)
#pragma unroll
                    for (int e = 0; e < E; e += 4) store4(s_slab + h8 * (HD + 4) + d0 + e, make_float4(a[e], a[e + 1], a[e + 2], a[e + 3]));
                    if (d0 == 0) {
                        s_m[0][h8] = top;
                        s_l[0][h8] = sum;
                    }
                    bar_consumers();
                    if (set == 0) {
                        float all = -INFINITY;
                        for (int q = 0; q < sets; ++q) all = fmaxf(all, s_m[0][q * heads + h8]);
                        const float tf = finite_max(all);
                        sum = 0.f;
#pragma unroll
                        for (int e = 0; e < E; ++e) a[e] = 0.f;
                        for (int q = 0; q < sets; ++q) {
                            const int y = q * heads + h8;
                            const float f = ex2(s_m[0][y] - tf);
                            sum = fmaf(f, s_l[0][y], sum);
#pragma unroll
                            for (int e = 0; e < E; ++e) a[e] = fmaf(f, s_slab[y * (HD + 4) + d0 + e], a[e]);
                        }
                    }
                }
                if (set == 0) put(b, pass, h, a, sum);
            }
        }
    }
    if (tid == 0 && s_abort) atomicExch(p.status, 2);
}

int32_t decode_configure(DeviceState& ds) {
    constexpr auto attr = cudaFuncAttributeMaxDynamicSharedMemorySize;
    auto set = [&](auto kernel, int smem) { return cudaFuncSetAttribute(kernel, attr, smem); };
    RSTQ_CUDA(set(paged_decode_kernel<__nv_bfloat16, 64, 8>, dec_smem<64>()));
    RSTQ_CUDA(set(paged_decode_kernel<__nv_bfloat16, 64, 16>, dec_smem<64>()));
    RSTQ_CUDA(set(paged_decode_kernel<float, 64, 1>, dec_smem<64>()));
    RSTQ_CUDA(set(paged_decode_kernel<float, 64, 4>, dec_smem<64>()));
    RSTQ_CUDA(set(paged_decode_kernel<float, 64, 8>, dec_smem<64>()));
    RSTQ_CUDA(set(paged_decode_kernel<__nv_bfloat16, 128, 8>, dec_smem<128>()));
    RSTQ_CUDA(set(paged_decode_kernel<__nv_bfloat16, 128, 16>, dec_smem<128>()));
    RSTQ_CUDA(set(paged_decode_kernel<float, 128, 1>, dec_smem<128>()));
    RSTQ_CUDA(set(paged_decode_kernel<float, 128, 4>, dec_smem<128>()));
    RSTQ_CUDA(set(paged_decode_kernel<float, 128, 8>, dec_smem<128>()));
    RSTQ_CUDA(set(paged_decode_kernel<__nv_bfloat16, 256, 8>, dec_smem<256>()));
    RSTQ_CUDA(set(paged_decode_kernel<__nv_bfloat16, 256, 16>, dec_smem<256>()));
    RSTQ_CUDA(set(paged_decode_kernel<float, 256, 1>, dec_smem<256>()));
    RSTQ_CUDA(set(paged_decode_kernel<float, 256, 4>, dec_smem<256>()));
    RSTQ_CUDA(set(paged_decode_kernel<float, 256, 8>, dec_smem<256>()));
    RSTQ_CUDA(cudaMalloc((void**)&ds.seq_starts, (size_t)(kMaxSeqs + 1) * 8));
    return RSTQ_OK;
}

int32_t rows_tensor_map(CUtensorMap* m, const void* base, int32_t dtype, int64_t rows, int64_t ld, int heads, int head_dim, int box) {
    const EncodeTiledFn enc = encode_tiled_fn();
    RSTQ_REQUIRE(enc, RSTQ_E_CUDA, "cuTensorMapEncodeTiled is not available");
    const cuuint64_t es = (cuuint64_t)elem_bytes(dtype);
    const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)heads, (cuuint64_t)(rows > 0 ? rows : 1)};
    const cuuint64_t strides[2] = {head_dim * es, (cuuint64_t)ld * es};
    const cuuint32_t bx[3] = {(cuuint32_t)(128 / es), 1u, (cuuint32_t)box}, ones[3] = {1u, 1u, 1u};
    const CUresult r = enc(m, dtype == RSTQ_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void*>(base), dims,
                           strides, bx, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    RSTQ_REQUIRE(r == CUDA_SUCCESS, RSTQ_E_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return RSTQ_OK;
}

int32_t launch_paged_decode(DeviceState& ds, const PromptArgs& a, int* launches) {
    DecodeParams p;
    p.q = a.q; p.k = a.k; p.v = a.v; p.out = a.out;
    p.kv = a.kv;
    p.ldq = a.ldq;
    p.seqs = a.seqs; p.n_q = a.n_q; p.group = a.group; p.n_kv = a.n_kv; p.head_dim = a.head_dim;
    const int per = a.dtype == RSTQ_BF16 ? dec_heads<__nv_bfloat16>() : dec_heads<float>();
    p.gz = (a.group + per - 1) / per;
    p.scale2 = a.scale * 1.4426950408889634f;
    p.part = ds.partials;
    p.counters = ds.counters;
    p.status = ds.status;
    const int page = 1 << a.kv.shift, tile = a.dtype == RSTQ_BF16 ? dec_tile<__nv_bfloat16>() : dec_tile<float>();
    p.box = std::min(page, tile);
    CUtensorMap kmap, vmap;
    int32_t rc = rows_tensor_map(&kmap, a.k, a.dtype, a.kv_rows, a.kv.ld, a.n_kv, a.head_dim, p.box);
    if (rc == RSTQ_OK) rc = rows_tensor_map(&vmap, a.v, a.dtype, a.kv_rows, a.kv.ld, a.n_kv, a.head_dim, p.box);
    if (rc != RSTQ_OK) return rc;
    const int64_t blocks = (a.head_dim > 128 ? dec_blocks<256>() : dec_blocks<128>()) * (int64_t)ds.sm_count;
    const int64_t slot = a.head_dim > 128 ? dec_slot<256>() : dec_slot<128>();
    constexpr int sums = kDecWarps * dec_sums<256, kPagedGroup>();
    p.sums = ds.prompt_slots;
    RSTQ_REQUIRE(2 * blocks * slot * 4 <= ds.partials_bytes && blocks <= ds.counters_len && blocks * sums <= kPromptSlotFloats, RSTQ_E_LIMIT,
                 "%lld thread blocks", (long long)blocks);
    *launches = 1;
    p.start = nullptr;
    if (a.seqs > kDecSums) {
        if ((rc = launch_sums(ds, a, tile, kDecEnd)) != RSTQ_OK) return rc;
        p.start = ds.seq_starts;
        ++*launches;
    }
    const int g = std::min(a.group, per);
    auto go = [&](auto kernel, int smem) { return launch_pdl(kernel, dim3((unsigned)blocks), dim3(kDecThreads), (size_t)smem, ds, p, kmap, vmap); };
    auto sized = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        using B = __nv_bfloat16;
        if (a.dtype == RSTQ_BF16) return g <= 8 ? go(paged_decode_kernel<B, HD, 8>, dec_smem<HD>()) : go(paged_decode_kernel<B, HD, 16>, dec_smem<HD>());
        return g == 1   ? go(paged_decode_kernel<float, HD, 1>, dec_smem<HD>())
               : g <= 4 ? go(paged_decode_kernel<float, HD, 4>, dec_smem<HD>())
                        : go(paged_decode_kernel<float, HD, 8>, dec_smem<HD>());
    };
    const cudaError_t e = a.head_dim <= 64 ? sized(std::integral_constant<int, 64>()) : a.head_dim <= 128 ? sized(std::integral_constant<int, 128>())
                                                                                                        : sized(std::integral_constant<int, 256>());
    RSTQ_CUDA(e);
    return RSTQ_OK;
}

}  // namespace rstq
