// Attention of one new token per sequence over a paged cache, head_dim up to 128.
//
//   out[b, h] = sum_j p_j V[b, j] / sum_j p_j,   p_j = exp(scale q.K[b, j] - m),   j < lens[b]
//
// Bound by HBM: every cached row is read once, for all query heads of its KV head (up to 16, in f32 8; larger groups in several passes).
//
// Work.  A unit is a tile of positions (64 in bf16, 32 in f32) of one sequence and KV head; the units of all sequences lie
// on one line (sequence, head, tile) and every thread block takes an equal range of it, so that lengths may be as different as they
// like and few long sequences use all SMs.  The ranges follow from the lengths alone, which are read on the device: one recorded
// launch serves every step.  A (sequence, head) pair that lies in one range is finished there; the parts of one that spans
// several are left in slots, and the block that comes last (an arrival counter) joins them in the order of the ranges, so the
// result does not depend on who came last.  Nobody waits for another block.
//
// Block.  A thread brings K and V by TMA, a box per page (its rows 128 bytes wide, swizzled), through a ring of 96 KB, two blocks
// per SM, and the queries of each part ahead of it; four warps take a quarter of each tile's positions and keep a softmax of their own
// (running maximum, sum, weighted V), joined at the end of a range's part.  V's rows behind the end are zeroed in shared memory before they
// are used and their scores masked, so what stale pages hold never reaches a result.
//   bf16: m16n8k16 MMAs, the query heads of the group in the 16 rows; scores and weights stay in registers.  A weight enters
//         P.V as the sum of two bf16 terms (16 bits): the second product is free beside the copies.
//   f32:  a lane forms a quarter of a dot product in f32 FMAs for each head of the group, then owns four (two) columns of V.
#include <algorithm>
#include <type_traits>

#include "paged.cuh"
#include "sync_helpers.cuh"
#include "tcgen05_helpers.cuh"

namespace rstq {

constexpr int kDecWarps = 4;                          // consumers; one more warp copies
constexpr int kDecThreads = (kDecWarps + 1) * 32;
constexpr int kDecRing = 96 * 1024;
constexpr int kDecMerge = 8 * 1024;                   // sums on their way from warp to warp
constexpr int kDecQ = 8 * 1024 - 1024;                // queries of the parts to come (1 KB of it: the ring's alignment)
constexpr int kDecSmem = kDecRing + kDecMerge + 8 * 1024;

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
};
template <typename T>
__host__ __device__ constexpr int dec_tile() { return sizeof(T) == 2 ? 64 : 32; }
template <typename T, int HD>
__host__ __device__ constexpr int dec_stage() { return dec_tile<T>() * HD * (int)sizeof(T) * 2; }
// Query heads of a KV head that one pass serves.  f32: eight, so that a pass's sums fit its registers; a larger group's other
// heads find the rows in L2.
template <typename T>
__host__ __device__ constexpr int dec_heads() { return sizeof(T) == 2 ? kPagedGroup : kPagedGroup / 2; }
// a slot: HD / 2 sums per lane, then the heads' maxima and sums of weights
template <int HD>
__host__ __device__ constexpr int dec_slot() { return HD / 2 * 32 + 2 * kPagedGroup; }

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
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.f : m; }   // nothing seen yet: exp2(-inf - 0) = 0
__device__ __forceinline__ void bar_consumers() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

constexpr float kRest = 7.8886091e-31f;      // 2^-100

// Where a block's range of units lies.  Units of sequence b: its tiles for each of H heads.  All lanes of a warp hold the same,
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
// Total units, and the place of the first one of the range that `range` gives for it.
template <int TILE, typename F>
__device__ __forceinline__ int64_t dec_find(const DecodeParams& p, int H, Walk* w, F range) {
    const int lane = threadIdx.x & 31;
    const int head = dec_len(p, lane);
    int64_t total = (head + TILE - 1) / TILE;
    for (int b0 = 32; b0 < p.seqs; b0 += 128) {
        int n[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) n[u] = dec_len(p, b0 + u * 32 + lane);
#pragma unroll
        for (int u = 0; u < 4; ++u) total += (n[u] + TILE - 1) / TILE;
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    total *= H;
    int64_t first, last;
    range(total, &first, &last);
    w->left = last - first;
    if (w->left <= 0) return total;
    int64_t base = 0;
    for (int b0 = 0; b0 < p.seqs; b0 += 32) {
        const int len = b0 ? dec_len(p, b0 + lane) : head;
        const int n = (len + TILE - 1) / TILE;
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
            w->nt = __shfl_sync(0xffffffffu, n, src);
            const int64_t in = first - (end - (int64_t)w->nt * H);
            w->h = (int)(in / w->nt);
            w->t = (int)(in - (int64_t)w->h * w->nt);
            return total;
        }
        base += __shfl_sync(0xffffffffu, x, 31);
    }
    w->left = 0;
    return total;
}
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

// GH: query heads served at once (bf16: 8 or 16; f32: what the group needs)
template <typename T, int HD, int GH>
__global__ void __launch_bounds__(kDecThreads, 2)
paged_decode_kernel(const DecodeParams p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    constexpr int TILE = dec_tile<T>(), STAGE = dec_stage<T, HD>(), NST = kDecRing / STAGE, R = HD / 2;
    constexpr int ES = (int)sizeof(T), BLKS = HD * ES / 128, BLK = TILE * 128;      // a tile's rows in pieces of 128 bytes: BLKS blocks
    constexpr bool BF = ES == 2;
    constexpr int SLOT = dec_slot<HD>(), QB = GH * HD * ES, NQ = kDecQ / QB >= 4 ? 4 : kDecQ / QB;
    constexpr int PER = dec_heads<T>();               // query heads of a pass
    static_assert(NST >= 3 && NST <= 6 && NQ >= 1 && GH <= PER, "ring");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ uint8_t s_raw0[];
    uint8_t* s_raw = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(s_raw0) + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t s_bar[2 * NST + 2 * NQ];
    __shared__ uint32_t s_seen[NST];                  // which sixteens of a stage's positions are there
    __shared__ float s_m[kDecWarps][kPagedGroup], s_l[kDecWarps][kPagedGroup];
    __shared__ int s_abort, s_last;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t ring = smem_u32(s_raw), full = smem_u32(s_bar), empty = full + 8 * NST, qfull = empty + 8 * NST, qempty = qfull + 8 * NQ;
    float* s_merge = reinterpret_cast<float*>(s_raw + kDecRing);
    uint8_t* s_q = s_raw + kDecRing + kDecMerge;
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
    int64_t blocks = gridDim.x, r0 = 0, r1 = 0, total = 0;
    Walk w;
    w.left = 0;
    total = dec_find<TILE>(p, H, &w, [&](int64_t n, int64_t* a, int64_t* e) {
        if (blocks > n) blocks = n;                   // every range has a unit at least
        r0 = blockIdx.x < blocks ? blockIdx.x * n / blocks : 0;
        r1 = blockIdx.x < blocks ? (blockIdx.x + 1) * n / blocks : 0;
        *a = r0;
        *e = r1;
    });

    if (warp == kDecWarps) {
        // ---- copies ----
        int s = 0, sq = 0;
        uint32_t ph = 0, phq = 0;
        bool bad = false, ok = true, first = true;
        // Page of the lane's sixteen of a tile's positions (lanes 0 .. TILE/16 - 1 matter), asked for a tile ahead.
        auto page_of = [&]() {
            const int pos = w.t * TILE + lane * 16;
            return w.left > 0 && lane < TILE / 16 && pos < w.len ? p.kv.table[(int64_t)w.b * p.kv.width + (pos >> p.kv.shift)] : 0;
        };
        int page = page_of();
        while (w.left > 0 && ok) {
            const int hkv = w.h / p.gz, pos0 = w.t * TILE, len = w.len;
            if (first) {      // the part's queries: rows of the group's heads, one behind the other
                first = false;
                const int g0 = (w.h - hkv * p.gz) * PER, G = min(p.group - g0, PER);
                ok = __all_sync(0xffffffffu, mbar_block(qempty + 8 * sq, phq ^ 1u, abort_flag));
                if (!ok) break;
                if (lane == 0) {
                    const uint32_t bytes = (uint32_t)(G * p.head_dim * ES);
                    mbar_expect_tx(qfull + 8 * sq, bytes);
                    bulk_copy_g2s(smem_u32(s_q) + sq * QB, (const T*)p.q + (int64_t)w.b * p.ldq + (int64_t)(hkv * p.group + g0) * p.head_dim, bytes, qfull + 8 * sq);
                }
                if (++sq == NQ) { sq = 0; phq ^= 1u; }
            }
            const bool there = (uint32_t)page < (uint64_t)p.kv.n_pages;
            const unsigned seen = __ballot_sync(0xffffffffu, there) & ((1u << (TILE / 16)) - 1);
            bad |= !there;
            const int row = there ? (page << p.kv.shift) + ((pos0 + lane * 16) & ((1 << p.kv.shift) - 1)) : 0;
            // the walk goes on: the next tile's pages are asked for before this one's copies
            --w.left;
            if (++w.t == w.nt && w.left > 0) {
                dec_next<TILE>(p, H, &w);
                first = true;
            }
            page = page_of();
            ok = __all_sync(0xffffffffu, mbar_block(empty + 8 * s, ph ^ 1u, abort_flag));
            if (!ok) break;
            const int per = p.box >> 4;               // sixteens of a box
            // boxes that begin before the end and whose page is one
            unsigned boxes = 0;
            for (int g = 0; g < TILE / 16; g += per) boxes |= pos0 + g * 16 < len && ((seen >> g) & 1) ? 1u << g : 0u;
            const uint32_t bar = full + 8 * s, dst = ring + s * STAGE;
            if (lane == 0) {
                s_seen[s] = seen;
                if (boxes) mbar_expect_tx(bar, (uint32_t)(__popc(boxes) * p.box * 128 * BLKS * 2));
                else mbar_arrive(bar);
            }
            for (int g = 0; g < TILE / 16; g += per) {
                const int y = __shfl_sync(0xffffffffu, row, g);
                if (lane == 0 && ((boxes >> g) & 1)) {
#pragma unroll
                    for (int c = 0; c < BLKS; ++c) {
                        tma_load_3d(dst + c * BLK + g * 16 * 128, &kmap, c * (128 / ES), hkv, y, bar);
                        tma_load_3d(dst + (BLKS + c) * BLK + g * 16 * 128, &vmap, c * (128 / ES), hkv, y, bar);
                    }
                }
            }
            if (++s == NST) { s = 0; ph ^= 1u; }
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
    while (w.left > 0) {
        const int hkv = w.h / p.gz, g0 = (w.h - hkv * p.gz) * PER;
        const int G = min(p.group - g0, PER);
        const int n = (int)(w.left < w.nt - w.t ? w.left : w.nt - w.t);
        const int len = w.len;
        const int64_t unit0 = r1 - w.left;                      // this part's first unit
        if (ok) ok = __all_sync(0xffffffffu, mbar_spin(qfull + 8 * sq, phq, abort_flag));
        const uint32_t qaddr = smem_u32(s_q) + sq * QB;
        float o[R];
#pragma unroll
        for (int i = 0; i < R; ++i) o[i] = 0.f;
        constexpr int NH = BF ? 2 : GH;                         // heads whose maximum and sum a lane holds
        float m[NH], l[NH];
#pragma unroll
        for (int i = 0; i < NH; ++i) { m[i] = -INFINITY; l[i] = 0.f; }

        if constexpr (BF) {
            const int hr = lane >> 2, cc = (lane & 3) * 2;
            uint32_t qa[HD / 16][4];
#pragma unroll
            for (int k = 0; k < HD / 16; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int h = hr + (i & 1) * 8, d = k * 16 + cc + (i >> 1) * 8;
                    qa[k][i] = 0u;
                    if (GH == 8 && (i & 1)) continue;
                    const uint32_t x = lds32(qaddr + (uint32_t)(min(h, G - 1) * p.head_dim + min(d, p.head_dim - 2)) * 2u);
                    qa[k][i] = h < G && d < p.head_dim ? x : 0u;
                }
            __syncwarp();
            if (lane == 0) mbar_arrive(qempty + 8 * sq);
            for (int i = 0; i < n; ++i) {
                if (ok) ok = __all_sync(0xffffffffu, mbar_spin(full + 8 * s, ph, abort_flag));
                const int pos = (w.t + i) * TILE + warp * 16;
                if (ok && pos < len && (s_seen[s] >> warp) & 1) {
                    const uint32_t kb = ring + s * STAGE + warp * 16 * 128, vb = kb + BLKS * BLK;
                    const int end = len - pos < 16 ? len - pos : 16;
                    if (end < 16) {          // V's rows behind the end: zeros, whatever was in the page
                        for (int e = end * 8 * BLKS + lane; e < 16 * 8 * BLKS; e += 32) {
                            const int r = e / (8 * BLKS), c = e - r * (8 * BLKS);
                            sts128(vb + (c >> 3) * BLK + r * 128 + ((c & 7) << 4), 0u, 0u, 0u, 0u);
                        }
                        fence_async_smem();
                        __syncwarp();
                    }
                    float sc[2][4] = {};
                    // matrices of an x4: positions 0-7 / 8-15 by the lane's bit 4, dims 0-7 / 8-15 by bit 3
                    const int kr = (lane & 7) + ((lane >> 4) << 3), kc = (lane >> 3) & 1;
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k) {
                        uint32_t b[4];
                        ldsm4(kb + (k >> 2) * BLK + kr * 128 + (((2 * (k & 3) + kc) ^ (kr & 7)) << 4), b);
                        mma_bf16(sc[0], qa[k], b[0], b[1]);
                        mma_bf16(sc[1], qa[k], b[2], b[3]);
                    }
                    float top[2] = {m[0], m[1]};
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (GH == 8 && e >= 2) continue;
                            sc[j][e] = j * 8 + cc + (e & 1) < end ? sc[j][e] * p.scale2 : -INFINITY;
                            top[e >> 1] = fmaxf(top[e >> 1], sc[j][e]);
                        }
                    bool grown = false;
#pragma unroll
                    for (int x = 0; x < (GH == 8 ? 1 : 2); ++x) {
                        top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 1));
                        top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 2));
                        grown |= top[x] > m[x];
                    }
                    if (__any_sync(0xffffffffu, grown)) {
                        float f[2];
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            f[x] = ex2(m[x] - finite_max(top[x]));
                            m[x] = top[x];
                            l[x] *= f[x];
                        }
#pragma unroll
                        for (int r = 0; r < R; ++r) o[r] *= f[(r >> 1) & 1];
                    }
                    const float m0 = finite_max(m[0]), m1 = finite_max(m[1]);
                    uint32_t hi[4] = {0u, 0u, 0u, 0u}, lo[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int x = 0; x < (GH == 8 ? 1 : 2); ++x) {
                            const float a = ex2(sc[j][2 * x] - (x ? m1 : m0)), b = ex2(sc[j][2 * x + 1] - (x ? m1 : m0));
                            l[x] += a + b;
                            // (cut, not rounded, and the rest never zero: both terms of an infinite value have one sign)
                            const uint32_t h2 = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
                            hi[2 * j + x] = h2;
                            lo[2 * j + x] = bf16_pair(a - __uint_as_float(h2 << 16) + kRest, b - __uint_as_float(h2 & 0xFFFF0000u) + kRest);
                        }
                    // (transposed) matrices: positions by the lane's bit 3, dims by bit 4
                    const int vr = (lane & 7) + (((lane >> 3) & 1) << 3), vc = lane >> 4;
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k) {
                        uint32_t b[4];
                        ldsm4t(vb + (k >> 2) * BLK + vr * 128 + (((2 * (k & 3) + vc) ^ (vr & 7)) << 4), b);
                        float(&d0)[4] = *reinterpret_cast<float(*)[4]>(&o[8 * k]);
                        float(&d1)[4] = *reinterpret_cast<float(*)[4]>(&o[8 * k + 4]);
                        mma_bf16(d0, hi, b[0], b[1]);
                        mma_bf16(d1, hi, b[2], b[3]);
                        mma_bf16(d0, lo, b[0], b[1]);
                        mma_bf16(d1, lo, b[2], b[3]);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(empty + 8 * s);
                if (++s == NST) { s = 0; ph ^= 1u; }
            }
            // sums of weights over the four lanes of a row
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
                l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
                if ((lane & 3) == 0) {
                    s_m[warp][hr + 8 * x] = m[x];
                    s_l[warp][hr + 8 * x] = l[x];
                }
            }
        } else {
            constexpr int VE = HD / 32;               // columns of V a lane owns
            // position of the warp's eight (a quarter-warp reads rows of both halves of the swizzle), quarter of the pieces
            const int pr = ((lane >> 2) & 1) * 4 + (lane >> 3), pc = lane & 3;
            for (int i = 0; i < n; ++i) {
                if (ok) ok = __all_sync(0xffffffffu, mbar_spin(full + 8 * s, ph, abort_flag));
                const int pos = (w.t + i) * TILE + warp * 8;
                if (ok && pos < len && (s_seen[s] >> (warp >> 1)) & 1) {
                    uint8_t* kb = s_raw + s * STAGE + warp * 8 * 128;
                    uint8_t* vb = kb + BLKS * BLK;
                    const int end = len - pos < 8 ? len - pos : 8;
                    if (end < 8) {           // V's rows behind the end: zeros, whatever was in the page
                        for (int e = end * 8 * BLKS + lane; e < 8 * 8 * BLKS; e += 32) {
                            const int r = e / (8 * BLKS), c = e - r * (8 * BLKS);
                            *reinterpret_cast<float4*>(vb + (c >> 3) * BLK + r * 128 + ((c & 7) << 4)) = make_float4(0.f, 0.f, 0.f, 0.f);
                        }
                        fence_async_smem();
                        __syncwarp();
                    }
                    float4 kk[HD / 16];
#pragma unroll
                    for (int j = 0; j < HD / 16; ++j)
                        kk[j] = *reinterpret_cast<const float4*>(kb + (j >> 1) * BLK + pr * 128 + (((pc + 4 * (j & 1)) ^ pr) << 4));
                    float vv[8][VE];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if constexpr (VE == 4) {
                            const float4 x = *reinterpret_cast<const float4*>(vb + (lane >> 3) * BLK + j * 128 + (((lane & 7) ^ j) << 4));
                            vv[j][0] = x.x; vv[j][1] = x.y; vv[j][2] = x.z; vv[j][3] = x.w;
                        } else {
                            const float2 x = *reinterpret_cast<const float2*>(vb + (lane >> 4) * BLK + j * 128 + ((((lane >> 1) & 7) ^ j) << 4) + (lane & 1) * 8);
                            vv[j][0] = x.x; vv[j][1] = x.y;
                        }
                    }
                    const bool in = pos + pr < len;
#pragma unroll
                    for (int h = 0; h < GH; ++h) {
                        if (h < G) {
                            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                            for (int j = 0; j < HD / 16; ++j) {
                                const float4 x = (pc + 4 * j) * 4 < p.head_dim ? lds128(qaddr + (uint32_t)(h * p.head_dim + (pc + 4 * j) * 4) * 4u) : make_float4(0.f, 0.f, 0.f, 0.f);
                                a.x = fmaf(x.x, kk[j].x, a.x);
                                a.y = fmaf(x.y, kk[j].y, a.y);
                                a.z = fmaf(x.z, kk[j].z, a.z);
                                a.w = fmaf(x.w, kk[j].w, a.w);
                            }
                            float sc = (a.x + a.y) + (a.z + a.w);
                            sc += __shfl_xor_sync(0xffffffffu, sc, 1);
                            sc += __shfl_xor_sync(0xffffffffu, sc, 2);
                            sc = in ? sc * p.scale2 : -INFINITY;
                            float top = fmaxf(m[h], sc);
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                            const float mf = finite_max(top);
                            if (top > m[h]) {
                                const float f = ex2(m[h] - mf);
                                m[h] = top;
                                l[h] *= f;
#pragma unroll
                                for (int e = 0; e < VE; ++e) o[h * VE + e] *= f;
                            }
                            const float pw = ex2(sc - mf);
                            l[h] += pw;
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const float pj = __shfl_sync(0xffffffffu, pw, ((j >> 2) & 1) * 4 + (j & 3) * 8);
#pragma unroll
                                for (int e = 0; e < VE; ++e) o[h * VE + e] = fmaf(pj, vv[j][e], o[h * VE + e]);
                            }
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(empty + 8 * s);
                if (++s == NST) { s = 0; ph ^= 1u; }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(qempty + 8 * sq);
#pragma unroll
            for (int h = 0; h < GH; ++h) {
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 4);
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 8);
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 16);
                if (lane == 0) {
                    s_m[warp][h] = m[h];
                    s_l[warp][h] = l[h];
                }
            }
        }

        if (++sq == NQ) { sq = 0; phq ^= 1u; }

        // ---- the warps' states joined: sums of all to the common maximum, then added (2 + 3 to 0 + 1, 1 to 0; where two warps'
        // do not fit, 1 .. 3 to 0 one by one) ----
        constexpr int HEADS = BF ? GH : GH;
        auto head_of = [&](int r) { return BF ? (lane >> 2) + ((r >> 1) & 1) * 8 : r / (BF ? 1 : HD / 32); };
        constexpr int LIVE = BF ? R : GH * (HD / 32);     // sums of a lane that mean something
        bar_consumers();
        {
            float f[NH];
#pragma unroll
            for (int x = 0; x < NH; ++x) {
                const int h = BF ? (lane >> 2) + 8 * x : x;
                if (h < HEADS) {
                    const float top = finite_max(fmaxf(fmaxf(s_m[0][h], s_m[1][h]), fmaxf(s_m[2][h], s_m[3][h])));
                    f[x] = ex2(m[x] - top);
                } else f[x] = 0.f;
            }
#pragma unroll
            for (int r = 0; r < LIVE; ++r) {
                const float fr = f[BF ? (r >> 1) & 1 : (r / (BF ? 1 : HD / 32)) % NH];
                o[r] = fr == 0.f ? 0.f : o[r] * fr;
            }
        }
        // (bf16, up to eight heads: every second pair of sums belongs to the rows that no head has)
        auto live = [](int r) { return !(BF && GH == 8 && (r >> 1 & 1)); };
        auto packed = [](int r) { return BF && GH == 8 ? (r >> 2) * 2 + (r & 1) : r; };
        constexpr int SLAB = (BF && GH == 8 ? R / 2 : LIVE) * 32;
        auto hand = [&](float* to) {
#pragma unroll
            for (int r = 0; r < LIVE; ++r)
                if (live(r)) to[packed(r) * 32 + lane] = o[r];
        };
        auto take = [&](const float* from) {
#pragma unroll
            for (int r = 0; r < LIVE; ++r)
                if (live(r)) o[r] += from[packed(r) * 32 + lane];
        };
        if constexpr (2 * SLAB * 4 <= kDecMerge) {
            if (warp >= 2) hand(s_merge + (warp & 1) * SLAB);
            bar_consumers();
            if (warp < 2) take(s_merge + (warp & 1) * SLAB);
            bar_consumers();
            if (warp == 1) hand(s_merge);
            bar_consumers();
            if (warp == 0) take(s_merge);
        } else {
            for (int x = 1; x < kDecWarps; ++x) {
                if (warp == x) hand(s_merge);
                bar_consumers();
                if (warp == 0) take(s_merge);
                bar_consumers();
            }
        }

        const bool whole = w.t == 0 && n == w.nt;
        const int64_t orow = (int64_t)w.b * p.n_q + (int64_t)hkv * p.group + g0;
        // sums rfirst .. of this lane, times what `inv` holds: the reciprocals of the two rows' sums of weights (f32: of the heads')
        auto put = [&](const auto& v, int rfirst, auto nr, const auto& inv) {
            if constexpr (BF) {
#pragma unroll
                for (int j = 0; j < nr.value; j += 2) {
                    if (!live(j)) continue;
                    const int r = rfirst + j, x = (j >> 1) & 1, h = (lane >> 2) + 8 * x, d = (r >> 2) * 8 + (lane & 3) * 2;
                    if (h < G && d < p.head_dim)
                        *reinterpret_cast<uint32_t*>((T*)p.out + (orow + h) * p.head_dim + d) = bf16_pair(v[j] * inv[x], v[j + 1] * inv[x]);
                }
            } else {
                constexpr int VE = HD / 32;
#pragma unroll
                for (int j = 0; j < nr.value; j += VE) {
                    const int h = (rfirst + j) / VE, d = lane * VE;
                    if (h < G && d < p.head_dim) {
#pragma unroll
                        for (int e = 0; e < VE; ++e) ((float*)p.out)[(orow + h) * p.head_dim + d + e] = v[j + e] * inv[j / VE];
                    }
                }
            }
        };
        auto state_of = [&](int h, float* top) {     // the block's maximum and sum of a head
            *top = fmaxf(fmaxf(s_m[0][h], s_m[1][h]), fmaxf(s_m[2][h], s_m[3][h]));
            const float t = finite_max(*top);
            float sum = 0.f;
#pragma unroll
            for (int x = 0; x < kDecWarps; ++x) sum += s_l[x][h] == 0.f ? 0.f : s_l[x][h] * ex2(s_m[x][h] - t);
            return sum;
        };
        if (warp == 0) {
            float top = -INFINITY, sum = 0.f;             // lane h: of head h
            if (lane < HEADS) sum = state_of(lane, &top);
            if (whole) {
                const float i = sum == 0.f ? 0.f : 1.f / sum;
                float inv[NH];
#pragma unroll
                for (int x = 0; x < NH; ++x) inv[x] = __shfl_sync(0xffffffffu, i, BF ? (lane >> 2) + 8 * x : x);
                put(o, 0, std::integral_constant<int, LIVE>{}, inv);
            } else {
                float* slot = p.part + (2 * (int64_t)blockIdx.x + (w.t == 0 ? 1 : 0)) * SLOT;
#pragma unroll
                for (int r = 0; r < LIVE; ++r)
                    if (live(r)) slot[r * 32 + lane] = o[r];
                if (lane < HEADS) {
                    slot[R * 32 + kPagedGroup + lane] = sum;
                    slot[R * 32 + lane] = top;
                }
                __threadfence();
                __syncwarp();
            }
        }
        if (!whole) {
            // blocks of this pair: those of its first and last unit, and all between
            const int64_t f = unit0 - w.t, e = f + w.nt - 1;
            const int c0 = (int)(((f + 1) * blocks - 1) / total), c1 = (int)(((e + 1) * blocks - 1) / total);
            if (tid == 0) s_last = atomicAdd(&p.counters[c0], 1) == c1 - c0;
            bar_consumers();
            if (s_last) {
                __threadfence();
                if (tid == 0) p.counters[c0] = 0;
                // warp x joins a quarter of the sums of all parts, in the order of the blocks
                constexpr int Q = LIVE / kDecWarps > 0 ? LIVE / kDecWarps : 1;
                const int rf = warp * Q;
                if (rf < LIVE) {
                    float a[Q];
#pragma unroll
                    for (int j = 0; j < Q; ++j) a[j] = 0.f;
                    constexpr int NA = BF ? 2 : 1;        // heads among this lane's sums here
                    static_assert(BF || Q % (HD / 32) == 0 || (HD / 32) % Q == 0, "a lane's quarter");
#pragma unroll
                    for (int j0 = 0; j0 < Q; j0 += BF ? Q : (Q < HD / 32 ? Q : HD / 32)) {
                        constexpr int STEP = BF ? Q : (Q < HD / 32 ? Q : HD / 32);
                        float top[NA], sum[NA];
#pragma unroll
                        for (int x = 0; x < NA; ++x) {
                            const int h = BF ? (lane >> 2) + 8 * x : head_of(rf + j0);
                            top[x] = -INFINITY;
                            sum[x] = 0.f;
                            if (h >= HEADS) continue;
#pragma unroll 8
                            for (int c = c0; c <= c1; ++c)
                                top[x] = fmaxf(top[x], __ldcg(p.part + (2 * (int64_t)c + (c == c0 ? 1 : 0)) * SLOT + R * 32 + h));
                            top[x] = finite_max(top[x]);
                        }
#pragma unroll (BF && GH == 16 ? 2 : 4)
                        for (int c = c0; c <= c1; ++c) {
                            const float* slot = p.part + (2 * (int64_t)c + (c == c0 ? 1 : 0)) * SLOT;
                            float f2[NA];
#pragma unroll
                            for (int x = 0; x < NA; ++x) {
                                const int h = BF ? (lane >> 2) + 8 * x : head_of(rf + j0);
                                f2[x] = 0.f;
                                if (h >= HEADS) continue;
                                const float li = __ldcg(slot + R * 32 + kPagedGroup + h);
                                f2[x] = ex2(__ldcg(slot + R * 32 + h) - top[x]);
                                sum[x] += li == 0.f ? 0.f : li * f2[x];
                            }
                            float part[STEP];      // (all asked for before any is used)
#pragma unroll
                            for (int j = 0; j < STEP; ++j)
                                if (live(j)) part[j] = __ldcg(slot + (rf + j0 + j) * 32 + lane);
#pragma unroll
                            for (int j = 0; j < STEP; ++j) {
                                if (!live(j)) continue;
                                const float fr = f2[BF ? ((rf + j) >> 1) & 1 : 0];
                                a[j0 + j] = fr == 0.f ? a[j0 + j] : fmaf(part[j], fr, a[j0 + j]);
                            }
                        }
                        if constexpr (!BF) {
                            const float i = sum[0] == 0.f ? 0.f : 1.f / sum[0];
                            const int h = head_of(rf + j0), d = lane * (HD / 32) + (rf + j0) % (HD / 32);
                            if (h < G)
#pragma unroll
                                for (int j = 0; j < STEP; ++j)
                                    if (d + j < p.head_dim) ((float*)p.out)[(orow + h) * p.head_dim + d + j] = a[j0 + j] * i;
                        } else {
                            float inv[NA];
#pragma unroll
                            for (int x = 0; x < NA; ++x) inv[x] = sum[x] == 0.f ? 0.f : 1.f / sum[x];
                            put(a, rf, std::integral_constant<int, Q>{}, inv);
                        }
                    }
                }
            }
        }
        bar_consumers();       // s_m, s_l, s_merge, s_last are the next part's
        w.left -= n;
        if (w.left > 0) dec_next<TILE>(p, H, &w);
    }
    if (tid == 0 && s_abort) atomicExch(p.status, 2);
}

int32_t decode_configure(DeviceState& ds) {
    constexpr auto attr = cudaFuncAttributeMaxDynamicSharedMemorySize;
    auto set = [&](auto kernel) { return cudaFuncSetAttribute(kernel, attr, kDecSmem); };
    RSTQ_CUDA(set(paged_decode_kernel<__nv_bfloat16, 64, 8>));
    RSTQ_CUDA(set(paged_decode_kernel<__nv_bfloat16, 64, 16>));
    RSTQ_CUDA(set(paged_decode_kernel<__nv_bfloat16, 128, 8>));
    RSTQ_CUDA(set(paged_decode_kernel<__nv_bfloat16, 128, 16>));
    RSTQ_CUDA(set(paged_decode_kernel<float, 64, 1>));
    RSTQ_CUDA(set(paged_decode_kernel<float, 64, 4>));
    RSTQ_CUDA(set(paged_decode_kernel<float, 64, 8>));
    RSTQ_CUDA(set(paged_decode_kernel<float, 128, 1>));
    RSTQ_CUDA(set(paged_decode_kernel<float, 128, 4>));
    RSTQ_CUDA(set(paged_decode_kernel<float, 128, 8>));
    (void)ds;
    return RSTQ_OK;
}

// A pool (or packed rows) as [rows][n_kv][head_dim], read in boxes of 128 bytes x `box` rows of one head.
int32_t kv_tensor_map(CUtensorMap* m, const void* base, int32_t dtype, int64_t rows, int64_t ld, int n_kv, int head_dim, int box) {
    const EncodeTiledFn enc = encode_tiled_fn();
    RSTQ_REQUIRE(enc, RSTQ_E_CUDA, "cuTensorMapEncodeTiled is not available");
    const cuuint64_t es = (cuuint64_t)elem_bytes(dtype);
    const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)n_kv, (cuuint64_t)(rows > 0 ? rows : 1)};
    const cuuint64_t strides[2] = {head_dim * es, (cuuint64_t)ld * es};
    const cuuint32_t bx[3] = {(cuuint32_t)(128 / es), 1u, (cuuint32_t)box}, ones[3] = {1u, 1u, 1u};
    const CUresult r = enc(m, dtype == RSTQ_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void*>(base), dims,
                           strides, bx, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    RSTQ_REQUIRE(r == CUDA_SUCCESS, RSTQ_E_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return RSTQ_OK;
}

int32_t launch_paged_decode(DeviceState& ds, const PromptArgs& a) {
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
    int32_t rc = kv_tensor_map(&kmap, a.k, a.dtype, a.kv_rows, a.kv.ld, a.n_kv, a.head_dim, p.box);
    if (rc == RSTQ_OK) rc = kv_tensor_map(&vmap, a.v, a.dtype, a.kv_rows, a.kv.ld, a.n_kv, a.head_dim, p.box);
    if (rc != RSTQ_OK) return rc;
    const int64_t blocks = 2 * (int64_t)ds.sm_count;
    static_assert(2 * dec_slot<128>() >= 2 * dec_slot<64>(), "slots");
    RSTQ_REQUIRE(2 * blocks * dec_slot<128>() * 4 <= ds.partials_bytes && blocks <= ds.counters_len, RSTQ_E_LIMIT, "%lld thread blocks", (long long)blocks);
    const int g = std::min(a.group, per);
    auto go = [&](auto kernel) { return launch_pdl(kernel, dim3((unsigned)blocks), dim3(kDecThreads), kDecSmem, ds, p, kmap, vmap); };
    cudaError_t e;
    if (a.dtype == RSTQ_BF16) {
        if (a.head_dim <= 64) e = g <= 8 ? go(paged_decode_kernel<__nv_bfloat16, 64, 8>) : go(paged_decode_kernel<__nv_bfloat16, 64, 16>);
        else e = g <= 8 ? go(paged_decode_kernel<__nv_bfloat16, 128, 8>) : go(paged_decode_kernel<__nv_bfloat16, 128, 16>);
    } else if (a.head_dim <= 64) {
        e = g == 1 ? go(paged_decode_kernel<float, 64, 1>) : g <= 4 ? go(paged_decode_kernel<float, 64, 4>) : go(paged_decode_kernel<float, 64, 8>);
    } else {
        e = g == 1 ? go(paged_decode_kernel<float, 128, 1>) : g <= 4 ? go(paged_decode_kernel<float, 128, 4>) : go(paged_decode_kernel<float, 128, 8>);
    }
    RSTQ_CUDA(e);
    return RSTQ_OK;
}

}  // namespace rstq
