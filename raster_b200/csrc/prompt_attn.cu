// Causal attention of whole prompts, bf16, on the tcgen05 tensor cores.
//
//   out[i] = sum_j p_ij V[j] / sum_j p_ij,   p_ij = exp(scale q_i.K_j - m_i),   j <= i + (keys - rows) of its sequence
//
// A block of rows is two query tiles of 128 (row, head) pairs of one sequence: 256 rows of a head, or 128 / group rows per tile of all heads of
// a group, which then read K and V once, fill the tiles with few rows and see less beyond the diagonal (12 prompts of 28 heads over 4: 90 -> 77
// us; 20 rows each behind 200 caches 527 -> 92).  Its keys go by in tiles of 128:
//
//   S = Q K^T   (tcgen05, Q and K from shared memory, S in tensor memory)
//   P = exp2(scale2 S - m)   (a warpgroup per query tile, a thread per row: S from tensor memory, P back over it in bf16)
//   O += P V    (tcgen05, P from tensor memory, V from shared memory as it lies: an operand with head_dim innermost)
//
// While one tile's warpgroup is at its exponentials the tensor core works for the other tile.  The running maximum of a row moves
// only when it grows by more than 2^8 (a published refinement of the softmax taken in one pass), so O is read and written back for a few tiles at
// the start of a row and hardly ever after.  Weights are taken relative to 2^8 times it: none is more than 1.  (Sums are f32 and P's relative
// rounding does not depend on its size; the 2^8 leaves with the sum of the weights.)
// P is rounded to bf16, the type of V (2^-9 rms of each weight, no more than the result's own rounding); its sum is taken before that.
// P is handed to the tensor core in halves, as soon as each is written.
//
// K and V come by TMA through one ring, a box of 128 packed rows or one per page (the table is read a tile ahead).  Keys a row does not see
// get -inf before the maximum.  V's rows behind a sequence's end (another sequence's, a stale page's) are zeroed in shared memory before the
// product, for 0 * NaN is NaN; what lies above the diagonal cannot be zeroed, it belongs to other rows: a warp looks through those few tiles,
// and where it finds an infinity or NaN the block's rows are computed again one by one, from the positions they see alone (attend_row).
// So are those of a block whose table names no page.
//
// A thread block stays on its SM and takes the next block of rows, those with most keys of a sequence first, when its copies for this one are
// out (a counter): the next rows' Q, K and V are on their way during the last products.  Few blocks of rows that see many keys are cut
// into parts along the keys (prompt_share); a part leaves its sums, maximum and weight in a slot, and a second launch joins them in order, so
// that results do not depend on who was first.
//
// What it takes.  A step (256 rows, 128 keys, head_dim 128) takes 1.9 us, of which the MMAs are 1.05 at the tensor core's own pace (1.5 at the rate
// that a large matrix product reaches on the device) and the exponentials, on the SM's 16 special-function lanes, as much: the chain S, maximum,
// exponentials, P V, next S of each tile does not close any tighter in 512 columns of tensor memory, two places for S per tile would need 768
// (of 64 columns 640; there a third one for both tiles would fit).  8192 rows, 32 heads over 8: 442 us, 1245 TFLOP/s (515 in a row, at the power
// limit: 1070); 4096 rows 127 us; 8192 of 64 columns 400 us.  Beside the steps a block of rows costs 2.6 us, mostly its stores, and a launch 5 to
// 7 us until the first S.  512 rows behind 16000 keys 162 us (in parts; 255 with one query tile per block), 2 rows 33 us.
// A polynomial in place of a part of the exponentials was slower, so were 64 keys per tile with two places for S.
#include <algorithm>
#include <type_traits>

#include "prompt.cuh"

namespace rstq {

constexpr int kPrThreads = 384;      // two warpgroups of softmax; copies, MMAs, V's edges
constexpr int kPrRows = 128;         // rows of a query tile, keys of a tile
// Tiles of keys whose P V stays in tensor memory.  Its additions cut off, towards zero, so after as many O goes to a slot in memory, where it is added
// to the rows' sums in f32, and starts anew: 2^20 keys lost 7e-3 of a result, 2^18 1.3e-3; now 1e-4.
constexpr int kPromptFold = 256;
template <int HD>
struct PromptShape {
    // (of 256 columns one query tile: K and V of a step and Q take 192 KB, S and O 384 columns of tensor memory)
    static constexpr int blks = HD / 64, tile = kPrRows * HD * 2, stages = HD == 256 ? 2 : HD == 128 ? 5 : 8, queries = HD == 256 ? 1 : 2;
    static constexpr int smem = 1024 + (queries + stages) * tile;
};

struct PromptParams {
    PromptArgs a;
    int tiles;                       // query tiles of a block: 1 or 2
    int pack, rpt;                   // heads of a group that share a tile (1: none), rows of q of a tile: its rows are (row of q, head), the head innermost
    int heads;                       // items per block of rows: n_kv, or n_q without packing
    int bound;                       // items there are at most
    int sms;                         // blocks of threads that take the items of a call whose blocks' keys may be cut into parts
    int box;                         // rows of a box of keys
    int sectors;                     // the rows of out begin on 32-byte boundaries, and so do their pieces of 16 columns
    float scale2;
    int* status;
    PromptJoin join;                 // where the parts of a block's keys go
    int* counters;                   // [0] items dealt out beyond the first of every block, [1] blocks that are done: zero between launches
};
// what a warp has to know of a block of rows
struct PromptWork {
    PromptItem it;
    int h;                           // query head, or the packed ones' KV head
    int item;
};
// 16 columns of a row, and g times (`there`) what a slot of R rows has of them; `back`: to the slot.
template <int R>
__device__ __forceinline__ void add_slot(uint32_t (&o)[16], float* slot, bool there, float g, bool back) {
#pragma unroll
    for (int u = 0; u < 16; u += 4) {
        float* at = slot + u * R;
        float4 v = make_float4(__uint_as_float(o[u]), __uint_as_float(o[u + 1]), __uint_as_float(o[u + 2]), __uint_as_float(o[u + 3]));
        if (there) {
            const float4 x = load4(at);
            v = make_float4(fmaf(x.x, g, v.x), fmaf(x.y, g, v.y), fmaf(x.z, g, v.z), fmaf(x.w, g, v.w));
        }
        o[u] = __float_as_uint(v.x);
        o[u + 1] = __float_as_uint(v.y);
        o[u + 2] = __float_as_uint(v.z);
        o[u + 3] = __float_as_uint(v.w);
        if (back) store4(at, v);
    }
}
// PARTS: a block's keys may be cut into parts.  LONG: they may be more than kPromptFold tiles.  (Calls that cannot have as many do without: 12 ragged
// prompts 79 us, and 82 with it; 512 rows behind 16000 keys 163 and 167; of 64 columns it makes no difference for the worse.)
template <int HD, bool PARTS, bool LONG>
__global__ void __launch_bounds__(kPrThreads, 1)
prompt_kernel(const PromptParams p, const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
              const __grid_constant__ CUtensorMap vmap) {
    using Sh = PromptShape<HD>;
    constexpr int NST = Sh::stages, TILE = Sh::tile, BLK = kPrRows * 128, R = Sh::queries * kPrRows;     // BLK: 64 columns of a tile; R: rows of a slot
    extern __shared__ uint8_t s_raw0[];
    uint8_t* s_raw = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(s_raw0) + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t s_bar[2 * NST + 19];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort[2];       // somebody gave up; rows taken again one by one, for which others may have to wait long
    __shared__ volatile int s_again[2];
    __shared__ PromptWork s_work[2];
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;      // (the same in all lanes, for the compiler too)
    const uint32_t sq = smem_u32(s_raw), ring = sq + Sh::queries * TILE;
    // full / empty: a stage of the ring (empty: by the MMAs that read it and by the warp at V's edges); qfull / qempty; sfull[t]: S of a
    // tile is there; phalf[t], pfull[t]: half of P is, all of it, and O has its scale; odone[t]: P V is added; vfix[2]: the last V's edge is
    // zeroed; fixed[2]: no V of these rows will be looked at any more; wfull[2] / wempty[2]: what to work on (all six by the number of the block
    // of rows: a warp may be one ahead of another, never two); over: all products are done, after a wait ran out
    const uint32_t full = smem_u32(s_bar), empty = full + 8 * NST, qfull = empty + 8 * NST, qempty = qfull + 8, sfull = qempty + 8,
                   phalf = sfull + 16, pfull = phalf + 16, odone = pfull + 16, vfix = odone + 16, fixed = vfix + 16, wfull = fixed + 16,
                   wempty = wfull + 16, over = wempty + 16;
    volatile int* abort_flag = s_abort;
    if (tid == 0) {
        s_abort[0] = s_abort[1] = 0;
        for (int i = 0; i < NST; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 2);
        }
        mbar_init(qfull, 1);
        mbar_init(qempty, 1);
        for (int t = 0; t < 2; ++t) {
            mbar_init(sfull + 8 * t, 1);
            mbar_init(phalf + 8 * t, 4);
            mbar_init(pfull + 8 * t, 4);
            mbar_init(odone + 8 * t, 1);
            mbar_init(wfull + 8 * t, 1);
            mbar_init(wempty + 8 * t, 10);
            mbar_init(vfix + 8 * t, 1);
            mbar_init(fixed + 8 * t, 1);
        }
        mbar_init(over, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    for (int e = p.rpt * p.pack * 8 + tid; e < kPrRows * 8; e += kPrThreads)      // rows of Q's tiles that no copy fills
        for (int c = 0; c < Sh::queries * Sh::blks; ++c) sts128(sq + c * BLK + e * 16, 0u, 0u, 0u, 0u);
    fence_async_smem();
    if (warp == 9) {
        tmem_alloc(smem_u32(&s_tmem), 512);
        tmem_relinquish();
    }
    if (tid == 8 * 32) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&qmap)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&kmap)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&vmap)) : "memory");
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    PromptItem first;                // the block's first work, looked up while tensor memory is on its way
    first.rows = 0;
    const int per = p.tiles * p.rpt;                     // rows of q of a block
    int share = 1 << 30;
    if (warp == 8) {
        if (PARTS) {
            int items;
            share = prompt_share(p.a, per, kPrRows, p.heads, p.sms, 2, 3, &items);      // (a step 2 us)
            if (blockIdx.x == 0 && lane == 0) *p.join.listed = items;
        }
        first = PARTS ? prompt_item(p.a, per, kPrRows, share, blockIdx.x / p.heads) : prompt_block(p.a, per, kPrRows, blockIdx.x / p.heads);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = (uint32_t)uniform((int)s_tmem);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");     // (not before this block has its tensor memory)
    const uint32_t tS[2] = {tmem, tmem + 128}, tO[2] = {tmem + 256, tmem + 256 + HD};
    // keys that row r of a block sees, and the steps of a tile: tiles of keys, of the item's, that some row of it sees
    auto sees = [&](const PromptItem& it, int r) { return it.sees(r, p.a.causal); };
    auto steps_of = [&](const PromptItem& it, int t) {
        const int last = min(it.rows, (t + 1) * p.rpt) - 1;
        return uniform(t < p.tiles && last >= t * p.rpt ? max(min(it.j1, (sees(it, last) + kPrRows - 1) / kPrRows) - it.j0, 0) : 0);
    };
    bool ok = true;
    // The next block of rows, of which `w` is the number; false: there is none.
    auto next_work = [&](int w, PromptWork* x) {
        if (!wait_phase<true>(wfull + 8 * (w & 1), (w >> 1) & 1, abort_flag)) {
            ok = false;
            return false;
        }
        *x = s_work[w & 1];
        return uniform(x->it.rows) > 0;
    };
    auto done_work = [&](int w) {
        __syncwarp();
        if (lane == 0) mbar_arrive(wempty + 8 * (w & 1));
    };

    if (warp < 8) {
        // ---- softmax: a thread per row ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int t = warp >> 2;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, tSt = tS[0] + t * 128 + lanes, tOt = tO[0] + t * HD + lanes;
        const int rt = (warp & 3) * 32 + lane, slot_row = t * kPrRows + rt, r = t * p.rpt + rt / p.pack, mine_of = rt % p.pack;      // row of the block, head
        uint32_t c = 0;                      // steps of this tile so far (their parity is that of its barriers)
        PromptWork x;
        for (int w = 0; ok && next_work(w, &x); ++w) {
            const PromptItem& it = x.it;
            const int steps = steps_of(it, t);
            // keys of this row, of the tile's first, from the item's first on
            const int mine = sees(it, r) - it.j0 * kPrRows, least = sees(it, t * p.rpt) - it.j0 * kPrRows;
            float m = -INFINITY, m2 = 0.f, sum = 0.f;      // running maximum of S; scale2 times it (0: nothing seen yet)
            auto slot_of = [&]() { return p.join.part + (int64_t)(PARTS ? x.item : (int)blockIdx.x) * prompt_slot<HD>(); };
            float ref = -INFINITY;                         // what the sums in the slot refer to, as m2 (-inf: nothing)
            for (int j = 0; j < steps; ++j) {
                ok = wait_phase<true>(sfull + 8 * t, (c + j) & 1, abort_flag);
                if (!ok) break;
                tc_fence_after();
                uint32_t s[128];
#pragma unroll
                for (int i = 0; i < 128; i += 32) tmem_ld32_wait(tSt + i, s + i);
                if ((j + 1) * kPrRows > least) {           // some row of the tile does not see all of these keys
                    const int lim = mine - j * kPrRows;
#pragma unroll
                    for (int i = 0; i < 128; ++i) s[i] = i < lim ? s[i] : 0xFF800000u;
                }
                float top[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) top[i] = fmaxf(__uint_as_float(s[i]), __uint_as_float(s[i + 4]));
#pragma unroll
                for (int i = 8; i < 128; i += 8)
#pragma unroll
                    for (int u = 0; u < 4; ++u) top[u] = fmaxf(fmaxf(top[u], __uint_as_float(s[i + u])), __uint_as_float(s[i + 4 + u]));
                const float rowmax = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                const bool grown = rowmax > m && !(rowmax * p.scale2 <= m2 + kGrow && m != -INFINITY);
                if (__any_sync(0xffffffffu, grown) || (LONG && j % kPromptFold == 0)) {
                    float f = 1.f;
                    if (grown) {
                        const float next = rowmax * p.scale2;
                        f = m == -INFINITY ? 0.f : ex2f(m2 - next);
                        m = rowmax;
                        m2 = next;
                        sum *= f;
                    }
                    if (j > 0) {      // (S of this step came after the P V of the last but one)
                        ok = wait_phase<true>(odone + 8 * t, (c + j - 1) & 1, abort_flag);
                        if (!ok) break;
                        tc_fence_after();
                        const bool taken = LONG && j % kPromptFold == 0;
                        const float g = j > kPromptFold ? ex2f(ref - m2) : 0.f;
#pragma unroll 1
                        for (int i = 0; i < HD; i += 16) {
                            uint32_t o[16];
                            tmem_ld16_wait(tOt + i, o);
#pragma unroll
                            for (int u = 0; u < 16; ++u) o[u] = __float_as_uint(__uint_as_float(o[u]) * f);
                            if (taken) add_slot<R>(o, slot_of() + (i / 4 * R + slot_row) * 4, j > kPromptFold, g, true);
                            else tmem_st16(tOt + i, o);
                        }
                        if (taken) ref = m == -INFINITY ? m : m2;
                    }
                }
                // (2^-8 in every weight, so that none is more than 1 and a large value stays one)
                const float below = -m2 - kGrow;
                const uint64_t scale = pack2(p.scale2, p.scale2), minus = pack2(below, below);
                uint64_t part[2] = {0ull, 0ull};
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    uint32_t v[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float a, b;
                        unpack2(fma2(pack2(__uint_as_float(s[32 * g + 2 * i]), __uint_as_float(s[32 * g + 2 * i + 1])), scale, minus), a, b);
                        a = ex2f(a);
                        b = ex2f(b);
                        part[i & 1] = add2(part[i & 1], pack2(a, b));
                        v[i] = bf16_pair(a, b);
                    }
                    tmem_st16(tSt + 16 * g, v);
                    if (g & 1) {
                        tmem_st_wait();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive((g == 3 ? pfull : phalf) + 8 * t);
                    }
                }
                float a, b;
                unpack2(add2(part[0], part[1]), a, b);
                sum += a + b;
            }
            // ---- the rows' results ----
            c += steps;
            if (ok) ok = wait_phase<true>(fixed + 8 * (w & 1), (w >> 1) & 1, abort_flag);
            if (steps > 0 && ok) ok = wait_phase<true>(odone + 8 * t, (c - 1) & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            const bool has_row = t < p.tiles && rt < p.rpt * p.pack && r < it.rows;
            __nv_bfloat16* out = (__nv_bfloat16*)p.a.out + ((it.row + r) * p.a.n_q + x.h * p.pack + mine_of) * p.a.head_dim;
            const bool again = s_again[w & 1] != 0;
            // (a part of a block's keys: what it has found goes to its slot, for prompt_join_kernel)
            const bool whole = !PARTS || it.parts == 1;
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            if (LONG && steps > kPromptFold) {      // what is in the slot back to O
                const float g = ex2f(ref - m2);
#pragma unroll 1
                for (int i = 0; i < HD; i += 16) {
                    uint32_t o[16];
                    tmem_ld16_wait(tOt + i, o);
                    add_slot<R>(o, slot_of() + (i / 4 * R + slot_row) * 4, true, g, false);
                    tmem_st16(tOt + i, o);
                }
                tmem_st_wait();
            }
            float* slot = slot_of();
            if (!whole || !again)
#pragma unroll
                for (int i = 0; i < HD; i += 32) {
                    uint32_t o[32];
                    if (steps > 0) tmem_ld32_wait(tOt + i, o);
                    if (has_row && whole) {
#pragma unroll
                        for (int u = 0; u < 32; u += 16) {
                            if (i + u >= p.a.head_dim) continue;
                            uint32_t v[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                v[e] = sum == 0.f ? 0u : bf16_pair(__uint_as_float(o[u + 2 * e]) * inv, __uint_as_float(o[u + 2 * e + 1]) * inv);
                            if (p.sectors) st_sector(out + i + u, v);
                            else {
                                *reinterpret_cast<uint4*>(out + i + u) = make_uint4(v[0], v[1], v[2], v[3]);
                                if (i + u + 8 < p.a.head_dim) *reinterpret_cast<uint4*>(out + i + u + 8) = make_uint4(v[4], v[5], v[6], v[7]);
                            }
                        }
                    } else if (PARTS && has_row && steps > 0) {
#pragma unroll
                        for (int u = 0; u < 32; u += 4)
                            *reinterpret_cast<uint4*>(slot + ((i + u) / 4 * R + slot_row) * 4) = make_uint4(o[u], o[u + 1], o[u + 2], o[u + 3]);
                    }
                }
            if (PARTS && !whole) {
                if (has_row) {
                    slot[R * HD + slot_row] = m2;
                    slot[R * (HD + 1) + slot_row] = sum;      // (0: the columns say nothing)
                }
                if (tid == 0) slot[R * (HD + 2)] = again ? 1.f : 0.f;
            }
            tc_fence_before();       // O has been read before the next rows' P is handed on
            if (again && whole)
                for (int i = 0; i < p.pack; ++i) prompt_rows<__nv_bfloat16>(p.a, it, x.h * p.pack + i, warp, 8, s_abort + 1);
            done_work(w);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 8) {
            // ---- work dealt out; copies: Q, then K and V tile by tile ----
            const int boxes = kPrRows / p.box;
            int s = 0, item = blockIdx.x;
            uint32_t ph = 0, cq = 0;
            // The next item, asked for when the last copies of this one are on their way.  (Asked for with the item itself, the long ones'
            // blocks would take it from those that are done sooner: 2048 rows, 32 heads 48 -> 61 us.)
            auto claim = [&]() {
                first.rows = 0;
                if (p.bound <= (int)gridDim.x) return;
                if (lane == 0) item = atomicAdd(p.counters, 1) + (int)gridDim.x;
                item = __shfl_sync(0xffffffffu, item, 0);
                first = PARTS ? prompt_item(p.a, per, kPrRows, share, item / p.heads) : prompt_block(p.a, per, kPrRows, item / p.heads);
            };
            for (int w = 0;; ++w) {
                PromptWork x;
                x.it = first;
                x.h = item % p.heads;
                x.item = item;
                const PromptItem& it = x.it;
                ok = wait_phase<true>(wempty + 8 * (w & 1), ((w >> 1) & 1) ^ 1u, abort_flag);
                if (!ok) break;
                if (lane == 0) {
                    s_again[w & 1] = 0;
                    s_work[w & 1] = x;
                    mbar_arrive(wfull + 8 * (w & 1));
                }
                if (it.rows == 0) break;
                if (PARTS && lane == 0 && share < 1 << 30) p.join.list[item] = it;
                const int n = max(steps_of(it, 0), steps_of(it, 1)), hkv = p.pack > 1 ? x.h : x.h / p.a.group;
                // rows of a tile's boxes, a lane each (-1: behind the last key, -2: no page), looked up a tile ahead
                auto rows_at = [&](int j) {
                    const int pos = (it.j0 + j) * kPrRows + lane * p.box;
                    if (j >= n || lane >= boxes || pos >= it.keys) return -1;
                    const int row = (int)kv_row(p.a.kv, it.b, it.row0, pos);
                    return row < 0 ? -2 : row;
                };
                int ahead = rows_at(0);
                if (n > 0) {
                    ok = wait_phase<true>(qempty, (cq & 1) ^ 1u, abort_flag);
                    if (!ok) break;
                    ++cq;
                    if (lane == 0) {
                        mbar_expect_tx(qfull, (uint32_t)(p.tiles * p.rpt * p.pack * HD * 2));
                        for (int t = 0; t < p.tiles; ++t)
                            for (int c = 0; c < Sh::blks; ++c)
                                tma_load_4d(sq + t * TILE + c * BLK, &qmap, c * 64, p.pack > 1 ? 0 : x.h % p.a.group, hkv, (int)it.row + t * p.rpt, qfull);
                    }
                }
                for (int j = 0; j < n && ok; ++j) {
                    const int y = ahead;
                    ahead = rows_at(j + 1);
                    if (y == -2) s_again[w & 1] = 1;
                    __syncwarp();
                    const unsigned there = __ballot_sync(0xffffffffu, y >= 0);
                    const uint32_t bytes = (uint32_t)(__popc(there) * p.box * 128 * Sh::blks);
                    for (int kv = 0; kv < 2; ++kv) {
                        if (ok) ok = wait_phase<true>(empty + 8 * s, ph ^ 1u, abort_flag);
                        if (!ok) break;
                        const uint32_t bar = full + 8 * s, dst = ring + s * TILE;
                        if (lane == 0) {
                            if (bytes) mbar_expect_tx(bar, bytes);
                            else mbar_arrive(bar);
                        }
                        for (int g = 0; g < boxes; ++g) {
                            const int row = __shfl_sync(0xffffffffu, y, g);
                            if (lane == 0 && row >= 0)
                                for (int c = 0; c < Sh::blks; ++c) tma_load_3d(dst + c * BLK + g * p.box * 128, kv ? &vmap : &kmap, c * 64, hkv, row, bar);
                        }
                        if (++s == NST) { s = 0; ph ^= 1u; }
                    }
                }
                if (!ok) break;
                claim();
            }
            if (!ok) {      // copies under way are waited for (again with a limit)
                volatile int none = 0;
                if (cq) wait_phase(qfull, (cq - 1) & 1, const_cast<volatile int*>(&none));
                for (int i = 0; i < NST; ++i) wait_phase(full + 8 * i, ph ^ (i >= s ? 1u : 0u), const_cast<volatile int*>(&none));
            }
        } else if (warp == 9) {
            // ---- MMAs ----
            constexpr uint32_t id_s = idesc_bf16(128), id_o = idesc_bf16(HD) | (1u << 16);     // (bit 16: B with N innermost)
            const bool leader = elect_one();
            int s = 0;                                            // the ring's next stage
            uint32_t ph = 0, c[2] = {0, 0}, cq = 0;               // steps so far; blocks of rows with any
            auto wait = [&](uint32_t bar, uint32_t parity) {
                if (ok) ok = wait_phase<true>(bar, parity, abort_flag);
                tc_fence_after();
            };
            auto step = [&]() { if (++s == NST) { s = 0; ph ^= 1u; } };
            // low words of descriptors (in 16 bytes) and their high word; V's: the blocks of 64 columns apart
            const uint32_t hi = (uint32_t)(smem_desc_sw128(0) >> 32), lead = (uint32_t)smem_desc_sw128(0), lead_v = (uint32_t)smem_desc_rows(0, BLK);
            auto product_s = [&](int t, int stage) {
                if (!ok) return;
                const uint32_t a = lead + ((sq + t * TILE) >> 4), b = lead + ((ring + stage * TILE) >> 4);
#pragma unroll
                for (int k = 0; k < HD / 16; ++k) {
                    const uint32_t o = (k >> 2) * (BLK >> 4) + (k & 3) * 2;
                    if (leader) umma_ss(tS[t], a + o, b + o, hi, id_s, k > 0);
                }
                umma_commit_if(sfull + 8 * t, leader);
            };
            PromptWork x;
            for (int w = 0; ok && next_work(w, &x); ++w) {
                const int nt[2] = {steps_of(x.it, 0), steps_of(x.it, 1)}, n = max(nt[0], nt[1]);
                if (n > 0) {
                    wait(qfull, cq & 1);
                    wait(full + 8 * s, ph);
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        if (nt[t] > 0) product_s(t, s);
                    if (ok) umma_commit_if(empty + 8 * s, leader);
                    if (ok && n == 1) umma_commit_if(qempty, leader);
                    step();
                }
                for (int j = 0; j < n && ok; ++j) {
                    const int vs = s;
                    const uint32_t vph = ph;
                    step();
                    const int ks = s;
                    const uint32_t kph = ph;
                    if (j + 1 < n) step();
                    wait(full + 8 * vs, vph);
                    if (j == n - 1) wait(vfix + 8 * (w & 1), (w >> 1) & 1);
                    bool have_k = false;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (j < nt[t]) {
                            const uint32_t b = lead_v + ((ring + vs * TILE) >> 4);
#pragma unroll
                            for (int half = 0; half < 2; ++half) {       // P's first half is there sooner
                                wait((half ? pfull : phalf) + 8 * t, (c[t] + j) & 1);
                                if (!ok) break;
#pragma unroll
                                for (int k = half * 4; k < half * 4 + 4; ++k) if (leader) umma_ts(tO[t], tS[t] + k * 8, b + k * (2048 >> 4), hi, id_o, (LONG ? j % kPromptFold : j) > 0 || k > 0);
                            }
                            if (ok) umma_commit_if(odone + 8 * t, leader);
                        }
                        if (t == 1 && ok) umma_commit_if(empty + 8 * vs, leader);
                        if (j + 1 < nt[t]) {
                            if (!have_k) wait(full + 8 * ks, kph);
                            have_k = true;
                            product_s(t, ks);
                        }
                        if (t == 1 && j + 1 < n && ok) umma_commit_if(empty + 8 * ks, leader);
                    }
                    if (ok && j + 2 == n) umma_commit_if(qempty, leader);      // Q's last product is issued
                }
                c[0] += nt[0];
                c[1] += nt[1];
                cq += n > 0;
                done_work(w);
            }
            if (!ok) {      // products under way are waited for (with a limit) before the memory they use is given up
                volatile int none = 0;
                umma_commit_if(over, leader);
                wait_phase(over, 0, const_cast<volatile int*>(&none));
            }
        } else if (warp == 10) {
            // ---- V's edges ----
            int s = 0;
            uint32_t ph = 0;
            PromptWork x;
            for (int w = 0; ok && next_work(w, &x); ++w) {
                const PromptItem& it = x.it;
                const int n = max(steps_of(it, 0), steps_of(it, 1)), base = it.j0 * kPrRows, seen_by_all = sees(it, 0) - base;
                for (int i = 0; i < 2 * n; ++i) {
                    ok = wait_phase<true>(full + 8 * s, ph, abort_flag);
                    if (!ok) break;
                    if (i & 1) {
                        const int j = i >> 1;
                        const uint32_t v = ring + s * TILE;
                        const int end = min(it.keys - base - j * kPrRows, kPrRows);
                        for (int e = end * 8 * Sh::blks + lane; e < kPrRows * 8 * Sh::blks; e += 32) {     // behind the last key: zeros
                            const int row = e / (8 * Sh::blks), c = e - row * (8 * Sh::blks);
                            sts128(v + (c >> 3) * BLK + row * 128 + ((c & 7) << 4), 0u, 0u, 0u, 0u);
                        }
                        if (j == n - 1) {
                            fence_async_smem();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(vfix + 8 * (w & 1));
                        }
                        // keys that some rows see and some do not
                        const int from = max(seen_by_all - j * kPrRows, 0);
                        uint32_t found = 0;
                        if (from < end) {
#pragma unroll 8
                            for (int e = from * 8 * Sh::blks + lane; e < end * 8 * Sh::blks; e += 32) {
                                const int row = e / (8 * Sh::blks), c = e - row * (8 * Sh::blks);
                                uint32_t y[4];
                                asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(y[0]), "=r"(y[1]), "=r"(y[2]), "=r"(y[3]) : "r"(v + (c >> 3) * BLK + row * 128 + ((c & 7) << 4)));
#pragma unroll
                                for (int u = 0; u < 4; ++u) found |= ((y[u] & 0x7FFF7FFFu) + 0x00800080u) & 0x80008000u;   // exponent of ones
                            }
                        }
                        if (found) s_again[w & 1] = 1;
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(empty + 8 * s);
                    if (++s == NST) { s = 0; ph ^= 1u; }
                }
                if (!ok) break;
                if (lane == 0) {
                    if (n == 0) mbar_arrive(vfix + 8 * (w & 1));
                    mbar_arrive(fixed + 8 * (w & 1));
                }
                done_work(w);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) tmem_dealloc(tmem, 512);
    if (tid == 0) {
        if (s_abort[0]) atomicExch(p.status, 2);
        if (atomicAdd(p.counters + 1, 1) == (int)gridDim.x - 1) p.counters[0] = p.counters[1] = 0;      // the last block: for the next launch
    }
}

// The parts of a block joined, in their order: blocks of threads per item, a slice of the columns each, of which those of the first part do it.
constexpr int kJoinSlices = 8;
// R: rows of a block.
template <typename T, int HD, int R>
__global__ void __launch_bounds__(256, 3)
prompt_join_kernel(const PromptJoin p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int SLOT = prompt_slot<HD>();
    const int tid = threadIdx.x, all = *p.listed * kJoinSlices;
    for (int job = blockIdx.x; job < all; job += gridDim.x) {
    const int item = job / kJoinSlices, slice = job - item * kJoinSlices;
    const PromptItem it = p.list[item];
    if (it.parts == 1 || it.part != 0) continue;
    const int h = item % p.heads;
    const float* from = p.part + (int64_t)item * SLOT;
    const int64_t step = (int64_t)p.heads * SLOT;
    bool again = false;
#pragma unroll
    for (int q = 0; q < kMaxParts; ++q) again |= __ldcg(from + min(q, it.parts - 1) * step + R * (HD + 2)) != 0.f;
    if (again) {
        if (slice == 0)
            for (int i = 0; i < p.pack; ++i) prompt_rows<T>(p.a, it, h * p.pack + i, tid >> 5, 8);
        continue;
    }
    // eight columns of a row per thread: rows side by side
    const int rows = it.rows * p.pack, pieces = p.a.head_dim / 8, mine = (pieces - slice + kJoinSlices - 1) / kJoinSlices;
    for (int e = tid; e < rows * mine; e += 256) {
        const int x = e / rows, y = e - x * rows, i = x * kJoinSlices + slice, row = y / p.pack, t = row / p.rpt;
        const int r = t * (128 - p.rpt * p.pack) + y;      // (the tile's rows that hold none left out)
        float top = -INFINITY, total = 0.f, a[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int q0 = 0; q0 < it.parts; q0 += 4) {
            // (a load of a part that is not there is one of the last part's, with a weight of 0: loads behind a branch would wait for one another)
            float4 u[4], v[4];
            float f[4], s[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float* x = from + min(q0 + q, it.parts - 1) * step;
                s[q] = __ldcg(x + R * (HD + 1) + r);
                f[q] = __ldcg(x + R * HD + r);
                u[q] = __ldcg(reinterpret_cast<const float4*>(x) + 2 * i * R + r);
                v[q] = __ldcg(reinterpret_cast<const float4*>(x) + (2 * i + 1) * R + r);
            }
            float next = top;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (q0 + q >= it.parts) s[q] = 0.f;
                f[q] = s[q] != 0.f ? f[q] : -INFINITY;
                next = fmaxf(next, f[q]);
            }
            const float ref = next == -INFINITY ? 0.f : next, g = ex2f(top - ref);
            top = next;
            total *= g;
#pragma unroll
            for (int x = 0; x < 8; ++x) a[x] *= g;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (s[q] == 0.f) continue;      // (not where the weight is: 0 times what is no number is none either)
                const float w = ex2f(f[q] - ref);
                total = fmaf(w, s[q], total);
                a[0] = fmaf(w, u[q].x, a[0]); a[1] = fmaf(w, u[q].y, a[1]); a[2] = fmaf(w, u[q].z, a[2]); a[3] = fmaf(w, u[q].w, a[3]);
                a[4] = fmaf(w, v[q].x, a[4]); a[5] = fmaf(w, v[q].y, a[5]); a[6] = fmaf(w, v[q].z, a[6]); a[7] = fmaf(w, v[q].w, a[7]);
            }
        }
        const float inv = total == 0.f ? 0.f : 1.f / total;
        T* out = (T*)p.a.out + ((it.row + row) * p.a.n_q + h * p.pack + y - row * p.pack) * p.a.head_dim + 8 * i;
        if constexpr (sizeof(T) == 2)
            *reinterpret_cast<uint4*>(out) = make_uint4(bf16_pair(a[0] * inv, a[1] * inv), bf16_pair(a[2] * inv, a[3] * inv), bf16_pair(a[4] * inv, a[5] * inv),
                                                        bf16_pair(a[6] * inv, a[7] * inv));
        else {
            store4(out, make_float4(a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv));
            store4(out + 4, make_float4(a[4] * inv, a[5] * inv, a[6] * inv, a[7] * inv));
        }
    }
    }
}

PromptJoin prompt_join(DeviceState& ds, const PromptArgs& a, int pack, int rpt, int heads) {
    PromptJoin j;
    j.a = a;
    j.pack = pack;
    j.rpt = rpt;
    j.heads = heads;
    j.part = ds.prompt_slots;
    j.list = (PromptItem*)(ds.prompt_slots + (int64_t)kPromptSlots * prompt_slot<128>());
    j.listed = (int*)(j.list + kPromptSlots);
    return j;
}
int32_t launch_prompt_join(DeviceState& ds, const PromptJoin& j) {
    const dim3 grid((unsigned)(12 * ds.sm_count));
    auto go = [&](auto kernel) { return launch_pdl(kernel, grid, dim3(256), 0, ds, j); };
    using B = __nv_bfloat16;
    if (j.a.dtype == RSTQ_BF16)
        RSTQ_CUDA(j.a.head_dim <= 64    ? go(prompt_join_kernel<B, 64, 256>)
                  : j.a.head_dim <= 128 ? go(prompt_join_kernel<B, 128, 256>)
                                        : go(prompt_join_kernel<B, 256, 128>));
    else RSTQ_CUDA(j.a.head_dim <= 64 ? go(prompt_join_kernel<float, 64, 128>) : go(prompt_join_kernel<float, 128, 128>));
    return RSTQ_OK;
}

int32_t prompt_configure(DeviceState& ds) {
    constexpr auto attr = cudaFuncAttributeMaxDynamicSharedMemorySize;
    auto set = [&](auto hd) {
        constexpr int HD = decltype(hd)::value, smem = PromptShape<HD>::smem;
        cudaError_t e = cudaFuncSetAttribute((prompt_kernel<HD, false, false>), attr, smem);
        if (e == cudaSuccess) e = cudaFuncSetAttribute((prompt_kernel<HD, false, true>), attr, smem);
        if (e == cudaSuccess) e = cudaFuncSetAttribute((prompt_kernel<HD, true, false>), attr, smem);
        return e == cudaSuccess ? cudaFuncSetAttribute((prompt_kernel<HD, true, true>), attr, smem) : e;
    };
    RSTQ_CUDA(set(std::integral_constant<int, 64>()));
    RSTQ_CUDA(set(std::integral_constant<int, 128>()));
    RSTQ_CUDA(set(std::integral_constant<int, 256>()));
    const size_t slots = (size_t)kPromptSlots * (prompt_slot<128>() * 4 + sizeof(PromptItem));
    RSTQ_CUDA(cudaMalloc((void**)&ds.prompt_slots, slots + 64));
    RSTQ_CUDA(cudaMemsetAsync((char*)ds.prompt_slots + slots, 0, 64, ds.stream));
    return RSTQ_OK;
}

// q as [rows][n_kv][group][head_dim], in boxes of a tile's rows
static int32_t prompt_q_map(CUtensorMap* m, const PromptArgs& a, int heads, int rows) {
    const EncodeTiledFn enc = encode_tiled_fn();
    RSTQ_REQUIRE(enc, RSTQ_E_CUDA, "cuTensorMapEncodeTiled is not available");
    const cuuint64_t dims[4] = {(cuuint64_t)a.head_dim, (cuuint64_t)a.group, (cuuint64_t)a.n_kv, (cuuint64_t)a.rows};
    const cuuint64_t strides[3] = {(cuuint64_t)a.head_dim * 2, (cuuint64_t)a.group * a.head_dim * 2, (cuuint64_t)a.ldq * 2};
    const cuuint32_t box[4] = {64u, (cuuint32_t)heads, 1u, (cuuint32_t)rows}, ones[4] = {1u, 1u, 1u, 1u};
    const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(a.q), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    RSTQ_REQUIRE(r == CUDA_SUCCESS, RSTQ_E_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return RSTQ_OK;
}

int32_t launch_prompt(DeviceState& ds, const PromptArgs& a, int* launches) {
    PromptParams p;
    p.a = a;
    p.scale2 = a.scale * 1.4426950408889634f;
    p.status = ds.status;
    p.sectors = ((uintptr_t)a.out & 31) == 0 && a.head_dim % 16 == 0;
    p.box = a.kv.table ? std::min(1 << a.kv.shift, kPrRows) : kPrRows;
    p.pack = prompt_pack(a.group);
    p.rpt = kPrRows / p.pack;
    p.heads = a.n_q / p.pack;
    // Two query tiles per block keep the tensor core busy; with fewer blocks than SMs one each does the rows sooner.
    p.tiles = a.head_dim > 128 || a.rows * a.n_q <= kPrRows * (int64_t)ds.sm_count ? 1 : 2;
    // Few blocks of rows that may see many keys are cut into parts, which a second launch joins.  (A sequence's rows of more than a tile then
    // take two as well: there is no lack of parts.)
    const int64_t some = std::min<int64_t>(a.seqs, a.rows);
    const int tiles = a.head_dim <= 128 && a.rows > p.rpt * some ? 2 : 1;
    const bool parts = prompt_may_part(a, 1024) && (a.rows / (tiles * p.rpt) + some) * p.heads <= ds.sm_count;
    if (parts) p.tiles = tiles;
    const int per = p.tiles * p.rpt;
    const int64_t blocks = (a.rows / per + some) * p.heads;     // no sequence has more than this of them
    RSTQ_REQUIRE(blocks < (1ll << 31), RSTQ_E_LIMIT, "%lld thread blocks", (long long)blocks);
    p.sms = prompt_sms(ds);
    p.bound = parts ? 1 << 30 : (int)blocks;
    p.join = prompt_join(ds, a, p.pack, p.rpt, p.heads);
    CUtensorMap qmap, kmap, vmap;
    int32_t rc = prompt_q_map(&qmap, a, p.pack, p.rpt);
    if (rc == RSTQ_OK) rc = rows_tensor_map(&kmap, a.k, a.dtype, a.kv_rows, a.kv.ld, a.n_kv, a.head_dim, p.box);
    if (rc == RSTQ_OK) rc = rows_tensor_map(&vmap, a.v, a.dtype, a.kv_rows, a.kv.ld, a.n_kv, a.head_dim, p.box);
    if (rc != RSTQ_OK) return rc;
    p.counters = p.join.listed + 4;
    *launches = parts ? 2 : 1;
    if (!parts && a.seqs > kSumSeqs) {
        if ((rc = launch_sums(ds, a, per, 0)) != RSTQ_OK) return rc;
        p.a.start = ds.seq_starts;
        ++*launches;
    }
    const dim3 grid((unsigned)(parts ? p.sms : std::min<int64_t>(blocks, std::min(ds.sm_count, kPromptSlots))));
    const bool many = (a.kv.table ? (int64_t)a.kv.width << a.kv.shift : a.kv_rows) > kPromptFold * kPrRows;
    auto go = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        auto run = [&](auto kernel) { return launch_pdl(kernel, grid, dim3(kPrThreads), (size_t)PromptShape<HD>::smem, ds, p, qmap, kmap, vmap); };
        if (parts) return many ? run(prompt_kernel<HD, true, true>) : run(prompt_kernel<HD, true, false>);
        return many ? run(prompt_kernel<HD, false, true>) : run(prompt_kernel<HD, false, false>);
    };
    const cudaError_t e = a.head_dim <= 64 ? go(std::integral_constant<int, 64>()) : a.head_dim <= 128 ? go(std::integral_constant<int, 128>())
                                                                                                     : go(std::integral_constant<int, 256>());
    RSTQ_CUDA(e);
    return parts ? launch_prompt_join(ds, p.join) : RSTQ_OK;
}

}  // namespace rstq
