// What the kernels of prompt attention share: tensor memory in rows, operands as rows lie, the block's part of the work.
#pragma once
#include "paged.cuh"
#include "sync_helpers.cuh"
#include "tcgen05_helpers.cuh"

namespace rstq {

// ---- keys cut into parts ----
// What a part of a block of rows has found goes to its slot; a second launch joins the parts in their order.  (prompt_attn.cu)
struct PromptItem;
struct PromptJoin {
    PromptArgs a;
    int pack, rpt, heads;            // as the kernel that leaves the parts has them
    float* part;                     // a slot per item
    PromptItem* list;                // what each item was; their number, 0 where no block's keys are cut
    int* listed;
};
PromptJoin prompt_join(DeviceState& ds, const PromptArgs& a, int pack, int rpt, int heads);
int32_t launch_prompt_join(DeviceState& ds, const PromptJoin& j);
// A call's rows may see more than `most` keys: a cache, or more keys than rows.  Not of many sequences: every block of threads goes through their
// lengths a few times to share the work out (four of them with 4 rows behind 4000 keys, of 4 in all 39 us, of 256 53, of 1000 92, and 100
// without parts).
inline bool prompt_may_part(const PromptArgs& a, int most) {
    if (a.seqs > 1024) return false;
    const int64_t keys = a.kv.table ? (int64_t)a.kv.width << a.kv.shift : a.kv_rows > a.rows ? a.kv_rows : 0;
    return keys > most;
}

// Heads of a group that share a query tile of 128 rows, (row of q, head) with the head innermost: all of them where they fill seven eighths of it.
inline int prompt_pack(int group) { return 128 / group * group >= 112 ? group : 1; }

constexpr float kGrow = 8.f;         // bf16: log2 of how far a row's scores may go beyond the running maximum before it moves

// 32 columns of this thread's row, there when the instruction is over: what follows cannot be moved before the wait.
__device__ __forceinline__ void tmem_ld32_wait(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
        "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
          "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
          "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
// 16 columns of this thread's row, there when the instruction is over.
__device__ __forceinline__ void tmem_ld16_wait(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
// 32 bytes at once: a thread per row writes whole sectors, half the requests of 16 bytes each
__device__ __forceinline__ void st_sector(void* p, const uint32_t (&v)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
                 "r"(v[6]), "r"(v[7])
                 : "memory");
}
// pairs of f32 in one instruction
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// 16 (8) columns of this thread's row at two places, there when the instruction is over.
__device__ __forceinline__ void tmem_ld_x2_wait(uint32_t t0, uint32_t t1, uint32_t (&r)[16], uint32_t (&q)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];"
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]),
          "=r"(q[4]), "=r"(q[5]), "=r"(q[6]), "=r"(q[7]), "=r"(q[8]), "=r"(q[9]), "=r"(q[10]), "=r"(q[11]), "=r"(q[12]), "=r"(q[13]),
          "=r"(q[14]), "=r"(q[15])
        : "r"(t0), "r"(t1)
        : "memory");
}
__device__ __forceinline__ void tmem_ld_x2_wait(uint32_t t0, uint32_t t1, uint32_t (&r)[8], uint32_t (&q)[8]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%16];"
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%8,%9,%10,%11,%12,%13,%14,%15}, [%17];"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(q[0]), "=r"(q[1]), "=r"(q[2]),
          "=r"(q[3]), "=r"(q[4]), "=r"(q[5]), "=r"(q[6]), "=r"(q[7])
        : "r"(t0), "r"(t1)
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
                 "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
                 : "memory");
}
// A wait of a whole warp, in line (kernels that move registers between warps cannot call a function): true once the phase is
// complete, false after the limit or when another warp gave up.  BEAT: the word behind the flag changes while somebody is at work that takes
// longer than the limit allows; the limit then begins anew.
template <bool BEAT = false>
__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    unsigned long long t0 = 0;
    int seen = 0;
#pragma unroll 1
    for (uint32_t i = 1;; ++i) {
        if (__all_sync(0xffffffffu, mbar_try(bar, parity))) return true;
        if ((i & 255) == 0) {
            const unsigned long long now = gtime_ns();
            if (!t0) t0 = now;
            if (__any_sync(0xffffffffu, *abort_flag || now - t0 > kWaitLimitNs)) {
                const int is = BEAT ? __shfl_sync(0xffffffffu, abort_flag[1], 0) : 0;
                if (is == seen || *abort_flag) {
                    *abort_flag = 1;
                    return false;
                }
                seen = is;
                t0 = now;
            }
        }
    }
}
// One lane of the warp, the same one every time: what it does in a branch on this is known to be done once, so operands stay in uniform
// registers.
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(r));
    return r != 0;
}
// D[tmem] (+)= A * B, by the elected lane, from values that are the same in all lanes for the compiler too (a vote's or a reduction's result, not
// what was read from memory): an MMA is then issued in 13 cycles, else in 65 - 80, more than it takes.  Descriptors: low words, their
// common high word; A from shared or tensor memory.
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{ .reg .pred p; .reg .b64 a, b; setp.ne.b32 p, %5, 0; mov.b64 a, {%1, %3}; mov.b64 b, {%2, %3}; "
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p; }" ::"r"(d),
        "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{ .reg .pred p; .reg .b64 b; setp.ne.b32 p, %5, 0; mov.b64 b, {%2, %3}; "
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p; }" ::"r"(d),
        "r"(a_tmem), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ int uniform(int v) { return (int)__reduce_max_sync(0xffffffffu, v); }     // (the lanes' value is one already)
// V as it lies, [keys][head_dim] in blocks of 64 columns: an operand whose N is innermost.  128-byte swizzle; 64-column blocks
// `block` bytes apart, groups of eight keys 1024.
__device__ __forceinline__ uint64_t smem_desc_rows(uint32_t saddr, uint32_t block) {
    uint64_t d = smem_desc_sw128(saddr);
    d &= ~(0x3FFFull << 16);
    return d | (uint64_t)(block >> 4) << 16;
}
__device__ __forceinline__ float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// What a block works on: rows [row, row + rows) of the packed q, of sequence b, against tiles j0 .. j1 - 1 of its keys.
struct PromptItem {
    int b, rows;           // sequence, rows of it in this block (0: nothing left to do)
    int64_t row;           // the first one, packed
    int place;             // the first one's position in the sequence (below 0, or beyond its keys: it has none)
    int keys, row0;        // keys of the sequence; packed: the first one's row
    int j0, j1;            // tiles of keys
    int part, parts;       // which of how many parts of the block's keys
    // keys that row r of the block sees
    __device__ __forceinline__ int sees(int r, int causal) const {
        return causal ? min(max(place + 1 + r, 0), keys) : keys;
    }
};
constexpr int kMaxParts = 16, kPartRounds = 3;
inline int prompt_sms(const DeviceState& ds) { return ds.sm_count < kPromptSlots / kPartRounds ? ds.sm_count : kPromptSlots / kPartRounds; }
// One lane's sequence cut into blocks of `per` rows, and the tiles of `tile` keys that block k sees.
struct PromptSequence {
    int n, keys, end, row0, first, blocks;      // rows; keys; the position behind its last row; packed: first key; first row; blocks
    __device__ __forceinline__ void load(const PromptArgs& a, int b, int per) {
        n = keys = end = row0 = first = 0;
        if (b < a.seqs) {
            int64_t f, l, r;
            packed_range(a.cu_q, b, a.rows, &f, &l);
            keys = (int)kv_length(a.kv, b, &r);
            end = (int)min(kv_end(a.kv, b, keys), keys + kMaxRows);      // (farther, every row sees everything too)
            n = (int)(l - f);
            first = (int)f;
            row0 = (int)r;
        }
        blocks = (n + per - 1) / per;
    }
    __device__ __forceinline__ int tiles(int k, int per, int causal, int tile) const {
        const int last = min(n, (k + 1) * per) - 1, s = causal ? min(max(end - n + 1 + last, 0), keys) : keys;
        return (s + tile - 1) / tile;
    }
};
// parts of a block that sees w tiles, where a part should have about `share`
__device__ __forceinline__ int prompt_parts(int w, int share) { return w > share + (share >> 2) ? min((w + share - 1) / share, kMaxParts) : 1; }
__device__ __forceinline__ int prompt_count(const PromptSequence& q, int per, int causal, int tile, int share) {
    if (q.blocks == 0 || prompt_parts(q.tiles(q.blocks - 1, per, causal, tile), share) == 1) return q.blocks;     // (the last sees most)
    int c = 0;
    for (int k = 0; k < q.blocks; ++k) c += prompt_parts(q.tiles(k, per, causal, tile), share);
    return c;
}
// Items of all sequences with parts of about `share` tiles; more than `most`: that they are more.
static __device__ __forceinline__ int prompt_items(const PromptArgs& a, int per, int tile, int share, int most) {
    const int lane = threadIdx.x & 31;
    int items = 0;
    for (int b0 = 0; b0 < a.seqs && items <= most; b0 += 32) {
        PromptSequence q;
        q.load(a, b0 + lane, per);
        if (__any_sync(0xffffffffu, q.blocks > most)) return most + 1;
        items += __reduce_add_sync(0xffffffffu, prompt_count(q, per, a.causal, tile, share));
    }
    return items;
}
// How many tiles of keys a part should have; all (no parts, *total = 0) where that is sooner done.  `sms` blocks of threads take the items in
// rounds: for one, two and three of them the shortest parts that do not need another, and of these and of whole blocks what takes the
// fewest tiles one after the other.  item, join: what an item costs beside its tiles and what the joining launch does, in tiles.  Parts of
// fewer than four tiles are not made.  heads: items per block of rows.
static __device__ __forceinline__ int prompt_share(const PromptArgs& a, int per, int tile, int heads, int sms, int item, int join, int* total) {
    const int lane = threadIdx.x & 31;
    float all = 0.f;       // (sums of integers below 2^24, or large enough not to matter)
    int longest = 0, blocks = 0;
    for (int b0 = 0; b0 < a.seqs; b0 += 32) {
        PromptSequence q;
        q.load(a, b0 + lane, per);
        const int last = q.blocks ? q.tiles(q.blocks - 1, per, a.causal, tile) : 0;
        float w = q.blocks ? 0.5f * (float)q.blocks * (float)(q.tiles(0, per, a.causal, tile) + last) : 0.f;
#pragma unroll
        for (int d = 16; d; d >>= 1) w += __shfl_xor_sync(0xffffffffu, w, d);
        all += w;
        longest = max(longest, __reduce_max_sync(0xffffffffu, last));
        blocks = min(blocks + __reduce_add_sync(0xffffffffu, min(q.blocks, 1 << 20)), 1 << 25);
    }
    int best = 1 << 30, items = 0;
    int64_t cost = ((int64_t)blocks * heads + sms - 1) / sms * (longest + item);
    for (int rounds = 1; rounds <= kPartRounds; ++rounds) {
        const int most = rounds * sms / heads;
        int share = (int)fminf(fmaxf(ceilf(all * (float)heads / (float)(rounds * sms)), 4.f), 1e6f);
        for (int tries = 0; tries < 6; ++tries, share += (share >> 3) + 1) {
            const int64_t now = (int64_t)rounds * (share + item) + join;
            if (now >= cost) break;
            const int n = prompt_items(a, per, tile, share, most);
            if (n > most) continue;
            cost = now;
            best = share;
            items = n * heads;
            break;
        }
    }
    *total = items;
    return best;
}
// Block `item` of those of all sequences, `per` rows each, all of its keys; counted from the end, so that the blocks with most keys of a
// long sequence come first.  A warp's lanes work together and get the same answer.
static __device__ __forceinline__ PromptItem prompt_block(const PromptArgs& a, int per, int tile, int item) {
    const int lane = threadIdx.x & 31;
    PromptItem it;
    it.rows = 0;
    if (a.start) {
        const int64_t at = a.start[a.seqs] - 1 - item;
        if (at < 0) return it;
        const int b = find_start(a.start, a.seqs, at);
        PromptSequence q;
        q.load(a, b, per);
        const int k = (int)(at - a.start[b]);
        if ((int64_t)k * per >= q.n) return it;
        it.b = b;
        it.keys = q.keys;
        it.row = q.first + (int64_t)k * per;
        it.place = q.end - q.n + k * per;
        it.rows = min(q.n - k * per, per);
        it.row0 = q.row0;
        it.parts = 1;
        it.part = it.j0 = 0;
        it.j1 = q.tiles(k, per, a.causal, tile);
        return it;
    }
    for (int b0 = (a.seqs - 1) & ~31; b0 >= 0; b0 -= 32) {
        PromptSequence q;
        q.load(a, b0 + 31 - lane, per);
        int x = q.blocks;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += y;
        }
        const unsigned behind = __ballot_sync(0xffffffffu, x > item);
        if (!behind) {
            item -= __shfl_sync(0xffffffffu, x, 31);
            if (item < 0) return it;                       // (sequences that overlap beyond counting)
            continue;
        }
        const int src = __ffs((int)behind) - 1, k = __shfl_sync(0xffffffffu, x, src) - 1 - item;      // of the sequence, from its start
        q.n = __shfl_sync(0xffffffffu, q.n, src);
        if (k < 0 || (int64_t)k * per >= q.n) return it;
        it.keys = q.keys = __shfl_sync(0xffffffffu, q.keys, src);
        q.end = __shfl_sync(0xffffffffu, q.end, src);
        it.b = b0 + 31 - src;
        it.row = __shfl_sync(0xffffffffu, q.first, src) + (int64_t)k * per;
        it.place = q.end - q.n + k * per;
        it.rows = min(q.n - k * per, per);
        it.row0 = __shfl_sync(0xffffffffu, q.row0, src);
        it.parts = 1;
        it.part = it.j0 = 0;
        it.j1 = q.tiles(k, per, a.causal, tile);
        return it;
    }
    return it;
}
// Item `item` of those of all sequences: blocks of `per` rows, from the end of each sequence (those that see most keys first), in
// parts.  A warp's lanes work together and get the same answer.
static __device__ __forceinline__ PromptItem prompt_item(const PromptArgs& a, int per, int tile, int share, int item) {
    const int lane = threadIdx.x & 31;
    PromptItem it;
    it.rows = 0;
    for (int b0 = (a.seqs - 1) & ~31; b0 >= 0; b0 -= 32) {
        PromptSequence q;
        q.load(a, b0 + 31 - lane, per);
        const int m = prompt_count(q, per, a.causal, tile, share);
        int x = m;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += y;
        }
        const unsigned behind = __ballot_sync(0xffffffffu, x > item);
        if (!behind) {
            item -= __shfl_sync(0xffffffffu, x, 31);
            if (item < 0) return it;                       // (sequences that overlap beyond counting)
            continue;
        }
        const int src = __ffs((int)behind) - 1;
        int left = item - __shfl_sync(0xffffffffu, x - m, src);      // items of this sequence before it
        const int blocks = __shfl_sync(0xffffffffu, q.blocks, src);
        const bool whole = __shfl_sync(0xffffffffu, m, src) == blocks;
        q.n = __shfl_sync(0xffffffffu, q.n, src);
        q.keys = __shfl_sync(0xffffffffu, q.keys, src);
        q.end = __shfl_sync(0xffffffffu, q.end, src);
        int k = blocks - 1 - (whole ? left : 0), parts = 1;
        if (!whole)
            for (;; --k) {
                if (k < 0) return it;
                parts = prompt_parts(q.tiles(k, per, a.causal, tile), share);
                if (left < parts) break;
                left -= parts;
            }
        if (left < 0 || k < 0 || (int64_t)k * per >= q.n) return it;
        const int w = q.tiles(k, per, a.causal, tile);
        it.b = b0 + 31 - src;
        it.row = __shfl_sync(0xffffffffu, q.first, src) + (int64_t)k * per;
        it.place = q.end - q.n + k * per;
        it.rows = min(q.n - k * per, per);
        it.keys = q.keys;
        it.row0 = __shfl_sync(0xffffffffu, q.row0, src);
        it.parts = parts;
        it.part = whole ? 0 : left;
        it.j0 = (int)((int64_t)w * it.part / parts);
        it.j1 = (int)((int64_t)w * (it.part + 1) / parts);
        return it;
    }
    return it;
}

// The block's rows one by one, from the positions they see alone.
template <typename T>
__device__ __forceinline__ void prompt_rows(const PromptArgs& a, const PromptItem& it, int h, int warp, int warps, int* beat = nullptr) {     // (of one head)
    const int lane = threadIdx.x & 31;
    using S = RowState<T>;      // (f32: head_dim <= 128; one piece of a lane)
    bool bad = false;
    for (int r = warp; r < it.rows; r += warps) {
        S st;
        bad |= attend_row(a, it.b, it.row + r, h, it.sees(r, a.causal), 0, kRowPos, &st, beat);
        const float inv = st.l == 0.f ? 0.f : 1.f / st.l;
        if (lane * S::V < a.head_dim)
#pragma unroll
            for (int i = 0; i < S::V; i += 4)
                store4((T*)a.out + ((it.row + r) * a.n_q + h) * a.head_dim + lane * S::V + i,
                       make_float4(st.o[0][i] * inv, st.o[0][i + 1] * inv, st.o[0][i + 2] * inv, st.o[0][i + 3] * inv));
    }
    if (bad && lane == 0) a.kv.status[kStatusPage] = 1;
}

}  // namespace rstq
