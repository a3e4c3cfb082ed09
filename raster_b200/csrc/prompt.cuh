// What the kernels of prompt attention share: tensor memory in rows, operands as rows lie, the block's part of the work.
#pragma once
#include "paged.cuh"
#include "sync_helpers.cuh"
#include "tcgen05_helpers.cuh"

namespace rstq {

constexpr float kGrow = 8.f;         // log2 of how far a row's largest weight may go beyond 1

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
        "%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
          "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
          "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
        "%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
        "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
        : "memory");
}
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
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
                 "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
                 : "memory");
}
// A wait of a whole warp, in line (kernels that move registers between warps cannot call a function): true once the phase is
// complete, false after the limit or when another warp gave up.
__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    unsigned long long t0 = 0;
#pragma unroll 1
    for (uint32_t i = 1;; ++i) {
        if (__all_sync(0xffffffffu, mbar_try(bar, parity))) return true;
        if ((i & 255) == 0) {
            const unsigned long long now = gtime_ns();
            if (!t0) t0 = now;
            if (__any_sync(0xffffffffu, *abort_flag || now - t0 > kWaitLimitNs)) {
                *abort_flag = 1;
                return false;
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

// What a block works on: rows [first, first + n) of the packed q, sequence b.
struct PromptItem {
    int b, rows;           // sequence, rows of it in this block (0: nothing to do)
    int64_t row;           // the first one, packed
    int behind;            // rows from the first one to the sequence's end
    int keys, row0;        // keys of the sequence; packed: the first one's row
    // keys that row r of the block sees
    __device__ __forceinline__ int sees(int r, int causal) const {
        return causal ? min(max(keys - behind + 1 + r, 0), keys) : keys;
    }
};
// Block `item` of those of all sequences, `per` rows each; counted from the end, so that the blocks with most keys of a
// long sequence come first.  A warp's lanes work together and get the same answer.
static __device__ __forceinline__ PromptItem prompt_item(const PromptArgs& a, int per, int item) {
    const int lane = threadIdx.x & 31;
    auto rows_of = [&](int b, int64_t* first) {
        int64_t last;
        *first = 0;
        if (b >= a.seqs) return 0;
        packed_range(a.cu_q, b, a.rows, first, &last);
        return (int)(last - *first);
    };
    PromptItem it;
    it.rows = 0;
    int base = 0;
    for (int b0 = (a.seqs - 1) & ~31; b0 >= 0; b0 -= 32) {
        int64_t first;
        const int b = b0 + 31 - lane, n = rows_of(b, &first), m = (n + per - 1) / per;
        int x = m;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += y;
        }
        const unsigned behind = __ballot_sync(0xffffffffu, base + x > item);
        if (behind) {
            const int src = __ffs((int)behind) - 1;
            const int end = __shfl_sync(0xffffffffu, base + x, src), rows = __shfl_sync(0xffffffffu, n, src);
            const int block = end - 1 - item;              // (of the sequence, from its start)
            if (block < 0 || (int64_t)block * per >= rows) return it;     // (sequences that overlap beyond counting)
            it.b = b0 + 31 - src;
            it.row = __shfl_sync(0xffffffffu, (int)first, src) + (int64_t)block * per;
            it.behind = rows - block * per;
            it.rows = it.behind < per ? it.behind : per;
            int64_t row0;
            it.keys = (int)kv_length(a.kv, it.b, &row0);
            it.row0 = (int)row0;
            return it;
        }
        base += __shfl_sync(0xffffffffu, x, 31);
    }
    return it;
}

// The block's rows one by one, from the positions they see alone.
template <typename T>
__device__ __forceinline__ void prompt_rows(const PromptArgs& a, const PromptItem& it, int h, int warp, int warps) {
    const int lane = threadIdx.x & 31;
    using S = RowState<T>;      // (head_dim <= 128: one piece of a lane)
    bool bad = false;
    for (int r = warp; r < it.rows; r += warps) {
        S st;
        bad |= attend_row(a, it.b, it.row + r, h, it.behind - r, 0, kRowPos, &st);
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
