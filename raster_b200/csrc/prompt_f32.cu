// Causal attention of whole prompts, f32, head_dim up to 128, on the tcgen05 tensor cores: prompt_attn.cu's walk with every operand as
// three bf16 terms.
//
//   x = x1 + x2 + x3, each the leading 8 bits of what is left (24 bits in all: exact);
//   x y = x1 y1 + (x1 y2 + x2 y1 + x2 y2 + x1 y3 + x3 y1)          to 2^-24 of it
//
// for Q K^T and for P V alike: six MMAs instead of one.  The tensor core's additions cut off, always towards zero, so no sum stays there for
// long: the first product has one of its own and the five small ones another, in tensor memory, and P V of every tile of keys is taken out and
// added, to nearest, to sums in registers.  (Left in tensor memory over all keys a result lost 6e-9 of itself with every key: 1.2e-5 of it after
// 4000, 7.7e-5 after 16000, 3.7e-4 after 64000; as it is 2e-7, 3e-7, 6e-7.  It costs nothing: O is not rescaled in tensor memory any more; 1024
// rows of 16 heads x 64 38 and 39 us, x 128 59 and 57.)  f32 FMAs would be bound by 72 TFLOP/s of the whole device, the six MMAs by a
// sixth of bf16's rate.
//
// A block has a tile of 128 (row, head) pairs of one sequence: rows of a head, or rows of all heads of a group as in prompt_attn.cu.  Four warps
// (eight above 64 columns) fetch K and V, a tile of 64 keys at a time and one ahead in registers, split them and write the terms to shared memory,
// swizzled as the tensor core wants them (zeros behind the last key); eight warps are the softmax, two threads per row with half of the keys
// each, P's three terms over S in tensor memory; one thread issues.  There are two places for S and P, and the next tile's S is formed while this
// one's exponentials are.  (Of 64 columns two blocks with one place each would fit an SM: two sequences of 1000 rows 63 us, against 46.)  A step of
// 64 keys takes 1.7 us with 64 columns, 3.0 with 128, of which the MMAs are 1 and 2 (an MMA of S is bound by reading Q and K from shared memory, 48
// cycles): the rest is the way of K and V through registers and their split, one tile at a time, which a second tile ahead only lengthens (spills).
// 1024 rows of 16 heads: 39 and 57 us.
// Few blocks that see many keys are cut into parts as in prompt_attn.cu: 2 rows behind 4000 keys of 8 heads of 128 212 -> 39 us, 300 of 64 columns
// 129 -> 50.
//
// An infinity or NaN has no such terms: a block that meets one (in keys or values its rows may not even see) computes its rows one by one
// (attend_row), and so does one whose table names no page.
#include <algorithm>

#include "prompt.cuh"

namespace rstq {

constexpr int kPfRows = 128, kPfKeys = 64, kPfPlaces = 2;      // places for S in tensor memory
template <int HD>
struct PromptShapeF {
    static constexpr int blks = HD / 64, qblk = kPfRows * 128, kblk = kPfKeys * 128;     // 64 columns of a term
    static constexpr int qplane = blks * qblk, kplane = blks * kblk;
    static constexpr int smem = 1024 + 3 * (qplane + 2 * kplane);
    static constexpr int soft = 8, split = HD == 128 ? 8 : 4;      // warps: softmax, split, and one for the MMAs
    // Registers of a thread: 128 columns' softmax has 64 sums of its row, so there the split's and the MMAs' threads (a warpgroup of which one warp
    // works) give some of theirs up.  (With 17 warps none could have more than 96, and the sums would be spilled.)
    static constexpr bool moved = HD == 128;
    static constexpr int threads = (soft + split + (moved ? 4 : 1)) * 32;
    static constexpr int launched = 96, soft_regs = 128, split_regs = 96, mma_regs = 32;
    static_assert(soft * soft_regs + split * split_regs + 4 * mma_regs <= (soft + split + 4) * launched || !moved, "more than there are: the wait for them would not end");
};

struct PromptParamsF {
    PromptArgs a;
    int pack, rpt, heads;            // heads of a group that share a tile (1: none), rows of q of a tile, blocks per rows of a tile
    int over_pack;                   // 2^16 / pack, rounded up: x / pack = x * over_pack >> 16 for x < 128 (off by less than 128 / 2^16 < 1 / pack)
    float scale2;
    int* status;
    int sms;                         // blocks that run at once
    PromptJoin join;                 // where the parts of a block's keys go
};

// The next eight bits of a pair of values, as bf16 pair; the values become what is left.
__device__ __forceinline__ uint32_t next_term(float& a, float& b) {
    const uint32_t w = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
    unpack2(fma2(pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)), pack2(-1.f, -1.f), pack2(a, b)), a, b);
    return w;
}

// PARTS: a block's keys may be cut into parts.
template <int HD, bool PARTS>
__global__ void __launch_bounds__(PromptShapeF<HD>::threads, 1)
prompt_f32_kernel(const PromptParamsF p) {
    using Sh = PromptShapeF<HD>;
    constexpr int NB = kPfPlaces, SOFT = Sh::soft, SPLIT = Sh::split;
    extern __shared__ uint8_t s_raw0[];
    uint8_t* s_raw = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(s_raw0) + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t s_bar[15];
    __shared__ float s_pair[2][2][kPfRows];      // what the two threads of a row tell each other: [turn][half][row]
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort, s_again;
    __shared__ PromptItem s_item;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;      // (the same in all lanes, for the compiler too)
    const uint32_t sq = smem_u32(s_raw), sk = sq + 3 * Sh::qplane, sv = sk + 3 * Sh::kplane;
    // qfull, kfull, vfull: the terms are written; kfree, vfree: the products that read them are done; sfull, pfull: S, P of a place;
    // odone: P V is added; over: everything is, after a wait ran out
    const uint32_t qfull = smem_u32(s_bar), kfull = qfull + 8, kfree = qfull + 16, vfull = qfull + 24, vfree = qfull + 32, sfull = qfull + 40,
                   pfull = qfull + 56, odone = qfull + 72, over = qfull + 80, pair = qfull + 88;
    volatile int* abort_flag = &s_abort;
    const int h = blockIdx.x % p.heads, hkv = p.pack > 1 ? h : h / p.a.group;      // query head, or the packed ones' KV head
    if (tid == 0) {
        s_abort = s_again = 0;
        mbar_init(qfull, SPLIT);
        mbar_init(kfull, SPLIT);
        mbar_init(kfree, 1);
        mbar_init(vfull, SPLIT);
        mbar_init(vfree, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(sfull + 8 * i, 1);
            mbar_init(pfull + 8 * i, SOFT);
        }
        mbar_init(odone, 1);
        mbar_init(over, 1);
        for (int i = 0; i < 4; ++i) mbar_init(pair + 8 * i, 2);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == SOFT + SPLIT) {
        tmem_alloc(smem_u32(&s_tmem), 512);
        tmem_relinquish();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp == 0) {
        PromptItem it;
        if (PARTS) {
            int items;
            const int share = prompt_share(p.a, p.rpt, kPfKeys, p.heads, p.sms, HD == 64 ? 5 : 3, HD == 64 ? 8 : 4, &items);      // (a block's begin and end 8 us)
            it = prompt_item(p.a, p.rpt, kPfKeys, share, blockIdx.x / p.heads);
            if (lane == 0) {
                if (blockIdx.x == 0) *p.join.listed = items;
                if ((int)blockIdx.x < items) p.join.list[blockIdx.x] = it;
            }
        } else it = prompt_block(p.a, p.rpt, kPfKeys, blockIdx.x / p.heads);
        if (lane == 0) s_item = it;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = (uint32_t)uniform((int)s_tmem);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");     // (not before this block has its tensor memory)
    const PromptItem it = s_item;
    const int key0 = PARTS && it.rows > 0 ? it.j0 * kPfKeys : 0;      // the part's first key
    auto sees = [&](int r) { return it.sees(r, p.a.causal) - key0; };     // keys that row r sees, from there
    const int n = uniform(it.rows > 0 ? it.j1 - (PARTS ? it.j0 : 0) : 0);      // (the last row's tiles)
    const bool whole = !PARTS || it.rows == 0 || it.parts == 1;
    const uint32_t tO = tmem + NB * 128;

    if (warp < SOFT) {
        // ---- softmax: two threads per row, half of the keys each ----
        if constexpr (Sh::moved) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Sh::soft_regs));
        const int half = warp >> 2, quarter = warp & 3;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16, bar = pair + 8 * quarter;
        const int rt = quarter * 32 + lane, r = rt * p.over_pack >> 16, head = h * p.pack + rt - r * p.pack, mine = sees(r) - half * 32, least = sees(0) - half * 32;
        float m = -INFINITY, m2 = 0.f, sum = 0.f;
        uint32_t turn = 0;
        bool ok = true;
        // What the row's other thread says.  Both warps have read what they read of tensor memory before either goes on.
        auto other = [&](float x) {
            s_pair[turn & 1][half][rt] = x;
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
            ok = wait_phase(bar, turn & 1, abort_flag);
            tc_fence_after();
            const float y = s_pair[turn & 1][half ^ 1][rt];
            ++turn;
            return y;
        };
        // Sums of P V so far, of this thread's half of the columns; a tile's P V added to them.
        uint64_t o[HD / 4];
#pragma unroll
        for (int i = 0; i < HD / 4; ++i) o[i] = 0ull;
        auto fold = [&]() {
#pragma unroll
            for (int c = 0; c < HD / 2; c += 16) {
                uint32_t a[16], b[16];
                tmem_ld_x2_wait(tO + lanes + half * (HD / 2) + c, tO + lanes + HD + half * (HD / 2) + c, a, b);
#pragma unroll
                for (int i = 0; i < 16; i += 2)
                    o[(c + i) / 2] = add2(o[(c + i) / 2], add2(pack2(__uint_as_float(a[i]), __uint_as_float(a[i + 1])), pack2(__uint_as_float(b[i]), __uint_as_float(b[i + 1]))));
            }
        };
        for (int j = 0; j < n; ++j) {
            const int buf = j % NB;
            const uint32_t tS = tmem + buf * 128 + lanes;
            if (ok) ok = wait_phase(sfull + 8 * buf, (j / NB) & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            float s[32];
            constexpr int SW = Sh::moved ? 8 : 16;      // columns at a time: what the registers hold beside the sums
#pragma unroll
            for (int c = 0; c < 32; c += SW) {
                uint32_t a[SW], b[SW];
                tmem_ld_x2_wait(tS + half * 32 + c, tS + 64 + half * 32 + c, a, b);
#pragma unroll
                for (int i = 0; i < SW; i += 2)
                    unpack2(add2(pack2(__uint_as_float(a[i]), __uint_as_float(a[i + 1])), pack2(__uint_as_float(b[i]), __uint_as_float(b[i + 1]))), s[c + i], s[c + i + 1]);
            }
            if (j * kPfKeys + 32 > least) {
                const int lim = mine - j * kPfKeys;
#pragma unroll
                for (int i = 0; i < 32; ++i) s[i] = i < lim ? s[i] : -INFINITY;
            }
            float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int i = 4; i < 32; ++i) top[i & 3] = fmaxf(top[i & 3], s[i]);
            float rowmax = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
            rowmax = fmaxf(rowmax, other(rowmax));
            if (!ok) break;
            const bool grown = rowmax > m;
            const bool any = __any_sync(0xffffffffu, grown);
            float f = 1.f;
            if (grown) {
                const float next = rowmax * p.scale2;
                f = m == -INFINITY ? 0.f : ex2f(m2 - next);
                m = rowmax;
                m2 = next;
                sum *= f;
            }
            uint64_t part[2] = {0ull, 0ull};
            const uint64_t scale = pack2(p.scale2, p.scale2), minus = pack2(-m2, -m2);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                uint32_t w[3][8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float a, b;
                    unpack2(fma2(pack2(s[16 * g + 2 * i], s[16 * g + 2 * i + 1]), scale, minus), a, b);
                    a = ex2f(a);
                    b = ex2f(b);
                    part[i & 1] = add2(part[i & 1], pack2(a, b));
                    w[0][i] = next_term(a, b);
                    w[1][i] = next_term(a, b);
                    w[2][i] = next_term(a, b);
                }
#pragma unroll
                for (int x = 0; x < 3; ++x) tmem_st8(tS + x * 32 + half * 16 + g * 8, w[x]);
            }
            float a, b;
            unpack2(add2(part[0], part[1]), a, b);
            sum += a + b;
            // the last tile's P V, before this one's takes its place
            if (j > 0) {
                ok = wait_phase(odone, (j - 1) & 1, abort_flag);
                if (!ok) break;
                tc_fence_after();
                fold();
                if (any) {
                    const uint64_t f2 = pack2(f, f);
#pragma unroll
                    for (int i = 0; i < HD / 4; ++i) o[i] = mul2(o[i], f2);
                }
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(pfull + 8 * buf);
        }
        if (ok && n > 0) {
            ok = wait_phase(odone, (n - 1) & 1, abort_flag);
            tc_fence_after();
            if (ok) fold();
        }
        if (ok) {
            const float y = other(sum);
            sum = half ? y + sum : sum + y;      // (the same in both)
        }
        tc_fence_after();
        // (s_again is set before the terms it is about are handed on, and the last product came after all of them)
        const bool again = *(volatile int*)&s_again;
        if (ok && !whole) {
            // a part: sums, reference and sum of weights to its slot
            float* slot = p.join.part + (int64_t)blockIdx.x * prompt_slot<HD>();
            if (!half && rt < p.rpt * p.pack && r < it.rows) {
                slot[kPfRows * HD + rt] = m2;
                slot[kPfRows * (HD + 1) + rt] = sum;
            }
            if (tid == 0) slot[kPfRows * (HD + 2)] = again ? 1.f : 0.f;
#pragma unroll
            for (int i = 0; i < HD / 2; i += 4) {
                float4 v;
                unpack2(o[i / 2], v.x, v.y);
                unpack2(o[i / 2 + 1], v.z, v.w);
                store4(slot + ((half * (HD / 2) + i) / 4 * kPfRows + rt) * 4, v);
            }
        } else if (ok && !again) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const bool has_row = rt < p.rpt * p.pack && r < it.rows;
            float* out = (float*)p.a.out + ((it.row + r) * p.a.n_q + head) * p.a.head_dim;
            if (has_row)
#pragma unroll
                for (int i = 0; i < HD / 2; i += 4) {
                    const int c = half * (HD / 2) + i;
                    if (c >= p.a.head_dim) continue;
                    float4 v;
                    unpack2(o[i / 2], v.x, v.y);
                    unpack2(o[i / 2 + 1], v.z, v.w);
                    store4(out + c, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
                }
        }
        if (ok && whole && again)
            for (int i = 0; i < p.pack; ++i) prompt_rows<float>(p.a, it, h * p.pack + i, warp, SOFT);
    } else if (warp < SOFT + SPLIT) {
        // ---- split ----
        if constexpr (Sh::moved) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Sh::split_regs));
        constexpr int LPR = HD / 4, RPI = 32 / LPR, ROWS = kPfKeys / SPLIT, NI = ROWS / RPI;      // lanes of a row; rows of a load; a warp's rows of a tile, and loads
        const int w = warp - SOFT, d = (lane % LPR) * 4, sub = lane / LPR;
        const bool in = d < p.a.head_dim;
        const int din = in ? d : 0;
        uint32_t top = 0;             // largest magnitude seen, as bits
        auto write = [&](uint32_t base, int plane, int blk, int row, float4 x) {
            top = max(max(top, max(__float_as_uint(x.x) & 0x7FFFFFFFu, __float_as_uint(x.y) & 0x7FFFFFFFu)),
                      max(__float_as_uint(x.z) & 0x7FFFFFFFu, __float_as_uint(x.w) & 0x7FFFFFFFu));
            const uint32_t at = base + (d >> 6) * blk + row * 128 + ((((d & 63) >> 3) ^ (row & 7)) << 4) + (d & 4) * 2;
#pragma unroll
            for (int t = 0; t < 3; ++t) {
                const uint32_t a = next_term(x.x, x.y), b = next_term(x.z, x.w);
                asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at + t * plane), "r"(a), "r"(b) : "memory");
            }
        };
        auto hand = [&](uint32_t bar) {
            if (top >= 0x7F800000u) s_again = 1;
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        bool ok = n > 0;
        // this warp's rows of a tile of K and V: their places, a lane each
        auto places = [&](int j) {
            const int pos = key0 + j * kPfKeys + w * ROWS + (lane & (ROWS - 1));
            int64_t row = -1;
            if (j < n && pos < it.keys) {
                row = kv_row(p.a.kv, it.b, it.row0, pos);
                if (row < 0) s_again = 1;
            }
            return (int)row;
        };
        // Loads are made of some row in any case, so that all of them are under way at once; `live` says which rows count (a bit each).
        auto fetch = [&](float4 (&x)[NI], const void* base, int rows) {
            const float* from = (const float*)base + (int64_t)hkv * p.a.head_dim + din;
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int row = max(__shfl_sync(0xffffffffu, rows, i * RPI + sub), 0);
                x[i] = *reinterpret_cast<const float4*>(from + (int64_t)row * p.a.kv.ld);
            }
        };
        auto rows_in = [&](int rows) {
            const uint32_t there = __ballot_sync(0xffffffffu, rows >= 0) >> sub;
            return in ? there : 0u;
        };
        auto only = [&](bool there, float4 x) {
            return make_float4(there ? x.x : 0.f, there ? x.y : 0.f, there ? x.z : 0.f, there ? x.w : 0.f);
        };
        // K is written a tile ahead of V: the next S comes before this tile's P V
        float4 k[NI], v[NI];
        int r1 = places(0), r2 = places(1);
        uint32_t klive = 0, vlive = 0;
        if (ok) {
            fetch(k, p.a.k, r1);
            klive = rows_in(r1);
            for (int half = 0; half < 2; ++half) {      // (of its rows of Q, twice as many)
                float4 x[NI];
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const int rt = (w * 2 + half) * ROWS + i * RPI + sub, row = rt * p.over_pack >> 16, head = h * p.pack + rt - row * p.pack;
                    x[i] = *reinterpret_cast<const float4*>((const float*)p.a.q + (it.row + min(row, it.rows - 1)) * p.a.ldq + (int64_t)head * p.a.head_dim + din);
                }
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const int rt = (w * 2 + half) * ROWS + i * RPI + sub;
                    write(sq, Sh::qplane, Sh::qblk, rt, only(in && rt < it.rows * p.pack, x[i]));
                }
            }
            hand(qfull);
        }
        // (the fence of a hand-over waits for loads under way: both fetches come behind both)
        auto write_k = [&](int j) {
            if (!ok || j >= n) return;
            ok = wait_phase(kfree, (j & 1) ^ 1u, abort_flag);
            if (!ok) return;
#pragma unroll
            for (int i = 0; i < NI; ++i) write(sk, Sh::kplane, Sh::kblk, w * ROWS + i * RPI + sub, only(klive >> (i * RPI) & 1, k[i]));
            hand(kfull);
        };
        write_k(0);
        for (int j = 0; j < n && ok; ++j) {
            fetch(v, p.a.v, r1);
            vlive = rows_in(r1);
            if (j + 1 < n) fetch(k, p.a.k, r2);
            klive = rows_in(r2);
            r1 = r2;
            r2 = places(j + 2);
            write_k(j + 1);
            if (ok) ok = wait_phase(vfree, (j & 1) ^ 1u, abort_flag);
            if (!ok) break;
#pragma unroll
            for (int i = 0; i < NI; ++i) write(sv, Sh::kplane, Sh::kblk, w * ROWS + i * RPI + sub, only(vlive >> (i * RPI) & 1, v[i]));
            hand(vfull);
        }
    } else {
        // ---- MMAs ----
        if constexpr (Sh::moved) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Sh::mma_regs));
        if (warp == SOFT + SPLIT) {
        constexpr uint32_t id_s = idesc_bf16(kPfKeys), id_o = idesc_bf16(HD) | (1u << 16);     // (bit 16: B with N innermost)
        const bool leader = elect_one();
        bool ok = n > 0;
        auto wait = [&](uint32_t bar, uint32_t parity) {
            if (ok) ok = wait_phase(bar, parity, abort_flag);
            tc_fence_after();
        };
        // terms of the products: the first to the first sum, the others to the second
        // (two bits of a word each: the six are a loop, whose descriptors as constants would take a hundred registers)
        constexpr uint32_t terms_a = 0x850u, terms_b = 0x244u;      // 0 0 1 1 0 2 and 0 1 0 1 2 0, the first in the lowest bits
        auto term = [](uint32_t terms, int x) { return (terms >> (2 * x)) & 3u; };
        // low words of descriptors (in 16 bytes) and their high word; V's: the blocks of 64 columns apart
        const uint32_t hi = (uint32_t)(smem_desc_sw128(0) >> 32), lead = (uint32_t)smem_desc_sw128(0), lead_v = (uint32_t)smem_desc_rows(0, Sh::kblk);
        const uint32_t q0 = lead + (sq >> 4), k0 = lead + (sk >> 4), v0 = lead_v + (sv >> 4);
        auto product_s = [&](int j) {
            const uint32_t tS = tmem + (j % NB) * 128;
            wait(kfull, j & 1);
            if (!ok) return;
#pragma unroll 1
            for (int x = 0; x < 6; ++x) {
                const uint32_t d = tS + (x ? 64 : 0), q = q0 + term(terms_a, x) * (Sh::qplane >> 4), kk = k0 + term(terms_b, x) * (Sh::kplane >> 4);
#pragma unroll
                for (int k = 0; k < HD / 16; ++k)
                    if (leader) umma_ss(d, q + (k >> 2) * (Sh::qblk >> 4) + (k & 3) * 2, kk + (k >> 2) * (Sh::kblk >> 4) + (k & 3) * 2, hi, id_s, x > 1 || k > 0);
            }
            umma_commit_if(sfull + 8 * (j % NB), leader);
            umma_commit_if(kfree, leader);
        };
        wait(qfull, 0);
        if (n > 0) product_s(0);
        for (int j = 0; j < n && ok; ++j) {
            const uint32_t tP = tmem + (j % NB) * 128;
            if (j + 1 < n) product_s(j + 1);
            wait(vfull, j & 1);
            wait(pfull + 8 * (j % NB), (j / NB) & 1);
            if (!ok) break;
#pragma unroll 1
            for (int x = 0; x < 6; ++x) {
                const uint32_t d = tO + (x ? HD : 0), pp = tP + term(terms_a, x) * 32, vv = v0 + term(terms_b, x) * (Sh::kplane >> 4);
#pragma unroll
                for (int k = 0; k < kPfKeys / 16; ++k)
                    if (leader) umma_ts(d, pp + k * 8, vv + k * (2048 >> 4), hi, id_o, x > 1 || k > 0);
            }
            umma_commit_if(odone, leader);
            umma_commit_if(vfree, leader);
        }
        if (!ok && n > 0) {      // products under way are waited for (with a limit) before the memory they use is given up
            volatile int none = 0;
            umma_commit_if(over, leader);
            wait_phase(over, 0, const_cast<volatile int*>(&none));
        }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == SOFT + SPLIT) tmem_dealloc(tmem, 512);
    if (tid == 0 && s_abort) atomicExch(p.status, 2);
}

int32_t prompt_f32_configure() {
    constexpr auto attr = cudaFuncAttributeMaxDynamicSharedMemorySize;
    RSTQ_CUDA(cudaFuncSetAttribute((prompt_f32_kernel<64, false>), attr, PromptShapeF<64>::smem));
    RSTQ_CUDA(cudaFuncSetAttribute((prompt_f32_kernel<64, true>), attr, PromptShapeF<64>::smem));
    RSTQ_CUDA(cudaFuncSetAttribute((prompt_f32_kernel<128, false>), attr, PromptShapeF<128>::smem));
    RSTQ_CUDA(cudaFuncSetAttribute((prompt_f32_kernel<128, true>), attr, PromptShapeF<128>::smem));
    // registers are moved between warps: a block has to be launched with as many as are shared out
    using Sh = PromptShapeF<128>;
    cudaFuncAttributes a[2];
    RSTQ_CUDA(cudaFuncGetAttributes(&a[0], (prompt_f32_kernel<128, false>)));
    RSTQ_CUDA(cudaFuncGetAttributes(&a[1], (prompt_f32_kernel<128, true>)));
    RSTQ_REQUIRE(a[0].numRegs >= Sh::launched && a[1].numRegs >= Sh::launched, RSTQ_E_CUDA, "prompt_f32_kernel was built for %d and %d registers",
                 a[0].numRegs, a[1].numRegs);
    return RSTQ_OK;
}

int32_t launch_prompt_f32(DeviceState& ds, const PromptArgs& a, int* launches) {
    PromptParamsF p;
    p.a = a;
    p.scale2 = a.scale * 1.4426950408889634f;
    p.status = ds.status;
    p.pack = prompt_pack(a.group);
    p.rpt = kPfRows / p.pack;
    p.heads = a.n_q / p.pack;
    p.over_pack = (65536 + p.pack - 1) / p.pack;
    const int64_t blocks = (a.rows / p.rpt + std::min<int64_t>(a.seqs, a.rows)) * p.heads;
    RSTQ_REQUIRE(blocks < (1ll << 31), RSTQ_E_LIMIT, "%lld thread blocks", (long long)blocks);
    p.sms = prompt_sms(ds);
    p.join = prompt_join(ds, a, p.pack, p.rpt, p.heads);
    const bool parts = prompt_may_part(a, 768) && blocks <= p.sms;
    *launches = parts ? 2 : 1;
    if (!parts && a.seqs > kSumSeqs) {
        const int32_t rc = launch_sums(ds, a, p.rpt, 0);
        if (rc != RSTQ_OK) return rc;
        p.a.start = ds.seq_starts;
        ++*launches;
    }
    const dim3 grid((unsigned)(parts ? kPartRounds * p.sms : blocks));
    auto go = [&](auto kernel, auto shape) { return launch_pdl(kernel, grid, dim3(decltype(shape)::threads), (size_t)decltype(shape)::smem, ds, p); };
    if (a.head_dim <= 64) RSTQ_CUDA(parts ? go(prompt_f32_kernel<64, true>, PromptShapeF<64>()) : go(prompt_f32_kernel<64, false>, PromptShapeF<64>()));
    else RSTQ_CUDA(parts ? go(prompt_f32_kernel<128, true>, PromptShapeF<128>()) : go(prompt_f32_kernel<128, false>, PromptShapeF<128>()));
    return parts ? launch_prompt_join(ds, p.join) : RSTQ_OK;
}

}  // namespace rstq
