// What the kernels over a paged cache share: where a sequence's rows are, element types, argument checks.
//
// A pool holds n_pages pages of `page` positions (a power of two), a position n_kv heads of head_dim elements: the rows
// of the contiguous caches [position][n_kv][head_dim], cut into pages.  A sequence's row of the table names its pages in
// order, so a contiguous cache is the pool whose table counts up.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>

#include "internal.h"

namespace rstq {

constexpr int kMaxSeqs = 65536;
constexpr int64_t kMaxPages = 1 << 20;      // of a pool
constexpr int64_t kMaxRows = 1ll << 30;     // packed rows of a call
constexpr int kStatusPage = 1;              // word of DeviceState::status: a table named a page outside the pool
constexpr int kPagedGroup = 16;             // query heads of a KV head that one thread block of the decode kernel serves

// What attention keeps in memory between (and for long sums, beside) the registers of its blocks of threads: slots of floats.
constexpr int kPromptSlots = 512;      // items of a call whose blocks' keys are cut into parts
// a slot, in floats: up to 256 rows' sums (of more than 128 columns 128 rows'), four columns at a time; their references; their sums of weights; whether they have to be taken again
template <int HD>
__host__ __device__ constexpr int prompt_slot() { return (HD > 128 ? 128 : 256) * (HD + 2) + 32; }
static_assert(prompt_slot<256>() <= prompt_slot<128>() && prompt_slot<64>() <= prompt_slot<128>(), "the slots are laid out for 128 columns");
constexpr int64_t kPromptSlotFloats = (int64_t)kPromptSlots * prompt_slot<128>();

template <typename T>
struct Elem;
template <>
struct Elem<float> {
    static constexpr int kVec = 4;   // elements of 16 bytes
    static __device__ __forceinline__ void load(const float* p, float (&v)[4]) {
        const float4 x = *reinterpret_cast<const float4*>(p);
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    }
};
template <>
struct Elem<__nv_bfloat16> {
    static constexpr int kVec = 8;
    static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&v)[8]) {
        const uint4 x = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
};
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {   // rounded to nearest, ties to even
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// four consecutive elements
__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    return make_float4(__uint_as_float(x.x << 16), __uint_as_float(x.x & 0xFFFF0000u), __uint_as_float(x.y << 16),
                       __uint_as_float(x.y & 0xFFFF0000u));
}
__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store4(__nv_bfloat16* p, float4 v) {
    *reinterpret_cast<uint2*>(p) = make_uint2(bf16_pair(v.x, v.y), bf16_pair(v.z, v.w));
}

// The rows of the sequences' keys and values: in the pages of a pool, or packed one sequence after the other.
struct KvPlace {
    const int32_t* table;   // [seqs][width]; null: packed
    const int32_t* lens;    // paged: positions of each sequence, this call's own among them
    const int32_t* cu;      // packed: first row of each sequence, and the end of the last
    int64_t rows;           // packed: rows there are
    int64_t n_pages;
    int64_t ld;             // elements from a row to the next
    int width, shift;       // pages of a row of the table; log2 of a page's positions
    int* status;
};
__device__ __forceinline__ int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); }
// Rows of sequence b of a packed array: whatever the words of `cu` hold, inside [0, rows].
__device__ __forceinline__ void packed_range(const int32_t* cu, int b, int64_t rows, int64_t* first, int64_t* last) {
    *first = clamp64(cu[b], 0, rows);
    *last = clamp64(cu[b + 1], *first, rows);
}
// Positions of sequence b that have a place; packed: *row0 = its first row.
__device__ __forceinline__ int64_t kv_length(const KvPlace& kv, int b, int64_t* row0) {
    if (kv.table) {
        *row0 = 0;
        return clamp64(kv.lens[b], 0, (int64_t)kv.width << kv.shift);
    }
    int64_t last;
    packed_range(kv.cu, b, kv.rows, row0, &last);
    return last - *row0;
}
// Where sequence b, of n positions that have a place, ends: the position behind its last row.  That is n, but for a length beyond the
// sequence's pages.
__device__ __forceinline__ int64_t kv_end(const KvPlace& kv, int b, int64_t n) { return kv.table && kv.lens[b] > n ? kv.lens[b] : n; }
// Row of the pool (of the packed array) that holds position `pos` of sequence b; -1: the table names no page of the pool.
__device__ __forceinline__ int64_t kv_row(const KvPlace& kv, int b, int64_t row0, int64_t pos) {
    if (!kv.table) return row0 + pos;
    const int page = kv.table[(int64_t)b * kv.width + (pos >> kv.shift)];
    if ((uint32_t)page >= (uint64_t)kv.n_pages) return -1;
    return ((int64_t)page << kv.shift) + (pos & ((1 << kv.shift) - 1));
}
// The sequence of a packed row: the last one that begins at or before it; -1: none holds it.
__device__ __forceinline__ int row_sequence(const int32_t* cu, int seqs, int64_t row) {
    int lo = 0, hi = seqs;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] <= row) lo = mid + 1;
        else hi = mid;
    }
    const int b = lo - 1;
    return b >= 0 && row < cu[b + 1] ? b : -1;
}

// ---- argument checks of the entry points ----
inline bool paged_buf(const rstq_buf* b, const rstq_ctx* ctx, int64_t bytes) {
    return b && b->magic == kBufMagic && b->ctx == ctx && b->bytes >= bytes && ((uintptr_t)b->ptr & 15) == 0;
}
// Bytes of an array that a call reads or writes.
struct Span {
    const void* p;
    int64_t n;
};
inline bool apart(const Span& a, const Span& b) {
    const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
    return a.n <= 0 || b.n <= 0 || x + (uintptr_t)a.n <= y || y + (uintptr_t)b.n <= x;
}
// No array that is written lies over another one, read or written.
template <size_t W, size_t R>
inline bool apart(const Span (&written)[W], const Span (&read)[R]) {
    for (size_t i = 0; i < W; ++i) {
        for (size_t j = i + 1; j < W; ++j)
            if (!apart(written[i], written[j])) return false;
        for (size_t j = 0; j < R; ++j)
            if (!apart(written[i], read[j])) return false;
    }
    return true;
}
inline int elem_bytes(int32_t dtype) { return dtype == RSTQ_BF16 ? 2 : 4; }
inline int log2_of(int64_t v) {
    int s = 0;
    while ((1ll << s) < v) ++s;
    return s;
}
// n_q = group x n_kv heads of head_dim, of a type these kernels take
int32_t check_heads(int64_t n_q, int64_t group, int64_t n_kv, int64_t head_dim, int32_t dtype);
// a pool's and a table's sizes
int32_t check_pages(int64_t seqs, int64_t page, int64_t n_pages, int64_t max_pages);
template <typename... B>
inline bool same_device(const rstq_buf* a, const B*... rest) {
    return ((rest == nullptr || rest->dev == a->dev) && ...);
}

struct PromptArgs {
    const void *q, *k, *v;
    void* out;
    const int32_t* cu_q;    // null: one row per sequence
    KvPlace kv;
    int64_t rows, ldq;
    int seqs, n_q, group, n_kv, head_dim;
    float scale;
    int causal;
    int32_t dtype;
    int64_t kv_rows;        // rows of the pool or of the packed arrays
    const int64_t* start;   // what launch_sums wrote; null: few sequences
};
// ---- a row's attention by one warp, any shape ----
// The lanes hold 16-byte pieces of the head, a dot product is a sum over them; kRowPos positions at a time, the softmax runs
// along.  Only positions that the row sees are read, so what lies elsewhere (NaN too) cannot reach it.  Every sum in f32.
constexpr int kRowPos = 4;
template <typename T>
struct RowState {
    static constexpr int V = Elem<T>::kVec, C = 256 / (32 * V) < 1 ? 1 : 256 / (32 * V);   // elements of a piece; pieces of a lane
    float o[C][V], m, l;
};
// Row `row` of head h, which sees `len` positions of sequence b, against positions first .. first + kRowPos - 1, and so on every `step`.
// True: a position had no page.  beat: a word that changes every few thousand positions, for those who wait.
template <typename T>
__device__ __forceinline__ bool attend_row(const PromptArgs& p, int b, int64_t row, int h, int64_t len, int64_t first, int64_t step,
                                           RowState<T>* st, int* beat = nullptr) {
    constexpr int V = RowState<T>::V, C = RowState<T>::C;
    const int lane = threadIdx.x & 31, hd = p.head_dim, hkv = h / p.group;
    int64_t row0;
    kv_length(p.kv, b, &row0);
    float q[C][V];
    st->m = -INFINITY;
    st->l = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int e = (c * 32 + lane) * V;
#pragma unroll
        for (int i = 0; i < V; ++i) q[c][i] = st->o[c][i] = 0.f;
        if (e < hd) Elem<T>::load((const T*)p.q + row * p.ldq + (int64_t)h * hd + e, q[c]);
    }
    bool bad = false;
    const float scale2 = p.scale * 1.4426950408889634f;
    for (int64_t j0 = first; j0 < len; j0 += step) {
        if (beat && (j0 & 16383) < step && lane == 0) atomicAdd(beat, 1);
        float s[kRowPos];
        int64_t at[kRowPos];
#pragma unroll
        for (int u = 0; u < kRowPos; ++u) {
            at[u] = j0 + u < len ? kv_row(p.kv, b, row0, j0 + u) : -1;
            bad |= j0 + u < len && at[u] < 0;
            s[u] = 0.f;
            if (at[u] >= 0) {
                const T* k = (const T*)p.k + at[u] * p.kv.ld + (int64_t)hkv * hd;
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const int e = (c * 32 + lane) * V;
                    float x[V];
                    if (e < hd) {
                        Elem<T>::load(k + e, x);
#pragma unroll
                        for (int i = 0; i < V; ++i) s[u] = fmaf(q[c][i], x[i], s[u]);
                    }
                }
            }
        }
#pragma unroll
        for (int d = 16; d; d >>= 1)
#pragma unroll
            for (int u = 0; u < kRowPos; ++u) s[u] += __shfl_xor_sync(0xffffffffu, s[u], d);
        float top = st->m;
#pragma unroll
        for (int u = 0; u < kRowPos; ++u) {
            s[u] = at[u] >= 0 ? s[u] * scale2 : -INFINITY;
            top = s[u] > top || s[u] != s[u] ? s[u] : top;     // (a NaN stays one)
        }
        if (top == -INFINITY) continue;
        const float w = exp2f(st->m - top);
        st->l *= w;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < V; ++i) st->o[c][i] *= w;
        st->m = top;
#pragma unroll
        for (int u = 0; u < kRowPos; ++u) {
            if (at[u] < 0) continue;
            const float e2 = exp2f(s[u] - top);
            st->l += e2;
            const T* v = (const T*)p.v + at[u] * p.kv.ld + (int64_t)hkv * hd;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int e = (c * 32 + lane) * V;
                float x[V];
                if (e < hd) {
                    Elem<T>::load(v + e, x);
#pragma unroll
                    for (int i = 0; i < V; ++i) st->o[c][i] = fmaf(e2, x[i], st->o[c][i]);
                }
            }
        }
    }
    return bad;
}

// ---- many sequences: where each one's work begins ----
// Up to this many a kernel adds the lengths up itself, 32 at a time, for every place that it looks for; above, one launch ahead of it writes
// the sums (start[b], and all of it in start[seqs]), and a place is found by search.  (Prompts of 100 rows, 128 of them 85 us without and 90 with
// that launch, 300 240 and 192; 4000 of 4 rows 6.2 and 1.1 ms.)
constexpr int kSumSeqs = 128;
// The last sequence that begins at or before unit `at` < start[seqs].  A warp's lanes work together and get the same answer.
__device__ __forceinline__ int find_start(const int64_t* start, int seqs, int64_t at) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = seqs;                // it is one of lo .. lo + n - 1
    while (n > 1) {
        const int step = (n + 31) >> 5, i = lo + lane * step;
        const unsigned in = __ballot_sync(0xffffffffu, lane * step < n && start[i] <= at);      // (a run from lane 0 on)
        const int l = 31 - __clz((int)(in | 1u));
        n = min(step, n - l * step);
        lo += l * step;
    }
    return lo;
}
// Sums of ceil(rows of a sequence / per) for packed rows, of ceil(positions / per) + extra (of none: 0) where cu_q is null.
int32_t launch_sums(DeviceState& ds, const PromptArgs& a, int per, int extra);

// A pool (or packed rows) as [rows][heads][head_dim], read in boxes of 128 bytes x `box` rows of one head.
int32_t rows_tensor_map(CUtensorMap* m, const void* base, int32_t dtype, int64_t rows, int64_t ld, int heads, int head_dim, int box);
// prompt_attn.cu (bf16), prompt_f32.cu (head_dim <= 128): scale > 0, keys to read.  (*launches: how many)
int32_t launch_prompt(DeviceState& ds, const PromptArgs& a, int* launches);
int32_t launch_prompt_f32(DeviceState& ds, const PromptArgs& a, int* launches);
// paged_attn.cu: any head_dim and length, a warp per position
int32_t launch_attention_rows(DeviceState& ds, const PromptArgs& a);
// paged_decode.cu: one row per sequence, paged
int32_t launch_paged_decode(DeviceState& ds, const PromptArgs& a, int* launches);

}  // namespace rstq
