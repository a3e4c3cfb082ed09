// Serving many sequences from a paged cache: rows turned and written to their pages, and attention over them.
// The conventions (pool, table, lengths, packed rows) are those of paged.cuh.
#include <math.h>

#include "paged.cuh"
#include "sync_helpers.cuh"
#include "tcgen05_helpers.cuh"

namespace rstq {

int32_t check_heads(int64_t n_q, int64_t group, int64_t n_kv, int64_t head_dim, int32_t dtype) {
    RSTQ_REQUIRE(dtype == RSTQ_F32 || dtype == RSTQ_BF16, RSTQ_E_INVALID, "unknown element type %d", (int)dtype);
    RSTQ_REQUIRE(n_kv >= 1 && n_kv <= 65536 && group >= 1 && group <= 65536 && n_q == group * n_kv, RSTQ_E_SHAPE,
                 "n_q = %lld must be group (%lld) x n_kv (%lld)", (long long)n_q, (long long)group, (long long)n_kv);
    RSTQ_REQUIRE(head_dim >= 8 && head_dim % 8 == 0 && head_dim <= 256, RSTQ_E_SHAPE,
                 "head_dim = %lld (a multiple of 8, at most 256)", (long long)head_dim);
    return RSTQ_OK;
}
int32_t check_pages(int64_t seqs, int64_t page, int64_t n_pages, int64_t max_pages) {
    RSTQ_REQUIRE(seqs >= 1 && seqs <= kMaxSeqs, RSTQ_E_LIMIT, "seqs = %lld (1 .. %d)", (long long)seqs, kMaxSeqs);
    RSTQ_REQUIRE(page >= 16 && page <= 256 && (page & (page - 1)) == 0, RSTQ_E_SHAPE,
                 "page = %lld positions (16, 32, 64, 128 or 256)", (long long)page);
    RSTQ_REQUIRE(n_pages >= 1 && n_pages <= kMaxPages, RSTQ_E_LIMIT, "n_pages = %lld (1 .. %lld)", (long long)n_pages,
                 (long long)kMaxPages);
    RSTQ_REQUIRE(max_pages >= 1 && max_pages <= kMaxPages, RSTQ_E_LIMIT, "max_pages = %lld (1 .. %lld)", (long long)max_pages,
                 (long long)kMaxPages);
    return RSTQ_OK;
}

// ---- rope + append of packed rows --------------------------------------------------------------
struct AppendParams {
    const void *q, *k, *v;
    void *qout, *kpool, *vpool;
    const int32_t* cu;      // null: row t is sequence t's only one
    KvPlace kv;
    int64_t rows, ldq, ldkv;
    int seqs, n_q, n_kv, head_dim;
    double ln_theta;
};
// Items of a thread whose loads are under way together (1, 4: 4600 rows of 48 heads of 128, f32 to bf16 32.2, 31.5 us, to f32 44.1, 40.9).
constexpr int kAppendItems = 4;
// out = (x0 cos - x1 sin, x1 cos + x0 sin) over the halves of a head, in f32, rounded once to the type stored.  The angle
// pos * theta^(-2i/d) is formed and reduced to [-pi, pi] in f64, so that far positions keep f32's accuracy; sine and cosine are
// taken in f32 of the reduced angle's leading part and corrected by the rest of it.  They are shared by all heads of a row:
// a block works them out once for each of its rows, into shared memory.  Bound by HBM: each element in once, out once; 4556 rows of 32 + 8 + 8
// heads of 128, f32 to bf16, 168 MB: 32 us, 80 % of the copy rate, beside which are the places and angles at the start of each block.
template <typename TI, typename TO>
__global__ void __launch_bounds__(256)
paged_rope_append_kernel(const AppendParams p, const int per_block) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ __align__(16) uint8_t s_append[];
    int64_t* s_row = reinterpret_cast<int64_t*>(s_append);                 // row of the pool, -1: nothing to do
    int64_t* s_pos = s_row + per_block;
    float2* s_cs = reinterpret_cast<float2*>(s_pos + per_block);           // [per_block][head_dim / 2]: cosine, sine
    const int tid = threadIdx.x, h2 = p.head_dim >> 1;
    const int64_t t0 = (int64_t)blockIdx.x * per_block;
    const int n = p.rows - t0 < per_block ? (int)(p.rows - t0) : per_block;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (tid < n) {
        const int64_t t = t0 + tid;
        int64_t row = -1, pos = 0;
        const int b = p.cu ? row_sequence(p.cu, p.seqs, t) : (int)t;
        if (b >= 0) {
            const int64_t behind = p.cu ? (int64_t)p.cu[b + 1] - t : 1;    // rows from this one to the sequence's end
            pos = (int64_t)p.kv.lens[b] - behind;
            if (pos >= 0 && pos < ((int64_t)p.kv.width << p.kv.shift)) row = kv_row(p.kv, b, 0, pos);
            // (a sequence that holds nothing has no row in a step of all sequences: its slot is idle, which is no error)
            if (row < 0 && (p.cu || pos >= 0 || p.kv.table[(int64_t)b * p.kv.width] != -1)) p.kv.status[kStatusPage] = 1;
        }
        s_row[tid] = row;
        s_pos[tid] = pos;
    }
    __syncthreads();
    for (int i = tid; i < n * h2; i += 256) {
        const int r = i / h2, j = i - r * h2;
        const double a = (double)s_pos[r] * exp((-2.0 * (double)j) / (double)p.head_dim * p.ln_theta);
        const double turns = rint(a * 0.15915494309189535);
        const double red = fma(turns, -2.4492935982947064e-16, fma(turns, -6.283185307179586, a));
        const float hi = (float)red, lo = (float)(red - (double)hi);
        float s, c;
        sincosf(hi, &s, &c);
        s_cs[i] = make_float2(fmaf(-lo, s, c), fmaf(lo, c, s));
    }
    __syncthreads();
    const int quads = h2 >> 2, heads = p.n_q + 2 * p.n_kv;     // items of four pairs (of V: of eight elements)
    const int per_row = heads * quads, step = 256 * gridDim.y;
    constexpr int U = kAppendItems;
    for (int i0 = blockIdx.y * 256 + tid; i0 < n * per_row; i0 += U * step) {
        float4 a[U], b[U];
        TO* dst[U];
        int cs[U], gap[U];                                     // where the angles are (-1: none), how far the other half is
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * step;
            dst[u] = nullptr;
            if (i >= n * per_row) continue;
            const int r = i / per_row, e = i - r * per_row, h = e / quads, j = (e - h * quads) * 4;
            const int64_t row = s_row[r], t = t0 + r;
            if (row < 0) continue;
            const int hk = h - p.n_q, hv = hk - p.n_kv;
            const int64_t pool = row * p.kv.ld;
            cs[u] = hv < 0 ? r * h2 + j : -1;
            gap[u] = hv < 0 ? h2 : 4;
            const TI* src;
            if (hv >= 0) {
                src = (const TI*)p.v + t * p.ldkv + (int64_t)hv * p.head_dim + 2 * j;
                dst[u] = (TO*)p.vpool + pool + (int64_t)hv * p.head_dim + 2 * j;
            } else if (hk >= 0) {
                src = (const TI*)p.k + t * p.ldkv + (int64_t)hk * p.head_dim + j;
                dst[u] = (TO*)p.kpool + pool + (int64_t)hk * p.head_dim + j;
            } else {
                src = (const TI*)p.q + t * p.ldq + (int64_t)h * p.head_dim + j;
                dst[u] = (TO*)p.qout + (t * p.n_q + h) * p.head_dim + j;
            }
            a[u] = load4(src);
            b[u] = load4(src + gap[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!dst[u]) continue;
            float4 x = a[u], y = b[u];
            if (cs[u] >= 0) {
                const float4 cs0 = *reinterpret_cast<const float4*>(s_cs + cs[u]), cs1 = *reinterpret_cast<const float4*>(s_cs + cs[u] + 2);
                x.x = a[u].x * cs0.x - b[u].x * cs0.y; y.x = b[u].x * cs0.x + a[u].x * cs0.y;
                x.y = a[u].y * cs0.z - b[u].y * cs0.w; y.y = b[u].y * cs0.z + a[u].y * cs0.w;
                x.z = a[u].z * cs1.x - b[u].z * cs1.y; y.z = b[u].z * cs1.x + a[u].z * cs1.y;
                x.w = a[u].w * cs1.z - b[u].w * cs1.w; y.w = b[u].w * cs1.z + a[u].w * cs1.w;
            }
            store4(dst[u], x);
            store4(dst[u] + gap[u], y);
        }
    }
}

// ---- many sequences ------------------------------------------------------------------------------
// One block: a thread per sequence of 1024 at a time, sums over warps and then over the block.
constexpr int kSumThreads = 1024;
__global__ void __launch_bounds__(kSumThreads)
sums_kernel(const PromptArgs a, const int per, const int extra, int64_t* __restrict__ start) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __shared__ int64_t s_warp[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t base = 0;
    for (int b0 = 0; b0 < a.seqs; b0 += kSumThreads) {
        const int b = b0 + threadIdx.x;
        int64_t v = 0;
        if (b < a.seqs) {
            int64_t first, last;
            if (a.cu_q) {
                packed_range(a.cu_q, b, a.rows, &first, &last);
                v = (last - first + per - 1) / per;
            } else {
                const int64_t len = kv_length(a.kv, b, &first);
                v = len > 0 ? (len + per - 1) / per + extra : 0;
            }
        }
        int64_t x = v;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += y;
        }
        if (lane == 31) s_warp[warp] = x;
        __syncthreads();
        if (warp == 0) {
            int64_t w = s_warp[lane];
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int64_t y = __shfl_up_sync(0xffffffffu, w, d);
                if (lane >= d) w += y;
            }
            s_warp[lane] = w;
        }
        __syncthreads();
        if (b < a.seqs) start[b] = base + x - v + (warp ? s_warp[warp - 1] : 0);
        base += s_warp[31];
        __syncthreads();
    }
    if (threadIdx.x == 0) start[a.seqs] = base;
}
int32_t launch_sums(DeviceState& ds, const PromptArgs& a, int per, int extra) {
    RSTQ_CUDA(launch_pdl(sums_kernel, dim3(1), dim3(kSumThreads), 0, ds, a, per, extra, ds.seq_starts));
    return RSTQ_OK;
}

// ---- attention, any shape -----------------------------------------------------------------------
// One query row and head per thread block: its four warps take four positions in turn (attend_row), and their states are joined
// through shared memory.  For what the tiled kernels do not take: f32 prompts of head_dim above 128 (three terms of 128 rows of Q alone would fill shared memory; 1024 rows
// of 16 heads of 256 1.2 ms, where six MMAs per product would take 61 us), a scale that is not positive (they find the maximum
// before they scale), no keys at all.  Bound by L2: every row reads its keys and values itself.
constexpr int kRowWarps = 4;
template <typename T>
__global__ void __launch_bounds__(kRowWarps * 32)
attention_rows_kernel(const PromptArgs p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __shared__ float s_o[kRowWarps][256];
    __shared__ float s_ml[kRowWarps][2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hd = p.head_dim;
    const int64_t item = blockIdx.x, row = item / p.n_q;
    const int h = (int)(item - row * p.n_q);
    int b = (int)row;
    int64_t behind = 1;
    if (p.cu_q) {
        b = row_sequence(p.cu_q, p.seqs, row);
        if (b < 0) return;
        behind = (int64_t)p.cu_q[b + 1] - row;
    }
    int64_t row0;
    const int64_t keys = kv_length(p.kv, b, &row0), sees = p.causal ? clamp64(kv_end(p.kv, b, keys) - behind + 1, 0, keys) : keys;
    RowState<T> st;
    if (attend_row(p, b, row, h, sees, warp * kRowPos, kRowWarps * kRowPos, &st) && lane == 0) p.kv.status[kStatusPage] = 1;
#pragma unroll
    for (int c = 0; c < RowState<T>::C; ++c)
#pragma unroll
        for (int i = 0; i < RowState<T>::V; ++i)
            if ((c * 32 + lane) * RowState<T>::V < hd) s_o[warp][(c * 32 + lane) * RowState<T>::V + i] = st.o[c][i];
    if (lane == 0) {
        s_ml[warp][0] = st.m;
        s_ml[warp][1] = st.l;
    }
    __syncthreads();
    float top = -INFINITY, total = 0.f, w[kRowWarps];
#pragma unroll
    for (int i = 0; i < kRowWarps; ++i) top = s_ml[i][0] > top || s_ml[i][0] != s_ml[i][0] ? s_ml[i][0] : top;
#pragma unroll
    for (int i = 0; i < kRowWarps; ++i) {
        w[i] = s_ml[i][0] == -INFINITY ? 0.f : exp2f(s_ml[i][0] - top);
        total = fmaf(w[i], s_ml[i][1], total);
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;      // nothing to see: zeros
    for (int e = threadIdx.x * 4; e < hd; e += kRowWarps * 128) {
        float r[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kRowWarps; ++i)
            if (w[i] != 0.f)
#pragma unroll
                for (int j = 0; j < 4; ++j) r[j] = fmaf(w[i], s_o[i][e + j], r[j]);
        store4((T*)p.out + (row * p.n_q + h) * hd + e, make_float4(r[0] * inv, r[1] * inv, r[2] * inv, r[3] * inv));
    }
}

int32_t launch_attention_rows(DeviceState& ds, const PromptArgs& a) {
    const int64_t items = a.rows * a.n_q;
    RSTQ_REQUIRE(items < (1ll << 31), RSTQ_E_LIMIT, "rows x heads = %lld is beyond 2^31", (long long)items);
    if (a.dtype == RSTQ_BF16)
        RSTQ_CUDA(launch_pdl(attention_rows_kernel<__nv_bfloat16>, dim3((unsigned)items), dim3(kRowWarps * 32), 0, ds, a));
    else
        RSTQ_CUDA(launch_pdl(attention_rows_kernel<float>, dim3((unsigned)items), dim3(kRowWarps * 32), 0, ds, a));
    return RSTQ_OK;
}

}  // namespace rstq

using namespace rstq;

extern "C" {

int32_t rstq_paged_rope_append(rstq_ctx* ctx, rstq_buf* q, rstq_buf* k, rstq_buf* v, rstq_buf* qout, rstq_buf* kcache,
                               rstq_buf* vcache, rstq_buf* table, rstq_buf* lens, rstq_buf* cu, int64_t rows, int64_t seqs,
                               int64_t n_q, int64_t n_kv, int64_t head_dim, int64_t page, int64_t n_pages, int64_t max_pages,
                               int64_t ldq, int64_t ldkv, double theta, int32_t in_dtype, int32_t dtype) {
    RSTQ_REQUIRE(ctx && ctx->magic == kCtxMagic, RSTQ_E_INVALID, "invalid context handle");
    RSTQ_REQUIRE(n_kv >= 1 && n_q >= 1 && n_q <= 65536 && n_kv <= 65536, RSTQ_E_SHAPE, "n_q = %lld, n_kv = %lld", (long long)n_q,
                 (long long)n_kv);
    int32_t rc = check_heads(n_kv, 1, n_kv, head_dim, dtype);
    if (rc == RSTQ_OK) rc = check_heads(n_kv, 1, n_kv, head_dim, in_dtype);
    if (rc == RSTQ_OK) rc = check_pages(seqs, page, n_pages, max_pages);
    if (rc != RSTQ_OK) return rc;
    RSTQ_REQUIRE(rows >= 0 && rows <= kMaxRows && (cu || rows == seqs), RSTQ_E_SHAPE, "rows = %lld of %lld sequences (without cu, one each)",
                 (long long)rows, (long long)seqs);
    RSTQ_REQUIRE(theta > 0.0 && isfinite(theta), RSTQ_E_SHAPE, "theta = %g", theta);
    if (rows == 0) return RSTQ_OK;
    const int64_t qrow = n_q * head_dim, kvrow = n_kv * head_dim, ib = elem_bytes(in_dtype), ob = elem_bytes(dtype);
    if (!ldq) ldq = qrow;
    if (!ldkv) ldkv = kvrow;
    RSTQ_REQUIRE(ldq >= qrow && ldkv >= kvrow && ldq < (1ll << 31) && ldkv < (1ll << 31), RSTQ_E_SHAPE, "ldq = %lld, ldkv = %lld are shorter than a row", (long long)ldq,
                 (long long)ldkv);
    RSTQ_REQUIRE(ldq * ib % 16 == 0 && ldkv * ib % 16 == 0, RSTQ_E_ALIGN, "rows must start on 16-byte boundaries");
    const int64_t pool = n_pages * page * kvrow * ob;
    RSTQ_REQUIRE(paged_buf(q, ctx, ((rows - 1) * ldq + qrow) * ib) && paged_buf(k, ctx, ((rows - 1) * ldkv + kvrow) * ib) &&
                     paged_buf(v, ctx, ((rows - 1) * ldkv + kvrow) * ib) && paged_buf(qout, ctx, rows * qrow * ob) &&
                     paged_buf(kcache, ctx, pool) && paged_buf(vcache, ctx, pool) && paged_buf(table, ctx, seqs * max_pages * 4) &&
                     paged_buf(lens, ctx, seqs * 4) && (!cu || paged_buf(cu, ctx, (seqs + 1) * 4)),
                 RSTQ_E_INVALID, "invalid, unaligned or too small buffer");
    RSTQ_REQUIRE(same_device(q, k, v, qout, kcache, vcache, table, lens, cu), RSTQ_E_DEVICE, "buffers live on different devices");
    // in place: every pair of elements is read and written by one thread, if it stays where it is
    const bool in_place = qout->ptr == q->ptr && in_dtype == dtype && (ldq == qrow || rows == 1);
    const Span written[] = {{qout->ptr, rows * qrow * ob}, {kcache->ptr, pool}, {vcache->ptr, pool}};
    const Span read[] = {{k->ptr, ((rows - 1) * ldkv + kvrow) * ib}, {v->ptr, ((rows - 1) * ldkv + kvrow) * ib}, {table->ptr, seqs * max_pages * 4},
                         {lens->ptr, seqs * 4}, {cu ? cu->ptr : nullptr, cu ? (seqs + 1) * 4 : 0}};
    const Span qs = {q->ptr, ((rows - 1) * ldq + qrow) * ib};
    RSTQ_REQUIRE(apart(written, read) && (in_place || apart(written[0], qs)) && apart(written[1], qs) && apart(written[2], qs), RSTQ_E_INVALID,
                 "an array that is written lies over another one");
    DeviceState& ds = ctx->devs[q->dev];
    if ((rc = use_dev(ctx, q->dev)) != RSTQ_OK) return rc;
    AppendParams p;
    p.q = q->ptr; p.k = k->ptr; p.v = v->ptr;
    p.qout = qout->ptr; p.kpool = kcache->ptr; p.vpool = vcache->ptr;
    p.cu = cu ? (const int32_t*)cu->ptr : nullptr;
    p.kv = KvPlace{(const int32_t*)table->ptr, (const int32_t*)lens->ptr, nullptr, 0, n_pages, kvrow, (int)max_pages, log2_of(page), ds.status};
    p.rows = rows; p.ldq = ldq; p.ldkv = ldkv;
    p.seqs = (int)seqs; p.n_q = (int)n_q; p.n_kv = (int)n_kv; p.head_dim = (int)head_dim;
    p.ln_theta = log(theta);
    // Few rows: one per block, its heads over as many blocks as there is work of 256 threads; many: four per block, which share
    // the wait for their page numbers and angles.
    const int64_t items = (n_q + 2 * n_kv) * head_dim / 8;
    const int per = rows >= 8 * (int64_t)ds.sm_count ? 4 : 1;
    int64_t gy = per > 1 ? 1 : (items + 255) / 256;
    if (gy > 1 && gy * rows > 4 * (int64_t)ds.sm_count) gy = std::max<int64_t>(1, 4 * ds.sm_count / rows);
    if (gy > 65535) gy = 65535;
    const size_t smem = (size_t)per * (16 + head_dim / 2 * 8);
    const dim3 grid((unsigned)((rows + per - 1) / per), (unsigned)gy);
    auto go = [&](auto kernel) { return launch_pdl(kernel, grid, dim3(256), smem, ds, p, per); };
    cudaError_t e;
    if (in_dtype == RSTQ_F32) e = dtype == RSTQ_F32 ? go(paged_rope_append_kernel<float, float>) : go(paged_rope_append_kernel<float, __nv_bfloat16>);
    else e = dtype == RSTQ_F32 ? go(paged_rope_append_kernel<__nv_bfloat16, float>) : go(paged_rope_append_kernel<__nv_bfloat16, __nv_bfloat16>);
    RSTQ_CUDA(e);
    ctx->launches++;
    return RSTQ_OK;
}

// what the three attention entry points have in common
static int32_t attention_args(rstq_ctx* ctx, rstq_buf* q, rstq_buf* k, rstq_buf* v, rstq_buf* out, rstq_buf* table, rstq_buf* cu_q,
                              rstq_buf* lens_or_cu, int64_t rows, int64_t kv_rows, int64_t seqs, int64_t n_q, int64_t group,
                              int64_t n_kv, int64_t head_dim, int64_t page, int64_t n_pages, int64_t max_pages, int64_t ldq,
                              int64_t ldk, double scale, int32_t causal, int32_t dtype, bool packed, PromptArgs* a) {
    RSTQ_REQUIRE(ctx && ctx->magic == kCtxMagic, RSTQ_E_INVALID, "invalid context handle");
    int32_t rc = check_heads(n_q, group, n_kv, head_dim, dtype);
    if (rc == RSTQ_OK) rc = check_pages(seqs, packed ? 16 : page, packed ? 1 : n_pages, packed ? 1 : max_pages);
    if (rc != RSTQ_OK) return rc;
    RSTQ_REQUIRE(rows >= 0 && rows <= kMaxRows && kv_rows >= 0 && kv_rows <= kMaxRows, RSTQ_E_SHAPE, "rows = %lld, kv_rows = %lld",
                 (long long)rows, (long long)kv_rows);
    RSTQ_REQUIRE(causal == 0 || causal == 1, RSTQ_E_INVALID, "causal = %d (0 or 1)", (int)causal);
    RSTQ_REQUIRE(fabs(scale) <= 1e30, RSTQ_E_SHAPE, "scale = %g", scale);       // (log2(e) times it is a float too)
    const int64_t qrow = n_q * head_dim, kvrow = n_kv * head_dim, eb = elem_bytes(dtype);
    if (!ldq) ldq = qrow;
    if (!ldk) ldk = kvrow;
    RSTQ_REQUIRE(ldq >= qrow && ldk >= kvrow && ldq < (1ll << 31) && ldk < (1ll << 31), RSTQ_E_SHAPE, "ldq = %lld, ldk = %lld: shorter than a row",
                 (long long)ldq, (long long)ldk);
    RSTQ_REQUIRE(ldq * eb % 16 == 0 && ldk * eb % 16 == 0, RSTQ_E_ALIGN, "rows must start on 16-byte boundaries");
    const int64_t qb = rows ? ((rows - 1) * ldq + qrow) * eb : 0, kb = kv_rows ? ((kv_rows - 1) * ldk + kvrow) * eb : 0;
    RSTQ_REQUIRE(paged_buf(q, ctx, qb) && paged_buf(out, ctx, rows * qrow * eb) && paged_buf(k, ctx, kb) && paged_buf(v, ctx, kb) &&
                     (packed || paged_buf(table, ctx, seqs * max_pages * 4)) && (!cu_q || paged_buf(cu_q, ctx, (seqs + 1) * 4)) &&
                     paged_buf(lens_or_cu, ctx, (packed ? seqs + 1 : seqs) * 4),
                 RSTQ_E_INVALID, "invalid, unaligned or too small buffer");
    RSTQ_REQUIRE(same_device(q, k, v, out, table, cu_q, lens_or_cu), RSTQ_E_DEVICE, "buffers live on different devices");
    const Span written[] = {{out->ptr, rows * qrow * eb}};
    const Span read[] = {{q->ptr, qb}, {k->ptr, kb}, {v->ptr, kb}, {packed ? nullptr : table->ptr, packed ? 0 : seqs * max_pages * 4},
                         {cu_q ? cu_q->ptr : nullptr, cu_q ? (seqs + 1) * 4 : 0}, {lens_or_cu->ptr, (packed ? seqs + 1 : seqs) * 4}};
    RSTQ_REQUIRE(apart(written, read), RSTQ_E_INVALID, "out lies over an array that is read");
    DeviceState& ds = ctx->devs[q->dev];
    const int32_t* w = (const int32_t*)lens_or_cu->ptr;
    a->q = q->ptr; a->k = k->ptr; a->v = v->ptr; a->out = out->ptr;
    a->cu_q = cu_q ? (const int32_t*)cu_q->ptr : nullptr;
    a->kv = packed ? KvPlace{nullptr, nullptr, w, kv_rows, 0, ldk, 0, 0, ds.status}
                   : KvPlace{(const int32_t*)table->ptr, w, nullptr, 0, n_pages, ldk, (int)max_pages, log2_of(page), ds.status};
    a->rows = rows; a->ldq = ldq;
    a->seqs = (int)seqs; a->n_q = (int)n_q; a->group = (int)group; a->n_kv = (int)n_kv; a->head_dim = (int)head_dim;
    a->scale = (float)scale; a->causal = causal; a->dtype = dtype; a->kv_rows = kv_rows;
    a->start = nullptr;
    return use_dev(ctx, q->dev);
}

int32_t rstq_paged_decode_attention(rstq_ctx* ctx, rstq_buf* q, rstq_buf* kcache, rstq_buf* vcache, rstq_buf* out, rstq_buf* table,
                                    rstq_buf* lens, int64_t seqs, int64_t n_q, int64_t group, int64_t n_kv, int64_t head_dim,
                                    int64_t page, int64_t n_pages, int64_t max_pages, int64_t ldq, double scale, int32_t dtype) {
    PromptArgs a;
    int32_t rc = attention_args(ctx, q, kcache, vcache, out, table, nullptr, lens, seqs, n_pages * page, seqs, n_q, group, n_kv, head_dim,
                                page, n_pages, max_pages, ldq, 0, scale, 0, dtype, false, &a);
    if (rc != RSTQ_OK) return rc;
    DeviceState& ds = ctx->devs[q->dev];
    int launches = 1;
    rc = launch_paged_decode(ds, a, &launches);
    if (rc == RSTQ_OK) ctx->launches += launches;
    return rc;
}

static int32_t run_prompt(rstq_ctx* ctx, rstq_buf* q, const PromptArgs& a) {
    if (a.rows == 0) return RSTQ_OK;
    DeviceState& ds = ctx->devs[q->dev];
    int32_t rc;
    int launches = 1;
    if ((a.head_dim > 128 && a.dtype == RSTQ_F32) || a.scale <= 0.f || a.kv_rows == 0) rc = launch_attention_rows(ds, a);
    else rc = a.dtype == RSTQ_BF16 ? launch_prompt(ds, a, &launches) : launch_prompt_f32(ds, a, &launches);
    if (rc == RSTQ_OK) ctx->launches += launches;
    return rc;
}

int32_t rstq_prompt_attention(rstq_ctx* ctx, rstq_buf* q, rstq_buf* k, rstq_buf* v, rstq_buf* out, rstq_buf* cu_q, rstq_buf* cu_k,
                              int64_t rows, int64_t kv_rows, int64_t seqs, int64_t n_q, int64_t group, int64_t n_kv,
                              int64_t head_dim, int64_t ldq, int64_t ldk, double scale, int32_t causal, int32_t dtype) {
    PromptArgs a;
    RSTQ_REQUIRE(cu_q, RSTQ_E_INVALID, "null buffer: the rows' sequences");
    const int32_t rc = attention_args(ctx, q, k, v, out, nullptr, cu_q, cu_k, rows, kv_rows, seqs, n_q, group, n_kv, head_dim, 16, 1, 1, ldq, ldk,
                                      scale, causal, dtype, true, &a);
    return rc != RSTQ_OK ? rc : run_prompt(ctx, q, a);
}

int32_t rstq_paged_prompt_attention(rstq_ctx* ctx, rstq_buf* q, rstq_buf* kcache, rstq_buf* vcache, rstq_buf* out, rstq_buf* table,
                                    rstq_buf* cu_q, rstq_buf* lens, int64_t rows, int64_t seqs, int64_t n_q, int64_t group,
                                    int64_t n_kv, int64_t head_dim, int64_t page, int64_t n_pages, int64_t max_pages,
                                    int64_t ldq, double scale, int32_t causal, int32_t dtype) {
    PromptArgs a;
    RSTQ_REQUIRE(cu_q, RSTQ_E_INVALID, "null buffer: the rows' sequences");
    const int32_t rc = attention_args(ctx, q, kcache, vcache, out, table, cu_q, lens, rows, n_pages * page, seqs, n_q, group, n_kv, head_dim,
                                      page, n_pages, max_pages, ldq, 0, scale, causal, dtype, false, &a);
    return rc != RSTQ_OK ? rc : run_prompt(ctx, q, a);
}

}  // extern "C"
