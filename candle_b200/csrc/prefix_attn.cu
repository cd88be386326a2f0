// Attention of a decode batch whose sequences share the pages of a prefix: the plan, the join, and the entry points.
// prefix_attn.cuh has the decomposition.
#include <cmath>
#include <cstdio>

#include "prefix_attn.cuh"

namespace {
using namespace cq_attn;
using cq_kv::State;

constexpr int kThreads = 1024;

__device__ __forceinline__ int scan_before(int v, int *sums, int &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, m);
        if (lane >= m) x += y;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    int w = sums[lane];
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, w, m);
        if (lane >= m) w += y;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    const int before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
    return x - v + (warp ? before : 0);
}
// Index of the last entry of an ascending column that is not above `v`.
template <typename F> __device__ __forceinline__ int last_not_above(int n, int v, F column) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (column(mid) <= v) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// One CTA.  The pages that a group shares are found by comparing the tables, so a plan cannot be wrong about them: the leading
// entries that agree in all its sequences, as far as the shortest context among its queries fills pages.
__global__ void __launch_bounds__(kThreads) prefix_plan_kernel(const cq_kv_cache cache, const Call call, const int *__restrict__ slots) {
    __shared__ int sums[32];
    const State s = cq_kv::state_of(cache);
    const Shape &sh = call.sh;
    const Plan &pl = call.plan;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int t = sh.queries, hkv = sh.kv_heads, cap = s.max_pages * s.page, nq = sh.n_queries(), shared_items = call.items_shared;
    cq_pdl_wait();
    // groups: [start] first sequence with a context for each query, [tiles] how many of them, [shared] pages, as minima and counts
    for (int g = tid; g < sh.groups; g += kThreads) pl.groups[g] = Group{INT32_MAX, 0, INT32_MAX, -1};
    __syncthreads();
    auto length = [&](int b) {          // -1: no such slot
        const int slot = slots[b];
        return slot >= 0 && slot < s.max_seqs ? min(max(s.lens[slot], 0), cap) : -1;
    };
    auto group_of = [&](int b) { return last_not_above(sh.groups, b * t, [&](int g) { return pl.shapes[g].query0; }); };
    for (int b = tid; b < sh.batch; b += kThreads) {
        const int len = length(b), g = group_of(b);
        if (len < 0) atomicCAS(s.header, cq_kv::kOk, cq_kv::kBadSlot);
        pl.query[b * t] = Query{0, 0, len, g};
        if (len >= t) {
            atomicMin(&pl.groups[g].start, b);
            atomicAdd(&pl.groups[g].tiles, 1);
        }
    }
    __syncthreads();
    for (int b = warp; b < sh.batch; b += kThreads / 32) {
        const int len = pl.query[b * t].len, g = pl.query[b * t].group;
        const Group gr = pl.groups[g];
        if (len < t || gr.tiles < 2) continue;          // the whole warp
        const int *mine = s.tables + (size_t)slots[b] * s.max_pages, *first = s.tables + (size_t)slots[gr.start] * s.max_pages;
        int n = (len - t + 1) / s.page;
        for (int j0 = 0; j0 < n; j0 += 128) {
            int bad = INT32_MAX;
#pragma unroll
            for (int i = 3; i >= 0; --i) {
                const int j = j0 + 32 * i + lane;
                if (j < n) {
                    const int p = mine[j];
                    if (p != first[j] || p < 0 || p >= s.pages) bad = j;
                }
            }
            bad = __reduce_min_sync(0xffffffffu, bad);
            if (bad != INT32_MAX) { n = bad; break; }
        }
        if (lane == 0) atomicMin(&pl.groups[g].shared, n);
    }
    __syncthreads();
    int line = 0;
    for (int g0 = 0; g0 < sh.groups; g0 += kThreads) {
        const int g = g0 + tid;
        Group gr{0, 0, 0, -1};
        int n = 0, all;
        if (g < sh.groups) {
            const Group was = pl.groups[g];
            if (was.tiles >= 2 && was.shared > 0) {
                gr.shared = was.shared * s.page;
                gr.slot = slots[was.start];
                gr.tiles = (gr.shared + kKeyTile - 1) / kKeyTile;
            }
            n = gr.tiles * hkv * pl.shapes[g].row_tiles;
        }
        gr.start = line + scan_before(n, sums, all);
        if (g < sh.groups) pl.groups[g] = gr;
        line += all;
    }
    __syncthreads();
    // queries, the last of a sequence first: entry 0 of a sequence still holds its length and group
    for (int b = tid; b < sh.batch; b += kThreads) {
        const int len = pl.query[b * t].len, g = pl.query[b * t].group;
        const int shared = len >= t ? pl.groups[g].shared : 0;
        for (int i = t - 1; i >= 0; --i) {
            const int n = len - t + 1 + i;
            pl.query[b * t + i] = Query{0, n > shared ? (n - shared + kKeyTile - 1) / kKeyTile : 0, n, shared ? g : -1};
        }
    }
    __syncthreads();
    for (int i0 = 0; i0 < nq; i0 += kThreads) {
        const int i = i0 + tid;
        int all;
        const int start = line + scan_before(i < nq ? pl.query[i].tiles * hkv : 0, sums, all);
        if (i < nq) pl.query[i].start = start;
        line += all;
    }
    const int chunk = max((line + sh.ctas - 1) / sh.ctas, 1);
    if (tid == 0) { pl.header[0] = line; pl.header[1] = chunk; }
    __syncthreads();
    // segments of an item that starts at `start` of the line
    auto write = [&](int item, int start, int tiles, Segment seg, int key0, int key1, int c_first, int c_step) {
        const int c0 = start / chunk, c1 = tiles ? (start + tiles - 1) / chunk : c0;
        if (c_first == 0) pl.item[item] = tiles ? make_int2(c0, c1) : make_int2(1, 0);
        for (int c = c0 + c_first; c <= c1; c += c_step) {
            if (c >= sh.ctas) break;                    // an empty item at the very end of the line
            const int a = max(start, c * chunk), b = min(start + tiles, (c + 1) * chunk);
            seg.tiles = b - a;
            seg.key0 = key0 + (a - start) * kKeyTile;
            seg.key1 = min(key1, key0 + (b - start) * kKeyTile);
            seg.part = (int)part_of(sh, shared_items, item, c);
            pl.segments[item + c] = seg;
            if (tiles && c * chunk >= start) pl.first[c] = item + c;
        }
    };
    const int per = sh.per_kv();
    for (int i = warp; i < shared_items; i += kThreads / 32) {
        const int g = last_not_above(sh.groups, i, [&](int x) { return pl.shapes[x].item0; });
        const GroupShape gs = pl.shapes[g];
        const Group gr = pl.groups[g];
        const int local = i - gs.item0, tile = local % gs.row_tiles, row0 = gs.query0 * per + tile * sh.row_tile;
        Segment seg{};
        seg.row0 = row0;
        seg.rows = min(sh.row_tile, pl.shapes[g + 1].query0 * per - row0);
        seg.head = local / gs.row_tiles;
        seg.slot = gr.slot;
        write(i, gr.start + local * gr.tiles, gr.tiles, seg, 0, gr.shared, lane, 32);
    }
    for (int i = tid; i < nq * hkv; i += kThreads) {
        const int n = i / hkv, h = i % hkv;
        const Query q = pl.query[n];
        Segment seg{};
        seg.row0 = n * per;
        seg.rows = per;
        seg.head = h;
        seg.slot = slots[n / t];
        write(shared_items + i, q.start + h * q.tiles, q.tiles, seg, q.group >= 0 ? pl.groups[q.group].shared : 0, q.len, 0, 1);
    }
}

// One warp per row: its shared item's segments, then its own item's, in the order of their keys.
template <typename T> struct Two { T x, y; };
template <typename T, int D> __global__ void __launch_bounds__(256) prefix_join_kernel(const Call call, T *__restrict__ out) {
    const Shape &sh = call.sh;
    const Plan &pl = call.plan;
    cq_pdl_launch_dependents();
    cq_pdl_wait();
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, per = sh.per_kv();
    if (row >= (int64_t)sh.n_queries() * sh.heads) return;
    const int n = (int)(row / sh.heads), hq = (int)(row % sh.heads), h = hq / per, in = hq % per;
    const Query q = pl.query[n];
    constexpr int V = D / 32;
    float acc[V] = {}, m = -INFINITY, l = 0.0f;
    auto add = [&](int64_t part) {
        const float2 ml = call.ml[part];
        const float big = fmaxf(m, ml.x);
        // two maxima of -inf: no score so far, nothing to scale
        const float a = m == big ? 1.0f : exp2f(m - big), b = ml.x == big ? 1.0f : exp2f(ml.x - big);
        l = __fmaf_rn(l, a, __fmul_rn(ml.y, b));
        const float *o = call.o + part * D + V * lane;
        float v[V];
        if constexpr (V == 4) *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(o);
        else *reinterpret_cast<float2 *>(v) = *reinterpret_cast<const float2 *>(o);
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = __fmaf_rn(acc[i], a, __fmul_rn(v[i], b));
        m = big;
    };
    if (q.len > 0) {
        if (q.group >= 0) {
            const GroupShape gs = pl.shapes[q.group];
            const int r = (n - gs.query0) * per + in, item = gs.item0 + h * gs.row_tiles + r / sh.row_tile;
            const int2 c = pl.item[item];
            for (int x = c.x; x <= c.y; ++x) add(part_of(sh, call.items_shared, item, x) + r % sh.row_tile);
        }
        const int item = call.items_shared + n * sh.kv_heads + h;
        const int2 c = pl.item[item];
        for (int x = c.x; x <= c.y; ++x) add(part_of(sh, call.items_shared, item, x) + in);
    }
    T *to = out + row * D + V * lane;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float r = q.len > 0 ? __fdiv_rn(acc[i], l) : 0.0f;        // no key: zeros
        if constexpr (sizeof(T) == 4) to[i] = r;
        else if constexpr (std::is_same<T, __half>::value) to[i] = __float2half_rn(r);
        else to[i] = __float2bfloat16_rn(r);
    }
}

template <int D> void join_launch(const Call &c, void *out, cudaStream_t st) {
    const dim3 grid((unsigned)(((int64_t)c.sh.n_queries() * c.sh.heads + 7) / 8));
    if (c.sh.elem == CQ_F32) cq_launch_k(prefix_join_kernel<float, D>, grid, dim3(256), 0, st, c, (float *)out);
    else if (c.sh.elem == CQ_F16) cq_launch_k(prefix_join_kernel<__half, D>, grid, dim3(256), 0, st, c, (__half *)out);
    else cq_launch_k(prefix_join_kernel<__nv_bfloat16, D>, grid, dim3(256), 0, st, c, (__nv_bfloat16 *)out);
}

bool shape_ok(const cq_kv_cache *cache, const cq_prefix_plan *p, const char *who, Shape &s) {
    if (!cq_kv::cache_ok(cache, who)) return false;
    char msg[160];
    const char *why = nullptr;
    int status = CQ_ERR_BAD_ARG;
    if (!p) why = "null plan";
    else if (p->batch <= 0 || p->queries <= 0 || p->heads <= 0 || p->heads % cache->kv_heads) why = "batch, queries, heads must be positive, heads a multiple of kv_heads";
    else if (p->groups <= 0 || p->groups > p->batch) why = "between one group and one per sequence";
    else {
        status = CQ_ERR_UNSUPPORTED;
        if ((int64_t)p->batch * p->queries > 4096) why = "at most 4096 queries (batch * queries)";
        else if (p->heads / cache->kv_heads > 32) why = "at most 32 query heads per KV head";
        else if ((int64_t)p->batch * p->queries * p->heads * ((int64_t)cache->max_pages * cache->page_size / kKeyTile + 1) > INT32_MAX)
            why = "too many (query, key) tiles for one call";
    }
    if (why) {
        std::snprintf(msg, sizeof msg, "%s: %s", who, why);
        cq_set_status(status, msg);
        return false;
    }
    s = Shape{p->batch, p->queries, p->heads, cache->kv_heads, p->groups, cache->head_dim, cache->elem, p->row_tile, p->ctas};
    return true;
}
Call call_of(const cq_prefix_plan *p, const Shape &s) {
    Call c;
    c.sh = s;
    c.items_shared = p->shared_items;
    c.plan = plan_of(p->ints, s, p->shared_items);
    c.o = p->scratch;
    c.ml = reinterpret_cast<float2 *>(p->scratch + part_rows(s, p->shared_items) * s.head_dim);
    return c;
}
bool plan_ready(const cq_prefix_plan *p, const Shape &s, const char *who) {
    char msg[160];
    if (!p->ints || !p->scratch || (((uintptr_t)p->ints | (uintptr_t)p->scratch) & 31) || p->row_tile <= 0 || p->ctas <= 0 || p->shared_items <= 0 ||
        p->n_ints != plan_ints(s, p->shared_items) || p->n_floats != part_rows(s, p->shared_items) * (s.head_dim + 2)) {
        std::snprintf(msg, sizeof msg, "%s: the plan is not one that cq_prefix_plan_shape has filled for this cache, or its memory is missing", who);
        cq_set_status(CQ_ERR_BAD_ARG, msg);
        return false;
    }
    return true;
}

}  // namespace

extern "C" int cq_prefix_plan_shape(const cq_kv_cache *cache, cq_prefix_plan *plan, const int *group_sizes, int *shapes) {
    Shape s;
    if (!shape_ok(cache, plan, "prefix_plan_shape", s)) return 1;
    s.row_tile = plan->row_tile = s.elem == CQ_F32 ? 32 : 128;
    s.ctas = plan->ctas = 2 * cq_sm_count();
    int64_t items = 0, seqs = 0;
    for (int g = 0; g < plan->groups; ++g) {
        const int n = group_sizes ? group_sizes[g] : plan->groups == 1 ? plan->batch : 1;
        if (n <= 0) { cq_set_status(CQ_ERR_BAD_ARG, "prefix_plan_shape: a group without sequences"); return 1; }
        const int64_t tiles = ((int64_t)n * s.queries * s.per_kv() + s.row_tile - 1) / s.row_tile;
        if (shapes) { shapes[3 * g] = (int)(seqs * s.queries); shapes[3 * g + 1] = (int)items; shapes[3 * g + 2] = (int)tiles; }
        items += tiles * s.kv_heads;
        seqs += n;
    }
    if (seqs != plan->batch) { cq_set_status(CQ_ERR_BAD_ARG, "prefix_plan_shape: the groups' sizes do not add up to the batch"); return 1; }
    if (shapes) { shapes[3 * plan->groups] = (int)(seqs * s.queries); shapes[3 * plan->groups + 1] = (int)items; shapes[3 * plan->groups + 2] = 0; }
    plan->shared_items = (int)items;
    plan->n_ints = plan_ints(s, items);
    plan->n_floats = part_rows(s, items) * (s.head_dim + 2);
    return 0;
}

extern "C" void cq_prefix_plan_update(const cq_kv_cache *cache, const cq_prefix_plan *plan, const int *slots, void *stream) {
    Shape s;
    if (!shape_ok(cache, plan, "prefix_plan_update", s) || !plan_ready(plan, s, "prefix_plan_update")) return;
    if (!slots) { cq_set_status(CQ_ERR_BAD_ARG, "prefix_plan_update: null slots"); return; }
    cq_launch_k(prefix_plan_kernel, dim3(1), dim3(kThreads), 0, (cudaStream_t)stream, *cache, call_of(plan, s), slots);
    cq_check_launch("prefix_plan_update");
}

extern "C" void cq_prefix_attention(const cq_kv_cache *cache, int layer, const cq_prefix_plan *plan, const void *q, int64_t q_stride, void *out, float scale,
                                    void *stream) {
    Shape s;
    if (!shape_ok(cache, plan, "prefix_attention", s) || !plan_ready(plan, s, "prefix_attention")) return;
    if (!q || !out || layer < 0 || layer >= cache->layers || q_stride < (int64_t)s.heads * s.head_dim || q_stride * cq_kv::elem_bytes(s.elem) % 16 ||
        (((uintptr_t)q | (uintptr_t)out) & 15) || !(scale > 0.0f) || std::isinf(scale)) {
        cq_set_status(CQ_ERR_BAD_ARG, "prefix_attention: null pointer, layer out of range, rows not 16-byte aligned, or a scale that is not positive");
        return;
    }
    const Call c = call_of(plan, s);
    cudaStream_t st = (cudaStream_t)stream;
    if (s.elem == CQ_F32) simt_launch(c, *cache, layer, q, q_stride, scale, st);
    else if (!mma_launch(c, *cache, layer, q, q_stride, scale, st)) return;
    if (s.head_dim == 128) join_launch<128>(c, out, st);
    else join_launch<64>(c, out, st);
    cq_check_launch("prefix_attention");
}
