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
// Bound by latency: slots, lengths and tables are three reads that depend on one another, the rest works in shared memory.
__global__ void __launch_bounds__(kThreads) prefix_plan_kernel(const cq_kv_cache cache, const Call call, const int *__restrict__ slots) {
    extern __shared__ int dyn[];
    __shared__ int sums[32], most;
    const State s = cq_kv::state_of(cache);
    const Shape &sh = call.sh;
    const Plan &pl = call.plan;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int t = sh.queries, hkv = sh.kv_heads, cap = s.max_pages * s.page, nq = sh.n_queries(), per = sh.per_kv();
    int *slot_of = dyn, *len_of = slot_of + sh.batch, *group_of = len_of + sh.batch;         // by sequence
    int *first_of = group_of + sh.batch, *count_of = first_of + sh.groups, *least_of = count_of + sh.groups;      // by group: of its sequences that
                                                                    // have a context for each query: the first, how many, pages that agree
    for (int g = tid; g < sh.groups; g += kThreads) { first_of[g] = INT32_MAX; count_of[g] = 0; least_of[g] = INT32_MAX; }
    if (tid == 0) most = 0;
    cq_pdl_launch_dependents();
    cq_pdl_wait();
    __syncthreads();
    for (int b = tid; b < sh.batch; b += kThreads) {
        const int slot = slots[b];
        const bool there = slot >= 0 && slot < s.max_seqs;
        const int len = there ? min(max(s.lens[slot], 0), cap) : -1, g = last_not_above(sh.groups, b * t, [&](int x) { return pl.shapes[x].query0; });
        if (!there) atomicCAS(s.header, cq_kv::kOk, cq_kv::kBadSlot);
        slot_of[b] = slot;
        len_of[b] = len;
        group_of[b] = g;
        if (len >= t) {
            atomicMin(&first_of[g], b);
            atomicAdd(&count_of[g], 1);
            atomicMin(&least_of[g], (len - t + 1) / s.page);
            atomicMax(&most, (len - t + 1) / s.page);
        }
    }
    __syncthreads();
    // a warp compares 128 entries of a sequence with those of its group's first one
    const int blocks = (most + 127) / 128;
    for (int u = warp; u < sh.batch * blocks; u += kThreads / 32) {
        const int b = u / blocks, j0 = u % blocks * 128 + lane, g = group_of[b];
        if (len_of[b] < t || count_of[g] < 2) continue;         // the whole warp
        const int n = (len_of[b] - t + 1) / s.page;
        const int *mine = s.tables + (size_t)slot_of[b] * s.max_pages, *first = s.tables + (size_t)slot_of[first_of[g]] * s.max_pages;
        int p[4], f[4], bad = INT32_MAX;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool in = j0 + 32 * i < n;
            p[i] = in ? mine[j0 + 32 * i] : 0;
            f[i] = in ? first[j0 + 32 * i] : 0;
        }
#pragma unroll
        for (int i = 3; i >= 0; --i)
            if (p[i] != f[i] || p[i] < 0 || p[i] >= s.pages) bad = j0 + 32 * i;
        bad = __reduce_min_sync(0xffffffffu, bad);
        if (lane == 0 && bad != INT32_MAX) atomicMin(&least_of[g], bad);
    }
    __syncthreads();
    // the shared line
    int line = 0;
    for (int g0 = 0; g0 < sh.groups; g0 += kThreads) {
        const int g = g0 + tid;
        Group gr{0, 0, 0, -1};
        int n = 0, all;
        if (g < sh.groups) {
            if (count_of[g] >= 2 && least_of[g] > 0) {
                gr.shared = least_of[g] * s.page;
                gr.slot = slot_of[first_of[g]];
                gr.units = (gr.shared + kKeyTile - 1) / kKeyTile;
            }
            n = gr.units * hkv * pl.shapes[g].row_tiles;
        }
        gr.start = line + scan_before(n, sums, all);
        if (g < sh.groups) {
            pl.groups[g] = gr;
            least_of[g] = gr.shared;
        }
        line += all;
    }
    __syncthreads();
    const int chunk = max((line + sh.ctas - 1) / sh.ctas, 1), shared_line = line;
    // the own line
    const int tiles = sh.own_tiles();
    line = 0;
    for (int i0 = 0; i0 < nq; i0 += kThreads) {
        const int i = i0 + tid;
        Query q{};
        int all;
        if (i < nq) {
            const int b = i / t, g = group_of[b], len = len_of[b], shared = len >= t ? least_of[g] : 0;
            const GroupShape gs = pl.shapes[g];
            q.len = len - t + 1 + i % t;
            q.group = shared ? g : -1;
            q.units = q.len > shared ? (q.len - shared + sh.own_step - 1) / sh.own_step : 0;
            q.query0 = gs.query0; q.item0 = gs.item0; q.row_tiles = gs.row_tiles;
        }
        q.start = line + scan_before(q.units * hkv * tiles, sums, all);
        if (i < nq) pl.query[i] = q;
        line += all;
    }
    const int own_chunk = max((line + sh.own_workers - 1) / sh.own_workers, 1);
    if (tid == 0) {
        pl.shared.header[0] = shared_line; pl.shared.header[1] = chunk;
        pl.own.header[0] = line; pl.own.header[1] = own_chunk;
    }
    __syncthreads();
    // segments of an item that starts at `start` of its line
    auto write = [&](const Line &l, int workers, int chunk, int item, int start, int units, int step, Segment seg, int key0, int key1, int64_t part0, int part_step,
                     int w_first, int w_step) {
        const int w0 = start / chunk, w1 = units ? (start + units - 1) / chunk : w0;
        if (w_first == 0) l.item[item] = units ? make_int2(w0, w1) : make_int2(1, 0);
        for (int w = w0 + w_first; w <= w1; w += w_step) {
            if (w >= workers) break;                    // an empty item at the very end of the line
            const int a = max(start, w * chunk), b = min(start + units, (w + 1) * chunk);
            seg.units = b - a;
            seg.key0 = key0 + (a - start) * step;
            seg.key1 = min(key1, key0 + (b - start) * step);
            seg.part = (int)(part0 + (int64_t)(item + w) * part_step);
            l.segments[item + w] = seg;
            if (units && w * chunk >= start) l.first[w] = item + w;
        }
    };
    for (int i = warp; i < call.shared_items; i += kThreads / 32) {
        const int g = last_not_above(sh.groups, i, [&](int x) { return pl.shapes[x].item0; });
        const GroupShape gs = pl.shapes[g];
        const Group gr = pl.groups[g];
        const int local = i - gs.item0, row0 = gs.query0 * per + local % gs.row_tiles * sh.row_tile;
        Segment seg{};
        seg.row0 = row0;
        seg.rows = min(sh.row_tile, pl.shapes[g + 1].query0 * per - row0);
        seg.head = local / gs.row_tiles;
        seg.slot = gr.slot;
        write(pl.shared, sh.ctas, chunk, i, gr.start + local * gr.units, gr.units, kKeyTile, seg, 0, gr.shared, part_shared(sh, 0), sh.row_tile, lane, 32);
    }
    for (int i = tid; i < sh.own_items(); i += kThreads) {
        const int tile = i % tiles, h = i / tiles % hkv, n = i / tiles / hkv;
        const Query q = pl.query[n];
        Segment seg{};
        seg.row0 = n * per + tile * sh.own_rows;
        seg.rows = min(sh.own_rows, per - tile * sh.own_rows);
        seg.head = h;
        seg.slot = slot_of[n / t];
        write(pl.own, sh.own_workers, own_chunk, i, q.start + (h * tiles + tile) * q.units, q.units, sh.own_step, seg, q.group >= 0 ? least_of[q.group] : 0, q.len,
              part_own(sh, call.shared_items, 0), sh.own_slot(), 0, 1);
    }
}

// One warp per row: lane x weighs segment x - those of the row's shared item, then those of its own one, in the order of their keys - and the
// outputs are added in that order.
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
    if (q.len > 0) {
        const int own_item = (n * sh.kv_heads + h) * sh.own_tiles() + in / sh.own_rows;
        const int2 own = pl.own.item[own_item];
        int2 shared = make_int2(1, 0);
        int64_t shared0 = 0;
        if (q.group >= 0) {
            const int r = (n - q.query0) * per + in, item = q.item0 + h * q.row_tiles + r / sh.row_tile;
            shared = pl.shared.item[item];
            shared0 = part_shared(sh, item + shared.x) + r % sh.row_tile;
        }
        const int n_shared = shared.y - shared.x + 1, n_all = n_shared + own.y - own.x + 1;
        const int64_t own0 = part_own(sh, call.shared_items, own_item + own.x) + in % sh.own_rows;
        for (int x0 = 0; x0 < n_all; x0 += 32) {
            const int x = x0 + lane, count = min(32, n_all - x0);
            const int part = (int)(x < n_shared ? shared0 + (int64_t)x * sh.row_tile : own0 + (int64_t)(x - n_shared) * sh.own_slot());
            const float2 ml = lane < count ? call.ml[part] : make_float2(-INFINITY, 0.0f);
            float big = fmaxf(m, ml.x);
#pragma unroll
            for (int k = 16; k > 0; k >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, k));
            // all scores so far -inf: no weight can be given, as in the formula (lanes without a segment have none)
            const float w = lane < count ? exp2f(ml.x - big) : 0.0f, f = x0 ? exp2f(m - big) : 0.0f;
            float sum = lane < count ? __fmul_rn(ml.y, w) : 0.0f;
#pragma unroll
            for (int k = 16; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
            l = x0 ? __fmaf_rn(l, f, sum) : sum;
            m = big;
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = x0 ? __fmul_rn(acc[i], f) : 0.0f;
#pragma unroll 4
            for (int y = 0; y < count; ++y) {
                const float wy = __shfl_sync(0xffffffffu, w, y);
                const float *o = call.o + (int64_t)__shfl_sync(0xffffffffu, part, y) * D + V * lane;
                float v[V];
                if constexpr (V == 4) *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(o);
                else *reinterpret_cast<float2 *>(v) = *reinterpret_cast<const float2 *>(o);
#pragma unroll
                for (int i = 0; i < V; ++i) acc[i] = __fmaf_rn(wy, v[i], acc[i]);
            }
        }
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
        else if ((int64_t)p->batch * p->queries * p->heads * ((int64_t)cache->max_pages * cache->page_size / 16 + 1) > INT32_MAX)
            why = "more than 2^35 (query head, key) pairs in one call";
    }
    if (why) {
        std::snprintf(msg, sizeof msg, "%s: %s", who, why);
        cq_set_status(status, msg);
        return false;
    }
    s = Shape{p->batch, p->queries, p->heads, cache->kv_heads, p->groups, cache->head_dim, cache->elem, 0, p->ctas, 0, 0, 0};
    if (cache->elem == CQ_F32) { s.row_tile = s.own_rows = 32; s.own_step = 64; s.own_workers = s.ctas; }
    else { s.row_tile = 128; s.own_rows = 16; s.own_step = 16; s.own_workers = s.ctas * kMmaWarps; }
    return true;
}
Call call_of(const cq_prefix_plan *p, const Shape &s) {
    Call c;
    c.sh = s;
    c.shared_items = p->shared_items;
    c.plan = plan_of(p->ints, s, p->shared_items);
    c.o = p->scratch;
    c.ml = reinterpret_cast<float2 *>(p->scratch + part_rows(s, p->shared_items) * s.head_dim);
    return c;
}
bool plan_ready(const cq_prefix_plan *p, const Shape &s, const char *who) {
    char msg[160];
    if (!p->ints || !p->scratch || (((uintptr_t)p->ints | (uintptr_t)p->scratch) & 31) || p->ctas <= 0 || p->shared_items <= 0 ||
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
    s.ctas = plan->ctas = 2 * cq_sm_count();
    s.own_workers = s.elem == CQ_F32 ? s.ctas : s.ctas * kMmaWarps;
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
    const size_t smem = 12 * ((size_t)s.batch + s.groups);
    if (smem > 48 * 1024) cudaFuncSetAttribute(prefix_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    cq_launch_k(prefix_plan_kernel, dim3(1), dim3(kThreads), smem, (cudaStream_t)stream, *cache, call_of(plan, s), slots);
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
