// Attention of a decode batch whose sequences share the pages of a prefix: the plan, the join, and the entry points.
// prefix_attn.cuh has the decomposition.
#include <cmath>
#include <cstdio>

#include "prefix_attn.cuh"

namespace {
using namespace cq_attn;
using cq_kv::State;

constexpr int kThreads = 256, kPlanCtas = 8;

// Units per worker of the own line.  f16 and bf16: the four warps of a CTA that have nothing else, and the eight that come when its `units` shared ones are done.  In clocks
// of a B200 SM: a shared unit takes 4,300 and the first of them 5,000 more, one of the four warps takes some 1,700 a step beside them, and twelve warps together are bound by
// HBM with 400 a step.  All finish together by that; a model that is off by a third leaves the one kind of warps idle for a tenth of the time.  (Measured with heads of 128; those of
// 64 have the same division.)
__device__ __forceinline__ void own_chunks(const Shape &s, int units, int line, int &chunk, int &chunk2) {
    chunk2 = 1;
    if (s.own_first == s.own_workers) { chunk = max((line + s.own_workers - 1) / s.own_workers, 1); return; }
    const int per_cta = (line + s.ctas - 1) / s.ctas;
    const int beside = units ? (int)min(((int64_t)units * 4300 + 5000) / 1700, (int64_t)per_cta) : 0;          // steps a warp does in that time
    const int rest = per_cta - kMmaWarps * beside;
    if (rest <= 0) { chunk = max((per_cta + kMmaWarps - 1) / kMmaWarps, 1); return; }
    const int share = (rest + kMmaWarps + kMmaHelpers - 1) / (kMmaWarps + kMmaHelpers);
    chunk = beside + share;
    chunk2 = share;
}

// Sum of `v` over the threads before this one, two counts in one 64-bit word; `total` over all.
__device__ __forceinline__ uint64_t scan_before(uint64_t v, uint64_t *sums, uint64_t &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint64_t x = v;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, x, m);
        if (lane >= m) x += y;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    uint64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w == warp) before = total;
        total += sums[w];
    }
    return before + x - v;
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

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// One cluster.  The pages that a group shares are found by comparing the tables, so a plan cannot be wrong about them: the leading
// entries that agree in all its sequences, as far as the shortest context among its queries fills pages.
// Bound by latency: slots, lengths and tables are three reads that depend on one another, and a warp by itself takes some five clocks an instruction.
// So the comparison and the records are divided over the CTAs, everything else each does for itself, and divisions are kept out of the way (one CTA of 1024 threads
// took 16 - 33 us for 64 - 128 sequences).  In a graph: 5.4 us for 8 sequences of 8 pages, 6.6 for 64 of 143, 7.9 for 128 of 264.
__global__ void __launch_bounds__(kThreads) prefix_plan_kernel(const cq_kv_cache cache, const Call call, const int *slots) {
    extern __shared__ int dyn[];
    __shared__ uint64_t sums[kThreads / 32];
    __shared__ int most;
    const State s = cq_kv::state_of(cache);
    const Shape &sh = call.sh;
    const Plan &pl = call.plan;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)blockIdx.x, shift = 31 - __clz(s.page);
    const int t = sh.queries, hkv = sh.kv_heads, cap = s.max_pages * s.page, nq = sh.n_queries();
    int *slot_of = dyn, *len_of = slot_of + sh.batch, *group_of = len_of + sh.batch;         // by sequence
    int *first_of = group_of + sh.batch, *count_of = first_of + sh.groups, *least_of = count_of + sh.groups;      // by group: of its sequences that
                                                                    // have a context for each query: the first, how many, pages that agree
    int *group_start = least_of + sh.groups, *start_of = group_start + sh.groups, *units_of = start_of + nq;      // first units; by query
    for (int g = tid; g < sh.groups; g += kThreads) { first_of[g] = INT32_MAX; count_of[g] = 0; least_of[g] = INT32_MAX; }
    if (tid == 0) most = 0;
    __syncwarp();
    cluster_arrive();                       // the others may write this CTA's least_of
    cq_pdl_launch_dependents();
    cq_pdl_wait();
    __syncthreads();
    for (int b = tid; b < sh.batch; b += kThreads) {
        const int slot = slots[b];
        const bool there = slot >= 0 && slot < s.max_seqs;
        const int len = there ? min(max(s.lens[slot], 0), cap) : -1;
        const int g = sh.groups == 1 ? 0 : last_not_above(sh.groups, b * t, [&](int x) { return pl.shapes[x].query0; });
        if (!there) atomicCAS(s.header, cq_kv::kOk, cq_kv::kBadSlot);
        slot_of[b] = slot;
        len_of[b] = len;
        group_of[b] = g;
        if (len >= t) {
            atomicMin(&first_of[g], b);
            atomicAdd(&count_of[g], 1);
            atomicMin(&least_of[g], (len - t + 1) >> shift);
            atomicMax(&most, (len - t + 1) >> shift);
        }
    }
    __syncthreads();
    cluster_wait();
    // a warp compares 128 entries of a sequence with those of its group's first one
    for (int j0 = 0; j0 < most; j0 += 128)
#pragma unroll 1
        for (int b = rank * (kThreads / 32) + warp; b < sh.batch; b += kPlanCtas * (kThreads / 32)) {
            const int g = group_of[b], n = (len_of[b] - t + 1) >> shift, from = first_of[g];
            if (len_of[b] < t || b == from || j0 >= n) continue;        // the whole warp
            const int *mine = s.tables + (size_t)slot_of[b] * s.max_pages + j0 + lane, *first = s.tables + (size_t)slot_of[from] * s.max_pages + j0 + lane;
            int p[4], f[4], bad = INT32_MAX;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool in = j0 + 32 * i + lane < n;
                p[i] = in ? mine[32 * i] : 0;
                f[i] = in ? first[32 * i] : 0;
            }
#pragma unroll
            for (int i = 3; i >= 0; --i)
                if (p[i] != f[i] || (unsigned)p[i] >= (unsigned)s.pages) bad = j0 + 32 * i + lane;
            bad = __reduce_min_sync(0xffffffffu, bad);
            if (bad != INT32_MAX && lane < kPlanCtas) {
                uint32_t at;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(cq_smem_u32(&least_of[g])), "r"(lane));
                asm volatile("red.relaxed.cluster.shared::cluster.min.s32 [%0], %1;" ::"r"(at), "r"(bad) : "memory");
            }
        }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    auto shared_of = [&](int g) { return count_of[g] >= 2 ? least_of[g] << shift : 0; };       // positions
    // both lines at once: the units of group i, and of query i
    uint64_t before = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < max(nq, sh.groups); i0 += kThreads) {
        const int i = i0 + tid;
        int n_shared = 0, units = 0;
        if (i < sh.groups) n_shared = ((shared_of(i) + sh.tile - 1) / sh.tile) * hkv * pl.shapes[i].row_tiles;
        if (i < nq) {
            const int b = t == 1 ? i : i / t, len = len_of[b], shared = len >= t ? shared_of(group_of[b]) : 0, n = len - t + 1 + (i - b * t);
            units = n > shared ? (n - shared + (1 << sh.own_shift) - 1) >> sh.own_shift : 0;
        }
        uint64_t all;
        const uint64_t at = before + scan_before((uint64_t)n_shared << 32 | (unsigned)(units * hkv * sh.own_tiles), sums, all);
        if (i < sh.groups) group_start[i] = (int)(at >> 32);
        if (i < nq) { start_of[i] = (int)(uint32_t)at; units_of[i] = units; }
        before += all;
    }
    __syncthreads();
    const int shared_line = (int)(before >> 32), own_line = (int)(uint32_t)before;
    const int chunk = max((shared_line + sh.ctas - 1) / sh.ctas, 1);
    int own_chunk, own_chunk2;
    own_chunks(sh, shared_line ? chunk : 0, own_line, own_chunk, own_chunk2);
    auto group_at = [&](int g) {
        const GroupShape gs = pl.shapes[g];
        const int shared = shared_of(g);
        return Group{(shared + sh.tile - 1) / sh.tile, shared, count_of[g] ? slot_of[first_of[g]] : -1, group_start[g], gs.query0, gs.rows, gs.item0, gs.row_tiles};
    };
    // records, dealt out one a CTA: of the workers, the queries, the groups
    const int workers = sh.ctas + sh.own_workers;
#pragma unroll 1
    for (int i = tid * kPlanCtas + rank; i < workers + nq + sh.groups; i += kPlanCtas * kThreads) {
        if (i < workers) {
            const bool own = i >= sh.ctas;
            const int w = own ? i - sh.ctas : i, later = w - sh.own_first;
            const int u = !own ? w * chunk : later < 0 ? w * own_chunk : sh.own_first * own_chunk + later * own_chunk2;
            Start st{};
            st.left = own ? min(own_line - u, later < 0 ? own_chunk : own_chunk2) : min(shared_line - u, chunk);
            if (st.left > 0) {
                // the last group (query) that begins here or before; those without units begin where the next one does
                const int *starts = own ? start_of : group_start;
                const int x = last_not_above(own ? nq : sh.groups, u, [&](int y) { return starts[y]; });
                int units, tiles;
                st.index = x;
                if (own) {
                    const int b = t == 1 ? x : x / t, len = len_of[b];
                    units = units_of[x];
                    tiles = sh.own_tiles;
                    st.copy[0] = len - t + 1 + (x - b * t);
                    st.copy[1] = slot_of[b];
                    st.copy[2] = len >= t ? shared_of(group_of[b]) : 0;
                    st.copy[3] = units;
                } else {
                    const Group g = group_at(x);
                    units = g.units;
                    tiles = g.row_tiles;
                    st.copy[0] = g.units; st.copy[1] = g.shared; st.copy[2] = g.slot; st.copy[3] = g.start;
                    st.copy[4] = g.query0; st.copy[5] = g.rows; st.copy[6] = g.item0; st.copy[7] = g.row_tiles;
                }
                const int local = (u - starts[x]) / units;
                st.unit = u - starts[x] - local * units;
                st.head = tiles == 1 ? local : local / tiles;
                st.tile = local - st.head * tiles;
            }
            (own ? pl.own : pl.shared)[w] = st;
        } else if (i < workers + nq) {
            const int x = i - workers, b = t == 1 ? x : x / t, len = len_of[b];
            Query q{};
            q.len = len - t + 1 + (x - b * t);
            q.slot = slot_of[b];
            q.units = units_of[x];
            q.start = start_of[x];
            if (len >= t && shared_of(group_of[b])) {
                const Group g = group_at(group_of[b]);
                q.shared = g.shared;
                q.group_start = g.start; q.group_units = g.units; q.query0 = g.query0; q.item0 = g.item0; q.row_tiles = g.row_tiles;
            }
            pl.query[x] = q;
        } else pl.groups[i - workers - nq] = group_at(i - workers - nq);
    }
    if (rank == 0 && tid == 0) { pl.header[0] = shared_line; pl.header[1] = chunk; pl.header[2] = own_line; pl.header[3] = own_chunk; pl.header[4] = own_chunk2; }
}

// W warps per row, each with a share of its segments: lane x weighs segment x of 32 - those of the row's shared item, then those of its own one, in the order of their keys - and the
// outputs are added in that order.
template <typename T, int D, int W> __global__ void __launch_bounds__(256) prefix_join_kernel(const Call call, T *out) {
    __shared__ __align__(16) float all_acc[W > 1 ? W : 1][W > 1 ? D : 4];
    __shared__ float2 all_ml[W];
    const Shape &sh = call.sh;
    const Plan &pl = call.plan;
    cq_pdl_launch_dependents();
    cq_pdl_wait();
    const int lane = threadIdx.x & 31, per = sh.per_kv, n = blockIdx.y, warp = threadIdx.x >> 5, hq = W > 1 ? blockIdx.x : blockIdx.x * 8 + warp;
    if (hq >= sh.heads) return;
    const int h = div_per(hq, sh), in = hq - h * per, tile = in / sh.own_rows;
    const int64_t row = (int64_t)n * sh.heads + hq;
    const Query q = pl.query[n];
    const int chunk = pl.header[1], own_chunk = pl.header[3], own_chunk2 = pl.header[4];
    constexpr int V = D / 32;
    float acc[V] = {}, m = -INFINITY, l = 0.0f;
    if (q.len > 0) {
        // segments of an item: its units [start, start + units) of the line, cut at multiples of the chunk
        const int local = h * sh.own_tiles + tile, own_item = n * sh.kv_heads * sh.own_tiles + local;
        const int own_start = q.start + local * q.units, own_w = own_worker(sh, own_start, own_chunk, own_chunk2);
        const int n_own = q.units ? own_worker(sh, own_start + q.units - 1, own_chunk, own_chunk2) - own_w + 1 : 0;
        int n_shared = 0;
        int64_t shared0 = 0;
        if (q.shared) {
            const int r = (n - q.query0) * per + in, local = h * q.row_tiles + r / sh.row_tile, start = q.group_start + local * q.group_units, w = start / chunk;
            n_shared = (start + q.group_units - 1) / chunk - w + 1;
            shared0 = part_shared(sh, q.item0 + local + w) + r % sh.row_tile;
        }
        const int n_all = n_shared + n_own;
        const int64_t own0 = part_own(sh, call.shared_items, own_item + own_w) + in - tile * sh.own_rows;
        const int share = (n_all + W - 1) / W, begin = W > 1 ? warp * share : 0, end = W > 1 ? min(n_all, begin + share) : n_all;
        for (int x0 = begin; x0 < end; x0 += 32) {
            const bool more = x0 > begin;
            const int x = x0 + lane, count = min(32, end - x0);
            const int part = (int)(x < n_shared ? shared0 + (int64_t)x * sh.row_tile : own0 + (int64_t)(x - n_shared) * sh.own_slot());
            const float2 ml = lane < count ? call.ml[part] : make_float2(-INFINITY, 0.0f);
            // four outputs at a time on their way, the first of them beside the maxima
            float v[4][V];
            auto fetch = [&](int y0) {
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const float *o = call.o + (int64_t)__shfl_sync(0xffffffffu, part, (y0 + y) & 31) * D + V * lane;
                    if (y0 + y < count) {
                        if constexpr (V == 4) *reinterpret_cast<float4 *>(v[y]) = *reinterpret_cast<const float4 *>(o);
                        else *reinterpret_cast<float2 *>(v[y]) = *reinterpret_cast<const float2 *>(o);
                    }
                }
            };
            fetch(0);
            float big = fmaxf(m, ml.x);
#pragma unroll
            for (int k = 16; k > 0; k >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, k));
            // all scores so far -inf: no weight yet, relative to anything finite; where it stays so the quotient of the sums is 0 / 0, a NaN as in the formula
            const float base = big == -INFINITY ? 0.0f : big;
            const float w = lane < count ? exp2f(ml.x - base) : 0.0f, f = more ? exp2f(m - base) : 0.0f;
            float sum = lane < count ? __fmul_rn(ml.y, w) : 0.0f;
#pragma unroll
            for (int k = 16; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
            l = more ? __fmaf_rn(l, f, sum) : sum;
            m = big;
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = more ? __fmul_rn(acc[i], f) : 0.0f;
            for (int y0 = 0; y0 < count; y0 += 4) {
                if (y0) fetch(y0);
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const float wy = __shfl_sync(0xffffffffu, w, (y0 + y) & 31);
                    if (y0 + y < count)
#pragma unroll
                        for (int i = 0; i < V; ++i) acc[i] = __fmaf_rn(wy, v[y][i], acc[i]);
                }
            }
        }
    }
    if constexpr (W > 1) {                  // the warps' shares, in their order
        if (lane == 0) all_ml[warp] = make_float2(m, l);            // a share without segments: -inf, no weight
#pragma unroll
        for (int i = 0; i < V; ++i) all_acc[warp][V * lane + i] = acc[i];
        __syncthreads();
        if (warp) return;
        m = -INFINITY;
#pragma unroll
        for (int w = 0; w < W; ++w) m = fmaxf(m, all_ml[w].x);
        const float base = m == -INFINITY ? 0.0f : m;
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float2 ml = all_ml[w];
            const float f = exp2f(ml.x - base);
            l = __fmaf_rn(f, ml.y, l);
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = __fmaf_rn(f, all_acc[w][V * lane + i], acc[i]);
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

template <int D, int W> void join_launch(const Call &c, void *out, cudaStream_t st) {
    const dim3 grid((unsigned)(W > 1 ? c.sh.heads : (c.sh.heads + 7) / 8), (unsigned)c.sh.n_queries()), threads(W > 1 ? 32 * W : 256);
    if (c.sh.elem == CQ_F32) cq_launch_k(prefix_join_kernel<float, D, W>, grid, threads, 0, st, c, (float *)out);
    else if (c.sh.elem == CQ_F16) cq_launch_k(prefix_join_kernel<__half, D, W>, grid, threads, 0, st, c, (__half *)out);
    else cq_launch_k(prefix_join_kernel<__nv_bfloat16, D, W>, grid, threads, 0, st, c, (__nv_bfloat16 *)out);
}
// Few rows have many segments, a hundred and more where one sequence's keys are divided over the whole device: several warps a row where all of them are on the
// device at once, 64 an SM.  With plan and attention, in us: 32 rows of 4,000 keys 42 with one warp a row, 18 with eight; 2,048 rows of 8,700 keys 56.6, with two 53.9; but 3,200
// rows of 300 keys 20.7, with two 22.4, which is where two stop.
template <int D> void join_launch(const Call &c, void *out, cudaStream_t st) {
    const int rows = c.sh.n_queries() * c.sh.heads, warps = 64 * cq_sm_count();
    if (rows * 8 <= warps) join_launch<D, 8>(c, out, st);
    else if (rows * 3 <= warps) join_launch<D, 2>(c, out, st);
    else join_launch<D, 1>(c, out, st);
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
        else if ((int64_t)p->batch * p->queries * p->heads * ((int64_t)cache->max_pages * cache->page_size / 16 + 1) > (1 << 30))
            why = "more than 2^34 (query head, key) pairs in one call";
    }
    if (why) {
        std::snprintf(msg, sizeof msg, "%s: %s", who, why);
        cq_set_status(status, msg);
        return false;
    }
    s = Shape{p->batch, p->queries, p->heads, cache->kv_heads, p->groups, cache->head_dim, cache->elem, p->heads / cache->kv_heads};
    s.ctas = p->ctas;
    s.own_rows = 8;
    s.own_shift = 4;
    if (cache->elem == CQ_F32) { s.row_tile = 8; s.tile = 16; s.own_workers = s.own_first = s.ctas; }
    else { s.row_tile = 256; s.tile = 128; s.own_first = s.ctas * kMmaWarps; s.own_workers = s.own_first + s.ctas * kMmaHelpers; }
    s.own_tiles = (s.per_kv + s.own_rows - 1) / s.own_rows;
    if (s.per_kv > 1) s.rcp = (unsigned)(((1ull << 32) + s.per_kv - 1) / s.per_kv);
    return true;
}
Call call_of(const cq_prefix_plan *p, const Shape &s) {
    Call c;
    c.sh = s;
    c.shared_items = p->shared_items;
    c.plan = plan_of(p->ints, s);
    c.o = p->scratch;
    c.ml = reinterpret_cast<float2 *>(p->scratch + part_rows(s, p->shared_items) * s.head_dim);
    return c;
}
bool plan_ready(const cq_prefix_plan *p, const Shape &s, const char *who) {
    char msg[160];
    if (!p->ints || !p->scratch || (((uintptr_t)p->ints | (uintptr_t)p->scratch) & 63) || p->ctas <= 0 || p->shared_items <= 0 ||
        p->n_ints != plan_ints(s) || p->n_floats != part_rows(s, p->shared_items) * (s.head_dim + 2)) {
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
    s.ctas = plan->ctas = (s.elem == CQ_F32 ? f32_warps(s.head_dim) : 1) * cq_sm_count();
    s.own_first = s.elem == CQ_F32 ? s.ctas : s.ctas * kMmaWarps;
    s.own_workers = s.own_first + (s.elem == CQ_F32 ? 0 : s.ctas * kMmaHelpers);
    int64_t items = 0, seqs = 0;
    for (int g = 0; g < plan->groups; ++g) {
        const int n = group_sizes ? group_sizes[g] : plan->groups == 1 ? plan->batch : 1;
        if (n <= 0) { cq_set_status(CQ_ERR_BAD_ARG, "prefix_plan_shape: a group without sequences"); return 1; }
        const int64_t tiles = ((int64_t)n * s.queries * s.per_kv + s.row_tile - 1) / s.row_tile;
        if (shapes) {
            int *to = shapes + 4 * g;
            to[0] = (int)(seqs * s.queries); to[1] = n * s.queries * s.per_kv; to[2] = (int)items; to[3] = (int)tiles;
        }
        items += tiles * s.kv_heads;
        seqs += n;
    }
    if (seqs != plan->batch) { cq_set_status(CQ_ERR_BAD_ARG, "prefix_plan_shape: the groups' sizes do not add up to the batch"); return 1; }
    plan->shared_items = (int)items;
    plan->n_ints = plan_ints(s);
    plan->n_floats = part_rows(s, items) * (s.head_dim + 2);
    return 0;
}

extern "C" void cq_prefix_plan_update(const cq_kv_cache *cache, const cq_prefix_plan *plan, const int *slots, void *stream) {
    Shape s;
    if (!shape_ok(cache, plan, "prefix_plan_update", s) || !plan_ready(plan, s, "prefix_plan_update")) return;
    if (!slots) { cq_set_status(CQ_ERR_BAD_ARG, "prefix_plan_update: null slots"); return; }
    const size_t smem = 4 * (3 * (size_t)s.batch + 4 * (size_t)s.groups + 2 * (size_t)s.n_queries());
    if (smem > 47 * 1024) cudaFuncSetAttribute(prefix_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    cq_launch_cluster_k(prefix_plan_kernel, dim3(kPlanCtas), dim3(kThreads), smem, (cudaStream_t)stream, kPlanCtas, *cache, call_of(plan, s), slots);
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
    if (s.elem == CQ_F32) f32_launch(c, *cache, layer, q, q_stride, scale, st);
    else if (!mma_launch(c, *cache, layer, q, q_stride, scale, st)) return;
    if (s.head_dim == 128) join_launch<128>(c, out, st);
    else join_launch<64>(c, out, st);
    cq_check_launch("prefix_attention");
}
