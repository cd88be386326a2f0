// Attention of a decode batch over the pages of a KV cache, shared pages read once: the plan that its kernels work from.
//
// A row is one query of one head; the rows of a KV head are numbered (sequence * queries + query) * group + head in group, so the
// rows of consecutive sequences are consecutive.  Two kinds of items cover all (row, key) pairs:
//   shared : up to `row_tile` rows of one group of sequences x one KV head x the keys of the pages that all of them share;
//   own    : up to `own_rows` rows of one query x one KV head x the keys behind these pages.
// An item is a number of units (`tile` keys of a shared item, 2^own_shift of an own one); the units of all items of a kind form a line, which
// its workers (CTAs or warps) take in equal parts.  A part of an item that one worker takes
// is a segment; it leaves (maximum, sum, unnormalised output) per row, and a second kernel joins a row's segments in the order of their keys:
// m = max m_i,  l = sum 2^(m_i - m) l_i,  o = sum 2^(m_i - m) o_i / l.
#pragma once
#include "kv_cache.cuh"

namespace cq_attn {

struct Segment {
    int row0, rows;         // rows of the KV head
    int head;               // KV head
    int slot;               // whose table holds the pages
    int key0, key1;         // positions [key0, key1), key0 a multiple of 16
    int part;               // first row of the partial results
    int units;
};
struct Group {              // 32 bytes
    int units, shared, slot, start;             // units per item, shared positions, a slot whose table holds them, first unit on the line
    int query0, rows, item0, row_tiles;         // from the sizes of the groups alone
};
struct Query {              // 64 bytes
    int len, slot, shared, units;               // context length, slot, positions that its group shares (its own keys begin there), own units per item
    int start, group_start, group_units, query0;
    int item0, row_tiles, pad[6];
};
// Where a worker begins: the group (query), head and row tile of its first item, the unit in that, and how many units the worker has.
struct Start { int index, head, tile, unit, left, pad[3], copy[8]; };       // 64 bytes; copy: the Group, or the first half of the Query
struct GroupShape { int query0, rows, item0, row_tiles; };

struct Shape {
    int batch, queries, heads, kv_heads, groups, head_dim, elem, per_kv;
    int row_tile, tile, ctas;                                   // rows of a shared item, keys of a unit of it (a multiple of the largest page or a part of the smallest), workers
    int own_rows, own_shift;                                    // rows of an own item, 2^own_shift keys a unit
    int own_workers, own_first;                                 // workers of the own line; the first own_first have chunks of one size, the others of another
    int own_tiles;          // row tiles of a KV head's query heads
    unsigned rcp;           // ceil(2^32 / query heads per KV head); 0 for one
    __host__ __device__ int n_queries() const { return batch * queries; }
    __host__ __device__ int own_slot() const { return per_kv < own_rows ? per_kv : own_rows; }      // rows of a partial result
    __host__ __device__ int own_items() const { return n_queries() * kv_heads * own_tiles; }        // query, then head, then row tile
};

// The plan's ints.
struct Plan {
    int *header;            // units of the shared line, units per CTA; units of the own line, per worker of the first and of the second kind
    GroupShape *shapes;     // [groups], written by the host's part of the plan
    Group *groups;
    Query *query;
    Start *shared, *own;    // [ctas], [own_workers]
};

// Everything a call has in hand besides its tensors.
struct Call {
    Shape sh;
    Plan plan;
    float *o;               // partial outputs [rows][head_dim]
    float2 *ml;             // maximum (times scale and log2 e) and sum [rows]
    int shared_items;
};

inline int64_t part_rows(const Shape &s, int64_t shared) { return (shared + s.ctas) * s.row_tile + ((int64_t)s.own_items() + s.own_workers) * s.own_slot(); }
inline Plan plan_of(int *base, const Shape &s, int64_t *ints = nullptr) {
    Plan r;
    int *p = base + 16;
    r.header = base;
    r.shapes = (GroupShape *)p; p += (4LL * s.groups + 15) / 16 * 16;
    r.groups = (Group *)p; p += (8LL * s.groups + 15) / 16 * 16;
    r.query = (Query *)p; p += 16LL * s.n_queries();
    r.shared = (Start *)p; p += 16LL * s.ctas;
    r.own = (Start *)p; p += 16LL * s.own_workers;
    if (ints) *ints = p - base;
    return r;
}
inline int64_t plan_ints(const Shape &s) {
    int64_t n;
    (void)plan_of((int *)nullptr, s, &n);
    return n;
}

// Which worker has unit u of the own line.
__host__ __device__ inline int own_worker(const Shape &s, int u, int chunk, int chunk2) {
    const int first = s.own_first * chunk;
    return u < first ? u / chunk : s.own_first + (u - first) / chunk2;
}

// First row of the partial results of segment (item, worker) of a kind, at = item + worker: that sum is another one for every segment of a line.
__host__ __device__ inline int64_t part_shared(const Shape &s, int at) { return (int64_t)at * s.row_tile; }
__host__ __device__ inline int64_t part_own(const Shape &s, int shared_items, int at) {
    return (int64_t)(shared_items + s.ctas) * s.row_tile + (int64_t)at * s.own_slot();
}

// The segments of a worker, one after the other.
struct SharedWalk {
    int group, head, tile, unit, left, cta;
    Group g;
    __device__ __forceinline__ void take(const int4 &b, const int4 &d) { g = Group{b.x, b.y, b.z, b.w, d.x, d.y, d.z, d.w}; }
    __device__ __forceinline__ SharedWalk(const Call &c, int cta) : cta(cta) {
        const int4 *p = reinterpret_cast<const int4 *>(c.plan.shared + cta);
        const int4 a = p[0];
        left = p[1].x;
        group = a.x; head = a.y; tile = a.z; unit = a.w;
        take(p[2], p[3]);
    }
    __device__ __forceinline__ bool next(const Call &c, Segment &s) {
        if (left <= 0) return false;
        const Shape &sh = c.sh;
        while (g.units == 0 || head == sh.kv_heads) {
            const int4 *p = reinterpret_cast<const int4 *>(c.plan.groups + ++group);
            take(p[0], p[1]);
            head = 0;
        }
        s.head = head;
        s.row0 = g.query0 * sh.per_kv + tile * sh.row_tile;
        s.rows = min(sh.row_tile, g.rows - tile * sh.row_tile);
        s.slot = g.slot;
        s.units = min(left, g.units - unit);
        s.key0 = unit * sh.tile;
        s.key1 = min(g.shared, (unit + s.units) * sh.tile);
        s.part = (int)part_shared(sh, g.item0 + head * g.row_tiles + tile + cta);
        left -= s.units;
        unit += s.units;
        if (unit == g.units) {
            unit = 0;
            if (++tile == g.row_tiles) { tile = 0; ++head; }
        }
        return true;
    }
};
struct OwnWalk {
    int query, head, tile, unit, left, worker;
    int len, slot, shared, units;
    __device__ __forceinline__ OwnWalk(const Call &c, int worker) : worker(worker) {
        const int4 *p = reinterpret_cast<const int4 *>(c.plan.own + worker);
        const int4 a = p[0], b = p[2];
        left = p[1].x;
        query = a.x; head = a.y; tile = a.z; unit = a.w;
        len = b.x; slot = b.y; shared = b.z; units = b.w;
    }
    __device__ __forceinline__ bool next(const Call &c, Segment &s) {
        if (left <= 0) return false;
        const Shape &sh = c.sh;
        while (units == 0 || head == sh.kv_heads) {
            const int4 b = *reinterpret_cast<const int4 *>(c.plan.query + ++query);
            len = b.x; slot = b.y; shared = b.z; units = b.w;
            head = 0;
        }
        s.head = head;
        s.row0 = query * sh.per_kv + tile * sh.own_rows;
        s.rows = min(sh.own_rows, sh.per_kv - tile * sh.own_rows);
        s.slot = slot;
        s.units = min(left, units - unit);
        s.key0 = shared + (unit << sh.own_shift);
        s.key1 = min(len, s.key0 + (s.units << sh.own_shift));
        s.part = (int)part_own(sh, c.shared_items, (query * sh.kv_heads + head) * sh.own_tiles + tile + worker);
        left -= s.units;
        unit += s.units;
        if (unit == units) {
            unit = 0;
            if (++tile == sh.own_tiles) { tile = 0; ++head; }
        }
        return true;
    }
};
// n / per for the rows of a call, by a multiplication: exact for n < 2^22, per <= 32, with rcp = ceil(2^32 / per)
__device__ __forceinline__ int div_per(int n, const Shape &s) { return s.rcp ? (int)__umulhi((unsigned)n, s.rcp) : n; }

// The kernels that make the segments' results (prefix_attn_f32.cu: f32; prefix_attn_mma.cu: f16 and bf16).
void f32_launch(const Call &c, const cq_kv_cache &cache, int layer, const void *q, int64_t q_stride, float scale, cudaStream_t st);
bool mma_launch(const Call &c, const cq_kv_cache &cache, int layer, const void *q, int64_t q_stride, float scale, cudaStream_t st);
constexpr int f32_warps(int head_dim) { return head_dim == 128 ? 6 : 12; }      // of a CTA of the former, one per SM: each is a worker of both lines
constexpr int kMmaWarps = 4, kMmaHelpers = 8;       // warps of a CTA of the latter that are workers of the own line from the start, and after the shared items

}  // namespace cq_attn
