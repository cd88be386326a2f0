// Attention of a decode batch over the pages of a KV cache, shared pages read once: the plan that its kernels work from.
//
// A row is one query of one head; the rows of a KV head are numbered (sequence * queries + query) * group + head in group, so the
// rows of consecutive sequences are consecutive.  Two kinds of items cover all (row, key) pairs:
//   shared : up to `row_tile` rows of one group of sequences x one KV head x the keys of the pages that all of them share;
//   own    : up to `own_rows` rows of one query x one KV head x the keys behind these pages.
// An item is a number of units (128 keys of a shared item, `own_step` keys of an own one); the units of all items of a kind form a line, which
// its workers (CTAs for the shared items; CTAs or warps for the own ones) take in equal parts.  A part of an item that one worker takes
// is a segment; it leaves (maximum, sum, unnormalised output) per row, and a second kernel joins a row's segments in the order of their keys:
// m = max m_i,  l = sum 2^(m_i - m) l_i,  o = sum 2^(m_i - m) o_i / l.
#pragma once
#include "kv_cache.cuh"

namespace cq_attn {

constexpr int kKeyTile = 128;       // keys of a shared unit

struct Segment {            // 32 bytes
    int row0, rows;         // rows of the KV head
    int head;               // KV head
    int slot;               // whose table holds the pages
    int key0, key1;         // positions [key0, key1), key0 a multiple of the page size
    int part;               // first row of the partial results
    int units;
};
struct Query {              // 32 bytes
    int len, group;         // context length; group with shared keys, or -1
    int start, units;       // its first own unit on the line, units per item
    int query0, item0, row_tiles, pad;          // of its group
};
struct Group { int start, units, shared, slot; };       // first unit, units per item, shared positions, a slot whose table holds them
struct GroupShape { int query0, item0, row_tiles; };    // from the sizes of the groups alone

struct Shape {
    int batch, queries, heads, kv_heads, groups, head_dim, elem;
    int row_tile, ctas, own_rows, own_step, own_workers;
    __host__ __device__ int per_kv() const { return heads / kv_heads; }
    __host__ __device__ int n_queries() const { return batch * queries; }
    __host__ __device__ int own_tiles() const { return (per_kv() + own_rows - 1) / own_rows; }
    __host__ __device__ int own_slot() const { return per_kv() < own_rows ? per_kv() : own_rows; }      // rows of a partial result
    __host__ __device__ int own_items() const { return n_queries() * kv_heads * own_tiles(); }          // query, then head, then row tile
};

// One kind of items: its segments (that of item i and worker w at i + w), the first segment of each worker, the workers of each item.
struct Line {
    int *header;            // units in all, units per worker
    int *first;             // [workers]
    int2 *item;             // first and last worker (first > last: no keys)
    Segment *segments;      // [items + workers]
};
// The plan's ints.
struct Plan {
    GroupShape *shapes;     // [groups + 1], written by the host's part of the plan
    Group *groups;
    Query *query;
    Line shared, own;
};

// Everything a call has in hand besides its tensors.
struct Call {
    Shape sh;
    Plan plan;
    float *o;               // partial outputs [rows][head_dim]
    float2 *ml;             // maximum (times scale and log2 e) and sum [rows]
    int shared_items;
};

inline int64_t align8(int64_t n) { return (n + 7) / 8 * 8; }
inline int64_t part_rows(const Shape &s, int64_t shared) { return (shared + s.ctas) * s.row_tile + ((int64_t)s.own_items() + s.own_workers) * s.own_slot(); }
inline Line line_of(int *&p, int *header, int64_t items, int64_t workers) {
    Line l;
    l.header = header;
    l.first = p; p += align8(workers);
    l.item = (int2 *)p; p += align8(2 * items);
    l.segments = (Segment *)p; p += 8 * (items + workers);
    return l;
}
inline Plan plan_of(int *base, const Shape &s, int64_t shared, int64_t *ints = nullptr) {
    Plan r;
    int *p = base + 16;
    r.shapes = (GroupShape *)p; p += align8(3LL * (s.groups + 1));
    r.groups = (Group *)p; p += align8(4LL * s.groups);
    r.query = (Query *)p; p += 8LL * s.n_queries();
    r.shared = line_of(p, base, shared, s.ctas);
    r.own = line_of(p, base + 2, s.own_items(), s.own_workers);
    if (ints) *ints = p - base;
    return r;
}
inline int64_t plan_ints(const Shape &s, int64_t shared) {
    int64_t n;
    (void)plan_of((int *)nullptr, s, shared, &n);
    return n;
}

// First row of the partial results of segment i + w of a kind.
__host__ __device__ inline int64_t part_shared(const Shape &s, int at) { return (int64_t)at * s.row_tile; }
__host__ __device__ inline int64_t part_own(const Shape &s, int shared_items, int at) {
    return (int64_t)(shared_items + s.ctas) * s.row_tile + (int64_t)at * s.own_slot();
}

// The kernels that make the segments' results (prefix_attn_simt.cu: f32; prefix_attn_mma.cu: f16 and bf16).
void simt_launch(const Call &c, const cq_kv_cache &cache, int layer, const void *q, int64_t q_stride, float scale, cudaStream_t st);
bool mma_launch(const Call &c, const cq_kv_cache &cache, int layer, const void *q, int64_t q_stride, float scale, cudaStream_t st);
constexpr int kMmaWarps = 6;            // of a CTA of the latter: each is a worker of the own line

}  // namespace cq_attn
