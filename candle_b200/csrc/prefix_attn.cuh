// Attention of a decode batch over the pages of a KV cache, shared pages read once: the plan that its kernels work from.
//
// A row is one query of one head; the rows of a KV head are numbered (sequence * queries + query) * group + head in group, so the
// rows of consecutive sequences are consecutive.  Two kinds of items cover all (row, key) pairs:
//   shared : up to `row_tile` rows of one group of sequences x one KV head x the keys of the pages that all of them share;
//   own    : the rows of one query x one KV head x the keys behind these pages.
// An item is a number of key tiles; the tiles of all items form one line, which the `ctas` CTAs take in equal parts.  A part of an
// item that one CTA takes is a segment; it leaves (maximum, sum, unnormalised output) per row, and a second kernel joins a row's
// segments in the order of their keys:  m = max m_i,  l = sum 2^(m_i - m) l_i,  o = sum 2^(m_i - m) o_i / l.
#pragma once
#include "kv_cache.cuh"

namespace cq_attn {

constexpr int kKeyTile = 128;
constexpr int kMaxQueries = 1 << 16;        // sequences x queries of a call

struct Segment {            // 32 bytes
    int row0, rows;         // rows of the KV head
    int head;               // KV head
    int slot;               // whose table holds the pages
    int key0, key1;         // positions [key0, key1), key0 a multiple of the page size
    int part;               // first row of the partial results
    int tiles;
};
struct Query { int start, tiles, len, group; };         // its first own tile on the line, tiles per head, context length; group -1: no shared keys
struct Group { int start, tiles, shared, slot; };       // first tile, tiles per item, shared positions, a slot whose table holds them
struct GroupShape { int query0, item0, row_tiles; };    // from the sizes of the groups alone

struct Shape {
    int batch, queries, heads, kv_heads, groups, head_dim, elem;
    int row_tile, ctas;
    __host__ __device__ int per_kv() const { return heads / kv_heads; }
    __host__ __device__ int n_queries() const { return batch * queries; }
};

// The plan's ints.  header: [0] tiles in all, [1] tiles per CTA
struct Plan {
    int *header;
    GroupShape *shapes;     // [groups + 1], written by the host's part of the plan
    Group *groups;
    Query *query;
    int2 *item;             // first and last CTA of an item (first > last: no keys)
    int *first;             // first segment of a CTA
    Segment *segments;      // [items + ctas], segment of item i and CTA c at i + c
};

}  // namespace cq_attn

namespace cq_attn {

// Everything a call has in hand besides its tensors.
struct Call {
    Shape sh;
    Plan plan;
    float *o;               // partial outputs [rows][head_dim]
    float2 *ml;             // maximum (times scale and log2 e) and sum [rows]
    int items_shared;
};

inline int64_t align8(int64_t n) { return (n + 7) / 8 * 8; }
inline int64_t items_own(const Shape &s) { return (int64_t)s.n_queries() * s.kv_heads; }
inline int64_t part_rows(const Shape &s, int64_t shared) { return (shared + s.ctas) * s.row_tile + (items_own(s) + s.ctas) * s.per_kv(); }
inline int64_t plan_ints(const Shape &s, int64_t shared) {
    const int64_t items = shared + items_own(s);
    return 16 + align8(3LL * (s.groups + 1)) + 4LL * s.groups + 4LL * s.n_queries() + 8 + align8(2 * items) + align8(s.ctas) + 8 * (items + s.ctas);
}
inline Plan plan_of(int *p, const Shape &s, int64_t shared) {
    const int64_t items = shared + items_own(s);
    Plan r;
    r.header = p; p += 16;
    r.shapes = (GroupShape *)p; p += align8(3LL * (s.groups + 1));
    r.groups = (Group *)p; p += 4LL * s.groups;
    r.query = (Query *)p; p += 4LL * s.n_queries();
    p += (8 - ((4LL * s.groups + 4LL * s.n_queries()) & 7)) & 7;
    r.item = (int2 *)p; p += align8(2 * items);
    r.first = p; p += align8(s.ctas);
    r.segments = (Segment *)p;
    return r;
}

// First row of the partial results of segment (item, CTA).
__host__ __device__ inline int64_t part_of(const Shape &s, int shared, int item, int cta) {
    return item < shared ? (int64_t)(item + cta) * s.row_tile : (int64_t)(shared + s.ctas) * s.row_tile + (int64_t)(item - shared + cta) * s.per_kv();
}

// One CTA's kernel for all segments, by element type (prefix_attn_simt.cu, prefix_attn_mma.cu).
void simt_launch(const Call &c, const cq_kv_cache &cache, int layer, const void *q, int64_t q_stride, float scale, cudaStream_t st);
bool mma_launch(const Call &c, const cq_kv_cache &cache, int layer, const void *q, int64_t q_stride, float scale, cudaStream_t st);

}  // namespace cq_attn
