// The paged KV cache as the kernels see it (kv_pages.cu: its pages; prefix_attn*.cu: the attention that reads them).
//
//   k, v  : [layers, pages, kv_heads, page_size, head_dim] of one element type
//   state : int32, device: a header, the reference count of every page, the length of every sequence, its row of page numbers, and
//           room that the page operations work in.
#pragma once
#include "../../include/candle_q_b200.h"
#include "common.cuh"

namespace cq_kv {

constexpr int kHeader = 16;             // ints; [0] fault code, [1] copies listed by the last page operation
enum Fault : int { kOk = 0, kBadSlot = 1, kNoPages = 2, kTooLong = 3, kOccupied = 4, kBadPage = 5, kBadPosition = 6, kTimeout = 7 };

struct State {
    int *header, *refs, *lens, *tables, *offsets, *copies, *map;        // copies: (source, destination, rows) per page
    int pages, max_seqs, max_pages, page;
};
__host__ __device__ inline size_t state_ints(int pages, int max_seqs, int max_pages) {
    return (size_t)kHeader + (size_t)pages * 5 + (size_t)max_seqs * 2 + (size_t)max_seqs * max_pages;
}
__host__ __device__ inline State state_of(const cq_kv_cache &c) {
    State s;
    s.pages = c.pages; s.max_seqs = c.max_seqs; s.max_pages = c.max_pages; s.page = c.page_size;
    s.header = c.state;
    s.refs = s.header + kHeader;
    s.lens = s.refs + c.pages;
    s.tables = s.lens + c.max_seqs;
    s.offsets = s.tables + (size_t)c.max_seqs * c.max_pages;
    s.copies = s.offsets + c.max_seqs;
    s.map = s.copies + 3 * (size_t)c.pages;
    return s;
}
__host__ __device__ inline int elem_bytes(int elem) { return elem == CQ_F32 ? 4 : 2; }

// Records `msg` and returns false when the description of the cache is not usable.
bool cache_ok(const cq_kv_cache *c, const char *who);

}  // namespace cq_kv
