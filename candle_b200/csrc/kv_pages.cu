// Pages of a KV cache: reserving, forking, freeing and compacting them, and the store of new keys and values.
//
// The bookkeeping (reference counts, lengths, tables) lives on the device, so that a decode step that grows its sequences, or forks
// one, is a sequence of launches that a graph can hold.  One CTA does it: a pool has some thousands of pages, and a page's number
// depends on all that are taken before it.  What it decides, a second kernel copies with the whole device.
// On a B200, each kernel by itself with cold caches: 63 forks of 16 pages 10 - 13 us, bound by some ten reads that depend on one another; the list of a compaction of 320
// pages 5 us.  In a graph: a token reserved for 1 / 64 / 128 sequences 3.0 / 3.7 / 4.5 us, 16 pages each freed 3.0 / 4.8 / 7.1.
#include <cstdio>

#include "kv_cache.cuh"

namespace cq_kv {

bool cache_ok(const cq_kv_cache *c, const char *who) {
    char msg[160];
    const char *why = nullptr;
    int status = CQ_ERR_BAD_ARG;
    if (!c || !c->k || !c->v || !c->state) why = "null pointer";
    else if (c->layers <= 0 || c->pages <= 0 || c->kv_heads <= 0 || c->max_seqs <= 0 || c->max_pages <= 0) why = "sizes must be positive";
    else if (c->elem != CQ_F32 && c->elem != CQ_F16 && c->elem != CQ_BF16) why = "element type must be f32, f16 or bf16";
    else if (((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->state) & 15) why = "k, v and state must be 16-byte aligned";
    else {
        status = CQ_ERR_UNSUPPORTED;
        if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) why = "page_size must be 16, 32, 64 or 128";
        else if (c->head_dim != 64 && c->head_dim != 128) why = "head_dim must be 64 or 128";
        else if (c->max_seqs > 65536 || (int64_t)c->max_seqs * c->max_pages > (1 << 28) || (int64_t)c->max_pages * c->page_size > (1 << 30))
            why = "at most 65536 slots, 2^28 table entries and 2^30 positions";
        // rows of head_dim elements of one layer are numbered in 32 bits
        else if ((int64_t)c->pages * c->kv_heads * c->page_size > INT32_MAX || (int64_t)c->pages * c->layers * c->kv_heads > (1 << 26))
            why = "at most 2^31 rows in a layer and 2^26 pages over all layers and heads";
    }
    if (!why) return true;
    std::snprintf(msg, sizeof msg, "%s: %s", who, why);
    cq_set_status(status, msg);
    return false;
}

}  // namespace cq_kv

namespace {
using namespace cq_kv;

constexpr int kMeta = 1024;

// Sum of `v` over the threads before this one; `total` over all.
__device__ __forceinline__ int block_scan(int v, int *sums, int &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, m);
        if (lane >= m) x += y;
    }
    __syncthreads();                    // the sums of the call before have been read
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

__device__ __forceinline__ int pages_of(int len, int page) { return (len + page - 1) / page; }

// The `total` lowest free pages into copies[3 f + 1]; false when there are fewer.
__device__ bool take_free(const State &s, int total, int *sums) {
    int found = 0;
    for (int p0 = 0; p0 < s.pages && found < total; p0 += 4 * kMeta) {
        const int p = p0 + 4 * threadIdx.x;
        int r[4] = {1, 1, 1, 1};
        if (p + 3 < s.pages) {
            const int4 q = *reinterpret_cast<const int4 *>(s.refs + p);
            r[0] = q.x; r[1] = q.y; r[2] = q.z; r[3] = q.w;
        } else
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (p + i < s.pages) r[i] = s.refs[p + i];
        int mine = 0, all;
#pragma unroll
        for (int i = 0; i < 4; ++i) mine += r[i] == 0;
        int f = found + block_scan(mine, sums, all);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (r[i] == 0) {
                if (f < total) s.copies[3 * (size_t)f + 1] = p + i;
                ++f;
            }
        found += all;
    }
    __syncthreads();
    return found >= total;
}

// Whether the pages in the row of a slot of length `len` are in the pool and taken; one warp.
__device__ __forceinline__ bool row_ok(const State &s, int slot, int len, int lane) {
    bool ok = true;
    for (int j = lane; j < pages_of(len, s.page); j += 32) {
        const int p = s.tables[(size_t)slot * s.max_pages + j];
        ok = ok && p >= 0 && p < s.pages && s.refs[p] > 0;
    }
    return __all_sync(0xffffffffu, ok);
}

enum MetaOp { kReserve, kFork, kFree };

// Three passes: everything is checked; the pages each slot needs are numbered in the order of the list; then the state changes.
template <int OP>
__global__ void __launch_bounds__(kMeta) kv_meta_kernel(const cq_kv_cache cache, const int *slots, const int *dst, int n, int arg) {
    extern __shared__ unsigned seen[];              // one bit per slot
    __shared__ int sums[32], err;
    const State s = state_of(cache);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cap = s.max_pages * s.page;
    cq_pdl_wait();
    for (int i = tid; i < (s.max_seqs + 31) / 32; i += kMeta) seen[i] = 0;
    if (tid == 0) {
        err = s.header[0] ? -1 : 0;
        s.header[1] = 0;
    }
    __syncthreads();
    const int stop = err;
    __syncthreads();                                // read by all before any thread adds to it
    if (stop) return;
    auto in_range = [&](int slot) { return slot >= 0 && slot < s.max_seqs; };
    auto fail = [&](int code) { atomicMax(&err, code); };
    const int *changed = OP == kFork ? dst : slots;
    for (int i = tid; i < n; i += kMeta) {
        const int slot = changed[i];
        if (!in_range(slot) || (OP == kFork && !in_range(slots[i]))) { fail(kBadSlot); continue; }
        const unsigned bit = 1u << (slot & 31);
        if (atomicOr(&seen[slot >> 5], bit) & bit) fail(kBadSlot);
        const int len = s.lens[slot];
        if (len < 0 || len > cap) fail(kBadPage);
        if (OP == kFork && len != 0) fail(kOccupied);
        if (OP == kReserve && (int64_t)len + arg > cap) fail(kTooLong);
        if (OP == kFork) {
            const int from = s.lens[slots[i]];
            if (from < 0 || from > cap) fail(kBadPage);
        }
    }
    __syncthreads();
    if (!err && OP != kReserve)
        for (int i = warp; i < n; i += kMeta / 32) {
            const int slot = slots[i];
            if (OP == kFork && (seen[slot >> 5] >> (slot & 31) & 1)) { fail(kBadSlot); continue; }
            if (!row_ok(s, slot, s.lens[slot], lane)) fail(kBadPage);
        }
    __syncthreads();
    int total = 0;
    if (!err && OP != kFree) {
        for (int i0 = 0; i0 < n; i0 += kMeta) {
            const int i = i0 + tid;
            int need = 0, all;
            if (i < n) {
                const int len = s.lens[slots[i]];
                if (OP == kReserve) need = pages_of(len + arg, s.page) - pages_of(len, s.page);
                else need = arg ? pages_of(len, s.page) : (len % s.page ? 1 : 0);
            }
            const int at = total + block_scan(need, sums, all);
            if (i < n) s.offsets[i] = at;
            total += all;
        }
        // more than the pool has: take_free would not need to look, and its list would not hold them
        if (total > s.pages || !take_free(s, total, sums)) fail(kNoPages);
    }
    __syncthreads();
    if (err) {
        if (tid == 0) s.header[0] = err;
        return;
    }
    for (int i = warp; i < n; i += kMeta / 32) {
        const int slot = slots[i], len = s.lens[slot];
        int *row = s.tables + (size_t)slot * s.max_pages;
        __syncwarp();
        if (OP == kReserve) {
            const int have = pages_of(len, s.page), need = pages_of(len + arg, s.page) - have;
            for (int j = lane; j < need; j += 32) {
                const int p = s.copies[3 * (size_t)(s.offsets[i] + j) + 1];
                row[have + j] = p;
                s.refs[p] = 1;
            }
            if (lane == 0) s.lens[slot] = len + arg;
        } else if (OP == kFree) {
            for (int j = lane; j < pages_of(len, s.page); j += 32) {
                atomicSub(&s.refs[row[j]], 1);
                row[j] = -1;
            }
            if (lane == 0) s.lens[slot] = 0;
        } else {
            int *to = s.tables + (size_t)dst[i] * s.max_pages;
            const int shared = arg ? 0 : len / s.page;
            for (int j = lane; j < pages_of(len, s.page); j += 32) {
                const int p = row[j];
                if (j < shared) {
                    to[j] = p;
                    atomicAdd(&s.refs[p], 1);
                } else {
                    int *c = s.copies + 3 * (size_t)(s.offsets[i] + j - shared);
                    c[0] = p;
                    c[2] = min(s.page, len - j * s.page);
                    to[j] = c[1];
                    s.refs[c[1]] = 1;
                }
            }
            if (lane == 0) s.lens[dst[i]] = len;
        }
    }
    if (OP == kFork && tid == 0) s.header[1] = total;
}

// Live pages are counted, then the free ones below that number meet the live ones at or above it, both in ascending order.
__global__ void __launch_bounds__(kMeta) kv_compact_kernel(const cq_kv_cache cache) {
    __shared__ int sums[32], stop;
    const State s = state_of(cache);
    const int tid = threadIdx.x;
    cq_pdl_wait();
    if (tid == 0) {
        stop = s.header[0];
        s.header[1] = 0;
    }
    __syncthreads();
    if (stop) return;
    int mine = 0, live;
    for (int p = tid; p < s.pages; p += kMeta) mine += s.refs[p] > 0;
    block_scan(mine, sums, live);
    int holes = 0, movers = 0;
    for (int p0 = 0; p0 < s.pages; p0 += kMeta) {
        const int p = p0 + tid;
        const bool used = p < s.pages && s.refs[p] > 0;
        const bool hole = p < live && !used, mover = p >= live && used;
        int nh, nm;
        const int ah = block_scan(hole, sums, nh), am = block_scan(mover, sums, nm);
        if (hole) s.copies[3 * (size_t)(holes + ah) + 1] = p;
        if (mover) {
            s.copies[3 * (size_t)(movers + am)] = p;
            s.copies[3 * (size_t)(movers + am) + 2] = s.page;
        }
        if (p >= live && p < s.pages) s.map[p] = -1;
        holes += nh;
        movers += nm;
    }
    __syncthreads();
    for (int m = tid; m < movers; m += kMeta) {         // as many as holes: both are live - (live pages below `live`)
        const int from = s.copies[3 * (size_t)m], to = s.copies[3 * (size_t)m + 1];
        s.refs[to] = s.refs[from];
        s.refs[from] = 0;
        s.map[from] = to;
    }
    __syncthreads();
    if (tid == 0) {
        s.header[1] = movers;
        s.header[2] = live;
    }
}

// The listed copies over all layers, keys and values.  A warp moves pieces of kPiece bytes, eight 16-byte loads of a lane in flight
// before the first store.  REMAP: the table entries of moved pages follow (compaction).  Bound by HBM: 64 pages of 32 layers, 1074 MB read and written, in 173 us, 6.2 TB/s
// (a plain copy of the device: 6.5); 63 part-full pages, 336 MB, in 57 us, 5.9 TB/s.
constexpr int kPiece = 4096, kCopyThreads = 256;
template <bool REMAP>
__global__ void __launch_bounds__(kCopyThreads) kv_copy_kernel(const cq_kv_cache cache) {
    const State s = state_of(cache);
    const int lane = threadIdx.x & 31;
    cq_pdl_wait();
    const int n = s.header[1];
    if (n == 0) return;
    const int row_bytes = cache.head_dim * elem_bytes(cache.elem);
    const unsigned pieces = (unsigned)(s.page * row_bytes + kPiece - 1) / kPiece, heads = cache.kv_heads;
    const unsigned per_copy = 2u * cache.layers * heads * pieces;
    const int64_t page_bytes = (int64_t)s.page * row_bytes;
    const unsigned total = (unsigned)n * per_copy, warps = gridDim.x * (kCopyThreads / 32);
    for (unsigned u = blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5); u < total; u += warps) {
        const unsigned c = u / per_copy, r = u % per_copy, seg = r / pieces, piece = r % pieces, layer_kv = seg / heads, head = seg % heads;
        const int bytes = min(s.copies[3 * (size_t)c + 2] * row_bytes - (int)piece * kPiece, kPiece);
        if (bytes <= 0) continue;
        uint8_t *pool = reinterpret_cast<uint8_t *>(layer_kv & 1 ? cache.v : cache.k);
        const int64_t layer = (int64_t)(layer_kv >> 1) * cache.pages;
        const uint4 *from = reinterpret_cast<const uint4 *>(pool + ((layer + s.copies[3 * (size_t)c]) * heads + head) * page_bytes + piece * kPiece) + lane;
        uint4 *to = reinterpret_cast<uint4 *>(pool + ((layer + s.copies[3 * (size_t)c + 1]) * heads + head) * page_bytes + piece * kPiece) + lane;
        uint4 w[kPiece / 512];
#pragma unroll
        for (int i = 0; i < kPiece / 512; ++i)
            if (i * 512 + lane * 16 < bytes) w[i] = from[32 * i];
#pragma unroll
        for (int i = 0; i < kPiece / 512; ++i)
            if (i * 512 + lane * 16 < bytes) to[32 * i] = w[i];
    }
    if constexpr (REMAP) {
        const int live = s.header[2];
        const int64_t entries = (int64_t)s.max_seqs * s.max_pages;
        for (int64_t e = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x; e < entries; e += (int64_t)gridDim.x * kCopyThreads) {
            const int p = s.tables[e];
            if (p >= live && p < s.pages) s.tables[e] = s.map[p];
        }
    }
}

__global__ void __launch_bounds__(256) kv_reset_kernel(const cq_kv_cache cache) {
    cq_pdl_wait();
    const State s = state_of(cache);
    const int64_t n = (int64_t)state_ints(s.pages, s.max_seqs, s.max_pages), t0 = s.tables - s.header, t1 = s.offsets - s.header;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) s.header[i] = i >= t0 && i < t1 ? -1 : 0;
}

// ---- new keys and values ----
template <typename T, int N> struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Vec { T v[N]; };
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

struct AppendArgs {
    const int *slots;
    const void *q, *k, *v;
    void *q_out;
    const float *cosv, *sinv;
    int64_t q_stride, k_stride, v_stride;
    int layer, batch, t, hq, max_pos, neox;
};

// What is looked at before any row of an append is stored: each slot, and the pages of its last t positions, at most `per` of them.
__device__ __forceinline__ int append_fault(const State &s, const AppendArgs &a, int slot, int len, int page, int refs) {
    if (slot < 0 || slot >= s.max_seqs) return kBadSlot;
    if (len < a.t || len > s.max_pages * s.page || (a.cosv && len > a.max_pos)) return kBadPosition;
    if (page < 0 || page >= s.pages) return kBadPage;
    return refs > 1 ? kBadPosition : kOk;                   // others read it
}
// The table entry of position `pos` of a slot, kept inside the tables so that it can be read before slot and position are known to be right.
__device__ __forceinline__ int entry_of(const State &s, int slot, int pos, int shift) {
    const bool there = slot >= 0 && slot < s.max_seqs;
    return there ? slot * s.max_pages + min(max(pos >> shift, 0), s.max_pages - 1) : 0;
}
// The item-th check by itself; `seen`: the slots that were named so far.
__device__ __forceinline__ int append_check(const State &s, const AppendArgs &a, unsigned *seen, int item, int per, int shift) {
    const int b = item / per, j = item - b * per, slot = a.slots[b];
    if (slot < 0 || slot >= s.max_seqs) return kBadSlot;
    if (j == 0 && atomicOr(&seen[slot >> 5], 1u << (slot & 31)) >> (slot & 31) & 1) return kBadSlot;
    const int len = s.lens[slot], pos = min(((len - a.t) >> shift << shift) + (j << shift), len - 1), page = s.tables[entry_of(s, slot, pos, shift)];
    return append_fault(s, a, slot, len, page, page >= 0 && page < s.pages ? s.refs[page] : 0);
}

// The checks of a call with many: a fault before the rows' kernel looks for one.
__global__ void __launch_bounds__(kMeta) kv_append_check_kernel(const cq_kv_cache cache, const AppendArgs a, int per) {
    extern __shared__ unsigned seen[];
    __shared__ int err;
    const State s = state_of(cache);
    const int shift = 31 - __clz(s.page);
    for (int i = threadIdx.x; i < (s.max_seqs + 31) / 32; i += kMeta) seen[i] = 0;
    if (threadIdx.x == 0) err = kOk;
    cq_pdl_launch_dependents();
    __syncthreads();
    cq_pdl_wait();
    int wrong = kOk;
#pragma unroll 4
    for (int64_t item = threadIdx.x; item < (int64_t)a.batch * per; item += kMeta) wrong = max(wrong, append_check(s, a, seen, (int)item, per, shift));
    if (wrong) atomicMax(&err, wrong);
    __syncthreads();
    if (threadIdx.x == 0 && err) atomicCAS(s.header, kOk, err);
}

// A thread takes four rotary pairs of one head: eight consecutive elements (interleaved), or four and the four half a head further.
// grid.x covers the heads of q, k and v of a row, grid.y the rows, R of them at a time: their elements are asked for before their places are looked up, which is a chain of
// three reads, with cos and sin at its end.  Every CTA makes all `checks` of the call, one a thread beside its first rows' chain, so all of them come to the same answer without
// a word between them, and a call is stored whole or not at all.  (0.25 us of 64 rows; an arrival counter, so that a fault shows when all CTAs have read that there was none
// before, took 2.5 ns a CTA: 300 rows 9.1 us.)
// One read and one write of each element are the bound: 2047 rows of 48 heads of 128, f32, 102 MB in 21.4 us, 4.8 TB/s; 64 rows take 2.95 us, a launch and the chain, 300 rows 5.1
// (all in a graph).
template <typename In, typename T, int R>
__global__ void __launch_bounds__(128) kv_append_kernel(const cq_kv_cache cache, const AppendArgs a, int checks, int per) {
    extern __shared__ unsigned seen[];
    const State s = state_of(cache);
    const int tid = threadIdx.x;
    cq_pdl_launch_dependents();
    if (checks && a.batch > 1) {
        for (int i = tid; i < (s.max_seqs + 31) / 32; i += 128) seen[i] = 0;
        __syncthreads();
    }
    cq_pdl_wait();
    const int shift = 31 - __clz(s.page), d = cache.head_dim, log_per = d == 128 ? 4 : 3, hkv = cache.kv_heads, hq = a.q ? a.hq : 0;
    const int unit = blockIdx.x * 128 + tid, x = unit & ((1 << log_per) - 1);
    const bool there = unit >> log_per < hq + 2 * hkv;              // the last CTA's other threads only check
    const int head = there ? unit >> log_per : 0;
    const bool is_q = head < hq, is_v = head >= hq + hkv;
    const int first = a.neox ? 4 * x : 8 * x, second = a.neox ? first + d / 2 : first + 4, own = is_q ? head : is_v ? head - hq - hkv : head - hq;
    const In *from = reinterpret_cast<const In *>(is_q ? a.q : is_v ? a.v : a.k) + (int64_t)own * d;
    const int64_t stride = is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride;
    const int rows = a.batch * a.t, step = gridDim.y;
    const int fault = s.header[0];
    int wrong = kOk;
    for (int item = tid + 128; item < checks; item += 128) wrong = max(wrong, append_check(s, a, seen, item, per, shift));
    bool stop = false;
    for (int row0 = blockIdx.y; row0 < rows; row0 += R * step) {
        Vec<In, 4> lo[R], hi[R];
        int pos[R], page[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const In *src = from + (int64_t)min(row0 + i * step, rows - 1) * stride;
            lo[i] = *reinterpret_cast<const Vec<In, 4> *>(src + first);
            hi[i] = *reinterpret_cast<const Vec<In, 4> *>(src + second);
        }
        // The chains: those of the rows and, the first time, that of a check.  All read inside the tables, whatever the numbers are; what they mean is looked at behind.
        const bool check = row0 == blockIdx.y && tid < checks;
        int slot[R + 1], len[R + 1], entry[R + 1];
#pragma unroll
        for (int i = 0; i <= R; ++i) {
            const int row = min(row0 + i * step, rows - 1), b = i < R ? (a.t == 1 ? row : row / a.t) : check ? (per == 1 ? tid : tid / per) : 0;
            slot[i] = a.slots[b];
            if (i < R) pos[i] = row - b * a.t - a.t;
        }
        const int j = per == 1 ? 0 : tid % per;
        unsigned twice = 0;                     // a slot named twice would have two writers for its positions
        if (check && a.batch > 1 && j == 0 && slot[R] >= 0 && slot[R] < s.max_seqs) twice = atomicOr(&seen[slot[R] >> 5], 1u << (slot[R] & 31)) >> (slot[R] & 31) & 1;
#pragma unroll
        for (int i = 0; i <= R; ++i) len[i] = s.lens[slot[i] >= 0 && slot[i] < s.max_seqs ? slot[i] : 0];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            pos[i] += len[i];
            entry[i] = entry_of(s, slot[i], pos[i], shift);
        }
        entry[R] = entry_of(s, slot[R], min(((len[R] - a.t) >> shift << shift) + (j << shift), len[R] - 1), shift);
#pragma unroll
        for (int i = 0; i < R; ++i) page[i] = s.tables[entry[i]];
        const int check_page = s.tables[entry[R]];
        float4 c[R], n[R];
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (!is_v && a.cosv) {
                const int64_t at = (int64_t)min(max(pos[i], 0), a.max_pos - 1) * (d / 2) + 4 * x;
                c[i] = *reinterpret_cast<const float4 *>(a.cosv + at);
                n[i] = *reinterpret_cast<const float4 *>(a.sinv + at);
            }
        if (row0 == blockIdx.y) {
            if (check) wrong = max(wrong, twice ? (int)kBadSlot : append_fault(s, a, slot[R], len[R], check_page, s.refs[check_page >= 0 && check_page < s.pages ? check_page : 0]));
            stop = checks ? __syncthreads_or(fault | wrong) != 0 : fault != 0;
            if (wrong && blockIdx.x == 0 && blockIdx.y == 0) atomicCAS(s.header, kOk, wrong);
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int64_t row = row0 + (int64_t)i * step;
            if (row >= rows || !there || (stop && !is_q)) break;
            Vec<T, 4> out_lo, out_hi;
            if (is_v || !a.cosv) {
#pragma unroll
                for (int y = 0; y < 4; ++y) { out_lo.v[y] = from_f<T>(to_f(lo[i].v[y])); out_hi.v[y] = from_f<T>(to_f(hi[i].v[y])); }
            } else {
                const float cs[4] = {c[i].x, c[i].y, c[i].z, c[i].w}, sn[4] = {n[i].x, n[i].y, n[i].z, n[i].w};
                float p0[4], p1[4], r0[4], r1[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    p0[y] = a.neox ? to_f(lo[i].v[y]) : y < 2 ? to_f(lo[i].v[2 * (y & 1)]) : to_f(hi[i].v[2 * (y & 1)]);
                    p1[y] = a.neox ? to_f(hi[i].v[y]) : y < 2 ? to_f(lo[i].v[2 * (y & 1) + 1]) : to_f(hi[i].v[2 * (y & 1) + 1]);
                }
#pragma unroll
                for (int y = 0; y < 4; ++y) {               // the operations of cq_rope_store_kv_f32
                    r0[y] = __fmaf_rn(p0[y], cs[y], -__fmul_rn(p1[y], sn[y]));
                    r1[y] = __fmaf_rn(p0[y], sn[y], __fmul_rn(p1[y], cs[y]));
                }
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    out_lo.v[y] = from_f<T>(a.neox ? r0[y] : y & 1 ? r1[y >> 1] : r0[y >> 1]);
                    out_hi.v[y] = from_f<T>(a.neox ? r1[y] : y & 1 ? r1[2 + (y >> 1)] : r0[2 + (y >> 1)]);
                }
            }
            T *dst;
            if (is_q) {
                if (stop)
#pragma unroll
                    for (int y = 0; y < 4; ++y) out_lo.v[y] = out_hi.v[y] = from_f<T>(0.0f);
                dst = reinterpret_cast<T *>(a.q_out) + (row * hq + head) * d;
            } else
                dst = reinterpret_cast<T *>(is_v ? cache.v : cache.k) +
                      (((((int64_t)a.layer * s.pages + page[i]) * hkv + own) << shift) + (pos[i] & (s.page - 1))) * d;
            *reinterpret_cast<Vec<T, 4> *>(dst + first) = out_lo;
            *reinterpret_cast<Vec<T, 4> *>(dst + second) = out_hi;
        }
    }
}

// Up to this many checks every CTA makes them all (2047 rows over pages of 16: 129, two a thread); beyond, a kernel before it.
constexpr int kChecksInside = 512;

template <typename In, typename T> void append_launch(const cq_kv_cache &c, const AppendArgs &a, cudaStream_t st) {
    const unsigned units = ((a.q ? a.hq : 0) + 2 * c.kv_heads) * (c.head_dim / 8), x = (units + 127) / 128, rows = (unsigned)a.batch * a.t;
    const size_t smem = (size_t)(c.max_seqs + 31) / 32 * 4;
    const int per = (a.t + c.page_size - 2) / c.page_size + 1;             // pages that t positions can lie in
    const bool inside = (int64_t)a.batch * per <= kChecksInside;
    const int checks = inside ? a.batch * per : 0;
    if (!inside) cq_launch_k(kv_append_check_kernel, dim3(1), dim3(kMeta), smem, st, c, a, per);
    // four rows a thread where that still fills the device (16 such CTAs an SM); one where latency counts
    if (x * rows >= 4u * 16 * cq_sm_count())
        cq_launch_k(kv_append_kernel<In, T, 4>, dim3(x, (rows + 3) / 4 < 65535 ? (rows + 3) / 4 : 65535), dim3(128), smem, st, c, a, checks, per);
    else cq_launch_k(kv_append_kernel<In, T, 1>, dim3(x, rows < 65535 ? rows : 65535), dim3(128), smem, st, c, a, checks, per);
}

bool slots_ok(const cq_kv_cache *c, const int *a, const int *b, int n, const char *who) {
    if (!cache_ok(c, who)) return false;
    if ((n && (!a || !b)) || n < 0 || n > c->max_seqs) {
        char msg[160];
        std::snprintf(msg, sizeof msg, "%s: null list, or more slots than the cache has", who);
        cq_set_status(CQ_ERR_BAD_ARG, msg);
        return false;
    }
    return true;
}
size_t seen_bytes(const cq_kv_cache *c) { return (size_t)(c->max_seqs + 31) / 32 * 4; }

}  // namespace

extern "C" size_t cq_kv_state_ints(int pages, int max_seqs, int max_pages) {
    return pages > 0 && max_seqs > 0 && max_pages > 0 ? state_ints(pages, max_seqs, max_pages) : 0;
}

extern "C" void cq_kv_reset(const cq_kv_cache *cache, void *stream) {
    if (!cache_ok(cache, "kv_reset")) return;
    const int64_t n = (int64_t)state_ints(cache->pages, cache->max_seqs, cache->max_pages);
    cq_launch_k(kv_reset_kernel, dim3((unsigned)(n / 1024 < 1 ? 1 : n / 1024 < 1024 ? n / 1024 : 1024)), dim3(256), 0, (cudaStream_t)stream, *cache);
    cq_check_launch("kv_reset");
}

extern "C" void cq_kv_reserve(const cq_kv_cache *cache, const int *slots, int n, int tokens, void *stream) {
    if (!slots_ok(cache, slots, slots, n, "kv_reserve")) return;
    if (tokens < 0) { cq_set_status(CQ_ERR_BAD_ARG, "kv_reserve: negative number of tokens"); return; }
    if (n == 0 || tokens == 0) return;
    cq_launch_k(kv_meta_kernel<kReserve>, dim3(1), dim3(kMeta), seen_bytes(cache), (cudaStream_t)stream, *cache, slots, nullptr, n, tokens);
    cq_check_launch("kv_reserve");
}

extern "C" void cq_kv_fork(const cq_kv_cache *cache, const int *src, const int *dst, int n, int deep, void *stream) {
    if (!slots_ok(cache, src, dst, n, "kv_fork")) return;
    if (n == 0) return;
    cq_launch_k(kv_meta_kernel<kFork>, dim3(1), dim3(kMeta), seen_bytes(cache), (cudaStream_t)stream, *cache, src, dst, n, deep ? 1 : 0);
    cq_launch_k(kv_copy_kernel<false>, dim3(cq_sm_count() * 8), dim3(kCopyThreads), 0, (cudaStream_t)stream, *cache);
    cq_check_launch("kv_fork");
}

extern "C" void cq_kv_free(const cq_kv_cache *cache, const int *slots, int n, void *stream) {
    if (!slots_ok(cache, slots, slots, n, "kv_free")) return;
    if (n == 0) return;
    cq_launch_k(kv_meta_kernel<kFree>, dim3(1), dim3(kMeta), seen_bytes(cache), (cudaStream_t)stream, *cache, slots, nullptr, n, 0);
    cq_check_launch("kv_free");
}

extern "C" void cq_kv_compact(const cq_kv_cache *cache, void *stream) {
    if (!cache_ok(cache, "kv_compact")) return;
    cq_launch_k(kv_compact_kernel, dim3(1), dim3(kMeta), 0, (cudaStream_t)stream, *cache);
    cq_launch_k(kv_copy_kernel<true>, dim3(cq_sm_count() * 8), dim3(kCopyThreads), 0, (cudaStream_t)stream, *cache);
    cq_check_launch("kv_compact");
}

extern "C" void cq_kv_append(const cq_kv_cache *cache, int layer, const int *slots, int batch, int t, const void *q, const void *k, const void *v, int in_elem,
                             int hq, int64_t q_stride, int64_t k_stride, int64_t v_stride, const float *cosv, const float *sinv, int max_pos, int neox,
                             void *q_out, void *stream) {
    if (!slots_ok(cache, slots, slots, batch, "kv_append")) return;
    if (!k || !v || t <= 0 || layer < 0 || layer >= cache->layers || !q != !q_out || (q && hq <= 0) || !cosv != !sinv || (cosv && max_pos <= 0) ||
        (in_elem != CQ_F32 && in_elem != CQ_F16 && in_elem != CQ_BF16)) {
        cq_set_status(CQ_ERR_BAD_ARG, "kv_append: null pointer, layer, head count, or element type out of range");
        return;
    }
    const int es = elem_bytes(in_elem);
    const int64_t width = (int64_t)cache->kv_heads * cache->head_dim, q_width = (int64_t)hq * cache->head_dim;
    if (((k_stride | v_stride) * es) % 16 || (q && (q_stride * es) % 16) || k_stride < width || v_stride < width || (q && q_stride < q_width) ||
        (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)cosv | (uintptr_t)sinv) & 15)) {
        cq_set_status(CQ_ERR_BAD_ARG, "kv_append: rows must be 16-byte aligned and not overlap");
        return;
    }
    if (q && q == q_out && (in_elem != cache->elem || (q_stride != q_width && (int64_t)batch * t > 1))) {
        cq_set_status(CQ_ERR_BAD_ARG, "kv_append: q_out may be q only with the same type and rows without gaps");
        return;
    }
    if ((int64_t)batch * t > (1 << 30)) { cq_set_status(CQ_ERR_UNSUPPORTED, "kv_append: at most 2^30 rows in a call"); return; }
    if (batch == 0) return;
    const AppendArgs a{slots, q, k, v, q_out, cosv, sinv, q_stride, k_stride, v_stride, layer, batch, t, hq, max_pos, neox};
    cudaStream_t st = (cudaStream_t)stream;
    switch (in_elem * 3 + cache->elem) {
        case 0: append_launch<float, float>(*cache, a, st); break;
        case 1: append_launch<float, __half>(*cache, a, st); break;
        case 2: append_launch<float, __nv_bfloat16>(*cache, a, st); break;
        case 3: append_launch<__half, float>(*cache, a, st); break;
        case 4: append_launch<__half, __half>(*cache, a, st); break;
        case 5: append_launch<__half, __nv_bfloat16>(*cache, a, st); break;
        case 6: append_launch<__nv_bfloat16, float>(*cache, a, st); break;
        case 7: append_launch<__nv_bfloat16, __half>(*cache, a, st); break;
        default: append_launch<__nv_bfloat16, __nv_bfloat16>(*cache, a, st);
    }
    cq_check_launch("kv_append");
}

extern "C" int cq_kv_take_fault(const cq_kv_cache *cache, void *stream) {
    if (!cache_ok(cache, "kv_take_fault")) return -1;
    static const char *const text[] = {"", "a slot is out of range, named twice, or source and destination at once", "out of pages",
                                       "a sequence would be longer than its table", "fork into a slot that is not empty", "a table names a page that is not there",
                                       "a position before the sequence, in a shared page, or past its table or the rotary tables", "a wait inside the attention gave up"};
    int fault = 0;
    const int zero = 0;
    cudaStream_t st = (cudaStream_t)stream;
    if (cudaMemcpyAsync(&fault, cache->state, sizeof fault, cudaMemcpyDeviceToHost, st) != cudaSuccess || cudaStreamSynchronize(st) != cudaSuccess ||
        (fault && (cudaMemcpyAsync(cache->state, &zero, sizeof zero, cudaMemcpyHostToDevice, st) != cudaSuccess || cudaStreamSynchronize(st) != cudaSuccess))) {
        cq_check_launch("kv_take_fault");
        return -1;
    }
    if (fault) {
        char msg[160];
        std::snprintf(msg, sizeof msg, "kv cache: %s", fault > 0 && fault <= kTimeout ? text[fault] : "unknown fault");
        cq_set_status(fault == kTimeout ? CQ_ERR_TIMEOUT : CQ_ERR_BAD_ARG, msg);
    }
    return fault;
}
