// Log probabilities of given tokens, the entropy of their distributions, and the best alternatives, from rows of logits.
//
//   S = sum e^(x - M),  T = sum e^(x - M) (x - M):   log p(t) = (x_t - M) - ln S,   entropy = ln S - T / S
// with any M near the maximum: here an element of the row, the maximum or no more than 2 below it.  With the maximum T <= 0 and the entropy is a sum of two terms that are not
// negative.  With less T may be positive and the entropy a difference, but not a small one: M's own element has at least e^-2 of the largest weight then, so that the entropy is
// 0.36 or more.  Parts of a row are joined by M = max M_p, f_p = e^(M_p - M), S = sum f_p S_p, T = sum f_p (T_p + S_p (M_p - M)).
//
// One read of the logits is the bound.  A warp walks one segment of a row in chunks of 1024 elements, 32 a lane, the next chunk on its way to shared memory; nothing waits
// for another warp.  Each lane keeps a maximum, S and T of its own; the maximum follows only where a chunk's is more than 2 higher (S and T have any base near the maximum;
// lanes, then segments, are joined as above).  The best `top` so far lie in the lanes in order; a chunk whose maximum does not pass the last of them - after the first few
// nearly every one - costs them a vote.  Else its elements from there on are ranked against the list by counting.  (With a CTA per 8192 elements, a maximum of the
// CTA first and a list for its candidates, 1024 rows of 128256 f32 took 141 us: a warp in search of candidates held up the seven others.)
// Those 1024 rows, 525 MB: 94 us, 5.6 TB/s.  64 rows of 151936 bf16 with five alternatives: 14.5 us from cold caches, where HBM would want 3: each warp has three chunks, and the first of
// them costs it a list.
#include "../../include/candle_q_b200.h"
#include "common.cuh"

// Pointers carry no __restrict__: a read-only one would let the compiler move loads over the wait for the kernel before.
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kCtas = 3, kPer = 32, kChunk = 32 * kPer, kMaxTop = 32, kMaxSegments = 128;

// Keys order elements by (value descending, index ascending) as one unsigned comparison; 0: not an element of the row.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);               // -0 is 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }

struct Part { float m, s, t, pad; };

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}
// A row's values from its joined parts.
struct Out {
    const int64_t *tokens;
    float *logprob, *entropy, *top_logprobs;
    int64_t *top_ids;
};
template <typename T> __device__ __forceinline__ float load_f(const T *p) {
    if constexpr (sizeof(T) == 4) return *p;
    else if constexpr (std::is_same<T, __half>::value) return __half2float(*p);
    else return __bfloat162float(*p);
}
__device__ __forceinline__ void write_top(const Out &o, int64_t r, int top, int rank, uint64_t key, bool ok, float m, float ls) {
    o.top_logprobs[r * top + rank] = ok ? (value_of((uint32_t)(key >> 32)) - m) - ls : NAN;
    o.top_ids[r * top + rank] = ok ? (int64_t)(~(uint32_t)key) : -1;
}

template <typename T> __device__ __forceinline__ float element(const uint4 &w, int j) {
    const uint32_t b[4] = {w.x, w.y, w.z, w.w};
    if constexpr (sizeof(T) == 4) return __uint_as_float(b[j]);
    else if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)(b[j / 2] >> (16 * (j & 1)))));
    else return __uint_as_float(j & 1 ? b[j / 2] & 0xffff0000u : b[j / 2] << 16);
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// two f32 operations per instruction
__device__ __forceinline__ uint64_t pack2(float a, float b) { return (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a); }
__device__ __forceinline__ float lo(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

template <typename T> struct Warp {
    static constexpr int kUnits = kPer * (int)sizeof(T) / 16;          // 16-byte units of a chunk, a lane
    uint4 ring[2][kUnits][32];
    uint64_t found[64];                                               // candidates not yet in the list
};

template <typename T>
__global__ void __launch_bounds__(kThreads, kCtas) logprobs_segment_kernel(const T *logits, int64_t stride, int vocab, int segments, int per_segment, int total, int top, Part *part_out,
                                                                           uint64_t *keys_out) {
    constexpr int V = 16 / sizeof(T), N = Warp<T>::kUnits;
    constexpr uint32_t kLowest = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;      // -inf, for what is not there
    extern __shared__ __align__(16) uint8_t raw[];
    const int lane = threadIdx.x & 31;
    Warp<T> &sm = reinterpret_cast<Warp<T> *>(raw)[threadIdx.x >> 5];
    cq_pdl_launch_dependents();
    cq_pdl_wait();
#pragma unroll 1
    for (int at = blockIdx.x * kWarps + (threadIdx.x >> 5); at < total; at += gridDim.x * kWarps) {
        // 16-byte units from the one that holds the row's first element; elements before and behind the row are masked
        const int r = at / segments, sg = at - r * segments;
        const T *row = logits + r * stride;
        const int shift = (int)(((uintptr_t)row & 15) / sizeof(T)), units = (vocab + shift + V - 1) / V;
        const int u0 = sg * per_segment * N * 32, chunks = min(per_segment, max((units - u0 + N * 32 - 1) / (N * 32), 0));
        const uint4 *src = reinterpret_cast<const uint4 *>(row - shift) + lane;
        auto bring = [&](int c) {
            if (c < chunks) {
                const int u = u0 + c * N * 32;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    uint4 *to = &sm.ring[c & 1][i][lane];
                    if (u + i * 32 + lane < units) cq_cp_async16(to, src + u + i * 32);
                    else *to = make_uint4(kLowest, kLowest, kLowest, kLowest);
                }
            }
            cq_cp_async_commit();
        };
        float m = -INFINITY, s = 0.0f, t = 0.0f;
        uint64_t best = 0;                      // the lane-th best so far
        float bound = -INFINITY;                // elements from here on may belong to them
        bring(0);
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
            bring(c + 1);
            cq_cp_async_wait<1>();
            const int u = u0 + c * N * 32 + lane;
            const bool edge = u0 + c == 0 || u0 + (c + 1) * N * 32 >= units;            // of the row: with elements that are not of it
            auto index_of = [&](int i, int j) { return (u + i * 32) * V + j - shift; };
            float x[kPer];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const uint4 w = sm.ring[c & 1][i][lane];
#pragma unroll
                for (int j = 0; j < V; ++j) x[i * V + j] = element<T>(w, j);
            }
            if (edge)
#pragma unroll
                for (int i = 0; i < kPer; ++i)
                    if ((unsigned)index_of(i / V, i % V) >= (unsigned)vocab) x[i] = -INFINITY;
            float mine = -INFINITY, other = -INFINITY;
#pragma unroll
            for (int i = 0; i < kPer; i += 4) { mine = max3(mine, x[i], x[i + 1]); other = max3(other, x[i + 2], x[i + 3]); }
            mine = fmaxf(mine, other);
            if (__any_sync(0xffffffffu, mine > m + 2.0f)) {
                if (mine > m + 2.0f) {
                    const float d = fmaxf(m - mine, -150.0f), f = ex2(d * 1.44269504f);      // from -inf: S and T are 0
                    t = f * __fmaf_rn(s, d, t);
                    s *= f;
                    m = mine;
                }
            }
            const float base = m == -INFINITY ? 0.0f : m;
            const uint64_t nbase = pack2(-base, -base), log2e = pack2(1.44269504f, 1.44269504f);
            uint64_t s2 = 0, t2 = 0;
#pragma unroll
            for (int i = 0; i < kPer; i += 2) {
                const uint64_t z = add2(pack2(x[i], x[i + 1]), nbase), y = mul2(z, log2e), e = pack2(ex2(lo(y)), ex2(hi(y)));
                s2 = add2(s2, e);
                t2 = fma2(e, z, t2);
            }
            float tc = lo(t2) + hi(t2);
            if (tc != tc) {             // 0 times an infinite distance: a logit of -inf has no share in it (from 150 on the weight is 0)
                tc = 0.0f;
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    const float z = x[i] - base;
                    tc = __fmaf_rn(ex2(z * 1.44269504f), fmaxf(z, -150.0f), tc);
                }
            }
            s += lo(s2) + hi(s2);
            t += tc;
            if (top == 0) continue;
            if (top == 1) {                     // a lane's own best, its first among equals
                if (mine > bound || best == 0) {
                    int at_i = kPer;
#pragma unroll
                    for (int i = kPer - 1; i >= 0; --i)
                        if (x[i] == mine && (!edge || (u + i / V * 32 < units && (unsigned)index_of(i / V, i % V) < (unsigned)vocab))) at_i = i;
                    if (at_i < kPer && u + at_i / V * 32 < units) {
                        best = (uint64_t)ordered(mine) << 32 | (uint32_t)~index_of(at_i / V, at_i % V);
                        bound = mine;
                    }
                }
                continue;
            }
            const unsigned over = __ballot_sync(0xffffffffu, mine >= bound);
            if (!over) continue;
            // the top-th largest of the lanes' maxima is no higher than the chunk's top-th element
            if (__popc(over) >= top) {
                float *maxima = reinterpret_cast<float *>(sm.found);
                maxima[lane] = mine;
                __syncwarp();
                int rank = 0;
#pragma unroll
                for (int y = 0; y < 32; y += 4) {
                    const float4 v = *reinterpret_cast<const float4 *>(maxima + y);
                    rank += (v.x > mine || (v.x == mine && y < lane)) + (v.y > mine || (v.y == mine && y + 1 < lane)) + (v.z > mine || (v.z == mine && y + 2 < lane)) +
                            (v.w > mine || (v.w == mine && y + 3 < lane));
                }
                bound = fmaxf(bound, __shfl_sync(0xffffffffu, mine, __ffs(__ballot_sync(0xffffffffu, rank == top - 1)) - 1));
                __syncwarp();
            }
            uint32_t hits = 0;
#pragma unroll
            for (int i = 0; i < kPer; ++i) hits |= (uint32_t)(x[i] >= bound) << i;
            int n = 0;
            // 32 found ones and the list, each ranked among all
            auto merge = [&](int from, int count) {
                __syncwarp();
                const uint64_t key = lane < count ? sm.found[from + lane] : 0;
                int rank_list = lane, rank_key = 0;
#pragma unroll 4
                for (int y = 0; y < count; ++y) {
                    const uint64_t k = __shfl_sync(0xffffffffu, key, y);
                    const int above = __popc(__ballot_sync(0xffffffffu, best > k));
                    rank_list += k > best;
                    rank_key += (k > key) + (y == lane ? above : 0);
                }
                __syncwarp();
                // over the keys that were just read
                if (best != 0 && rank_list < 32) sm.found[from + rank_list] = best;
                if (key != 0 && rank_key < 32) sm.found[from + rank_key] = key;
                const int filled = min(32, __popc(__ballot_sync(0xffffffffu, best != 0)) + count);
                __syncwarp();
                best = lane < filled ? sm.found[from + lane] : 0;
                __syncwarp();
                const uint64_t last = __shfl_sync(0xffffffffu, best, top - 1);
                if (last != 0) bound = fmaxf(bound, value_of((uint32_t)(last >> 32)));
            };
#pragma unroll 1
            while (__any_sync(0xffffffffu, hits != 0)) {            // one of each lane's at a time
                const int i = __ffs(hits) - 1, e = index_of(i / V, i % V);
                const bool there = hits != 0 && u + i / V * 32 < units && (unsigned)e < (unsigned)vocab;
                const float v = there ? load_f(reinterpret_cast<const T *>(&sm.ring[c & 1][i / V][lane]) + i % V) : 0.0f;
                const bool in = there && v >= bound;                // it may have risen
                const unsigned votes = __ballot_sync(0xffffffffu, in);
                if (in) sm.found[n + __popc(votes & ((1u << lane) - 1))] = (uint64_t)ordered(v) << 32 | (uint32_t)~e;
                n += __popc(votes);
                hits &= hits - 1;
                if (n >= 32) { n -= 32; merge(n, 32); }
            }
            if (n) merge(0, n);
            // later chunks have higher indices: an equal one is no better
            const uint64_t last = __shfl_sync(0xffffffffu, best, top - 1);
            bound = last ? value_of((uint32_t)(last >> 32) + 1) : -INFINITY;
        }
        // the lanes' sums, relative to their largest maximum
        float big = m;
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, k));
        const float d = s != 0.0f ? fmaxf(m - big, -150.0f) : 0.0f, f = expf(d);
        t = warp_sum(f * __fmaf_rn(s, d, t));
        s = warp_sum(f * s);
        if (lane == 0) part_out[at] = Part{big, s, t, 0.0f};
        if (top == 1)
#pragma unroll
            for (int k = 16; k > 0; k >>= 1) {
                const uint64_t o = __shfl_xor_sync(0xffffffffu, best, k);
                best = o > best ? o : best;
            }
        if (lane < top) keys_out[(int64_t)at * top + lane] = best;
    }
}

// One CTA per row.  All bring the segments' lists to shared memory; one warp then joins the sums, another one merges the lists, which are in order: a lane has the heads of four, and
// the largest of all heads is the next one.  (With what remains above a bound ranked by all warps one row of 128256 took, in a graph, 11.1 us for five alternatives and 13.5 for 20;
// so it takes 6.2 and 10.3.  Where 32 are asked for of 8 rows or more the ranking was 1.3 us faster.)
constexpr int kJoin = 256;
template <typename T>
__global__ void __launch_bounds__(kJoin) logprobs_join_kernel(const T *logits, int64_t stride, int vocab, int segments, int top, const Part *part_in, const uint64_t *keys_in,
                                                              const Out o) {
    extern __shared__ uint64_t lists[];             // [segments][top]
    __shared__ float row_m, row_s;
    __shared__ uint64_t best[kMaxTop];
    constexpr int kLane = kMaxSegments / 32, kAtOnce = 8;
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, all = segments * top;
    cq_pdl_launch_dependents();
    cq_pdl_wait();
    const Part *part = part_in + r * segments;
    const uint64_t *keys = keys_in + r * all;
    int64_t tok = -1;
    Part a[kLane];
    if (warp == 1) {
        if (o.tokens) tok = o.tokens[r];
#pragma unroll
        for (int i = 0; i < kLane; ++i) a[i] = lane + 32 * i < segments ? part[lane + 32 * i] : Part{-INFINITY, 0.0f, 0.0f, 0.0f};
    }
#pragma unroll 1
    for (int i0 = tid; i0 < all; i0 += kAtOnce * blockDim.x) {
        uint64_t v[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) v[i] = i0 + i * (int)blockDim.x < all ? keys[i0 + i * blockDim.x] : 0;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
            if (i0 + i * (int)blockDim.x < all) lists[i0 + i * blockDim.x] = v[i];
    }
    const float at_tok = tok >= 0 && tok < vocab ? load_f(logits + r * stride + tok) : 0.0f;
    __syncthreads();
    if (warp == 1) {
        float m = -INFINITY, s = 0.0f, t = 0.0f;
#pragma unroll
        for (int i = 0; i < kLane; ++i) m = fmaxf(m, a[i].m);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
#pragma unroll
        for (int i = 0; i < kLane; ++i)
            if (a[i].s != 0.0f) {                               // nothing but -inf: no weight, and no difference of infinities
                const float d = fmaxf(a[i].m - m, -150.0f), f = expf(d);        // the difference of two finite values may be -inf
                s = __fmaf_rn(f, a[i].s, s);
                t = __fmaf_rn(f, __fmaf_rn(a[i].s, d, a[i].t), t);
            }
        s = warp_sum(s);
        t = warp_sum(t);
        if (lane == 0) {
            const bool ok = s > 0.0f && m < INFINITY;       // a NaN or +inf among the logits, or nothing but -inf: no distribution
            const float ls = logf(s);
            o.entropy[r] = ok ? ls - __fdiv_rn(t, s) : NAN;
            if (o.tokens) o.logprob[r] = tok < 0 ? 0.0f : tok >= vocab || !ok ? NAN : (at_tok - m) - ls;
            row_m = m;
            row_s = s;
        }
    } else if (warp == 0) {
        uint64_t head[kLane], after[kLane];
        int next[kLane];
#pragma unroll
        for (int i = 0; i < kLane; ++i) {
            const int first = (lane + 32 * i) * top;
            head[i] = first < all ? lists[first] : 0;
            after[i] = first < all && top > 1 ? lists[first + 1] : 0;
            next[i] = first + 2;
        }
#pragma unroll 1
        for (int k = 0; k < top; ++k) {
            uint64_t mine = head[0];
#pragma unroll
            for (int i = 1; i < kLane; ++i) mine = head[i] > mine ? head[i] : mine;
            const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(mine >> 32));
            const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(mine >> 32) == hi ? (uint32_t)mine : 0u);
            const uint64_t key = (uint64_t)hi << 32 | lo;
            if (lane == 0) best[k] = key;
#pragma unroll
            for (int i = 0; i < kLane; ++i)
                if (head[i] == key && key != 0) {               // one lane's: indices differ
                    head[i] = after[i];
                    after[i] = next[i] < (lane + 32 * i + 1) * top ? lists[next[i]] : 0;
                    ++next[i];
                }
        }
    }
    if (top == 0) return;
    __syncthreads();
    const float m = row_m, s = row_s;
    if (tid < top) write_top(o, r, top, tid, best[tid], s > 0.0f && m < INFINITY, m, logf(s));
}

int chunks_of(int vocab) { return (int)(((int64_t)vocab + 8 + kChunk - 1) / kChunk); }     // + 8: a row may start inside a 16-byte unit

// Segments of a row: one for every warp that the device holds, or, with more rows than warps, the number up to eight that leaves the fewest chunks to the busiest warp.
int segments_of(int rows, int vocab) {
    const int chunks = chunks_of(vocab), warps = kCtas * kWarps * cq_sm_count();
    int s = rows <= warps ? warps / rows : 1;
    if (rows > warps) {
        int64_t least = INT64_MAX;
        for (int x = 1; x <= 8; ++x) {
            const int64_t cost = ((int64_t)rows * x + warps - 1) / warps * ((chunks + x - 1) / x);
            if (cost < least) { least = cost; s = x; }
        }
    }
    if (s > chunks) s = chunks;
    if (s > kMaxSegments) s = kMaxSegments;
    const int per = (chunks + s - 1) / s;
    return (chunks + per - 1) / per;
}

template <typename T>
void launch(const void *logits, int64_t stride, int rows, int vocab, int top, const Out &o, void *scratch, cudaStream_t st) {
    const int segments = segments_of(rows, vocab), per = (chunks_of(vocab) + segments - 1) / segments, total = rows * segments;
    Part *part = reinterpret_cast<Part *>(scratch);
    uint64_t *keys = reinterpret_cast<uint64_t *>(part + total);
    constexpr int smem = kWarps * (int)sizeof(Warp<T>);
    static bool done[64];
    cq_smem_once((const void *)logprobs_segment_kernel<T>, smem, done);
    const int most = kCtas * cq_sm_count(), want = (total + kWarps - 1) / kWarps;
    cq_launch_k(logprobs_segment_kernel<T>, dim3((unsigned)(want < most ? want : most)), dim3(kThreads), smem, st, (const T *)logits, stride, vocab, segments, per, total, top, part,
                keys);
    cq_launch_k(logprobs_join_kernel<T>, dim3((unsigned)rows), dim3(top > 1 ? kJoin : 64), 8 * segments * top, st, (const T *)logits, stride, vocab, segments, top, (const Part *)part,
                (const uint64_t *)keys, o);
}

}  // namespace

extern "C" size_t cq_token_logprobs_scratch_bytes(int rows, int vocab, int top) {
    if (rows <= 0 || vocab <= 0 || vocab > (1 << 30) || top < 0 || top > kMaxTop || top > vocab || (int64_t)rows * kMaxSegments > (1 << 30)) return 0;
    return (size_t)rows * segments_of(rows, vocab) * (sizeof(Part) + 8 * (size_t)top);
}

extern "C" void cq_token_logprobs(const void *logits, int elem, int64_t row_stride, int rows, int vocab, const int64_t *tokens, int top, float *logprob, float *entropy,
                                  float *top_logprobs, int64_t *top_ids, void *scratch, void *stream) {
    if (!logits || !entropy || !scratch || !tokens != !logprob || (top > 0 && (!top_logprobs || !top_ids)) || ((uintptr_t)scratch & 15) ||
        (elem != CQ_F32 && elem != CQ_F16 && elem != CQ_BF16) || (uintptr_t)logits % (elem == CQ_F32 ? 4 : 2)) {
        cq_set_status(CQ_ERR_BAD_ARG, "token_logprobs: null or misaligned pointer, or an element type that is not f32, f16 or bf16");
        return;
    }
    if (cq_token_logprobs_scratch_bytes(rows, vocab, top) == 0 || row_stride < 0) {
        cq_set_status(CQ_ERR_BAD_ARG, "token_logprobs: rows and vocab must be positive, 0 <= top <= min(32, vocab)");
        return;
    }
    const Out o{tokens, logprob, entropy, top_logprobs, top_ids};
    cudaStream_t st = (cudaStream_t)stream;
    if (elem == CQ_F32) launch<float>(logits, row_stride, rows, vocab, top, o, scratch, st);
    else if (elem == CQ_F16) launch<__half>(logits, row_stride, rows, vocab, top, o, scratch, st);
    else launch<__nv_bfloat16>(logits, row_stride, rows, vocab, top, o, scratch, st);
    cq_check_launch("token_logprobs");
}
