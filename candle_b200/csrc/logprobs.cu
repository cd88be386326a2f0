// Log probabilities of given tokens, the entropy of their distributions, and the best alternatives, from rows of logits.
//
//   M = max x,  S = sum e^(x - M),  T = sum e^(x - M) (x - M):   log p(t) = (x_t - M) - ln S,   entropy = ln S - T / S
// (T <= 0, so the entropy is a sum of two terms that are not negative.)  Parts of a row are joined by M = max M_p, f_p = e^(M_p - M),
// S = sum f_p S_p, T = sum f_p (T_p + S_p (M_p - M)).
//
// One read of the logits is the bound.  A CTA holds a part of 8192 elements in registers, 32 a thread, so all its loads are in flight at
// once and the maximum, the sums and the alternatives need no second read.  The best `top` of a part: 64 groups of four threads have a
// maximum each, and the top-th largest of these is no higher than the top-th largest element; the elements from there on, some more
// than `top`, go to a list in shared memory and are ranked by counting.  Ties make the list long (a row of one value has 8192 of
// them): then the best is taken `top` times instead.
#include "../../include/candle_q_b200.h"
#include "common.cuh"

// Pointers carry no __restrict__: a read-only one would let the compiler move loads over the wait for the kernel before.
namespace {

constexpr int kThreads = 256, kPart = 8192, kPer = kPart / kThreads, kList = 512, kMaxTop = 32;

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
__device__ __forceinline__ uint64_t warp_max(uint64_t v) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) {
        const uint64_t o = __shfl_xor_sync(0xffffffffu, v, m);
        v = o > v ? o : v;
    }
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

// 16 bytes that are read once
__device__ __forceinline__ uint4 load16(const uint4 *p) {
    uint4 v;
    asm volatile("ld.global.cs.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
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

// Issue slots, not HBM, bound the first form of this kernel (some 2,000 a warp, 262 us for 1024 rows of 128256 f32); the parts inside a row have no masks, pairs
// of elements share an instruction, and the search for alternatives is only as long as `top` asks for.
template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_part_kernel(const T *logits, int64_t stride, int vocab, int parts, int top, Part *part_out,
                                                                 uint64_t *keys_out) {
    constexpr int V = 16 / sizeof(T), N = kPer / V;
    constexpr uint32_t kLowest = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;      // -inf, for what is not there
    __shared__ float red[3][8];
    __shared__ __align__(16) float group[64];
    __shared__ float least_s;
    __shared__ uint64_t list[kList];
    __shared__ int count;
    __shared__ uint64_t best[8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t r = blockIdx.x / parts;
    const int p = blockIdx.x - (int)r * parts;
    cq_pdl_launch_dependents();
    cq_pdl_wait();
    // 16-byte units from the one that holds the row's first element; elements before and behind the row are masked
    const T *row = logits + r * stride;
    const int shift = (int)(((uintptr_t)row & 15) / sizeof(T)), units = (vocab + shift + V - 1) / V, per = (units + parts - 1) / parts;
    const int u0 = p * per, u1 = min(units, u0 + per);
    const uint4 *src = reinterpret_cast<const uint4 *>(row - shift) + u0 + tid;
    uint4 w[N];
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = u0 + i * kThreads + tid < u1 ? load16(src + i * kThreads) : make_uint4(kLowest, kLowest, kLowest, kLowest);
    float x[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = element<T>(w[i / V], i % V);
    auto index_of = [&](int i) { return (u0 + i / V * kThreads + tid) * V + i % V - shift; };
    auto valid = [&](int i) { return u0 + i / V * kThreads + tid < u1 && (unsigned)index_of(i) < (unsigned)vocab; };
    if (p == 0 || p == parts - 1)               // the row's ends
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (!valid(i)) x[i] = -INFINITY;
    float mine = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPer; i += 2) mine = max3(mine, x[i], x[i + 1]);
    float m = mine;
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    if (top > 1 && (lane & 3) == 0) group[tid >> 2] = m;
#pragma unroll
    for (int k = 16; k > 2; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
    if (lane == 0) red[0][warp] = m;
    if (tid == 0) count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i += 2) m = max3(m, red[0][i], red[0][i + 1]);
    const float base = m == -INFINITY ? 0.0f : m;
    const uint64_t nbase = pack2(-base, -base), log2e = pack2(1.44269504f, 1.44269504f);
    uint64_t s2 = 0, t2 = 0;
#pragma unroll
    for (int i = 0; i < kPer; i += 2) {
        const uint64_t z = add2(pack2(x[i], x[i + 1]), nbase), y = mul2(z, log2e), e = pack2(ex2(lo(y)), ex2(hi(y)));
        s2 = add2(s2, e);
        t2 = fma2(e, z, t2);
    }
    float s = lo(s2) + hi(s2), t = lo(t2) + hi(t2);
    if (t != t) {               // 0 times an infinite distance: a logit of -inf has no share in it (from 150 on the weight is 0)
        t = 0.0f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const float z = x[i] - base;
            t = __fmaf_rn(ex2(z * 1.44269504f), fmaxf(z, -150.0f), t);
        }
    }
    s = warp_sum(s);
    t = warp_sum(t);
    if (lane == 0) { red[1][warp] = s; red[2][warp] = t; }
    // the top-th largest of the 64 groups' maxima: a warp ranks eight of them, four lanes each
    if (top > 1) {
        const int at = warp * 8 + (lane >> 2), j0 = (lane & 3) * 16;
        const float v = group[at];
        int rank = 0;
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            const float4 o = *reinterpret_cast<const float4 *>(&group[j0 + j]);
            rank += (o.x > v || (o.x == v && j0 + j < at)) + (o.y > v || (o.y == v && j0 + j + 1 < at)) + (o.z > v || (o.z == v && j0 + j + 2 < at)) +
                    (o.w > v || (o.w == v && j0 + j + 3 < at));
        }
        rank += __shfl_xor_sync(0xffffffffu, rank, 1);
        rank += __shfl_xor_sync(0xffffffffu, rank, 2);
        if (rank == top - 1 && (lane & 3) == 0) least_s = v;
    }
    __syncthreads();
    if (tid == 0) {
        s = red[1][0]; t = red[2][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) { s += red[1][i]; t += red[2][i]; }
        part_out[blockIdx.x] = Part{m, s, t, 0.0f};
    }
    if (top == 0) return;
    const float least = top > 1 ? least_s : m;
    if (mine >= least) {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (x[i] >= least && valid(i)) {
                const int at = atomicAdd(&count, 1);
                if (at < kList) list[at] = (uint64_t)ordered(x[i]) << 32 | (uint32_t)~index_of(i);
            }
    }
    __syncthreads();
    uint64_t *keys = keys_out + (int64_t)blockIdx.x * top;
    const int n = count;
    if (n <= kList) {
        for (int i = tid; i < n; i += kThreads) {
            const uint64_t k = list[i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += list[j] > k;
            if (rank < top) keys[rank] = k;
        }
        for (int i = n + tid; i < top; i += kThreads) keys[i] = 0;      // a part of fewer elements than `top`
        return;
    }
    uint64_t below = ~0ull;
    for (int a = 0; a < top; ++a) {
        uint64_t k = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const uint64_t c = valid(i) ? (uint64_t)ordered(x[i]) << 32 | (uint32_t)~index_of(i) : 0;
            if (c < below && c > k) k = c;
        }
        k = warp_max(k);
        __syncthreads();
        if (lane == 0) best[warp] = k;
        __syncthreads();
        below = best[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) below = best[i] > below ? best[i] : below;
        if (tid == 0) keys[a] = below;
    }
}

// One CTA per row: the parts' sums (first warp) beside the best of their lists.  The largest of the parts' last keys is no higher than the row's top-th key, which leaves few
// keys to rank.
constexpr int kJoin = 128, kHeld = 8;           // threads; keys a thread holds
template <typename T>
__global__ void __launch_bounds__(kJoin) logprobs_join_kernel(const T *logits, int64_t stride, int vocab, int parts, int top, const Part *part_in,
                                                              const uint64_t *keys_in, const Out o) {
    __shared__ float row_m, row_s;
    __shared__ uint64_t least_of[kJoin / 32];
    __shared__ uint64_t list[kList];
    __shared__ int count;
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, all = parts * top;
    cq_pdl_launch_dependents();
    cq_pdl_wait();
    const Part *part = part_in + r * parts;
    const uint64_t *keys = keys_in + r * all;
    // what every row needs is asked for at once
    uint64_t k[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) k[i] = tid + i * kJoin < all ? keys[tid + i * kJoin] : 0;
    if (warp == 0) {
        const int64_t tok = o.tokens ? o.tokens[r] : -1;
        const float at_tok = tok >= 0 && tok < vocab ? load_f(logits + r * stride + tok) : 0.0f;
        float m = -INFINITY, s = 0.0f, t = 0.0f;
        const Part first = lane < parts ? part[lane] : Part{-INFINITY, 0.0f, 0.0f, 0.0f};
        m = first.m;
        for (int p = lane + 32; p < parts; p += 32) m = fmaxf(m, part[p].m);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
        for (int p = lane; p < parts; p += 32) {
            const Part a = p == lane ? first : part[p];
            if (a.s != 0.0f) {                              // nothing but -inf: no weight, and no difference of infinities
                const float d = fmaxf(a.m - m, -150.0f), f = expf(d);       // the difference of two finite values may be -inf
                s = __fmaf_rn(f, a.s, s);
                t = __fmaf_rn(f, __fmaf_rn(a.s, d, a.t), t);
            }
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
    }
    if (top == 0) return;
    uint64_t least = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) least = (tid + i * kJoin) % top == top - 1 && k[i] > least ? k[i] : least;
    for (int i = tid + kHeld * kJoin; i < all; i += kJoin) least = i % top == top - 1 && keys[i] > least ? keys[i] : least;
    least = warp_max(least);
    if (lane == 0) least_of[warp] = least;
    if (tid == 0) count = 0;
    __syncthreads();
    least = least_of[0];
#pragma unroll
    for (int i = 1; i < kJoin / 32; ++i) least = least_of[i] > least ? least_of[i] : least;
    const float m = row_m, s = row_s, ls = logf(s);
    const bool ok = s > 0.0f && m < INFINITY;
    if (!ok) {
        if (tid < top) write_top(o, r, top, tid, 0, false, m, ls);
        return;
    }
    auto take = [&](uint64_t key) {
        if (key >= least && key != 0) {
            const int at = atomicAdd(&count, 1);
            if (at < kList) list[at] = key;
        }
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i) take(k[i]);
    for (int i = tid + kHeld * kJoin; i < all; i += kJoin) take(keys[i]);
    __syncthreads();
    // keys differ, so at most (parts - 1) * (top - 1) + top of them are not below `least`; where the list is too short for that, all are ranked
    const int n = count;
    const uint64_t *from = n <= kList ? list : keys;
    const int total = n <= kList ? n : all;
    for (int i = tid; i < total; i += kJoin) {
        const uint64_t key = from[i];
        if (key < least || key == 0) continue;
        int rank = 0;
        for (int j = 0; j < total; ++j) rank += from[j] > key;
        if (rank < top) write_top(o, r, top, rank, key, ok, m, ls);
    }
}

int parts_of(int vocab) { return (int)(((int64_t)vocab + 8 + kPart - 1) / kPart); }        // + 8: a row may start inside a 16-byte unit

template <typename T>
void launch(const void *logits, int64_t stride, int rows, int vocab, int top, const Out &o, void *scratch, cudaStream_t st) {
    const int parts = parts_of(vocab);
    Part *part = reinterpret_cast<Part *>(scratch);
    uint64_t *keys = reinterpret_cast<uint64_t *>(part + (int64_t)rows * parts);
    cq_launch_k(logprobs_part_kernel<T>, dim3((unsigned)((int64_t)rows * parts)), dim3(kThreads), 0, st, (const T *)logits, stride, vocab, parts, top, part, keys);
    cq_launch_k(logprobs_join_kernel<T>, dim3((unsigned)rows), dim3(kJoin), 0, st, (const T *)logits, stride, vocab, parts, top, (const Part *)part,
                (const uint64_t *)keys, o);
}

}  // namespace

extern "C" size_t cq_token_logprobs_scratch_bytes(int rows, int vocab, int top) {
    if (rows <= 0 || vocab <= 0 || top < 0 || top > kMaxTop || top > vocab || (int64_t)rows * parts_of(vocab) > INT32_MAX) return 0;
    return (size_t)rows * parts_of(vocab) * (sizeof(Part) + 8 * (size_t)top);
}

extern "C" void cq_token_logprobs(const void *logits, int elem, int64_t row_stride, int rows, int vocab, const int64_t *tokens, int top, float *logprob, float *entropy,
                                  float *top_logprobs, int64_t *top_ids, void *scratch, void *stream) {
    if (!logits || !entropy || !scratch || !tokens != !logprob || (top > 0 && (!top_logprobs || !top_ids)) || ((uintptr_t)scratch & 15) ||
        (elem != CQ_F32 && elem != CQ_F16 && elem != CQ_BF16) || (uintptr_t)logits % (elem == CQ_F32 ? 4 : 2)) {
        cq_set_status(CQ_ERR_BAD_ARG, "token_logprobs: null or misaligned pointer, or an element type that is not f32, f16 or bf16");
        return;
    }
    if (cq_token_logprobs_scratch_bytes(rows, vocab, top) == 0 || row_stride < 0 || vocab > (1 << 30)) {
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
