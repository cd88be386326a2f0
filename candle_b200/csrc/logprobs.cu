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
template <typename T>
__device__ __forceinline__ void write_row(const Out &o, const T *row, int64_t r, int vocab, float m, float s, float t) {
    const bool ok = s > 0.0f && m < INFINITY;       // a NaN or +inf among the logits, or nothing but -inf: no distribution
    const float ls = logf(s);
    o.entropy[r] = ok ? ls - __fdiv_rn(t, s) : NAN;
    if (o.tokens) {
        const int64_t tok = o.tokens[r];
        o.logprob[r] = tok < 0 ? 0.0f : tok >= vocab || !ok ? NAN : (load_f(row + tok) - m) - ls;
    }
}
__device__ __forceinline__ void write_top(const Out &o, int64_t r, int top, int rank, uint64_t key, bool ok, float m, float ls) {
    o.top_logprobs[r * top + rank] = ok ? (value_of((uint32_t)(key >> 32)) - m) - ls : NAN;
    o.top_ids[r * top + rank] = ok ? (int64_t)(~(uint32_t)key) : -1;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_part_kernel(const T *__restrict__ logits, int64_t stride, int vocab, int parts, int top, Part *__restrict__ part_out,
                                                                 uint64_t *__restrict__ keys_out) {
    constexpr int V = 16 / sizeof(T), N = kPer / V;
    __shared__ float red[3][8];
    __shared__ uint32_t group[64];
    __shared__ uint64_t list[kList];
    __shared__ int count;
    __shared__ uint64_t best[8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t r = blockIdx.x / parts;
    const int p = blockIdx.x % parts;
    cq_pdl_launch_dependents();
    cq_pdl_wait();
    // 16-byte units from the one that holds the row's first element; elements before and behind the row are masked
    const T *row = logits + r * stride;
    const int shift = (int)(((uintptr_t)row & 15) / sizeof(T)), units = (vocab + shift + V - 1) / V, per = (units + parts - 1) / parts;
    const int u0 = p * per, u1 = min(units, u0 + per);
    const uint4 *src = reinterpret_cast<const uint4 *>(row - shift);
    uint4 w[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int u = u0 + i * kThreads + tid;
        w[i] = u < u1 ? __ldcs(src + u) : make_uint4(0, 0, 0, 0);
    }
    float x[kPer];
    float mine = -INFINITY;
    uint32_t valid = 0;             // bit per element
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t b[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
        const int u = u0 + i * kThreads + tid, e0 = u * V - shift;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float f;
            if constexpr (sizeof(T) == 4) f = __uint_as_float(b[j]);
            else if constexpr (std::is_same<T, __half>::value) f = __half2float(__ushort_as_half((unsigned short)(b[j / 2] >> (16 * (j & 1)))));
            else f = __uint_as_float(j & 1 ? b[j / 2] & 0xffff0000u : b[j / 2] << 16);
            const bool in = u < u1 && e0 + j >= 0 && e0 + j < vocab;
            x[i * V + j] = in ? f : -INFINITY;
            valid |= (uint32_t)in << (i * V + j);
            mine = fmaxf(mine, x[i * V + j]);
        }
    }
    float g = mine;
    g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, 1));
    g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, 2));
    if ((lane & 3) == 0) group[tid >> 2] = ordered(g);
    float m = g;
#pragma unroll
    for (int k = 16; k > 2; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
    if (lane == 0) red[0][warp] = m;
    if (tid == 0) count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, red[0][i]);
    const float base = m == -INFINITY ? 0.0f : m;
    float s = 0.0f, t = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const float z = x[i] - base, e = exp2f(z * 1.44269504f);
        s += e;
        t = __fmaf_rn(e, fmaxf(z, -150.0f), t);         // e is 0 from there on: -inf must not meet it
    }
    s = warp_sum(s);
    t = warp_sum(t);
    if (lane == 0) { red[1][warp] = s; red[2][warp] = t; }
    // the top-th largest of the 64 groups' maxima
    uint32_t least = 1;
    if (top > 0) {
        const uint32_t a = group[lane], b = group[lane + 32];
        int ra = 0, rb = 0;
#pragma unroll 8
        for (int i = 0; i < 64; ++i) {
            const uint32_t o = group[i];
            ra += o > a || (o == a && i < lane);
            rb += o > b || (o == b && i < lane + 32);
        }
        least = __reduce_max_sync(0xffffffffu, ra == top - 1 ? a : rb == top - 1 ? b : 0u);
        const uint32_t omine = ordered(mine);
        if (omine >= least && valid) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const uint32_t o = ordered(x[i]);
                if ((valid >> i & 1) && o >= least) {
                    const int at = atomicAdd(&count, 1), e = (u0 + i / V * kThreads + tid) * V + i % V - shift;
                    if (at < kList) list[at] = (uint64_t)o << 32 | (uint32_t)~e;
                }
            }
        }
    }
    __syncthreads();
    if (tid == 0) {
        s = red[1][0]; t = red[2][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) { s += red[1][i]; t += red[2][i]; }
        part_out[blockIdx.x] = Part{m, s, t, 0.0f};
    }
    if (top == 0) return;
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
            const int e = (u0 + i / V * kThreads + tid) * V + i % V - shift;
            const uint64_t c = valid >> i & 1 ? (uint64_t)ordered(x[i]) << 32 | (uint32_t)~e : 0;
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

// One CTA per row: the parts' sums, then the best of their lists.  The largest of the parts' last keys is no higher than the row's top-th key.
template <typename T>
__global__ void __launch_bounds__(128) logprobs_join_kernel(const T *__restrict__ logits, int64_t stride, int vocab, int parts, int top, const Part *__restrict__ part_in,
                                                            const uint64_t *__restrict__ keys_in, const Out o) {
    __shared__ float row_m, row_s;
    __shared__ uint64_t least_of[4];
    __shared__ uint64_t list[kList];
    __shared__ int count;
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    cq_pdl_launch_dependents();
    cq_pdl_wait();
    const Part *part = part_in + r * parts;
    const uint64_t *keys = keys_in + r * parts * top;
    if (warp == 0) {
        float m = -INFINITY;
        for (int p = lane; p < parts; p += 32) m = fmaxf(m, part[p].m);
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
        float s = 0.0f, t = 0.0f;
        for (int p = lane; p < parts; p += 32) {
            const Part a = part[p];
            if (a.s != 0.0f) {                              // nothing but -inf: no weight, and no difference of infinities
                const float d = fmaxf(a.m - m, -150.0f), f = expf(d);       // the difference of two finite values may be -inf
                s = __fmaf_rn(f, a.s, s);
                t = __fmaf_rn(f, __fmaf_rn(a.s, d, a.t), t);
            }
        }
        s = warp_sum(s);
        t = warp_sum(t);
        if (lane == 0) {
            write_row(o, logits + r * stride, r, vocab, m, s, t);
            row_m = m;
            row_s = s;
        }
    }
    if (top == 0) return;
    uint64_t least = 0;
    for (int p = tid; p < parts; p += 128) {
        const uint64_t k = keys[(int64_t)p * top + top - 1];
        least = k > least ? k : least;
    }
    least = warp_max(least);
    if (lane == 0) least_of[warp] = least;
    if (tid == 0) count = 0;
    __syncthreads();
    least = least_of[0];
#pragma unroll
    for (int i = 1; i < 4; ++i) least = least_of[i] > least ? least_of[i] : least;
    const float m = row_m, s = row_s, ls = logf(s);
    const bool ok = s > 0.0f && m < INFINITY;
    if (!ok) {
        if (tid < top) write_top(o, r, top, tid, 0, false, m, ls);
        return;
    }
    // keys differ, so at most (parts - 1) * (top - 1) + top of them are not below `least`; the list may still be too short for that
    for (int i = tid; i < parts * top; i += 128) {
        const uint64_t k = keys[i];
        if (k >= least && k != 0) {
            const int at = atomicAdd(&count, 1);
            if (at < kList) list[at] = k;
        }
    }
    __syncthreads();
    const int n = count;
    const bool all = n <= kList;
    const uint64_t *from = all ? list : keys;
    const int total = all ? n : parts * top;
    for (int i = tid; i < total; i += 128) {
        const uint64_t k = from[i];
        if (k < least || k == 0) continue;
        int rank = 0;
        for (int j = 0; j < total; ++j) rank += from[j] > k;
        if (rank < top) write_top(o, r, top, rank, k, ok, m, ls);
    }
}

int parts_of(int vocab) { return (int)(((int64_t)vocab + 8 + kPart - 1) / kPart); }        // + 8: a row may start inside a 16-byte unit

template <typename T>
void launch(const void *logits, int64_t stride, int rows, int vocab, int top, const Out &o, void *scratch, cudaStream_t st) {
    const int parts = parts_of(vocab);
    Part *part = reinterpret_cast<Part *>(scratch);
    uint64_t *keys = reinterpret_cast<uint64_t *>(part + (int64_t)rows * parts);
    cq_launch_k(logprobs_part_kernel<T>, dim3((unsigned)((int64_t)rows * parts)), dim3(kThreads), 0, st, (const T *)logits, stride, vocab, parts, top, part, keys);
    cq_launch_k(logprobs_join_kernel<T>, dim3((unsigned)rows), dim3(128), 0, st, (const T *)logits, stride, vocab, parts, top, (const Part *)part,
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
