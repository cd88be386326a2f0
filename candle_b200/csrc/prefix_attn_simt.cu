// Segments of the shared-prefix attention (prefix_attn.cuh) in f32 arithmetic, for every element type.
//
// A CTA walks its segments in steps of 64 keys: keys and values go to shared memory as f32, scores are made by warps that hold R rows
// x 32 keys, the softmax of a row runs with its maximum and sum so far, and the outputs stay in registers: a warp holds R rows x all
// dims and half of the keys; the halves meet when the segment ends.
#include "prefix_attn.cuh"

namespace {
using namespace cq_attn;

constexpr int kRows = 32, kStep = 64, kThreads = 256;

template <int D> struct Smem {
    float q[kRows][D + 4];
    float k[kStep][D + 4];          // 16-byte units of neighbouring keys in different banks
    float v[kStep][D];
    float p[kRows][kStep + 4];
    float m[kRows], l[kRows], f[kRows];
};

__device__ __forceinline__ void put4(float *to, const float *from) { cq_cp_async16(to, from); }
__device__ __forceinline__ void put4(float *to, const __half *from) {
    const uint2 w = *reinterpret_cast<const uint2 *>(from);
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&w.y));
    *reinterpret_cast<float4 *>(to) = make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void put4(float *to, const __nv_bfloat16 *from) {
    const uint2 w = *reinterpret_cast<const uint2 *>(from);
    *reinterpret_cast<float4 *>(to) = make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                                                  __uint_as_float(w.y & 0xffff0000u));
}

// scores of rows r0 .. r0 + R - 1 and key `key` of the step
template <int D, int R> __device__ __forceinline__ void scores(Smem<D> &sm, int r0, int key) {
    float s[R] = {};
#pragma unroll 4
    for (int d = 0; d < D; d += 4) {
        const float4 k = *reinterpret_cast<const float4 *>(&sm.k[key][d]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float4 q = *reinterpret_cast<const float4 *>(&sm.q[r0 + r][d]);
            s[r] = __fmaf_rn(q.x, k.x, s[r]); s[r] = __fmaf_rn(q.y, k.y, s[r]);
            s[r] = __fmaf_rn(q.z, k.z, s[r]); s[r] = __fmaf_rn(q.w, k.w, s[r]);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) sm.p[r0 + r][key] = s[r];
}
template <int D, int R> __device__ __forceinline__ void outputs(const Smem<D> &sm, int r0, int key0, int lane, float (&o)[8][D / 32]) {
    constexpr int V = D / 32;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < V; ++i) o[r][i] = __fmul_rn(o[r][i], sm.f[r0 + r]);
    for (int j = key0; j < key0 + kStep / 2; j += 4) {
        float p[R][4], v[4][V];
#pragma unroll
        for (int r = 0; r < R; ++r) *reinterpret_cast<float4 *>(p[r]) = *reinterpret_cast<const float4 *>(&sm.p[r0 + r][j]);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            if constexpr (V == 4) *reinterpret_cast<float4 *>(v[x]) = *reinterpret_cast<const float4 *>(&sm.v[j + x][V * lane]);
            else *reinterpret_cast<float2 *>(v[x]) = *reinterpret_cast<const float2 *>(&sm.v[j + x][V * lane]);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < V; ++i) o[r][i] = __fmaf_rn(p[r][x], v[x][i], o[r][i]);
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) prefix_simt_kernel(const cq_kv_cache cache, const Call call, int layer, const T *q, int64_t q_stride,
                                                               float c) {
    extern __shared__ __align__(16) uint8_t raw[];
    Smem<D> &sm = *reinterpret_cast<Smem<D> *>(raw);
    const cq_kv::State s = cq_kv::state_of(cache);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, per = call.sh.per_kv;
    cq_pdl_launch_dependents();
    cq_pdl_wait();
    const T *k_pool = reinterpret_cast<const T *>(cache.k), *v_pool = reinterpret_cast<const T *>(cache.v);
    SharedWalk shared(call, blockIdx.x);
    OwnWalk own(call, blockIdx.x);
    Segment seg;
    while (shared.next(call, seg) || own.next(call, seg)) {
        const int *table = s.tables + (size_t)seg.slot * s.max_pages;
        __syncthreads();
        for (int i = tid; i < kRows * (D / 4); i += kThreads) {
            const int r = i / (D / 4), d = i % (D / 4) * 4;
            if (r < seg.rows) {
                const int row = seg.row0 + r;
                put4(&sm.q[r][d], q + (int64_t)(row / per) * q_stride + (int64_t)(seg.head * per + row % per) * D + d);
            } else *reinterpret_cast<float4 *>(&sm.q[r][d]) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        if (tid < kRows) { sm.m[tid] = -INFINITY; sm.l[tid] = 0.0f; }
        float o[8][D / 32] = {};
        const int wide = seg.rows <= 4 ? 1 : seg.rows <= 8 ? 2 : seg.rows <= 16 ? 4 : 8, r0 = (warp >> 1) * wide, half = warp & 1;
        for (int key0 = seg.key0; key0 < seg.key1; key0 += kStep) {
            const int n = min(kStep, seg.key1 - key0);
            __syncthreads();                // the step before has been read
            for (int i = tid; i < kStep * (D / 4); i += kThreads) {
                const int j = i / (D / 4), d = i % (D / 4) * 4;
                bool there = j < n;
                if (there) {
                    const int pos = key0 + j, page = table[pos / s.page];
                    there = page >= 0 && page < s.pages;
                    if (there) {
                        const int64_t row = (((int64_t)layer * s.pages + page) * cache.kv_heads + seg.head) * s.page + pos % s.page;
                        put4(&sm.k[j][d], k_pool + row * D + d);
                        put4(&sm.v[j][d], v_pool + row * D + d);
                    } else atomicCAS(s.header, cq_kv::kOk, cq_kv::kBadPage);
                }
                if (!there) {               // whatever lies behind the context must not meet a weight of zero as a NaN
                    *reinterpret_cast<float4 *>(&sm.k[j][d]) = make_float4(0.f, 0.f, 0.f, 0.f);
                    *reinterpret_cast<float4 *>(&sm.v[j][d]) = make_float4(0.f, 0.f, 0.f, 0.f);
                }
            }
            cq_cp_async_commit();
            cq_cp_async_wait<0>();
            __syncthreads();
            const int key = half * 32 + lane;
            if (wide == 1) scores<D, 1>(sm, r0, key);
            else if (wide == 2) scores<D, 2>(sm, r0, key);
            else if (wide == 4) scores<D, 4>(sm, r0, key);
            else scores<D, 8>(sm, r0, key);
            __syncthreads();
            for (int r = warp; r < 4 * wide; r += kThreads / 32) {
                const float a = lane < n ? sm.p[r][lane] : -INFINITY, b = lane + 32 < n ? sm.p[r][lane + 32] : -INFINITY;
                float mx = fmaxf(a, b);
#pragma unroll
                for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
                const float was = sm.m[r], now = fmaxf(was, __fmul_rn(mx, c)), base = now == -INFINITY ? 0.0f : now;
                const float pa = lane < n ? exp2f(__fmaf_rn(a, c, -base)) : 0.0f, pb = lane + 32 < n ? exp2f(__fmaf_rn(b, c, -base)) : 0.0f;
                sm.p[r][lane] = pa;
                sm.p[r][lane + 32] = pb;
                float sum = pa + pb;
#pragma unroll
                for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
                __syncwarp();
                if (lane == 0) {
                    const float f = was == now ? 1.0f : exp2f(was - now);
                    sm.m[r] = now;
                    sm.l[r] = __fmaf_rn(sm.l[r], f, sum);
                    sm.f[r] = f;
                }
            }
            __syncthreads();
            if (wide == 1) outputs<D, 1>(sm, r0, half * 32, lane, o);
            else if (wide == 2) outputs<D, 2>(sm, r0, half * 32, lane, o);
            else if (wide == 4) outputs<D, 4>(sm, r0, half * 32, lane, o);
            else outputs<D, 8>(sm, r0, half * 32, lane, o);
        }
        __syncthreads();
        constexpr int V = D / 32;
        float *mine = &sm.k[0][0] + r0 * D + V * lane;          // the halves meet where the keys were
        if (half == 1)
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (r < wide)
#pragma unroll
                    for (int i = 0; i < V; ++i) mine[r * D + i] = o[r][i];
        __syncthreads();
        if (half == 0)
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (r < wide && r0 + r < seg.rows)
#pragma unroll
                    for (int i = 0; i < V; ++i) call.o[(int64_t)(seg.part + r0 + r) * D + V * lane + i] = o[r][i] + mine[r * D + i];
        if (tid < seg.rows) call.ml[seg.part + tid] = make_float2(sm.m[tid], sm.l[tid]);
    }
}

template <typename T, int D>
void launch(const Call &c, const cq_kv_cache &cache, int layer, const void *q, int64_t q_stride, float scale, cudaStream_t st) {
    static bool done[64];
    cq_smem_once((const void *)prefix_simt_kernel<T, D>, (int)sizeof(Smem<D>), done);
    cq_launch_k(prefix_simt_kernel<T, D>, dim3(c.sh.ctas), dim3(kThreads), sizeof(Smem<D>), st, cache, c, layer, (const T *)q, q_stride,
                (float)(scale * 1.4426950408889634));
}

}  // namespace

void cq_attn::simt_launch(const Call &c, const cq_kv_cache &cache, int layer, const void *q, int64_t q_stride, float scale, cudaStream_t st) {
    const bool wide = c.sh.head_dim == 128;
    if (c.sh.elem == CQ_F32) wide ? launch<float, 128>(c, cache, layer, q, q_stride, scale, st) : launch<float, 64>(c, cache, layer, q, q_stride, scale, st);
    else if (c.sh.elem == CQ_F16) wide ? launch<__half, 128>(c, cache, layer, q, q_stride, scale, st) : launch<__half, 64>(c, cache, layer, q, q_stride, scale, st);
    else wide ? launch<__nv_bfloat16, 128>(c, cache, layer, q, q_stride, scale, st) : launch<__nv_bfloat16, 64>(c, cache, layer, q, q_stride, scale, st);
}
