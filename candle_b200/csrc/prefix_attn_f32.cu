// Segments of the shared-prefix attention (prefix_attn.cuh) of f32 caches: f32 products from three tf32 ones on the tensor cores.
//
// x = h + l with h the nearest number of 11 significant bits, l = x - h exact, of either sign, no more than 2^-11 |x| and 12 bits long, cut to 11 by the instruction:
// a b = h h' + h l' + l h' up to 2^-22 (l l', of either sign) and 2^-23 for each of the two cuts, together 2^-21 of |a b|.  (With h cut instead of rounded all errors have one sign: an output was
// 2e-6 off where plain f32 is 6e-7.)  The instruction's own sums are cut as well, so chains are short: scores have an accumulator for every 32 dims and two for the low parts, and the outputs' products of a step
// go to fresh ones that are added to the outputs by f32 additions.
// mma.sync m16n8k8 does 474 products a clock and SM here (measured), so 158 of these, against 128 fused products of the f32 pipe that would want their
// operands from shared memory all the time.
//
// A warp is a worker of both lines: eight rows, S^T = K Q^T (16 keys x 8 rows a step), O^T += V^T P^T (dims x 8 rows), the next step of keys and values on its way by
// asynchronous copies.  Shared keys are read once for every eight rows, from L2 but for the first: at 16 KB for 16 keys x 8 rows the tensor cores ask
// for 60 bytes a clock of an SM when nothing else is in the way, about what L2 gives.
// By itself, cold caches: 32 sequences over 4 x 1500 shared keys, 32 heads of 64: 25 us, 0.45 GFLOP; 8 over 512, 32 heads of 128: 9.6 us, all of it latency.
// Rows of K lie 4 floats more than their length apart and those of V 8 more, so that the fragments' reads meet every bank once.
#include "prefix_attn.cuh"

namespace {
using namespace cq_attn;

constexpr int kStep = 16, kStages = 2;
// Weights are up to 2^8, the maximum being let be so far: times 2^-24, which the quotient of the sums loses again, 65536 of them add up to no more than 1, and values of any
// size do not overflow where their mean does not.  Values lose bits for it below 2^-80.
constexpr float kDown = 1.0f / (1 << 24);

template <int D> struct Step { float k[kStep][D + 4], v[kStep][D + 8]; };

__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t high(uint32_t x) { return (x + 0x1000u) & 0xffffe000u; }
__device__ __forceinline__ uint32_t low(uint32_t x, uint32_t h) { return __float_as_uint(__uint_as_float(x) - __uint_as_float(h)); }
// The same for any number: what would round to infinity is cut.  Of an infinity nothing is left, and it meets the other side's high part only: a low part of 0 would make a
// NaN of it.  A NaN's low part is a NaN, whatever the cut makes of the high one.
__device__ __forceinline__ bool infinite(uint32_t x) { return (x & 0x7fffffffu) == 0x7f800000u; }
__device__ __forceinline__ uint32_t safe_high(uint32_t x) { return (x & 0x7fffffffu) >= 0x7f7ff000u ? x & 0xffffe000u : high(x); }
__device__ __forceinline__ uint32_t safe_low(uint32_t x) { return infinite(x) ? 0u : low(x, safe_high(x)); }
__device__ __forceinline__ uint32_t finite_high(uint32_t x) { return infinite(x) ? 0u : safe_high(x); }

// The copies of a warp's steps, ahead of their use and across its segments: the shared line, then the own one.  Sixteen rows of a page are one block of memory, copied 16 bytes
// a lane; rows behind the last key come as zeros.
template <int D> struct Loader {
    SharedWalk shared;
    OwnWalk own;
    Segment seg;
    int step, steps;                // in the segment
    int base, ids, shift;           // page numbers base .. base + 31 of the segment's table, one a lane
    __device__ __forceinline__ Loader(const Call &call, int worker, int own_worker, int page_shift) : shared(call, worker), own(call, own_worker), step(0), steps(0), shift(page_shift) {}
    __device__ __forceinline__ void send(Step<D> &to, const cq_kv_cache &cache, const float *k, const float *v, const Call &call, const cq_kv::State &st, int lane) {
        constexpr int kPieces = kStep * D / 128, kRows = 128 / D;               // of 512 bytes; rows of a piece
        if (step == steps && (shared.next(call, seg) || own.next(call, seg))) {
            step = 0;
            steps = (seg.key1 - seg.key0 + kStep - 1) / kStep;
            base = INT32_MIN / 2;
        }
        if (step < steps) {
            const int key = seg.key0 + kStep * step, j = key >> shift;
            if (j - base >= 32) {
                base = j;
                ids = (j + lane) << shift < seg.key1 ? st.tables[(size_t)seg.slot * st.max_pages + j + lane] : -1;
            }
            int id = __shfl_sync(0xffffffffu, ids, j - base), n = seg.key1 - key;
            if ((unsigned)id >= (unsigned)st.pages) {
                if (lane == 0) atomicCAS(st.header, cq_kv::kOk, cq_kv::kBadPage);
                id = n = 0;
            }
            const int64_t at = (int64_t)(((id * cache.kv_heads + seg.head) << shift) + (key & (st.page - 1))) * D + lane * 4;
            const float *ks = k + at, *vs = v + at;
            const int row = lane / (D / 4), x = lane % (D / 4) * 4;
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int r = row + i * kRows, bytes = r < n ? 16 : 0;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(cq_smem_u32(&to.k[r][x])), "l"(ks + i * 128), "r"(bytes) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(cq_smem_u32(&to.v[r][x])), "l"(vs + i * 128), "r"(bytes) : "memory");
            }
            ++step;
        }
        cq_cp_async_commit();           // one group a step, an empty one behind the last
    }
};

template <int D>
__global__ void __launch_bounds__(32 * f32_warps(D), 1) prefix_f32_kernel(const cq_kv_cache cache, const Call call, const float *k_layer, const float *v_layer, const float *q,
                                                                          int64_t q_stride, float c) {
    extern __shared__ __align__(16) uint8_t raw[];
    const cq_kv::State st = cq_kv::state_of(cache);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, per = call.sh.per_kv;
    Step<D> *steps = reinterpret_cast<Step<D> *>(raw) + warp * kStages;
    cq_pdl_launch_dependents();
    cq_pdl_wait();
    // Neighbours on the lines are on different SMs, and the first of the one line are the last of the other: a small call's work is spread (8 sequences over 512 shared keys,
    // 32 heads of 128: 20.0 us with the plan; 21.5 with neighbours on one SM, 22.3 with the same first ones).
    const int worker = warp * gridDim.x + blockIdx.x;
    Loader<D> load(call, worker, gridDim.x * f32_warps(D) - 1 - worker, 31 - __clz(st.page));
    SharedWalk shared = load.shared;
    OwnWalk own = load.own;
#pragma unroll 1
    for (int i = 0; i < kStages; ++i) load.send(steps[i], cache, k_layer, v_layer, call, st, lane);
    Segment seg;
    int stage = 0;
#pragma unroll 1
    while (shared.next(call, seg) || own.next(call, seg)) {
        // Q^T: a lane has dims t and t + 4 of each eight, row g
        uint32_t qh[D / 8][2], ql[D / 8][2];
        const int query = div_per(seg.row0 + g, call.sh);
        const float *src = q + (int64_t)query * q_stride + (int64_t)(seg.head * per + seg.row0 + g - query * per) * D + t;
#pragma unroll
        for (int x = 0; x < D / 8; ++x)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t w = g < seg.rows ? __float_as_uint(src[8 * x + 4 * i]) : 0u;
                qh[x][i] = safe_high(w);
                ql[x][i] = safe_low(w);
            }
        float o[D / 16][4] = {}, m0 = 0.0f, m1 = 0.0f, l0 = 0.0f, l1 = 0.0f;       // rows 2 t and 2 t + 1
#pragma unroll 1
        for (int key = seg.key0; key < seg.key1; key += kStep) {
            const int n = seg.key1 - key;                       // keys of this step, if fewer than 16
            cq_cp_async_wait<kStages - 1>();
            __syncwarp();
            const Step<D> &kv = steps[stage];
            const uint32_t ka = cq_smem_u32(&kv.k[(lane >> 3 & 1) * 8 + (lane & 7)][(lane >> 4) * 4]);
            constexpr int kChains = D / 32;
            float s[kChains][4] = {}, sl[2][4] = {};
#pragma unroll
            for (int x = 0; x < D / 8; ++x) {
                uint32_t a[4], h[4], r[4];
                ldsm(a, ka + 32 * x);
#pragma unroll
                for (int i = 0; i < 4; ++i) { h[i] = high(a[i]); r[i] = low(a[i], h[i]); }
                mma(sl[0], r, qh[x][0], qh[x][1]);
                mma(sl[1], h, ql[x][0], ql[x][1]);
                mma(s[x % kChains], h, qh[x][0], qh[x][1]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float small = sl[0][i] + sl[1][i];
#pragma unroll
                for (int x = 1; x < kChains; ++x) s[0][i] += s[x][i];
                s[0][i] += small;
            }
            // An infinite key has a NaN for its low part: the scores once more, with care.
            const float sum = s[0][0] + s[0][1] + s[0][2] + s[0][3];
            if (__any_sync(0xffffffffu, sum != sum)) {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[0][i] = 0.0f;
#pragma unroll
                for (int x = 0; x < D / 8; ++x) {
                    uint32_t a[4], h[4], f[4], r[4];
                    ldsm(a, ka + 32 * x);
#pragma unroll
                    for (int i = 0; i < 4; ++i) { h[i] = safe_high(a[i]); f[i] = finite_high(a[i]); r[i] = safe_low(a[i]); }
                    mma(s[0], r, qh[x][0], qh[x][1]);
                    mma(s[0], f, ql[x][0], ql[x][1]);
                    mma(s[0], h, qh[x][0], qh[x][1]);
                }
            }
            if (g >= n) s[0][0] = s[0][1] = -INFINITY;
            if (g + 8 >= n) s[0][2] = s[0][3] = -INFINITY;
            float mx0 = fmaxf(s[0][0], s[0][2]), mx1 = fmaxf(s[0][1], s[0][3]);
#pragma unroll
            for (int x = 4; x <= 16; x <<= 1) {
                mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, x));
                mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, x));
            }
            mx0 *= c;
            mx1 *= c;
            if (key == seg.key0) { m0 = mx0; m1 = mx1; }
            else {          // the maximum so far stays until a score passes it by 2^8
                const bool up0 = mx0 > m0 + 8.0f, up1 = mx1 > m1 + 8.0f;
                if (__any_sync(0xffffffffu, up0 || up1)) {
                    const float f0 = up0 ? exp2f(m0 - mx0) : 1.0f, f1 = up1 ? exp2f(m1 - mx1) : 1.0f;
                    if (up0) m0 = mx0;
                    if (up1) m1 = mx1;
                    l0 *= f0;
                    l1 *= f1;
#pragma unroll
                    for (int x = 0; x < D / 16; ++x) { o[x][0] *= f0; o[x][1] *= f1; o[x][2] *= f0; o[x][3] *= f1; }
                }
            }
            const float b0 = m0 == -INFINITY ? 0.0f : m0, b1 = m1 == -INFINITY ? 0.0f : m1;
            float p[4] = {exp2f(__fmaf_rn(s[0][0], c, -b0)), exp2f(__fmaf_rn(s[0][1], c, -b1)), exp2f(__fmaf_rn(s[0][2], c, -b0)), exp2f(__fmaf_rn(s[0][3], c, -b1))};
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] *= kDown;
            l0 += p[0] + p[2];
            l1 += p[1] + p[3];
            // P^T changes sides: this lane's row is g now, its keys t, t + 4, t + 8, t + 12
            uint32_t ph[4], pr[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int from = (t + 4 * (i & 1)) * 4 + (g >> 1);
                const float even = __shfl_sync(0xffffffffu, i < 2 ? p[0] : p[2], from), odd = __shfl_sync(0xffffffffu, i < 2 ? p[1] : p[3], from);
                const uint32_t w = __float_as_uint(g & 1 ? odd : even);
                ph[i] = high(w);
                pr[i] = low(w, ph[i]);
            }
#pragma unroll
            for (int x0 = 0; x0 < D / 16; x0 += 4) {            // 64 dims at a time
                uint32_t w[4][2][4];
                float care = 0.0f;                              // the largest: infinities, and what would round to one, need care
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int y = 0; y < 2; ++y)                 // keys 8 y .. 8 y + 7
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float e = kv.v[8 * y + t + 4 * (i >> 1)][16 * (x0 + x) + g + 8 * (i & 1)];
                            care = fmaxf(care, fabsf(e));
                            w[x][y][i] = __float_as_uint(e);
                        }
                if (!__any_sync(0xffffffffu, care > 3e38f)) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        float hh[4] = {}, hl[4] = {};
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            uint32_t h[4], r[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) { h[i] = high(w[x][y][i]); r[i] = low(w[x][y][i], h[i]); }
                            mma(hl, r, ph[2 * y], ph[2 * y + 1]);
                            mma(hl, h, pr[2 * y], pr[2 * y + 1]);
                            mma(hh, h, ph[2 * y], ph[2 * y + 1]);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[x0 + x][i] += hh[i] + hl[i];
                    }
                } else {
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        float hh[4] = {}, hl[4] = {};
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            uint32_t h[4], f[4], r[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) { h[i] = safe_high(w[x][y][i]); f[i] = finite_high(w[x][y][i]); r[i] = safe_low(w[x][y][i]); }
                            mma(hl, r, ph[2 * y], ph[2 * y + 1]);
                            mma(hl, f, pr[2 * y], pr[2 * y + 1]);
                            mma(hh, h, ph[2 * y], ph[2 * y + 1]);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[x0 + x][i] += hh[i] + hl[i];
                    }
                }
            }
            __syncwarp();
            load.send(steps[stage], cache, k_layer, v_layer, call, st, lane);
            if (++stage == kStages) stage = 0;
        }
#pragma unroll
        for (int x = 4; x <= 16; x <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, x);
            l1 += __shfl_xor_sync(0xffffffffu, l1, x);
        }
        float *to = call.o + ((int64_t)seg.part + 2 * t) * D + g;
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {
            if (2 * t < seg.rows) { to[16 * x] = o[x][0]; to[16 * x + 8] = o[x][2]; }
            if (2 * t + 1 < seg.rows) { to[D + 16 * x] = o[x][1]; to[D + 16 * x + 8] = o[x][3]; }
        }
        if (g == 0) {
            if (2 * t < seg.rows) call.ml[seg.part + 2 * t] = make_float2(m0, l0);
            if (2 * t + 1 < seg.rows) call.ml[seg.part + 2 * t + 1] = make_float2(m1, l1);
        }
    }
}

template <int D>
void launch(const Call &c, const cq_kv_cache &cache, const float *k, const float *v, const float *q, int64_t q_stride, float scale, cudaStream_t st) {
    constexpr int warps = f32_warps(D), smem = warps * kStages * (int)sizeof(Step<D>);
    static bool done[64];
    cq_smem_once((const void *)prefix_f32_kernel<D>, smem, done);
    cq_launch_k(prefix_f32_kernel<D>, dim3(c.sh.ctas / warps), dim3(32 * warps), smem, st, cache, c, k, v, q, q_stride, (float)(scale * 1.4426950408889634));
}

}  // namespace

void cq_attn::f32_launch(const Call &c, const cq_kv_cache &cache, int layer, const void *q, int64_t q_stride, float scale, cudaStream_t st) {
    const int64_t offset = (int64_t)cache.pages * cache.kv_heads * cache.page_size * cache.head_dim * layer;
    const float *k = (const float *)cache.k + offset, *v = (const float *)cache.v + offset;
    if (c.sh.head_dim == 128) launch<128>(c, cache, k, v, (const float *)q, q_stride, scale, st);
    else launch<64>(c, cache, k, v, (const float *)q, q_stride, scale, st);
}
