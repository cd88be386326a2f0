// Segments of the shared-prefix attention (prefix_attn.cuh) on the tensor cores: f16 and bf16 caches.
//
// Shared items (many rows, keys mostly from L2): tiles of 128 rows x 64 keys by tcgen05.  S = Q K^T goes to tensor memory; thread r of the softmax
// warps owns row r, reads it there, and writes the weights 2^(s c - m), c = scale log2 e, back over it in 16 bits as the first operand of O += P V.
// Warps: 0-3 softmax (TMEM lanes 32 w ..), 4 copies, 5 MMA.  256 columns a CTA: the scores of two tiles, so that one tile's softmax has the products
// of its neighbours beside it, and the outputs.  Two CTAs per SM.
//
// Own items (as many rows as a KV head has query heads, keys from HBM): a warp is a worker of its own, 16 rows x 16 keys a step by mma.sync, with two
// steps of keys and values on their way.  Through the first form an item of four rows costs the waits of a whole tile chain - QK,
// softmax, PV, some 10,000 clocks for 64 KB - where HBM gives an SM 64 KB in 2,850; here twelve warps of an SM have 190 KB in flight and
// nothing to wait for but that.
//
// In both m is the row's maximum so far, kept until a score passes it by 2^8 (weights up to 256 are as good as any, the sum has the same
// factor), so that outputs are scaled in the first tiles only.  The sum adds the weights as rounded: rounding moves weight between keys but
// not the total.  Keys and values come by tiled TMA copies of 64 dims and a page (own items: 16 rows) at a time, 128-byte swizzle: K as it is
// for the first product, V for the second with its rows as the K dimension.  Rows of a tile behind the last key hold whatever the page or the tile
// before left there: their scores are masked, their values set to zero before the second product, since 0 x NaN is not 0.
#include <cuda.h>

#include <mutex>

#include "prefix_attn.cuh"
#include "prompt_f16.cuh"

namespace {
using namespace cq_attn;
using namespace cq_prompt;

constexpr int kThreads = 32 * kMmaWarps, kStages = 2, kCols = 256, kHalfBytes = 128 * 128;       // 128 rows of 64 elements
constexpr int kS = 0, kO = 128;                                      // columns of scores / weights (two tiles) and of outputs

// operands there (q, k, v), scores there (and K free), weights there, outputs there (and V, weights free)
struct Bars { uint64_t q, k[2], v[2], s[2], p[2], o[2]; };

constexpr int kStep = 16;                // keys of a step of an own item
template <int D> struct Step { uint8_t k[D / 64][kStep * 128], v[D / 64][kStep * 128]; };
template <int D> struct Tiles {
    union {
        struct { uint8_t q[D / 64][kHalfBytes], k[2][D / 64][kKeyTile * 128], v[2][D / 64][kKeyTile * 128]; };
        Step<D> step[kMmaWarps][kStages];
    };
    Bars bar;
    uint64_t step_bar[kMmaWarps][kStages];
    uint32_t tmem;
    int abort;
};

// 128-byte swizzle, 8-row groups 1024 bytes apart.  K-major operands ignore the low word's upper half; N-major ones find there the distance
// between blocks of 64 columns.
__device__ __forceinline__ uint64_t desc_sw(uint32_t lo) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"((1024u >> 4) | (1u << 14) | (2u << 29)));
    return r;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(desc_sw(a)), "l"(desc_sw(b)), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(desc_sw(b)), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
                 "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
                   "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// two weights in the type's 16 bits, and their sum as rounded
template <bool BF16> __device__ __forceinline__ uint32_t pack(float a, float b, float &sum) {
    uint32_t w;
    if constexpr (BF16) {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
        sum += __uint_as_float(w << 16) + __uint_as_float(w & 0xffff0000u);
    } else {
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
        sum += f.x + f.y;
    }
    return w;
}

// The CTA's share of the shared line.  False: a wait gave up.
// The scores of two tiles have room, so QK of the next tile and PV of the one before run beside a tile's softmax; a barrier per buffer, since
// no waiter may fall two phases behind.
template <int D, bool BF16>
__device__ bool shared_part(Tiles<D> &sm, const cq_kv_cache &cache, const cq_kv::State &st, const Call &call, const CUtensorMap &k_map, const CUtensorMap &v_map,
                            const uint8_t *__restrict__ q, int64_t q_stride, float c, uint32_t tmem) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, page = st.page;
    constexpr uint32_t kIdescQK = (1u << 4) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)kKeyTile >> 3) << 17 | (128u >> 4) << 24;
    constexpr uint32_t kIdescPV = (1u << 4) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | (1u << 16) | ((uint32_t)D >> 3) << 17 | (128u >> 4) << 24;
    volatile int *abort_flag = &sm.abort;
    SharedWalk walk(call, blockIdx.x);
    Segment seg;
    bool ok = true;
    unsigned tile = 0;              // buffer tile & 1, phase tile / 2
    if (warp < 4) {
        const int per = call.sh.per_kv, row = warp * 32 + lane;
        const uint32_t mine = tmem + ((uint32_t)(warp * 32) << 16);
        while (ok && walk.next(call, seg)) {
            // Q: all rows of the segment by the four warps; rows behind them keep what was there, and nobody reads their results
            const uint8_t *src = q + (int64_t)seg.head * per * D * 2;
            for (int i = tid; i < seg.rows * (D / 8); i += 128) {
                const int r = i / (D / 8), x = i % (D / 8), n = div_per(seg.row0 + r, call.sh), in = seg.row0 + r - n * per;
                cq_cp_async16(&sm.q[x >> 3][r * 128 + ((x & 7) ^ (r & 7)) * 16], src + ((int64_t)n * q_stride + (int64_t)in * D + x * 8) * 2);
            }
            cq_cp_async_commit();
            cq_cp_async_wait<0>();
            fence_proxy_async_smem();
            arrive_warp(&sm.bar.q, lane);
            const bool active = warp * 32 < seg.rows;
            float m = -INFINITY, l = 0.0f;
            for (int j = 0; j < seg.units; ++j, ++tile) {
                const int n = seg.key1 - seg.key0 - j * kKeyTile;          // keys of this tile, if fewer than kKeyTile
                const unsigned b = tile & 1, phase = tile >> 1 & 1;
                const uint32_t sp = mine + kS + b * kKeyTile;
                if (!(ok = wait_warp(&sm.bar.s[b], phase, abort_flag))) break;
                tc_fence_after();
                if (active) {
                    uint32_t s[2][32];
                    tmem_ld32(sp, s[0]);
                    tmem_ld32(sp + 32, s[1]);
                    tmem_ld_wait();
                    if (n < kKeyTile) {
#pragma unroll
                        for (int i = 0; i < kKeyTile; ++i)
                            if (i >= n) s[i >> 5][i & 31] = 0xff800000u;        // -inf
                    }
                    float mx = -INFINITY, my = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 32; ++i) { mx = fmaxf(mx, __uint_as_float(s[0][i])); my = fmaxf(my, __uint_as_float(s[1][i])); }
                    mx = fmaxf(mx, my) * c;
                    if (j == 0) m = mx;
                    else {
                        const bool up = mx > m + 8.0f;          // from -inf as well
                        if (__any_sync(0xffffffffu, up)) {
                            const float f = up ? ex2(m - mx) : 1.0f;
                            if (up) m = mx;
                            l *= f;
                            if (!(ok = wait_warp(&sm.bar.o[b ^ 1], (tile - 1) >> 1 & 1, abort_flag))) break;        // the outputs so far
                            tc_fence_after();
#pragma unroll
                            for (int x = 0; x < D / 16; ++x) {
                                uint32_t o[16];
                                tmem_ld16(mine + kO + 16 * x, o);
                                tmem_ld_wait();
#pragma unroll
                                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                                tmem_st16(mine + kO + 16 * x, o);
                            }
                        }
                    }
                    const float base = m == -INFINITY ? 0.0f : m;
                    float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        uint32_t w[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            w[i] = pack<BF16>(ex2(__fmaf_rn(__uint_as_float(s[x][2 * i]), c, -base)), ex2(__fmaf_rn(__uint_as_float(s[x][2 * i + 1]), c, -base)),
                                              i & 1 ? sum1 : sum0);
                        tmem_st16(sp + 16 * x, w);              // over the scores
                    }
                    l += sum0 + sum1;
                    tmem_st_wait();
                    tc_fence_before();
                }
                if (n < kKeyTile) {
                    if (!(ok = wait_warp(&sm.bar.v[b], phase, abort_flag))) break;
                    for (int i = tid; i < (kKeyTile - n) * (D / 8); i += 128) {
                        const int r = n + i / (D / 8), x = i % (D / 8);
                        *reinterpret_cast<uint4 *>(&sm.v[b][x >> 3][r * 128 + (x & 7) * 16]) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_smem();
                }
                arrive_warp(&sm.bar.p[b], lane);
            }
            if (!ok || !(ok = wait_warp(&sm.bar.o[(tile - 1) & 1], (tile - 1) >> 1 & 1, abort_flag))) break;
            tc_fence_after();
            if (active) {
                float *to = call.o + (int64_t)(seg.part + row) * D;
#pragma unroll
                for (int x = 0; x < D / 32; ++x) {
                    uint32_t s[32];
                    tmem_ld32(mine + kO + 32 * x, s);
                    tmem_ld_wait();
                    if (row < seg.rows)
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            *reinterpret_cast<uint4 *>(to + 32 * x + 4 * i) = make_uint4(s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]);
                }
                if (row < seg.rows) call.ml[seg.part + row] = make_float2(m, l);
                tc_fence_before();
            }
        }
    } else if (warp == 4) {
        const int shift = 31 - __clz(page), box = min(page, kKeyTile);
        while (ok && walk.next(call, seg)) {
            const int *table = st.tables + (size_t)seg.slot * st.max_pages;
            int base = INT32_MIN / 2, ids = -1;             // page numbers base .. base + 31 of the table, one a lane
            for (int j = 0; j < seg.units; ++j, ++tile) {
                const unsigned b = tile & 1, before = (tile >> 1 & 1) ^ 1;
                const int key = seg.key0 + j * kKeyTile, p0 = key >> shift, mine = key + lane * box;
                if (((key + kKeyTile - 1) >> shift) - base >= 32) {
                    base = p0;
                    ids = (p0 + lane) << shift < seg.key1 ? table[p0 + lane] : -1;
                }
                int id = __shfl_sync(0xffffffffu, ids, ((mine >> shift) - base) & 31);           // a lane takes a box
                if (lane * box >= kKeyTile || mine >= seg.key1) id = -1;
                else if (id < 0 || id >= st.pages) { id = -1; atomicCAS(st.header, cq_kv::kOk, cq_kv::kBadPage); }
                const unsigned bytes = (unsigned)__popc(__ballot_sync(0xffffffffu, id >= 0)) * box * D * 2;
                const int y = ((id * cache.kv_heads + seg.head) << shift) + (mine & (page - 1));
                if (tile >= 2 && !(ok = wait_warp(&sm.bar.s[b], before, abort_flag))) break;
                if (lane == 0) cq_mbar_expect_tx(&sm.bar.k[b], bytes);
                __syncwarp();
                if (id >= 0)
#pragma unroll
                    for (int h = 0; h < D / 64; ++h) cq_tmap::load_2d(&sm.k[b][h][lane * box * 128], &k_map, 64 * h, y, &sm.bar.k[b]);
                if (tile >= 2 && !(ok = wait_warp(&sm.bar.o[b], before, abort_flag))) break;
                if (lane == 0) cq_mbar_expect_tx(&sm.bar.v[b], bytes);
                __syncwarp();
                if (id >= 0)
#pragma unroll
                    for (int h = 0; h < D / 64; ++h) cq_tmap::load_2d(&sm.v[b][h][lane * box * 128], &v_map, 64 * h, y, &sm.bar.v[b]);
            }
        }
        if (!ok)                        // leaving early: not before what is on its way has come (a copy that was never sent costs the wait's bound)
            for (unsigned b = 0; b < 2; ++b)
                if (tile >= b) {
                    const unsigned last = (tile - b) >> 1 & 1;          // phase of the newest copy that may be out
                    (void)(cq_mbar_wait_bounded(&sm.bar.k[b], last ^ 1) && cq_mbar_wait_bounded(&sm.bar.k[b], last));
                    (void)(cq_mbar_wait_bounded(&sm.bar.v[b], last ^ 1) && cq_mbar_wait_bounded(&sm.bar.v[b], last));
                }
    } else {
        unsigned segment = 0, qk = 0;           // tiles whose first product is under way
        const uint32_t qa = uniform(cq_smem_u32(&sm.q[0][0]) >> 4), ka = uniform(cq_smem_u32(&sm.k[0][0][0]) >> 4), va = uniform(cq_smem_u32(&sm.v[0][0][0]) >> 4);
        const uint32_t t0 = uniform(tmem);
        constexpr uint32_t kHalfK = kKeyTile * 128 >> 4, kBuf = D / 64 * kHalfK;
        auto scores = [&]() {                   // S = Q K^T of tile qk
            const unsigned b = qk & 1, phase = qk >> 1 & 1;
            if (!wait_warp(&sm.bar.k[b], phase, abort_flag)) return false;
            if (qk >= 2 && !wait_warp(&sm.bar.o[b], phase ^ 1, abort_flag)) return false;          // the weights there have been read
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int x = 0; x < D / 16; ++x)
                    mma_ss(t0 + kS + b * kKeyTile, qa + (x >> 2) * (kHalfBytes >> 4) + (x & 3) * 2, ka + b * kBuf + (x >> 2) * kHalfK + (x & 3) * 2, kIdescQK, x > 0);
                tc_commit(&sm.bar.s[b]);
            }
            __syncwarp();
            ++qk;
            return true;
        };
        while (ok && walk.next(call, seg)) {
            const int units = (int)uniform((uint32_t)seg.units);
            if (!(ok = wait_warp(&sm.bar.q, segment++ & 1, abort_flag) && scores())) break;
            for (int j = 0; j < units; ++j, ++tile) {
                const unsigned b = tile & 1, phase = tile >> 1 & 1;
                if (j + 1 < units && !(ok = scores())) break;
                if (!(ok = wait_warp(&sm.bar.v[b], phase, abort_flag)) || !(ok = wait_warp(&sm.bar.p[b], phase, abort_flag))) break;
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int x = 0; x < kKeyTile / 16; ++x)
                        mma_ts(t0 + kO, t0 + kS + b * kKeyTile + 8 * x, (va + b * kBuf + x * (2048 >> 4)) | kHalfK << 16, kIdescPV, j > 0 || x > 0);
                    tc_commit(&sm.bar.o[b]);
                }
                __syncwarp();
            }
        }
        if (!ok)                        // nor before the products have ended
            for (unsigned b = 0; b < 2; ++b) {
                if (qk > b) (void)cq_mbar_wait_bounded(&sm.bar.s[b], (qk - 1 - b) >> 1 & 1);
                if (tile > b) (void)cq_mbar_wait_bounded(&sm.bar.o[b], (tile - 1 - b) >> 1 & 1);
            }
    }
    return ok;
}

// ---- own items ----
__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool BF16> __device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The copies of a warp's steps, ahead of their use and across its segments.
template <int D> struct Loader {
    OwnWalk walk;
    Segment seg;
    int step, sent;                 // step in the segment, steps sent
    int base, ids, shift;           // page numbers base .. base + 31 of the segment's table, one a lane
    __device__ __forceinline__ Loader(const Call &call, int worker, int page_shift) : walk(call, worker), step(0), sent(0), shift(page_shift) { seg.units = 0; }
    __device__ __forceinline__ void send(Step<D> &to, uint64_t *bar, const Call &call, const cq_kv::State &st, int kv_heads, const CUtensorMap &k_map, const CUtensorMap &v_map,
                                         int lane) {
        if (step == seg.units) {
            if (!walk.next(call, seg)) return;
            step = 0;
            base = INT32_MIN / 2;
        }
        const int key = seg.key0 + kStep * step, j = key >> shift;
        if (j - base >= 32) {
            base = j;
            ids = (j + lane) << shift < seg.key1 ? st.tables[(size_t)seg.slot * st.max_pages + j + lane] : -1;
        }
        const int id = __shfl_sync(0xffffffffu, ids, j - base);
        const bool there = id >= 0 && id < st.pages;
        if (lane == 0) {
            cq_mbar_expect_tx(bar, there ? (unsigned)sizeof(Step<D>) : 0u);
            if (there) {
                const int y = ((id * kv_heads + seg.head) << shift) + (key & (st.page - 1));
#pragma unroll
                for (int h = 0; h < D / 64; ++h) {
                    cq_tmap::load_2d(to.k[h], &k_map, 64 * h, y, bar);
                    cq_tmap::load_2d(to.v[h], &v_map, 64 * h, y, bar);
                }
            } else atomicCAS(st.header, cq_kv::kOk, cq_kv::kBadPage);
        }
        ++step;
        ++sent;
    }
};

// The warp's share of the own line.  Fragments as mma.sync m16n8k16 has them: a lane holds rows lane / 4 and lane / 4 + 8.
template <int D, bool BF16>
__device__ bool own_part(Tiles<D> &sm, const cq_kv_cache &cache, const cq_kv::State &st, const Call &call, const CUtensorMap &k_map, const CUtensorMap &v_map,
                         const uint8_t *__restrict__ q, int64_t q_stride, float c) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, x2 = (lane & 3) * 2, per = call.sh.per_kv;
    const int worker = blockIdx.x * kMmaWarps + warp;
    Step<D> *steps = sm.step[warp];
    uint64_t *bars = sm.step_bar[warp];
    Loader<D> load(call, worker, 31 - __clz(st.page));
    OwnWalk walk = load.walk;
    const int units = walk.left;
    if (units <= 0) return true;
#pragma unroll
    for (int i = 0; i < kStages; ++i) load.send(steps[i], &bars[i], call, st, cache.kv_heads, k_map, v_map, lane);
    Segment seg;
    seg.units = 0;
    int step = 0;
    bool ok = true;
    uint32_t qa[D / 16][4];
    float o[D / 8][4], m0 = 0.0f, m1 = 0.0f, l0 = 0.0f, l1 = 0.0f;
    for (int u = 0; u < units; ++u) {
        const int stage = u % kStages;
        if (step == seg.units) {
            walk.next(call, seg);
            step = 0;
            const int query = div_per(seg.row0, call.sh);
            const uint8_t *src = q + ((int64_t)query * q_stride + (int64_t)(seg.head * per + seg.row0 - query * per) * D) * 2;
#pragma unroll
            for (int x = 0; x < D / 16; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = g + (i & 1) * 8;
                    qa[x][i] = r < seg.rows ? *reinterpret_cast<const uint32_t *>(src + ((int64_t)r * D + 16 * x + (i >> 1) * 8 + x2) * 2) : 0u;
                }
#pragma unroll
            for (int x = 0; x < D / 8; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[x][i] = 0.0f;
            l0 = l1 = 0.0f;
        }
        const int n = seg.key1 - seg.key0 - kStep * step;        // keys of this step, if fewer than 16
        const bool upper = seg.rows > 8;
        if (!(ok = wait_warp(&bars[stage], (u / kStages) & 1, &sm.abort))) break;
        const uint32_t kb = cq_smem_u32(steps[stage].k), vb = cq_smem_u32(steps[stage].v);
        float s[2][4] = {};
#pragma unroll
        for (int x = 0; x < D / 32; ++x)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int key = 8 * t + (lane & 7), unit = 4 * x + (lane >> 3);
                uint32_t b[4];
                ldsm(b, kb + (unit >> 3) * (kStep * 128) + key * 128 + ((unit & 7) ^ (key & 7)) * 16);
                mma16816<BF16>(s[t], qa[2 * x], b[0], b[1]);
                mma16816<BF16>(s[t], qa[2 * x + 1], b[2], b[3]);
            }
        if (n < kStep) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (8 * t + x2 + (i & 1) >= n) s[t][i] = -INFINITY;
            for (int i = lane; i < (kStep - n) * (D / 8); i += 32) {
                const int r = n + i / (D / 8), x = i % (D / 8);
                *reinterpret_cast<uint4 *>(&steps[stage].v[x >> 3][r * 128 + (x & 7) * 16]) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
        }
        float mx0 = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1])), mx1 = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2)) * c;
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2)) * c;
        if (step == 0) { m0 = mx0; m1 = mx1; }
        else {
            const bool up0 = mx0 > m0 + 8.0f, up1 = upper && mx1 > m1 + 8.0f;
            if (__any_sync(0xffffffffu, up0 || up1)) {
                const float f0 = up0 ? ex2(m0 - mx0) : 1.0f, f1 = up1 ? ex2(m1 - mx1) : 1.0f;
                if (up0) m0 = mx0;
                if (up1) m1 = mx1;
                l0 *= f0;
                l1 *= f1;
#pragma unroll
                for (int x = 0; x < D / 8; ++x) { o[x][0] *= f0; o[x][1] *= f0; o[x][2] *= f1; o[x][3] *= f1; }
            }
        }
        const float b0 = m0 == -INFINITY ? 0.0f : m0, b1 = m1 == -INFINITY ? 0.0f : m1;
        uint32_t p[4];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            p[2 * t] = pack<BF16>(ex2(__fmaf_rn(s[t][0], c, -b0)), ex2(__fmaf_rn(s[t][1], c, -b0)), l0);
            p[2 * t + 1] = upper ? pack<BF16>(ex2(__fmaf_rn(s[t][2], c, -b1)), ex2(__fmaf_rn(s[t][3], c, -b1)), l1) : 0u;
        }
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {
            const int key = lane & 15, unit = 2 * x + (lane >> 4);
            uint32_t b[4];
            ldsm_t(b, vb + (unit >> 3) * (kStep * 128) + key * 128 + ((unit & 7) ^ (key & 7)) * 16);
            mma16816<BF16>(o[2 * x], p, b[0], b[1]);
            mma16816<BF16>(o[2 * x + 1], p, b[2], b[3]);
        }
        __syncwarp();
        load.send(steps[stage], &bars[stage], call, st, cache.kv_heads, k_map, v_map, lane);
        if (++step == seg.units) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
            l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
            l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
            l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
            float *to = call.o + ((int64_t)seg.part + g) * D + x2;
#pragma unroll
            for (int x = 0; x < D / 8; ++x) {
                if (g < seg.rows) *reinterpret_cast<float2 *>(to + 8 * x) = make_float2(o[x][0], o[x][1]);
                if (g + 8 < seg.rows) *reinterpret_cast<float2 *>(to + 8 * D + 8 * x) = make_float2(o[x][2], o[x][3]);
            }
            if (x2 == 0) {
                if (g < seg.rows) call.ml[seg.part + g] = make_float2(m0, l0);
                if (g + 8 < seg.rows) call.ml[seg.part + g + 8] = make_float2(m1, l1);
            }
        }
    }
    if (!ok)                            // leaving early: not before what is on its way has come
        for (int i = 0; i < kStages; ++i) {
            const int sent = (load.sent - i + kStages - 1) / kStages;       // copies into this stage
            if (sent > 0) (void)cq_mbar_wait_bounded(&bars[i], (sent - 1) & 1);
        }
    return ok;
}

// The first half of the CTAs begins with shared items, the second with own ones, so that the tensor cores and HBM are both in use.
template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads, 2) prefix_mma_kernel(const cq_kv_cache cache, const Call call, const __grid_constant__ CUtensorMap k_map,
                                                                 const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CUtensorMap k_step,
                                                                 const __grid_constant__ CUtensorMap v_step, const uint8_t *__restrict__ q, int64_t q_stride, float c) {
    extern __shared__ uint8_t raw[];
    Tiles<D> &sm = *reinterpret_cast<Tiles<D> *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const cq_kv::State st = cq_kv::state_of(cache);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        cq_mbar_init(&sm.bar.q, 4);
        for (int i = 0; i < 2; ++i) {
            cq_mbar_init(&sm.bar.k[i], 1); cq_mbar_init(&sm.bar.v[i], 1);
            cq_mbar_init(&sm.bar.s[i], 1); cq_mbar_init(&sm.bar.p[i], 4); cq_mbar_init(&sm.bar.o[i], 1);
        }
        for (int i = 0; i < kMmaWarps * kStages; ++i) cq_mbar_init(&sm.step_bar[0][i], 1);
        sm.abort = 0;
        cq_fence_mbar_init();
    }
    if (warp == 5) {
        tmem_alloc(&sm.tmem, kCols);
        tmem_relinquish();
        tc_fence_before();
    }
    cq_pdl_launch_dependents();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem;
    cq_pdl_wait();
    const bool own_first = blockIdx.x >= gridDim.x / 2;
    bool ok = true;
    if (own_first) {
        ok = own_part<D, BF16>(sm, cache, st, call, k_step, v_step, q, q_stride, c);
        __syncthreads();
    }
    if (!sm.abort) ok = shared_part<D, BF16>(sm, cache, st, call, k_map, v_map, q, q_stride, c, tmem) && ok;
    if (!own_first) {
        __syncthreads();
        if (!sm.abort) ok = own_part<D, BF16>(sm, cache, st, call, k_step, v_step, q, q_stride, c) && ok;
    }
    if (!ok && lane == 0) atomicCAS(st.header, cq_kv::kOk, cq_kv::kTimeout);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 5) tmem_dealloc(tmem, kCols);
}

// One layer of a pool as rows of D elements; box: rows of one page x 64 elements, 128-byte swizzle.
bool pool_map(const void *base, int64_t rows, int d, int box_rows, CUtensorMap &out) {
    using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult res;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &res) != cudaSuccess || res != cudaDriverEntryPointSuccess) {
            (void)cudaGetLastError();
            fn = nullptr;
        }
        return (Encode)fn;
    }();
    if (!encode) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)d, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)d * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, one[2] = {1, 1};
    return encode(&out, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void *>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool BF16>
void launch(const Call &c, const cq_kv_cache &cache, const CUtensorMap (&m)[4], const void *q, int64_t q_stride, float scale, cudaStream_t st) {
    constexpr int smem = (int)sizeof(Tiles<D>) + 1024;
    cudaFuncSetAttribute(prefix_mma_kernel<D, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    cq_launch_k(prefix_mma_kernel<D, BF16>, dim3(c.sh.ctas), dim3(kThreads), smem, st, cache, c, m[0], m[1], m[2], m[3], (const uint8_t *)q, q_stride,
                (float)(scale * 1.4426950408889634));
}

}  // namespace

bool cq_attn::mma_launch(const Call &c, const cq_kv_cache &cache, int layer, const void *q, int64_t q_stride, float scale, cudaStream_t st) {
    const int64_t rows = (int64_t)cache.pages * cache.kv_heads * cache.page_size, offset = rows * layer * cache.head_dim * 2;
    const uint8_t *k = (const uint8_t *)cache.k + offset, *v = (const uint8_t *)cache.v + offset;
    const int box = cache.page_size < kKeyTile ? cache.page_size : kKeyTile;
    CUtensorMap m[4];
    if (!pool_map(k, rows, cache.head_dim, box, m[0]) || !pool_map(v, rows, cache.head_dim, box, m[1]) ||
        !pool_map(k, rows, cache.head_dim, kStep, m[2]) || !pool_map(v, rows, cache.head_dim, kStep, m[3])) {
        cq_set_status(CQ_ERR_CUDA, "prefix_attention: cuTensorMapEncodeTiled is not available or refused the pool");
        return false;
    }
    const bool bf16 = c.sh.elem == CQ_BF16;
    if (c.sh.head_dim == 128) bf16 ? launch<128, true>(c, cache, m, q, q_stride, scale, st) : launch<128, false>(c, cache, m, q, q_stride, scale, st);
    else bf16 ? launch<64, true>(c, cache, m, q, q_stride, scale, st) : launch<64, false>(c, cache, m, q, q_stride, scale, st);
    return true;
}
