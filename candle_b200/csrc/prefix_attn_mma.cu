// Segments of the shared-prefix attention (prefix_attn.cuh) on the tensor cores: f16 and bf16 caches.
//
// Shared items (many rows, keys mostly from L2): tiles of 2 x 128 rows x 128 keys by tcgen05.  S = Q K^T goes to tensor memory; thread r of a
// half's softmax warps owns row r, reads it there, and writes the weights 2^(s c - m), c = scale log2 e, back over it in 16 bits as the first operand of
// O += P V.  512 columns, a half's scores and outputs twice: one half's softmax has the other's products beside it.
//
// Own items (as many rows as a KV head has query heads, keys from HBM): a warp is a worker of its own, 8 rows x 16 keys a step by mma.sync, with its
// next steps of keys and values on their way.  Through the first form an item of four rows costs the waits of a whole tile chain - QK, softmax, PV, some
// 10,000 clocks for 64 KB - where HBM gives an SM 64 KB in 2,850.  Four such warps run beside the others, so that HBM and tensor
// cores are both in use, and the softmax warps join them when the shared items are done.
//
// By itself, cold caches: 128 sequences over 32768 shared keys, 32 / 8 heads of 128 (70 GFLOP, 405 MB) 97 us: 28 shared units of 4,300 clocks a CTA, in which the tensor cores
// and the exponentials would each take 2,050, beside some 220 own steps; 64 over 8191 (9 GFLOP, 185 MB) 41 us.
//
// In both m is the row's maximum so far, kept until a score passes it by 2^8 (weights up to 256 are as good as any, the sum has the same
// factor), so that outputs are scaled in the first tiles only.  The sum adds the weights as rounded: rounding moves weight between keys, but
// the weights given add up to 1.  Keys and values of shared items come by tiled TMA copies of 64 dims and a page at a time, 128-byte swizzle: K as it is
// for the first product, V for the second with its rows as the K dimension.  Rows of a tile behind the last key hold whatever the page or the tile
// before left there: their scores are masked, their values set to zero before the second product, since 0 x NaN is not 0.
#include <cuda.h>

#include "prefix_attn.cuh"
#include "prompt_f16.cuh"

namespace {
using namespace cq_attn;
using namespace cq_prompt;

// Warps: 0-3 and 4-7 softmax of a row tile's halves, 8 copies, 9 products, 12-15 own items.
constexpr int kThreads = 512, kCopyWarp = kMmaHelpers, kMmaWarp = 9, kOwnWarp = 12;
constexpr int kKeyTile = 128, kRing = 3, kCols = 512;                        // buffers that hold K, V, K, V, ... of the tiles in turn
constexpr int kHalfBytes = 128 * 128;                        // 128 rows of 64 elements
constexpr int kGroup = 256, kO = 128;                        // columns of a half; in it the scores / weights and the outputs
constexpr int kStep = 16;                                    // keys of a step of an own item
// Weights of bf16 are 2^-24 of what was said, which the quotient of the sums loses again: 65536 of them add up to no more than 1, and values of any size do not overflow where
// their mean does not.  Those of f16 are 2^7 times that, up to 2^15 of the type's 65504, so that they are rounded by no more than 2^-11 of themselves down to 2^-21 of the
// kept maximum and by 2^-32 of it below (without: 2^-14 and 2^-25, and 9,000 keys of 2^-24.5 beside one of 1 were 0.6 % off in sum); 2^15 * 65504 * 2^30 keys are finite in f32.
template <bool BF16> constexpr float kDown = BF16 ? 24.0f : -7.0f;
// registers a thread by warpgroup: 128 * (160 + 160 + 64 + 128) is what the block was launched with, 512 * 128
constexpr int kRegsSoft = 160, kRegsMisc = 64, kRegsOwn = 128;
static_assert(kCopyWarp == 8 && kMmaWarps == 4, "warp roles");
static_assert(2 * kRegsSoft + kRegsMisc + kRegsOwn == 512 && kRegsSoft >= 128 && kRegsOwn >= 128 && kRegsMisc <= 128, "setmaxnreg: up only from 128, down only from 128");

template <int D> struct Step { uint8_t k[D / 64][kStep * 128], v[D / 64][kStep * 128]; };
template <int D> struct Tiles {
    static constexpr int kStages = D == 64 ? 4 : 2;          // steps of an own warp: 64 KB for four of them
    uint8_t q[2][D / 64][kHalfBytes], kv[kRing][D / 64][kHalfBytes];
    Step<D> step[kMmaWarps][kStages];
    uint64_t full[kRing], free[kRing];
    uint64_t q_bar[2], s_bar[2], p_bar[2], o_bar[2], e_bar[2];         // by half: rows there, scores there, weights there, outputs there, outputs on their way out
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
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// 2^x of two exponents in the type's 16 bits; `sum` adds them as rounded
template <bool BF16> __device__ __forceinline__ uint32_t weights(uint64_t x, uint64_t &sum) {
    const float a = ex2(__uint_as_float((uint32_t)x)), b = ex2(__uint_as_float((uint32_t)(x >> 32)));
    uint32_t w;
    if constexpr (BF16) {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
        sum = add2(sum, pack2(w << 16, w & 0xffff0000u));
    } else {
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
        sum = add2(sum, pack2f(f.x, f.y));
    }
    return w;
}

__device__ __forceinline__ void load_3d(uint32_t smem, const void *map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem), "l"(map), "r"(x), "r"(y), "r"(z),
                 "r"(bar) : "memory");
}
__device__ __forceinline__ void expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// ---- shared items ----
// No waiter can fall two phases behind its barrier: what completes the next phase needs what the waiter does after the wait.

// Softmax of one half of the row tiles.  False: a wait gave up.
template <int D, bool BF16>
__device__ bool softmax_part(Tiles<D> &sm, const Call &call, const CUtensorMap &o_map, const uint8_t *q, int64_t q_stride, float c, int half) {
    const int tid = threadIdx.x & 127, lane = tid & 31, warp = tid >> 5, row = tid, per = call.sh.per_kv;
    const uint32_t mine = sm.tmem + ((uint32_t)(warp * 32) << 16) + half * kGroup;
    volatile int *abort_flag = &sm.abort;
    SharedWalk walk(call, blockIdx.x);
    Segment seg;
    unsigned tile = 0, segments = 0;        // of this half
    while (walk.next(call, seg)) {
        const int rows = min(seg.rows - half * 128, 128), row0 = seg.row0 + half * 128;
        if (rows <= 0) continue;
        // Q: rows behind the last keep what was there, and nobody reads their results
        const uint8_t *src = q + (int64_t)seg.head * per * D * 2;
        for (int i = tid; i < rows * (D / 8); i += 128) {
            const int r = i / (D / 8), x = i % (D / 8), n = div_per(row0 + r, call.sh), in = row0 + r - n * per;
            cq_cp_async16(&sm.q[half][x >> 3][r * 128 + ((x & 7) ^ (r & 7)) * 16], src + ((int64_t)n * q_stride + (int64_t)in * D + x * 8) * 2);
        }
        cq_cp_async_commit();
        cq_cp_async_wait<0>();
        fence_proxy_async_smem();
        arrive_warp(&sm.q_bar[half], lane);
        const bool active = warp * 32 < rows;
        float m = -INFINITY, l = 0.0f;
        for (int j = 0; j < seg.units; ++j, ++tile) {
            const int n = seg.key1 - seg.key0 - j * kKeyTile;          // keys of this tile, if fewer than kKeyTile
            if (!wait_warp(&sm.s_bar[half], tile & 1, abort_flag)) return false;
            tc_fence_after();
            if (active) {
                uint32_t s[kKeyTile / 32][32];
#pragma unroll
                for (int x = 0; x < kKeyTile / 32; ++x) tmem_ld32(mine + 32 * x, s[x]);
                tmem_ld_wait();
                if (n < kKeyTile) {
#pragma unroll
                    for (int i = 0; i < kKeyTile; ++i)
                        if (i >= n) s[i >> 5][i & 31] = 0xff800000u;        // -inf
                }
                float mx = -INFINITY, my = -INFINITY;
#pragma unroll
                for (int i = 0; i < kKeyTile; i += 4) {
                    mx = max3(mx, __uint_as_float(s[i >> 5][i & 31]), __uint_as_float(s[i >> 5][(i & 31) + 1]));
                    my = max3(my, __uint_as_float(s[i >> 5][(i & 31) + 2]), __uint_as_float(s[i >> 5][(i & 31) + 3]));
                }
                mx = fmaxf(mx, my) * c;
                if (j == 0) m = mx;
                else {
                    const bool up = mx > m + 8.0f;          // from -inf as well
                    if (__any_sync(0xffffffffu, up)) {
                        const float f = up ? ex2(m - mx) : 1.0f;
                        if (up) m = mx;
                        l *= f;
#pragma unroll 1
                        for (int x = 0; x < D / 8; ++x) {           // QK of this tile has waited for the outputs so far
                            uint32_t o[8];
                            tmem_ld8(mine + kO + 8 * x, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            tmem_st8(mine + kO + 8 * x, o);
                        }
                    }
                }
                const float base = (m == -INFINITY ? 0.0f : m) + kDown<BF16>;
                const uint64_t c2 = pack2f(c, c), base2 = pack2f(-base, -base);
                uint64_t sum = 0;
#pragma unroll
                for (int x = 0; x < kKeyTile / 32; ++x) {
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) w[i] = weights<BF16>(fma2(pack2(s[x][2 * i], s[x][2 * i + 1]), c2, base2), sum);
                    tmem_st16(mine + 16 * x, w);            // over scores that have been read
                }
                l += __uint_as_float((uint32_t)sum) + __uint_as_float((uint32_t)(sum >> 32));
                tmem_st_wait();
                tc_fence_before();
            }
            if (n < kKeyTile && half == 0) {                // before either half's product: the second follows the first
                const unsigned v = 2 * tile + 1, buf = v % kRing;       // the first half has a part in every tile
                if (!wait_warp(&sm.full[buf], v / kRing & 1, abort_flag)) return false;
                for (int i = tid; i < (kKeyTile - n) * (D / 8); i += 128) {
                    const int r = n + i / (D / 8), x = i % (D / 8);
                    *reinterpret_cast<uint4 *>(&sm.kv[buf][x >> 3][r * 128 + (x & 7) * 16]) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();
            }
            arrive_warp(&sm.p_bar[half], lane);
        }
        if (!wait_warp(&sm.o_bar[half], (tile - 1) & 1, abort_flag)) return false;
        tc_fence_after();
        if (active) {
            // The outputs go out as 32 x 32 boxes of 128-byte rows, one warp's each, from where Q was.  (Stored by their threads, a row each, they
            // took the load / store unit 8,000 clocks, and the own warps' fragments with them.)
            const int part = seg.part + half * 128 + warp * 32;
#pragma unroll
            for (int x = 0; x < D / 32; ++x) {
                uint32_t o[32];
                tmem_ld32(mine + kO + 32 * x, o);
                tmem_ld_wait();
                uint8_t *box = &sm.q[half][x % (D / 64)][warp * 4096];
                if (x == D / 64) {
                    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                    __syncwarp();
                }
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    *reinterpret_cast<uint4 *>(box + lane * 128 + (i ^ (lane & 7)) * 16) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0)
                    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];\n\tcp.async.bulk.commit_group;"
                                 ::"l"(&o_map), "r"(32 * x), "r"(part), "r"(cq_smem_u32(box)) : "memory");
            }
            if (row < rows) call.ml[part + lane] = make_float2(m, l);
            tc_fence_before();
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        arrive_warp(&sm.e_bar[half], lane);                 // before the next Q; not a barrier without a limit, since a warp may have given up
        if (!wait_warp(&sm.e_bar[half], segments++ & 1, abort_flag)) return false;
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    return true;
}

template <int D>
__device__ bool copy_part(Tiles<D> &sm, const cq_kv_cache &cache, const cq_kv::State &st, const Call &call, const CUtensorMap &k_map, const CUtensorMap &v_map) {
    const int lane = threadIdx.x & 31, page = st.page, shift = 31 - __clz(page), boxes = page < kKeyTile ? D / 64 : 1;
    volatile int *abort_flag = &sm.abort;
    SharedWalk walk(call, blockIdx.x);
    Segment seg;
    unsigned buf = 0, phase = 1, sent = 0;          // phase: of the use before
    bool ok = true;
    while (ok && walk.next(call, seg)) {
        const int *table = st.tables + (size_t)seg.slot * st.max_pages;
        int base = INT32_MIN / 2, ids = -1;             // page numbers base .. base + 31 of the table, one a lane
        for (int j = 0; ok && j < seg.units; ++j) {
            const int key = seg.key0 + j * kKeyTile, mine = key + lane * page;
            if (((key + kKeyTile - 1) >> shift) - base >= 32) {
                base = key >> shift;
                ids = (base + lane) << shift < seg.key1 ? table[base + lane] : -1;
            }
            int id = __shfl_sync(0xffffffffu, ids, ((mine >> shift) - base) & 31);           // a lane takes a page
            if (lane * page >= kKeyTile || mine >= seg.key1) id = -1;
            else if (id < 0 || id >= st.pages) { id = -1; atomicCAS(st.header, cq_kv::kOk, cq_kv::kBadPage); }
            const unsigned bytes = (unsigned)__popc(__ballot_sync(0xffffffffu, id >= 0)) * page * D * 2;
            const int y = (id * cache.kv_heads + seg.head) << shift;
            for (int kind = 0; kind < 2; ++kind) {
                if (sent >= kRing && !(ok = wait_warp(&sm.free[buf], phase, abort_flag))) break;
                const uint32_t bar = cq_smem_u32(&sm.full[buf]);
                if (lane == 0) expect_tx(bar, bytes);
                __syncwarp();
                if (id >= 0)
                    for (int h = 0; h < boxes; ++h) load_3d(cq_smem_u32(&sm.kv[buf][h][lane * page * 128]), kind ? &v_map : &k_map, 0, y, h, bar);
                ++sent;
                if (++buf == kRing) { buf = 0; phase ^= 1; }
            }
        }
    }
    if (!ok)                        // leaving early: not before what is on its way has come
        for (unsigned b = 0; b < kRing; ++b)
            if (sent > b) (void)cq_mbar_wait_bounded(&sm.full[b], (sent - 1 - b) / kRing & 1);
    return ok;
}

template <int D, bool BF16> __device__ bool mma_part(Tiles<D> &sm, const Call &call) {
    constexpr uint32_t kTypes = BF16 ? (1u << 7) | (1u << 10) : 0u;
    constexpr uint32_t kIdescQK = (1u << 4) | kTypes | ((uint32_t)kKeyTile >> 3) << 17 | (128u >> 4) << 24;
    constexpr uint32_t kIdescPV = (1u << 4) | kTypes | (1u << 16) | ((uint32_t)D >> 3) << 17 | (128u >> 4) << 24;
    constexpr uint32_t kBlock = kHalfBytes >> 4, kBuf = D / 64 * kBlock;
    const uint32_t qa = uniform(cq_smem_u32(&sm.q[0][0][0]) >> 4), kva = uniform(cq_smem_u32(&sm.kv[0][0][0]) >> 4), t0 = uniform(sm.tmem);
    volatile int *abort_flag = &sm.abort;
    SharedWalk walk(call, blockIdx.x);
    Segment seg;
    unsigned segments[2] = {0, 0}, tiles[2] = {0, 0}, done[2] = {0, 0};             // by half: segments, tiles with QK, with PV under way
    unsigned buf = 0, phase = 0;
    bool ok = true;
    auto advance = [&]() { if (++buf == kRing) { buf = 0; phase ^= 1; } };
    // S = Q K^T of the tile in `buf` for half h; the last half sets the buffer free
    auto scores = [&](int h, bool last) {
        if (elect_one()) {
#pragma unroll
            for (int x = 0; x < D / 16; ++x)
                mma_ss(t0 + h * kGroup, qa + h * kBuf + (x >> 2) * kBlock + (x & 3) * 2, kva + buf * kBuf + (x >> 2) * kBlock + (x & 3) * 2, kIdescQK, x > 0);
            tc_commit(&sm.s_bar[h]);
            if (last) tc_commit(&sm.free[buf]);
        }
        __syncwarp();
        ++tiles[h];
    };
    while (ok && walk.next(call, seg)) {
        const int units = (int)uniform((uint32_t)seg.units), halves = uniform((uint32_t)seg.rows) > 128 ? 2 : 1;
        if (!(ok = wait_warp(&sm.full[buf], phase, abort_flag))) break;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (h >= halves || !(ok = ok && wait_warp(&sm.q_bar[h], segments[h]++ & 1, abort_flag))) break;
            tc_fence_after();
            scores(h, h == halves - 1);
        }
        advance();
        for (int j = 0; ok && j < units; ++j) {
            const unsigned v_buf = buf;
            if (!(ok = wait_warp(&sm.full[buf], phase, abort_flag))) break;
            advance();                      // to K of the next tile
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h >= halves || !(ok = ok && wait_warp(&sm.p_bar[h], done[h] & 1, abort_flag))) break;
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int x = 0; x < kKeyTile / 16; ++x)
                        mma_ts(t0 + h * kGroup + kO, t0 + h * kGroup + 8 * x, (kva + v_buf * kBuf + x * (2048 >> 4)) | kBlock << 16, kIdescPV, j > 0 || x > 0);
                    tc_commit(&sm.o_bar[h]);
                    if (h == halves - 1) tc_commit(&sm.free[v_buf]);
                }
                __syncwarp();
                ++done[h];
                if (j + 1 < units) {        // the scores go where the weights are: not before those have been read
                    if (!(ok = (h > 0 || wait_warp(&sm.full[buf], phase, abort_flag)) && wait_warp(&sm.o_bar[h], (done[h] - 1) & 1, abort_flag))) break;
                    tc_fence_after();
                    scores(h, h == halves - 1);
                }
            }
            if (j + 1 < units) advance();
        }
    }
    if (!ok)                        // nor before the products have ended
        for (int h = 0; h < 2; ++h) {
            if (tiles[h]) (void)cq_mbar_wait_bounded(&sm.s_bar[h], (tiles[h] - 1) & 1);
            if (done[h]) (void)cq_mbar_wait_bounded(&sm.o_bar[h], (done[h] - 1) & 1);
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

// The copies of a warp's steps, ahead of their use and across its segments.  Sixteen rows of a page are one block of memory, which the lanes copy 16 bytes
// at a time; rows behind the last key come as zeros.  (By TMA a step cost its warp 500 clocks of issue against some 100.)
template <int D> struct Loader {
    OwnWalk walk;
    Segment seg;
    int step;                       // in the segment
    int base, ids, shift;           // page numbers base .. base + 31 of the segment's table, one a lane
    const uint8_t *k, *v;           // the layer, at this lane's 16 bytes
    uint32_t off[D / 32];           // of this lane's pieces in shared memory, by piece modulo D / 32
    __device__ __forceinline__ Loader(const Call &call, int worker, int page_shift, const void *kp, const void *vp, int lane)
        : walk(call, worker), step(0), shift(page_shift), k((const uint8_t *)kp + lane * 16), v((const uint8_t *)vp + lane * 16) {
        seg.units = 0;
        constexpr int kUnits = D / 8, kRows = 32 / kUnits;              // 16-byte units of a row, rows of a piece
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const int row = lane / kUnits + i * kRows, x = lane % kUnits;
            off[i] = (x >> 3) * (kStep * 128) + row * 128 + ((x & 7) ^ (row & 7)) * 16;
        }
    }
    __device__ __forceinline__ void send(uint32_t to, const Call &call, const cq_kv::State &st, int kv_heads, int lane) {
        constexpr int kPieces = D / 16, kPeriod = D / 32, kRows = 256 / D;      // pieces of 512 bytes; after kPeriod of them (8 rows) the pattern repeats
        if (step == seg.units && walk.next(call, seg)) {
            step = 0;
            base = INT32_MIN / 2;
        }
        if (step < seg.units) {
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
            const int64_t at = (int64_t)(((id * kv_heads + seg.head) << shift) + (key & (st.page - 1))) * (D * 2);
            const uint8_t *ks = k + at, *vs = v + at;
            const uint32_t vt = to + (uint32_t)sizeof(Step<D>) / 2;
            if (n >= kStep) {
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    const uint32_t o = off[i % kPeriod] + i / kPeriod * 1024;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + o), "l"(ks + i * 512) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(vt + o), "l"(vs + i * 512) : "memory");
                }
            } else {
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    const uint32_t o = off[i % kPeriod] + i / kPeriod * 1024;
                    const int bytes = lane / (D / 8) + i * kRows < n ? 16 : 0;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + o), "l"(ks + i * 512), "r"(bytes) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(vt + o), "l"(vs + i * 512), "r"(bytes) : "memory");
                }
            }
            ++step;
        }
        cq_cp_async_commit();           // one group a step, an empty one behind the last
    }
};

// 8 x 8 of 16 bits, a lane holding two of row lane / 4, to the same of its transpose
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <bool BF16> __device__ __forceinline__ uint32_t pack(float a, float b, float &sum_a, float &sum_b) {
    uint32_t w;
    if constexpr (BF16) {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
        sum_a += __uint_as_float(w << 16);
        sum_b += __uint_as_float(w & 0xffff0000u);
    } else {
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
        sum_a += f.x;
        sum_b += f.y;
    }
    return w;
}

// The warp's share of the own line: S^T = K Q^T (16 keys x 8 rows), O^T += V^T P^T (dims x 8 rows) by mma.sync m16n8k16.  With rows as the narrow side eight of them
// cost half the products and half the registers that they would cost as half of a 16-row side.  A lane holds rows 2 (lane % 4) and the next, keys (dims)
// lane / 4 and + 8; the weights change sides by a transposition.
// `stages_at`: shared memory of kStages steps, `stride` bytes apart.
template <int D, bool BF16, int kStages>
__device__ void own_part(uint32_t stages_at, uint32_t stride, int worker, const cq_kv_cache &cache, const cq_kv::State &st, const Call &call,
                         const uint8_t *k_layer, const uint8_t *v_layer, const uint8_t *q, int64_t q_stride, float c) {
    const int lane = threadIdx.x & 31, g = lane >> 2, x2 = (lane & 3) * 2, per = call.sh.per_kv;
    const uint32_t steps_at = uniform(stages_at);
    Loader<D> load(call, worker, 31 - __clz(st.page), k_layer, v_layer, lane);
    OwnWalk walk = load.walk;
    const int units = walk.left;
    if (units <= 0) return;
    auto send = [&](int i) { load.send(steps_at + i * stride, call, st, cache.kv_heads, lane); };
#pragma unroll 1
    for (int i = 0; i < kStages; ++i) send(i);
    // this lane's row address in the fragments' 8 x 8 blocks: of K by key and half of a 16-dim step, of V by key and half of a 16-dim tile
    const int k_key = (lane >> 3 & 1) * 8 + (lane & 7), k_half = lane >> 4, v_key = (lane >> 4) * 8 + (lane & 7), v_half = lane >> 3 & 1;
    Segment seg;
    seg.units = 0;
    int step = 0;
    uint32_t qb[D / 16][2];
    float o[D / 16][4], m0 = 0.0f, m1 = 0.0f, l0 = 0.0f, l1 = 0.0f;
    int stage = 0;
#pragma unroll 1
    for (int u = 0; u < units; ++u) {
        if (step == seg.units) {
            walk.next(call, seg);
            step = 0;
            const int query = div_per(seg.row0, call.sh);
            const uint8_t *src = q + ((int64_t)query * q_stride + (int64_t)(seg.head * per + seg.row0 - query * per + g) * D + x2) * 2;
#pragma unroll
            for (int x = 0; x < D / 16; ++x)
#pragma unroll
                for (int i = 0; i < 2; ++i) qb[x][i] = g < seg.rows ? *reinterpret_cast<const uint32_t *>(src + (16 * x + 8 * i) * 2) : 0u;
#pragma unroll
            for (int x = 0; x < D / 16; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[x][i] = 0.0f;
            l0 = l1 = 0.0f;
        }
        const int n = seg.key1 - seg.key0 - kStep * step;        // keys of this step, if fewer than 16
        cq_cp_async_wait<kStages - 1>();
        __syncwarp();
        const uint32_t kb = steps_at + stage * stride, vb = kb + (uint32_t)sizeof(Step<D>) / 2;
        float s[2][4] = {};
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {
            const int unit = 2 * x + k_half;
            uint32_t a[4];
            ldsm(a, kb + (unit >> 3) * (kStep * 128) + k_key * 128 + ((unit & 7) ^ (k_key & 7)) * 16);
            mma16816<BF16>(s[x & 1], a, qb[x][0], qb[x][1]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) s[0][i] += s[1][i];
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
        if (step == 0) { m0 = mx0; m1 = mx1; }
        else {
            const bool up0 = mx0 > m0 + 8.0f, up1 = mx1 > m1 + 8.0f;
            if (__any_sync(0xffffffffu, up0 || up1)) {
                const float f0 = up0 ? ex2(m0 - mx0) : 1.0f, f1 = up1 ? ex2(m1 - mx1) : 1.0f;
                if (up0) m0 = mx0;
                if (up1) m1 = mx1;
                l0 *= f0;
                l1 *= f1;
#pragma unroll
                for (int x = 0; x < D / 16; ++x) { o[x][0] *= f0; o[x][1] *= f1; o[x][2] *= f0; o[x][3] *= f1; }
            }
        }
        const float b0 = (m0 == -INFINITY ? 0.0f : m0) + kDown<BF16>, b1 = (m1 == -INFINITY ? 0.0f : m1) + kDown<BF16>;
        const uint32_t p0 = transpose8(pack<BF16>(ex2(__fmaf_rn(s[0][0], c, -b0)), ex2(__fmaf_rn(s[0][1], c, -b1)), l0, l1));
        const uint32_t p1 = transpose8(pack<BF16>(ex2(__fmaf_rn(s[0][2], c, -b0)), ex2(__fmaf_rn(s[0][3], c, -b1)), l0, l1));
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {
            const int unit = 2 * x + v_half;
            uint32_t a[4];
            ldsm_t(a, vb + (unit >> 3) * (kStep * 128) + v_key * 128 + ((unit & 7) ^ (v_key & 7)) * 16);
            mma16816<BF16>(o[x], a, p0, p1);
        }
        __syncwarp();
        send(stage);
        if (++stage == kStages) stage = 0;
        if (++step == seg.units) {
#pragma unroll
            for (int x = 4; x <= 16; x <<= 1) {
                l0 += __shfl_xor_sync(0xffffffffu, l0, x);
                l1 += __shfl_xor_sync(0xffffffffu, l1, x);
            }
            float *to = call.o + ((int64_t)seg.part + x2) * D + g;
#pragma unroll
            for (int x = 0; x < D / 16; ++x) {
                if (x2 < seg.rows) { to[16 * x] = o[x][0]; to[16 * x + 8] = o[x][2]; }
                if (x2 + 1 < seg.rows) { to[D + 16 * x] = o[x][1]; to[D + 16 * x + 8] = o[x][3]; }
            }
            if (g == 0) {
                if (x2 < seg.rows) call.ml[seg.part + x2] = make_float2(m0, l0);
                if (x2 + 1 < seg.rows) call.ml[seg.part + x2 + 1] = make_float2(m1, l1);
            }
        }
    }
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads, 1) prefix_mma_kernel(const cq_kv_cache cache, const Call call, const __grid_constant__ CUtensorMap k_map,
                                                                 const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CUtensorMap o_map,
                                                                 const uint8_t *k_layer, const uint8_t *v_layer,
                                                                 const uint8_t *q, int64_t q_stride, float c) {
    extern __shared__ uint8_t raw[];
    Tiles<D> &sm = *reinterpret_cast<Tiles<D> *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const cq_kv::State st = cq_kv::state_of(cache);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) { cq_mbar_init(&sm.q_bar[i], 4); cq_mbar_init(&sm.s_bar[i], 1); cq_mbar_init(&sm.p_bar[i], 4); cq_mbar_init(&sm.o_bar[i], 1); cq_mbar_init(&sm.e_bar[i], 4); }
        for (int i = 0; i < kRing; ++i) { cq_mbar_init(&sm.full[i], 1); cq_mbar_init(&sm.free[i], 1); }
        sm.abort = 0;
        cq_fence_mbar_init();
    }
    if (warp == kMmaWarp) {
        tmem_alloc(&sm.tmem, kCols);
        tmem_relinquish();
        tc_fence_before();
    }
    cq_pdl_launch_dependents();
    __syncthreads();
    tc_fence_after();
    cq_pdl_wait();
    bool ok = true;
    if (warp < kCopyWarp) {
        regs_up<kRegsSoft>();
        ok = softmax_part<D, BF16>(sm, call, o_map, q, q_stride, c, warp >> 2);
        // then own items as well, in the room of Q, K and V: no product or copy is under way when both halves are here
        asm volatile("bar.sync 3, 256;" ::: "memory");
        if (!sm.abort)
            own_part<D, BF16, 2>(cq_smem_u32(&sm.q[0][0][0]) + warp * (uint32_t)sizeof(Step<D>), (uint32_t)sizeof(sm.q), call.sh.own_first + blockIdx.x * kCopyWarp + warp, cache,
                                 st, call, k_layer, v_layer, q, q_stride, c);
    }
    else if (warp < kOwnWarp) {
        regs_down<kRegsMisc>();
        if (warp == kCopyWarp) ok = copy_part<D>(sm, cache, st, call, k_map, v_map);
        else if (warp == kMmaWarp) ok = mma_part<D, BF16>(sm, call);
    } else {
        regs_up<kRegsOwn>();            // workers from the last CTA on: where there is less than one item or tile for each, the first ones have the shared tiles
        own_part<D, BF16, Tiles<D>::kStages>(cq_smem_u32(sm.step[warp - kOwnWarp]), (uint32_t)sizeof(Step<D>), (gridDim.x - 1 - blockIdx.x) * kMmaWarps + warp - kOwnWarp, cache, st, call,
                                             k_layer, v_layer, q, q_stride, c);
    }
    if (!ok && lane == 0) atomicCAS(st.header, cq_kv::kOk, cq_kv::kTimeout);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kMmaWarp) tmem_dealloc(sm.tmem, kCols);
}

bool encode(CUtensorMap &out, CUtensorMapDataType type, int rank, const void *base, const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box) {
    using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode fn = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult res;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &res) != cudaSuccess || res != cudaDriverEntryPointSuccess) {
            (void)cudaGetLastError();
            f = nullptr;
        }
        return (Encode)f;
    }();
    const cuuint32_t one[3] = {1, 1, 1};
    return fn && fn(&out, type, rank, const_cast<void *>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// One layer of a pool as [D / 64][rows][64]; box: `boxes` blocks of 64 dims of some rows of a page.
bool pool_map(const void *base, int64_t rows, int d, int box_rows, int boxes, CUtensorMap &out) {
    const cuuint64_t dims[3] = {64, (cuuint64_t)rows, (cuuint64_t)d / 64}, strides[2] = {(cuuint64_t)d * 2, 128};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, (cuuint32_t)boxes};
    return encode(out, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, base, dims, strides, box);
}
// The partial outputs of shared items as [rows][D] f32; box: 32 x 32.
bool part_map(const Call &c, CUtensorMap &out) {
    const cuuint64_t dims[2] = {(cuuint64_t)c.sh.head_dim, (cuuint64_t)(c.shared_items + c.sh.ctas) * c.sh.row_tile}, strides[1] = {(cuuint64_t)c.sh.head_dim * 4};
    const cuuint32_t box[2] = {32, 32};
    return encode(out, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, c.o, dims, strides, box);
}

template <int D, bool BF16>
void launch(const Call &c, const cq_kv_cache &cache, const CUtensorMap (&m)[3], const uint8_t *k, const uint8_t *v, const void *q, int64_t q_stride, float scale, cudaStream_t st) {
    constexpr int smem = (int)sizeof(Tiles<D>) + 1024;
    static bool done[64];
    cq_smem_once((const void *)prefix_mma_kernel<D, BF16>, smem, done);
    cq_launch_k(prefix_mma_kernel<D, BF16>, dim3(c.sh.ctas), dim3(kThreads), smem, st, cache, c, m[0], m[1], m[2], k, v, (const uint8_t *)q, q_stride,
                (float)(scale * 1.4426950408889634));
}

}  // namespace

bool cq_attn::mma_launch(const Call &c, const cq_kv_cache &cache, int layer, const void *q, int64_t q_stride, float scale, cudaStream_t st) {
    const int64_t rows = (int64_t)cache.pages * cache.kv_heads * cache.page_size, offset = rows * layer * cache.head_dim * 2;
    const uint8_t *k = (const uint8_t *)cache.k + offset, *v = (const uint8_t *)cache.v + offset;
    const int d = cache.head_dim, box = cache.page_size, boxes = box < kKeyTile ? 1 : d / 64;
    CUtensorMap m[3];
    if (!pool_map(k, rows, d, box, boxes, m[0]) || !pool_map(v, rows, d, box, boxes, m[1]) || !part_map(c, m[2])) {
        cq_set_status(CQ_ERR_CUDA, "prefix_attention: cuTensorMapEncodeTiled is not available or refused the pool");
        return false;
    }
    const bool bf16 = c.sh.elem == CQ_BF16;
    if (c.sh.head_dim == 128) bf16 ? launch<128, true>(c, cache, m, k, v, q, q_stride, scale, st) : launch<128, false>(c, cache, m, k, v, q, q_stride, scale, st);
    else bf16 ? launch<64, true>(c, cache, m, k, v, q, q_stride, scale, st) : launch<64, false>(c, cache, m, k, v, q, q_stride, scale, st);
    return true;
}
