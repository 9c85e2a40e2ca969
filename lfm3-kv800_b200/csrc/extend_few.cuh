// kv800_extend for few queries a row (up to 6, or 8: drafted tokens, short extends), where rebuilding the keys is the work and a
// 128-row tile would be mostly padding.  The roles in the MMAs are turned round: keys are the 128 rows of the tile, the 32
// (query, query head) pairs of a KV head its columns,
//   S' = K Q'      A = K in tensor memory, B = Q' in shared memory: 128 keys x 32 columns
//   O' += V' P'    A = V' (dims x keys), B = P' (keys x columns): 128 dims x 32 columns
// so that the MMAs cost a quarter of the padded tile's, and thread t of a CTA's 128 is key t throughout: it rebuilds its key in
// registers and stores it to its lane of tensor memory (no shared memory on the way), and scales its weights by its own V scale.
// Sums over the keys stay in the threads' registers, one per column, until the segment ends.
//
// The maximum of a column lies across the threads.  It is taken for a tile only where some weight would pass 2^6; the
// group agrees on that in the barrier it needs anyway.
//
// V' wants dims in the lanes.  A quantized tile's bytes go through 4 KB of shared memory turned round (a byte in 16 bits, keys
// side by side): thread d then reads byte d % 16 of all keys, and one AND with bit d / 16 of two keys at a time leaves the pair
// of f16 subnormals 2^(d / 16 - 24), which go to tensor memory over K (done with by then).  Exact values are read there by the
// threads of their dims.
//
// A CTA is 4 groups of 128 threads, one a KV head, each with its own barriers and 128 columns of tensor memory, so that one's
// waits are another's work.  They share the tile's bytes: a ring of 3 stages filled by TMA holds the codes and bits of all heads
// (one DRAM line each), the scales and the rotation rows of the 128 positions.  (Loading them per thread, rows apart, cost 4
// times the instruction time in L1 wavefronts: 750 us where this form took 652, at 64 rows x 5 queries of 32K.)
//
// A rotated pair is summed in 32 bits and rounded once, as in extend_tc (64 rows x 5 queries of 32K 467 us; in packed bf16 438).
//
// Measured at 64 rows x 5 queries of 32K: 467 us as a graph, 452 MB at 0.97 TB/s (the floor is 69 us).  The bound is the
// instructions, about 1,050 a warp and tile of 32 keys x 20 columns, two fifths of them for the key: 58 % of the issue slots are
// used by the 16 warps that the registers allow, the rest goes in the chain from key to scores to weights to output.
// On a window or sliding layer (64 x 5, 31 us for 35 MB; 1 x 4, 21 us) a CTA has one or two tiles: latency, with instruction fetch.
// Where other forms' times stand below, they were taken side by side while the rotation was still packed (438 us).
#pragma once
#include <cuda.h>

#include "extend_tc.cuh"

namespace kv800 {

constexpr int EF_COLS = 32, EF_STAGES = 3;

// A stage: codes of 128 keys (rows of 128 bytes, all heads, 128-byte swizzle), V bits (2 keys a row, the same), cos and sin rows
// (64 bytes, 64-byte swizzle), the sub-block's scales.
struct EfStage {
    static constexpr int CODE = 0, BITS = 16384, COS = 24576, SIN = 32768, SCALE = 40960, BYTES = 43008;
};
static_assert(EF_STAGES * EfStage::BYTES <= 4 * 32768, "the ring and the heads' exact tiles share their memory");
struct EfSmem {
    static constexpr int Q = 4 * 32768, P = Q + 4 * 8192, TURN = P + 4 * 8192, TABLE = TURN + 4 * 16 * 272,
                         MAX = TABLE + 4 * 512, RED = MAX + 4 * 128, SEG = RED + 4 * 1024, BARS = SEG + 4 * 64,
                         BYTES = BARS + 192 + 1024;
};

__device__ __forceinline__ void group_sync(int id) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool group_or(int id, bool x) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"((uint32_t)x), "r"(id) : "memory");
    return r != 0;
}

// One of a group's 4 warps is ready (all lanes: operands stored and fenced): true in one lane of the last of them, which issues.
// Nobody waits here (with a barrier of the group before each: 522 us against 489 at 64 rows x 5 queries of 32K).
__device__ __forceinline__ bool last_warp(uint32_t count, int lane) {
    __syncwarp();
    uint32_t before = 0;
    if (lane == 0)
        asm volatile("atom.acq_rel.cta.shared::cta.add.u32 %0, [%1], 1;" : "=r"(before) : "r"(count) : "memory");
    return lane == 0 && (before & 3) == 3;
}

// byte offset of 16-byte chunk c (of 4) of row k (a key: 32 columns of 16 bits) in P': 64-byte rows, 64-byte swizzle
__device__ __forceinline__ uint32_t p_at(int k, int c) {
    return (uint32_t)((k >> 3) * 512 + (k & 7) * 64 + ((c ^ ((k >> 1) & 3)) << 4));
}
__device__ __forceinline__ uint64_t smem_desc64(uint32_t addr, uint32_t lbo, uint32_t sbo) {   // 64-byte swizzle
    return (uint64_t)((addr & 0x3ffff) >> 4) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) | (1ull << 46) |
           (4ull << 61);
}
// NC columns of tensor memory (a multiple of 4), waited for
template <int NC>
__device__ __forceinline__ void tmem_cols(uint32_t a, uint32_t (&r)[NC]) {
#pragma unroll
    for (int i = 0; i < NC / 8; i++) tmem_ld8(a + 8 * i, r + 8 * i);
    if (NC % 8) {
        uint32_t* x = r + NC / 8 * 8;
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(a + NC / 8 * 8));
        asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(x[0]), "+r"(x[1]), "+r"(x[2]), "+r"(x[3])::"memory");
    }
#pragma unroll
    for (int i = 0; i < NC / 8; i++) tmem_wait_ld8(r + 8 * i);
}

// Over the warp's 32 lanes of N <= 32 values a lane: lane i < N is left with the sum, or the maximum, of
// value i.  The first step folds lanes 16 apart and keeps N values or, for N > 16, sends the upper 16 one way and the lower the
// other; each later one halves the values.
template <int N, bool MAX>
__device__ __forceinline__ float fold_lanes(float (&x)[N], int lane) {
    auto both = [](float a, float b) { return MAX ? fmaxf(a, b) : a + b; };
    float y[16];
    const bool up = lane & 16;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const float hi = 16 + i < N ? x[16 + i < N ? 16 + i : 0] : (MAX ? -INFINITY : 0.0f);
        if (N <= 16) {
            y[i] = i < N ? both(x[i < N ? i : 0], __shfl_xor_sync(0xffffffffu, x[i < N ? i : 0], 16)) : 0.0f;
        } else if (16 + i < N) {
            y[i] = both(up ? hi : x[i], __shfl_xor_sync(0xffffffffu, up ? x[i] : hi, 16));
        } else {
            y[i] = both(x[i], __shfl_xor_sync(0xffffffffu, x[i], 16));
        }
    }
#pragma unroll
    for (int o = 8; o; o >>= 1) {
        const bool u = lane & o;
#pragma unroll
        for (int i = 0; i < o; i++) {
            const float keep = u ? y[i + o] : y[i], send = u ? y[i] : y[i + o];
            y[i] = both(keep, __shfl_xor_sync(0xffffffffu, send, o));
        }
    }
    return y[0];
}

// O' from the Hadamard domain to the plain one, in place: thread = dim, sum P' bit in units of 2^(dim / 16 - 24) for the NC
// columns.  Two butterfly levels across the warps through `buf` (8 columns, 4 KB, at a time), five across the lanes.  off, the
// threads' parts of sum p * offset, adds to dim 0 alone, times sqrt(128); it is left at zero.
template <int NC>
__device__ __forceinline__ void ef_turn(uint32_t o, f2 (&off2)[NC / 2], float* red, float* buf, int tid, int id) {
    const int lane = tid & 31, warp = tid >> 5;
    {
        float off[NC];
#pragma unroll
        for (int r = 0; r < NC / 2; r++) {
            off2[r].get(off[2 * r], off[2 * r + 1]);
            off2[r] = f2(0.0f, 0.0f);
        }
        red[warp * 32 + lane] = fold_lanes<NC, false>(off, lane);
    }
    const float unit = __uint_as_float((uint32_t)(127 + 24 - (tid >> 4)) << 23);
    const float s1 = warp & 1 ? -1.0f : 1.0f, s2 = warp & 2 ? -1.0f : 1.0f;
#pragma unroll
    for (int g = 0; g < (NC + 7) / 8; g++) {
        uint32_t x[8];
        tmem_ld8(o + 8 * g, x);
        tmem_wait_ld8(x);
        group_sync(id);
#pragma unroll
        for (int i = 0; i < 8; i++) buf[i * 128 + tid] = __uint_as_float(x[i]) * unit;
        group_sync(id);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float* c = buf + i * 128 + lane;
            float y = fmaf(s2, fmaf(s1, c[96], c[64]), fmaf(s1, c[32], c[0]));
#pragma unroll
            for (int k = 1; k < 32; k <<= 1) {
                const float z = __shfl_xor_sync(0xffffffffu, y, k);
                y = lane & k ? z - y : y + z;
            }
            y *= 0.08838834764831845f;
            const int r = 8 * g + i;
            if (tid == 0) y = fmaf(red[r] + red[32 + r] + red[64 + r] + red[96 + r], 11.313708498984761f, y);
            x[i] = __float_as_uint(y);
        }
        tmem_st8(o + 8 * g, x);
    }
    tmem_wait_st();
    group_sync(id);     // red and buf are free again
}

// The segment a CTA works on, in shared memory (registers are what this kernel lacks): one copy for each group, which may be a
// segment apart.
struct EfSeg {
    int t0, t1, slot, more;
    ExItem item;
};

// What a group of 128 threads (one KV head) carries through its tiles.
template <int NC>
struct EfGroup {
    int tid, lane, warp, h, id;
    uint32_t T_KV, T_S, T_O, lanes;         // tensor memory: 64 + 32 + 32 columns; this warp's lanes
    uint32_t b_s, b_p, ns, np;              // barriers of S and of O, MMA groups waited for
    uint32_t n_k, n_v;                      // counts of warps that are ready with K, with V' and P'
    uint32_t q_sm, p_sm, turn_sm, table_sm;
    float *s_neg, *s_red, *buf;             // minus the columns' maxima (log2 domain); reductions; P' as floats
    volatile int* gave_up;
    f2 l[NC / 2], off[NC / 2];
    bool turned;                            // O' is in the plain domain, or empty

    __device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity) {
        return !group_or(id, !bar_wait(bar, parity, gave_up));
    }
};

// A warp's 32 rows of 256 bytes (lane i holds row i's address, null for zeros) into a tile in shared memory, 16 lanes a row.
// -> rows with a value that is not finite, if asked for; they are stored as zeros.
template <bool CHECK>
__device__ __forceinline__ uint32_t ef_gather(const uint16_t* row, uint32_t tile, int warp, int lane) {
    uint32_t bads = 0;
#pragma unroll 1
    for (int half = 0; half < 2; half++) {
        uint4 v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint4* src = reinterpret_cast<const uint4*>(
                __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(row), 16 * half + 2 * i + (lane >> 4)));
            v[i] = src ? __ldg(src + (lane & 15)) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int r = 16 * half + 2 * i;
            if (CHECK) {
                uint32_t nan = bf2_fma(v[i].x & 0x7fff7fffu, 0u, 0u);   // stays +0 while every value is finite: x * 0 + nan
                nan = bf2_fma(v[i].y & 0x7fff7fffu, 0u, nan);
                nan = bf2_fma(v[i].z & 0x7fff7fffu, 0u, nan);
                nan = bf2_fma(v[i].w & 0x7fff7fffu, 0u, nan);
                const uint32_t any = __ballot_sync(0xffffffffu, nan != 0);
                if (any) {
                    if (any >> (lane & 16) & 0xffffu) v[i] = make_uint4(0, 0, 0, 0);
                    bads |= ((any & 0xffffu ? 1u : 0u) | (any >> 16 ? 2u : 0u)) << r;
                }
            }
            st_shared16(tile + tile_at(32 * warp + r + (lane >> 4), lane & 15), v[i].x, v[i].y, v[i].z, v[i].w);
        }
    }
    return bads;
}

// One tile of 128 keys.  stage: a quantized tile's stage of the ring (good: the key's sub-block and rotation exist), or the
// 32 KB an exact tile's rows kr, vr pass through (K on its way to the threads of its keys, then V as an MMA operand).
// failed: a wait before this tile was given up.  The group leaves together, where it agrees on the maxima.
template <bool QUANT, int NC, typename Release>
__device__ __forceinline__ bool ef_tile(const ExtendArgs& a, EfGroup<NC>& g, const volatile ExItem& t, bool begin, bool failed, int kp, bool good,
                                        uint32_t stage, int half, const uint16_t* kr, const uint16_t* vr,
                                        Release release) {
    using G = EfStage;
    const int tid = g.tid, h = g.h;
    // ---- K: 16 columns of tensor memory per pair of code words
    if (!QUANT) {
        if (!begin) {      // the tile before is done with V, K and O
            failed |= !warp_wait(g.b_p, g.np & 1, g.gave_up);
            g.np++;
            tc_fence_after();
        }
        if (good) {        // on its way while K is built
            asm volatile("prefetch.global.L2 [%0];" ::"l"(vr));
            asm volatile("prefetch.global.L2 [%0];" ::"l"(vr + 64));
        }
        ef_gather<false>(kr, stage, g.warp, g.lane);
        __syncwarp();
    }
    // (64 rows x 5 queries of 32K: a turn at a time 465 us, two 449, all four 438)
#pragma unroll
    for (int u = 0; u < 4; u++) {
        uint32_t k[16];     // [plane][even, odd of word 2 u; even, odd of word 2 u + 1]
        uint4 c, s;
        if (QUANT) {
            const uint2 code = ld_shared8(stage + G::CODE + tid * 128 + (((2 * h + (u >> 1)) ^ tid) & 7) * 16 + (u & 1) * 8);
            const uint32_t at = stage + tid * 64 + ((u ^ ((tid >> 1) & 3)) << 4);
            c = ld_shared16(at + G::COS);
            s = ld_shared16(at + G::SIN);
#pragma unroll
            for (int v = 0; v < 2; v++) {
                const uint32_t ev = v ? code.y : code.x, od = ev >> 8;
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const uint4 x = ld_shared16(g.table_sm + ((2 * u + v) * 4 + q) * 16);
                    k[4 * q + 2 * v] = bf2_fma(ev & (0x00030003u << (2 * q)), x.x, x.y);
                    k[4 * q + 2 * v + 1] = bf2_fma(od & (0x00030003u << (2 * q)), x.z, x.w);
                }
            }
        } else {
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const uint4 x = ld_shared16(stage + tile_at(tid, 4 * q + u));
                k[4 * q] = prmt(x.x, x.y, 0x5410), k[4 * q + 1] = prmt(x.x, x.y, 0x7632);
                k[4 * q + 2] = prmt(x.z, x.w, 0x5410), k[4 * q + 3] = prmt(x.z, x.w, 0x7632);
            }
            c = s = make_uint4(0, 0, 0, 0);
            if (a.cos_t && good) {
                c = __ldg(reinterpret_cast<const uint4*>(a.cos_t + (int64_t)kp * 32) + u);
                s = __ldg(reinterpret_cast<const uint4*>(a.sin_t + (int64_t)kp * 32) + u);
            }
        }
        if (QUANT || a.cos_t) {
            turn_packed(k[0], k[8], prmt(c.x, c.y, 0x5410), prmt(s.x, s.y, 0x5410));
            turn_packed(k[1], k[9], prmt(c.x, c.y, 0x7632), prmt(s.x, s.y, 0x7632));
            turn_packed(k[2], k[10], prmt(c.z, c.w, 0x5410), prmt(s.z, s.w, 0x5410));
            turn_packed(k[3], k[11], prmt(c.z, c.w, 0x7632), prmt(s.z, s.w, 0x7632));
        }
        if (QUANT && u == 0 && !begin) {      // the tile before is done with K / V and O
            failed |= !warp_wait(g.b_p, g.np & 1, g.gave_up);
            g.np++;
            tc_fence_after();
        }
        tmem_st16(g.T_KV + g.lanes + 16 * u, k);
    }
    tmem_wait_st();
    tc_fence_before();
    if (last_warp(g.n_k, g.lane)) {
        constexpr uint32_t D = mma_desc(1, 128, EF_COLS, 0, 0);
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < 8; k++)
            mma_ts(g.T_S, g.T_KV + 8 * k, smem_desc(g.q_sm + (k >> 2) * 4096 + (k & 3) * 32, 16, 1024), D, k > 0);
        mma_commit(g.b_s);
    }
    // ---- while the scores are made: the V bytes, the V scales, which queries see the key (bit i of hide: query i does not)
    float vs = 1.0f, vl = 0.0f;
    if (QUANT) {
        const uint4 x = ld_shared16(stage + G::BITS + (tid >> 1) * 128 + ((((tid & 1) * 4 + h) ^ (tid >> 1)) & 7) * 16);
        const uint32_t v[4] = {x.x, x.y, x.z, x.w};
        const uint32_t turn = g.turn_sm + tid * 2;
#pragma unroll
        for (int j = 0; j < 16; j++)
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(turn + j * 272), "h"((uint16_t)prmt(v[j >> 2], 0, 0x4440 + (j & 3))) : "memory");
        const uint32_t at = stage + G::SCALE + (half * EX_TILE + tid) * 2 + (h >> 1);
        uint32_t bs, bl;
        asm volatile("ld.shared.u8 %0, [%1];" : "=r"(bs) : "r"(at + (VSC_O - VLO_O)));
        asm volatile("ld.shared.u8 %0, [%1];" : "=r"(bl) : "r"(at));
        f8_pair(good ? bs : 0u, good ? bl : 0u, vs, vl);
        release();
    }
    bool bad = false;      // the key's value is not finite: zeros stand for it, which no weight of zero turns into NaN
    if (QUANT) {
        if (!(vs + vl < INFINITY)) bad = true, vs = vl = 0.0f;
    } else {
        bad = ef_gather<true>(vr, stage, g.warp, g.lane) >> g.lane & 1;
    }
    uint32_t hide = good ? below(kp - t.p0) : 0xffu;
    if (!QUANT && a.P.win && !(a.P.sk && kp < (int)a.P.nsink)) hide |= ~below((int)min((int64_t)kp - t.p0 + a.P.win, (int64_t)32));
    hide &= 0xffu;
    if (bad) {             // whoever sees it becomes NaN
        const float nan = __uint_as_float(0x7fc00000u);
#pragma unroll
        for (int i = 0; i < NC / 4; i++)
            if (!((hide >> i) & 1)) g.l[2 * i] = g.l[2 * i + 1] = f2(nan, nan);
    }
    // ---- weights
    failed |= !warp_wait(g.b_s, g.ns & 1, g.gave_up);
    g.ns++;
    tc_fence_after();
    const float sc = QUANT ? EX_SCALE * 16384.0f : EX_SCALE;
    const bool any = __any_sync(0xffffffffu, hide != 0);
    uint32_t s[NC];
    tmem_cols<NC>(g.T_S + g.lanes, s);
    if (any)
#pragma unroll
        for (int i = 0; i < NC; i++)
            if ((hide >> (i >> 2)) & 1) s[i] = 0xff800000u;
    float top = -INFINITY;
    {
        const f2 sc2(sc, sc);
#pragma unroll
        for (int i = 0; i < NC / 4; i++) {
            const float4 m = *reinterpret_cast<const float4*>(g.s_neg + 4 * i);
            float x, y, z, w;
            fma2(f2(__uint_as_float(s[4 * i]), __uint_as_float(s[4 * i + 1])), sc2, f2(m.x, m.y)).get(x, y);
            fma2(f2(__uint_as_float(s[4 * i + 2]), __uint_as_float(s[4 * i + 3])), sc2, f2(m.z, m.w)).get(z, w);
            top = fmaxf(fmaxf(top, fmaxf(x, y)), fmaxf(z, w));
            s[4 * i] = __float_as_uint(x), s[4 * i + 1] = __float_as_uint(y);
            s[4 * i + 2] = __float_as_uint(z), s[4 * i + 3] = __float_as_uint(w);
        }
    }
    if (group_or(g.id, top > EX_LAZY || failed)) {     // move the maxima (of a column's first keys: set them)
        if (group_or(g.id, failed)) return false;
        tmem_cols<NC>(g.T_S + g.lanes, s);
        {
            float x[NC];
#pragma unroll
            for (int i = 0; i < NC; i++) {
                x[i] = (hide >> (i >> 2)) & 1 ? -INFINITY : __uint_as_float(s[i]) * sc;
                s[i] = __float_as_uint(x[i]);
            }
            g.s_red[g.warp * 32 + g.lane] = fold_lanes<NC, true>(x, g.lane);
        }
        group_sync(g.id);
        if (tid < 32) {
            const float m0 = -g.s_neg[tid];
            float m1 = fmaxf(fmaxf(g.s_red[tid], g.s_red[32 + tid]), fmaxf(g.s_red[64 + tid], g.s_red[96 + tid]));
            m1 = fmaxf(m1, m0);
            g.s_neg[tid] = -m1;
            g.s_red[128 + tid] = exp2_approx(m0 - m1);
        }
        group_sync(g.id);
#pragma unroll
        for (int r = 0; r < NC / 2; r++) {
            const f2 f(g.s_red[128 + 2 * r], g.s_red[128 + 2 * r + 1]);
            g.l[r] = mul2(g.l[r], f);
            g.off[r] = mul2(g.off[r], f);
        }
#pragma unroll
        for (int i = 0; i < NC; i++) s[i] = __float_as_uint(__uint_as_float(s[i]) + g.s_neg[i]);
        if (!begin) {
#pragma unroll
            for (int i = 0; i < (NC + 7) / 8; i++) {
                uint32_t o[8];
                tmem_ld8(g.T_O + g.lanes + 8 * i, o);
                tmem_wait_ld8(o);
#pragma unroll
                for (int k = 0; k < 8; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * g.s_red[128 + 8 * i + k]);
                tmem_st8(g.T_O + g.lanes + 8 * i, o);
            }
            tmem_wait_st();
        }
    }
    if (!QUANT && !g.turned) {
        g.turned = true;
        ef_turn<NC>(g.T_O + g.lanes, g.off, g.s_red, g.buf, tid, g.id);
    }
    if (QUANT) g.turned = false;
    const f2 vs2(vs, vs), vl2(vl, vl);
#pragma unroll
    for (int i = 0; i < (NC + 7) / 8; i++) {
        uint32_t pk[4] = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < 4 && 8 * i + 2 * k < NC; k++) {
            float x = exp2_approx(__uint_as_float(s[8 * i + 2 * k])), y = exp2_approx(__uint_as_float(s[8 * i + 2 * k + 1]));
            const f2 pp(x, y);
            g.l[4 * i + k] = add2(g.l[4 * i + k], pp);
            if (QUANT) {
                g.off[4 * i + k] = fma2(pp, vl2, g.off[4 * i + k]);
                mul2(pp, vs2).get(x, y);
            }
            pk[k] = QUANT ? pack2_f16(x, y) : pack2_bf16(x, y);
        }
        st_shared16(g.p_sm + p_at(tid, i), pk[0], pk[1], pk[2], pk[3]);
    }
    // ---- V': thread = dim
    if (QUANT) {
        const uint32_t bit = 0x00010001u << (tid >> 4), src = g.turn_sm + (tid & 15) * 272;
#pragma unroll 1
        for (int i = 0; i < 4; i++) {
            uint32_t k[16];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint4 x = ld_shared16(src + 64 * i + 16 * j);
                k[4 * j] = x.x & bit, k[4 * j + 1] = x.y & bit, k[4 * j + 2] = x.z & bit, k[4 * j + 3] = x.w & bit;
            }
            tmem_st16(g.T_KV + g.lanes + 16 * i, k);
        }
    }
    tmem_wait_st();
    fence_async_smem();
    tc_fence_before();
    if (last_warp(g.n_v, g.lane)) {
        constexpr uint32_t D = mma_desc(QUANT ? 0 : 1, 128, EF_COLS, QUANT ? 0 : 1, 1);
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const uint64_t p = smem_desc64(g.p_sm + k * 1024, 16, 512);
            if (QUANT) mma_ts(g.T_O, g.T_KV + 8 * k, p, D, !begin || k > 0);
            else mma_ss(g.T_O, smem_desc(stage + k * 2048, 16384, 1024), p, D, !begin || k > 0);
        }
        mma_commit(g.b_p);
    }
    return true;
}

// The plan of extend_plan, made by each CTA for its own part, a row a thread (at most 512 rows): one load's latency and two barriers
// instead of a launch and its results' way through memory.  64 rows x 5 queries of a window take 31 us so, 33
// with extend_plan, a single row of 4 queries 22.4 and 23.7.
__device__ __forceinline__ void ef_plan(const ExtendArgs& a, const ExPlan& pl, volatile int* sums) {
    const int r = threadIdx.x, lane = r & 31, warp = r >> 5;
    ExItem it{};
    int units = 0;
    if (blockIdx.x == 0) ex_clear_first(a);
    if (r < a.R) {
        const int64_t q0 = a.qsl[r], q1 = a.qsl[r + 1];
        ExRow row;
        ex_row(a, r, row);
        int64_t ql = row.q1 - row.q0;
        if (blockIdx.x == 0 && (q1 < q0 || q0 < 0 || q1 > a.T || ql > a.max_qlen)) {
            ex_flag(a, ST_TABLE);
            for (int64_t t = row.q0 + a.max_qlen; t < row.q1; t++)
                for (int d = 0; d < 16 * DIM; d++) a.out[t * 16 * DIM + d] = 0;
        }
        if (ql > a.max_qlen) ql = a.max_qlen;
        if (ql > 0) {
            ExKeys k;
            ex_keys(a, row, row.n0, row.n0 + ql - 1, k);
            it.b = r, it.nq = (int)ql, it.q0 = (int)row.q0, it.p0 = (int)row.n0, it.ns = (int)row.ns;
            it.nexact = (int)k.nexact, it.nsk = (int)k.nsk, it.xlo = (int)k.xlo;
            it.quant = (int)((k.nquant + EX_TILE - 1) / EX_TILE);
            const int n = it.quant + (int)((k.nexact + EX_TILE - 1) / EX_TILE);
            it.tiles = n > 0 ? n : 1;
            it.lead = pl.lead;
            units = it.lead + it.tiles;
        }
    }
    auto plus = [](int x, int y) { return (int)min((uint32_t)x + (uint32_t)y, 0x40000000u); };   // stops at 2^30
    int x = units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x = plus(x, y);
    }
    const uint32_t some = __ballot_sync(0xffffffffu, units > 0);
    if (lane == 31) sums[warp] = x, sums[16 + warp] = __popc(some);
    __syncthreads();
    const int left = __shfl_up_sync(0xffffffffu, x, 1);
    int W = 0, index = __popc(some & ((1u << lane) - 1));
    it.base = lane ? left : 0;
#pragma unroll
    for (int w = 0; w < 16; w++) {
        if (w == warp) it.base = plus(W, it.base);
        if (w < warp) index += sums[16 + w];
        W = plus(W, sums[w]);
    }
    if (W >= 0x40000000) {     // no cache holds this many keys
        if (r == 0 && blockIdx.x == 0) ex_flag(a, ST_TABLE);
        W = 0;
    }
    const ExCut cut(W, pl.parts);
    const int u0 = cut.start(blockIdx.x), u1 = cut.start(blockIdx.x + 1);
    if (u0 < u1 && units && it.base < u1 && it.base + units > u0) {
        pl.items[index] = it;
        if (it.base <= u0) pl.part[blockIdx.x] = ExPart{u0, u1, W, index, it};
    }
    if (u0 >= u1 && r == 0) pl.part[blockIdx.x] = ExPart{W, W, W, 0, ExItem{}};
    __syncthreads();
}

template <int NC>     // columns in use: 4 heads x 4 to 8 queries
__global__ void __launch_bounds__(512, 1)
    extend_few(const __grid_constant__ ExtendArgs a, const __grid_constant__ ExPlan pl, const __grid_constant__ ExMaps maps) {
    using L = EfSmem;
    using G = EfStage;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t sm0 = smem_u32(smem_raw), sm = (sm0 + 1023) & ~1023u;
    uint8_t* smp = smem_raw + (sm - sm0);
    EfGroup<NC> g;
    const int h = g.h = threadIdx.x >> 7, tid = g.tid = threadIdx.x & 127;
    g.lane = tid & 31, g.warp = tid >> 5, g.id = 1 + h;
    const uint32_t bars = sm + L::BARS, b_full = bars, b_free = bars + 24, b_ring = bars + 144;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smp + L::BARS + 112);
    g.gave_up = reinterpret_cast<volatile int*>(smp + L::BARS + 116);
    volatile int* s_ok = reinterpret_cast<volatile int*>(smp + L::BARS + 128);   // a stage's sub-block lies in the pool
    g.b_s = bars + 48 + 16 * h, g.b_p = g.b_s + 8, g.ns = g.np = 0;
    g.n_k = bars + 160 + 8 * h, g.n_v = g.n_k + 4;
    g.q_sm = sm + L::Q + h * 8192, g.p_sm = sm + L::P + h * 8192, g.turn_sm = sm + L::TURN + h * (16 * 272);
    g.table_sm = sm + L::TABLE + h * 512;
    g.s_neg = reinterpret_cast<float*>(smp + L::MAX + h * 128);
    g.s_red = reinterpret_cast<float*>(smp + L::RED + h * 1024);
    g.buf = reinterpret_cast<float*>(smp + L::P + h * 8192);
    // A wait by parity tells a phase from the next one only.  None here can fall further behind: a stage's next fill waits for its
    // release by all 16 warps, its next release for that fill; a group's next product for all its warps to be ready again, each of
    // which has waited for the one before; the ring's next return for the copies of the segment it was returned in.
    if (threadIdx.x == 0) {
        for (int i = 0; i < EF_STAGES; i++) {
            bar_init(b_full + 8 * i, 1);
            bar_init(b_free + 8 * i, 16);
        }
        for (int i = 0; i < 8; i++) bar_init(bars + 48 + 8 * i, 1);
        bar_init(b_ring, 16);
        for (int i = 0; i < 8; i++) reinterpret_cast<volatile uint32_t*>(smp + L::BARS + 160)[i] = 0;
        *g.gave_up = 0;
        if (a.own) a.status[1 + blockIdx.x] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x < 32) tmem_alloc(smem_u32(tmem_slot), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    g.T_KV = *tmem_slot + 128 * h, g.T_S = g.T_KV + 64, g.T_O = g.T_KV + 96, g.lanes = (uint32_t)(g.warp * 32) << 16;
    pdl_wait();
    pdl_launch_dependents();
    if (a.own) ef_plan(a, pl, reinterpret_cast<volatile int*>(smp + L::RED));
    // tokens after the last row's, which no row owns
    const int64_t owned = a.R && a.qsl[a.R] > 0 ? a.qsl[a.R] : 0;
    for (int64_t t = owned + (int64_t)blockIdx.x; t < a.T; t += gridDim.x)
        for (int d = threadIdx.x; d < 16 * DIM / 8; d += 512)
            reinterpret_cast<uint4*>(a.out + t * 16 * DIM)[d] = make_uint4(0, 0, 0, 0);
    uint32_t kq = 0, issued = 0;   // quantized tiles used; tiles fetched (thread 0)
    bool lent = false;             // exact tiles have borrowed the ring since this head's last quantized one
    uint32_t taken = 0;            // times it was taken back (thread 0)
    bool ok = true;                // no wait has been given up

    volatile EfSeg& seg = *reinterpret_cast<volatile EfSeg*>(smp + L::SEG + h * 64);
    volatile ExItem& t = seg.item;
    int u, u1, it;              // thread 0 of the group: the part's tiles left, the item
    if (tid == 0) {
        const int4* src = reinterpret_cast<const int4*>(pl.part + blockIdx.x);
        const int4 x = src[0];
        u = x.x, u1 = x.y, it = x.w;
#pragma unroll
        for (int i = 0; i < 3; i++) reinterpret_cast<int4*>(smp + L::SEG + h * 64 + 16)[i] = src[1 + i];
    }
    const int u0 = u;
    for (;;) {
        if (tid == 0) {
            bool more = u < u1;
            if (more) {
                if (u >= t.base + t.lead + t.tiles) {
                    const int4* src = reinterpret_cast<const int4*>(pl.items + ++it);
#pragma unroll
                    for (int i = 0; i < 3; i++) reinterpret_cast<int4*>(smp + L::SEG + h * 64 + 16)[i] = src[i];
                }
                const int tiles = t.tiles, from = u - t.base - t.lead, t0 = max(from, 0), t1 = min(tiles, from + (u1 - u));
                more = t1 > 0;           // the part may end before the item's first tile
                seg.t0 = t0, seg.t1 = t1;
                seg.slot = (t0 == 0 && t1 == tiles) ? -1 : ((u == u0 ? 2 * (int)blockIdx.x : 2 * (int)blockIdx.x + 1) * HEADS + h);
                u += t1 - from;
            }
            seg.more = more;
        }
        group_sync(g.id);
        if (!seg.more) break;
        const int rows = 4 * t.nq, t0 = seg.t0, t1 = seg.t1, qend = min(t1, t.quant);
        auto fetch = [&](int ti) {     // thread 0 of the CTA: the bytes of a quantized tile into the ring's next stage
            const uint32_t st = issued % EF_STAGES, ph = (issued / EF_STAGES) & 1;
            if (!bar_wait(b_free + 8 * st, ph ^ 1, g.gave_up)) return;
            const uint8_t* sb = ex_subblock(a, t.b, ti >> 1);
            s_ok[st] = sb != nullptr;
            const uint32_t bar = b_full + 8 * st, dst = sm + st * G::BYTES;
            if (sb) {
                const int row = (int)((sb - a.P.qpool) / 128), half = ti & 1;
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(G::BYTES) : "memory");
                ex_tma(dst + G::CODE, &maps.rows, 0, row + KC_O / 128 + 128 * half, bar);
                ex_tma(dst + G::CODE + 8192, &maps.rows, 0, row + KC_O / 128 + 128 * half + 64, bar);
                ex_tma(dst + G::BITS, &maps.rows, 0, row + VB_O / 128 + 64 * half, bar);
                ex_tma(dst + G::COS, &maps.cos, 0, ti * EX_TILE, bar);
                ex_tma(dst + G::SIN, &maps.sin, 0, ti * EX_TILE, bar);
                ex_tma(dst + G::SCALE, &maps.scales, 0, row + VLO_O / 128, bar);
            } else {
                bar_arrive(bar);
            }
            issued++;
        };
        // exact tiles borrow the ring.  Each warp gives it back where its next segment with quantized tiles begins (the group's
        // exact tiles are done then), and copies wait until all 16 have.  No head gets past that segment before the copies, so the
        // barrier is one phase ahead of this wait at most; a count of the segments with exact tiles would be any number ahead, for
        // the heads walk such segments apart, and a parity cannot tell two phases from none.
        if (t0 < qend) {
            if (lent && g.lane == 0) bar_arrive(b_ring);
            if (threadIdx.x == 0) {
                const bool clear = !lent || bar_wait(b_ring, taken++ & 1, g.gave_up);
                for (int k = 0; clear && k < EF_STAGES - 1 && t0 + k < qend; k++) fetch(t0 + k);
            }
            lent = false;
        }
        {   // Q': natural dims of chunk c = 4 plane + pair, stored as chunk 4 pair + plane, groups of four as (0, 2, 1, 3)
            const int r = tid >> 2;
            const uint4* src = reinterpret_cast<const uint4*>(a.q + ((int64_t)(t.q0 + (r >> 2)) * 16 + h * 4 + (r & 3)) * DIM);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int c = 4 * i + (tid & 3), pos = 4 * (tid & 3) + i;
                const uint4 x = r < rows ? __ldg(src + c) : make_uint4(0, 0, 0, 0);
                st_shared16(g.q_sm + (pos >> 3) * 4096 + (r >> 3) * 1024 + (r & 7) * 128 + (((pos ^ r) & 7) << 4),
                            prmt(x.x, x.y, 0x5410), prmt(x.x, x.y, 0x7632), prmt(x.z, x.w, 0x5410), prmt(x.z, x.w, 0x7632));
            }
            fence_async_smem();
            if (tid < 32) g.s_neg[tid] = 1e30f;
            group_sync(g.id);
        }
#pragma unroll
        for (int r = 0; r < NC / 2; r++) g.l[r] = g.off[r] = f2(0.0f, 0.0f);
        g.turned = true;
        int table = -1;
        for (int ti = t0; ok && ti < qend; ti++) {
            const uint32_t st = kq % EF_STAGES;
            if (threadIdx.x == 0 && ti + EF_STAGES - 1 < qend) fetch(ti + EF_STAGES - 1);
            const bool failed = !warp_wait(b_full + 8 * st, (kq / EF_STAGES) & 1, g.gave_up);
            const int kp = ti * EX_TILE + tid;
            const bool sub = s_ok[st] != 0, good = sub && kp < a.npos;
            if (sub && !good) ex_flag(a, ST_TABLE);
            if (table != (ti >> 1)) {   // [word][plane]: (scale, offset) of its even dims, of its odd dims
                table = ti >> 1;
                {
                    const int e = tid & 63, lo = tid >> 6, wd = e >> 3, q = (e >> 1) & 3, od = e & 1, d = 32 * q + 4 * wd + od;
                    const uint8_t* src = smp + st * G::BYTES + G::SCALE + (lo ? KLO_O - VLO_O : KSC_O - VLO_O) + h * DIM + d;
                    float x = 0, y = 0;
                    if (sub) f8_pair(src[0], src[2], x, y);
                    const float by = lo ? 6.103515625e-05f : __uint_as_float((uint32_t)(127 + 119 - 2 * q) << 23);
                    *reinterpret_cast<uint32_t*>(smp + L::TABLE + h * 512 + e * 8 + lo * 4) = pack2_bf16(x * by, y * by);
                }
                group_sync(g.id);
            }
            ok = ef_tile<true, NC>(a, g, t, ti == t0, failed, kp, good, sm + st * G::BYTES, ti & 1, nullptr, nullptr, [&] {
                __syncwarp();
                if (g.lane == 0) bar_arrive(b_free + 8 * st);
            });
            kq++;
        }
        const int x0 = max(t0, t.quant);
        if (x0 < t1)      // the ring's last tiles are done with by all heads
            for (uint32_t k = kq < EF_STAGES ? 0 : kq - EF_STAGES; ok && k < kq; k++)
                ok = g.wait(b_free + 8 * (k % EF_STAGES), (k / EF_STAGES) & 1);
        for (int ti = x0; ok && ti < t1; ti++) {
            const int e = (ti - t.quant) * EX_TILE + tid;
            bool good = e < t.nexact;
            const int kp = e < t.nsk ? e : t.xlo + (e - t.nsk);
            const uint16_t *kr = nullptr, *vr = nullptr;
            if (good) good = ex_exact(a, t.b, t.ns, h, kp, kr, vr);
            if (good && a.cos_t && kp >= a.npos) {
                ex_flag(a, ST_TABLE);
                good = false;
            }
            if (!good) kr = vr = nullptr;
            ok = ef_tile<false, NC>(a, g, t, ti == t0, false, kp, good, sm + h * 32768, 0, kr, vr, [] {});
        }
        if (!ok) break;
        ok = g.wait(g.b_p, g.np & 1);
        g.np++;
        if (!ok) break;
        tc_fence_after();
        lent |= x0 < t1;
        if (!g.turned) ef_turn<NC>(g.T_O + g.lanes, g.off, g.s_red, g.buf, tid, g.id);
        // sums over the keys
        {
            float x[NC];
#pragma unroll
            for (int r = 0; r < NC / 2; r++) g.l[r].get(x[2 * r], x[2 * r + 1]);
            g.s_red[g.warp * 32 + g.lane] = fold_lanes<NC, false>(x, g.lane);
        }
        group_sync(g.id);
        if (tid < NC) {
            const float sum = g.s_red[tid] + g.s_red[32 + tid] + g.s_red[64 + tid] + g.s_red[96 + tid];
            g.s_red[128 + tid] = seg.slot < 0 ? (sum == 0.0f ? 0.0f : 1.0f / sum) : 1.0f;
            if (seg.slot >= 0 && tid < rows) pl.ml[(int64_t)seg.slot * 32 + tid] = make_float2(-g.s_neg[tid], sum);
        }
        group_sync(g.id);
#pragma unroll
        for (int i = 0; i < (NC + 7) / 8; i++) {
            uint32_t o[8];
            tmem_ld8(g.T_O + g.lanes + 8 * i, o);
            tmem_wait_ld8(o);
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int r = 8 * i + k;
                if (r < rows) {
                    if (seg.slot < 0)
                        a.out[((int64_t)(t.q0 + (r >> 2)) * 16 + h * 4 + (r & 3)) * DIM + tid] =
                            f2bf(__uint_as_float(o[k]) * g.s_red[128 + r]);
                    else
                        pl.o[((int64_t)seg.slot * 32 + r) * DIM + tid] = __uint_as_float(o[k]);
                }
            }
        }
        tc_fence_before();
        group_sync(g.id);     // O, Q', the maxima and the sums are free
        tc_fence_after();
    }
    if (threadIdx.x == 0 && *g.gave_up) {      // copies still in flight land before the CTA ends
        const uint64_t t0 = now_ns();
        for (uint32_t k = kq; k < issued; k++)
            while (!bar_try(b_full + 8 * (k % EF_STAGES), (k / EF_STAGES) & 1) && now_ns() - t0 < 1000000000ull) {
            }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x < 32) {
        tc_fence_after();
        tmem_free(*tmem_slot, 512);
    }
    if (threadIdx.x == 0 && *g.gave_up) ex_flag(a, ST_TIMEOUT);
}

}  // namespace kv800
