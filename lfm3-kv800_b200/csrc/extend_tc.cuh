// kv800_extend on the tensor cores (tcgen05), for tiles of MT x 128 rows: a row is one (query, query head) pair, the 4 heads
// of a KV head side by side, so a tile of 128 rows is 32 queries against one KV head.
//
//   S = Q K^T      per 128 keys, M = 128 rows, N = 128 keys: both operands in shared memory, S in tensor memory
//   P = 2^(S c - m)  one thread a row, the running maximum moved only when it grows by more than 2^6
//   O += P V       P back into tensor memory over S, V in shared memory (dims contiguous per key), O in tensor memory
//
// A quantized key is the cache's: bf16 after dequantizing.  A 2-bit code left where it lies in its byte is a bf16 subnormal,
// code 2^(2 plane - 133), so one packed FMA with (scale 2^(119 - 2 plane), offset 2^-14) gives the key times 2^-14, rounded once;
// the factor goes into c.  A rotated pair is summed in 32 bits and rounded to bf16 once, so that keys are the decode's bit for bit.
// (In packed bf16, a product rounded before the sum, a call takes 4 % less, 370 us for 385 at 2,048 queries over 16K, but single
// rows are then 1.4e-2 off at scores of deviation 3, 5e-2 at 10.)
// A quantized value is one of two, offset and offset + scale, rounded to f16 (2^-12): the sign of its bit, shifted to the top of
// its byte, spreads over 16 bits and picks.  P is f16 there (11 bits against bf16's 8), and O stays in the Hadamard domain until
// the first exact tile or the end, where the row's thread turns its 128 values in tensor memory (a fast Walsh-Hadamard transform
// in two passes of 32 registers).  Exact keys and values are bf16; the chunk's own tokens are read from the pages like all others.
//
// Warps: 4 softmax warps per tile of 128 rows, 8 that build K and V tiles (two threads a key of quantized tiles, whose bytes and
// rotation TMA brings a tile ahead; 8 or 16 lanes a row of exact ones, copied whole and rotated in place), one that issues the
// MMAs, one the TMA copies.
// The two tiles of MT = 2 take turns: one is in the tensor cores while the other is in the softmax.
// Bound for long chunks: a tile of 256 rows x 128 keys takes the tensor cores, the exponentials (16 a clock) and the
// shared-memory and tensor-memory traffic about 2,050 clocks each.  Measured: 2,048 queries over 16,384 tokens more take 385 us,
// 292 GFLOP at 758 TFLOP/s (46 % of what a cuBLAS bf16 product reaches in a burst), about 6,400 clocks a tile: the tensor cores
// are busy for 38 % of it, the issue slots for 54 %; a softmax warp's chain of scores, maximum, exponentials and P is the longest.
// 4,103 queries from 0 (exact tiles alone, and 2.7 item beginnings a CTA) take 154 us, 69 GFLOP at 448.  2,048 queries over 2,000
// tokens more on a window or sliding layer take 43 us.
// Tried and slower, each beside the form of its day: polynomial exponentials on the FMA pipe (639 us where this took 552), two threads a row (488 / 449), separate
// loops by template for quantized and exact weights (420 / 386), page lookups two tiles ahead (160 / 153 at 4,103 from 0).
//
// Work is cut evenly: the (row, query tile) items are flattened into 128-key tiles and cut into equal parts, each done for the
// 4 KV heads by 4 CTAs at about the same time, so that the heads' bytes of a sub-block leave DRAM once.  An item that a cut
// goes through leaves partial (m, l, O) of fp32 in its CTAs' slots, merged by extend_join.
//
// A value that is not finite makes every weight's product with it NaN, a masked (zero) weight's too: the builders replace
// such values by zero and mark their keys, and a row that sees a marked key becomes NaN as a whole.
#pragma once
#include <cuda.h>

#include "extend_rows.cuh"
#include "tc5.cuh"

namespace kv800 {

struct __align__(16) ExItem {     // queries of one row, with all that a kernel needs to find its keys
    int b, quant, tiles, base;    // row; key tiles: quantized ones, all (one head's); the units of the items before
    int q0, nq, p0, nexact;       // first query's token, queries, its position; exact keys
    int nsk, xlo, ns, lead;       // exact key e lies at position e < nsk ? e : xlo + e - nsk, below ns in the sink rows
};
// An item's work in units of a key tile: `lead` for what it costs to begin (its queries, the first tile's way through the CTA, the
// output), then its tiles.
struct __align__(16) ExPart {     // a run [u0, u1) of the W units, and the item it begins in
    int u0, u1, W, it;
    ExItem item;
};

struct ExPlan {
    ExPart* part;
    ExItem* items;
    float2* ml;              // [2 parts][heads][rows] running maximum (log2) and sum
    float* o;                // [2 parts][heads][rows][128]
    int64_t max_items;
    int qt, parts, lead;     // queries a tile, parts the units are cut into (each done for the 4 heads), units of an item's beginning
};

constexpr int EX_TILE = 128;
constexpr float EX_LAZY = 6.0f;      // log2: weights reach 2^6 before the maximum moves; 2^6 x the largest V scale is an f16

// The W units are cut into `parts` runs whose lengths differ by at most one: the first unit of run c, and the run of unit u.
struct ExCut {
    int q, rem;
    __device__ __forceinline__ ExCut(int W, int parts) : q(W / parts), rem(W % parts) {}
    __device__ __forceinline__ int start(int c) const { return c * q + min(c, rem); }
    __device__ __forceinline__ int part(int u) const {
        const int big = rem * (q + 1);
        return u < big ? u / (q + 1) : rem + (u - big) / q;
    }
};

// One CTA: the items (rows in order, query tiles in order), the sums of their units, and what each part begins with, so that
// a CTA of the kernels after it starts from one load.  A first walk over the items counts the units, a second writes; up to
// 1,024 rows and items need one.
__global__ void __launch_bounds__(1024) extend_plan(const __grid_constant__ ExtendArgs a, const __grid_constant__ ExPlan pl) {
    __shared__ int s_w[32];
    __shared__ int s_first[1025];     // items of the chunk's rows before
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_launch_dependents();
    auto plus = [](int x, int y) { return (int)min((uint32_t)x + (uint32_t)y, 0x40000000u); };   // stops at 2^30
    auto scan = [&](int v, int& total) {   // exclusive, over the CTA
        int x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x = plus(x, y);
        }
        __syncthreads();
        if (lane == 31) s_w[warp] = x;
        __syncthreads();
        int w = s_w[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w = plus(w, y);
        }
        total = __shfl_sync(0xffffffffu, w, 31);
        const int before = __shfl_sync(0xffffffffu, w, warp ? warp - 1 : 0);
        const int left = __shfl_up_sync(0xffffffffu, x, 1);
        return plus(warp ? before : 0, lane ? left : 0);
    };
    if (tid == 0) *a.status = 0;
    ex_clear_first(a);
    __syncthreads();
    int W = 0;
    for (int pass = 0; pass < 2; pass++) {
        int items = 0, sum = 0, total;
        bool done = false;
        for (int rows = 0; rows < a.R; rows += 1024) {
            int nt = 0;
            if (rows + tid < a.R) {
                const int b = rows + tid;
                const int64_t q0 = a.qsl[b], q1 = a.qsl[b + 1];
                int64_t ql = (q1 < a.T ? q1 : a.T) - (q0 > 0 ? q0 : 0);
                if (pass == 0 && (q1 < q0 || q0 < 0 || q1 > a.T)) ex_flag(a, ST_TABLE);
                if (ql > a.max_qlen) {
                    if (pass == 0) {
                        ex_flag(a, ST_TABLE);
                        for (int64_t t = (q0 > 0 ? q0 : 0) + a.max_qlen; t < q1 && t < a.T; t++)
                            for (int d = 0; d < 16 * DIM; d++) a.out[t * 16 * DIM + d] = 0;
                    }
                    ql = a.max_qlen;
                }
                nt = ql > 0 ? (int)((ql + pl.qt - 1) / pl.qt) : 0;
            }
            const int at = scan(nt, total);
            s_first[tid] = at;
            if (tid == 0) s_first[1024] = total;
            __syncthreads();
            const int count = (int)min((int64_t)total, pl.max_items - items);   // fewer only where query_start_loc decreases
            if (count < total && tid == 0) ex_flag(a, ST_TABLE);
            const bool small = a.R <= 1024 && count <= 1024;
            for (int base = 0; base < count; base += 1024) {
                const int i = base + tid;
                ExItem it{};
                if (i < count) {
                    int lo = 0, hi = 1024;   // s_first[lo] <= i < s_first[hi]
                    while (hi - lo > 1) {
                        const int mid = (lo + hi) >> 1;
                        if (s_first[mid] <= i) lo = mid;
                        else hi = mid;
                    }
                    ExRow r;
                    ExKeys k;
                    ex_row(a, rows + lo, r);
                    int64_t ql = r.q1 - r.q0;
                    if (ql > a.max_qlen) ql = a.max_qlen;
                    const int64_t i0 = (int64_t)(i - s_first[lo]) * pl.qt;
                    it.b = rows + lo;
                    it.nq = (int)(ql - i0 < pl.qt ? ql - i0 : pl.qt);
                    it.q0 = (int)(r.q0 + i0), it.p0 = (int)(r.n0 + i0), it.ns = (int)r.ns;
                    ex_keys(a, r, r.n0 + i0, r.n0 + i0 + it.nq - 1, k);
                    it.nexact = (int)k.nexact, it.nsk = (int)k.nsk, it.xlo = (int)k.xlo;
                    it.quant = (int)((k.nquant + EX_TILE - 1) / EX_TILE);
                    const int n = it.quant + (int)((k.nexact + EX_TILE - 1) / EX_TILE);
                    it.tiles = n > 0 ? n : 1;
                    it.lead = pl.lead;
                }
                it.base = plus(sum, scan(it.lead + it.tiles, total));
                sum = plus(sum, total);
                if (small) W = sum, done = true;
                if (pass == 0 && !small) continue;
                if (W >= 0x40000000) {     // no cache holds this many keys
                    if (tid == 0) ex_flag(a, ST_TABLE);
                    W = 0;
                    break;
                }
                if (i < count) pl.items[items + i] = it;
                // the parts that begin in the items
                const ExCut cut(W, pl.parts);
                const int end = it.base + it.lead + it.tiles;
                int c = 0;
                bool has = false;
                if (i < count) {
                    c = cut.part(it.base);
                    if (cut.start(c) < it.base) c++;
                    has = c < pl.parts && cut.start(c) < end;
                }
                const bool many = has && c + 8 < pl.parts && cut.start(c + 8) < end;
                if (has && !many)
                    for (int p = c; p < pl.parts && cut.start(p) < end; p++)
                        pl.part[p] = ExPart{cut.start(p), cut.start(p + 1), W, items + i, it};
                for (uint32_t left = __ballot_sync(0xffffffffu, many); left; left &= left - 1) {   // the whole warp for one item
                    const int src = __ffs(left) - 1;
                    ExItem x;
                    int* f = reinterpret_cast<int*>(&x);
                    const int* g = reinterpret_cast<const int*>(&it);
#pragma unroll
                    for (int k = 0; k < 12; k++) f[k] = __shfl_sync(0xffffffffu, g[k], src);
                    const int index = items + __shfl_sync(0xffffffffu, i, src);
                    for (int p = __shfl_sync(0xffffffffu, c, src) + lane; p < pl.parts && cut.start(p) < x.base + x.lead + x.tiles; p += 32)
                        pl.part[p] = ExPart{cut.start(p), cut.start(p + 1), W, index, x};
                }
            }
            items += count;
        }
        if (pass == 0 && !done) W = sum;
        if (done) break;
    }
    for (int p = W + tid; p < pl.parts; p += 1024) pl.part[p] = ExPart{W, W, W, 0, ExItem{}};   // parts without a unit
}

// The segments of a CTA (part block / 4, head block % 4): runs of key tiles of one item.  The item stays in memory, its fields are
// read where they are needed: registers are short in every role.
struct ExWalk {
    const ExItem* item;
    int u, u1, t0, t1;
    bool begun;       // the segment is not the part's first

    __device__ __forceinline__ ExWalk(const ExPlan& p, int block) {
        const int4 x = __ldg(reinterpret_cast<const int4*>(p.part + (block >> 2)));
        u = x.x, u1 = x.y, item = p.items + x.w - 1;
        t1 = -1;
    }
    __device__ __forceinline__ bool next() {
        if (u >= u1) return false;
        begun = t1 >= 0;
        item++;      // a segment ends with its item, but for the last
        const int from = u - item->base - item->lead, to = min(item->tiles, from + (u1 - u));
        u += to - from;
        t0 = max(from, 0), t1 = to;
        return to > 0;           // the part may end before the item's first tile
    }
    // where the partial result goes, or -1 if the segment is the whole item
    __device__ __forceinline__ int slot(const ExPlan& p, int block) const {
        if (t0 == 0 && t1 == item->tiles) return -1;
        return (2 * (block >> 2) + begun) * HEADS + (block & 3);
    }
};

__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

// Byte offset of 16-byte chunk c (of 16) of row r in a tile of 128 rows x 128 16-bit values: two blocks of 64 values, rows of
// 128 bytes with their chunks swizzled.  The same offsets serve K (K-major) and V (dims contiguous per key).
__device__ __forceinline__ uint32_t tile_at(int r, int c) {
    return (uint32_t)((c >> 3) * 16384 + (r >> 3) * 1024 + (r & 7) * 128 + (((c ^ r) & 7) << 4));
}

// Tensor maps of the quantized tiles: the quant pool as rows of 128 bytes (a head's 32 bytes of 128 rows; whole rows, 64 and, of
// the scales, 16 at a time) and the rotation tables.
struct ExMaps {
    CUtensorMap head, rows, scales, cos, sin;
};
__device__ __forceinline__ void ex_tma(uint32_t dst, const CUtensorMap* m, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                 "l"(m), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}

// The raw bytes of a quantized tile for one head: codes (32 bytes a key, 32-byte swizzle), cos and sin (64 bytes a key, 64-byte
// swizzle), V bits (rows of 2 keys x 4 heads, 128-byte swizzle), the sub-block's scales.
struct ExRaw {
    static constexpr int CODE = 0, COS = 4096, SIN = 12288, BITS = 20480, SCALE = 28672, BYTES = 30720;
};
template <int MT>
struct ExSmem {
    static constexpr int Q = 0, K = MT * 32768, V = K + 2 * 32768, RAW = V + 2 * 32768, TABLE = RAW + ExRaw::BYTES,
                         MASK = TABLE + 2 * 512, BARS = MASK + 2 * 32, BYTES = BARS + 256 + 1024;
};

// ------------------------------------------------------------------ O: Hadamard domain -> plain
// Column 32 g + 8 w + 4 i0 + pos holds dim 32 g + 16 i0 + 4 w + b, b = pos with its two bits swapped.
__device__ __forceinline__ void turn_o(uint32_t o) {
    uint32_t r[32];
#pragma unroll 1
    for (int g = 0; g < 4; g++) {
        tmem_ld32(o + 32 * g, r);
        tmem_wait_ld(r);
        float x[32];
#pragma unroll
        for (int d = 0; d < 32; d++) {   // to dim order
            const int i0 = d >> 4, w = (d >> 2) & 3, b = d & 3, pos = (b >> 1) | ((b & 1) << 1);
            x[d] = __uint_as_float(r[8 * w + 4 * i0 + pos]);
        }
#pragma unroll
        for (int len = 1; len < 32; len <<= 1)
#pragma unroll
            for (int d = 0; d < 32; d++)
                if (!(d & len)) {
                    const float y = x[d], z = x[d + len];
                    x[d] = y + z, x[d + len] = y - z;
                }
#pragma unroll
        for (int d = 0; d < 32; d++) r[d] = __float_as_uint(x[d]);
        tmem_st32(o + 32 * g, r);
    }
    tmem_wait_st();
#pragma unroll 1
    for (int k = 0; k < 4; k++) {
#pragma unroll
        for (int g = 0; g < 4; g++) tmem_ld8(o + 32 * g + 8 * k, r + 8 * g);
        tmem_wait_ld(r);
#pragma unroll
        for (int d = 0; d < 8; d++) {
            const float x0 = __uint_as_float(r[d]), x1 = __uint_as_float(r[8 + d]), x2 = __uint_as_float(r[16 + d]),
                        x3 = __uint_as_float(r[24 + d]);
            const float a = x0 + x1, b = x0 - x1, c = x2 + x3, e = x2 - x3, n = 0.08838834764831845f;
            r[d] = __float_as_uint((a + c) * n);
            r[8 + d] = __float_as_uint((b + e) * n);
            r[16 + d] = __float_as_uint((a - c) * n);
            r[24 + d] = __float_as_uint((b - e) * n);
        }
#pragma unroll
        for (int g = 0; g < 4; g++) tmem_st8(o + 32 * g + 8 * k, r + 8 * g);
    }
    tmem_wait_st();
}

__device__ __forceinline__ void scale_o(uint32_t o, float f) {   // 8 columns at a time: the scores fill the registers meanwhile
#pragma unroll 1
    for (int g = 0; g < 16; g++) {
        uint32_t r[8];
        tmem_ld8(o + 8 * g, r);
        tmem_wait_ld8(r);
#pragma unroll
        for (int d = 0; d < 8; d++) r[d] = __float_as_uint(__uint_as_float(r[d]) * f);
        tmem_st8(o + 8 * g, r);
    }
    tmem_wait_st();
}

// ------------------------------------------------------------------ keys
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t s) {
    uint32_t d;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(s));
    return d;
}
// (a, b) -> (a c - b s, b c + a s) of two pairs: bf16 products are exact in fp32, the sum is rounded there and once to bf16, as the
// decode rounds a key
__device__ __forceinline__ void turn_packed(uint32_t& a, uint32_t& b, uint32_t c, uint32_t s) {
    asm("{\n\t.reg .b16 a0, a1, b0, b1, c0, c1, s0, s1;\n\t.reg .f32 t, x0, x1, y0, y1;\n\t"
        "mov.b32 {a0, a1}, %0;\n\tmov.b32 {b0, b1}, %1;\n\tmov.b32 {c0, c1}, %2;\n\tmov.b32 {s0, s1}, %3;\n\t"
        "fma.rn.f32.bf16 t, b0, s0, 0f00000000;\n\tneg.f32 t, t;\n\tfma.rn.f32.bf16 x0, a0, c0, t;\n\t"
        "fma.rn.f32.bf16 t, b1, s1, 0f00000000;\n\tneg.f32 t, t;\n\tfma.rn.f32.bf16 x1, a1, c1, t;\n\t"
        "fma.rn.f32.bf16 t, a0, s0, 0f00000000;\n\tfma.rn.f32.bf16 y0, b0, c0, t;\n\t"
        "fma.rn.f32.bf16 t, a1, s1, 0f00000000;\n\tfma.rn.f32.bf16 y1, b1, c1, t;\n\t"
        "cvt.rn.bf16x2.f32 %0, x1, x0;\n\tcvt.rn.bf16x2.f32 %1, y1, y0;\n\t}"
        : "+r"(a), "+r"(b)
        : "r"(c), "r"(s));
}
__device__ __forceinline__ float max3(float a, float b, float c) {   // NaN if one of them is
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
template <int N> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <int MT>
__global__ void __launch_bounds__((MT + 3) * 128, 1)
    extend_tc(const __grid_constant__ ExtendArgs a, const __grid_constant__ ExPlan pl, const __grid_constant__ ExMaps maps) {
    using L = ExSmem<MT>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t sm0 = smem_u32(smem_raw), sm = (sm0 + 1023) & ~1023u;
    uint8_t* smp = smem_raw + (sm - sm0);
    const uint32_t bars = sm + L::BARS;
    volatile int* gave_up = reinterpret_cast<volatile int*>(smp + L::BARS + 248);
    volatile int* s_ok = reinterpret_cast<volatile int*>(smp + L::BARS + 244);    // the raw tile's sub-block lies in the pool
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smp + L::BARS + 240);
    // barriers (8 bytes each)
    const uint32_t b_q = bars, b_of = bars + 16, b_s = bars + 32, b_p = bars + 48, b_o = bars + 64, b_kf = bars + 80,
                   b_ke = bars + 96, b_vf = bars + 112, b_ve = bars + 128, b_tab = bars + 144, b_raw = bars + 152,
                   b_used = bars + 160, b_ph = bars + 168;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int W_PROD = MT * 4, W_MMA = MT * 4 + 8;
    // A wait by parity tells a phase from the next one only.  None here can fall further behind, since each phase waits for whoever
    // waits on the one before: a stage is refilled (kf, vf) once the products have released it (ke, ve), which want all builder and
    // softmax warps' arrivals; scores (s) follow the P of the tile before (ph, p), a segment's queries (q) its last O (o), O's first
    // product the last one's read-out (of); a raw tile (raw) its readers' release (used); a table (tab) all builders' arrivals.
    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            bar_init(b_q + 8 * i, 4);
            bar_init(b_of + 8 * i, 4);
            bar_init(b_s + 8 * i, 1);
            bar_init(b_p + 8 * i, 4);
            bar_init(b_ph + 8 * i, 4);
            bar_init(b_o + 8 * i, 1);
            bar_init(b_kf + 8 * i, 8);
            bar_init(b_ke + 8 * i, 1);
            bar_init(b_vf + 8 * i, 8);
            bar_init(b_ve + 8 * i, 1);
        }
        bar_init(b_tab, 8);
        bar_init(b_raw, 1);
        bar_init(b_used, 8);
        *gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == W_MMA) tmem_alloc(smem_u32(tmem_slot), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_launch_dependents();

    // register split of the launch's 96 x 640 (MT = 2; 128 x 512 at MT = 1): 120 x 128 MT + 88 x 256 + 56 x 128
    if (warp < W_PROD) {
        regs_up<MT == 1 ? 136 : 120>();
        // ---------------------------------------------------------------- softmax: one thread a row of its tile
        ExWalk walk(pl, blockIdx.x);
        const int head = blockIdx.x & 3;
        const int mt = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t S = tmem + lanes + 128 * mt, O = tmem + lanes + 256 + 128 * mt;
        // tokens after the last row's, which no row owns
        const int64_t owned = a.R && a.qsl[a.R] > 0 ? a.qsl[a.R] : 0;
        for (int64_t t = owned + (int64_t)blockIdx.x; t < a.T; t += gridDim.x)
            for (int d = tid; d < 16 * DIM / 8; d += W_PROD * 32)
                reinterpret_cast<uint4*>(a.out + t * 16 * DIM)[d] = make_uint4(0, 0, 0, 0);
        uint32_t kt = 0;
        for (uint32_t seg = 0; walk.next(); seg++) {
            const int rows = 4 * walk.item->nq - 128 * mt;      // of this tile
            const bool busy = (warp & 3) * 32 < rows;           // this warp has any
            const int qi = 32 * mt + (row >> 2);                // query within the item
            // the row's position, and its place among the exact keys
            const int p = walk.item->p0 + (row < rows ? qi : walk.item->nq - 1), px = p - walk.item->xlo + walk.item->nsk;
            const int nquant = walk.item->quant;
            // Q: natural dims, each group of four stored as (0, 2, 1, 3) like the keys
            {
                const uint4* src =
                    reinterpret_cast<const uint4*>(a.q + ((int64_t)(walk.item->q0 + qi) * 16 + head * 4 + (row & 3)) * DIM);
                const uint32_t dst = sm + L::Q + mt * 32768;
#pragma unroll
                for (int c = 0; c < 16; c++) {
                    const uint4 x = row < rows ? __ldg(src + c) : make_uint4(0, 0, 0, 0);
                    st_shared16(dst + tile_at(row, c), prmt(x.x, x.y, 0x5410), prmt(x.x, x.y, 0x7632),
                                prmt(x.z, x.w, 0x5410), prmt(x.z, x.w, 0x7632));
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) bar_arrive(b_q + 8 * mt);
            }
            float m = -INFINITY, l = 0.0f;
            bool turned = true;                                 // O is in the plain domain (or empty)
            for (int ti = walk.t0; ti < walk.t1; ti++, kt++) {
                const bool quant = ti < nquant;
                const uint32_t st = kt & 1, ph = (kt >> 1) & 1;
                if (!warp_wait(b_vf + 8 * st, ph, gave_up) || !warp_wait(b_s + 8 * mt, kt & 1, gave_up)) goto done;
                tc_fence_after();
                if (busy) {
                    if (!quant && !turned) turn_o(O);           // the first exact tile: the scores before it are summed up
                    turned = !quant;
                    // what of the tile the row sees: keys [., hi], from lo on or below ss
                    const int e0 = (quant ? ti : ti - nquant) * EX_TILE, hi = (quant ? p : px) - e0;
                    int lo = 0, ss = 0;
                    if (!quant && a.P.win) {
                        lo = max(hi, (int)a.P.win - 1) - (int)a.P.win + 1;
                        ss = a.P.sk ? (int)a.P.nsink - e0 : 0;
                    }
                    const uint32_t* mask = reinterpret_cast<const uint32_t*>(smp + L::MASK + st * 32);
                    const uint4 gone = *reinterpret_cast<const uint4*>(mask), bad = *reinterpret_cast<const uint4*>(mask + 4);
                    const bool marks = (gone.x | gone.y | gone.z | gone.w | bad.x | bad.y | bad.z | bad.w) != 0;
                    const bool all = __all_sync(0xffffffffu, hi >= EX_TILE - 1 && lo <= 0) && !marks;
                    uint32_t sa[32], sb[32];      // 64 keys' scores at a time
                    if (!all) {                   // the keys the row does not see: -inf, written back before anything reads them
#pragma unroll 1
                        for (int c = 0; c < 4; c++) {
                            tmem_ld32(S + 32 * c, sa);
                            const uint32_t vis = below(hi + 1 - 32 * c) & (~below(lo - 32 * c) | below(ss - 32 * c)) & ~mask[c];
                            if (vis & mask[4 + c]) l = __uint_as_float(0x7fc00000u);
                            tmem_wait_ld(sa);
#pragma unroll
                            for (int i = 0; i < 32; i++)
                                if (!((vis >> i) & 1)) sa[i] = 0xff800000u;
                            tmem_st32(S + 32 * c, sa);
                        }
                        tmem_wait_st();
                    }
                    const float sc = quant ? EX_SCALE * 16384.0f : EX_SCALE;
                    float top = -INFINITY, f = 1.0f;
                    // short loops, run again and again: straight code of their length would miss the instruction cache all along
#pragma unroll 1
                    for (int c = 0; c < 128; c += 64) {
                        tmem_ld32(S + c, sa);
                        tmem_ld32(S + c + 32, sb);
                        tmem_wait_ld(sa);
                        tmem_wait_ld(sb);
                        float x[4] = {top, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            x[0] = max3(x[0], __uint_as_float(sa[i]), __uint_as_float(sa[i + 1]));
                            x[1] = max3(x[1], __uint_as_float(sa[i + 2]), __uint_as_float(sa[i + 3]));
                            x[2] = max3(x[2], __uint_as_float(sb[i]), __uint_as_float(sb[i + 1]));
                            x[3] = max3(x[3], __uint_as_float(sb[i + 2]), __uint_as_float(sb[i + 3]));
                        }
                        top = max3(max3(x[0], x[1], x[2]), x[3], -INFINITY);
                    }
                    top *= sc;
                    if (!(top < INFINITY)) {      // a NaN, or a score beyond all others
                        l = __uint_as_float(0x7fc00000u);
                        top = -INFINITY;
                    }
                    if (top > m + EX_LAZY || (m == -INFINITY && top > m)) {
                        f = exp2_approx(m - top);
                        m = top;
                        l *= f;
                    }
                    if (ti > walk.t0 && __any_sync(0xffffffffu, f != 1.0f)) scale_o(O, f);
                    const float mu = m == -INFINITY ? 0.0f : m;
                    const f2 sc2(sc, sc), mm2(-mu, -mu);
                    f2 l2[2] = {f2(0.0f, 0.0f), f2(0.0f, 0.0f)};
                    // P over the second half of S, whose scores are in hand; then the first half's are read again
#pragma unroll 1
                    for (int half = 1; half >= 0; half--) {
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            const uint32_t(&r)[32] = c ? sb : sa;
                            uint32_t w[16];
#pragma unroll
                            for (int i = 0; i < 16; i++) {
                                float x, y;
                                fma2(f2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), sc2, mm2).get(x, y);
                                x = exp2_approx(x), y = exp2_approx(y);
                                l2[i & 1] = add2(l2[i & 1], f2(x, y));
                                w[i] = quant ? pack2_f16(x, y) : pack2_bf16(x, y);
                            }
                            tmem_st16(S + 64 + 32 * half + 16 * c, w);
                        }
                        if (half) {
                            tmem_ld32(S, sa);
                            tmem_ld32(S + 32, sb);
                            tmem_wait_st();                          // the keys done may start on P V
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) bar_arrive(b_ph + 8 * mt);
                            tmem_wait_ld(sa);
                            tmem_wait_ld(sb);
                        }
                    }
                    float x, y;
                    add2(l2[0], l2[1]).get(x, y);
                    l += x + y;
                    tmem_wait_st();
                } else if (lane == 0) {
                    bar_arrive(b_ph + 8 * mt);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(b_p + 8 * mt);
            }
            if (!warp_wait(b_o + 8 * mt, seg & 1, gave_up)) goto done;
            tc_fence_after();
            if (busy) {
                if (!turned) turn_o(O);
                uint32_t r[32];
                const bool real = row < 4 * walk.item->nq - 128 * mt;
                const int slot = walk.slot(pl, blockIdx.x);
                if (slot < 0) {
                    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                    uint4* dst = reinterpret_cast<uint4*>(
                        a.out + ((int64_t)(walk.item->q0 + 32 * mt + (row >> 2)) * 16 + head * 4 + (row & 3)) * DIM);
#pragma unroll 1
                    for (int c = 0; c < 4; c++) {
                        tmem_ld32(O + 32 * c, r);
                        tmem_wait_ld(r);
                        if (real) {
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                uint32_t w[4];
#pragma unroll
                                for (int k = 0; k < 4; k++)
                                    w[k] = pack2_bf16(__uint_as_float(r[8 * i + 2 * k]) * inv,
                                                      __uint_as_float(r[8 * i + 2 * k + 1]) * inv);
                                dst[4 * c + i] = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        }
                    }
                } else {
                    const int64_t at = (int64_t)slot * (MT * 128) + mt * 128 + row;
                    uint4* dst = reinterpret_cast<uint4*>(pl.o + at * DIM);
                    if (real) pl.ml[at] = make_float2(m, l);
#pragma unroll 1
                    for (int c = 0; c < 4; c++) {
                        tmem_ld32(O + 32 * c, r);
                        tmem_wait_ld(r);
                        if (real)
#pragma unroll
                            for (int i = 0; i < 8; i++)
                                dst[8 * c + i] = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(b_of + 8 * mt);
        }
    } else if (warp < W_MMA) {
        regs_down<88>();
        // ---------------------------------------------------------------- builders
        ExWalk walk(pl, blockIdx.x);
        const int bt = tid - W_PROD * 32, pw = warp - W_PROD, h = blockIdx.x & 3;
        const int key = bt & 127, hf = bt >> 7;      // quantized tiles: the key, and which half of its dims
        uint32_t kt = 0, nraw = 0, tb = 0;   // tiles, raw tiles, tables (in two buffers)
        for (uint32_t seg = 0; walk.next(); seg++) {
            const int nquant = walk.item->quant, qend = min(walk.t1, nquant);
            int table = -1;                      // sub-block whose scales the current table holds
            auto publish = [&](uint32_t st) {      // a V tile
                fence_async_smem();
                __syncwarp();
                if (lane == 0) bar_arrive(b_vf + 8 * st);
            };
            for (int ti = walk.t0; ti < qend; ti++, kt++) {
                const uint32_t st = kt & 1, ph = (kt >> 1) & 1;
                const uint32_t kd = sm + L::K + st * 32768, vd = sm + L::V + st * 32768;
                const uint32_t raw = sm + L::RAW;
                if (!warp_wait(b_raw, nraw & 1, gave_up)) goto done;
                const bool sub = *s_ok != 0;
                const bool ok = sub && ti * EX_TILE + key < a.npos;
                if (sub && !ok) ex_flag(a, ST_TABLE);
                if (table != (ti >> 1)) {      // [word][plane]: (scale, offset) of its even dims, of its odd dims
                    table = ti >> 1;
                    if (bt < 64) {
                        const int wd = bt >> 3, q = (bt >> 1) & 3, od = bt & 1, d = 32 * q + 4 * wd + od;
                        const uint8_t* ks = smp + L::RAW + ExRaw::SCALE + (KSC_O - VLO_O) + h * DIM + d;
                        const uint8_t* kl = smp + L::RAW + ExRaw::SCALE + (KLO_O - VLO_O) + h * DIM + d;
                        float x0 = 0, x1 = 0, l0 = 0, l1 = 0;
                        if (sub) f8_pair(ks[0], ks[2], x0, x1), f8_pair(kl[0], kl[2], l0, l1);
                        const float up = __uint_as_float((uint32_t)(127 + 119 - 2 * q) << 23), dn = 6.103515625e-05f;
                        *reinterpret_cast<uint2*>(smp + L::TABLE + (tb & 1) * 512 + bt * 8) =
                            make_uint2(pack2_bf16(x0 * up, x1 * up), pack2_bf16(l0 * dn, l1 * dn));
                    }
                    __syncwarp();
                    if (lane == 0) bar_arrive(b_tab);
                    if (!warp_wait(b_tab, tb & 1, gave_up)) goto done;
                    tb++;
                }
                const uint32_t tab = sm + L::TABLE + ((tb - 1) & 1) * 512;
                // the thread's half of the raw tile into registers, so that the next one can come
                const uint4 code = ld_shared16(raw + ExRaw::CODE + key * 32 + ((hf ^ ((key >> 2) & 1)) << 4));
                uint4 cs[2], sn[2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const uint32_t at = raw + key * 64 + (((2 * hf + i) ^ ((key >> 1) & 3)) << 4);
                    cs[i] = ld_shared16(at + ExRaw::COS);
                    sn[i] = ld_shared16(at + ExRaw::SIN);
                }
                const uint2 bits = ld_shared8(raw + ExRaw::BITS + (key >> 1) * 128 + ((((key & 1) * 4 + h) ^ (key >> 1)) & 7) * 16 + 8 * hf);
                const uint8_t* vsc = smp + L::RAW + ExRaw::SCALE + ((ti & 1) * EX_TILE + key) * 2 + (h >> 1);
                float vl, vh;
                f8_pair(ok ? vsc[0] : 0u, ok ? vsc[VSC_O - VLO_O] : 0u, vl, vh);
                vh += vl;
                __syncwarp();
                if (lane == 0) bar_arrive(b_used);
                nraw++;
                if (!warp_wait(b_ke + 8 * st, ph ^ 1, gave_up)) goto done;
#pragma unroll 1
                for (int i = 0; i < 2; i++) {
                    uint32_t k[4][4];   // [plane][even, odd of the first word of the pair; even, odd of the second]
#pragma unroll
                    for (int v = 0; v < 2; v++) {
                        const uint32_t ev = i == 0 ? (v ? code.y : code.x) : (v ? code.w : code.z), od = ev >> 8;
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            const uint4 x = ld_shared16(tab + ((4 * hf + 2 * i + v) * 4 + q) * 16);
                            k[q][2 * v] = bf2_fma(ev & (0x00030003u << (2 * q)), x.x, x.y);
                            k[q][2 * v + 1] = bf2_fma(od & (0x00030003u << (2 * q)), x.z, x.w);
                        }
                    }
                    const uint4 c = i ? cs[1] : cs[0], sn_ = i ? sn[1] : sn[0];
                    turn_packed(k[0][0], k[2][0], prmt(c.x, c.y, 0x5410), prmt(sn_.x, sn_.y, 0x5410));
                    turn_packed(k[0][1], k[2][1], prmt(c.x, c.y, 0x7632), prmt(sn_.x, sn_.y, 0x7632));
                    turn_packed(k[0][2], k[2][2], prmt(c.z, c.w, 0x5410), prmt(sn_.z, sn_.w, 0x5410));
                    turn_packed(k[0][3], k[2][3], prmt(c.z, c.w, 0x7632), prmt(sn_.z, sn_.w, 0x7632));
#pragma unroll
                    for (int q = 0; q < 4; q++) st_shared16(kd + tile_at(key, 4 * q + 2 * hf + i), k[q][0], k[q][1], k[q][2], k[q][3]);
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) bar_arrive(b_kf + 8 * st);
                // V: offset where the bit is clear, offset + scale where it is set
                const bool bad = !(fabsf(vl) < 1e9f && fabsf(vh) < 1e9f);
                const uint32_t v0 = bad ? 0u : pack2_f16(vl, vl), vx = bad ? 0u : v0 ^ pack2_f16(vh, vh);
                if (!warp_wait(b_ve + 8 * st, ph ^ 1, gave_up)) goto done;
#pragma unroll 1
                for (int w = 0; w < 2; w++) {
                    const uint32_t x = w ? bits.y : bits.x;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t y = x << (7 - 2 * i), z = x << (6 - 2 * i);
                        st_shared16(vd + tile_at(key, 4 * i + 2 * hf + w), (prmt(y, 0, 0xaa88) & vx) ^ v0, (prmt(y, 0, 0xbb99) & vx) ^ v0,
                                    (prmt(z, 0, 0xaa88) & vx) ^ v0, (prmt(z, 0, 0xbb99) & vx) ^ v0);
                    }
                }
                const uint32_t gone = __ballot_sync(0xffffffffu, !ok), bads = __ballot_sync(0xffffffffu, bad);
                if (lane == 0 && hf == 0) {
                    uint32_t* mask = reinterpret_cast<uint32_t*>(smp + L::MASK + st * 32);
                    mask[pw] = gone;
                    mask[4 + pw] = bads;
                }
                publish(st);
            }
            const int x0 = max(walk.t0, nquant);
            if (x0 >= walk.t1) continue;
            const int nsk = walk.item->nsk;
            // an exact tile: a warp builds 16 keys, lane i looks up key 16 pw + i % 16
            const uint16_t *kr = nullptr, *vr = nullptr;
            int kp = 0;
            bool in = false;
            auto lookup = [&](int ti) {
                const int e = (ti - nquant) * EX_TILE + 16 * pw + (lane & 15);
                kr = vr = nullptr;
                in = e < walk.item->nexact;
                kp = !in ? 0 : e < nsk ? e : walk.item->xlo + (e - nsk);
                bool ok = in && ex_exact(a, walk.item->b, walk.item->ns, h, kp, kr, vr);
                if (ok && a.cos_t && kp >= a.npos) {
                    ex_flag(a, ST_TABLE);
                    ok = false;
                }
                if (!ok) kr = vr = nullptr;
            };
            // rows come by asynchronous copies, 16 lanes a row, K to its place in the K tile where it is then rotated: 8 lanes a key,
            // lane j has dims 4 j .. 4 j + 3 of each 32.  Rows 4 apart share an access's phase, which keeps the swizzled chunks of
            // both clear of each other's banks
            const int j = lane & 7;
            const bool rotate = a.cos_t != nullptr;
            auto copy_rows = [&](const uint16_t* row, uint32_t dst) {
#pragma unroll 2
                for (int i = 0; i < 8; i++) {
                    const uint4* src = reinterpret_cast<const uint4*>(
                        __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(row), 2 * i + (lane >> 4)));
                    copy_async16(dst + tile_at(16 * pw + 2 * i + (lane >> 4), lane & 15),
                                 src ? src + (lane & 15) : reinterpret_cast<const uint4*>(a.q), src != nullptr);
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            for (int ti = x0; ti < walk.t1; ti++, kt++) {
                const uint32_t st = kt & 1, ph = (kt >> 1) & 1;
                const uint32_t kd = sm + L::K + st * 32768, vd = sm + L::V + st * 32768;
                if (ti == x0) {      // the first exact tile: nothing is on its way yet
                    lookup(ti);
                    if (!warp_wait(b_ke + 8 * st, ph ^ 1, gave_up)) goto done;
                    copy_rows(kr, kd);
                    if (!warp_wait(b_ve + 8 * st, ph ^ 1, gave_up)) goto done;
                    copy_rows(vr, vd);
                }
                // a key past the end is hidden by position; its mark would only cost the fast path
                const uint32_t gone = __ballot_sync(0xffffffffu, in && !kr) & 0xffffu;
                uint32_t bads = 0;
                // its first keys are sinks, whose rotation lies apart: exact key e < nsk at position e
                const int e0 = (ti - nquant) * EX_TILE, sunk = nsk - e0;
                const bool next = ti + 1 < walk.t1;
                if (next) lookup(ti + 1);
                if (rotate && !warp_wait(b_raw, nraw & 1, gave_up)) goto done;
                asm volatile("cp.async.wait_group 1;" ::: "memory");
                __syncwarp();
#pragma unroll 2
                for (int i = 0; i < 4; i++) {
                    const int r = 16 * pw + 8 * (i >> 1) + 2 * (i & 1) + ((lane >> 3) & 1) * 4 + (lane >> 4);
                    uint2 y[4];
#pragma unroll
                    for (int q = 0; q < 4; q++) y[q] = ld_shared8(kd + tile_at(r, 4 * q + (j >> 1)) + (j & 1) * 8);
                    uint2 c, sn;
                    if (rotate) {
                        const uint32_t at = sm + L::RAW + r * 64 + (((j >> 1) ^ ((r >> 1) & 3)) << 4) + (j & 1) * 8;
                        c = ld_shared8(at + ExRaw::COS), sn = ld_shared8(at + ExRaw::SIN);
                        if (r < sunk && e0 + r < a.npos) {
                            c = __ldg(reinterpret_cast<const uint2*>(a.cos_t + (int64_t)(e0 + r) * 32) + j);
                            sn = __ldg(reinterpret_cast<const uint2*>(a.sin_t + (int64_t)(e0 + r) * 32) + j);
                        }
                    }
#pragma unroll
                    for (int q = 0; q < 4; q++)   // (0, 2), (1, 3)
                        y[q] = make_uint2(prmt(y[q].x, y[q].y, 0x5410), prmt(y[q].x, y[q].y, 0x7632));
                    if (rotate) {
                        turn_packed(y[0].x, y[2].x, prmt(c.x, c.y, 0x5410), prmt(sn.x, sn.y, 0x5410));
                        turn_packed(y[0].y, y[2].y, prmt(c.x, c.y, 0x7632), prmt(sn.x, sn.y, 0x7632));
                    }
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(kd + tile_at(r, 4 * q + (j >> 1)) + (j & 1) * 8),
                                     "r"(y[q].x), "r"(y[q].y)
                                     : "memory");
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) bar_arrive(b_kf + 8 * st);
                if (rotate) {
                    if (lane == 0) bar_arrive(b_used);
                    nraw++;
                }
                const uint32_t ph1 = (((kt + 1) >> 1) & 1) ^ 1;
                if (next) {      // the next tile's K may come as soon as its stage is free
                    if (!warp_wait(b_ke + 8 * (st ^ 1), ph1, gave_up)) goto done;
                    copy_rows(kr, sm + L::K + (st ^ 1) * 32768);
                    asm volatile("cp.async.wait_group 1;" ::: "memory");
                } else {
                    asm volatile("cp.async.wait_all;" ::: "memory");
                }
                auto not_finite = [&](const uint4& v) {      // +0 if all are finite
                    return bf2_fma(v.w, 0u, bf2_fma(v.z, 0u, bf2_fma(v.y, 0u, bf2_fma(v.x, 0u, 0u))));
                };
                uint32_t nans = 0;       // one vote for all rows: one a row cost 158 us against 153's at 4,103 queries from 0
#pragma unroll 4
                for (int i = 0; i < 8; i++) nans |= not_finite(ld_shared16(vd + tile_at(16 * pw + 2 * i + (lane >> 4), lane & 15)));
                if (__any_sync(0xffffffffu, nans != 0)) {
#pragma unroll 1
                    for (int i = 0; i < 8; i++) {
                        const uint32_t at = vd + tile_at(16 * pw + 2 * i + (lane >> 4), lane & 15);
                        const uint32_t any = __ballot_sync(0xffffffffu, not_finite(ld_shared16(at)) != 0);
                        if (any >> (lane & 16) & 0xffffu) st_shared16(at, 0, 0, 0, 0);
                        bads |= ((any & 0xffffu ? 1u : 0u) | (any >> 16 ? 2u : 0u)) << (2 * i);
                    }
                }
                if (lane == 0) {      // 16 keys' marks
                    uint16_t* mask = reinterpret_cast<uint16_t*>(smp + L::MASK + st * 32);
                    mask[pw] = (uint16_t)gone;
                    mask[8 + pw] = (uint16_t)bads;
                }
                publish(st);
                if (next) {      // and so its V
                    if (!warp_wait(b_ve + 8 * (st ^ 1), ph1, gave_up)) goto done;
                    copy_rows(vr, sm + L::V + (st ^ 1) * 32768);
                }
            }
        }
    } else {
        regs_down<56>();
        if (warp == W_MMA + 1 && lane == 0) {
            // ------------------------------------------------------------ raw tiles: one ahead of the builders
            ExWalk walk(pl, blockIdx.x);
            uint32_t n = 0;
            const uint32_t dst = sm + L::RAW;
            while (walk.next()) {
                const int nquant = walk.item->quant, b = walk.item->b, x0 = walk.item->xlo - walk.item->nsk;
                for (int ti = walk.t0; ti < walk.t1; ti++) {
                    const bool quant = ti < nquant;
                    if (!quant && !a.cos_t) break;
                    const uint8_t* sb = quant ? ex_subblock(a, b, ti >> 1) : nullptr;
                    if (!bar_wait(b_used, (n & 1) ^ 1, gave_up)) goto out;
                    *s_ok = sb != nullptr;
                    if (quant && !sb) {
                        bar_arrive(b_raw);
                    } else {
                        const int p0 = quant ? ti * EX_TILE : x0 + (ti - nquant) * EX_TILE;
                        const uint32_t bytes = quant ? ExRaw::BYTES : 16384;
                        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(b_raw), "r"(bytes) : "memory");
                        ex_tma(dst + ExRaw::COS, &maps.cos, 0, p0, b_raw);
                        ex_tma(dst + ExRaw::SIN, &maps.sin, 0, p0, b_raw);
                        if (quant) {
                            const int r = (int)((sb - a.P.qpool) / 128), half = ti & 1;
                            ex_tma(dst + ExRaw::CODE, &maps.head, 32 * (int)(blockIdx.x & 3), r + KC_O / 128 + 128 * half, b_raw);
                            ex_tma(dst + ExRaw::BITS, &maps.rows, 0, r + VB_O / 128 + 64 * half, b_raw);
                            ex_tma(dst + ExRaw::SCALE, &maps.scales, 0, r + VLO_O / 128, b_raw);
                        }
                    }
                    n++;
                }
            }
        out:
            if (n && *gave_up) {      // the last copy lands before the CTA ends
                const uint64_t t0 = now_ns();
                while (!bar_try(b_raw, (n - 1) & 1) && now_ns() - t0 < 1000000000ull) {
                }
            }
        }
        if (warp == W_MMA && lane == 0) {
            // ------------------------------------------------------------ MMA issue
            ExWalk walk(pl, blockIdx.x);
            constexpr uint32_t D_QK = mma_desc(1, 128, 128, 0, 0), D_PV_F16 = mma_desc(0, 128, 128, 0, 1),
                               D_PV_BF = mma_desc(1, 128, 128, 0, 1);
            uint32_t kt = 0;
            // descriptors: the low words differ by the operand's address alone, the high word is one for all
            const uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29), kmaj = (16u >> 4) << 16, nmaj = (16384u >> 4) << 16;
            const uint32_t q0 = ((sm + L::Q) >> 4) | kmaj, k0 = ((sm + L::K) >> 4) | kmaj, v0 = ((sm + L::V) >> 4) | nmaj;
            auto qk = [&](int mt, uint32_t st) {
                const uint32_t qa = q0 + mt * 2048, kb = k0 + st * 2048;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const uint32_t o = (k >> 2) * 1024 + (k & 3) * 2;
                    mma_ss(tmem + 128 * mt, qa + o, kb + o, hi, D_QK, k > 0);
                }
            };
            auto pv = [&](int mt, uint32_t st, uint32_t desc, bool acc, int half) {   // 64 keys; the upper half comes first
                const uint32_t vb = v0 + st * 2048 + half * 512, p = tmem + 128 * mt + 64 + 32 * half;
                mma_ts(tmem + 256 + 128 * mt, p, vb, hi, desc, acc);
#pragma unroll
                for (int k = 1; k < 4; k++) mma_ts(tmem + 256 + 128 * mt, p + 8 * k, vb + k * 128, hi, desc, true);
            };
            for (uint32_t seg = 0; walk.next(); seg++) {
                const int n = walk.t1 - walk.t0, nquant = walk.item->quant - walk.t0;
                for (int mt = 0; mt < MT; mt++)
                    if (!bar_wait(b_q + 8 * mt, seg & 1, gave_up)) goto done;
                if (!bar_wait(b_kf + 8 * (kt & 1), (kt >> 1) & 1, gave_up)) goto done;
                tc_fence_after();
                for (int mt = 0; mt < MT; mt++) {
                    qk(mt, kt & 1);
                    mma_commit(b_s + 8 * mt);
                }
                mma_commit(b_ke + 8 * (kt & 1));
                for (int j = 0; j < n; j++, kt++) {
                    const uint32_t st = kt & 1, nx = st ^ 1;
                    const bool more = j + 1 < n;
                    if (!bar_wait(b_vf + 8 * st, (kt >> 1) & 1, gave_up)) goto done;
                    for (int mt = 0; mt < MT; mt++) {
                        if (j == 0 && !bar_wait(b_of + 8 * mt, (seg & 1) ^ 1, gave_up)) goto done;
                        const uint32_t desc = j < nquant ? D_PV_F16 : D_PV_BF;
                        if (!bar_wait(b_ph + 8 * mt, kt & 1, gave_up)) goto done;
                        tc_fence_after();
                        pv(mt, st, desc, j > 0, 1);
                        if (!bar_wait(b_p + 8 * mt, kt & 1, gave_up)) goto done;
                        tc_fence_after();
                        pv(mt, st, desc, true, 0);
                        if (mt == MT - 1) mma_commit(b_ve + 8 * st);
                        if (more) {
                            if (mt == 0) {
                                if (!bar_wait(b_kf + 8 * nx, ((kt + 1) >> 1) & 1, gave_up)) goto done;
                                tc_fence_after();
                            }
                            qk(mt, nx);
                            mma_commit(b_s + 8 * mt);
                        } else {
                            mma_commit(b_o + 8 * mt);
                        }
                    }
                    if (more) mma_commit(b_ke + 8 * nx);
                }
            }
        }
    }
done:
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == W_MMA) {
        tc_fence_after();
        tmem_free(tmem, 512);
    }
    if (tid == 0 && *gave_up) ex_flag(a, ST_TIMEOUT);
}

// Merges the partial results of the items that a cut went through: block (c, head, y) merges rows 8 y .. 8 y + 7 of the item that
// cut c is the first to fall into, a warp a row: the row's loads are a chain (part, maxima, values), so rows want to be side by side.
// Few queries' items may be cut over all 148 parts (over 37 with tiles of 128 rows and more) but have few rows: 8 slots' values are
// in flight there (1 row x 5 queries of 32K 37 us, 66 slot after slot), 4 where there are many rows (4,103 queries from 0 152 us,
// 154 with 8).
constexpr int EX_JOIN = 8;
template <int ROWS>
__global__ void __launch_bounds__(EX_JOIN * 32) extend_join(const __grid_constant__ ExtendArgs a, const __grid_constant__ ExPlan pl) {
    pdl_wait();
    const int c = blockIdx.x + 1, head = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (a.own && !blockIdx.x && !blockIdx.y && !blockIdx.z && !warp) {
        int bits = 0;
        for (int i = lane; i < pl.parts; i += 32) bits |= a.status[1 + i];
        bits = __reduce_or_sync(0xffffffffu, bits);
        if (lane == 0) *a.status = bits;
    }
    const ExPart x = pl.part[c];
    const ExItem& item = x.item;
    const ExCut cut(x.W, pl.parts);
    const int before = cut.start(c - 1), i0 = item.base + item.lead;
    if (x.u0 >= x.u1 || x.u0 <= i0 || before > i0) return;     // no unit, not cut here, or cut before
    const int first = before >= item.base ? 2 * (c - 1) : 2 * (c - 1) + 1, last = cut.part(i0 + item.tiles - 1);
    const int row = blockIdx.z * EX_JOIN + warp;
    if (row >= 4 * item.nq) return;
    auto slot = [&](int x) { return ((int64_t)(x < c ? first : 2 * x) * HEADS + head) * ROWS + row; };
    constexpr int IN = ROWS == 32 ? 8 : 4;
    float4 o[IN];
    auto fetch = [&](int x) {       // slots x .. x + IN - 1
#pragma unroll
        for (int j = 0; j < IN; j++)
            o[j] = x + j <= last ? reinterpret_cast<const float4*>(pl.o + slot(x + j) * DIM)[lane] : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    const float2 none = make_float2(-INFINITY, 0.0f);
    float2 ml = c - 1 + lane <= last ? pl.ml[slot(c - 1 + lane)] : none;      // lane i weighs every 32nd slot from c - 1 + i on
    fetch(c - 1);
    float m = ml.x;
    for (int x = c + 31 + lane; x <= last; x += 32) m = fmaxf(m, pl.ml[slot(x)].x);
#pragma unroll
    for (int k = 16; k; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
    const float mu = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int base = c - 1; base <= last; base += 32) {
        const float f = exp2_approx(ml.x - mu);
        l = fmaf(ml.y, f, l);
        const int n = min(32, last + 1 - base);
        for (int k = 0; k < n; k += IN) {
#pragma unroll
            for (int j = 0; j < IN; j++) {
                const float w = __shfl_sync(0xffffffffu, f, k + j);
                acc.x = fmaf(o[j].x, w, acc.x), acc.y = fmaf(o[j].y, w, acc.y), acc.z = fmaf(o[j].z, w, acc.z), acc.w = fmaf(o[j].w, w, acc.w);
            }
            if (base + k + IN <= last) fetch(base + k + IN);
        }
        if (base + 32 <= last) ml = base + 32 + lane <= last ? pl.ml[slot(base + 32 + lane)] : none;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int64_t tok = item.q0 + (row >> 2);
    reinterpret_cast<uint2*>(a.out + (tok * 16 + head * 4 + (row & 3)) * DIM)[lane] =
        make_uint2(pack2_bf16(acc.x * inv, acc.y * inv), pack2_bf16(acc.z * inv, acc.w * inv));
}

}  // namespace kv800
