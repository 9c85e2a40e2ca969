// The steps around a chunked or speculative attention step, in one launch or two and without a host sync:
//   step_tables  positions, slots and owning rows of a step's tokens from the requests' lengths, with the block tables
//                grown from a ring of free pages and dead pages given back to it
//   verify       acceptance of drafted tokens against the target's probabilities, from given random numbers
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "kv800_common.cuh"
#include "tc5.cuh"

namespace kv800 {

// ------------------------------------------------------------------------------------------------ step tables
// With n = n0 + qlen tokens after the step, a group of pages of pg tokens covers `cover` tokens of a row and has no use
// for the first `gone` of them:
//   KV800_PAGES_ALL      cover n             gone 0
//   KV800_PAGES_TAIL     cover n             gone 256 nq(n0)      (exact pages of a quantized layer)
//   KV800_PAGES_WINDOW   cover n             gone n0 - 255        (exact pages of a window layer)
//   KV800_PAGES_FLUSHED  cover 256 nq(n)     gone 0               (pages of sub-blocks)
// need = ceil(cover / pg); the row takes max(0, need - owned) pages off the ring's head, in row order, and gives
// min(gone / pg, owned) - first pages back at its tail.  All offsets are exclusive sums over the rows.  Nothing that the
// launch reads is written by it (taken entries are read at the head, returned ones written behind the tail, the new
// state goes to another buffer), so the same call gives the same result again.
struct Group {
    int32_t* table;
    int64_t stride;
    int32_t* ring;
    const int64_t* state;   // owned[R] | first[R] | head | tail
    int64_t* out;
    uint32_t width, cap, pg;
    int kind;
};

struct TablesArgs {
    const int32_t* n0;
    const int32_t* qlen;
    int R;
    int64_t T;
    Group g[2];             // exact pages, pages of sub-blocks
    int ngroups;
    int32_t* qsl;
    int32_t* rows;
    int64_t* pos;
    int64_t* slots;
    int32_t* N;
    int32_t* NQ;
    int* status;
};

constexpr int ST_THREADS = 512;
constexpr int ST_MAX_ROWS = 16384;   // two ints of shared memory a row
constexpr int ST_SHARE = 128;        // rows a CTA may own: the grid is 148 CTAs at ST_MAX_ROWS
constexpr uint32_t NONE = 0xffffffffu;

__device__ __forceinline__ uint32_t flushed_tokens(uint32_t n) { return n > LAG ? (n - LAG) / BLK * BLK : 0u; }

// saturating sum: an overflowing total stays above every limit it is compared with
__device__ __forceinline__ uint32_t add_sat(uint32_t x, uint32_t y) {
    const uint32_t z = x + y;
    return z < x ? 0xffffffffu : z;
}

__device__ __forceinline__ void row_len(const TablesArgs& a, int r, uint32_t& n0, uint32_t& ql) {
    const int x = a.n0[r], y = a.qlen[r];
    n0 = x > 0 ? x : 0;
    ql = y > 0 ? y : 0;
    if (n0 + ql > 0x7fffffffu) ql = 0x7fffffffu - n0;
}

// pages row r of group g takes (take) and gives back (give)
__device__ __forceinline__ void row_pages(const Group& g, int R, int r, uint32_t n0, uint32_t n, uint32_t& owned,
                                          uint32_t& first, uint32_t& take, uint32_t& give, bool& wide) {
    owned = (uint32_t)g.state[r];
    first = (uint32_t)g.state[R + r];
    const uint32_t cover = g.kind == KV800_PAGES_FLUSHED ? flushed_tokens(n) : n;
    const uint32_t need = cover ? (cover - 1) / g.pg + 1 : 0;
    wide = need > g.width;
    take = (!wide && need > owned) ? need - owned : 0;
    give = 0;
    if (g.kind == KV800_PAGES_TAIL || g.kind == KV800_PAGES_WINDOW) {
        const uint32_t gone = g.kind == KV800_PAGES_TAIL ? flushed_tokens(n0) : (n0 > WIN - 1 ? n0 - (WIN - 1) : 0);
        uint32_t live = gone / g.pg;
        live = live < owned ? live : owned;
        if (live > g.width) live = g.width;
        give = live > first ? live - first : 0;
    }
}

// Bound: a launch and two dependent passes over the rows' lengths and page counts (L2 latency); every CTA scans all rows
// for itself, which costs less than a second launch up to thousands of rows, and then takes its share of the rows'
// columns (8 lanes a row) and of the tokens.  8 us for one row, 17 us for 2,048 rows of some 3 tokens, 12 us for 64 rows of some 550
// (as graphs; a call takes 25 us of the host's time).
__global__ void __launch_bounds__(ST_THREADS) step_tables_kernel(const __grid_constant__ TablesArgs a) {
    extern __shared__ uint32_t sm[];
    uint32_t* s_qsl = sm;              // [R + 1]
    uint32_t* s_off = sm + a.R + 1;    // exact group: pages taken by the rows before, NONE where the row's do not fit
    __shared__ uint32_t s_own[ST_SHARE][2][2];   // this CTA's rows: offsets of what they take and give, per group
    __shared__ uint32_t s_part[5][ST_THREADS / 32];
    __shared__ uint32_t s_used[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (a.R + ST_THREADS - 1) / ST_THREADS, r0 = min(a.R, tid * per), r1 = min(a.R, r0 + per);
    if (tid < 2) s_used[tid] = 0;
    uint32_t sum[5] = {0, 0, 0, 0, 0};   // tokens, exact taken / given, quant taken / given
    for (int r = r0; r < r1; r++) {
        uint32_t n0, ql;
        row_len(a, r, n0, ql);
        sum[0] = add_sat(sum[0], ql);
        for (int k = 0; k < a.ngroups; k++) {
            uint32_t ow, fi, ta, gi;
            bool wide;
            row_pages(a.g[k], a.R, r, n0, n0 + ql, ow, fi, ta, gi, wide);
            sum[1 + 2 * k] = add_sat(sum[1 + 2 * k], ta);
            sum[2 + 2 * k] = add_sat(sum[2 + 2 * k], gi);
            if (wide && blockIdx.x == 0) flag(a.status, ST_TABLE);
        }
    }
    uint32_t ex[5], total[5];   // exclusive sums, totals
#pragma unroll
    for (int v = 0; v < 5; v++) {
        uint32_t x = sum[v];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x = add_sat(x, y);
        }
        if (lane == 31) s_part[v][warp] = x;
        const uint32_t left = __shfl_up_sync(0xffffffffu, x, 1);
        ex[v] = lane ? left : 0;
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < 5; v++) {
        uint32_t before = 0, all = 0;
        for (int w = 0; w < ST_THREADS / 32; w++) {
            const uint32_t x = s_part[v][w];
            if (w < warp) before = add_sat(before, x);
            all = add_sat(all, x);
        }
        ex[v] = add_sat(ex[v], before);
        total[v] = all;
    }
    // room and ring positions of the groups
    uint32_t head[2] = {0, 0}, tail[2] = {0, 0}, room[2] = {0, 0};
    for (int k = 0; k < a.ngroups; k++) {
        const int64_t h = a.g[k].state[2 * a.R], t = a.g[k].state[2 * a.R + 1];
        const int64_t free = t - h;
        head[k] = (uint32_t)(h % a.g[k].cap);
        tail[k] = (uint32_t)(t % a.g[k].cap);
        room[k] = free < 0 ? 0 : (uint32_t)(free < a.g[k].cap ? free : a.g[k].cap);
        if (total[1 + 2 * k] > room[k] && blockIdx.x == 0 && tid == 0) flag(a.status, ST_TABLE);
    }
    // rows: offsets for the tokens in shared memory, and (this CTA's share) lengths and new states
    const int share = (a.R + gridDim.x - 1) / gridDim.x, b0 = min(a.R, (int)blockIdx.x * share), b1 = min(a.R, b0 + share);
    for (int r = r0; r < r1; r++) {
        uint32_t n0, ql;
        row_len(a, r, n0, ql);
        const bool mine = r >= b0 && r < b1;
        s_qsl[r] = ex[0];
        if (mine) {
            a.qsl[r] = (int)ex[0];
            a.N[r] = (int)(n0 + ql);
            a.NQ[r] = (int)(flushed_tokens(n0) / BLK);
        }
        ex[0] = add_sat(ex[0], ql);
        for (int k = 0; k < a.ngroups; k++) {
            const Group& g = a.g[k];
            uint32_t ow, fi, ta, gi;
            bool wide;
            row_pages(g, a.R, r, n0, n0 + ql, ow, fi, ta, gi, wide);
            const uint32_t off = ex[1 + 2 * k], back = ex[2 + 2 * k], end = add_sat(off, ta);
            const bool fits = end <= room[k];
            if (k == 0) s_off[r] = (fits && !wide) ? off : NONE;
            if (fits && ta && blockIdx.x == 0) atomicMax(&s_used[k], end);
            if (mine) {
                g.out[r] = ow + (fits ? ta : 0);
                g.out[a.R + r] = fi + gi;
                s_own[r - b0][k][0] = fits ? off : NONE;
                s_own[r - b0][k][1] = back;
            }
            ex[1 + 2 * k] = end;
            ex[2 + 2 * k] = add_sat(back, gi);
        }
    }
    if (tid == 0) s_qsl[a.R] = total[0];
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) {
        a.qsl[a.R] = (int)total[0];
        if ((int64_t)total[0] > a.T) flag(a.status, ST_TABLE);
        for (int k = 0; k < a.ngroups; k++) {
            a.g[k].out[2 * a.R] = a.g[k].state[2 * a.R] + s_used[k];
            a.g[k].out[2 * a.R + 1] = a.g[k].state[2 * a.R + 1] + total[2 + 2 * k];
        }
    }
    // columns of this CTA's rows, 8 lanes a row
    for (int r = b0 + (tid >> 3); r < b1; r += ST_THREADS / 8) {
        uint32_t n0, ql;
        row_len(a, r, n0, ql);
        for (int k = 0; k < a.ngroups; k++) {
            const Group& g = a.g[k];
            uint32_t ow, fi, ta, gi;
            bool wide;
            row_pages(g, a.R, r, n0, n0 + ql, ow, fi, ta, gi, wide);
            int32_t* row = g.table + (int64_t)r * g.stride;
            const uint32_t off = s_own[r - b0][k][0], back = s_own[r - b0][k][1];
            if (off != NONE)
                for (uint32_t c = tid & 7; c < ta; c += 8) row[ow + c] = g.ring[(head[k] + off + c) % g.cap];
            for (uint32_t c = tid & 7; c < gi; c += 8) g.ring[(tail[k] + back + c) % g.cap] = row[fi + c];
        }
    }
    // tokens
    const uint32_t pg = a.g[0].pg;
    for (int64_t t = (int64_t)blockIdx.x * ST_THREADS + tid; t < a.T; t += (int64_t)gridDim.x * ST_THREADS) {
        int row = -1;
        int64_t p = 0, slot = -1;
        if (t < (int64_t)total[0]) {
            int lo = 0, hi = a.R;   // s_qsl[lo] <= t < s_qsl[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if ((int64_t)s_qsl[mid] <= t) lo = mid;
                else hi = mid;
            }
            row = lo;
            uint32_t n0, ql;
            row_len(a, row, n0, ql);
            const uint32_t q = n0 + (uint32_t)(t - s_qsl[row]), col = q / pg;
            const uint32_t owned = (uint32_t)a.g[0].state[row];
            p = q;
            int page = -1;
            if (col < owned) {
                if (col < a.g[0].width) page = a.g[0].table[(int64_t)row * a.g[0].stride + col];
            } else if (s_off[row] != NONE) {
                page = a.g[0].ring[(head[0] + s_off[row] + (col - owned)) % a.g[0].cap];
            }
            if (page >= 0) slot = (int64_t)page * pg + (q - col * pg);
        }
        a.rows[t] = row;
        a.pos[t] = p;
        a.slots[t] = slot;
    }
}

// ------------------------------------------------------------------------------------------------ verify
// Row b holds k = qsl[b + 1] - qsl[b] - 1 drafts: tokens[qsl[b] + 1 + i], judged by the target row x_i = logits[qsl[b] + i].
// With p_i = softmax(x_i / T) and q_i the draft model's probabilities (1 at the draft without them), draft i stands while
// every one before it does and u q_i(d) < p_i(d), u = uniform[qsl[b] + i].  The token after the m accepted ones is
// argmax_v r(v) / e(v) with r = max(p_m - q_m, 0) where draft m was rejected (p_m without d itself, lacking q), r = p_k
// where all stand, and e = noise[b]: for exponential e that is a sample of r / sum r, without a running sum over the
// vocabulary whose rounding would decide the token.  T = 0: argmax on both sides.  Ties go to the lowest index.
// A target row without a finite maximum (everything masked to -inf) accepts nothing and gives no token; greedy, +inf is a maximum.
// Two launches, the second overlapping the first's end.  With q, verify_stats gives the maximum (with its first index) and the sum
// of exponentials of every slice of every target row, one CTA a slice with all its loads in flight at once; verify_pick, some CTAs a
// request, merges them, judges the drafts and takes the argmax over one row, which it has to read again: p - q wants the row's sum
// first.  Without q, r is p but for one token, and argmax p / e = argmax x / T - log e needs no sum: verify_race takes it
// along for every target row (a warp keeps its 512 tokens' log e in registers for all rows of the request), so that the logits and
// the noise are read once, and race_pick is left with the slices' results.  Both are bound by those reads.
// Sums are held in 32 bits, x / T - log e too: from the slice's maximum on, so that its error is that of numbers below 30.
struct VerifyArgs {
    const void* logits;
    int64_t ldx;
    const int32_t* tokens;
    const int32_t* qsl;
    const float* u;
    const float* noise;
    int64_t lde;
    const float* q;
    int64_t ldq, nq;
    const float* temp;
    int R, K;
    int64_t T;
    int V;
    int32_t* out;       // [R, K + 1]
    int32_t* emitted;   // [R]
    int* status;
    void* stats;        // [R (K + 1)][slices] of Stat, or of Race
    int slices;
    unsigned long long* wins;   // [R][parts]: Best of a CTA's share
    int parts;          // CTAs a request in verify_pick
    unsigned* done;     // [R] CTAs of verify_pick that have finished
};

constexpr int VT = 256;          // threads a CTA
constexpr int VK = 64;           // most target rows a request (drafts + 1)
constexpr int VLOADS = 8;        // 16-byte loads a thread, all in flight: a slice is 32 KB of a row
constexpr float NEG = -3.402823466e38f;

template <typename T> struct Vec;
template <> struct Vec<float> { static constexpr int n = 4; };
template <> struct Vec<__nv_bfloat16> { static constexpr int n = 8; };
template <> struct Vec<__half> { static constexpr int n = 8; };

__device__ __forceinline__ void unpack(const uint4& w, float (&f)[4], const float*) {
    f[0] = __uint_as_float(w.x), f[1] = __uint_as_float(w.y), f[2] = __uint_as_float(w.z), f[3] = __uint_as_float(w.w);
}
__device__ __forceinline__ void unpack(const uint4& w, float (&f)[8], const __nv_bfloat16*) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) f[2 * i] = __uint_as_float(v[i] << 16), f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
}
__device__ __forceinline__ void unpack(const uint4& w, float (&f)[8], const __half*) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&v[i]));
        f[2 * i] = t.x, f[2 * i + 1] = t.y;
    }
}
__device__ __forceinline__ float tof(float x) { return x; }
__device__ __forceinline__ float tof(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float tof(__half x) { return __half2float(x); }

__device__ __forceinline__ float rcpf(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// running maximum (with its first index) and sum of exp2((x - max) c)
struct Stat {
    float m, s;
    int i;
};
__device__ __forceinline__ void merge(Stat& a, const Stat& b, float c) {
    const float m = fmaxf(a.m, b.m);
    a.s = a.s * exp2_approx((a.m - m) * c) + b.s * exp2_approx((b.m - m) * c);   // both finite: NEG stands for "nothing yet"
    if (b.m > a.m || (b.m == a.m && b.i < a.i)) a.i = b.i;
    a.m = m;
}
struct Best {
    float v;
    int i;
};
__device__ __forceinline__ void merge(Best& a, const Best& b) {
    if (b.v > a.v || (b.v == a.v && b.i < a.i)) a = b;
}

// n of a request's target rows, or 0 (flagged) where they do not lie in [0, T) or are more than K + 1
__device__ __forceinline__ int target_rows(const VerifyArgs& a, int b, int64_t& q0) {
    q0 = a.qsl[b];
    const int64_t q1 = a.qsl[b + 1];
    return q0 < 0 || q1 < q0 || q1 > a.T || q1 - q0 > a.K + 1 ? -1 : (int)(q1 - q0);
}
// the factor of the exponents, log2(e) / temperature; 0 for greedy rows
__device__ __forceinline__ float factor_of(const VerifyArgs& a, int b) {
    const float t = a.temp ? a.temp[b] : 1.0f;
    return t > 0.0f ? fmaxf(1e-30f, fminf(1e30f, 1.4426950408889634f / t)) : 0.0f;
}

// grid (slices, K + 1, R).  The slice of a row starts at its first 16-byte boundary plus a multiple of the slice's vectors; the
// elements before that boundary and after the last whole vector go to slice 0.
template <typename T>
__global__ void __launch_bounds__(VT) verify_stats(const __grid_constant__ VerifyArgs a) {
    constexpr int n = Vec<T>::n;
    const int b = blockIdx.z, row = blockIdx.y, slice = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    __shared__ Stat s_warp[VT / 32];
    pdl_launch_dependents();
    if (row == 0 && slice == 0 && tid == 0) a.done[b] = 0;
    int64_t q0;
    if (row >= target_rows(a, b, q0)) return;
    const T* p = reinterpret_cast<const T*>(a.logits) + (q0 + row) * a.ldx;
    const int skip = min(a.V, (int)(((16u - (unsigned)(reinterpret_cast<uintptr_t>(p) & 15u)) & 15u) / sizeof(T)));
    const int nv = (a.V - skip) / n, v0 = slice * (VLOADS * VT) + tid;
    const uint4* w = reinterpret_cast<const uint4*>(p + skip);
    uint4 x[VLOADS];
#pragma unroll
    for (int k = 0; k < VLOADS; k++)
        if (v0 + k * VT < nv) x[k] = __ldg(w + v0 + k * VT);
    float edge = -INFINITY;
    int edge_at = 0x7fffffff;
    if (slice == 0) {
        const int e = tid < skip ? tid : nv * n + tid;   // nv * n + skip + (tid - skip)
        if (tid < skip + (a.V - skip - nv * n)) edge = tof(p[e]), edge_at = e;
    }
    const float c = factor_of(a, b);
    Stat st{fmaxf(edge, NEG), 0.0f, edge > -INFINITY ? edge_at : 0x7fffffff};
    float top = NEG;
#pragma unroll
    for (int k = 0; k < VLOADS; k++)
        if (v0 + k * VT < nv) {
            float f[n];
            unpack(x[k], f, (const T*)nullptr);
#pragma unroll
            for (int i = 0; i < n; i += 2) top = fmaxf(top, fmaxf(f[i], f[i + 1]));
        }
    if (c == 0.0f) {                 // only a greedy row asks where the maximum is
        int at = 0x7fffffff;
#pragma unroll
        for (int k = VLOADS - 1; k >= 0; k--)
            if (v0 + k * VT < nv) {
                float f[n];
                unpack(x[k], f, (const T*)nullptr);
#pragma unroll
                for (int i = n - 1; i >= 0; i--)
                    if (f[i] == top) at = skip + (v0 + k * VT) * n + i;
            }
        if (top > st.m || (top == st.m && at < st.i)) st.i = at;
    }
    st.m = fmaxf(st.m, top);
    if (edge_at < 0x7fffffff) st.s = exp2_approx((edge - st.m) * c);
    const f2 c2(c, c), m2(-st.m, -st.m);
    f2 s2(0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < VLOADS; k++)
        if (v0 + k * VT < nv) {
            float f[n];
            unpack(x[k], f, (const T*)nullptr);
#pragma unroll
            for (int i = 0; i < n; i += 2) {
                float y, z;
                mul2(add2(f2(f[i], f[i + 1]), m2), c2).get(y, z);
                s2 = add2(s2, f2(exp2_approx(y), exp2_approx(z)));
            }
        }
    {
        float y, z;
        s2.get(y, z);
        st.s += y + z;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        Stat t{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), __shfl_xor_sync(0xffffffffu, st.i, o)};
        merge(st, t, c);
    }
    if (lane == 0) s_warp[warp] = st;
    __syncthreads();
    if (tid == 0) {
        for (int k = 1; k < VT / 32; k++) merge(st, s_warp[k], c);
        static_cast<Stat*>(a.stats)[((int64_t)b * (a.K + 1) + row) * a.slices + slice] = st;
    }
}

// The race over the row that decides, with q: as many CTAs a request as are resident at once (4 an SM), each of which judges the
// request's drafts for itself (a few hundred bytes of statistics), then takes every parts-th chunk of 4,096 tokens of the row, of q
// and of the noise, the chunk's loads all in flight.  The last of a request's CTAs to finish joins their winners.  Ties go to the
// lowest token, so the order in which CTAs finish does not show.  Latency bounds it at 64 rows x 4 drafts of 65,536 bf16 logits
// (19 us with verify_stats, 63 MB), traffic at 200 x 2 of 100,001 (66 us, 290 MB; a cluster a request, walking in vector loads: 78;
// a CTA for every chunk: 93).
constexpr int PE = 16, PC = PE * VT;   // tokens a thread, a CTA
template <typename T>
__global__ void __launch_bounds__(VT, 4) verify_pick(const __grid_constant__ VerifyArgs a) {
    const int parts = a.parts, b = blockIdx.x / parts, part = blockIdx.x - b * parts;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    __shared__ Stat s_all[VK];
    __shared__ unsigned long long s_ok;
    __shared__ Best s_win[VT / 32];
    __shared__ int s_last;
    const float c = factor_of(a, b);
    const bool greedy = c == 0.0f;
    int64_t q0;
    int n = target_rows(a, b, q0);   // k + 1
    int64_t dq = 0;                  // the request's first row of q: drafts of the rows before it (their tokens less one each)
    {
        int empty = 0;
        for (int base = 0; base < b; base += VT) {
            const int r = base + tid;
            empty += __syncthreads_count(r < b && a.qsl[r + 1] <= a.qsl[r]);
        }
        dq = q0 - a.qsl[0] - (b - empty);
    }
    if (n < 0 || dq < 0 || (n && dq + n - 1 > a.nq)) {
        if (tid == 0 && part == 0) flag(a.status, ST_TABLE);
        n = 0;
    }
    const T* x0 = reinterpret_cast<const T*>(a.logits) + q0 * a.ldx;
    // what the judgement needs of the inputs, on its way while the statistics are made
    int d = -1;
    float xd = 0.0f, ud = 0.0f, qd = 0.0f;
    if (tid < n - 1) {
        d = a.tokens[q0 + tid + 1];
        if (d < 0 || d >= a.V) {
            if (part == 0) flag(a.status, ST_TABLE);
            d = -1;
        } else {
            xd = tof(x0[tid * a.ldx + d]);
            ud = a.u[q0 + tid];
            qd = a.q[(dq + tid) * a.ldq + d];
        }
    }
    if (tid == 0) s_ok = 0;
    __syncthreads();
    pdl_wait();
    for (int row = warp; row < n; row += VT / 32) {
        const Stat* src = static_cast<const Stat*>(a.stats) + ((int64_t)b * (a.K + 1) + row) * a.slices;
        Stat st{NEG, 0.0f, 0x7fffffff};
        for (int k = lane; k < a.slices; k += 32) merge(st, src[k], c);
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            Stat t{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), __shfl_xor_sync(0xffffffffu, st.i, o)};
            merge(st, t, c);
        }
        if (st.i == 0x7fffffff) st.i = -1;
        if (lane == 0) s_all[row] = st;
    }
    __syncthreads();
    if (d >= 0) {
        const Stat st = s_all[tid];
        if (greedy ? st.i == d : ud * qd < exp2_approx((xd - st.m) * c) / st.s) atomicOr(&s_ok, 1ull << tid);
    }
    __syncthreads();
    const int m = n > 0 ? __ffsll((long long)~s_ok) - 1 : 0;   // accepted drafts (bit n - 1 is never set)
    int chosen = n > 0 && greedy ? s_all[m].i : -1;
    const bool race = n > 0 && !greedy;
    if (race) {
        const Stat st = s_all[m];
        const T* x = x0 + (int64_t)m * a.ldx;
        const bool less = m < n - 1;
        const float *q = a.q + (less ? dq + m : 0) * a.ldq, *e = a.noise + (int64_t)b * a.lde;
        const float inv = 1.0f / st.s;
        // the winner among every `every`-th chunk from the first on: of the residual, or of p
        auto walk = [&](const float* q, int first, int every) {
            Best w{0.0f, 0x7fffffff};
            auto chunk = [&](int64_t j0, auto full) {
                T xv[PE];
                float ev[PE], qv[PE];
#pragma unroll
                for (int k = 0; k < PE; k++) {
                    const bool in = decltype(full)::value || j0 + VT * k < a.V;
                    ev[k] = in ? __ldcs(e + j0 + VT * k) : 1.0f;
                    xv[k] = in ? __ldcs(x + j0 + VT * k) : T(-INFINITY);
                    qv[k] = q && in ? __ldcs(q + j0 + VT * k) : 0.0f;
                }
#pragma unroll
                for (int k = 0; k < PE; k++) {
                    const float v = fmaf(exp2_approx((tof(xv[k]) - st.m) * c), inv, -qv[k]) * rcpf(ev[k]);
                    if (v > w.v) w = Best{v, (int)j0 + VT * k};   // j grows, so a tie keeps the lower token
                }
            };
            for (int64_t j = (int64_t)first * PC; j < a.V; j += (int64_t)every * PC) {
                if (j + PC <= a.V) chunk(j + tid, std::true_type{});
                else chunk(j + tid, std::false_type{});
            }
            return w;
        };
        auto across = [&](Best w, int from) {   // the warp's lanes below 2 * from
            for (int o = from; o; o >>= 1) merge(w, Best{__shfl_xor_sync(0xffffffffu, w.v, o), __shfl_xor_sync(0xffffffffu, w.i, o)});
            return w;
        };
        auto block = [&](Best w) {              // thread 0 is left with the CTA's
            w = across(w, 16);
            __syncthreads();
            if (lane == 0) s_win[warp] = w;
            __syncthreads();
            return across(s_win[lane & (VT / 32 - 1)], VT / 64);
        };
        Best w = block(walk(less ? q : nullptr, part, parts));
        unsigned long long* all = a.wins + (int64_t)b * parts;
        if (tid == 0) {
            all[part] = (unsigned long long)__float_as_uint(w.v) << 32 | (unsigned)w.i;
            __threadfence();
            s_last = atomicAdd(a.done + b, 1u) == (unsigned)parts - 1;
        }
        __syncthreads();
        if (!s_last) return;
        __threadfence();
        w = Best{0.0f, 0x7fffffff};
        for (int k = tid; k < parts; k += VT) {
            const unsigned long long t = __ldcg(all + k);
            merge(w, Best{__uint_as_float((unsigned)(t >> 32)), (int)(unsigned)t});
        }
        w = block(w);
        if (less && w.i == 0x7fffffff) w = block(walk(nullptr, 0, 1));     // no residual: rare, and this CTA's alone
        chosen = w.i == 0x7fffffff ? -1 : w.i;
    } else if (part) {
        return;
    }
    if (tid < a.K + 1) {
        a.out[(int64_t)b * (a.K + 1) + tid] = tid < m ? a.tokens[q0 + tid + 1] : tid == m ? chosen : -1;
        if (tid == 0) a.emitted[b] = m + (chosen >= 0 ? 1 : 0);
    }
}

// A slice of a target row without q: its maximum and sum as in Stat, and the winner of the race: v = max (x - m) c - log2 e over
// the tokens but the row's draft, at i.  Greedy rows race with c = 1 and e = 1, and with 0 for m, so that +inf wins like any other
// maximum (inf - inf would take it out): v is the maximum, i the argmax, drafts included, and s means nothing.
struct Race {
    float m, s, v;
    int i;
};
constexpr int RE = 16;               // tokens a lane
constexpr int RC = 32 * RE;          // tokens a warp: a slice
__device__ __forceinline__ void merge(Race& a, const Race& b, float c) {
    const float m = fmaxf(a.m, b.m), fa = (a.m - m) * c, fb = (b.m - m) * c;
    a.s = a.s * exp2_approx(fa) + b.s * exp2_approx(fb);
    const float va = fmaxf(a.v + fa, -INFINITY), vb = fmaxf(b.v + fb, -INFINITY);   // inf - inf: not a candidate
    if (vb > va || (vb == va && b.i < a.i)) a.i = b.i;
    a.v = fmaxf(va, vb);
    a.m = m;
}
__device__ __forceinline__ float lg2f(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float warp_max(float x) {   // NaN is skipped
    float y;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}

// grid (slices / 8, shares of the rows, R).  Lanes read neighbouring tokens one by one: no alignment is asked of rows whose
// vocabulary is odd, and 16 loads a lane are in flight for the row after the one that is worked on.  The winner's place is looked
// up once its value is known, which costs fewer instructions than to carry it along.  192 rows x 5 drafts of 128,000 fp32 logits
// take 80 us with race_pick, 485 MB at 6.05 TB/s (places carried along: 86; four CTAs an SM in 64 registers, measured so: three 99,
// five 98 us); bf16 logits 72 us, 292 MB at 4.05 TB/s, where the instructions a token are the limit.
template <typename T>
__global__ void __launch_bounds__(VT, 4) verify_race(const __grid_constant__ VerifyArgs a) {
    const int b = blockIdx.z, lane = threadIdx.x & 31, slice = blockIdx.x * (VT / 32) + (threadIdx.x >> 5);
    pdl_launch_dependents();
    int64_t q0;
    const int n = target_rows(a, b, q0), step = gridDim.y;
    int row = blockIdx.y;
    if (slice >= a.slices || row >= n) return;
    const int j0 = slice * RC + lane;
    const bool full = (slice + 1) * (int64_t)RC <= a.V;      // no bounds to watch
    const T* p = reinterpret_cast<const T*>(a.logits) + (q0 + row) * a.ldx + j0;
    T x[RE];
    auto load = [&](const T* src) {
        if (full) {
#pragma unroll
            for (int k = 0; k < RE; k++) x[k] = __ldcs(src + 32 * k);
        } else {
#pragma unroll
            for (int k = 0; k < RE; k++) x[k] = j0 + 32 * k < a.V ? __ldcs(src + 32 * k) : T(-INFINITY);
        }
    };
    load(p);
    float c = factor_of(a, b), l[RE];        // -log2 e
    const bool greedy = c == 0.0f;
    if (greedy) c = 1.0f;
    const float* e = a.noise + (int64_t)b * a.lde + j0;
#pragma unroll
    for (int k = 0; k < RE; k++) l[k] = !greedy && j0 + 32 * k < a.V ? __ldcs(e + 32 * k) : 1.0f;
#pragma unroll
    for (int k = 0; k < RE; k++) l[k] = -lg2f(l[k]);
    const f2 c2(c, c);
    for (; row < n; row += step) {
        float f[RE];
#pragma unroll
        for (int k = 0; k < RE; k++) f[k] = tof(x[k]);
        p += step * a.ldx;
        if (row + step < n) load(p);
        float m = f[0];
#pragma unroll
        for (int k = 1; k < RE; k++) m = fmaxf(m, f[k]);
        m = greedy ? 0.0f : fmaxf(warp_max(m), NEG);
        const f2 m2(-m, -m);
        f2 s2(0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < RE; k += 2) {
            const f2 d = add2(f2(f[k], f[k + 1]), m2);
            float y, z;
            mul2(d, c2).get(y, z);
            s2 = add2(s2, f2(exp2_approx(y), exp2_approx(z)));
            fma2(d, c2, f2(l[k], l[k + 1])).get(f[k], f[k + 1]);
        }
        if (!greedy && row + 1 < n) {      // the row's draft does not race
            const int out = a.tokens[q0 + row + 1] - slice * RC;
            if (out >= 0 && out < RC) {
#pragma unroll
                for (int k = 0; k < RE; k++)
                    if (out == 32 * k + lane) f[k] = -INFINITY;
            }
        }
        float s, v = f[0];
        {
            float y, z;
            s2.get(y, z);
            s = y + z;
        }
#pragma unroll
        for (int k = 1; k < RE; k++) v = fmaxf(v, f[k]);       // NaN is skipped
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        const float best = fmaxf(warp_max(v), -INFINITY);
        unsigned i = 0x7fffffffu;
        if (v == best && best > -INFINITY) {
#pragma unroll
            for (int k = RE - 1; k >= 0; k--)
                if (f[k] == best) i = j0 + 32 * k;
        }
        i = __reduce_min_sync(0xffffffffu, i);
        if (lane == 0)
            *reinterpret_cast<float4*>(static_cast<Race*>(a.stats) + ((int64_t)b * (a.K + 1) + row) * a.slices + slice) =
                make_float4(m, s, best, __int_as_float((int)i));
    }
}

template <typename T>
__global__ void __launch_bounds__(VT) race_pick(const __grid_constant__ VerifyArgs a) {
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    __shared__ Race s_all[VK];
    __shared__ unsigned long long s_ok;
    int64_t q0;
    int n = target_rows(a, b, q0);   // k + 1
    if (n < 0) {
        if (tid == 0) flag(a.status, ST_TABLE);
        n = 0;
    }
    float c = factor_of(a, b);
    const bool greedy = c == 0.0f;
    if (greedy) c = 1.0f;
    int d = -1;
    float xd = 0.0f, ud = 0.0f;
    if (tid < n - 1) {
        d = a.tokens[q0 + tid + 1];
        if (d < 0 || d >= a.V) {
            flag(a.status, ST_TABLE);
            d = -1;
        } else {
            xd = tof(__ldg(reinterpret_cast<const T*>(a.logits) + (q0 + tid) * a.ldx + d));
            ud = a.u[q0 + tid];
        }
    }
    if (tid == 0) s_ok = 0;
    __syncthreads();
    pdl_wait();
    for (int row = warp; row < n; row += VT / 32) {
        const float4* src = reinterpret_cast<const float4*>(static_cast<const Race*>(a.stats) + ((int64_t)b * (a.K + 1) + row) * a.slices);
        Race st{NEG, 0.0f, -INFINITY, 0x7fffffff};
        for (int k = lane; k < a.slices; k += 32) {
            const float4 x = src[k];
            merge(st, Race{x.x, x.y, x.z, __float_as_int(x.w)}, c);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1)
            merge(st, Race{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), __shfl_xor_sync(0xffffffffu, st.v, o),
                           __shfl_xor_sync(0xffffffffu, st.i, o)}, c);
        if (lane == 0) s_all[row] = st;
    }
    __syncthreads();
    float pd = 0.0f;                 // p of the thread's draft
    if (d >= 0) {
        const Race st = s_all[tid];
        pd = exp2_approx((xd - st.m) * c) / st.s;
        if (greedy ? st.i == d : ud < pd) atomicOr(&s_ok, 1ull << tid);
    }
    __syncthreads();
    const int m = n > 0 ? __ffsll((long long)~s_ok) - 1 : 0;   // accepted drafts (bit n - 1 is never set)
    __shared__ int s_left;           // the rejected draft, where nothing else has a weight
    if (tid == m) s_left = d >= 0 && pd > 0.0f ? d : -1;
    __syncthreads();
    if (tid < a.K + 1) {
        int chosen = -1;
        if (n > 0) {
            const Race st = s_all[m];
            if (greedy || (st.s > 0.0f && st.s < INFINITY)) chosen = st.i < 0x7fffffff ? st.i : greedy ? -1 : s_left;
        }
        a.out[(int64_t)b * (a.K + 1) + tid] = tid < m ? a.tokens[q0 + tid + 1] : tid == m ? chosen : -1;
        if (tid == 0) a.emitted[b] = m + (chosen >= 0 ? 1 : 0);
    }
}

}  // namespace kv800

using namespace kv800;

static bool group_of(const kv800_pages* p, int64_t R, Group& g) {
    if ((R && !p->table) || !p->ring || !p->state || !p->state_out || p->state == p->state_out || p->width <= 0 ||
        p->table_stride < p->width || p->width > 0x7fffffffLL || p->cap <= 0 || p->cap > 0x3fffffffLL ||
        p->page_tokens <= 0 || p->page_tokens > 0x7fffffffLL || p->kind < KV800_PAGES_ALL ||
        p->kind > KV800_PAGES_FLUSHED)
        return false;
    g = Group{p->table, p->table_stride, p->ring, p->state, p->state_out, (uint32_t)p->width, (uint32_t)p->cap,
              (uint32_t)p->page_tokens, (int)p->kind};
    return true;
}

extern "C" int kv800_step_tables(const int32_t* n0, const int32_t* qlen, int64_t R, int64_t T, const kv800_pages* exact,
                                 const kv800_pages* quant, int32_t* query_start_loc, int32_t* rows, int64_t* positions,
                                 int64_t* slots, int32_t* N, int32_t* NQ, int* status, void* stream) {
    if (R < 0 || T < 0) {
        set_error("kv800_step_tables: negative R or T");
        return KV800_ERR_ARG;
    }
    if (R > ST_MAX_ROWS || T > 0x7fffffffLL) {
        set_error("kv800_step_tables: at most %d rows and 2^31 - 1 tokens", ST_MAX_ROWS);
        return KV800_ERR_RANGE;
    }
    if (R == 0 && T == 0) return KV800_OK;
    if (!exact || !query_start_loc || (R && (!n0 || !qlen || !N || !NQ)) || (T && (!rows || !positions || !slots))) {
        set_error("kv800_step_tables: null pointer");
        return KV800_ERR_ARG;
    }
    TablesArgs a{};
    a.n0 = n0, a.qlen = qlen, a.R = (int)R, a.T = T, a.ngroups = quant ? 2 : 1;
    a.qsl = query_start_loc, a.rows = rows, a.pos = positions, a.slots = slots, a.N = N, a.NQ = NQ, a.status = status;
    if (!group_of(exact, R, a.g[0]) || (quant && !group_of(quant, R, a.g[1]))) {
        set_error("kv800_step_tables: a group of pages needs table, ring, state and another state_out, 0 < width <= stride, "
                  "0 < cap < 2^30, page_tokens > 0 and a KV800_PAGES kind");
        return KV800_ERR_ARG;
    }
    const size_t smem = (2 * (size_t)R + 1) * 4;
    if (smem > 40 * 1024) {
        const int rc = cuda_status(cudaFuncSetAttribute(step_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                        (2 * ST_MAX_ROWS + 1) * 4), "step_tables smem attribute");
        if (rc) return rc;
    }
    // one CTA for 1,024 tokens or 64 rows, whichever asks for more, on at most 148 SMs
    int64_t grid = (T + 1023) / 1024;
    if ((R + 63) / 64 > grid) grid = (R + 63) / 64;
    grid = grid < 1 ? 1 : grid > 148 ? 148 : grid;
    step_tables_kernel<<<(unsigned)grid, ST_THREADS, smem, as_stream(stream)>>>(a);
    return cuda_status(cudaGetLastError(), "kv800_step_tables launch");
}

// the race's slices are the smaller ones, its results of one the larger
extern "C" int64_t kv800_verify_workspace_size(int64_t R, int64_t K, int64_t V) {
    if (R < 0 || K < 0 || V < 0) return -1;
    return (R * (K + 1) * ((V + RC - 1) / RC) * (int64_t)sizeof(Race) + R * (((V + PC - 1) / PC) * 8 + 4) + 255) & ~(int64_t)255;
}

template <typename T>
static int launch_verify(const VerifyArgs& a, cudaStream_t st) {
    for (int64_t r0 = 0; r0 < a.R; r0 += 65535) {   // the grid's z dimension holds 65,535 rows
        VerifyArgs s = a;
        const int rows = a.R - r0 < 65535 ? (int)(a.R - r0) : 65535;
        const int64_t at = r0 * (a.K + 1) * a.slices;
        s.qsl += r0;
        if (s.temp) s.temp += r0;
        if (a.q) {
            s.stats = static_cast<Stat*>(a.stats) + at;
            s.done += r0;
            verify_stats<T><<<dim3(a.slices, a.K + 1, rows), VT, 0, st>>>(s);
        } else {
            s.stats = static_cast<Race*>(a.stats) + at;
            s.noise += r0 * a.lde;
            // a warp takes all rows of its tokens, or a share of them where that leaves warps unused: 148 SMs hold 32 each
            const int64_t share = 148 * 32 / ((int64_t)rows * a.slices);
            verify_race<T><<<dim3((a.slices + VT / 32 - 1) / (VT / 32), share < 1 ? 1 : share > a.K ? a.K + 1 : (int)share, rows), VT, 0, st>>>(s);
        }
    }
    const int rc = cuda_status(cudaGetLastError(), "kv800_verify launch");
    if (rc) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)((int64_t)a.R * a.parts));
    cfg.blockDim = dim3(VT);
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cuda_status(a.q ? cudaLaunchKernelEx(&cfg, verify_pick<T>, a) : cudaLaunchKernelEx(&cfg, race_pick<T>, a), "kv800_verify launch");
}

extern "C" int kv800_verify(const void* logits, int64_t dtype, int64_t ld_logits, int64_t T, int64_t V,
                            const int32_t* tokens, const int32_t* query_start_loc, int64_t R, int64_t K,
                            const float* uniform, const float* noise, int64_t ld_noise, const float* draft_probs,
                            int64_t draft_rows, int64_t ld_probs, const float* temperature, int32_t* out, int32_t* emitted, void* workspace,
                            int64_t workspace_bytes, int* status, void* stream) {
    if (R < 0 || K < 0 || T < 0 || V <= 0 || dtype < KV800_BF16 || dtype > KV800_F32) {
        set_error("kv800_verify: need R, K, T >= 0, V > 0 and a KV800 dtype");
        return KV800_ERR_ARG;
    }
    if (K + 1 > VK || V > 0x3fffffffLL || R > 0x7ffffffLL) {
        set_error("kv800_verify: at most %d drafts a row, 2^30 - 1 tokens in the vocabulary, 2^27 - 1 rows", VK - 1);
        return KV800_ERR_RANGE;
    }
    if (R == 0) return KV800_OK;
    if ((T && (!logits || !tokens || !uniform)) || !query_start_loc || !noise || !out || !emitted || ld_logits < V ||
        ld_noise < V || (draft_probs && (ld_probs < V || draft_rows < 0))) {
        set_error("kv800_verify: null pointer, or a row stride below the vocabulary");
        return KV800_ERR_ARG;
    }
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u) || workspace_bytes < kv800_verify_workspace_size(R, K, V)) {
        set_error("kv800_verify: workspace of %lld bytes needed (16-byte aligned), got %lld",
                  (long long)kv800_verify_workspace_size(R, K, V), (long long)workspace_bytes);
        return workspace && workspace_bytes < kv800_verify_workspace_size(R, K, V) ? KV800_ERR_RANGE : KV800_ERR_ARG;
    }
    const int n = dtype == KV800_F32 ? 4 : 8;
    const int slices = draft_probs ? (int)((V / n + VLOADS * VT - 1) / (VLOADS * VT) + (V < n)) : (int)((V + RC - 1) / RC);
    const int64_t chunks = (V + PC - 1) / PC, room = 148 * 4 / R;
    const int parts = !draft_probs || room < 1 ? 1 : (int)(room < chunks ? room : chunks);
    uint8_t* wins = static_cast<uint8_t*>(workspace) + R * (K + 1) * ((V + RC - 1) / RC) * (int64_t)sizeof(Race);
    unsigned* done = reinterpret_cast<unsigned*>(wins + R * chunks * 8);
    VerifyArgs a{logits, ld_logits, tokens, query_start_loc, uniform, noise, ld_noise, draft_probs, ld_probs, draft_rows, temperature,
                 (int)R, (int)K, T, (int)V, out, emitted, status, workspace, slices, reinterpret_cast<unsigned long long*>(wins), parts, done};
    cudaStream_t st = as_stream(stream);
    if (dtype == KV800_BF16) return launch_verify<__nv_bfloat16>(a, st);
    if (dtype == KV800_F16) return launch_verify<__half>(a, st);
    return launch_verify<float>(a, st);
}
