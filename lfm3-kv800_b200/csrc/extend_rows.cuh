// Which keys a query of kv800_extend sees, and where they lie.
//
// A row (request) of N tokens, q1 - q0 of them new, has n0 = N - (q1 - q0) old ones.  Its keys in the order they are
// walked: positions [0, nquant) from the sub-blocks, then `nexact` exact ones, first the sink positions that lie before
// the walk's window, then positions from xlo on.  Every key is masked by position (ex_seen), so a range made for several
// queries serves each of them.
#pragma once
#include "kv800_common.cuh"

namespace kv800 {

constexpr float EX_SCALE = 0.12751743074602467f;   // 128^-0.5 * log2(e): scores in the log2 domain

struct ExtendArgs {
    kv800_paged P;
    const uint16_t* q;
    const int32_t* qsl;
    int R;
    int64_t T, max_qlen;
    const uint16_t* cos_t;
    const uint16_t* sin_t;
    int64_t npos;
    uint16_t* out;
    int* status;
    int own;     // CTAs plan for themselves: each flags in its own word, status[1 + CTA], and extend_join gathers them
};
__device__ __forceinline__ void ex_flag(const ExtendArgs& a, int bit) { flag(a.status + (a.own ? 1 + blockIdx.x : 0), bit); }

struct ExRow {
    int64_t q0, q1, n0, N;   // queries [q0, q1), the first at position n0
    int64_t nq;              // quantized sub-blocks
    int64_t lo;              // first exact position any of its queries needs
    int64_t ns;              // positions below this come from the sink rows
};

struct ExKeys {
    int64_t nquant, nexact, nsk, xlo;
};

__device__ __forceinline__ void ex_row(const ExtendArgs& a, int b, ExRow& r) {
    r.q0 = a.qsl[b];
    r.q1 = a.qsl[b + 1];
    if (r.q0 < 0) r.q0 = 0;
    if (r.q1 > a.T) r.q1 = a.T;
    r.N = a.P.N[b];
    r.n0 = r.N - (r.q1 - r.q0);
    int64_t nq = a.P.NQ[b];
    if (nq < 0) nq = 0;
    r.nq = a.P.win ? 0 : (nq < a.P.nqmax ? nq : a.P.nqmax);
    r.lo = nq * BLK;
    if (a.P.win && r.n0 + 1 - a.P.win > r.lo) r.lo = r.n0 + 1 - a.P.win;
    r.ns = (a.P.win && a.P.sk) ? (a.P.nsink < r.lo ? a.P.nsink : r.lo) : 0;
}

// keys that queries at positions [p0, p1] see
__device__ __forceinline__ void ex_keys(const ExtendArgs& a, const ExRow& r, int64_t p0, int64_t p1, ExKeys& k) {
    const int64_t end = p1 + 1 < r.N ? p1 + 1 : r.N;
    k.nquant = r.nq * BLK < end ? r.nq * BLK : (end > 0 ? end : 0);
    k.xlo = r.lo;
    if (a.P.win && p0 + 1 - a.P.win > k.xlo) k.xlo = p0 + 1 - a.P.win;
    k.nsk = (a.P.win && a.P.sk) ? (a.P.nsink < k.xlo ? a.P.nsink : k.xlo) : 0;
    if (k.nsk > end) k.nsk = end > 0 ? end : 0;
    k.nexact = k.nsk + (end > k.xlo ? end - k.xlo : 0);
}

// sub-block j of row b, or null (flagged) where its offset is outside the pool
__device__ __forceinline__ const uint8_t* ex_subblock(const ExtendArgs& a, int b, int64_t j) {
    const int64_t off = j < a.P.boff_stride ? a.P.boff[b * a.P.boff_stride + j] : -1;
    if (off < 0 || (off & 127) || off + SUB > a.P.qpool_bytes) {
        ex_flag(a, ST_QPOOL);
        return nullptr;
    }
    return a.P.qpool + off;
}

// K and V rows of head h at position kp (16-byte aligned); false (flagged) where they are outside their pool
__device__ __forceinline__ bool ex_exact(const ExtendArgs& a, int b, int ns, int h, int64_t kp,
                                         const uint16_t*& k, const uint16_t*& v) {
    if (kp < ns) {
        const int64_t at = (kp * HEADS + h) * DIM, ko = a.P.skoff[b] + at, vo = a.P.svoff[b] + at;
        if (((ko | vo) & 7) || ko < 0 || vo < 0 || ko + DIM > a.P.sk_elems || vo + DIM > a.P.sv_elems) {
            ex_flag(a, ST_SINK);
            return false;
        }
        k = a.P.sk + ko;
        v = a.P.sv + vo;
        return true;
    }
    int64_t pg, sl;
    page_split(kp, a.P.ebs, pg, sl);
    if (kp < 0 || pg >= a.P.eoff_stride) {
        ex_flag(a, ST_TABLE);
        return false;
    }
    const int64_t off = a.P.eoff[b * a.P.eoff_stride + pg] + h * a.P.e_hs + sl * a.P.e_ts;
    const int64_t last = off + (a.P.e_v > 0 ? a.P.e_v : 0) + DIM;
    if ((off & 7) || off < 0 || off + a.P.e_v < 0 || last > a.P.epool_elems) {
        ex_flag(a, ST_EPOOL);
        return false;
    }
    k = a.P.epool + off;
    v = k + a.P.e_v;
    return true;
}

// Zeros for the tokens before the first row's, which no row owns, by one CTA: query_start_loc begins with 0 but for odd callers.
__device__ __forceinline__ void ex_clear_first(const ExtendArgs& a) {
    const int64_t n = a.R ? min((int64_t)a.qsl[0], a.T) * (QROWS * DIM / 8) : 0;
    for (int64_t i = threadIdx.x; i < n; i += blockDim.x) reinterpret_cast<uint4*>(a.out)[i] = make_uint4(0, 0, 0, 0);
}

}  // namespace kv800
