// Attention of a chunk of new tokens over the paged 800h cache (kv800_extend): the ragged, causal, multi-token form of
// the decode, over quantized sub-blocks, exact pages and sinks.
#include "extend_few.cuh"
#include "extend_tc.cuh"
#include "tmap.cuh"

#include <atomic>

using namespace kv800;

namespace {
constexpr int MAX_DEV = 64;

// SMs of the current device: the persistent grid
int sm_count() {
    static std::atomic<int> cache[MAX_DEV];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= MAX_DEV) return 148;
    int n = cache[dev].load(std::memory_order_relaxed);
    if (!n) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
        cache[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

// The kernel by the longest row.  Up to 6 queries (24 rows a KV head) extend_few, whose cost is the keys': 64 rows x 5 queries of
// 32K take 467 us there and 1,073 on 128-row tiles, of 2K 67 and 92, on a window layer 31 and 37 (a single row 39 and 36 at 32K, 22
// and 18 on a window layer, but a launch more).  7 and 8 queries, whose sums no longer fit its registers, only over many sub-blocks:
// 64 x 8 of 32K 753 and 1,081, 16 x 8 228 and 285, but 4 x 8 96 and 85, 64 x 8 of 2K 101 and 92, of a window layer 42 and 37.  The
// host knows the sub-blocks by their bound nqmax alone: where that is far above what the rows hold, as in a captured step, 7 and 8
// queries of short rows take the slower of these.  Above that the 128-row tile (32 queries), and two of them above 32 (16 rows of
// 32K x 16 queries: 287 us in one, 308 in two; x 33: 551 and 331).
// Counting what an item's beginning costs evens the parts out: 4,103 queries from 0, whose first query tiles have a key tile or two,
// take 200 us with 0 units, 168 with 1, 154 with 2, 156 with 3; 64 rows x 5 queries of a window 35 us with 0, 31 with 1, 37 with 2.
constexpr int EX_LEAD = 2, EX_LEAD_FEW = 1;
struct Shape {
    int qt, rows, parts, threads, lead;   // queries and rows a tile, parts of the work, threads a CTA, ExPlan::lead
};
// blocks: sub-blocks of a quantized layer, over all rows
Shape shape_of(int64_t max_qlen, int sms, int64_t blocks) {
    if (max_qlen <= (blocks > 1024 ? 8 : 6)) return Shape{8, 32, sms, 512, EX_LEAD_FEW};
    if (max_qlen <= 32) return Shape{32, 128, sms / 4 > 0 ? sms / 4 : 1, 4 * 128, EX_LEAD};
    return Shape{64, 256, sms / 4 > 0 ? sms / 4 : 1, 5 * 128, EX_LEAD};
}

int64_t up256(int64_t x) { return (x + 255) & ~(int64_t)255; }

struct Layout {
    int64_t items, part_off, item_off, ml_off, o_off, bytes;
};
Layout layout(int64_t R, int64_t T, const Shape& s) {
    Layout l;
    l.items = T / s.qt + R;     // sum of ceil(queries / tile) over the rows
    l.part_off = up256(4 * (1 + (int64_t)s.parts));     // after the status word and, where CTAs plan for themselves, theirs
    l.item_off = up256(l.part_off + s.parts * (int64_t)sizeof(ExPart));
    l.ml_off = up256(l.item_off + l.items * (int64_t)sizeof(ExItem));
    const int64_t slots = 2 * (int64_t)s.parts * HEADS * s.rows;
    l.o_off = up256(l.ml_off + slots * 8);
    l.bytes = up256(l.o_off + slots * DIM * 4);
    return l;
}

// A launch that, if early, may start while the kernel before it in the stream still runs (it waits where it reads its results).
template <typename... A>
cudaError_t launch_early(bool early, void (*kernel)(A...), dim3 grid, int threads, size_t smem, cudaStream_t st, const A&... args) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = early ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Tensor maps of a quantized layer.  Copies start at column 0, or at a head's 32 bytes of a row.
int make_maps(const ExtendArgs& a, ExMaps& m) {
    PFN_cuTensorMapEncodeTiled encode = nullptr;
    const int rc = tensor_map_encoder(encode);
    if (rc) return rc;
    const bool quant = !a.P.win && a.P.nqmax;
    const int64_t rows = quant ? a.P.qpool_bytes / 128 : 128;
    if (rows < 128 || rows > 0x7fffffffLL || a.npos > 0x7fffffffLL) {
        set_error("kv800_extend: the quant pool must hold between 16 KB and 2^31 x 128 bytes, the tables fewer than 2^31 rows");
        return KV800_ERR_ARG;
    }
    cuuint32_t es[2] = {1, 1};
    auto make = [&](CUtensorMap* t, CUtensorMapDataType type, const void* base, cuuint64_t cols, cuuint64_t bytes, cuuint64_t n,
                    cuuint32_t width, cuuint32_t box, CUtensorMapSwizzle sw) {
        cuuint64_t dims[2] = {cols, n}, strides[1] = {bytes};
        cuuint32_t b[2] = {width, box};
        return encode(t, type, 2, const_cast<void*>(base), dims, strides, b, es, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    };
    if ((quant && (!make(&m.head, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.P.qpool, 128, 128, rows, 32, 128, CU_TENSOR_MAP_SWIZZLE_32B) ||
                   !make(&m.rows, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.P.qpool, 128, 128, rows, 128, 64, CU_TENSOR_MAP_SWIZZLE_128B) ||
                   !make(&m.scales, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.P.qpool, 128, 128, rows, 128, 16, CU_TENSOR_MAP_SWIZZLE_NONE))) ||
        !make(&m.cos, CU_TENSOR_MAP_DATA_TYPE_UINT16, a.cos_t, 32, 64, a.npos, 32, 128, CU_TENSOR_MAP_SWIZZLE_64B) ||
        !make(&m.sin, CU_TENSOR_MAP_DATA_TYPE_UINT16, a.sin_t, 32, 64, a.npos, 32, 128, CU_TENSOR_MAP_SWIZZLE_64B)) {
        set_error("kv800_extend: cuTensorMapEncodeTiled failed");
        return KV800_ERR_CUDA;
    }
    return KV800_OK;
}

template <auto KERNEL, int ROWS, typename... M>
int launch(int ctas, int smem, const ExtendArgs& a, const ExPlan& pl, int threads, cudaStream_t st, const M&... maps) {
    static std::atomic<int> done[MAX_DEV];
    int dev = 0;
    int rc = cuda_status(cudaGetDevice(&dev), "kv800_extend device");
    if (rc) return rc;
    if (dev < 0 || dev >= MAX_DEV || !done[dev].load(std::memory_order_acquire)) {
        rc = cuda_status(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
                         "kv800_extend smem attribute");
        if (rc) return rc;
        if (dev >= 0 && dev < MAX_DEV) done[dev].store(1, std::memory_order_release);
    }
    if (!a.own) {
        extend_plan<<<1, 1024, 0, st>>>(a, pl);
        rc = cuda_status(cudaGetLastError(), "kv800_extend plan");
    }
    if (!rc) rc = cuda_status(launch_early(!a.own, KERNEL, dim3((unsigned)ctas), threads, smem, st, a, pl, maps...), "kv800_extend launch");
    if (!rc && pl.parts > 1)
        rc = cuda_status(launch_early(true, extend_join<ROWS>, dim3((unsigned)(pl.parts - 1), HEADS, ROWS / EX_JOIN), EX_JOIN * 32, 0, st, a, pl),
                         "kv800_extend join");
    return rc;
}
}  // namespace

extern "C" int64_t kv800_extend_workspace_size(int64_t R, int64_t T, int64_t max_qlen) {
    if (R < 0 || T < 0 || max_qlen < 0) return -1;
    const int64_t x = layout(R, T, shape_of(max_qlen, sm_count(), 0)).bytes, y = layout(R, T, shape_of(max_qlen, sm_count(), 1 << 20)).bytes;
    return x > y ? x : y;
}

extern "C" int kv800_extend(const kv800_paged* P, const uint16_t* q, const int32_t* query_start_loc, int64_t R,
                            int64_t T, int64_t max_qlen, const uint16_t* cos_t, const uint16_t* sin_t, int64_t npos,
                            uint16_t* out, void* workspace, int64_t workspace_bytes, void* stream) {
    if (R < 0 || T < 0 || max_qlen < 0 || npos < 0) {
        set_error("kv800_extend: negative R, T, max_qlen or npos");
        return KV800_ERR_ARG;
    }
    if (R > (1 << 20) || T > 0x7fffffffLL) {
        set_error("kv800_extend: at most 2^20 rows and 2^31 - 1 tokens");
        return KV800_ERR_RANGE;
    }
    if (T == 0) return KV800_OK;
    if (!q || !out || (R && !query_start_loc) || (cos_t == nullptr) != (sin_t == nullptr) || (cos_t && npos < 1)) {
        set_error("kv800_extend: null q, out or query_start_loc, one of cos_t / sin_t without the other, or empty tables");
        return KV800_ERR_ARG;
    }
    if (!P || !P->epool || !P->eoff || !P->N || !P->NQ || P->ebs <= 0 || P->ebs > 0x7fffffffLL || P->eoff_stride <= 0 ||
        P->win < 0 || P->nsink < 0 || P->nqmax < 0) {
        set_error("kv800_extend: null Paged record / epool / eoff / N / NQ, ebs outside [1, 2^31), eoff_stride <= 0, or a "
                  "negative win / nsink / nqmax");
        return KV800_ERR_ARG;
    }
    if (P->win == 0 && P->nqmax > 0 && (!P->qpool || !P->boff || P->boff_stride <= 0 || !cos_t ||
                                        (reinterpret_cast<uintptr_t>(P->qpool) & 15u))) {
        set_error("kv800_extend: quantized layer with nqmax > 0 needs qpool (16-byte aligned), boff and the rotation tables");
        return KV800_ERR_ARG;
    }
    if (P->win && P->sk && (!P->sv || !P->skoff || !P->svoff)) {
        set_error("kv800_extend: sinks need sk, sv, skoff and svoff");
        return KV800_ERR_ARG;
    }
    if (((reinterpret_cast<uintptr_t>(P->epool) | reinterpret_cast<uintptr_t>(P->sk) | reinterpret_cast<uintptr_t>(P->sv) |
          reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(cos_t) |
          reinterpret_cast<uintptr_t>(sin_t)) & 15u) || (P->e_hs | P->e_ts | P->e_v) & 7) {
        set_error("kv800_extend: q, out, the tables and the pools must start 16-byte aligned, and e_hs / e_ts / e_v be "
                  "multiples of 8 elements");
        return KV800_ERR_ARG;
    }
    const int64_t need = kv800_extend_workspace_size(R, T, max_qlen);
    if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u)) {
        set_error("kv800_extend: workspace of %lld bytes needed (256-byte aligned), got %lld", (long long)need,
                  (long long)workspace_bytes);
        return workspace && workspace_bytes < need ? KV800_ERR_RANGE : KV800_ERR_ARG;
    }
    ExtendArgs a{*P, q, query_start_loc, (int)R, T, max_qlen, cos_t, sin_t, npos, out, (int*)workspace, 0};
    // positions are below 2^31 - 1, so that no larger window hides and no larger count of sinks shows a key more
    if (a.P.win > 0x7fffffffLL) a.P.win = 0x7fffffffLL;
    if (a.P.nsink > 0x7fffffffLL) a.P.nsink = 0x7fffffffLL;
    const Shape sh = shape_of(max_qlen, sm_count(), P->win ? 0 : P->nqmax < (1 << 20) ? P->nqmax * R : 1 << 20);
    a.own = sh.rows == 32 && R <= sh.threads && sh.parts > 1;     // extend_few plans for itself: a row a thread
    const Layout l = layout(R, T, sh);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    ExPlan pl{reinterpret_cast<ExPart*>(ws + l.part_off), reinterpret_cast<ExItem*>(ws + l.item_off),
              reinterpret_cast<float2*>(ws + l.ml_off), reinterpret_cast<float*>(ws + l.o_off), l.items, sh.qt, sh.parts, sh.lead};
    cudaStream_t st = as_stream(stream);
    ExMaps maps;
    if (cos_t && (sh.rows > 32 || (!P->win && P->nqmax))) {      // extend_few takes exact tiles' rotation as it goes
        const int rc = make_maps(a, maps);
        if (rc) return rc;
    }
    const int ctas = sh.parts * HEADS;
    if (sh.rows == 32) {
        // a tile's scores cost by the column: 64 rows x 5 queries of 32K take 467 us in 20, 483 in 24
        constexpr int smem = EfSmem::BYTES;
        if (max_qlen <= 4) return launch<extend_few<16>, 32>(sh.parts, smem, a, pl, sh.threads, st, maps);
        if (max_qlen == 5) return launch<extend_few<20>, 32>(sh.parts, smem, a, pl, sh.threads, st, maps);
        if (max_qlen == 6) return launch<extend_few<24>, 32>(sh.parts, smem, a, pl, sh.threads, st, maps);
        if (max_qlen == 7) return launch<extend_few<28>, 32>(sh.parts, smem, a, pl, sh.threads, st, maps);
        return launch<extend_few<32>, 32>(sh.parts, smem, a, pl, sh.threads, st, maps);
    }
    if (sh.rows == 128) return launch<extend_tc<1>, 128>(ctas, ExSmem<1>::BYTES, a, pl, sh.threads, st, maps);
    return launch<extend_tc<2>, 256>(ctas, ExSmem<2>::BYTES, a, pl, sh.threads, st, maps);
}
