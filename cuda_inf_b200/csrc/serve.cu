// Serving operators of the C ABI (include/cuinf.h): causal attention over
// packed prompts, the paged FP8 KV cache's append, and attention of new tokens
// over that cache.
#include <math.h>

#include <algorithm>
#include <mutex>

#include "serve.cuh"
#include "serve_few.cuh"
#include "serve_tc.cuh"

#define ST(s) ((cudaStream_t)(s))
#define REQUIRE(cond, msg) \
    do {                   \
        if (!(cond)) return cuinf_set_arg_error(msg); \
    } while (0)

static __device__ unsigned g_serve_err, g_serve_taken;
static int serve_err_ptr(unsigned** p) {
    CUINF_TRY(cudaGetSymbolAddress((void**)p, g_serve_err));
    return CUINF_OK;
}

// Read and cleared at once, so that a bit set meanwhile (by a call of another host thread) is kept for the next asking.
__global__ void k_take_err() { g_serve_taken = atomicExch(&g_serve_err, 0u); }

extern "C" int cuinf_paged_error(unsigned* flags) {
    REQUIRE(flags, "null pointer");
    static std::mutex mu;  // of g_serve_taken
    std::lock_guard<std::mutex> lock(mu);
    // the default stream alone would not wait for non-blocking ones
    CUINF_TRY(cudaDeviceSynchronize());
    k_take_err<<<1, 1>>>();
    if (int rc = cuinf_launch_status()) return rc;
    unsigned v = 0;
    CUINF_TRY(cudaMemcpyFromSymbol(&v, g_serve_taken, sizeof(v)));
    *flags = v;
    return CUINF_OK;
}

// ---------------------------------------------------------------------------
// append: new rows of packed sequences into pages and tails
//
// A sequence with `ctx` cached tokens and L new ones touches the 64-token
// groups ctx/64 .. (ctx+L-1)/64.  One warp takes one (group, kv head) of the
// keys or of the values: 8 KB, all asked for at once into the warp's own part
// of shared memory, so a CTA's 8 warps need no barrier, an SM has 192 KB in
// flight, and the loops over it stay small (held in registers the rows made
// 28 KB of straight code, which a CTA's one pass spent its time fetching).
// The maximum is reduced over the warp and the codes written once, a head's
// page block being one run of 4096 bytes.  Bound by HBM: 256 bytes in and 128
// out per token and head; 4 x 16384 tokens of 8 kv heads (201 MB) take 35.0 us,
// 5.75 TB/s, 88 % of a copy's rate (62 us with the rows in registers and a
// division per value).
//
// The rows of the unfinished last group go to the tail.  The warp of the
// sequence's first group copies them, after it has read the old tail, so nobody
// reads what it overwrites.
//
// CTA -> (sequence, group) without a plan: sequence s owns the slots from
// (cu[s] + 62 s) / 64 + s on, which are at least the groups L new rows can
// touch ((L + 62) / 64 + 1).  That needs ascending offsets: where they are not,
// the largest offset so far takes the place of cu[s], and a sequence that begins
// before it is skipped like one whose own offsets are out of order.
// ---------------------------------------------------------------------------
struct AppendArgs {
    const __half *k, *v;
    long long k_stride, v_stride;
    PackedRows rows;
    const int* ctx;
    PagedKV kv;
    unsigned* err;
};
__host__ __device__ __forceinline__ long long append_slot(long long row, int s) { return (row + 62ll * s) / 64 + s; }

__device__ __forceinline__ uint32_t serve_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
#define APPEND_SMEM (8 * SERVE_PAGE_HEAD * 2)
__global__ void __launch_bounds__(256, 3) k_paged_append(const AppendArgs A) {
    extern __shared__ __align__(16) unsigned char append_raw[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int s = -1, begin = 0;
    bool disorder = false;
    auto offset = [&](int i) { return min(max(A.rows.cu[i], 0), A.rows.n_rows); };
    for (int b = 0; b < A.rows.n_seqs; b += 256) {
        const int i = b + tid;
        const bool mine = i < A.rows.n_seqs && append_slot(offset(i), i) <= (long long)blockIdx.x;
        disorder |= i < A.rows.n_seqs && A.rows.cu[i] > A.rows.cu[i + 1];
        s += __syncthreads_count(mine);
    }
    if (__syncthreads_or(disorder)) {
        s = -1;
#pragma unroll 1
        for (int i = 0; i < A.rows.n_seqs; i++) {
            const int most = max(begin, offset(i));
            if (append_slot(most, i) > (long long)blockIdx.x) break;
            begin = most, s = i;
        }
    }
    if (s < 0) return;
    int a, b;
    const int ctx = A.ctx[s];
    const bool fine = packed_range(A.rows, s, a, b) && a >= begin && ctx >= 0 && (long long)ctx + (b - a) < (1ll << 31);
    if (!fine) {
        if (tid == 0) atomicOr(A.err, SERVE_ERR_RANGE);
        return;
    }
    const int L = b - a, total = ctx + L, g0 = ctx / SERVE_PAGE, nkv = A.kv.nkv;
    const long long gl = (long long)blockIdx.x - append_slot(a, s);
    const int h = blockIdx.y * 4 + (warp >> 1);
    if (L == 0 || gl > (total - 1) / SERVE_PAGE - g0 || h >= nkv) return;
    const bool val = warp & 1;  // keys or values
    const int g = g0 + (int)gl, r0 = lane >> 3, c = (lane & 7) * 8;  // this lane: 8 values of rows r0 + 4 i
    __half* tail = (val ? A.kv.vtail : A.kv.ktail) + ((size_t)s * nkv + h) * SERVE_PAGE_HEAD + c;
    const long long stride = val ? A.v_stride : A.k_stride;
    const __half* src = (val ? A.v : A.k) + (size_t)a * stride + h * CUINF_HD + c;  // token ctx
    if (g < total / SERVE_PAGE) {
        const int page = g < A.kv.width ? A.kv.table[(size_t)s * A.kv.width + g] : -1;
        // a lane reads back what it has copied itself
        uint4* mine = reinterpret_cast<uint4*>(append_raw + warp * SERVE_PAGE_HEAD * 2) + lane;
#pragma unroll 4
        for (int i = 0; i < 16; i++) {
            const int r = r0 + 4 * i, pos = g * SERVE_PAGE + r;
            const __half* from = pos < ctx ? tail + r * CUINF_HD : src + (long long)(pos - ctx) * stride;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(smem_u32(mine + 32 * i)), "l"(from) : "memory");
        }
        asm volatile("cp.async.wait_all;\n" ::: "memory");
        __half2 mx = __float2half2_rn(0.f);  // (a maximum passes NaN by)
#pragma unroll 4
        for (int i = 0; i < 16; i++) {
            const uint4 x = mine[32 * i];
            const __half2* e = reinterpret_cast<const __half2*>(&x);
#pragma unroll
            for (int j = 0; j < 4; j++) mx = __hmax2(mx, __habs2(e[j]));
        }
        const float amax = warp_max(fmaxf(__low2float(mx), __high2float(mx)));
        // kv_commit_group's rule: fp32 scale for the codes, fp16 in the cache
        const float sc = amax / 448.0f + 1e-12f;
        // x / sc rounded to nearest (the codes have to be those of the division) by two products with the rounded
        // reciprocal: q = x y, q + (x - q sc) y (Markstein, IBM J. Res. Dev. 34, 1990; no step of it underflows for
        // fp16 x).  A row that is infinite makes every quotient 0 or NaN.
        const bool finite = sc < INFINITY;
        const float y = 1.f / sc, y2 = finite ? y : 0.f, nsc = finite ? -sc : 0.f;
        if (page >= 0 && page < A.kv.n_pages) {
            const size_t blk = (size_t)page * nkv + h;
            uint8_t* dst = (val ? A.kv.vp8 : A.kv.kp8) + blk * SERVE_PAGE_HEAD + c;
#pragma unroll 2
            for (int i = 0; i < 16; i++) {
                const uint4 x = mine[32 * i];
                const __half2* e = reinterpret_cast<const __half2*>(&x);
                float q[8];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float2 f = __half22float2(e[j]);
                    q[2 * j] = f.x * y, q[2 * j + 1] = f.y * y;
                    q[2 * j] = fmaf(fmaf(q[2 * j], nsc, f.x), y2, q[2 * j]);
                    q[2 * j + 1] = fmaf(fmaf(q[2 * j + 1], nsc, f.y), y2, q[2 * j + 1]);
                }
                *reinterpret_cast<uint2*>(dst + (r0 + 4 * i) * CUINF_HD) =
                    make_uint2(serve_e4m3x2(q[0], q[1]) | serve_e4m3x2(q[2], q[3]) << 16,
                               serve_e4m3x2(q[4], q[5]) | serve_e4m3x2(q[6], q[7]) << 16);
            }
            if (lane == 0) (val ? A.kv.vps : A.kv.kps)[blk] = __float2half_rn(sc);
        } else if (lane == 0) {
            atomicOr(A.err, SERVE_ERR_PAGE);
        }
    }
    if (g != g0) return;
    __syncwarp();  // the old tail has been read
    // the unfinished group: its new rows go to the tail, asked for at once too
    const int last = total / SERVE_PAGE * SERVE_PAGE;
    if (last == total) return;
    uint4* mine = reinterpret_cast<uint4*>(append_raw + warp * SERVE_PAGE_HEAD * 2) + lane;
#pragma unroll 4
    for (int i = 0; i < 16; i++) {
        const int pos = last + r0 + 4 * i;
        if (pos < total && pos >= ctx)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(smem_u32(mine + 32 * i)),
                         "l"(src + (long long)(pos - ctx) * stride)
                         : "memory");
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
#pragma unroll 4
    for (int i = 0; i < 16; i++) {
        const int pos = last + r0 + 4 * i;
        if (pos < total && pos >= ctx) *reinterpret_cast<uint4*>(tail + (r0 + 4 * i) * CUINF_HD) = mine[32 * i];
    }
}

// ---------------------------------------------------------------------------
// entry points
// ---------------------------------------------------------------------------
static int check_rows(const void* p, int64_t stride, int heads, const char* what) {
    if (((uintptr_t)p & 15) != 0) return cuinf_set_arg_error(what);
    if (stride < (int64_t)heads * CUINF_HD || stride % 8 != 0) return cuinf_set_arg_error(what);
    return CUINF_OK;
}
#define CHECK_ROWS(p, stride, heads, name)                                                              \
    do {                                                                                                \
        const int rc_ = check_rows(p, stride, heads,                                                    \
                                   name ": 16-byte aligned, token stride a multiple of 8 elements and " \
                                        "at least heads * 64");                                         \
        if (rc_) return rc_;                                                                            \
    } while (0)
#define CHECK_HEADS(nh, nkv)                                                                       \
    REQUIRE((nh) > 0 && (nkv) > 0 && (nkv) <= 65535 && (nh) % (nkv) == 0 && (nh) / (nkv) <= 128, \
            "nh must be a multiple of nkv, at most 128 query heads per kv head")
#define CHECK_CACHE(kp8, vp8, kps, vps, ktail, vtail, table, width, n_pages)                                   \
    do {                                                                                                       \
        REQUIRE((kp8) && (vp8) && (kps) && (vps) && (ktail) && (vtail) && (table), "null pointer");            \
        REQUIRE((n_pages) > 0 && (width) > 0, "n_pages and table_width must be positive");                     \
        REQUIRE((width) <= 1 << 24, "table_width must be at most 2^24 (positions are 32 bits)");               \
        REQUIRE((((uintptr_t)(kp8) | (uintptr_t)(vp8) | (uintptr_t)(ktail) | (uintptr_t)(vtail)) & 15) == 0,   \
                "pages and tails must be 16-byte aligned");                                                    \
        REQUIRE((((uintptr_t)(kps) | (uintptr_t)(vps)) & 1) == 0 && ((uintptr_t)(table) & 3) == 0,             \
                "misaligned scales or table");                                                                 \
    } while (0)

extern "C" int cuinf_kv_paged_append(const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                                     const int* cu_seqlens, const int* ctx_lens, int n_seqs, int n_rows,
                                     const int* table, int table_width, uint8_t* kp8, uint8_t* vp8, void* kps,
                                     void* vps, int n_pages, void* ktail, void* vtail, int nkv, void* stream) {
    REQUIRE(k && v && cu_seqlens && ctx_lens, "null pointer");
    REQUIRE(n_seqs > 0 && n_rows > 0, "n_seqs and n_rows must be positive");
    CHECK_HEADS(nkv, nkv);
    CHECK_CACHE(kp8, vp8, kps, vps, ktail, vtail, table, table_width, n_pages);
    CHECK_ROWS(k, k_stride, nkv, "k");
    CHECK_ROWS(v, v_stride, nkv, "v");
    AppendArgs A;
    A.k = (const __half*)k, A.v = (const __half*)v;
    A.k_stride = k_stride, A.v_stride = v_stride;
    A.rows = {cu_seqlens, n_seqs, n_rows};
    A.ctx = ctx_lens;
    A.kv = {kp8, vp8, (__half*)kps, (__half*)vps, (__half*)ktail, (__half*)vtail, table, table_width, n_pages, nkv};
    if (int rc = serve_err_ptr(&A.err)) return rc;
    const long long slots = append_slot(n_rows, n_seqs);
    REQUIRE(slots < (1ll << 31), "too many rows");
    CUINF_TRY(cudaFuncSetAttribute(k_paged_append, cudaFuncAttributeMaxDynamicSharedMemorySize, APPEND_SMEM));
    k_paged_append<<<dim3((unsigned)slots, (nkv + 3) / 4), 256, APPEND_SMEM, ST(stream)>>>(A);
    return cuinf_launch_status();
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = (EncodeTiledFn)p;
    });
    return fn;
}
// fp16 rows [n_rows][heads][64], `stride` elements apart: boxes of bh heads x bt rows, 128-byte swizzle
static int rows_map(CUtensorMap* m, const __half* base, int64_t stride, int heads, int n_rows, int bh, int bt) {
    EncodeTiledFn fn = encode_fn();
    REQUIRE(fn, "cuTensorMapEncodeTiled unavailable");
    const cuuint64_t dims[3] = {CUINF_HD, (cuuint64_t)heads, (cuuint64_t)n_rows};
    const cuuint64_t strides[2] = {CUINF_HD * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[3] = {CUINF_HD, (cuuint32_t)bh, (cuuint32_t)bt}, one[3] = {1, 1, 1};
    const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, (void*)base, dims, strides, box, one,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    REQUIRE(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled refused the rows (stride below 2^39 elements?)");
    return CUINF_OK;
}

// Items of at most this many key tiles are not cut.
#define SERVE_WHOLE_TILES 4
static bool sv_cuts(long long most_keys) { return most_keys > SERVE_WHOLE_TILES * SV_KT; }
static int check_ws(const void* ws, size_t have, size_t need) {
    REQUIRE(need == 0 || (ws && have >= need && ((uintptr_t)ws & 15) == 0),
            "workspace: 16-byte aligned and of the size the _workspace_size call gives");
    return CUINF_OK;
}
static int num_ctas(int* n) {
    int dev = 0, sms = 0;
    CUINF_TRY(cudaGetDevice(&dev));
    CUINF_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    *n = std::min(sms, SERVE_MAX_CTAS);
    return CUINF_OK;
}

static cudaLaunchConfig_t pdl_config(dim3 grid, int threads, size_t smem, cudaStream_t st, cudaLaunchAttribute* attr) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    attr->id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr->val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
}
template <bool PAGED>
static int launch_many(const AttnArgs& A, bool cuts, const SvWs& W, int ctas, bool beside, cudaStream_t st) {
    CUtensorMap qm, km, vm;
    const int G = A.nh / A.nkv;
    if (int rc = rows_map(&qm, A.q, A.q_stride, A.nh, A.rows.n_rows, G, 128 / G)) return rc;
    km = vm = qm;
    if (!PAGED) {
        if (int rc = rows_map(&km, A.k, A.k_stride, A.nkv, A.rows.n_rows, 1, SV_KT)) return rc;
        if (int rc = rows_map(&vm, A.v, A.v_stride, A.nkv, A.rows.n_rows, 1, SV_KT)) return rc;
    }
    CUINF_TRY(cudaFuncSetAttribute(k_serve_attn<PAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   (int)SV_SMEM_BYTES));
    k_serve_attn<PAGED><<<ctas, SvCfg<PAGED>::WARPS * 32, SV_SMEM_BYTES, st>>>(qm, km, vm, A, cuts, beside, W);
    return cuinf_launch_status();
}
// `beside`: the chunks' kernel of the same call is launched before and runs beside this one (neither reads the other's
// results)
static int launch_few(const AttnArgs& A, bool cuts, const SvWs& W, int ctas, bool beside, cudaStream_t st) {
    auto* kernel = beside ? k_serve_few<true> : k_serve_few<false>;
    CUINF_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)FW_SMEM_BYTES));
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = pdl_config(dim3(ctas), (FW_WARPS + 1) * 32, FW_SMEM_BYTES, st, attr);
    cfg.numAttrs = beside ? 1 : 0;
    CUINF_TRY(cudaLaunchKernelEx(&cfg, kernel, A, (int)cuts, W));
    return cuinf_launch_status();
}
static int launch_combine(const AttnArgs& A, const SvWs& Wm, const SvWs& Wf, int ctas, bool many, bool few,
                          cudaStream_t st) {
    cudaLaunchAttribute attr[1];
    const cudaLaunchConfig_t cfg = pdl_config(dim3(ctas, (many ? SV_JOIN_Y : 0) + (few ? 1 : 0)), 256, 0, st, attr);
    auto* kernel = !few ? k_serve_combine<true, false> : many ? k_serve_combine<true, true> : k_serve_combine<false, true>;
    CUINF_TRY(cudaLaunchKernelEx(&cfg, kernel, A, Wm, Wf, ctas));
    return cuinf_launch_status();
}

extern "C" size_t cuinf_attn_varlen_workspace_size(int n_seqs, int n_rows, int nh, int nkv) {
    return sv_cuts(n_rows) ? sv_ws_bytes(SERVE_MAX_CTAS, 256) : 0;
}
extern "C" int cuinf_attn_varlen(const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                                 int64_t v_stride, const int* cu_seqlens, int n_seqs, int n_rows, float scale,
                                 void* out, int nh, int nkv, void* workspace, size_t workspace_bytes,
                                 void* stream) {
    REQUIRE(q && k && v && cu_seqlens && out, "null pointer");
    REQUIRE(n_seqs > 0 && n_rows > 0, "n_seqs and n_rows must be positive");
    REQUIRE(scale > 0.f && isfinite(scale * SV_LOG2E), "scale must be positive and finite (times log2(e) too)");
    CHECK_HEADS(nh, nkv);
    CHECK_ROWS(q, q_stride, nh, "q");
    CHECK_ROWS(k, k_stride, nkv, "k");
    CHECK_ROWS(v, v_stride, nkv, "v");
    REQUIRE(((uintptr_t)out & 15) == 0, "out must be 16-byte aligned");
    AttnArgs A = {};
    A.q = (const __half*)q, A.k = (const __half*)k, A.v = (const __half*)v;
    A.q_stride = q_stride, A.k_stride = k_stride, A.v_stride = v_stride;
    A.rows = {cu_seqlens, n_seqs, n_rows};
    A.scale = scale, A.out = (__half*)out, A.nh = nh, A.nkv = nkv;
    const bool cuts = sv_cuts(n_rows);
    if (int rc = check_ws(workspace, workspace_bytes, cuinf_attn_varlen_workspace_size(n_seqs, n_rows, nh, nkv)))
        return rc;
    if (int rc = serve_err_ptr(&A.err)) return rc;
    int ctas;
    if (int rc = num_ctas(&ctas)) return rc;
    const SvWs W = sv_ws(workspace, ctas, 256);
    if (int rc = launch_many<false>(A, cuts, W, ctas, false, ST(stream))) return rc;
    return cuts ? launch_combine(A, W, W, ctas, true, false, ST(stream)) : CUINF_OK;
}

// Which of the two kernels a paged call can need.
static bool has_many(int max_q, int nh, int nkv) { return (long long)max_q * (nh / nkv) > SERVE_FEW_ROWS; }
static bool has_few(int nh, int nkv) { return nh / nkv <= SERVE_FEW_ROWS; }

extern "C" size_t cuinf_attn_paged_workspace_size(int n_seqs, int n_rows, int max_q, int nh, int nkv,
                                                  int table_width) {
    if (nkv <= 0 || !sv_cuts(((long long)table_width + 1) * SERVE_PAGE)) return 0;
    const bool many = has_many(max_q, nh, nkv), few = has_few(nh, nkv);
    return (many ? sv_ws_bytes(SERVE_MAX_CTAS, 256) : 0) + (few ? sv_ws_bytes(SERVE_MAX_CTAS, 16) : 0);
}
extern "C" int cuinf_attn_paged(const void* q, int64_t q_stride, const int* cu_seqlens, const int* kv_lens,
                                int n_seqs, int n_rows, int max_q, const int* table, int table_width,
                                const uint8_t* kp8, const uint8_t* vp8, const void* kps, const void* vps,
                                int n_pages, const void* ktail, const void* vtail, float scale, void* out, int nh,
                                int nkv, void* workspace, size_t workspace_bytes, void* stream) {
    REQUIRE(q && cu_seqlens && kv_lens && out, "null pointer");
    REQUIRE(n_seqs > 0 && n_rows > 0, "n_seqs and n_rows must be positive");
    REQUIRE(max_q > 0, "max_q must be positive");
    REQUIRE(scale > 0.f && isfinite(scale * SV_LOG2E), "scale must be positive and finite (times log2(e) too)");
    CHECK_HEADS(nh, nkv);
    CHECK_CACHE(kp8, vp8, kps, vps, ktail, vtail, table, table_width, n_pages);
    CHECK_ROWS(q, q_stride, nh, "q");
    REQUIRE(((uintptr_t)out & 15) == 0, "out must be 16-byte aligned");
    AttnArgs A = {};
    A.q = (const __half*)q, A.q_stride = q_stride;
    A.rows = {cu_seqlens, n_seqs, n_rows};
    A.kv_lens = kv_lens, A.max_q = max_q;
    A.kv = {(uint8_t*)kp8, (uint8_t*)vp8, (__half*)kps, (__half*)vps, (__half*)ktail, (__half*)vtail,
            table, table_width, n_pages, nkv};
    A.scale = scale, A.out = (__half*)out, A.nh = nh, A.nkv = nkv;
    const bool cuts = sv_cuts(((long long)table_width + 1) * SERVE_PAGE);
    if (int rc = check_ws(workspace, workspace_bytes,
                          cuinf_attn_paged_workspace_size(n_seqs, n_rows, max_q, nh, nkv, table_width)))
        return rc;
    if (int rc = serve_err_ptr(&A.err)) return rc;
    int ctas;
    if (int rc = num_ctas(&ctas)) return rc;
    const bool many = has_many(max_q, nh, nkv), few = has_few(nh, nkv);
    const SvWs Wm = sv_ws(workspace, ctas, 256);
    const SvWs Wf = sv_ws((char*)workspace + (many && cuts ? sv_ws_bytes(ctas, 256) : 0), ctas, 16);
    if (many)
        if (int rc = launch_many<true>(A, cuts, Wm, ctas, few, ST(stream))) return rc;
    if (few)
        if (int rc = launch_few(A, cuts, Wf, ctas, many, ST(stream))) return rc;
    return cuts ? launch_combine(A, Wm, Wf, ctas, many, few, ST(stream)) : CUINF_OK;
}
