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

static __device__ unsigned g_serve_err;
static int serve_err_ptr(unsigned** p) {
    CUINF_TRY(cudaGetSymbolAddress((void**)p, g_serve_err));
    return CUINF_OK;
}

extern "C" int cuinf_paged_error(unsigned* flags) {
    REQUIRE(flags, "null pointer");
    unsigned v = 0;
    const unsigned zero = 0;
    CUINF_TRY(cudaMemcpyFromSymbol(&v, g_serve_err, sizeof(v)));
    if (v) CUINF_TRY(cudaMemcpyToSymbol(g_serve_err, &zero, sizeof(zero)));
    *flags = v;
    return CUINF_OK;
}

// ---------------------------------------------------------------------------
// append: new rows of packed sequences into pages and tails
//
// A sequence with `ctx` cached tokens and L new ones touches the 64-token
// groups ctx/64 .. (ctx+L-1)/64.  One CTA takes one (group, kv head), keys and
// values; a group that the call completes is read once (its first rows from
// the old tail, the rest from the new rows), its maximum reduced over the CTA
// and its bytes written once: 16 values of one row per thread, so a head's
// page block is one run of 256 16-byte stores.  The rows of the unfinished
// last group go to the tail; that copy is made by the CTA of the sequence's
// first group, after it has read the old tail, so that no other CTA reads what
// it overwrites.
//
// CTA -> (sequence, group) without a plan: sequence s owns the slots from
// (cu[s] + 62 s) / 64 + s on, which are at least the groups L new rows can
// touch ((L + 62) / 64 + 1).
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

__device__ __forceinline__ uint8_t serve_e4m3(float x) {
    return (uint8_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}

__global__ void __launch_bounds__(256) k_paged_append(const AppendArgs A) {
    __shared__ float red[2][8];
    const int h = blockIdx.y, tid = threadIdx.x;
    int s = -1;
    for (int b = 0; b < A.rows.n_seqs; b += 256) {
        const int i = b + tid;
        const bool mine = i < A.rows.n_seqs &&
                          append_slot(min(max(A.rows.cu[i], 0), A.rows.n_rows), i) <= (long long)blockIdx.x;
        s += __syncthreads_count(mine);
    }
    if (s < 0) return;
    int a, b;
    const int ctx = A.ctx[s];
    const bool fine = packed_range(A.rows, s, a, b) && ctx >= 0 && (long long)ctx + (b - a) < (1ll << 31);
    if (!fine) {
        if (tid == 0) atomicOr(A.err, SERVE_ERR_RANGE);
        return;
    }
    const int L = b - a, total = ctx + L, g0 = ctx / SERVE_PAGE;
    const long long gl = (long long)blockIdx.x - append_slot(a, s);
    if (L == 0 || gl > (total - 1) / SERVE_PAGE - g0) return;
    const int g = g0 + (int)gl, nkv = A.kv.nkv;
    const int r = tid >> 2, c = (tid & 3) * 16;  // this thread: 16 values of row r
    const int pos = g * SERVE_PAGE + r;
    const size_t tail = ((size_t)s * nkv + h) * SERVE_PAGE_HEAD;
    const bool whole = g < total / SERVE_PAGE;

    uint4 x[2][2];
    if (whole) {
        const __half *ks, *vs;
        if (pos < ctx) {
            ks = A.kv.ktail + tail + r * CUINF_HD + c;
            vs = A.kv.vtail + tail + r * CUINF_HD + c;
        } else {
            const size_t row = (size_t)a + (pos - ctx);
            ks = A.k + row * A.k_stride + h * CUINF_HD + c;
            vs = A.v + row * A.v_stride + h * CUINF_HD + c;
        }
        x[0][0] = *reinterpret_cast<const uint4*>(ks);
        x[0][1] = *reinterpret_cast<const uint4*>(ks + 8);
        x[1][0] = *reinterpret_cast<const uint4*>(vs);
        x[1][1] = *reinterpret_cast<const uint4*>(vs + 8);
        float mx[2];
#pragma unroll
        for (int p = 0; p < 2; p++) {
            const __half* e = reinterpret_cast<const __half*>(x[p]);
            mx[p] = 0.f;
#pragma unroll
            for (int i = 0; i < 16; i++) mx[p] = fmaxf(mx[p], fabsf(__half2float(e[i])));
            mx[p] = warp_max(mx[p]);
            if ((tid & 31) == 0) red[p][tid >> 5] = mx[p];
        }
        __syncthreads();  // also: the old tail has been read before it is overwritten below
        const int page = g < A.kv.width ? A.kv.table[(size_t)s * A.kv.width + g] : -1;
        if (page >= 0 && page < A.kv.n_pages) {
#pragma unroll
            for (int p = 0; p < 2; p++) {
                float amax = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++) amax = fmaxf(amax, red[p][i]);
                // kv_commit_group's rule: fp32 scale for the codes, fp16 in the cache
                const float sc = amax / 448.0f + 1e-12f;
                const __half* e = reinterpret_cast<const __half*>(x[p]);
                uint8_t q[16];
#pragma unroll
                for (int i = 0; i < 16; i++) q[i] = serve_e4m3(__half2float(e[i]) / sc);
                const size_t blk = (size_t)page * nkv + h;
                *reinterpret_cast<uint4*>((p ? A.kv.vp8 : A.kv.kp8) + blk * SERVE_PAGE_HEAD + r * CUINF_HD + c) =
                    *reinterpret_cast<const uint4*>(q);
                if (tid == 0) (p ? A.kv.vps : A.kv.kps)[blk] = __float2half_rn(sc);
            }
        } else if (tid == 0) {
            atomicOr(A.err, SERVE_ERR_PAGE);
        }
    }
    if (g != g0) return;
    const int last = total / SERVE_PAGE;  // the unfinished group: its new rows go to the tail
    const int tp = last * SERVE_PAGE + r;
    if (tp < total && tp >= ctx) {
        const size_t row = (size_t)a + (tp - ctx);
        const uint4* ks = reinterpret_cast<const uint4*>(A.k + row * A.k_stride + h * CUINF_HD + c);
        const uint4* vs = reinterpret_cast<const uint4*>(A.v + row * A.v_stride + h * CUINF_HD + c);
        uint4* kd = reinterpret_cast<uint4*>(A.kv.ktail + tail + r * CUINF_HD + c);
        uint4* vd = reinterpret_cast<uint4*>(A.kv.vtail + tail + r * CUINF_HD + c);
        const uint4 k0 = ks[0], k1 = ks[1], v0 = vs[0], v1 = vs[1];
        kd[0] = k0, kd[1] = k1, vd[0] = v0, vd[1] = v1;
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
    k_paged_append<<<dim3((unsigned)slots, nkv), 256, 0, ST(stream)>>>(A);
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

// One CTA per SM, at most this many: the workspace holds two partial results of each.
#define SERVE_MAX_CTAS 148
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
static int launch_many(const AttnArgs& A, bool cuts, const SvWs& W, int ctas, cudaStream_t st) {
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
    k_serve_attn<PAGED><<<ctas, SvCfg<PAGED>::WARPS * 32, SV_SMEM_BYTES, st>>>(qm, km, vm, A, cuts, W);
    return cuinf_launch_status();
}
// `beside`: a chunks' kernel of the same call runs before (its results do not matter to this one)
static int launch_few(const AttnArgs& A, bool cuts, const SvWs& W, int ctas, bool beside, cudaStream_t st) {
    CUINF_TRY(cudaFuncSetAttribute(k_serve_few, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)FW_SMEM_BYTES));
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = pdl_config(dim3(ctas), (FW_WARPS + 1) * 32, FW_SMEM_BYTES, st, attr);
    cfg.numAttrs = beside ? 1 : 0;
    CUINF_TRY(cudaLaunchKernelEx(&cfg, k_serve_few, A, (int)cuts, W));
    return cuinf_launch_status();
}
static int launch_combine(const AttnArgs& A, const SvWs& Wm, const SvWs& Wf, int ctas, bool many, bool few,
                          cudaStream_t st) {
    cudaLaunchAttribute attr[1];
    const cudaLaunchConfig_t cfg = pdl_config(dim3(ctas, (many ? SV_JOIN_Y : 0) + (few ? 1 : 0)), 256, 0, st, attr);
    CUINF_TRY(cudaLaunchKernelEx(&cfg, k_serve_combine, A, Wm, Wf, ctas, (int)many));
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
    REQUIRE(scale > 0.f && isfinite(scale), "scale must be positive and finite");
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
    if (int rc = launch_many<false>(A, cuts, W, ctas, ST(stream))) return rc;
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
    REQUIRE(scale > 0.f && isfinite(scale), "scale must be positive and finite");
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
        if (int rc = launch_many<true>(A, cuts, Wm, ctas, ST(stream))) return rc;
    if (few)
        if (int rc = launch_few(A, cuts, Wf, ctas, many, ST(stream))) return rc;
    return cuts ? launch_combine(A, Wm, Wf, ctas, many, few, ST(stream)) : CUINF_OK;
}
