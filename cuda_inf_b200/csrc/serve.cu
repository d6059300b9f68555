// Serving operators of the C ABI (include/cuinf.h): causal attention over
// packed prompts, the paged FP8 KV cache's append, and attention of new tokens
// over that cache.
#include <math.h>

#include "serve.cuh"

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
// attention, simple form: one warp per (row, query head), one key per lane,
// running maximum and sum in fp32
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(128) k_attn_rows(const AttnArgs A) {
    __shared__ float qs[4][CUINF_HD];
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * 4 + w;
    const long long row = item / A.nh;
    const int h = (int)(item % A.nh), hk = h / (A.nh / A.nkv);
    if (row >= A.rows.n_rows) return;
    int s = -1;
    for (int b = 0; b < A.rows.n_seqs; b += 32) {
        const int i = b + lane;
        int x, y;
        if (i < A.rows.n_seqs && !packed_range(A.rows, i, x, y)) atomicOr(A.err, SERVE_ERR_RANGE);
        s += __popc(__ballot_sync(0xffffffffu, i < A.rows.n_seqs && A.rows.cu[i] <= row));
    }
    if (s < 0) return;
    int a, b;
    if (!packed_range(A.rows, s, a, b) && lane == 0) atomicOr(A.err, SERVE_ERR_RANGE);
    if (row >= b) return;  // behind the last sequence
    const int kv = A.kv_lens ? A.kv_lens[s] : b - a;
    if (A.kv_lens && (kv < 0 || kv / SERVE_PAGE > A.kv.width || b - a > A.max_q)) {
        if (lane == 0) atomicOr(A.err, SERVE_ERR_RANGE);
        return;
    }
    const int pos = kv - (b - a) + (int)(row - a);
    for (int d = lane; d < CUINF_HD; d += 32)
        qs[w][d] = __half2float(A.q[row * A.q_stride + h * CUINF_HD + d]) * A.scale;
    __syncwarp();
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int j0 = 0; j0 <= pos; j0 += 32) {
        const int j = j0 + lane;
        const __half *kr = nullptr, *vr = nullptr;
        const uint8_t *k8 = nullptr, *v8 = nullptr;
        float ks = 1.f, vs = 1.f;
        bool ok = j <= pos;
        if (!A.kv_lens) {
            kr = A.k + (size_t)(a + min(j, pos)) * A.k_stride + hk * CUINF_HD;
            vr = A.v + (size_t)(a + min(j, pos)) * A.v_stride + hk * CUINF_HD;
        } else if (j / SERVE_PAGE < kv / SERVE_PAGE) {
            const int page = A.kv.table[(size_t)s * A.kv.width + j / SERVE_PAGE];
            if (page >= 0 && page < A.kv.n_pages) {
                const size_t blk = (size_t)page * A.nkv + hk;
                k8 = A.kv.kp8 + blk * SERVE_PAGE_HEAD + (j % SERVE_PAGE) * CUINF_HD;
                v8 = A.kv.vp8 + blk * SERVE_PAGE_HEAD + (j % SERVE_PAGE) * CUINF_HD;
                ks = __half2float(A.kv.kps[blk]), vs = __half2float(A.kv.vps[blk]);
            } else {
                if (ok) atomicOr(A.err, SERVE_ERR_PAGE);
                ok = false;
            }
        } else {
            const size_t t = ((size_t)s * A.nkv + hk) * SERVE_PAGE_HEAD + (j % SERVE_PAGE) * CUINF_HD;
            kr = A.kv.ktail + t, vr = A.kv.vtail + t;
        }
        float x = 0.f;
        if (ok)
            for (int d = 0; d < CUINF_HD; d++)
                x += qs[w][d] * (kr ? __half2float(kr[d]) : ks * (float)*reinterpret_cast<const __nv_fp8_e4m3*>(k8 + d));
        x = ok ? x : -INFINITY;
        const float mn = fmaxf(m, warp_max(x));  // NaN scores pass the maximum by, and reach the sum through p
        const float ref = mn == -INFINITY ? 0.f : mn;
        const float f = __expf(m - ref);
        const float p = ok ? __expf(x - ref) : 0.f;
        l = l * f + p, o0 *= f, o1 *= f, m = mn;
        for (int t = 0; t < 32; t++) {
            const float pt = __shfl_sync(0xffffffffu, p, t);
            const float st = __shfl_sync(0xffffffffu, vs, t);
            const __half* vt = (const __half*)__shfl_sync(0xffffffffu, (unsigned long long)vr, t);
            const uint8_t* v8t = (const uint8_t*)__shfl_sync(0xffffffffu, (unsigned long long)v8, t);
            if (!__shfl_sync(0xffffffffu, (int)ok, t)) continue;
            if (vt) {
                o0 += pt * __half2float(vt[lane]), o1 += pt * __half2float(vt[lane + 32]);
            } else {
                o0 += pt * st * (float)*reinterpret_cast<const __nv_fp8_e4m3*>(v8t + lane);
                o1 += pt * st * (float)*reinterpret_cast<const __nv_fp8_e4m3*>(v8t + lane + 32);
            }
        }
    }
    l = warp_sum(l);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    __half* o = A.out + ((size_t)row * A.nh + h) * CUINF_HD;
    o[lane] = __float2half_rn(o0 * inv);
    o[lane + 32] = __float2half_rn(o1 * inv);
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

static int launch_attn(const AttnArgs& A, cudaStream_t st) {
    const long long blocks = ((long long)A.rows.n_rows * A.nh + 3) / 4;
    REQUIRE(blocks < (1ll << 31), "too many rows");
    k_attn_rows<<<(unsigned)blocks, 128, 0, st>>>(A);
    return cuinf_launch_status();
}

extern "C" size_t cuinf_attn_varlen_workspace_size(int n_seqs, int n_rows, int nh, int nkv) {
    return 0;
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
    if (int rc = serve_err_ptr(&A.err)) return rc;
    return launch_attn(A, ST(stream));
}

extern "C" size_t cuinf_attn_paged_workspace_size(int n_seqs, int n_rows, int max_q, int nh, int nkv,
                                                  int table_width) {
    return 0;
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
    if (int rc = serve_err_ptr(&A.err)) return rc;
    return launch_attn(A, ST(stream));
}
