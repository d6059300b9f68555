// The line of work units that the serving attention kernels share out: one CTA
// per SM, each takes an equal contiguous share of all sequences' units laid
// end to end (key tiles of the tensor-core kernel, pages of the single-token
// kernel), so the load is even whatever the lengths are.  An item that a
// share's end cuts is joined from partial results by k_serve_combine.
#pragma once
#include "serve.cuh"

// ---- waits (bounded; the first that gives up raises the CTA's abort word, and
// the kernel's end reports it) ----
// A try that fails has taken between 90 ns and 4 us, so this many end after
// 0.2 to 8 s.  Counting them keeps the 30 waits of a kernel small: its roles run
// side by side from one instruction cache.
#define SV_TRIES 2000000u
__device__ __forceinline__ bool sv_wait(uint64_t* bar, uint32_t parity, int* abort_) {
#pragma unroll 1
    for (uint32_t k = 0; k < SV_TRIES; k++) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*(volatile int*)abort_) return false;
    }
    *(volatile int*)abort_ = 1;
    return false;
}
// The same by all lanes of a warp, with one answer (lanes that part after an
// abort would wait for each other in the warp's next vote or TMEM access).
__device__ __forceinline__ bool sv_wait_all(uint64_t* bar, uint32_t parity, int* abort_) {
    return __all_sync(0xffffffffu, sv_wait(bar, parity, abort_));
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;\n" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
// Before the CTA ends: a phase that copies or products in flight complete.
__device__ __forceinline__ void sv_drain(uint64_t* bar, uint32_t parity) {
#pragma unroll 1
    for (uint32_t k = 0; k < SV_TRIES; k++)
        if (mbar_try_wait(bar, parity)) return;
}

// ---- arithmetic ----
#define SV_LOG2E 1.44269504088896340736f
__device__ __forceinline__ float sv_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];\n" ::"l"(p)); }
__device__ __forceinline__ uint32_t sv_pack_h2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t sv_e4m3x2(uint32_t two) {  // low 16 bits: two codes -> two halves, exact
    uint32_t r;
    asm("{\n .reg .b16 t;\n cvt.u16.u32 t, %1;\n cvt.rn.f16x2.e4m3x2 %0, t;\n}\n" : "=r"(r) : "r"(two));
    return r;
}
// The reference that scores are taken from follows a row's maximum when that
// has grown by more than 2^SV_GROWTH (fp16 holds such weights), so that sums and
// O are seldom rescaled.
#define SV_GROWTH 8.f
// FP8: a weight meets the values' codes times the page's value scale over the
// row's unit, and O counts in that unit.  The unit is a power of two, 1/64 to
// 1/128 of the largest scale among the pages that the row has attended, so
// weights stay below 2^8 * 128 = 2^15 and, of the pages that count, in fp16's
// normal range down to 2^-20 of the reference (2^-31 is the last that is not
// lost), whatever the values' size.  A page of larger scale raises the unit in
// the rare path that follows the maximum; O, in fp32, loses nothing by a power
// of two.  An infinite scale does not count: its page's values are no numbers.
#define SV_UNIT0 2147483648.f  // 1 / unit at first: below 2^-24, the smallest scale, so the first page sets it
#define SV_UNIT_TOP 128.f
__device__ __forceinline__ float sv_in_units(float scale, float per_unit) {
    return scale <= 65504.f ? scale * per_unit : 0.f;
}
__device__ __forceinline__ float sv_inverse(float power_of_two) {
    return __uint_as_float((254u << 23) - __float_as_uint(power_of_two));
}
// 64 over the power of two at or below x
__device__ __forceinline__ float sv_unit_step(float x) {
    return __uint_as_float(((127u + 127u + 6u) << 23) - (__float_as_uint(x) & 0x7f800000u));
}

// ---- sequences ----
enum { SV_PACKED = 0, SV_MANY = 1, SV_FEW = 2 };  // packed prompts; paged, many or few rows of a sequence
// One sequence as a kernel sees it: c new rows from row a on, the first at
// position p0 of kv keys.
struct SvSeq {
    int a, c, p0, kv;
};
// False: nothing for this kernel (empty, out of range, or the other kernel's).
template <int KIND>
__device__ __forceinline__ bool sv_seq(const AttnArgs& A, int s, SvSeq& q, bool report) {
    int b;
    bool fine = packed_range(A.rows, s, q.a, b);
    q.c = fine ? b - q.a : 0;
    if (KIND != SV_PACKED) {
        q.kv = __ldg(A.kv_lens + s);
        if (q.c > 0 && (q.kv < 0 || q.kv / SERVE_PAGE > A.kv.width || q.c > A.max_q)) {
            fine = false;
            q.c = 0;
        }
        const bool few = (long long)q.c * (A.nh / A.nkv) <= SERVE_FEW_ROWS;
        if (few != (KIND == SV_FEW)) q.c = 0;
    } else {
        q.kv = q.c;
    }
    q.p0 = q.kv - q.c;
    if (report && !fine) atomicOr(A.err, SERVE_ERR_RANGE);
    return q.c > 0;
}

// Many rows: the line's unit is a key, and an item (a block of tq rows of one
// kv head) takes
// the keys of its last row and SV_OVH more for its beginning and end, so the
// blocks of a sequence form an arithmetic series and a place on the line is
// found without a table.  Cuts fall on key tiles (sv_cut).
#define SV_OVH 256
__device__ __forceinline__ int sv_keys(const SvSeq& q, int end) {  // rows before `end`; a row without a key still
    return max(1, q.p0 + end);                                     // has its zeros written
}
// units of the first k blocks of a head (none of them the last)
__device__ __forceinline__ long long sv_prefix(const SvSeq& q, int tq, int k) {
    const int z = q.p0 < 0 ? min(k, -q.p0 / tq) : 0;  // blocks without a key
    return (long long)k * SV_OVH + z + (long long)(k - z) * q.p0 +
           (long long)tq * (((long long)k * (k + 1) - (long long)z * (z + 1)) / 2);
}
__device__ __forceinline__ long long sv_head_units(const SvSeq& q, int tq) {
    return sv_prefix(q, tq, (q.c + tq - 1) / tq - 1) + sv_keys(q, q.c) + SV_OVH;
}
#define FW_TAIL 32  // tail tokens of a unit
// Few rows: units of one kv head (at least one: rows without a key still become zero)
__device__ __forceinline__ int fw_units(const SvSeq& q) {
    return max(1, q.kv / SERVE_PAGE + (q.kv % SERVE_PAGE + FW_TAIL - 1) / FW_TAIL);
}

// The CTA's share of the line (equal parts, to a unit).
struct SvShare {
    int s;           // sequence in which it begins
    long long rem;   // units of that sequence before it
    long long left;  // its units (0: nothing to do)
    long long scan[32];
    long long work[32][2];
};
// Where a call's sequences are of both kinds, the two kernels run beside one
// another, each on a part of the SMs that follows its work (`beside`), and the
// CTAs behind that end at once: the single tokens' kernel is bound by memory and
// latencies, the chunks' by the softmax.  128 single tokens at contexts to 4096
// beside a chunk of 64 tokens take 107 us (one kernel after the other: 130), 24
// beside a chunk of 515 80 (86).  In keys of the chunks' kernel a unit of the
// other takes SV_FEW_COST and an item's end SV_FEW_END units (8 instead of 14:
// 109 and 99 us; 12: 105 and 82; 18: 120 and 85).
#define SV_FEW_COST 14
#define SV_FEW_END 11
// All threads call; `units` gives a sequence's units.  One pass over the
// sequences where the CTA has a thread for each, else one for the sum and one
// for the place.
template <int KIND, class F>
__device__ __forceinline__ void sv_share(const AttnArgs& A, SvShare* S, int cta, int n_ctas, int beside, F units) {
    constexpr int OTHER = KIND == SV_FEW ? SV_MANY : SV_FEW;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nt = blockDim.x, nw = nt >> 5, n = A.rows.n_seqs;
    auto cost = [&](int kind, const SvSeq& q) {  // of one kv head
        return kind == SV_FEW ? (long long)(fw_units(q) + SV_FEW_END) * SV_FEW_COST
                              : sv_head_units(q, 2 * (128 / (A.nh / A.nkv)));
    };
    long long total = 0, beg = 0, end = 0, base = 0, mine = 0, other = 0;
    if (tid == 0) S->left = 0;
    for (int pass = n <= nt ? 1 : 0; pass < 2; pass++) {
        const bool sum = pass == 0 || n <= nt;
        for (int b = 0; b < n; b += nt) {
            const int s = b + tid;
            SvSeq q;
            long long w = 0, x, work[2] = {0, 0};
            if (s < n && sv_seq<KIND>(A, s, q, sum && cta == 0)) w = units(q);
            if (beside && sum) {
                if (w)
                    work[0] = cost(KIND, q);
                else if (s < n && sv_seq<OTHER>(A, s, q, false))
                    work[1] = cost(OTHER, q);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1)
                    for (int k = 0; k < 2; k++) work[k] += __shfl_xor_sync(0xffffffffu, work[k], o);
            }
            x = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            if (b > 0 || pass == 1) __syncthreads();
            if (lane == 31) S->scan[warp] = x, S->work[warp][0] = work[0], S->work[warp][1] = work[1];
            __syncthreads();
            long long before = 0, all = 0;
            for (int i = 0; i < nw; i++) {
                const long long y = S->scan[i];
                if (i < warp) before += y;
                all += y;
                if (beside && sum) mine += S->work[i][0], other += S->work[i][1];
            }
            if (pass == 0) {
                total += all;
                continue;
            }
            if (n <= nt) total = all;
            if (b == 0) {
                if (mine > 0 && other > 0) {  // the single tokens' CTAs: the same number in both kernels
                    const float f = (float)(KIND == SV_FEW ? mine : other) / (float)(mine + other);
                    const int few = min(max(1, (int)(f * n_ctas + 0.5f)), n_ctas - 1);
                    n_ctas = KIND == SV_FEW ? few : n_ctas - few;
                }
                const long long per = total / n_ctas, more = total - per * n_ctas;
                beg = per * cta + min((long long)cta, more);
                end = beg + per + (cta < more);
            }
            const long long lo = base + before + x - w;
            if (end > beg && beg >= lo && beg < lo + w) {
                S->s = s;
                S->rem = beg - lo;
                S->left = end - beg;
            }
            base += all;
        }
    }
    __syncthreads();
}

// ---- partial results: [CTA][2] slots of `rows` rows; slot 0: the CTA's share
// began inside the item, slot 1: it began the item and did not finish it ----
struct SvPart {
    int valid, last, row0, tokens, h, pad[3];  // first token row, tokens of the item, kv head
};
struct SvWs {
    SvPart* part;  // [ctas][2]
    float* ml;     // [ctas][2][rows][2]: reference (power of two) and sum
    float* o;      // [ctas][2][rows][64], not divided by the sum
};
static inline size_t sv_ws_bytes(int ctas, int rows) {
    return (size_t)ctas * 2 * (sizeof(SvPart) + (size_t)rows * (2 + CUINF_HD) * 4);
}
static inline SvWs sv_ws(void* p, int ctas, int rows) {
    SvWs w;
    w.o = (float*)p;
    w.ml = w.o + (size_t)ctas * 2 * rows * CUINF_HD;
    w.part = (SvPart*)(w.ml + (size_t)ctas * 2 * rows * 2);
    return w;
}

// Joins the items that were cut: CTA (i, j) takes rows of the item that CTA i
// of the attention began and did not finish; the other parts are slot 0 of the
// CTAs behind it.  j < SV_JOIN_Y (with `many`): 32 rows each of the tensor-core
// kernel's items, else the up to 16 of the single-token kernel's.  A thread
// holds 4 columns of a row and asks for SV_JOIN parts at a time: 3 or 4, for 8
// leave fewer CTAs on an SM (12 prompts of up to 1500 tokens: 115 us for 112.5),
// or 8 in a decode step, with one CTA an SM.  Where the rows are few and the parts many,
// up to 256 / (16 rows) neighbouring threads share the parts of one place.  The
// time is that of dependent loads: one part after another, the 20 parts of a
// 32768-token context took 29 us in all, shared out 20.  Fixed order: the same
// bits every time.
#define SV_JOIN_Y 8
template <bool MANY, bool FEW>
__global__ void __launch_bounds__(256, !MANY ? 1 : FEW ? 4 : 5)
    k_serve_combine(const AttnArgs A, const SvWs Wm, const SvWs Wf, const int n_ctas) {
    constexpr int SV_JOIN = !MANY ? 8 : FEW ? 4 : 3;
    pdl_wait();
    const bool few = FEW && (!MANY || blockIdx.y == SV_JOIN_Y);
    const SvWs& W = few ? Wf : Wm;
    const int rows = few ? 16 : 256, i = blockIdx.x, lane = threadIdx.x & 31;
    __shared__ unsigned char list[SERVE_MAX_CTAS];  // the CTAs that hold a part of the item (a share can be empty)
    __shared__ int n_parts;
    auto flags = [&](int k) {  // of CTA k's first slot: there, the item's last
        return k < n_ctas ? *reinterpret_cast<const int2*>(W.part + (size_t)k * 2) : make_int2(0, 0);
    };
    const SvPart p = W.part[i * 2 + 1];
    int2 x = flags(i + 1 + lane);
    if (!p.valid) return;
    if (threadIdx.x < 32) {
        int cnt = 1;
        if (lane == 0) list[0] = i;
        for (int k = i + 1;;) {
            const unsigned last = __ballot_sync(0xffffffffu, x.x && x.y);
            const unsigned there = __ballot_sync(0xffffffffu, x.x) & (last ^ (last - 1));  // up to the last (none: all)
            if (there >> lane & 1) list[cnt + __popc(there & ((1u << lane) - 1))] = k + lane;
            cnt += __popc(there);
            if (last || (k += 32) >= n_ctas) break;
            x = flags(k + lane);
        }
        if (lane == 0) n_parts = cnt;
    }
    __syncthreads();
    const int parts = n_parts;
    const int G = A.nh / A.nkv, TOK = 128 / G;
    int lg = 0;  // 2^lg threads share a place's parts
    if (few)
        while (lg < 4 && SV_JOIN << lg < parts && p.tokens * G << lg <= 8) lg++;
    const int at = threadIdx.x >> lg, c = (at & 15) * 4, part0 = threadIdx.x & ((1 << lg) - 1);
    for (int r = (few ? 0 : blockIdx.y * 32) + (at >> 4), z = 0; z < (few ? 1 : 2); z++, r += 16) {
        const int row = r & 127, tok = (r >> 7) * TOK + row / G;
        const bool live = row < TOK * G && tok < p.tokens;
        float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
        for (int k0 = part0; k0 < parts; k0 += SV_JOIN << lg) {
            float2 ml[SV_JOIN];
            float4 x[SV_JOIN];
#pragma unroll
            for (int j = 0; j < SV_JOIN; j++) {
                const int k = k0 + (j << lg);
                ml[j] = make_float2(-INFINITY, 0.f), x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (live && k < parts) {
                    const size_t slot = (size_t)list[k] * 2 + (k == 0);
                    ml[j] = reinterpret_cast<const float2*>(W.ml)[slot * rows + r];
                    x[j] = *reinterpret_cast<const float4*>(W.o + (slot * rows + r) * CUINF_HD + c);
                }
            }
            float mn = m;
#pragma unroll
            for (int j = 0; j < SV_JOIN; j++) mn = fmaxf(mn, ml[j].x);
            const float ref = mn == -INFINITY ? 0.f : mn, f0 = m == -INFINITY ? 0.f : sv_exp2(m - ref);
            l *= f0, m = mn;
#pragma unroll
            for (int d = 0; d < 4; d++) o[d] *= f0;
#pragma unroll
            for (int j = 0; j < SV_JOIN; j++) {
                const float f = ml[j].x == -INFINITY ? 0.f : sv_exp2(ml[j].x - ref);
                l += ml[j].x == -INFINITY ? ml[j].y : ml[j].y * f;  // NaN scores alone have no maximum
                o[0] += x[j].x * f, o[1] += x[j].y * f, o[2] += x[j].z * f, o[3] += x[j].w * f;
            }
        }
        for (int t = 1; t < 1 << lg; t *= 2) {
            const float m2 = __shfl_xor_sync(0xffffffffu, m, t), mn = fmaxf(m, m2), ref = mn == -INFINITY ? 0.f : mn;
            const float f = m == -INFINITY ? 0.f : sv_exp2(m - ref), f2 = m2 == -INFINITY ? 0.f : sv_exp2(m2 - ref);
            l = l * f + __shfl_xor_sync(0xffffffffu, l, t) * f2;  // (0 * NaN: NaN)
#pragma unroll
            for (int d = 0; d < 4; d++) o[d] = o[d] * f + __shfl_xor_sync(0xffffffffu, o[d], t) * f2;
            m = mn;
        }
        if (!live || part0) continue;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        *reinterpret_cast<uint2*>(A.out + ((size_t)(p.row0 + tok) * A.nh + p.h * G + row % G) * CUINF_HD + c) =
            make_uint2(sv_pack_h2(o[0] * inv, o[1] * inv), sv_pack_h2(o[2] * inv, o[3] * inv));
    }
}
