// Attention of many new rows on the 5th-generation tensor cores: packed
// prompts (fp16 keys and values by TMA) and chunks over the paged FP8 cache
// (pages widened to fp16 by converter warps).
//
// Rows of the MMA are (token, query head of one kv head), TOK = 128 / G
// tokens x G heads, so each key tile serves all heads that share it.  A work
// item is one (sequence, kv head, block of 2 TOK tokens): two 128-row tiles
// t = 0, 1 that run against the same 128-key tiles, one's softmax beside the
// other's products.  Per key tile and row tile
//   S = Q K^T        tcgen05.mma, 128 x 128 x 64, fp32 in TMEM
//   P = exp2(c S - m) one thread per row: its 128 scores in registers, running
//                    reference m and sum l in fp32, P rounded to fp16 (the MMA
//                    operand) and written to TMEM
//   O += P V         tcgen05.mma with P from TMEM, 128 x 64 x 128, fp32 in TMEM
// The reference m follows the row's maximum only when that has grown by more
// than 2^8 since (SV_GROWTH), so O is rescaled seldom (P stays within fp16's
// range).  Over pages P also carries the page's value scale, in units of the
// row's largest (SV_UNIT0).
//
// A row tile's softmax gives its S back once the scores are in registers, so
// the next scores come while it works and the kernel runs at the softmax's
// pace.  With head_dim 64 the exponentials alone (128 x 128 of them at 16 a
// clock: 1024 clocks) take twice the products' 512.  Measured on B200, 32 query
// and 8 kv heads: one prompt of 16384 tokens 1.275 ms, 862 TFLOP/s (back to
// back, under the 1 kW power cap, 1.39 to 1.41 ms) of the 1648 that a library
// matrix product reaches (the exponentials' bound is 1150 at 1.9 GHz); 12
// prompts of up to 1500 tokens 110 us; over pages, 4 chunks of 1024 tokens
// behind 8192: 469 us, 621 TFLOP/s.  At 4096 tokens the exponential unit is
// busy 60 % and the tensor pipe 30 % of the time, and the 8 softmax warps issue
// on 41 % of the clocks: two warps a scheduler do not hide the TMEM loads' and
// each other's latencies.  Replacing exponentials by polynomials on the FMA
// pipes therefore gained nothing (1/8 to 1/2 of them).
//
// The row blocks' key tiles of all sequences are laid end to end, and each CTA
// takes an equal share of that line (or, where items are short, the items that
// begin in it).  An item that is cut is joined by k_serve_combine from at most
// two partial results per CTA.
//
// Masked places: scores are replaced, not added to.  A value that is no number
// would pass a weight of zero (0 * NaN), so in tiles where some row masks some
// key such values are set to zero in shared memory and noted by (column, first
// key); the epilogue adds them to the rows that do attend them.
#pragma once
#include <cuda.h>
#include "serve_line.cuh"

#define SV_KT 128        // keys per tile
#define SV_FST 4         // paged: stages of FP8 tiles (two pages' keys and values)
#define SV_F_BYTES (4 * SERVE_PAGE_HEAD)
#define SV_SC 16         // slots of the pages' scales (more tiles than can be in flight)
#define SV_TILE_BYTES (SV_KT * CUINF_HD * 2)
#define SV_TMEM_COLS 512
#define SV_P_COL 256     // S of row tile t at 128 t, P at 256 + 64 t, O at 384 + 64 t
#define SV_O_COL 384

// An item, or the part of it that falls to this CTA.
struct SvItem {
    int s, h, qb, nqb;  // sequence, kv head, row block of nqb
    SvSeq q;
    int t0, tb, te, n;  // first token of the block; key tiles [tb, te) of n
    int u;              // the item's units
    long long left;     // units from its beginning to the end of the CTA's share
};

struct SvSmem {
    uint64_t q_full[2], q_empty[2], k_full[4], k_empty[4], v_full[4], v_empty[4], v_ok[4], f_full[SV_FST], f_empty[SV_FST];
    uint64_t s_full[2], s_free[2], p_full[2], o_full[2], o_free[2], epi[2], conv, done;
    uint32_t tmem;
    int abort_;
    alignas(16) float sc[SV_SC][4];  // (read by float4) FP8: K scale of the tile's two pages (negative: absent), V scales
    int kind[SV_FST][2];  // FP8: what the tile's two groups are (SV_PAGE ...)
    int bad[2][3][CUINF_HD];  // by segment parity: first key whose value is +inf, -inf, NaN
    int any_bad[2];
    SvShare share;
    int h, qb;  // the item in which the share begins, and its units before that
    long long off;
    SvItem item[4];  // of segment seg, modulo 4 (published by q_full; n = 0: no more)
};
static constexpr size_t SV_Q_BYTES = 2 * SV_TILE_BYTES;  // both row tiles of an item
enum { SV_PAGE = 0, SV_TAIL = 1, SV_NONE = 2 };  // a page, the fp16 tail, no keys
// (packed: 4 stages of K and V; paged: 2 of each, and 4 of FP8 tiles, which are asked for ahead: waiting for each
// tile's pages in turn, the chunks above took 716 us)
static constexpr size_t SV_SMEM_BYTES = 1024 + 2 * SV_Q_BYTES + 8 * (size_t)SV_TILE_BYTES + sizeof(SvSmem);
static_assert(SV_FST * SV_F_BYTES == 4 * SV_TILE_BYTES, "the same shared memory for both kernels");

// ---- packed fp32 pairs ----
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// ---- tcgen05 ----
__device__ __forceinline__ void sv_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void sv_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void sv_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_u32(bar))
                 : "memory");
}
// Shared-memory descriptor, 128-byte swizzle, 8-row groups 1024 bytes apart:
// a K-major operand (rows of 64 values), and equally V [key][64], an MN-major
// operand whose one 64-wide atom spans the head.  Its low word moves with the
// address (in units of 16 bytes), its high word is constant.
__device__ __forceinline__ uint32_t sv_desc_lo(uint32_t addr) { return (addr >> 4) | (1u << 16); }
#define SV_DESC_HI ((1024u >> 4) | (1u << 14) | (2u << 29))
__device__ __forceinline__ void sv_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 x, y;\n setp.ne.b32 p, %4, 0;\n mov.b64 x, {%1, %5};\n mov.b64 y, {%2, %5};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(SV_DESC_HI)
        : "memory");
}
__device__ __forceinline__ void sv_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 y;\n setp.ne.b32 p, %4, 0;\n mov.b64 y, {%2, %5};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(SV_DESC_HI)
        : "memory");
}
__device__ __forceinline__ bool sv_elect() {
    uint32_t r;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r != 0;
}
// fp16 operands, fp32 accumulate, M = 128; bit 16: B is MN-major
#define SV_IDESC_QK ((1u << 4) | ((uint32_t)(SV_KT >> 3) << 17) | (8u << 24))
#define SV_IDESC_PV ((1u << 4) | (1u << 16) | ((uint32_t)(CUINF_HD >> 3) << 17) | (8u << 24))

#define SV_R8(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), \
                    "=r"(r[o + 6]), "=r"(r[o + 7])
#define SV_I8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), \
                    "r"(r[o + 6]), "r"(r[o + 7])
__device__ __forceinline__ void sv_ld32(uint32_t t, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        : SV_R8(r, 0), SV_R8(r, 8), SV_R8(r, 16), SV_R8(r, 24)
        : "r"(t));
}
__device__ __forceinline__ void sv_ld16(uint32_t t, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
        : SV_R8(r, 0), SV_R8(r, 8)
        : "r"(t));
}
__device__ __forceinline__ void sv_st16(uint32_t t, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};\n" ::
            SV_I8(r, 0),
        SV_I8(r, 8), "r"(t)
        : "memory");
}
__device__ __forceinline__ void sv_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void sv_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void sv_tma_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];\n" ::"r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

// ---------------------------------------------------------------------------
// the line of key tiles
// ---------------------------------------------------------------------------
// (its unit is a key; see sv_head_units)
// first key tile of a part that begins x units into an item of n tiles and u units
__device__ __forceinline__ int sv_cut(long long x, int u, int n) {
    return x >= u ? n : min(n, (int)max(0ll, x - SV_OVH + SV_KT / 2) / SV_KT);
}

// The CTA's share and the item in which it begins (all threads call).
template <int KIND>
__device__ void sv_start(const AttnArgs& A, SvSmem* S, int tq, int n_ctas, int beside) {
    sv_share<KIND>(A, &S->share, blockIdx.x, n_ctas, beside,
                   [&](const SvSeq& q) { return sv_head_units(q, tq) * A.nkv; });
    if (threadIdx.x == 0 && S->share.left > 0) {
        SvSeq q;
        sv_seq<KIND>(A, S->share.s, q, false);
        const long long per = sv_head_units(q, tq);
        const int h = (int)(S->share.rem / per);
        const long long rem = S->share.rem - h * per;
        int lo = 0, hi = (q.c + tq - 1) / tq;  // the block: prefix(lo) <= rem < prefix(hi)
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (sv_prefix(q, tq, mid) <= rem)
                lo = mid;
            else
                hi = mid;
        }
        S->h = h;
        S->qb = lo;
        S->off = rem - sv_prefix(q, tq, lo);
    }
    __syncthreads();
}

// Walks the items of the CTA's share (the lane that copies Q; the other roles
// read the items from a ring).
// left: units from the item's beginning to the share's end.
__device__ __forceinline__ void sv_item(SvItem& w, int tq, int split, long long off) {
    const int t0 = w.qb * tq, keys = sv_keys(w.q, min(t0 + tq, w.q.c)), n = (keys + SV_KT - 1) / SV_KT;
    const int u = keys + SV_OVH;
    w.t0 = t0, w.n = n, w.u = u;
    w.tb = split ? sv_cut(off, u, n) : 0;
    w.te = split ? sv_cut(w.left, u, n) : n;
}
template <int KIND>
__device__ __forceinline__ void sv_next(const AttnArgs& A, SvItem& w, int tq, int split) {
    w.left -= w.u;
    if (w.left <= 0) return;
    if (++w.qb >= w.nqb) {
        w.qb = 0;
        if (++w.h >= A.nkv) {
            w.h = 0;
            SvSeq q;
            int s = w.s;
            do s++;
            while (s < A.rows.n_seqs && !sv_seq<KIND>(A, s, q, false));
            if (s >= A.rows.n_seqs) {
                w.left = 0;
                return;
            }
            w.s = s, w.q = q;
            w.nqb = (q.c + tq - 1) / tq;
        }
    }
    sv_item(w, tq, split, 0);
    if (w.te == 0) w.left = 0;  // the share ends before the item's first tile
}
template <int KIND>
__device__ __forceinline__ void sv_first(const AttnArgs& A, const SvSmem* S, SvItem& w, int tq, int split) {
    w.s = S->share.s, w.h = S->h, w.qb = S->qb, w.left = S->share.left;
    if (w.left <= 0) return;
    const long long off = S->off;
    w.left += off;
    SvSeq q;
    sv_seq<KIND>(A, w.s, q, false);
    w.q = q;
    w.nqb = (q.c + tq - 1) / tq;
    sv_item(w, tq, split, off);
    // nothing of this item: its last tile is before the share, or (uncut) it belongs to the share in which it begins
    if (split ? w.tb == w.te : off > 0) sv_next<KIND>(A, w, tq, split);
}

// ---------------------------------------------------------------------------
// roles
// ---------------------------------------------------------------------------
// Does some row of the block mask some key of the tile?
__device__ __forceinline__ bool sv_masked(const SvSeq& q, int t0, int tile) {
    return (tile + 1) * SV_KT > q.p0 + t0 + 1;
}

template <bool PAGED>
struct SvCfg {
    // softmax warps 0-7; packed: 8 TMA, 9 and 10 MMA, 11 value check;
    // paged: 8-11 converters, 12 Q by TMA, 13 and 14 MMA (15 idle)
    static constexpr int KIND = PAGED ? SV_MANY : SV_PACKED;
    static constexpr int WARPS = PAGED ? 16 : 12;
    static constexpr int MMA_WARP = PAGED ? 13 : 9;
    static constexpr int Q_WARP = PAGED ? 12 : 8;
    static constexpr int KST = PAGED ? 2 : 4;  // K and V stages
    // registers: 512 x 128 = 256 x 200 + 256 x 56; 384 x 168 = 256 x 208 + 128 x 88
    static constexpr int REG_HI = PAGED ? 200 : 208;
    static constexpr int REG_LO = PAGED ? 56 : 88;
};

// ---- paged: pages widened to fp16 tiles by four warps ----
// Value `half` of key `key`, column d, of an item (notes `par`): if it is no number it is noted and becomes zero.
__device__ __forceinline__ void sv_note(SvSmem* S, int par, __half* p, int key, int d) {
    const float f = __half2float(*p);
    if (isfinite(f)) return;
    *p = __float2half_rn(0.f);
    atomicMin(&S->bad[par][isnan(f) ? 2 : f > 0.f ? 0 : 1][d], key);
    S->any_bad[par] = 1;
}
// output column d of a row at `pos` with the values that are no numbers
__device__ __forceinline__ float sv_with_bad(const SvSmem* S, int par, int d, int pos, float x) {
    if (S->bad[par][0][d] <= pos) x += INFINITY;
    if (S->bad[par][1][d] <= pos) x -= INFINITY;
    return S->bad[par][2][d] <= pos ? NAN : x;
}
// place of column d of row r in a 128-byte-swizzled tile of 64-value rows
__device__ __forceinline__ __half* sv_at(unsigned char* tile, int r, int d) {
    return reinterpret_cast<__half*>(tile + r * 128 + (((d >> 3) ^ (r & 7)) << 4)) + (d & 7);
}
__device__ __forceinline__ uint32_t sv_sticky(uint32_t x, uint32_t h) { return hfma2_u(h, 0, x); }  // 0 * x is NaN
__device__ __forceinline__ bool sv_stuck(uint32_t x) {                                                // or 0
    const __half2 y = *reinterpret_cast<const __half2*>(&x);
    return __hisnan(y.x) || __hisnan(y.y);
}
struct SvConv {
    SvSmem* S;
    int tid;
    // Widens a page's block (chunk u = tid + 128 i of its 256: row u / 4, 16 values from 16 (u % 4)) to rows 64 g..
    // of the tile.
    __device__ __forceinline__ void page(unsigned char* dst, int g, const unsigned char* src) const {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int u = tid + 128 * i, r = 64 * g + (u >> 2), c = 2 * (u & 3);
            const uint4 x = *reinterpret_cast<const uint4*>(src + 16 * u);
            unsigned char* row = dst + r * 128;
            *reinterpret_cast<uint4*>(row + ((c ^ (r & 7)) << 4)) =
                make_uint4(sv_e4m3x2(x.x), sv_e4m3x2(x.x >> 16), sv_e4m3x2(x.y), sv_e4m3x2(x.y >> 16));
            *reinterpret_cast<uint4*>(row + (((c + 1) ^ (r & 7)) << 4)) =
                make_uint4(sv_e4m3x2(x.z), sv_e4m3x2(x.z >> 16), sv_e4m3x2(x.w), sv_e4m3x2(x.w >> 16));
        }
    }
    // The fp16 tail's first `rest` rows (chunk u = tid + 128 i of 512: row u / 8, 8 values), zeros behind them.
    __device__ __forceinline__ void tail(unsigned char* dst, int g, const __half* src, int rest) const {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int u = tid + 128 * i, r = u >> 3, c = u & 7, rr = 64 * g + r;
            uint4 x = make_uint4(0, 0, 0, 0);
            if (r < rest) x = *reinterpret_cast<const uint4*>(src + r * CUINF_HD + c * 8);
            *reinterpret_cast<uint4*>(dst + rr * 128 + ((c ^ (rr & 7)) << 4)) = x;
        }
    }
    __device__ __forceinline__ void group(unsigned char* dst, int g, int kind, const unsigned char* src, const __half* tl,
                                          int rest) const {
        if (kind == SV_PAGE)
            page(dst, g, src);
        else
            tail(dst, g, tl, kind == SV_TAIL ? rest : 0);
    }
    // This thread's values of the tail once more, times a power of two.
    __device__ __forceinline__ void raise(unsigned char* dst, int g, float up) const {
        const __half2 f = __float2half2_rn(up);
#pragma unroll 1
        for (int i = 0; i < 4; i++) {
            const int u = tid + 128 * i, r = 64 * g + (u >> 3);
            uint4* p = reinterpret_cast<uint4*>(dst + r * 128 + (((u & 7) ^ (r & 7)) << 4));
            uint4 x = *p;
            __half2* e = reinterpret_cast<__half2*>(&x);
#pragma unroll
            for (int j = 0; j < 4; j++) e[j] = __hmul2(e[j], f);
            *p = x;
        }
    }
    // In tiles with masked places, this thread's 32 values of the group once more: is one no number?
    __device__ __forceinline__ void note(unsigned char* dst, int g, int kind, int par, int key0) const {
        const bool pg = kind == SV_PAGE;
#pragma unroll 1
        for (int i = 0; i < 4; i++) {  // its four 16-byte chunks of the tile
            const int u = tid + 128 * (pg ? i >> 1 : i), r = 64 * g + (pg ? u >> 2 : u >> 3);
            const int c = pg ? 2 * (u & 3) + (i & 1) : u & 7;
            const uint4 x = *reinterpret_cast<const uint4*>(dst + r * 128 + ((c ^ (r & 7)) << 4));
            if (!sv_stuck(sv_sticky(sv_sticky(sv_sticky(sv_sticky(0, x.x), x.y), x.z), x.w))) continue;
#pragma unroll 1
            for (int e = 0; e < 8; e++) sv_note(S, par, sv_at(dst, r, 8 * c + e), key0 + r, 8 * c + e);
        }
    }
};
// Four warps widen the FP8 tiles that the copying warp asks for.
__device__ __forceinline__ void sv_convert(const AttnArgs& A, SvSmem* S, unsigned char* Ks, unsigned char* Vs,
                                           const unsigned char* Fs, int tid) {
    constexpr int KST = SvCfg<true>::KST;
    const int lane = tid & 31, warp = tid >> 5;
    const SvConv cv = {S, tid};
    uint32_t seg = 0, kt = 0;
    bool ok = true;
    for (; ok; seg++) {
        const int par = seg & 1;
        if (!(ok = sv_wait_all(&S->q_full[par], (seg >> 1) & 1, &S->abort_))) break;
        const SvItem& w = S->item[seg & 3];
        if (w.n == 0) break;
        if (lane == 0) mbar_arrive(&S->q_empty[par]);
        // this parity's notes were last read two segments ago
        if (seg >= 2 && !(ok = sv_wait_all(&S->epi[par], ((seg >> 1) - 1) & 1, &S->abort_))) break;
        if (warp == 0) {
            for (int u = lane; u < 3 * CUINF_HD; u += 32) (&S->bad[par][0][0])[u] = 0x7fffffff;
            if (lane == 0) S->any_bad[par] = 0;
        }
        __threadfence_block();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S->conv);
        if (!(ok = sv_wait_all(&S->conv, seg & 1, &S->abort_))) break;

        const size_t tail = ((size_t)w.s * A.nkv + w.h) * SERVE_PAGE_HEAD;
        const int tb = w.tb, te = w.te, rest = w.q.kv % SERVE_PAGE, first_masked = (w.q.p0 + w.t0 + 1) >> 7;
        for (int i = tb; i < te; i++, kt++) {
            const uint32_t st = kt % KST, ph = ((kt / KST) & 1) ^ 1, fs = kt % SV_FST;
            const unsigned char* f = Fs + fs * SV_F_BYTES;  // keys of both groups, then values
            unsigned char *kd = Ks + st * SV_TILE_BYTES, *vd = Vs + st * SV_TILE_BYTES;
            if (!(ok = sv_wait_all(&S->f_full[fs], (kt / SV_FST) & 1, &S->abort_))) break;
            const int kind[2] = {S->kind[fs][0], S->kind[fs][1]};
            if (!(ok = sv_wait_all(&S->k_empty[st], ph, &S->abort_))) break;
#pragma unroll
            for (int g = 0; g < 2; g++) cv.group(kd, g, kind[g], f + g * SERVE_PAGE_HEAD, A.kv.ktail + tail, rest);
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&S->k_full[st]);
            if (!(ok = sv_wait_all(&S->v_empty[st], ph, &S->abort_))) break;
#pragma unroll
            for (int g = 0; g < 2; g++) {
                cv.group(vd, g, kind[g], f + (2 + g) * SERVE_PAGE_HEAD, A.kv.vtail + tail, rest);
                if (i >= first_masked) cv.note(vd, g, kind[g], par, i * SV_KT);
            }
            if (kind[1] == SV_TAIL) cv.raise(vd, 1, sv_inverse(S->sc[kt % SV_SC][3]));
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __threadfence_block();
            __syncwarp();
            if (lane == 0) mbar_arrive(&S->v_full[st]), mbar_arrive(&S->f_empty[fs]);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&S->epi[par]);
    }
}
// The scale of a tail's values beside a page: 2^-k where 2^k, at most 2^15, takes the largest of its `rows` rows below
// 2^15.  The tail's rows are times 2^k in shared memory.  (With a scale of 1 the page's weights, in units of that
// scale, would lose what values below 1/448 leave of them.)  All lanes of a warp call.
__device__ __forceinline__ float sv_tail_scale(const __half* src, int rows, int lane) {
    uint32_t mx = 0;  // of two halves' bits; infinities and NaN pass by
#pragma unroll 8
    for (int u = lane; u < rows * (CUINF_HD / 8); u += 32) {
        const uint4 x = *reinterpret_cast<const uint4*>(src + 8 * u);
        const uint32_t w[4] = {x.x & 0x7fff7fffu, x.y & 0x7fff7fffu, x.z & 0x7fff7fffu, x.w & 0x7fff7fffu};
#pragma unroll
        for (int j = 0; j < 4; j++) mx = __vmaxu2(mx, w[j] & __vcmpltu2(w[j], 0x7c007c00u));
    }
    const uint32_t e = __reduce_max_sync(0xffffffffu, max(mx & 0xffffu, mx >> 16)) >> 10;  // its exponent, biased by 15
    return __uint_as_float((127u - min(29u - min(e, 29u), 15u)) << 23);
}
// The tiles of an item, two pages each, by the copying warp; kt: tiles so far.  Lane l has the page index and the
// scales of group l of 16 tiles.
__device__ __forceinline__ bool sv_pages(const AttnArgs& A, SvSmem* S, const SvItem& w, unsigned char* Fs, uint32_t& kt,
                                         int lane) {
    const int ng = w.q.kv / SERVE_PAGE, te = w.te, rest = w.q.kv % SERVE_PAGE;
    const size_t tail = ((size_t)w.s * A.nkv + w.h) * SERVE_PAGE_HEAD;
    if (te == w.n)  // the tail's lines, here and by the converters read at once where they are needed
        for (int r = lane; r < rest; r += 32) {
            prefetch_l2(A.kv.vtail + tail + r * CUINF_HD);
            prefetch_l2(A.kv.ktail + tail + r * CUINF_HD);
        }
    for (int c = w.tb; c < te; c += 16) {
        const int g = 2 * c + lane;
        int kind = g < ng ? SV_PAGE : g == ng && w.q.kv % SERVE_PAGE ? SV_TAIL : SV_NONE;
        size_t blk = 0;
        float ks = 1.f, vs = 1.f;
        if (kind == SV_PAGE && g < 2 * te) {
            const int page = __ldg(A.kv.table + (size_t)w.s * A.kv.width + g);
            if (page >= 0 && page < A.kv.n_pages) {
                blk = (size_t)page * A.nkv + w.h;
                ks = __half2float(__ldg(A.kv.kps + blk)), vs = __half2float(__ldg(A.kv.vps + blk));
            } else {
                atomicOr(A.err, SERVE_ERR_PAGE);
                kind = SV_NONE, ks = -1.f;
            }
        }
        const int n = min(16, te - c);
        for (int i = 0; i < n; i++, kt++) {
            const uint32_t fs = kt % SV_FST;
            if (!sv_wait_all(&S->f_empty[fs], ((kt / SV_FST) & 1) ^ 1, &S->abort_)) return false;
            const bool mine = lane >> 1 == i;
            if (2 * (c + i) + 1 == ng && rest) {  // a page and the tail
                const float scale = sv_tail_scale(A.kv.vtail + tail, rest, lane);
                if (mine && kind == SV_TAIL) vs = scale;
            }
            if (mine) {
                S->sc[kt % SV_SC][lane & 1] = ks, S->sc[kt % SV_SC][2 + (lane & 1)] = vs;
                S->kind[fs][lane & 1] = kind;
            }
            const uint32_t pages = __popc(__ballot_sync(0xffffffffu, mine && kind == SV_PAGE));
            __syncwarp();  // scales and kinds before the arrival (a vote does not order memory)
            if (lane == 0) {
                if (pages)
                    mbar_arrive_expect_tx(&S->f_full[fs], pages * 2 * SERVE_PAGE_HEAD);
                else
                    mbar_arrive(&S->f_full[fs]);
            }
            __syncwarp();
            if (mine && kind == SV_PAGE) {
                unsigned char* dst = Fs + fs * SV_F_BYTES + (lane & 1) * SERVE_PAGE_HEAD;
                tma_load_1d(dst, A.kv.kp8 + blk * SERVE_PAGE_HEAD, SERVE_PAGE_HEAD, &S->f_full[fs]);
                tma_load_1d(dst + 2 * SERVE_PAGE_HEAD, A.kv.vp8 + blk * SERVE_PAGE_HEAD, SERVE_PAGE_HEAD, &S->f_full[fs]);
            }
        }
    }
    return true;
}

template <bool PAGED>
__global__ void __launch_bounds__(SvCfg<PAGED>::WARPS * 32, 1)
    k_serve_attn(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                 const __grid_constant__ CUtensorMap vmap, const AttnArgs A, const int split, const int beside,
                 const SvWs W) {
    using C = SvCfg<PAGED>;
    extern __shared__ __align__(1024) unsigned char sv_raw[];
    unsigned char* sm = sv_raw + ((1024 - (smem_u32(sv_raw) & 1023)) & 1023);
    unsigned char* Qs = sm;
    unsigned char* Ks = Qs + 2 * SV_Q_BYTES;
    constexpr int KST = C::KST;
    unsigned char* Vs = Ks + KST * SV_TILE_BYTES;
    unsigned char* Fs = Vs + KST * SV_TILE_BYTES;  // (paged)
    SvSmem* S = reinterpret_cast<SvSmem*>(Ks + 8 * SV_TILE_BYTES);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = A.nh / A.nkv, TOK = 128 / G, tq = 2 * TOK;

    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(&S->q_full[i], 1);
            // the last scores of both row tiles, and every role's warps once they have seen the item (so that no
            // phase of q_full goes by unseen)
            mbar_init(&S->q_empty[i], 2 + 8 + (PAGED ? 4 : 1));
            mbar_init(&S->s_full[i], 1), mbar_init(&S->s_free[i], 4), mbar_init(&S->p_full[i], 4);
            mbar_init(&S->o_full[i], 1), mbar_init(&S->o_free[i], 4), mbar_init(&S->epi[i], PAGED ? 12 : 9);
            S->any_bad[i] = 0;
        }
        for (int i = 0; i < SV_FST; i++) mbar_init(&S->f_full[i], 1), mbar_init(&S->f_empty[i], 4);
        for (int i = 0; i < KST; i++) {
            mbar_init(&S->k_full[i], PAGED ? 4 : 1), mbar_init(&S->k_empty[i], 2);
            mbar_init(&S->v_full[i], PAGED ? 4 : 1), mbar_init(&S->v_empty[i], 2);
            mbar_init(&S->v_ok[i], 1);
        }
        mbar_init(&S->conv, 4);
        mbar_init(&S->done, 2);
        S->abort_ = 0;
    }
    if (warp == C::MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&S->tmem)),
                     "r"(SV_TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
        // not before: a dependent kernel that allocates TMEM would hold it and wait for this one to end
        pdl_trigger();
    }
    if (split && tid < 2) W.part[blockIdx.x * 2 + tid].valid = 0;
    sv_start<C::KIND>(A, S, tq, gridDim.x, PAGED && beside);
    sv_fence_before();
    __syncthreads();
    sv_fence_after();
    const uint32_t tmem = S->tmem;

    if (warp < 8) {
        // ---- softmax and epilogue: one thread per row of row tile t ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(C::REG_HI));
        const int t = warp >> 2, row = tid & 127;
        const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t o_addr = lane_base + SV_O_COL + t * CUINF_HD;
        const float c2 = A.scale * SV_LOG2E;  // scores in powers of two
        const uint32_t s_addr = lane_base + t * 128, p_addr = lane_base + SV_P_COL + t * 64;
        const int row_t = row / G, row_h = row - row_t * G;  // the row's token and head in the row tile
        uint32_t ops = 0, tiles = 0, seg = 0;
        bool ok = true;
        for (; ok; seg++) {
            if (!(ok = sv_wait_all(&S->q_full[seg & 1], (seg >> 1) & 1, &S->abort_))) break;
            const SvItem& w = S->item[seg & 3];
            if (w.n == 0) break;
            if (lane == 0) mbar_arrive(&S->q_empty[seg & 1]);
            const bool act1 = w.t0 + TOK < w.q.c;
            // all who arrive at a segment's epi barrier have seen the one before of the same parity complete
            if (seg >= 2 && !(ok = sv_wait_all(&S->epi[seg & 1], ((seg >> 1) - 1) & 1, &S->abort_))) break;
            if (t == 1 && !act1) {
                tiles += w.te - w.tb;
                __syncwarp();
                if (lane == 0) mbar_arrive(&S->epi[seg & 1]);
                continue;
            }
            const int tok = w.t0 + t * TOK + row_t;
            const bool live_row = row < TOK * G && tok < w.q.c;
            const int pos = live_row ? w.q.p0 + tok : -1;
            float m = -INFINITY, per_unit = SV_UNIT0;
            uint64_t l2[2] = {0, 0};  // four partial sums
            const int tb = w.tb, te = w.te;
            const int first_masked = (w.q.p0 + w.t0 + t * TOK + 1) >> 7;  // from here some row masks some key
            for (int i = tb; i < te; i++, ops++, tiles++) {
                // (a wait that gave up ends the loop after the tile, for all lanes alike)
                ok = sv_wait(&S->s_full[t], ops & 1, &S->abort_);
                __syncwarp();  // lanes leave a wait one by one; TMEM accesses take the whole warp
                sv_fence_after();
                uint32_t sr[128];
                float* s = reinterpret_cast<float*>(sr);
                sv_ld32(s_addr, sr), sv_ld32(s_addr + 32, sr + 32);
                float kc[2] = {c2, c2}, vc[2] = {1.f, 1.f};
                bool masked = i >= first_masked, gone[2] = {false, false};
                if (PAGED) {
                    const float4 sc = *reinterpret_cast<const float4*>(S->sc[tiles % SV_SC]);
                    kc[0] = c2 * sc.x, kc[1] = c2 * sc.y;
                    vc[0] = sc.z, vc[1] = sc.w;
                    gone[0] = sc.x < 0.f, gone[1] = sc.y < 0.f;
                    masked |= gone[0] | gone[1];
                }
                sv_wait_ld();
                sv_ld32(s_addr + 64, sr + 64), sv_ld32(s_addr + 96, sr + 96);
                const int lim = pos - i * SV_KT;  // last key of the tile that the row attends
                float mx[2];
#pragma unroll
                for (int g = 0; g < 2; g++) {
                    if (g == 1) {
                        sv_wait_ld();
                        sv_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&S->s_free[t]);  // the next scores may come while these are worked on
                    }
                    if (masked) {
                        const int last = gone[g] ? -1 : lim;
#pragma unroll
                        for (int j = 64 * g; j < 64 * g + 64; j++) s[j] = j <= last ? s[j] : -INFINITY;
                        if (PAGED) {
                            // a page's scale that is no number reaches only rows that attend the page
                            if (last < 64 * g) kc[g] = c2, vc[g] = 0.f;
                            if (kc[g] == 0.f) kc[g] = 1e-30f;  // a page of zeros: -inf * 0 is no number
                        }
                    }
                    float a[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) a[j] = s[64 * g + j];
#pragma unroll
                    for (int j = 8; j < 64; j++) a[j & 7] = fmaxf(a[j & 7], s[64 * g + j]);
                    mx[g] = fmaxf(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])), fmaxf(fmaxf(a[4], a[5]), fmaxf(a[6], a[7]))) *
                            kc[g];
                }
                const float x = fmaxf(mx[0], mx[1]);
                // the last product has read P and written O
                if (i > tb) {
                    ok &= sv_wait(&S->o_full[t], (ops - 1) & 1, &S->abort_);
                    __syncwarp();
                    sv_fence_after();
                }
                if (i == tb && !PAGED) {
                    m = x;
                } else if (i == tb ||
                           __any_sync(0xffffffffu, x > m + SV_GROWTH ||
                                                       (PAGED && fmaxf(vc[0], vc[1]) * per_unit >= SV_UNIT_TOP))) {
                    // rare: the reference follows the maximum (and the unit the scales), sum and O with it; each row for
                    // itself, so that its bits do not go by the others of the warp, which may be nobody's
                    const float mn = x > m + SV_GROWTH ? x : m;
                    float f = m == -INFINITY ? 0.f : sv_exp2(m - mn);
                    m = mn;
#pragma unroll
                    for (int e = 0; e < 2; e++) l2[e] = f2_mul(l2[e], f2_pack(f, f));
                    if (PAGED) {
                        const float v = fmaxf(sv_in_units(vc[0], per_unit), sv_in_units(vc[1], per_unit));
                        const float step = v >= SV_UNIT_TOP ? sv_unit_step(v) : 1.f;
                        per_unit *= step, f *= step;
                    }
#pragma unroll 1
                    for (uint32_t j = i == tb ? CUINF_HD : 0; j < CUINF_HD; j += 16) {
                        uint32_t o[16];
                        sv_ld16(o_addr + j, o);
                        sv_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        sv_st16(o_addr + j, o);
                    }
                }
                const float ref = m == -INFINITY ? 0.f : m;
                const uint64_t nm = f2_pack(-ref, -ref);
                if (PAGED) vc[0] *= per_unit, vc[1] *= per_unit;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int g = j >> 1;
                    const uint64_t cc = f2_pack(kc[g], kc[g]), vv = f2_pack(vc[g], vc[g]);
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        uint64_t y = f2_fma(f2_pack(s[32 * j + 2 * e], s[32 * j + 2 * e + 1]), cc, nm);
                        float y0, y1;
                        f2_unpack(y, y0, y1);
                        y0 = sv_exp2(y0), y1 = sv_exp2(y1);
                        y = f2_pack(y0, y1);
                        l2[e & 1] = f2_add(l2[e & 1], y);
                        if (PAGED) f2_unpack(f2_mul(y, vv), y0, y1);
                        pk[e] = sv_pack_h2(y0, y1);
                    }
                    sv_st16(p_addr + 16 * j, pk);
                }
                sv_wait_st();
                sv_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&S->p_full[t]);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
            }
            if (!ok) break;
            // ---- epilogue of the item (or of the CTA's part of it) ----
            if (!(ok = sv_wait_all(&S->o_full[t], (ops - 1) & 1, &S->abort_))) break;
            sv_fence_after();
            float la, lb;
            f2_unpack(f2_add(l2[0], l2[1]), la, lb);
            const float l = la + lb;
            const float vs = PAGED ? sv_inverse(per_unit) : 1.f;
            const bool whole = w.tb == 0 && w.te == w.n, any_bad = S->any_bad[seg & 1] != 0;
            const size_t slot = (size_t)blockIdx.x * 2 + (w.tb == 0);
            const float inv = whole ? (l == 0.f ? 0.f : vs / l) : vs;
            __half* dst = A.out + ((size_t)(w.q.a + tok) * A.nh + w.h * G + row_h) * CUINF_HD;
            float* part = W.o + (slot * 256 + t * 128 + row) * CUINF_HD;
#pragma unroll 1
            for (int d0 = 0; d0 < CUINF_HD; d0 += 32) {
                uint32_t o[32];
                __syncwarp();
                sv_ld32(o_addr + d0, o);
                sv_wait_ld();
                const float* of = reinterpret_cast<const float*>(o);
                if (!live_row) continue;
                if (whole) {
#pragma unroll
                    for (int d = 0; d < 32; d += 8)
                        *reinterpret_cast<uint4*>(dst + d0 + d) =
                            make_uint4(sv_pack_h2(of[d] * inv, of[d + 1] * inv), sv_pack_h2(of[d + 2] * inv, of[d + 3] * inv),
                                       sv_pack_h2(of[d + 4] * inv, of[d + 5] * inv), sv_pack_h2(of[d + 6] * inv, of[d + 7] * inv));
                } else {
#pragma unroll
                    for (int d = 0; d < 32; d += 4)
                        *reinterpret_cast<float4*>(part + d0 + d) =
                            make_float4(of[d] * inv, of[d + 1] * inv, of[d + 2] * inv, of[d + 3] * inv);
                }
            }
            if (any_bad && live_row) {  // rare: the row once more, where it has gone
#pragma unroll 1
                for (int d = 0; d < CUINF_HD; d++) {
                    if (whole)
                        dst[d] = __float2half_rn(sv_with_bad(S, seg & 1, d, pos, __half2float(dst[d])));
                    else
                        part[d] = sv_with_bad(S, seg & 1, d, pos, part[d]);
                }
            }
            sv_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&S->o_free[t]);
            if (!whole) {
                if (live_row) reinterpret_cast<float2*>(W.ml)[slot * 256 + t * 128 + row] = make_float2(m, l);
                if (t == 0 && row == 0) {
                    SvPart p;
                    p.valid = 1, p.last = w.te == w.n, p.row0 = w.q.a + w.t0, p.tokens = min(tq, w.q.c - w.t0);
                    p.h = w.h;
                    W.part[slot] = p;
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&S->epi[seg & 1]);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(C::REG_LO));
        if (warp == C::Q_WARP) {
            // ---- the walk; Q (and, packed, K and V) by TMA ----
            SvItem w;  // (lane 0's)
            uint32_t seg = 0, kt = 0, nq = 0, nk = 0, nv = 0;  // copies issued
            if (lane == 0) sv_first<C::KIND>(A, S, w, tq, split);
            bool ok = true;
            for (; ok; seg++) {
                const uint32_t qsl = seg & 1;
                bool more = false;
                if (lane == 0) {
                    ok = sv_wait(&S->q_empty[qsl], ((seg >> 1) & 1) ^ 1, &S->abort_);
                    more = ok && w.left > 0;
                    if (more) {
                        S->item[seg & 3] = w;
                        const int nt = w.t0 + TOK < w.q.c ? 2 : 1;
                        mbar_arrive_expect_tx(&S->q_full[qsl], (uint32_t)(TOK * G * 128) * nt);
                        for (int t = 0; t < nt; t++)
                            sv_tma_3d(Qs + qsl * SV_Q_BYTES + t * SV_TILE_BYTES, &qmap, 0, w.h * G,
                                      w.q.a + w.t0 + t * TOK, &S->q_full[qsl]);
                        nq = seg + 1;
                    } else if (ok) {
                        S->item[seg & 3].n = 0;
                        mbar_arrive(&S->q_full[qsl]);
                    }
                }
                if constexpr (PAGED) {
                    if (!__shfl_sync(0xffffffffu, (int)more, 0)) break;
                    __syncwarp();
                    ok = sv_pages(A, S, S->item[seg & 3], Fs, kt, lane);
                } else {
                    if (!more) break;  // (lane 0 alone goes on)
                    for (int i = w.tb; i < w.te; i++, kt++) {
                        const uint32_t st = kt % KST, ph = ((kt / KST) & 1) ^ 1;
                        if (!(ok = sv_wait(&S->k_empty[st], ph, &S->abort_))) break;
                        mbar_arrive_expect_tx(&S->k_full[st], SV_TILE_BYTES);
                        sv_tma_3d(Ks + st * SV_TILE_BYTES, &kmap, 0, w.h, w.q.a + i * SV_KT, &S->k_full[st]);
                        nk++;
                        if (!(ok = sv_wait(&S->v_empty[st], ph, &S->abort_))) break;
                        mbar_arrive_expect_tx(&S->v_full[st], SV_TILE_BYTES);
                        sv_tma_3d(Vs + st * SV_TILE_BYTES, &vmap, 0, w.h, w.q.a + i * SV_KT, &S->v_full[st]);
                        nv++;
                    }
                }
                if (lane == 0) sv_next<C::KIND>(A, w, tq, split);
            }
            // every copy is waited for by those who use it; after an abort, what is in flight has to land before the
            // CTA can exit
            if (lane == 0 && *(volatile int*)&S->abort_) {
                for (uint32_t k = nq < 2 ? 0 : nq - 2; k < nq; k++) sv_drain(&S->q_full[k & 1], (k >> 1) & 1);
                for (uint32_t k = nk < KST ? 0 : nk - KST; k < nk; k++) sv_drain(&S->k_full[k % KST], (k / KST) & 1);
                for (uint32_t k = nv < KST ? 0 : nv - KST; k < nv; k++) sv_drain(&S->v_full[k % KST], (k / KST) & 1);
                if (PAGED)
                    for (uint32_t k = kt < SV_FST ? 0 : kt - SV_FST; k < kt; k++)
                        sv_drain(&S->f_full[k % SV_FST], (k / SV_FST) & 1);
            }
            __syncwarp();
        } else if (warp == C::MMA_WARP || warp == C::MMA_WARP + 1) {
            // ---- products of row tile t: S of the next key tile as soon as the scores are read, then O of this
            // one.  A warp for each row tile (one warp's instructions for both were the kernel's pace); all lanes
            // walk, one issues ----
            const uint32_t t = warp - C::MMA_WARP;
            const bool leader = sv_elect();
            const uint32_t q_lo = sv_desc_lo(smem_u32(Qs) + t * SV_TILE_BYTES), k_lo = sv_desc_lo(smem_u32(Ks));
            const uint32_t v_lo = sv_desc_lo(smem_u32(Vs));
            const uint32_t d_s = tmem + t * 128, d_p = tmem + SV_P_COL + t * 64, d_o = tmem + SV_O_COL + t * CUINF_HD;
            uint32_t seg = 0, kt = 0, vt = 0;
            uint32_t nq = 0, np = 0, segs = 0;  // products of this row tile so far; segments in which it is active
            bool ok = true;
            auto scores = [&](uint32_t qa) -> bool {
                const uint32_t st = kt % KST;
                bool fine = sv_wait(&S->k_full[st], (kt / KST) & 1, &S->abort_);
                if (nq > 0) fine &= sv_wait(&S->s_free[t], (nq - 1) & 1, &S->abort_);
                sv_fence_after();
                if (leader) {
                    const uint32_t ka = k_lo + st * (SV_TILE_BYTES >> 4);
                    sv_mma_ss(d_s, qa, ka, SV_IDESC_QK, 0);
#pragma unroll
                    for (int k = 1; k < CUINF_HD / 16; k++) sv_mma_ss(d_s, qa + 2 * k, ka + 2 * k, SV_IDESC_QK, 1);
                    sv_commit(&S->s_full[t]);
                    sv_commit(&S->k_empty[st]);
                }
                nq++, kt++;
                return fine;
            };
            for (; ok; seg++) {
                if (!(ok = sv_wait_all(&S->q_full[seg & 1], (seg >> 1) & 1, &S->abort_))) break;
                const SvItem& w = S->item[seg & 3];
                if (w.n == 0) break;
                const int nt = w.te - w.tb;
                if (t == 1 && w.t0 + TOK >= w.q.c) {  // the block has one row tile: only let the stages go
                    for (int i = 0; ok && i < nt; i++, kt++, vt++) {
                        const uint32_t st = kt % KST;
                        if (!(ok = sv_wait_all(&S->k_full[st], (kt / KST) & 1, &S->abort_))) break;
                        if (leader) mbar_arrive(&S->k_empty[st]);
                        if (!(ok = sv_wait_all(&S->v_full[st], (vt / KST) & 1, &S->abort_))) break;
                        if (leader) mbar_arrive(&S->v_empty[st]);
                    }
                    if (leader) mbar_arrive(&S->q_empty[seg & 1]);
                    continue;
                }
                const uint32_t qa = q_lo + (seg & 1) * (SV_Q_BYTES >> 4);
                ok = scores(qa);
                for (int i = 0; i < nt; i++) {
                    if (i + 1 < nt) ok &= scores(qa);
                    if (leader && i == max(nt - 2, 0)) sv_commit(&S->q_empty[seg & 1]);  // the last scores are under way
                    const uint32_t st = vt % KST;
                    ok &= sv_wait(&S->v_full[st], (vt / KST) & 1, &S->abort_);
                    if (!PAGED) ok &= sv_wait(&S->v_ok[st], (vt / KST) & 1, &S->abort_);
                    if (i == 0 && segs > 0) ok &= sv_wait(&S->o_free[t], (segs - 1) & 1, &S->abort_);
                    ok &= sv_wait(&S->p_full[t], np & 1, &S->abort_);
                    sv_fence_after();
                    if (leader) {
                        const uint32_t va = v_lo + st * (SV_TILE_BYTES >> 4);
                        sv_mma_ts(d_o, d_p, va, SV_IDESC_PV, i > 0);
#pragma unroll
                        for (int k = 1; k < SV_KT / 16; k++)
                            sv_mma_ts(d_o, d_p + 8 * k, va + k * (16 * 128 >> 4), SV_IDESC_PV, 1);
                        sv_commit(&S->o_full[t]);
                        sv_commit(&S->v_empty[st]);
                    }
                    np++, vt++;
                    if (!(ok = __all_sync(0xffffffffu, ok))) break;
                }
                segs++;
            }
            if (leader) sv_commit(&S->done);
            __syncwarp();
        } else if (!PAGED && warp == 11) {
            // ---- values that are no numbers, in tiles with masked places ----
            uint32_t seg = 0, kt = 0;
            bool ok = true;
            for (; ok; seg++) {
                if (!(ok = sv_wait_all(&S->q_full[seg & 1], (seg >> 1) & 1, &S->abort_))) break;
                const SvItem& w = S->item[seg & 3];
                if (w.n == 0) break;
                if (lane == 0) mbar_arrive(&S->q_empty[seg & 1]);
                // this parity's notes were last read two segments ago
                if (seg >= 2 && !(ok = sv_wait_all(&S->epi[seg & 1], ((seg >> 1) - 1) & 1, &S->abort_))) break;
                for (int u = lane; u < 3 * CUINF_HD; u += 32) (&S->bad[seg & 1][0][0])[u] = 0x7fffffff;
                if (lane == 0) S->any_bad[seg & 1] = 0;
                __syncwarp();
                for (int i = w.tb; i < w.te; i++, kt++) {
                    const uint32_t st = kt % KST;
                    // every tile passes here, so that no phase of v_full goes unseen
                    if (!(ok = sv_wait_all(&S->v_full[st], (kt / KST) & 1, &S->abort_))) break;
                    if (!sv_masked(w.q, w.t0, i)) {
                        if (lane == 0) mbar_arrive(&S->v_ok[st]);
                        continue;
                    }
                    unsigned char* V = Vs + st * SV_TILE_BYTES;
                    uint32_t nan = 0;
#pragma unroll 8
                    for (int u = lane; u < SV_TILE_BYTES / 16; u += 32) {
                        const uint4 v = *reinterpret_cast<const uint4*>(V + u * 16);
                        nan = sv_sticky(sv_sticky(sv_sticky(sv_sticky(nan, v.x), v.y), v.z), v.w);
                    }
                    if (__any_sync(0xffffffffu, sv_stuck(nan))) {
#pragma unroll 1
                        for (int u = lane; u < SV_KT * CUINF_HD; u += 32)
                            sv_note(S, seg & 1, sv_at(V, u >> 6, u & 63), i * SV_KT + (u >> 6), u & 63);
                        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                    }
                    __threadfence_block();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&S->v_ok[st]);
                }
                if (!ok) break;
                if (lane == 0) mbar_arrive(&S->epi[seg & 1]);
            }
            __syncwarp();
        } else if (PAGED && warp < 12) {
            if constexpr (PAGED) sv_convert(A, S, Ks, Vs, Fs, tid - 256);
        }
    }
    sv_fence_before();
    __syncthreads();
    if (warp == C::MMA_WARP) {
        sv_fence_after();
        if (lane == 0) {
            sv_drain(&S->done, 0);
            if (S->abort_) atomicOr(A.err, SERVE_ERR_WAIT);
        }
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(SV_TMEM_COLS)
                     : "memory");
    }
}
