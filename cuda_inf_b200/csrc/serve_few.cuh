// Attention of few new rows per sequence (one token, or some drafted ones: at
// most 16 rows of new tokens x query heads per kv head) over the paged cache.
//
// Bound by the pages' bytes: 8 KB of FP8 per page and kv head against 16 rows.
// A unit of the shared line is one page of one (sequence, kv head), or 32
// tokens of its fp16 tail (also 8 KB).  The last warp copies units with bulk
// copies into a ring of FW_ST stages, lane i filling stage i, each lane with
// its next unit's page index and scales already in registers; warp w takes
// units w, w + FW_WARPS, ... of the CTA's share, so a stage belongs to one warp
// and the warps meet only where an item ends, when their (m, l, O) are joined
// in shared memory.
//
// Products by mma.sync m16n8k16 with the rows as M (4 of 16 for one token and
// 4 heads per kv head; the tensor pipe has room: 64 products a page against
// 356 clocks of its HBM time per SM).  The sum over the head's dims may run in
// any order, so lane quad c takes dims 16 c .. 16 c + 15 of a key: one 16-byte
// shared load per key.  E4M3 becomes fp16 exactly; the page's key scale joins
// the scores, its value scale (in units of the row's largest, SV_UNIT0) the
// weights: one rounding of a weight to fp16.
//
// Measured on B200, 8 kv heads of 4 query heads, one token each: 64 contexts of
// 2048 tokens 40 us and of 4096 61 us (269 MB, 4.4 TB/s), 128 of up to 8191
// tokens 128 us (554 MB, 4.3 TB/s); one of 32768 18 us (33.6 MB).  From 2048
// to 4096 tokens the added bytes go at 6.3 TB/s, near the copy rate: the rest is
// a part per call (the launch, the line, the first pages' latency, the join: 8.5
// us for 63 tokens) and per item (the warps' join: the same 269 MB as 512
// contexts of 512 take 102 us, 1.7 us per further item of a CTA).  8 warps took
// 56 us for the first, 11 (what the registers allow) 53; most of the rest came of
// smaller code (128 to 83 KB).
#pragma once
#include "serve_line.cuh"

#define FW_WARPS 11        // and one that copies: 3 a scheduler, at up to 168 registers a thread
#define FW_ST 22           // stages; a multiple of FW_WARPS: a stage's phases are all seen by one warp
#define FW_UNIT 8192       // bytes of a unit: 4096 of keys, 4096 of values
#define FW_IDLE (1u << 24) // turns (of 50 clocks and more) without a free stage that end the kernel

struct FwSmem {
    uint64_t full[FW_ST], empty[FW_ST], merge, merged;
    int abort_;
    float sc[FW_ST][2];       // key scale (negative: absent), value scale
    int any_bad[3];
    int bad[3][3][CUINF_HD];  // by item, modulo 3: first key whose value is +inf, -inf, NaN
    SvShare share;
    int left;                 // units of the share
    float ml[FW_WARPS][16][2];
    alignas(16) float o[FW_WARPS][16][CUINF_HD];  // (read by float4)
};
static constexpr size_t FW_SMEM_BYTES = 128 + (size_t)FW_ST * FW_UNIT + sizeof(FwSmem);

// A place on the line: unit u of the n of (sequence s, kv head h).  Kept by
// steps (a 64-bit division per unit and lane: 83 us for 78).
struct FwPos {
    int s, h, u, n;
    SvSeq q;
};
__device__ __forceinline__ void fw_first(const AttnArgs& A, const SvShare& S, FwPos& p) {
    p.s = S.s;
    sv_seq<SV_FEW>(A, p.s, p.q, false);
    p.n = fw_units(p.q);
    p.h = (int)(S.rem / p.n);
    p.u = (int)(S.rem % p.n);
}
__device__ __forceinline__ void fw_skip(const AttnArgs& A, FwPos& p, int by) {
    p.u += by;
    while (p.u >= p.n) {
        p.u -= p.n;
        if (++p.h < A.nkv) continue;
        p.h = 0;
        do {
            if (++p.s >= A.rows.n_seqs) return;  // the line's end
        } while (!sv_seq<SV_FEW>(A, p.s, p.q, false));
        p.n = fw_units(p.q);
    }
}
// Page of a unit: the table's entry, whatever it is (-1 for a part of the tail, which its place alone tells).
__device__ __forceinline__ bool fw_tail(const FwPos& p) { return p.u >= p.q.kv / SERVE_PAGE; }
__device__ __forceinline__ int fw_page(const AttnArgs& A, const FwPos& p) {
    return fw_tail(p) ? -1 : __ldg(A.kv.table + (size_t)p.s * A.kv.width + p.u);
}

__device__ __forceinline__ void fw_producer(const AttnArgs& A, FwSmem* S, unsigned char* ring, int lane) {
    if (lane >= FW_ST) return;
    const int cnt = S->left;
    FwPos p, np;  // the unit to copy; the one after it (FW_ST further on)
    int npage = -1;
    fw_first(A, S->share, p);
    fw_skip(A, p, lane);
    int page = lane < cnt ? fw_page(A, p) : -1;
    auto scales = [&](const FwPos& x, int pg, __half& k, __half& v) {
        k = v = __float2half_rn(1.f);
        if (pg < 0 || pg >= A.kv.n_pages) return;
        const size_t blk = (size_t)pg * A.nkv + x.h;
        k = __ldg(A.kv.kps + blk), v = __ldg(A.kv.vps + blk);
    };
    __half ks, vs;
    scales(p, page, ks, vs);
    uint32_t k = 0;      // copies of this lane so far
    bool armed = false;  // copies of the last one are in flight
    int j = lane;
    uint32_t idle = 0;
#pragma unroll 1
    for (;;) {
        // one test per turn, so that a lane whose stage is free is not held up by the others
        const bool go = j < cnt && mbar_test_wait(&S->empty[lane], (k & 1) ^ 1);
        if (!__ballot_sync((1u << FW_ST) - 1, j < cnt)) break;
        if (__ballot_sync((1u << FW_ST) - 1, go)) {
            idle = 0;
        } else if (++idle >= FW_IDLE || *(volatile int*)&S->abort_) {
            *(volatile int*)&S->abort_ = 1;
            break;
        }
        if (!go) continue;
        unsigned char* dst = ring + (size_t)lane * FW_UNIT;
        const int u = p.u, h = p.h, ng = p.q.kv / SERVE_PAGE;
        auto put = [&] { S->sc[lane][0] = __half2float(ks), S->sc[lane][1] = __half2float(vs); };
        armed = true;
        if (fw_tail(p)) {
            const int first = (u - ng) * FW_TAIL, rows = min(FW_TAIL, p.q.kv % SERVE_PAGE - first);
            if (rows > 0) {
                const size_t at = ((size_t)p.s * A.nkv + h) * SERVE_PAGE_HEAD + (size_t)first * CUINF_HD;
                put();
                mbar_arrive_expect_tx(&S->full[lane], 2 * rows * CUINF_HD * 2);
                tma_load_1d(dst, A.kv.ktail + at, rows * CUINF_HD * 2, &S->full[lane]);
                tma_load_1d(dst + FW_UNIT / 2, A.kv.vtail + at, rows * CUINF_HD * 2, &S->full[lane]);
            } else {
                put();
                mbar_arrive(&S->full[lane]);
            }
        } else if (page >= 0 && page < A.kv.n_pages) {
            const size_t at = ((size_t)page * A.nkv + h) * SERVE_PAGE_HEAD;
            mbar_expect_tx(&S->full[lane], FW_UNIT);
            tma_load_1d(dst, A.kv.kp8 + at, FW_UNIT / 2, &S->full[lane]);
            tma_load_1d(dst + FW_UNIT / 2, A.kv.vp8 + at, FW_UNIT / 2, &S->full[lane]);
            put();  // (the first copies do not wait for their scales)
            mbar_arrive(&S->full[lane]);
        } else {
            atomicOr(A.err, SERVE_ERR_PAGE);
            S->sc[lane][0] = -1.f, S->sc[lane][1] = 1.f;
            mbar_arrive(&S->full[lane]);
        }
        if (k == 0 && j + FW_ST < cnt) {  // (nor for the place of the second)
            np = p;
            fw_skip(A, np, FW_ST);
            npage = fw_page(A, np);
        }
        if (j + FW_ST < cnt) {
            p = np, page = npage;
            scales(p, page, ks, vs);
            if (j + 2 * FW_ST < cnt) {
                fw_skip(A, np, FW_ST);
                npage = fw_page(A, np);
            }
        }
        j += FW_ST, k++;
    }
    if (armed) sv_drain(&S->full[lane], (k - 1) & 1);  // copies land before the CTA can exit
}

// A warp's running state of 16 rows: lane 4 g + c holds rows g and g + 8.
struct FwRows {
    uint32_t q[4][4];  // the rows' A fragments
    int pos[2];
    float c2;                    // score scale, in powers of two
    float m[2], l[2], o[8][4];   // reference, this lane's share of the sum, output columns 2 c, 2 c + 1 of 8 tiles
    float per_unit;              // O counts in units (see SV_UNIT0) of the warp's pages so far: a row that does not
                                 // attend a page attends none behind it either
};
struct FwUnit {
    const unsigned char* kd;
    float ks, vs;
    int key0, here;  // first key, keys
};
// Values that some row masks become numbers, since 0 * NaN would pass a weight
// of zero: those that are none are noted by (column, first key) and become
// zero, keys behind the last are zero.  The stage is the warp's own.
template <bool TAIL>
__device__ __forceinline__ void fw_clean(const FwUnit& x, FwSmem* S, int note, int lane) {
    unsigned char* vd = const_cast<unsigned char*>(x.kd) + FW_UNIT / 2;
    bool touched = false;
#pragma unroll 1
    for (int u = lane; u < FW_UNIT / 2 / 16; u += 32) {
        uint4* p = reinterpret_cast<uint4*>(vd + 16 * u);
        const int row = TAIL ? u >> 3 : u >> 2, d0 = TAIL ? 8 * (u & 7) : 16 * (u & 3);
        if (row >= x.here) {
            *p = make_uint4(0, 0, 0, 0);
            touched = true;
            continue;
        }
        uint32_t any = 0;
        const uint4 v = *p;
        if (TAIL)  // exponent all ones
            any = ((v.x & 0x7fff7fffu) + 0x04000400u | (v.y & 0x7fff7fffu) + 0x04000400u | (v.z & 0x7fff7fffu) + 0x04000400u |
                   (v.w & 0x7fff7fffu) + 0x04000400u) & 0x80008000u;
        else  // E4M3's NaN: all ones but the sign
            any = ((v.x & 0x7f7f7f7fu) + 0x01010101u | (v.y & 0x7f7f7f7fu) + 0x01010101u | (v.z & 0x7f7f7f7fu) + 0x01010101u |
                   (v.w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
        if (!any) continue;
        touched = true;
#pragma unroll 1
        for (int e = 0; e < (TAIL ? 8 : 16); e++) {
            int kind = 2;
            if (TAIL) {
                const uint16_t bits = reinterpret_cast<const uint16_t*>(p)[e];
                if ((bits & 0x7c00) != 0x7c00) continue;
                kind = bits & 0x3ff ? 2 : bits >> 15;
                reinterpret_cast<uint16_t*>(p)[e] = 0;
            } else {
                if ((reinterpret_cast<const uint8_t*>(p)[e] & 0x7f) != 0x7f) continue;
                reinterpret_cast<uint8_t*>(p)[e] = 0;
            }
            atomicMin(&S->bad[note][kind][d0 + e], x.key0 + row);
            S->any_bad[note] = 1;
        }
    }
    if (touched) asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");  // before the next copy into the stage
    __syncwarp();
}
// One unit of 64 keys (TAIL: 32, fp16) into the state.  TWO: rows 8 to 15 are
// in use.  MASKED: some row masks some key, or some keys are not there.
template <bool TWO, bool MASKED, bool TAIL>
__device__ __forceinline__ void fw_unit(const FwUnit& x, FwRows& R, FwSmem* S, int note, int lane) {
    constexpr int NT = TAIL ? FW_TAIL / 8 : 8;  // score tiles of 8 keys
    const int g = lane >> 2, c = lane & 3;
    const unsigned char *kd = x.kd, *vd = x.kd + FW_UNIT / 2;
    if (MASKED) fw_clean<TAIL>(x, S, note, lane);
    float s[NT][4];
    // four score tiles at a time, so that a product does not wait for the one before it
#pragma unroll
    for (int t0 = 0; t0 < NT; t0 += 4) {
        uint32_t w[4][8];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            if (TAIL) {
                const uint4* src = reinterpret_cast<const uint4*>(kd + (8 * (t0 + t) + g) * 128 + 32 * c);
                const uint4 a = src[0], b = src[1];
                w[t][0] = a.x, w[t][1] = a.y, w[t][2] = a.z, w[t][3] = a.w;
                w[t][4] = b.x, w[t][5] = b.y, w[t][6] = b.z, w[t][7] = b.w;
            } else {
                const uint4 a = *reinterpret_cast<const uint4*>(kd + (8 * (t0 + t) + g) * 64 + 16 * c);
                w[t][0] = sv_e4m3x2(a.x), w[t][1] = sv_e4m3x2(a.x >> 16);
                w[t][2] = sv_e4m3x2(a.y), w[t][3] = sv_e4m3x2(a.y >> 16);
                w[t][4] = sv_e4m3x2(a.z), w[t][5] = sv_e4m3x2(a.z >> 16);
                w[t][6] = sv_e4m3x2(a.w), w[t][7] = sv_e4m3x2(a.w >> 16);
            }
        }
#pragma unroll
        for (int t = 0; t < 4; t++) s[t0 + t][0] = s[t0 + t][1] = s[t0 + t][2] = s[t0 + t][3] = 0.f;
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int t = 0; t < 4; t++)
                mma_16816(s[t0 + t], R.q[k][0], R.q[k][1], R.q[k][2], R.q[k][3], w[t][2 * k], w[t][2 * k + 1]);
    }
    constexpr int NR = TWO ? 2 : 1;
    float kc[2], top[2];
    bool none[2] = {false, false};  // the row attends no key of the unit
#pragma unroll
    for (int r = 0; r < NR; r++) {
        kc[r] = R.c2 * x.ks;
        if (MASKED) {
            if (kc[r] == 0.f) kc[r] = 1e-30f;  // a page of zeros: -inf * 0 is no number
            // a page's scale that is no number reaches only rows that attend the page
            none[r] = R.pos[r] < x.key0;
            if (none[r]) kc[r] = R.c2;
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int e = 0; e < 2; e++)
                    if (x.key0 + 8 * t + 2 * c + e > R.pos[r]) s[t][2 * r + e] = -INFINITY;
        }
        float a[4];
#pragma unroll
        for (int j = 0; j < 4; j++) a[j] = s[j / 2][2 * r + (j & 1)];
#pragma unroll
        for (int j = 4; j < 2 * NT; j++) a[j & 3] = fmaxf(a[j & 3], s[j / 2][2 * r + (j & 1)]);
        top[r] = fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3]));
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2)) * kc[r];
    }
    const bool grown = top[0] > R.m[0] + SV_GROWTH || (TWO && top[NR - 1] > R.m[NR - 1] + SV_GROWTH);
    if (__any_sync(0xffffffffu, grown || x.vs * R.per_unit >= SV_UNIT_TOP)) {
        const float v = sv_in_units(x.vs, R.per_unit), step = v >= SV_UNIT_TOP ? sv_unit_step(v) : 1.f;
        R.per_unit *= step;
#pragma unroll
        for (int r = 0; r < NR; r++) {
            const float mn = top[r] > R.m[r] + SV_GROWTH ? top[r] : R.m[r];  // (each row for itself)
            float f = R.m[r] == -INFINITY ? 0.f : sv_exp2(R.m[r] - mn);
            R.m[r] = mn, R.l[r] *= f, f *= step;
#pragma unroll
            for (int i = 0; i < 8; i++) R.o[i][2 * r] *= f, R.o[i][2 * r + 1] *= f;
        }
    }
    uint32_t a[NT / 2][4];  // the weights' A fragments, 16 keys each
#pragma unroll
    for (int r = 0; r < 2; r++) {
        if (r >= NR) {
#pragma unroll
            for (int t = 0; t < NT; t++) a[t / 2][2 * (t & 1) + 1] = 0;
            continue;
        }
        const float ref = R.m[r] == -INFINITY ? 0.f : R.m[r], vu = none[r] ? 0.f : x.vs * R.per_unit;
        float l[2] = {0.f, 0.f};
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const float p0 = sv_exp2(fmaf(s[t][2 * r], kc[r], -ref)), p1 = sv_exp2(fmaf(s[t][2 * r + 1], kc[r], -ref));
            l[t & 1] += p0 + p1;
            a[t / 2][2 * (t & 1) + r] = sv_pack_h2(p0 * vu, p1 * vu);
        }
        R.l[r] += l[0] + l[1];
    }
#pragma unroll
    for (int q = 0; q < NT / 2; q++) {
        // values: keys 16 q + 2 c, + 1 (z = 0) and 8 further on, dims 8 g .. 8 g + 7
        uint32_t b[2][8];
#pragma unroll
        for (int z = 0; z < 2; z++) {
            const int key = 16 * q + 8 * z + 2 * c;
            if (TAIL) {
                const uint4 v = *reinterpret_cast<const uint4*>(vd + key * 128 + 16 * g);
                const uint4 y = *reinterpret_cast<const uint4*>(vd + (key + 1) * 128 + 16 * g);
                b[z][0] = __byte_perm(v.x, y.x, 0x5410), b[z][1] = __byte_perm(v.x, y.x, 0x7632);
                b[z][2] = __byte_perm(v.y, y.y, 0x5410), b[z][3] = __byte_perm(v.y, y.y, 0x7632);
                b[z][4] = __byte_perm(v.z, y.z, 0x5410), b[z][5] = __byte_perm(v.z, y.z, 0x7632);
                b[z][6] = __byte_perm(v.w, y.w, 0x5410), b[z][7] = __byte_perm(v.w, y.w, 0x7632);
            } else {
                const uint2 v = *reinterpret_cast<const uint2*>(vd + key * 64 + 8 * g);
                const uint2 y = *reinterpret_cast<const uint2*>(vd + (key + 1) * 64 + 8 * g);
                const uint32_t w0 = __byte_perm(v.x, y.x, 0x5140), w1 = __byte_perm(v.x, y.x, 0x7362);
                const uint32_t w2 = __byte_perm(v.y, y.y, 0x5140), w3 = __byte_perm(v.y, y.y, 0x7362);
                b[z][0] = sv_e4m3x2(w0), b[z][1] = sv_e4m3x2(w0 >> 16);
                b[z][2] = sv_e4m3x2(w1), b[z][3] = sv_e4m3x2(w1 >> 16);
                b[z][4] = sv_e4m3x2(w2), b[z][5] = sv_e4m3x2(w2 >> 16);
                b[z][6] = sv_e4m3x2(w3), b[z][7] = sv_e4m3x2(w3 >> 16);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) mma_16816(R.o[i], a[q][0], a[q][1], a[q][2], a[q][3], b[0][i], b[1][i]);
    }
}

template <bool BESIDE>  // (a kernel of its own: with the sums' code one token at 32768 took 20.1 us, without 19.7)
__global__ void __launch_bounds__((FW_WARPS + 1) * 32, 1)
    k_serve_few(const AttnArgs A, const int split, const SvWs W) {
    extern __shared__ __align__(128) unsigned char fw_raw[];
    unsigned char* ring = fw_raw + ((128 - (smem_u32(fw_raw) & 127)) & 127);
    FwSmem* S = reinterpret_cast<FwSmem*>(ring + (size_t)FW_ST * FW_UNIT);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_trigger();
    if (tid == 0) {
        for (int i = 0; i < FW_ST; i++) mbar_init(&S->full[i], 1), mbar_init(&S->empty[i], 1);
        mbar_init(&S->merge, FW_WARPS), mbar_init(&S->merged, FW_WARPS);
        S->abort_ = 0;
        for (int i = 0; i < 3; i++) S->any_bad[i] = 0;
    }
    for (int i = tid; i < 9 * CUINF_HD; i += blockDim.x) (&S->bad[0][0][0])[i] = 0x7fffffff;
    if (split && tid < 2) W.part[blockIdx.x * 2 + tid].valid = 0;
    sv_share<SV_FEW>(A, &S->share, blockIdx.x, gridDim.x, BESIDE, [&](const SvSeq& q) { return (long long)fw_units(q) * A.nkv; });
    if (tid == 0) {
        long long left = S->share.left;
        if (!split && left > 0) {
            // items are not cut: the share's items are those that begin in it
            FwPos p;
            fw_first(A, S->share, p);
            const long long skip = (p.n - p.u) % p.n;
            if (left <= skip) {
                left = 0;
            } else {
                left -= skip;
                fw_skip(A, p, (int)skip);
                S->share.s = p.s, S->share.rem = (long long)p.h * p.n;
                long long at = 0;  // whole items from here on
                while (at < left && p.s < A.rows.n_seqs) {
                    at += p.n;
                    fw_skip(A, p, p.n);
                }
                left = at;
            }
        }
        S->left = (int)left;
    }
    __syncthreads();
    const int cnt = S->left;
    if (cnt > 0) {
        if (warp == FW_WARPS) {
            fw_producer(A, S, ring, lane);
            __syncwarp();
        } else {
            const int G = A.nh / A.nkv, g = lane >> 2, c = lane & 3;
            const float c2 = A.scale * SV_LOG2E;
            FwPos p;
            fw_first(A, S->share, p);
            int j = 0;  // share's units before the item
            uint32_t item = 0;
            bool ok = true;
            // rows g and g + 8: dims 16 c .. 16 c + 15
            uint4 qn[2][2];
            auto load_q = [&](const FwPos& x) {
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const int row = g + 8 * r;
                    qn[r][0] = qn[r][1] = make_uint4(0, 0, 0, 0);
                    if (row < x.q.c * G) {
                        const uint4* src = reinterpret_cast<const uint4*>(
                            A.q + (size_t)(x.q.a + row / G) * A.q_stride + (x.h * G + row % G) * CUINF_HD +
                            16 * c);
                        qn[r][0] = src[0], qn[r][1] = src[1];
                    }
                }
            };
            load_q(p);
            while (j < cnt) {
                const int rows = p.q.c * G, h = p.h, tb = p.u;
                const int te = min(p.n, tb + (cnt - j));
                const int ng = p.q.kv / SERVE_PAGE;
                FwRows R;
                {
                    const uint32_t* q0 = reinterpret_cast<const uint32_t*>(qn[0]);
                    const uint32_t* q1 = reinterpret_cast<const uint32_t*>(qn[1]);
#pragma unroll
                    for (int t = 0; t < 4; t++)
                        R.q[t][0] = q0[2 * t], R.q[t][1] = q1[2 * t], R.q[t][2] = q0[2 * t + 1], R.q[t][3] = q1[2 * t + 1];
                }
                FwPos nx = p;
                if (j + te - tb < cnt) {  // the next item's rows, while this one runs
                    fw_skip(A, nx, te - tb);
                    load_q(nx);
                }
                R.c2 = c2, R.per_unit = SV_UNIT0;
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    R.pos[r] = p.q.p0 + (g + 8 * r) / G;
                    R.m[r] = -INFINITY, R.l[r] = 0.f;
                }
#pragma unroll
                for (int i = 0; i < 8; i++) R.o[i][0] = R.o[i][1] = R.o[i][2] = R.o[i][3] = 0.f;
                const int(*bad)[CUINF_HD] = S->bad[item % 3];

                for (int u = j + (warp + FW_WARPS - j % FW_WARPS) % FW_WARPS; u < j + te - tb; u += FW_WARPS) {
                    const int st = u % FW_ST, unit = tb + u - j;
                    if (!(ok = sv_wait_all(&S->full[st], (u / FW_ST) & 1, &S->abort_))) break;
                    FwUnit x;
                    x.kd = ring + (size_t)st * FW_UNIT;
                    x.ks = S->sc[st][0], x.vs = S->sc[st][1];
                    const bool tail = unit >= ng;
                    x.key0 = tail ? ng * SERVE_PAGE + (unit - ng) * FW_TAIL : unit * SERVE_PAGE;
                    x.here = tail ? min(FW_TAIL, p.q.kv - x.key0) : SERVE_PAGE;
                    // one straight path each: with these as branches inside, the loop's loads and products could not
                    // be interleaved
                    if (x.ks >= 0.f || x.ks != x.ks) {  // (negative: absent)
                        if (tail)
                            fw_unit<true, true, true>(x, R, S, item % 3, lane);
                        else if (x.key0 + SERVE_PAGE > p.q.p0 + 1)
                            fw_unit<true, true, false>(x, R, S, item % 3, lane);
                        else if (rows > 8)
                            fw_unit<true, false, false>(x, R, S, item % 3, lane);
                        else
                            fw_unit<false, false, false>(x, R, S, item % 3, lane);
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&S->empty[st]);
                }
                // ---- the item's end: join the warps ----
                // what the last item left there has been read
                if (!ok || (item > 0 && !(ok = sv_wait_all(&S->merged, (item - 1) & 1, &S->abort_)))) break;
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    R.l[r] += __shfl_xor_sync(0xffffffffu, R.l[r], 1);
                    R.l[r] += __shfl_xor_sync(0xffffffffu, R.l[r], 2);
                    const int row = g + 8 * r;
                    if (c == 0) S->ml[warp][row][0] = R.m[r], S->ml[warp][row][1] = R.l[r];
                    if (row >= rows) continue;
                    const float unit = sv_inverse(R.per_unit);
#pragma unroll
                    for (int e = 0; e < 2; e++) {  // columns 2 c + e of tile i: dims 8 (2 c + e) + i
                        const int z = 2 * r + e;
                        float4* d = reinterpret_cast<float4*>(&S->o[warp][row][16 * c + 8 * e]);
                        d[0] = make_float4(R.o[0][z] * unit, R.o[1][z] * unit, R.o[2][z] * unit, R.o[3][z] * unit);
                        d[1] = make_float4(R.o[4][z] * unit, R.o[5][z] * unit, R.o[6][z] * unit, R.o[7][z] * unit);
                    }
                }
                // notes of the next item: last read two items ago, written only after this barrier
                const int nb = (item + 1) % 3;
                for (int i = tid; i < 3 * CUINF_HD; i += FW_WARPS * 32) (&S->bad[nb][0][0])[i] = 0x7fffffff;
                if (tid == 0) S->any_bad[nb] = 0;
                __threadfence_block();
                __syncwarp();
                if (lane == 0) mbar_arrive(&S->merge);
                if (!(ok = sv_wait_all(&S->merge, item & 1, &S->abort_))) break;
                const bool whole = tb == 0 && te == p.n;
                const size_t slot = (size_t)blockIdx.x * 2 + (tb == 0);
                for (int i = tid; i < rows * 16; i += FW_WARPS * 32) {
                    const int row = i >> 4, d = (i & 15) * 4;
                    float m = -INFINITY, l = 0.f;
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int w = 0; w < FW_WARPS; w++) m = fmaxf(m, S->ml[w][row][0]);
                    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
                    for (int w = 0; w < FW_WARPS; w++) {
                        const float mw = S->ml[w][row][0], lw = S->ml[w][row][1];
                        const float f = mw == -INFINITY ? 0.f : sv_exp2(mw - ref);
                        l += mw == -INFINITY ? lw : lw * f;  // (NaN scores alone have no maximum)
                        const float4 y = *reinterpret_cast<const float4*>(&S->o[w][row][d]);
                        x.x += y.x * f, x.y += y.y * f, x.z += y.z * f, x.w += y.w * f;
                    }
                    float* xf = reinterpret_cast<float*>(&x);
                    if (S->any_bad[item % 3]) {
                        const int pos = p.q.p0 + row / G;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            if (bad[0][d + e] <= pos) xf[e] += INFINITY;
                            if (bad[1][d + e] <= pos) xf[e] -= INFINITY;
                            if (bad[2][d + e] <= pos) xf[e] = NAN;
                        }
                    }
                    if (whole) {
                        const float inv = l == 0.f ? 0.f : 1.f / l;
                        uint2 r;
                        r.x = sv_pack_h2(x.x * inv, x.y * inv), r.y = sv_pack_h2(x.z * inv, x.w * inv);
                        *reinterpret_cast<uint2*>(A.out + ((size_t)(p.q.a + row / G) * A.nh + h * G + row % G) * CUINF_HD +
                                                  d) = r;
                    } else {
                        if (d == 0) reinterpret_cast<float2*>(W.ml)[slot * 16 + row] = make_float2(m, l);
                        *reinterpret_cast<float4*>(W.o + (slot * 16 + row) * CUINF_HD + d) = x;
                    }
                }
                if (!whole && tid == 0) {
                    SvPart t;
                    t.valid = 1, t.last = te == p.n, t.row0 = p.q.a, t.tokens = p.q.c, t.h = h;
                    W.part[slot] = t;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&S->merged);
                j += te - tb;
                p = nx;
                item++;
            }
        }
    }
    __syncthreads();
    if (tid == 0 && S->abort_) atomicOr(A.err, SERVE_ERR_WAIT);
    pdl_wait();  // launched beside the chunks' kernel: what follows this kernel follows that one too
}
