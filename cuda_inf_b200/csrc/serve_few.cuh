// Attention of few new rows per sequence (one token, or some drafted ones: at
// most 16 rows of new tokens x query heads per kv head) over the paged cache.
//
// Bound by the pages' bytes: 8 KB of FP8 per page and kv head against 16 rows.
// A unit of the shared line is one page of one (sequence, kv head), or 32
// tokens of its fp16 tail (also 8 KB).  Warp 8 copies units with bulk copies
// into a ring of 16 stages, lane i filling stage i, each lane with its next
// unit's page index and scales already in registers; warp w takes units w, w +
// 8, ... of the CTA's share, so a stage belongs to one warp and the warps meet
// only where an item ends, when their (m, l, O) are joined in shared memory.
//
// Products by mma.sync m16n8k16 with the rows as M (4 of 16 for one token and
// 4 heads per kv head; the tensor pipe has room: 64 products a page against
// 356 clocks of its HBM time per SM).  The sum over the head's dims may run in
// any order, so lane quad c takes dims 16 c .. 16 c + 15 of a key: one 16-byte
// shared load per key.  E4M3 becomes fp16 exactly; the page's key scale joins
// the scores, its value scale the weights (one rounding of a weight to fp16).
#pragma once
#include "serve_line.cuh"

#define FW_WARPS 8
#define FW_ST 16           // stages; a multiple of FW_WARPS: a stage's phases are all seen by one warp
#define FW_UNIT 8192       // bytes of a unit: 4096 of keys, 4096 of values
#define FW_TAIL 32         // tail tokens of a unit
#define FW_THR 3.f         // the reference follows the maximum when it has grown by 2^THR

struct FwSmem {
    uint64_t full[FW_ST], empty[FW_ST], merge;
    int abort_;
    float sc[FW_ST][2];       // key scale (negative: absent), value scale
    int any_bad[3];
    int bad[3][3][CUINF_HD];  // by item, modulo 3: first key whose value is +inf, -inf, NaN
    SvShare share;
    float ml[2][FW_WARPS][16][2];  // by item, modulo 2
    float o[2][FW_WARPS][16][CUINF_HD];
};
static constexpr size_t FW_SMEM_BYTES = 128 + (size_t)FW_ST * FW_UNIT + sizeof(FwSmem);

// units of one kv head (at least one: rows without a key still become zero)
__device__ __forceinline__ int fw_units(const SvSeq& q) {
    return max(1, q.kv / SERVE_PAGE + (q.kv % SERVE_PAGE + FW_TAIL - 1) / FW_TAIL);
}
// A place on the line: unit `rem` of sequence s's n * nkv.
struct FwPos {
    int s, n;
    long long rem;
    SvSeq q;
};
__device__ __forceinline__ void fw_skip(const AttnArgs& A, FwPos& p, long long by) {
    p.rem += by;
    while (p.s < A.rows.n_seqs && p.rem >= (long long)p.n * A.nkv) {
        p.rem -= (long long)p.n * A.nkv;
        do p.s++;
        while (p.s < A.rows.n_seqs && !sv_seq<SV_FEW>(A, p.s, p.q, false));
        if (p.s < A.rows.n_seqs) p.n = fw_units(p.q);
    }
}
// Page of unit u: an index (unchecked), or -2 for a part of the tail.
__device__ __forceinline__ int fw_page(const AttnArgs& A, const FwPos& p) {
    if (p.s >= A.rows.n_seqs) return -2;
    const int u = (int)(p.rem % p.n);
    return u < p.q.kv / SERVE_PAGE ? __ldg(A.kv.table + (size_t)p.s * A.kv.width + u) : -2;
}

__device__ __forceinline__ void fw_producer(const AttnArgs& A, FwSmem* S, unsigned char* ring, int lane) {
    if (lane >= FW_ST) return;
    const long long cnt = S->share.left;
    FwPos p, np;  // the unit to copy; the one after it (FW_ST further on)
    p.s = S->share.s, p.rem = S->share.rem;
    sv_seq<SV_FEW>(A, p.s, p.q, false);
    p.n = fw_units(p.q);
    fw_skip(A, p, lane);
    int page = lane < cnt ? fw_page(A, p) : -2;
    auto scales = [&](const FwPos& x, int pg, __half& k, __half& v) {
        k = v = __float2half_rn(1.f);
        if (pg < 0 || pg >= A.kv.n_pages) return;
        const size_t blk = (size_t)pg * A.nkv + (int)(x.rem / x.n);
        k = __ldg(A.kv.kps + blk), v = __ldg(A.kv.vps + blk);
    };
    __half ks, vs;
    scales(p, page, ks, vs);
    np = p;
    fw_skip(A, np, FW_ST);
    int npage = lane + FW_ST < cnt ? fw_page(A, np) : -2;
    uint32_t k = 0;      // copies of this lane so far
    bool armed = false;  // copies of the last one are in flight
    long long j = lane;
    uint64_t t0 = globaltimer_ns();
    for (int spin = 1;; spin++) {
        // one test per turn, so that a lane whose stage is free is not held up by the others
        const bool go = j < cnt && mbar_test_wait(&S->empty[lane], (k & 1) ^ 1);
        if (!__ballot_sync((1u << FW_ST) - 1, j < cnt)) break;
        if (__ballot_sync((1u << FW_ST) - 1, go)) {
            t0 = globaltimer_ns();
        } else if ((spin & 63) == 0) {
            const bool late = globaltimer_ns() - t0 > SV_WAIT_LIMIT_NS;
            if (__ballot_sync((1u << FW_ST) - 1, late || *(volatile int*)&S->abort_)) {
                if (late) atomicOr(A.err, SERVE_ERR_WAIT);
                *(volatile int*)&S->abort_ = 1;
                break;
            }
        }
        if (!go) continue;
        unsigned char* dst = ring + (size_t)lane * FW_UNIT;
        const int u = (int)(p.rem % p.n), h = (int)(p.rem / p.n), ng = p.q.kv / SERVE_PAGE;
        S->sc[lane][0] = __half2float(ks), S->sc[lane][1] = __half2float(vs);
        armed = true;
        if (page == -2) {
            const int first = (u - ng) * FW_TAIL, rows = min(FW_TAIL, p.q.kv % SERVE_PAGE - first);
            if (rows > 0) {
                const size_t at = ((size_t)p.s * A.nkv + h) * SERVE_PAGE_HEAD + (size_t)first * CUINF_HD;
                mbar_arrive_expect_tx(&S->full[lane], 2 * rows * CUINF_HD * 2);
                tma_load_1d(dst, A.kv.ktail + at, rows * CUINF_HD * 2, &S->full[lane]);
                tma_load_1d(dst + FW_UNIT / 2, A.kv.vtail + at, rows * CUINF_HD * 2, &S->full[lane]);
            } else {
                mbar_arrive(&S->full[lane]);
            }
        } else if (page >= 0 && page < A.kv.n_pages) {
            const size_t at = ((size_t)page * A.nkv + h) * SERVE_PAGE_HEAD;
            mbar_arrive_expect_tx(&S->full[lane], FW_UNIT);
            tma_load_1d(dst, A.kv.kp8 + at, FW_UNIT / 2, &S->full[lane]);
            tma_load_1d(dst + FW_UNIT / 2, A.kv.vp8 + at, FW_UNIT / 2, &S->full[lane]);
        } else {
            atomicOr(A.err, SERVE_ERR_PAGE);
            S->sc[lane][0] = -1.f;
            mbar_arrive(&S->full[lane]);
        }
        p = np, page = npage;
        if (j + FW_ST < cnt) {
            scales(p, page, ks, vs);
            fw_skip(A, np, FW_ST);
            npage = j + 2 * FW_ST < cnt ? fw_page(A, np) : -2;
        }
        j += FW_ST, k++;
    }
    if (armed) sv_drain(&S->full[lane], (k - 1) & 1, A.err);  // copies land before the CTA can exit
}

__global__ void __launch_bounds__((FW_WARPS + 1) * 32, 1)
    k_serve_few(const AttnArgs A, const int split, const SvWs W) {
    extern __shared__ __align__(128) unsigned char fw_raw[];
    unsigned char* ring = fw_raw + ((128 - (smem_u32(fw_raw) & 127)) & 127);
    FwSmem* S = reinterpret_cast<FwSmem*>(ring + (size_t)FW_ST * FW_UNIT);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_trigger();
    if (tid == 0) {
        for (int i = 0; i < FW_ST; i++) mbar_init(&S->full[i], 1), mbar_init(&S->empty[i], 1);
        mbar_init(&S->merge, FW_WARPS);
        S->abort_ = 0;
        for (int i = 0; i < 3; i++) S->any_bad[i] = 0;
    }
    for (int i = tid; i < 9 * CUINF_HD; i += blockDim.x) (&S->bad[0][0][0])[i] = 0x7fffffff;
    if (split && tid < 2) W.part[blockIdx.x * 2 + tid].valid = 0;
    sv_share<SV_FEW>(A, &S->share, blockIdx.x, gridDim.x, [&](const SvSeq& q) { return (long long)fw_units(q) * A.nkv; });
    if (!split && tid == 0 && S->share.left > 0) {
        // items are not cut: the share's items are those that begin in it
        SvShare& h = S->share;
        FwPos p;
        p.s = h.s, p.rem = h.rem;
        sv_seq<SV_FEW>(A, p.s, p.q, false);
        p.n = fw_units(p.q);
        const int skip = (int)((p.n - p.rem % p.n) % p.n);
        const long long left = h.left;
        fw_skip(A, p, skip);
        h.s = p.s, h.rem = p.rem;
        FwPos e = p;
        fw_skip(A, e, left - skip > 0 ? left - skip : 0);
        const int more = e.s < A.rows.n_seqs ? (int)((e.n - e.rem % e.n) % e.n) : 0;
        h.left = left > skip ? left - skip + more : 0;
    }
    __syncthreads();
    const long long cnt = S->share.left;
    if (cnt > 0) {
        if (warp == FW_WARPS) {
            fw_producer(A, S, ring, lane);
            __syncwarp();
        } else {
            const int G = A.nh / A.nkv, g = lane >> 2, c = lane & 3;
            const float c2 = A.scale * 1.44269504088896340736f;
            FwPos p;
            p.s = S->share.s, p.rem = S->share.rem;
            sv_seq<SV_FEW>(A, p.s, p.q, false);
            p.n = fw_units(p.q);
            long long j = 0;  // share's units before the item
            uint32_t item = 0;
            bool ok = true;
            // rows g and g + 8: dims 16 c .. 16 c + 15
            uint4 qn[2][2];
            auto load_q = [&](const FwPos& x) {
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const int row = g + 8 * r;
                    qn[r][0] = qn[r][1] = make_uint4(0, 0, 0, 0);
                    if (x.s < A.rows.n_seqs && row < x.q.c * G) {
                        const uint4* src = reinterpret_cast<const uint4*>(
                            A.q + (size_t)(x.q.a + row / G) * A.q_stride + ((int)(x.rem / x.n) * G + row % G) * CUINF_HD +
                            16 * c);
                        qn[r][0] = src[0], qn[r][1] = src[1];
                    }
                }
            };
            load_q(p);
            while (j < cnt) {
                const int rows = p.q.c * G, h = (int)(p.rem / p.n), tb = (int)(p.rem % p.n);
                const int te = (int)min((long long)p.n, tb + (cnt - j));
                const int ng = p.q.kv / SERVE_PAGE;
                uint32_t qa[4][4];
                {
                    const uint32_t* q0 = reinterpret_cast<const uint32_t*>(qn[0]);
                    const uint32_t* q1 = reinterpret_cast<const uint32_t*>(qn[1]);
#pragma unroll
                    for (int t = 0; t < 4; t++)
                        qa[t][0] = q0[2 * t], qa[t][1] = q1[2 * t], qa[t][2] = q0[2 * t + 1], qa[t][3] = q1[2 * t + 1];
                }
                FwPos nx = p;
                fw_skip(A, nx, te - tb);
                if (j + te - tb < cnt) load_q(nx);  // the next item's, while this one runs
                const int pos0 = p.q.p0 + g / G, pos1 = p.q.p0 + (g + 8) / G;  // positions of rows g, g + 8
                const bool two = rows > 8;
                float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f, o[8][4];
#pragma unroll
                for (int i = 0; i < 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
                int(*bad)[CUINF_HD] = S->bad[item % 3];

                const long long u0 = j + ((warp - j) % FW_WARPS + FW_WARPS) % FW_WARPS;
                for (long long u = u0; u < j + te - tb; u += FW_WARPS) {
                    const int st = (int)(u % FW_ST), unit = tb + (int)(u - j);
                    if (!(ok = sv_wait(&S->full[st], (u / FW_ST) & 1, &S->abort_, A.err))) break;
                    const unsigned char* kd = ring + (size_t)st * FW_UNIT;
                    const unsigned char* vd = kd + FW_UNIT / 2;
                    const float ks = S->sc[st][0], vs = S->sc[st][1];
                    const bool tail = unit >= ng;
                    const int key0 = tail ? ng * SERVE_PAGE + (unit - ng) * FW_TAIL : unit * SERVE_PAGE;
                    if (ks >= 0.f || ks != ks) {  // not absent
                        const int here = tail ? min(FW_TAIL, p.q.kv - key0) : SERVE_PAGE;
                        const bool masked = key0 + SERVE_PAGE > p.q.p0 + 1;
                        float s[8][4];
#pragma unroll
                        for (int t = 0; t < 8; t++) {
                            s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
                            uint32_t w[8];
                            if (tail) {
                                if (t >= FW_TAIL / 8) continue;
                                const uint4* src = reinterpret_cast<const uint4*>(kd + (8 * t + g) * 128 + 32 * c);
                                const uint4 a = src[0], b = src[1];
                                w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
                                w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
                            } else {
                                const uint4 a = *reinterpret_cast<const uint4*>(kd + (8 * t + g) * 64 + 16 * c);
                                w[0] = sv_e4m3x2(a.x), w[1] = sv_e4m3x2(a.x >> 16);
                                w[2] = sv_e4m3x2(a.y), w[3] = sv_e4m3x2(a.y >> 16);
                                w[4] = sv_e4m3x2(a.z), w[5] = sv_e4m3x2(a.z >> 16);
                                w[6] = sv_e4m3x2(a.w), w[7] = sv_e4m3x2(a.w >> 16);
                            }
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                mma_16816(s[t], qa[k][0], qa[k][1], qa[k][2], qa[k][3], w[2 * k], w[2 * k + 1]);
                        }
                        const float kc = c2 * ks;
                        float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
                        for (int t = 0; t < 8; t++)
#pragma unroll
                            for (int e = 0; e < 2; e++) {
                                s[t][e] *= kc, s[t][2 + e] *= kc;
                                if (masked) {
                                    const int key = key0 + 8 * t + 2 * c + e;
                                    if (key > pos0 || 8 * t >= here) s[t][e] = -INFINITY;
                                    if (key > pos1 || 8 * t >= here) s[t][2 + e] = -INFINITY;
                                }
                                x0 = fmaxf(x0, s[t][e]), x1 = fmaxf(x1, s[t][2 + e]);
                            }
                        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
                        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
                        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
                        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
                        if (__any_sync(0xffffffffu, x0 > m0 + FW_THR || x1 > m1 + FW_THR)) {
                            const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
                            const float f0 = m0 == -INFINITY ? 0.f : sv_exp2(m0 - n0);
                            const float f1 = m1 == -INFINITY ? 0.f : sv_exp2(m1 - n1);
                            m0 = n0, m1 = n1, l0 *= f0, l1 *= f1;
#pragma unroll
                            for (int i = 0; i < 8; i++) o[i][0] *= f0, o[i][1] *= f0, o[i][2] *= f1, o[i][3] *= f1;
                        }
                        const float r0 = m0 == -INFINITY ? 0.f : m0, r1 = m1 == -INFINITY ? 0.f : m1;
                        const float vc = vs * SV_VEXP;
                        // a page's scale that is no number reaches only rows that attend the page
                        const float vc0 = pos0 < key0 ? 0.f : vc, vc1 = pos1 < key0 ? 0.f : vc;
#pragma unroll
                        for (int q = 0; q < 4; q++) {  // 16 keys: score tiles 2 q, 2 q + 1
                            if (tail && q >= FW_TAIL / 16) continue;
                            uint32_t a[4] = {0, 0, 0, 0};
#pragma unroll
                            for (int z = 0; z < 2; z++) {
                                const float p0 = sv_exp2(s[2 * q + z][0] - r0), p1 = sv_exp2(s[2 * q + z][1] - r0);
                                l0 += p0 + p1;
                                a[2 * z] = sv_pack_h2(p0 * vc0, p1 * vc0);
                                if (two) {
                                    const float p2 = sv_exp2(s[2 * q + z][2] - r1), p3 = sv_exp2(s[2 * q + z][3] - r1);
                                    l1 += p2 + p3;
                                    a[2 * z + 1] = sv_pack_h2(p2 * vc1, p3 * vc1);
                                }
                            }
                            // values: keys 16 q + 2 c, + 1 (z = 0) and 8 further on, dims 8 g .. 8 g + 7
                            uint32_t b[2][8];
#pragma unroll
                            for (int z = 0; z < 2; z++) {
                                const int key = 16 * q + 8 * z + 2 * c;
                                if (tail) {
                                    const uint4 x = *reinterpret_cast<const uint4*>(vd + key * 128 + 16 * g);
                                    const uint4 y = *reinterpret_cast<const uint4*>(vd + (key + 1) * 128 + 16 * g);
                                    b[z][0] = __byte_perm(x.x, y.x, 0x5410), b[z][1] = __byte_perm(x.x, y.x, 0x7632);
                                    b[z][2] = __byte_perm(x.y, y.y, 0x5410), b[z][3] = __byte_perm(x.y, y.y, 0x7632);
                                    b[z][4] = __byte_perm(x.z, y.z, 0x5410), b[z][5] = __byte_perm(x.z, y.z, 0x7632);
                                    b[z][6] = __byte_perm(x.w, y.w, 0x5410), b[z][7] = __byte_perm(x.w, y.w, 0x7632);
                                } else {
                                    const uint2 x = *reinterpret_cast<const uint2*>(vd + key * 64 + 8 * g);
                                    const uint2 y = *reinterpret_cast<const uint2*>(vd + (key + 1) * 64 + 8 * g);
                                    const uint32_t w0 = __byte_perm(x.x, y.x, 0x5140), w1 = __byte_perm(x.x, y.x, 0x7362);
                                    const uint32_t w2 = __byte_perm(x.y, y.y, 0x5140), w3 = __byte_perm(x.y, y.y, 0x7362);
                                    b[z][0] = sv_e4m3x2(w0), b[z][1] = sv_e4m3x2(w0 >> 16);
                                    b[z][2] = sv_e4m3x2(w1), b[z][3] = sv_e4m3x2(w1 >> 16);
                                    b[z][4] = sv_e4m3x2(w2), b[z][5] = sv_e4m3x2(w2 >> 16);
                                    b[z][6] = sv_e4m3x2(w3), b[z][7] = sv_e4m3x2(w3 >> 16);
                                }
                                if (masked) {  // what some row masks is a number: 0 * NaN would pass a weight of zero
#pragma unroll
                                    for (int i = 0; i < 8; i++)
#pragma unroll
                                        for (int e = 0; e < 2; e++) {
                                            const uint32_t bits = b[z][i] >> (16 * e) & 0xffffu;
                                            const bool gone = key + e >= here;
                                            if (gone || (bits & 0x7c00u) == 0x7c00u) {
                                                if (!gone) {
                                                    atomicMin(&bad[bits & 0x3ffu ? 2 : bits & 0x8000u ? 1 : 0][8 * g + i],
                                                              key0 + key + e);
                                                    S->any_bad[item % 3] = 1;
                                                }
                                                b[z][i] &= e ? 0x0000ffffu : 0xffff0000u;
                                            }
                                        }
                                }
                            }
#pragma unroll
                            for (int i = 0; i < 8; i++) mma_16816(o[i], a[0], a[1], a[2], a[3], b[0][i], b[1][i]);
                        }
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&S->empty[st]);
                }
                // ---- the item's end: join the warps ----
                l0 += __shfl_xor_sync(0xffffffffu, l0, 1), l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
                l1 += __shfl_xor_sync(0xffffffffu, l1, 1), l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
                const int par = item & 1;
                if (c == 0) {
                    S->ml[par][warp][g][0] = m0, S->ml[par][warp][g][1] = l0;
                    S->ml[par][warp][g + 8][0] = m1, S->ml[par][warp][g + 8][1] = l1;
                }
#pragma unroll
                for (int e = 0; e < 2; e++) {  // columns 2 c + e of tile i: dims 8 (2 c + e) + i
                    if (g < rows) {
                        float4* d = reinterpret_cast<float4*>(&S->o[par][warp][g][16 * c + 8 * e]);
                        d[0] = make_float4(o[0][e], o[1][e], o[2][e], o[3][e]);
                        d[1] = make_float4(o[4][e], o[5][e], o[6][e], o[7][e]);
                    }
                    if (g + 8 < rows) {
                        float4* d = reinterpret_cast<float4*>(&S->o[par][warp][g + 8][16 * c + 8 * e]);
                        d[0] = make_float4(o[0][2 + e], o[1][2 + e], o[2][2 + e], o[3][2 + e]);
                        d[1] = make_float4(o[4][2 + e], o[5][2 + e], o[6][2 + e], o[7][2 + e]);
                    }
                }
                // notes of the next item: last read two items ago, written only after this barrier
                const int nb = (item + 1) % 3;
                for (int i = tid; i < 3 * CUINF_HD; i += FW_WARPS * 32) (&S->bad[nb][0][0])[i] = 0x7fffffff;
                if (tid == 0) S->any_bad[nb] = 0;
                __threadfence_block();
                __syncwarp();
                if (lane == 0) mbar_arrive(&S->merge);
                if (!ok || !(ok = sv_wait(&S->merge, item & 1, &S->abort_, A.err))) break;
                const bool whole = tb == 0 && te == p.n;
                const size_t slot = (size_t)blockIdx.x * 2 + (tb == 0);
                for (int i = tid; i < rows * 16; i += FW_WARPS * 32) {
                    const int row = i >> 4, d = (i & 15) * 4;
                    float m = -INFINITY, l = 0.f;
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int w = 0; w < FW_WARPS; w++) m = fmaxf(m, S->ml[par][w][row][0]);
                    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
                    for (int w = 0; w < FW_WARPS; w++) {
                        const float mw = S->ml[par][w][row][0], lw = S->ml[par][w][row][1];
                        const float f = mw == -INFINITY ? 0.f : sv_exp2(mw - ref);
                        l += mw == -INFINITY ? lw : lw * f;  // (NaN scores alone have no maximum)
                        const float4 y = *reinterpret_cast<const float4*>(&S->o[par][w][row][d]);
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
                        const float inv = l == 0.f ? 0.f : 1.f / (SV_VEXP * l);
                        uint2 r;
                        r.x = sv_pack_h2(x.x * inv, x.y * inv), r.y = sv_pack_h2(x.z * inv, x.w * inv);
                        *reinterpret_cast<uint2*>(A.out + ((size_t)(p.q.a + row / G) * A.nh + h * G + row % G) * CUINF_HD +
                                                  d) = r;
                    } else {
                        const float v = 1.f / SV_VEXP;
                        if (d == 0) reinterpret_cast<float2*>(W.ml)[slot * 16 + row] = make_float2(m, l);
                        *reinterpret_cast<float4*>(W.o + (slot * 16 + row) * CUINF_HD + d) =
                            make_float4(x.x * v, x.y * v, x.z * v, x.w * v);
                    }
                }
                if (!whole && tid == 0) {
                    SvPart t;
                    t.valid = 1, t.last = te == p.n, t.row0 = p.q.a, t.tokens = p.q.c, t.h = h;
                    W.part[slot] = t;
                }
                j += te - tb;
                p = nx;
                item++;
            }
        }
    }
    __syncthreads();
    pdl_wait();  // launched beside the chunks' kernel: what follows this kernel follows that one too
}
