// Shared pieces of the serving attention operators (serve.cu): packed
// sequences, the paged FP8 cache, their error word.
#pragma once
#include "common.cuh"

// Bits of the paged operators' error word (cuinf_paged_error).
#define SERVE_ERR_WAIT 1u   // a bounded wait gave up
#define SERVE_ERR_PAGE 2u   // a page index outside the pool
#define SERVE_ERR_RANGE 4u  // lengths or row offsets outside their ranges

// One page: the framework's commit group (64 tokens), head-major, so that one
// kv head of one page is one block of 4096 contiguous bytes.
#define SERVE_PAGE CUINF_KVGROUP
#define SERVE_PAGE_HEAD (SERVE_PAGE * CUINF_HD)

// The paged cache: kp8/vp8 u8 [n_pages][nkv][64][64], kps/vps fp16
// [n_pages][nkv], ktail/vtail fp16 [n_seqs][nkv][64][64], table int
// [n_seqs][width] (page of each whole 64-token group of a sequence).
struct PagedKV {
    uint8_t *kp8, *vp8;
    __half *kps, *vps, *ktail, *vtail;
    const int* table;
    int width, n_pages, nkv;
};

// One CTA per SM, at most this many: the workspace holds two partial results of each.
#define SERVE_MAX_CTAS 148
// Paged: sequences of at most this many rows (new tokens x query heads per kv
// head) go to the single-token kernel, longer ones to the tensor-core kernel.
// It is that kernel's one M = 16 tile.  64 contexts of 2048 tokens, 8 kv heads,
// 4 to 16 rows: 40 to 44 us there, 111 in the other; 20 to 128 rows take 122 to
// 129 in the other.
#define SERVE_FEW_ROWS 16

// New rows of packed sequences: sequence s holds rows cu[s]..cu[s+1]-1 of
// n_rows.  Offsets outside [0, n_rows] are clamped, and a sequence whose own two
// are clamped or out of order is reported and skipped, so that no row outside
// the tensors is touched.
struct PackedRows {
    const int* cu;
    int n_seqs, n_rows;
};
__device__ __forceinline__ bool packed_range(const PackedRows& R, int s, int& a, int& b) {
    const int x = R.cu[s], y = R.cu[s + 1];
    a = min(max(x, 0), R.n_rows);
    b = min(max(y, a), R.n_rows);
    return a == x && b == y;
}

// Where the attention's keys come from.
struct AttnArgs {
    const __half* q;
    long long q_stride;  // elements between tokens
    const __half *k, *v; // packed prompts (null: the paged cache)
    long long k_stride, v_stride;
    PackedRows rows;
    const int* kv_lens;  // paged: tokens in the cache, the new ones among them
    int max_q;           // paged: the caller's bound of a sequence's new rows
    PagedKV kv;
    float scale;
    __half* out;         // [n_rows][nh][64]
    int nh, nkv;
    unsigned* err;
};
