// vq_cache_internal.h -- what the source files of the vector-quantised cache share.
#ifndef VQ_CACHE_INTERNAL_H
#define VQ_CACHE_INTERNAL_H

#include <hip/hip_runtime.h>
#include <atomic>
#include <math.h>
#include <stdint.h>

#include "vq_cache.h"
#include "vq_hip.h"

#define VQ_HIDDEN __attribute__((visibility("hidden")))

VQ_HIDDEN int vq_internal_fail(int code, const char *message);
// Lets a kernel take all of the LDS on the current device, once for each (`allowed`: the kernel's own, a bit a device).
VQ_HIDDEN hipError_t vq_internal_allow_lds(const void *kernel, std::atomic<uint64_t> &allowed);

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
typedef __attribute__((ext_vector_type(2))) uint16_t u16x2;

struct AttendArgs {
    const void *q;
    int64_t q_token_stride, q_head_stride, rows;
    int q_heads;
    const void *cb[2];
    int cb_heads, heads, K, Kp;
    const uint8_t *codes[2];
    int64_t pages;
    int page;
    const int32_t *table;
    int seqs, width;
    const int32_t *kv_lens, *starts;
    float scale2;                      // |scale| * log2(e), or fp32's least number: above 0, so that maxima can be taken before it
    uint32_t flip;                     // the sign bits of two 16-bit numbers where scale < 0: q is negated instead
    void *out;
    float *lse;
    bool split;                        // items may be cut between workgroups
    int join_at, join_rows;            // LDS behind the tables: its place, and how many rows' sums fit there
    int seq_at;                        // behind them SEQ_BYTES for a workgroup's range and 64 sequences' rows and lengths
    float *part_o;                     // (slots, rows of an item, D), against part_ml's maximum; two slots a workgroup
    float2 *part_ml;                   // (slots, rows of an item): maximum (base 2) and sum
    struct AttendNote *notes;          // one a workgroup
};

// An item (tile of rows `tile` of sequence `seq`) that begins in one workgroup's part and ends, with tile `end` of all the head's work, in a
// later one's.
struct AttendNote {
    int seq, tile, parts, unused;
    int64_t end, all;
};

struct SearchArgs {
    const void *x[2];
    int64_t token_stride[2], head_stride[2];
    const void *cb[2];
    int64_t tokens;
    int cb_heads, heads, dim, K;
    int pw, chunk;                     // parts a workgroup takes, tokens a wave takes
    const int64_t *slots;              // writing
    int64_t pages;
    int page, page_shift;              // page = 1 << page_shift, or page_shift < 0
    uint8_t *k_codes, *v_codes;
    float *part_sums;                  // training: (chunks, heads * parts, sub + 1, 256), the last plane the counts
    double2 *part_dist;                // (chunks, heads * parts): squared distances and vectors that count
};

struct SearchPlan {
    int pw, chunk, blocks, chunks;
};
// both: 2 where keys and values are searched by one launch
VQ_HIDDEN SearchPlan vq_internal_search_plan(int64_t tokens, int heads, int dim, int sub, int both);
VQ_HIDDEN hipError_t vq_internal_search(const SearchArgs &a, int sub, int dtype, bool train, int blocks, hipStream_t stream);
// What an LBG iteration leaves: sums and dist, or, where cb_new is given, the new codebook and the mean distance.
struct LbgOut {
    int heads, dim, K;
    double *sums;
    int64_t *counts;
    double *dist;
    const float *cb_old;
    float *cb_new;
};
VQ_HIDDEN hipError_t vq_internal_lbg_gather(const SearchArgs &a, int sub, int chunks, const LbgOut &out, hipStream_t stream);

// How an attention call is laid out: RB * 16 rows to a workgroup of NW waves.
struct AttendPlan {
    int rb, nw;
    bool values_in_lds;
    size_t lds;
};

// Launches k_cache_attend and, for several splits, the kernel that joins them; one for each element type.
VQ_HIDDEN hipError_t vq_internal_attend_bf16(const AttendArgs &a, const AttendPlan &p, int dim, int sub, dim3 grid, hipStream_t stream);
VQ_HIDDEN hipError_t vq_internal_attend_f16(const AttendArgs &a, const AttendPlan &p, int dim, int sub, dim3 grid, hipStream_t stream);

constexpr int LDS_MOST = 160 * 1024;
// The least that a workgroup is given: under two tiles a wave, staging and joining outweigh what is shared out (one row of 500 tokens: 10.8 us
// by 16 tiles, 12.8 by 8; of 2000: 14.7 by 16, 13.8 by 8, 16.4 by 32).
constexpr int LEAST_TILES = 16;
// Items that are no longer than this, and for each of which there is a workgroup, are not cut: nothing has to be joined then, and the call is one
// launch.  (One row of 1000 tokens, 32 tiles: 12.5 us whole, 13.5 cut in two, 12.7 in four; of 2000: 16.4 whole, 14.7 in three.  From
// Python a second launch and a workspace take another 4.)
constexpr int WHOLE_TILES = 3 * LEAST_TILES;
// The workgroups a head's work asks for: one for every item at least, since to change items costs as much as several tiles, and a
// multiple of the items, so that those of equal length are cut alike and nobody has to change (4 sequences of 5 rows and 4000 tokens:
// 30 us by 31 workgroups a head, 21 by 32).
__host__ __device__ inline int64_t parts_wanted(int64_t tiles, int64_t items) {
    if (items < 1) return 1;
    const int64_t n = tiles / LEAST_TILES;
    return n <= items ? items : (n + items - 1) / items * items;
}
constexpr int SEQ_BYTES = 64 * 12 + 48;
constexpr int TILE = 32;              // tokens a wave takes at a time: two groups of 16, each inside one page

constexpr int value_chunk(int D, int SUB) {
    int e = SUB;
    while (D % (16 * e)) e /= 2;
    return e;
}
// Key table: part m starts at m * key_stride bytes; the pad keeps the writes of a codebook row's parts in different banks.
__host__ __device__ inline int rows_padded(int K) {
    int p = 1;
    while (p < K) p *= 2;
    return p;
}
__host__ __device__ inline int key_stride(int Kp, int SUB) { return (Kp + 1) * SUB * 2; }
inline size_t key_bytes(int Kp, int D, int SUB) { return ((size_t)(D / SUB) * key_stride(Kp, SUB) + 15) / 16 * 16; }


#endif
