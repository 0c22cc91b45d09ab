// vq_cache_attend.hip -- attention over the paged codes of the vector-quantised cache (vq_cache_attention, vq_cache.h).
// Compiled once for each element type: VQ_CACHE_TYPE and VQ_CACHE_ATTEND, the name of the launching function.
//
// Rows of one cache head (new token i, query head of the group) are taken RB * 16 at a time by one workgroup, whose waves share
// them and take 32-token tiles of the context in turn.  Nothing is expanded into memory: the codebooks of the head lie in LDS, and
// a wave looks its operands of the matrix instructions up there, codes -> registers.
//
//   S^T = K Q^T   (16 tokens) x (16 rows), v_mfma 16x16x32.  A lane holds one token's numbers and 8 dims a step: with the dims
//                 dealt to the four lane groups in quarters, a lane's codes are D / (4 SUB) consecutive bytes and each
//                 look-up of SUB numbers lands in the operand as it is.
//   O^T = V^T P^T (16 dims) x (16 rows) over 32 tokens.  The sum over tokens may run in any order, so a lane group takes the 4 + 4 tokens whose
//                 weights its lanes hold already from the first product: P goes from accumulators to operand without a
//                 shuffle.  A lane looks up E numbers (one chunk of dims) of each of 8 tokens and transposes 8 x E in registers (v_perm); the
//                 codes of 4 tokens are one word of v_codes, which is why those lie part by part.
//   The value table is code-major: 16 lanes read 16 different chunks, so the banks never clash whatever the codes are.  The
//   key table is part-major: 16 lanes read 16 codes of one part, which clash as random numbers do.
//
// What it reaches (8 cache heads, 32 query heads, 128 dims, 256 codewords, parts of 4; bf16) and what bounds it:
//   16 sequences of 20000 tokens on average, a token each: 58 us, 54 here and 5 in the join.  A call on 501 tokens takes 10, nearly all of it tables,
//     range and one chain to the first tile; what is left for the 161 MB of codes is 44 us, 3.7 TB/s.  There one wave's chain (codes, look-ups,
//     products, softmax) is the limit: two waves a SIMD are all that the registers leave.  Of the busy cycles LDS has 49% and clashes of
//     key look-ups 30%, VALU 52%, the matrix unit 17%.
//   2048 new tokens on 16384: 665 us, 775 TFLOP/s, 57% of what the library's plain product reaches.  VALU 64%, LDS 45% and clashes 27%, matrix unit
//     33%: all eight waves hold the same 32 rows, so every tile of tokens is looked up and transposed for each 32 rows anew.
// Measured and not kept: 64 rows to a workgroup (863 us for that chunk, where 32 took 690), 16 waves (75 us where 8 took 62 for
// the 16 sequences).
//
// Softmax in base 2.  A row's weights are taken against a running reference: for bf16 the largest score so far, moved only once a score
// exceeds it by 8 (weights stay below 2^8, sums are fp32), so that most tiles need neither a reduction across lanes nor a rescaling.  Weights are
// rounded to the cache's type for the second product (half a step, as the values themselves are of that type); the sum of weights takes them
// unrounded.  fp16 has 2^-14 to 2^16 for that, so there the reference follows the scores both ways: see Reference.

#include "vq_cache_internal.h"

namespace {

template <typename T> __device__ inline f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c);
template <> __device__ inline f32x4 mfma16<__bf16>(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <> __device__ inline f32x4 mfma16<_Float16>(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <typename T> __device__ inline uint32_t pack2(float lo, float hi);
template <> __device__ inline uint32_t pack2<__bf16>(float lo, float hi) {
    const bf16x2 v = {(__bf16)lo, (__bf16)hi};
    return __builtin_bit_cast(uint32_t, v);
}
template <> __device__ inline uint32_t pack2<_Float16>(float lo, float hi) {
    const f16x2 v = {(_Float16)lo, (_Float16)hi};
    return __builtin_bit_cast(uint32_t, v);
}
// The mean of finite values is none larger than the largest; where the weights' rounding makes it so, it may not become fp16's infinity.
template <typename T> __device__ inline float bounded(float v) { return v; }
template <> __device__ inline float bounded<_Float16>(float v) { return v > 65504.0f ? 65504.0f : v < -65504.0f ? -65504.0f : v; }

// The rows and the length of sequence b, kept inside the tensors whatever the device arrays hold.
__device__ inline void sequence(const AttendArgs &a, int b, int64_t &first, int &n_q, int &n_kv) {
    int64_t s = a.starts[b], e = a.starts[b + 1];
    s = s < 0 ? 0 : (s > a.rows ? a.rows : s);
    e = e < s ? s : (e > a.rows ? a.rows : e);
    const int64_t most = (int64_t)a.width * a.page;
    const int n = a.kv_lens[b];
    first = s;
    n_q = (int)(e - s);
    n_kv = n < 0 ? 0 : (n > most ? (int)most : n);
}

// Addresses that come out of registers say that they are global memory's: a flat load would count as an LDS access too, and every
// wait for a look-up would wait for it.
#define GLOBAL __attribute__((address_space(1)))
typedef const GLOBAL uint8_t *global_bytes;

// NB consecutive bytes from an address that is a multiple of the largest power of two in NB (16 at most).
template <int NB> __device__ inline void load_bytes(uint32_t *w, global_bytes p) {
    if constexpr (NB % 16 == 0) {
#pragma unroll
        for (int i = 0; i < NB / 16; ++i) {
            const u32x4 v = *(const GLOBAL u32x4 *)(p + 16 * i);
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    } else if constexpr (NB % 8 == 0) {
#pragma unroll
        for (int i = 0; i < NB / 8; ++i) {
            const u32x2 v = *(const GLOBAL u32x2 *)(p + 8 * i);
            w[2 * i] = v.x, w[2 * i + 1] = v.y;
        }
    } else if constexpr (NB % 4 == 0) {
#pragma unroll
        for (int i = 0; i < NB / 4; ++i) w[i] = *(const GLOBAL uint32_t *)(p + 4 * i);
    } else if constexpr (NB % 2 == 0) {
#pragma unroll
        for (int i = 0; i < (NB + 3) / 4; ++i) {
            w[i] = *(const GLOBAL uint16_t *)(p + 4 * i);
            if (4 * i + 2 < NB) w[i] |= (uint32_t)*(const GLOBAL uint16_t *)(p + 4 * i + 2) << 16;
        }
    } else {
        w[0] = 0;
#pragma unroll
        for (int i = 0; i < NB; ++i) w[0] |= (uint32_t)p[i] << (8 * i);
    }
}

// Look-ups name LDS by its byte offset: the kernel has no other LDS, so s_mem lies at 0, and an address is what the code and
// the lane make of it without a base to be added each time.
template <typename V> __device__ inline V lds(uint32_t at) { return *(const __attribute__((address_space(3))) V *)(uintptr_t)at; }

// A barrier that waits for LDS alone: loads and stores of global memory stay under way.
__device__ inline void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// The maximum over the four lanes of one row, to each of them, by the VALU alone: a shuffle through LDS would wait for the look-ups under way.
__device__ inline float wave_any_max(float v) {
    uint32_t bits = __builtin_bit_cast(uint32_t, v);
    const auto rows = __builtin_amdgcn_permlane16_swap(bits, bits, false, false);       // rows 0, 0, 2, 2 and 1, 1, 3, 3 of 16 lanes
    const uint32_t even = rows[0], odd = rows[1];
    bits = __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, even), __builtin_bit_cast(float, odd)));
    const auto halves = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
    const uint32_t low = halves[0], high = halves[1];
    return fmaxf(__builtin_bit_cast(float, low), __builtin_bit_cast(float, high));
}

// A value that every lane holds, in scalar registers: what follows from it stays there.
__device__ inline int64_t uniform(int64_t v) {
    return (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)v) | (int64_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32;
}

// v of the lane that the DPP control names, 0 where it names none or ROWS leaves this row of 16 lanes out.
template <int CONTROL, int ROWS> __device__ inline int64_t moved(int64_t v) {
    const int lo = __builtin_amdgcn_update_dpp(0, (int)v, CONTROL, ROWS, 0xf, false);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), CONTROL, ROWS, 0xf, false);
    return (int64_t)(uint32_t)lo | (int64_t)hi << 32;
}
// The sum over the lanes up to this one.
__device__ inline int64_t running(int64_t v) {
    v += moved<0x111, 0xf>(v);       // one, two, four and eight lanes to the right inside a row
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);       // the last lane of a row to all of the next, for the second and the fourth
    v += moved<0x143, 0xc>(v);       // lane 31 to the upper half
    return v;
}
__device__ inline int64_t of_last_lane(int64_t v) {
    return (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)v, 63) | (int64_t)__builtin_amdgcn_readlane((int)(v >> 32), 63) << 32;
}

// 8 numbers of a finished row, place = row * q_heads + head: v against the reference `most` (base 2) and the sum of weights.
template <typename T>
__device__ inline void store_row(const AttendArgs &a, int64_t place, int D, int c, f32x4 v0, f32x4 v1, float most, float sum) {
    const float over = sum == 0.0f ? 0.0f : 1.0f / sum;              // 0: the row sees no token (of any other the largest weight is 1 or more)
    *reinterpret_cast<u32x4 *>(static_cast<T *>(a.out) + place * D + c * 8) =
        (u32x4){pack2<T>(bounded<T>(v0[0] * over), bounded<T>(v0[1] * over)), pack2<T>(bounded<T>(v0[2] * over), bounded<T>(v0[3] * over)),
                pack2<T>(bounded<T>(v1[0] * over), bounded<T>(v1[1] * over)), pack2<T>(bounded<T>(v1[2] * over), bounded<T>(v1[3] * over))};
    // (the sum's power of two goes to `most` first: where the reference came down far, the two are large and nearly cancel)
    if (c == 0 && a.lse)
        a.lse[place] = sum == 0.0f ? -INFINITY : ((most + (float)__builtin_amdgcn_frexp_expf(sum)) + log2f(__builtin_amdgcn_frexp_mantf(sum))) * 0.69314718055994531f;
}

// From here on a score's rounding is no longer small against 1: scores are then rounded as their maximum was before it is taken off, so that the
// largest weight is what the reference says.  (Multiplied and subtracted at once, a score of 10^10 missed its own maximum by up to
// 2^9, and its weight was infinite or nothing.)
constexpr float LARGE = 0x1p20f;

// How a row's reference follows its scores.  It is moved where a tile's largest weight leaves 2^LEAST .. 2^MOST, to where that is 2^AIM; for bf16,
// whose weights have fp32's range, to the maximum itself and never down.  In fp16 a weight below 2^-14 loses bits and one below 2^-25 is
// nothing, and a reference that only rose would do that to all tokens of a wave behind one heavy token: with a heavy token whose value is zero
// and 20000 others 17 to 26 nats below it, an eighth of the result was lost.  With one that comes down again a weight is off by half a
// step, or by 2^-19 of the largest in its own tile (2^-33 where that has just moved the reference).  The reference lies a whole number below
// the score that moved it, so that this one's weight is exact, as that of a row's only token.  It comes down only as far as
// the row's sum stays below 2^93 (the products' sums, up to 2^16 times that, then stay inside fp32).  Scores of a few nats move it no oftener
// than before (512 rows on 8192 tokens, 128 dims by 4: 128 us); with a deviation of 4 nats it takes 140 us where 125 were, of 8 nats 151.
template <typename T> struct Reference {
    static constexpr bool BOTH_WAYS = false;
    static constexpr float MOST = 8.0f;
};
template <> struct Reference<_Float16> {
    static constexpr bool BOTH_WAYS = true;
    static constexpr float MOST = 15.0f, AIM = 8.0f, LEAST = -6.0f;
    static constexpr int SUM_MOST = 90;
};

// The tiles that the rows of one item see: rows tile * RB * 16 on of a sequence, whose row i sees tokens 0 .. n_kv - n_q + i.
template <int RB> __device__ inline int tiles_of(int tile, int n_q, int n_kv, int group) {
    const int n_rows = n_q * group, past = (tile + 1) * RB * 16;
    const int end = n_kv - n_q + ((past < n_rows ? past : n_rows) - 1) / group + 1;
    return end <= 0 ? 0 : (end - 1) / TILE + 1;                      // (end may be near 2^31)
}
// What an item counts in the division of the work: its tiles, and one where it has none but zeros to be written.
template <int RB> __device__ inline int cost_of(int tile, int n_q, int n_kv, int group) {
    const int n = tiles_of<RB>(tile, n_q, n_kv, group);
    return n < 1 ? 1 : n;
}

// Where a part of the work begins: parts of equal length, to a tile; it rises with the part, and both kernels work it out alike.
__device__ inline int64_t part_begin(int64_t all, int parts, int part) {
    return part >= parts ? all : (int64_t)((double)all / (double)parts * (double)part);
}

// One head's work is all its items side by side, (sequence, tile of rows) after (sequence, tile of rows), cut into as many equal
// ranges of tiles as there are workgroups: causal and ragged lengths are balanced by themselves, and a workgroup stages its tables once.
// A range may begin and end inside an item.  Such an item's parts go to the workspace (`slots`, two a workgroup: the part that begins
// an item and the part that does not), and the workgroup that holds its beginning notes it for k_cache_join.  Without `split` an item
// counts as one, whatever its length, and is never cut.
struct Range {
    int64_t left, skip, now, all;      // tiles to be done, of them already done by others in the first item, where that begins; all of the head's
    int seq, tile, held, parts;        // the first item; the first of the 64 sequences beside this
};
template <typename T, int D, int SUB, int RB, int NW, bool VLDS>
__global__ __launch_bounds__(NW * 64) void k_cache_attend(const AttendArgs a) {
    constexpr int M = D / SUB, KS = D / 32, NB = M / 4, KW = (NB + 3) / 4;
    constexpr int E = value_chunk(D, SUB), U = D / (16 * E), ROWS = RB * 16;
    extern __shared__ __align__(16) uint8_t s_mem[];
    if ((uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)s_mem != 0) return;      // (never: see lds())
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = blockIdx.x, group = a.q_heads / a.heads;
    // Up to 128 dims the tables have room for 256 codewords whatever K is: any code is inside them as it is, and a look-up's part is
    // an offset in its instruction.
    const int Kp = D <= 128 ? 256 : a.Kp, kstride = key_stride(Kp, SUB);
    const int k_at = VLDS ? Kp * D * 2 : 0;                       // the value table comes first: see look-ups
    const int64_t cb0 = a.cb_heads == 1 ? 0 : (int64_t)h * a.K * D;
    const T *k_cb = static_cast<const T *>(a.cb[0]) + cb0, *v_cb = static_cast<const T *>(a.cb[1]) + cb0;
    const int page16 = a.page >> 4;
    const uint32_t fold = D <= 128 ? ~0u : (uint32_t)(Kp - 1) * 0x01010101u;      // keeps codes of no codeword inside the tables
    const int64_t page_bytes = (int64_t)a.heads * a.page * M;
    const int64_t head_at = (int64_t)h * a.page * M;
    const uint32_t k_lane = r * M + g * NB;
    uint32_t v_lane[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v_lane[u] = ((u * 16 + r) * E / SUB) * a.page + 4 * g;

    // Codebooks -> LDS, 16 bytes at a time, several loads under way at once; rows past K are zeros.  The first loads leave now and
    // are on their way while the range is worked out.
    constexpr int BATCH = D <= 128 ? 8 : 4;
    u32x4 stage_k[BATCH], stage_v[VLDS ? BATCH : 1];
    auto stage_load = [&](int i0) {
#pragma unroll
        for (int x = 0; x < BATCH; ++x) {
            const int i = i0 + x * NW * 64;
            stage_k[x] = (u32x4){0, 0, 0, 0};
            if constexpr (VLDS) stage_v[x] = (u32x4){0, 0, 0, 0};
            if (i < a.K * (D / 8)) {
                stage_k[x] = *reinterpret_cast<const u32x4 *>(k_cb + (int64_t)i * 8);
                if constexpr (VLDS) stage_v[x] = *reinterpret_cast<const u32x4 *>(v_cb + (int64_t)i * 8);
            }
        }
    };
    auto stage_store = [&](int i0) {
#pragma unroll
        for (int x = 0; x < BATCH; ++x) {
            const int i = i0 + x * NW * 64, k = i / (D / 8), c = i % (D / 8);
            if (i >= Kp * (D / 8)) continue;
            if constexpr (SUB == 8) {
                *reinterpret_cast<u32x4 *>(s_mem + k_at + c * kstride + k * 16) = stage_k[x];
            } else if constexpr (SUB == 4) {
                *reinterpret_cast<u32x2 *>(s_mem + k_at + (2 * c) * kstride + k * 8) = stage_k[x].xy;
                *reinterpret_cast<u32x2 *>(s_mem + k_at + (2 * c + 1) * kstride + k * 8) = stage_k[x].zw;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) *reinterpret_cast<uint32_t *>(s_mem + k_at + (4 * c + j) * kstride + k * 4) = stage_k[x][j];
            }
            if constexpr (VLDS) *reinterpret_cast<u32x4 *>(s_mem + i * 16) = stage_v[x];
        }
    };
    // This workgroup's range, worked out by one wave while the tables arrive, and left in LDS with the rows and lengths of 64 sequences.  (One
    // row on 500 tokens: 10.0 us; all eight waves working it out for themselves 10.8.)  The sequences' loads go before the tables':
    // loads come back in order.
    int *s_seq = reinterpret_cast<int *>(s_mem + a.seq_at);
    Range *s_range = reinterpret_cast<Range *>(s_seq + 64 * 3);
    const int me = h * gridDim.y + blockIdx.y;
    int64_t seq_first = 0;
    int seq_q = 0, seq_kv = 0;                                    // a lane's sequence
    if (wave == 0 && lane < a.seqs) sequence(a, lane, seq_first, seq_q, seq_kv);
    __builtin_amdgcn_sched_barrier(0);
    stage_load(threadIdx.x);
    __builtin_amdgcn_sched_barrier(0);
    if (wave == 0) {
        int64_t items = 0;
        int held = 0;                                             // the lanes hold the sequences from here on: 64 at a time,
        auto costs_from = [&](int b0) -> int64_t {                // and their running cost; the tiles of rows of a long one go 64 at a time too
            int64_t sum = 0;
            if (b0 != held) {
                seq_first = 0, seq_q = seq_kv = 0;
                if (b0 + lane < a.seqs) sequence(a, b0 + lane, seq_first, seq_q, seq_kv);
                held = b0;
            }
            const int tiles = (seq_q * group + ROWS - 1) / ROWS;
            items += of_last_lane(running(tiles));
            if (!a.split) sum = tiles;
            else if (tiles == 1) sum = cost_of<RB>(0, seq_q, seq_kv, group);
            for (uint64_t todo = a.split ? __ballot(tiles > 1) : 0; todo; todo &= todo - 1) {
                const int of = __builtin_ctzll(todo), x_q = __shfl(seq_q, of), x_kv = __shfl(seq_kv, of), x_tiles = __shfl(tiles, of);
                int64_t part = 0;
                for (int t = lane; t < x_tiles; t += 64) part += cost_of<RB>(t, x_q, x_kv, group);
                part = of_last_lane(running(part));
                if (lane == of) sum = part;
            }
            return running(sum);
        };
        int64_t costs = costs_from(0), all = of_last_lane(costs);
        for (int b0 = 64; b0 < a.seqs; b0 += 64) {
            costs = costs_from(b0);
            all += of_last_lane(costs);
        }
        const int64_t most_parts = a.split ? parts_wanted(all, items) : items < 1 ? 1 : items;
        const int parts = most_parts > (int64_t)gridDim.y ? (int)gridDim.y : (int)most_parts;
        const int64_t begin = uniform(part_begin(all, parts, blockIdx.y)), past = uniform(part_begin(all, parts, blockIdx.y + 1));
        const int64_t left = (int)blockIdx.y < parts && begin < past ? past - begin : 0;
        int64_t skip = begin;                                     // first: of the work before sequence b; then of item (b, tile)
        int b = 0, tile = 0, at;
        auto locate = [&](int64_t sum) -> bool {                  // sum: the lanes' running costs; finds the lane that skip falls to
            const bool here = skip < of_last_lane(sum);
            at = here ? __builtin_ctzll(__ballot(sum > skip)) : 64;
            skip -= at > 0 ? uniform(__shfl(sum, at - 1)) : 0;
            return here;
        };
        for (int b0 = 0; left > 0 && b0 < a.seqs; b0 += 64) {
            if (b0 != held) costs = costs_from(b0);
            const bool here = locate(costs);
            b = b0 + at;
            if (here) break;
        }
        int n_q = 0, n_kv = 0;
        if (left > 0 && b < a.seqs) n_q = __builtin_amdgcn_readlane(seq_q, b - held), n_kv = __builtin_amdgcn_readlane(seq_kv, b - held);
        const int tiles = (n_q * group + ROWS - 1) / ROWS;
        for (int t0 = 0; tiles > 1 && t0 < tiles; t0 += 64) {
            const int t = t0 + lane;
            const bool here = locate(running(t >= tiles ? 0 : a.split ? cost_of<RB>(t, n_q, n_kv, group) : 1));
            tile = t0 + at;
            if (here) break;
        }
        s_seq[3 * lane] = (int)seq_first, s_seq[3 * lane + 1] = seq_q, s_seq[3 * lane + 2] = seq_kv;
        if (lane == 0) *s_range = Range{left, skip, begin - skip, all, b, tile, held, parts};
    }
    stage_store(threadIdx.x);
    for (int i0 = threadIdx.x + BATCH * NW * 64; i0 < Kp * (D / 8); i0 += BATCH * NW * 64) {
        stage_load(i0);
        stage_store(i0);
    }
    __syncthreads();

    int64_t left = uniform(s_range->left), skip = uniform(s_range->skip), now = uniform(s_range->now);      // now: where item (b, tile) begins
    int b = __builtin_amdgcn_readfirstlane(s_range->seq), tile = __builtin_amdgcn_readfirstlane(s_range->tile);
    int held = __builtin_amdgcn_readfirstlane(s_range->held);
    int first = 0, n_q = 0, n_kv = 0;
    // Rows and length of sequence b: out of LDS for all waves alike, so that they come to every barrier together whatever becomes of the
    // tensors meanwhile; the next 64 are fetched by one wave.
    auto take_sequence = [&]() {
        if (b - held >= 64) {
            lds_barrier();
            if (wave == 0) {
                int64_t x = 0;
                int y = 0, z = 0;
                if (b + lane < a.seqs) sequence(a, b + lane, x, y, z);
                s_seq[3 * lane] = (int)x, s_seq[3 * lane + 1] = y, s_seq[3 * lane + 2] = z;
            }
            held = b;
            lds_barrier();
        }
        first = __builtin_amdgcn_readfirstlane(s_seq[3 * (b - held)]);
        n_q = __builtin_amdgcn_readfirstlane(s_seq[3 * (b - held) + 1]);
        n_kv = __builtin_amdgcn_readfirstlane(s_seq[3 * (b - held) + 2]);
    };
    AttendNote note = {-1, 0, 0, 0, 0, 0};

    // The item in hand, from its first loads on.
    int take = 0, cost = 1, row0 = 0, rows_here = 0, lo = 0, hi = 0, all_see = 0;
    const int32_t *table = a.table;
    u32x4 q[RB][KS];
    int sees[RB];
    // A wave's tiles: lo + wave, then every NW-th.  Where their codes lie is worked out for 32 tiles at a time, a lane for each half of a
    // tile (16 tokens, inside one page); a turn then takes its four addresses out of the lanes.  (Page numbers fetched and
    // multiplied out turn by turn took longer than all the rest: a wave waits for every scalar step.)
    // Codes are fetched AHEAD tiles before their use.
    constexpr int AHEAD = 2;
    int t = lo + wave, fetched = 0;                           // the tile in hand; how many have been fetched
    uint64_t k_ptr = 0, v_ptr = 0, there = 0;                 // a lane's addresses; one bit a lane: its tokens lie in a page of the cache
    auto place = [&]() {
        const int tile32 = lo + wave + (fetched + (lane & 31)) * NW, group16 = 2 * tile32 + (lane >> 5);
        const int at = group16 / page16, y = group16 - at * page16;
        const bool in = tile32 < hi && group16 * 16 < n_kv;
        const int n = in ? table[at] : -1;
        const bool good = n >= 0 && n < a.pages;
        const int64_t from = good ? (int64_t)n * page_bytes + head_at : head_at;      // (else page 0: read, not looked at)
        k_ptr = (uint64_t)(a.codes[0] + (from + (int64_t)(good ? y : 0) * 16 * M));
        v_ptr = (uint64_t)(a.codes[1] + (from + (good ? y : 0) * 16));
        there = __ballot(good);
    };
    auto of_lane = [](uint64_t v, int from) -> global_bytes {
        return (global_bytes)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)v, from) |
                              (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), from) << 32);
    };
    uint32_t kc[AHEAD][2][KW], vc[AHEAD][2][U], seen[AHEAD];   // seen: bits 0 and 1: the tile's halves are there
    auto fetch = [&](int slot) {
        const int at = fetched & 31;
        if (at == 0) place();
        seen[slot] = (uint32_t)(there >> at) & 1u | ((uint32_t)(there >> (32 + at)) & 1u) << 1;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            load_bytes<NB>(kc[slot][s], of_lane(k_ptr, 32 * s + at) + k_lane);
            const global_bytes from = of_lane(v_ptr, 32 * s + at);
#pragma unroll
            for (int u = 0; u < U; ++u) vc[slot][s][u] = *(const GLOBAL uint32_t *)(from + v_lane[u]);
        }
        ++fetched;
    };
    static_assert(AHEAD == 2, "turns go by twos");
    // Sends off the loads of item (b, tile): queries, page numbers, the codes of a wave's first tiles.
    auto open = [&]() {
        const int tiles = tiles_of<RB>(tile, n_q, n_kv, group), n_rows = n_q * group, back = n_kv - n_q;     // row i sees tokens 0 .. back + i
        cost = !a.split || tiles < 1 ? 1 : tiles;
        take = (int)(left < cost - skip ? left : cost - skip);
        lo = (int)skip < tiles ? (int)skip : tiles, hi = a.split && (int)skip + take < tiles ? (int)skip + take : tiles;
        table = a.table + (int64_t)b * a.width;
        row0 = tile * ROWS, rows_here = n_rows - row0 < ROWS ? n_rows - row0 : ROWS;
        all_see = back + row0 / group;                            // every row of the item sees tokens up to here
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int row = rb * 16 + r < rows_here ? row0 + rb * 16 + r : row0;
            const int i = row / group, head = h * group + row % group;
            const T *p = static_cast<const T *>(a.q) + (int64_t)(first + i) * a.q_token_stride + head * a.q_head_stride + g * (D / 4);
            sees[rb] = back + i;
#pragma unroll
            for (int s = 0; s < KS; ++s) q[rb][s] = *reinterpret_cast<const u32x4 *>(p + 8 * s);
        }
        t = lo + wave, fetched = 0;
        if (t < hi) {
            fetch(0);
            fetch(1);
        }
    };
    // On to the next item; false where there is none.
    auto advance = [&]() -> bool {
        left -= take;
        now += cost;
        skip = 0;
        ++tile;
        while (left > 0 && tile * ROWS >= n_q * group) {
            tile = 0;
            if (++b >= a.seqs) return false;
            take_sequence();
        }
        return left > 0;
    };
    bool more = left > 0 && b < a.seqs;
    if (more) {
        take_sequence();
        open();
    }
    while (more) {
        f32x4 o[RB][U][E];
        float top[RB], total[RB];
        bool large = false;                                       // some row's reference is LARGE
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            top[rb] = -INFINITY;
            total[rb] = 0.0f;
#pragma unroll
            for (int s = 0; s < KS; ++s) q[rb][s] ^= a.flip;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < E; ++e) o[rb][u][e] = (f32x4){0, 0, 0, 0};
        }
        // Look-ups.  Up to 128 dims all of a tile's go first, so that they pass through LDS one behind the other; beyond, registers are
        // short and they go one step before their use.  Either way the tile's codes are done with before the next ones are fetched to
        // their registers: where old and new are both alive, the new ones are copied, and a copy waits for its load.
        constexpr bool FIRST = D <= 128;
        auto look_k = [&](uint32_t const (&codes)[KW], int ks) -> u32x4 {
            u32x4 x;
#pragma unroll
            for (int j = 0; j < 8 / SUB; ++j) {
                const int n = ks * (8 / SUB) + j;                // the lane's n-th part, g * NB + n of the vector
                const uint32_t code = ((codes[n / 4] & fold) >> (8 * (n % 4))) & 255u;
                const uint32_t at = k_at + g * NB * kstride + n * kstride + code * (SUB * 2);
                if constexpr (SUB == 8) x = lds<u32x4>(at);
                else if constexpr (SUB == 4) {
                    const u32x2 v = lds<u32x2>(at);
                    x[2 * j] = v.x, x[2 * j + 1] = v.y;
                } else x[j] = lds<uint32_t>(at);
            }
            return x;
        };
        auto look_v = [&](uint32_t c0, uint32_t c1, int u, uint32_t (&x)[8][E / 2]) {
            const uint32_t codes[2] = {c0 & fold, c1 & fold};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                uint32_t at;
                if constexpr (VLDS && D == 128) {
                    // a row has 256 bytes: the code is the second byte of the address, put there with the first in one go
                    at = __builtin_amdgcn_perm(codes[j / 4], (uint32_t)(r * E * 2), 0x0c0c0000u | (4u + j % 4) << 8);
                } else {
                    uint32_t code = (codes[j / 4] >> (8 * (j % 4))) & 255u;
                    if constexpr (!VLDS) code = code < (uint32_t)a.K ? code : (uint32_t)a.K - 1;
                    at = code * (D * 2) + r * E * 2;
                }
                at += u * 16 * E * 2;
                const uint8_t *from = reinterpret_cast<const uint8_t *>(v_cb) + (VLDS ? 0 : at);
                if constexpr (E == 8) {
                    const u32x4 v = VLDS ? lds<u32x4>(at) : *reinterpret_cast<const u32x4 *>(from);
                    x[j][0] = v.x, x[j][1] = v.y, x[j][2] = v.z, x[j][3] = v.w;
                } else if constexpr (E == 4) {
                    const u32x2 v = VLDS ? lds<u32x2>(at) : *reinterpret_cast<const u32x2 *>(from);
                    x[j][0] = v.x, x[j][1] = v.y;
                } else x[j][0] = VLDS ? lds<uint32_t>(at) : *reinterpret_cast<const uint32_t *>(from);
            }
        };
        auto turn = [&](int slot) {
            f32x4 z[RB][2];
            uint32_t vx[FIRST ? U : 1][8][E / 2];
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) z[rb][0] = z[rb][1] = (f32x4){0, 0, 0, 0};
            const uint32_t have = seen[slot];
            if constexpr (FIRST) {
                u32x4 kx[2][KS];
                auto values = [&]() {
#pragma unroll
                    for (int u = 0; u < U; ++u) look_v(vc[slot][0][u], vc[slot][1][u], u, vx[u]);
                    __builtin_amdgcn_sched_barrier(0);
                    fetch(slot);
                };
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) kx[0][ks] = look_k(kc[slot][0], ks), kx[1][ks] = look_k(kc[slot][1], ks);
                if constexpr (RB == 1) values();
                else __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int s = 0; s < 2; ++s)
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) z[rb][s] = mfma16<T>(kx[s][ks], q[rb][ks], z[rb][s]);
                if constexpr (RB > 1) {                          // (more rows: the values take the keys' registers)
                    __builtin_amdgcn_sched_barrier(0);
                    values();
                }
            } else {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const u32x4 x = look_k(kc[slot][s], ks);
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) z[rb][s] = mfma16<T>(x, q[rb][ks], z[rb][s]);
                    }
            }
            // weights
            u32x4 w[RB];
            const bool whole = have == 3 && t * TILE + TILE - 1 <= all_see;
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                float by = large ? 1.0f : a.scale2;               // what is still to be multiplied by
                if (__builtin_expect(!whole || large, 0)) {
                    const float times = large ? a.scale2 : 1.0f;
#pragma unroll
                    for (int s = 0; s < 2; ++s)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            z[rb][s][i] = !(have >> s & 1) || t * TILE + 16 * s + 4 * g + i > sees[rb] ? -INFINITY : z[rb][s][i] * times;
                }
                float best = -INFINITY;
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) best = fmaxf(best, z[rb][s][i]);
                best *= by;
                using Ref = Reference<T>;
                bool leaves = best - top[rb] > Ref::MOST;         // (not best > top + MOST: large scores would round it away)
                if constexpr (Ref::BOTH_WAYS) leaves = leaves || best - top[rb] < Ref::LEAST;
                if (__builtin_expect(__any(leaves), 0)) {         // (both rare ways out of line: a chunk of 2048 rows is 2% faster so)
                    const float most = wave_any_max(best);
                    float now = fmaxf(top[rb], most);
                    if constexpr (Ref::BOTH_WAYS) {               // (most tiles that come here have a lane's 8 tokens below the row's 32, no more)
                        const bool falls = most - top[rb] < Ref::LEAST && most > -INFINITY;
                        const float aim = fabsf(most) < LARGE ? most - Ref::AIM : most;
                        now = most - top[rb] > Ref::MOST ? aim : top[rb];
                        if (__any(falls)) {
                            // (a lane has a quarter of its row's sum, and its exponent leaves out up to a bit more)
                            const float room = (float)(Ref::SUM_MOST + 127 - (int)(__builtin_bit_cast(uint32_t, wave_any_max(total[rb])) >> 23));
                            if (falls) now = fmaxf(aim, top[rb] - fmaxf(room, 0.0f));
                        }
                    }
                    if (!Ref::BOTH_WAYS || __any(now != top[rb])) {
                        const float keep = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top[rb] - now);
                        top[rb] = now;
                        total[rb] *= keep;
#pragma unroll
                        for (int u = 0; u < U; ++u)
#pragma unroll
                            for (int e = 0; e < E; ++e) o[rb][u][e] *= keep;
                        if (!large && __any(fabsf(now) >= LARGE && now > -INFINITY)) {
                            large = true, by = 1.0f;
#pragma unroll
                            for (int s = 0; s < 2; ++s)
#pragma unroll
                                for (int i = 0; i < 4; ++i) z[rb][s][i] *= a.scale2;
                        }
                    }
                }
                const float base = top[rb] == -INFINITY ? 0.0f : -top[rb];
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) z[rb][s][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[rb][s][i], by, base));
                total[rb] += ((z[rb][0][0] + z[rb][0][1]) + (z[rb][0][2] + z[rb][0][3])) + ((z[rb][1][0] + z[rb][1][1]) + (z[rb][1][2] + z[rb][1][3]));
                w[rb] = (u32x4){pack2<T>(z[rb][0][0], z[rb][0][1]), pack2<T>(z[rb][0][2], z[rb][0][3]),
                                pack2<T>(z[rb][1][0], z[rb][1][1]), pack2<T>(z[rb][1][2], z[rb][1][3])};
            }
            // values: E numbers of 8 tokens, transposed to E operands of 8 tokens
#pragma unroll
            for (int u = 0; u < U; ++u) {
                uint32_t(&x)[8][E / 2] = vx[FIRST ? u : 0];
                if constexpr (!FIRST) look_v(vc[slot][0][u], vc[slot][1][u], u, x);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    u32x4 v;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        v[j] = __builtin_amdgcn_perm(x[2 * j + 1][e / 2], x[2 * j][e / 2], e % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) o[rb][u][e] = mfma16<T>(v, w[rb], o[rb][u][e]);
                }
            }
            if constexpr (!FIRST) {
                __builtin_amdgcn_sched_barrier(0);
                fetch(slot);
            }
            t += NW;
        };
        __builtin_amdgcn_s_waitcnt(0x0f70);                       // all loads: inside the loop no wait is left but those of the codes
        // The two waves of a SIMD take turns in going first: left to itself the older one does, and the younger's last tiles are done with nobody
        // to fill its waits (80 and 92 thousand cycles for 39 tiles each).
        bool ahead = wave < NW / 2;
        while (t + NW < hi) {                                     // (left in one place only: leaving after the first turn as well would make
            if (ahead) __builtin_amdgcn_s_setprio(1);             // every wait for its codes one for all loads)
            else __builtin_amdgcn_s_setprio(0);
            ahead = !ahead;
            turn(0);
            turn(1);
        }
        __builtin_amdgcn_s_setprio(0);
        if (t < hi) turn(0);

        // The next item's loads leave before this one's rows are joined, where there are registers for both.
        constexpr bool EARLY = RB * D <= 192;
        const bool whole_item = take == cost;
        const int slot = 2 * me + (skip == 0 ? 1 : 0), its_first = first, its_row0 = row0, its_rows = rows_here;
        if (!whole_item && skip == 0) note = AttendNote{b, tile, s_range->parts, 0, now + cost - 1, s_range->all};
        more = advance();
        if (EARLY && more) open();

        // Join the waves: maxima and sums first, then every wave's part weighted by its maximum, added in the waves' order, as many
        // waves at a time as LDS has room for beside the tables.
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            total[rb] += __shfl_xor(total[rb], 16);
            total[rb] += __shfl_xor(total[rb], 32);
        }
        float2 *s_ml = reinterpret_cast<float2 *>(s_mem + a.join_at);
        float *s_o = reinterpret_cast<float *>(s_mem + a.join_at + NW * ROWS * 8);
        if (g == 0)
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) s_ml[wave * ROWS + rb * 16 + r] = make_float2(top[rb], total[rb]);
        constexpr int EACH = (16 * (D / 8) + NW * 64 - 1) / (NW * 64);         // pieces of 8 numbers a thread adds up
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int rows_rb = its_rows - rb * 16 < 16 ? its_rows - rb * 16 : 16;
            if (rows_rb <= 0) break;
            if (rb > 0) lds_barrier();                          // the sums of the rows before go to the same place
            const int at_once = a.join_rows / rows_rb;
            f32x4 v0[EACH], v1[EACH];
            float weight[EACH][NW], most[EACH], sum[EACH];
            for (int w0 = 0; w0 < NW; w0 += at_once) {
                if (wave >= w0 && wave < w0 + at_once && r < rows_rb) {
                    f32x4 *p = reinterpret_cast<f32x4 *>(s_o + ((wave - w0) * rows_rb + r) * (D + 4)) + g * E;
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int j = 0; j < E; ++j) {            // 4 chunks of E numbers side by side, written four numbers at a time
                            f32x4 v;
#pragma unroll
                            for (int n = 0; n < 4; ++n) v[n] = o[rb][u][(4 * j + n) % E][(4 * j + n) / E];
                            p[u * 4 * E + j] = v;
                        }
                }
                lds_barrier();
#pragma unroll
                for (int n = 0; n < EACH; ++n) {
                    const int i = threadIdx.x + n * NW * 64, x = i / (D / 8), c = i % (D / 8);
                    if (x >= rows_rb) continue;
                    if (w0 == 0) {
                        v0[n] = v1[n] = (f32x4){0, 0, 0, 0};
                        float2 ml[NW];
#pragma unroll
                        for (int y = 0; y < NW; ++y) ml[y] = s_ml[y * ROWS + rb * 16 + x];
                        most[n] = -INFINITY, sum[n] = 0.0f;
#pragma unroll
                        for (int y = 0; y < NW; ++y) most[n] = fmaxf(most[n], ml[y].x);
#pragma unroll
                        for (int y = 0; y < NW; ++y) {
                            weight[n][y] = ml[y].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml[y].x - most[n]);
                            sum[n] += ml[y].y * weight[n][y];
                        }
                    }
#pragma unroll
                    for (int y = 0; y < NW; ++y) {
                        if (y < w0 || y >= w0 + at_once) continue;
                        const float *p = s_o + ((y - w0) * rows_rb + x) * (D + 4) + c * 8;
                        v0[n] += *reinterpret_cast<const f32x4 *>(p) * weight[n][y];
                        v1[n] += *reinterpret_cast<const f32x4 *>(p + 4) * weight[n][y];
                    }
                }
                if (w0 + at_once < NW) lds_barrier();
            }
#pragma unroll
            for (int n = 0; n < EACH; ++n) {
                const int i = threadIdx.x + n * NW * 64, x = i / (D / 8), c = i % (D / 8);
                if (x >= rows_rb) continue;
                if (whole_item) {
                    const int row = its_row0 + rb * 16 + x;
                    store_row<T>(a, (int64_t)(its_first + row / group) * a.q_heads + h * group + row % group, D, c, v0[n], v1[n], most[n], sum[n]);
                } else {
                    const int64_t at = (int64_t)slot * ROWS + rb * 16 + x;
                    float *p = a.part_o + at * D + c * 8;
                    *reinterpret_cast<f32x4 *>(p) = v0[n];
                    *reinterpret_cast<f32x4 *>(p + 4) = v1[n];
                    if (c == 0) a.part_ml[at] = make_float2(most[n], sum[n]);
                }
            }
        }
        lds_barrier();                                            // the next item's sums go to the same place
        if (!EARLY && more) open();
    }
    if (a.split && threadIdx.x == 0) a.notes[me] = note;
}

// Joins an item's parts: the one of the workgroup that noted it, then the others in order.  4 to 6 us, nearly all of it the launch and two
// trips to memory; a workgroup without a note ends at once.
template <typename T, int D, int RB>
__global__ __launch_bounds__(256) void k_cache_join(const AttendArgs a) {
    constexpr int ROWS = RB * 16;
    const int h = blockIdx.x, me = h * gridDim.y + blockIdx.y, group = a.q_heads / a.heads;
    const AttendNote note = a.notes[me];
    if (note.seq < 0) return;
    int64_t first;
    int n_q, n_kv;
    sequence(a, note.seq, first, n_q, n_kv);
    int last = (int)((double)note.end / ((double)note.all / (double)note.parts));      // the part that the item's last tile falls to, to one or two
    last = last < note.parts - 1 ? last : note.parts - 1;
    while (last > 0 && part_begin(note.all, note.parts, last) > note.end) --last;
    while (last < note.parts - 1 && part_begin(note.all, note.parts, last + 1) <= note.end) ++last;
    const int pieces = last - (int)blockIdx.y + 1;
    auto slot = [&](int s) -> int64_t { return s == 0 ? 2 * (int64_t)me + 1 : 2 * ((int64_t)me + s); };
    for (int i = threadIdx.x; i < ROWS * (D / 8); i += 256) {
        const int x = i / (D / 8), c = i % (D / 8), row = note.tile * ROWS + x;
        if (row >= n_q * group) return;
        float most = -INFINITY, sum = 0.0f;
#pragma unroll 4
        for (int s = 0; s < pieces; ++s) most = fmaxf(most, a.part_ml[slot(s) * ROWS + x].x);
        f32x4 v0 = {0, 0, 0, 0}, v1 = {0, 0, 0, 0};
#pragma unroll 4
        for (int s = 0; s < pieces; ++s) {
            const float2 ml = a.part_ml[slot(s) * ROWS + x];
            const float keep = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - most);
            const float *p = a.part_o + (slot(s) * ROWS + x) * D + c * 8;
            sum += ml.y * keep;
            v0 += *reinterpret_cast<const f32x4 *>(p) * keep;
            v1 += *reinterpret_cast<const f32x4 *>(p + 4) * keep;
        }
        store_row<T>(a, (first + row / group) * a.q_heads + h * group + row % group, D, c, v0, v1, most, sum);
    }
}

template <int D, int SUB, int RB, int NW, bool VLDS>
hipError_t launch(const AttendArgs &a, const AttendPlan &p, dim3 grid, hipStream_t stream) {
    using T = VQ_CACHE_TYPE;
    auto *kernel = k_cache_attend<T, D, SUB, RB, NW, VLDS>;
    static std::atomic<uint64_t> allowed{0};                      // devices that know of the LDS this kernel takes, a bit each
    const hipError_t e = vq_internal_allow_lds(reinterpret_cast<const void *>(kernel), allowed);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kernel, grid, dim3(NW * 64), p.lds, stream, a);
    if (a.split) hipLaunchKernelGGL((k_cache_join<T, D, RB>), grid, dim3(256), 0, stream, a);
    return hipGetLastError();
}

template <int D, int SUB>
hipError_t launch_rows(const AttendArgs &a, const AttendPlan &p, dim3 grid, hipStream_t stream) {
#define VQ_TRY(RB, NW, VLDS) \
    if (p.rb == RB && p.nw == (NW) && p.values_in_lds == VLDS) return launch<D, SUB, RB, (NW), VLDS>(a, p, grid, stream)
    VQ_TRY(1, 8, true);
    VQ_TRY(2, D >= 192 ? 4 : 8, true);
    if constexpr (D >= 192) {
        VQ_TRY(1, 8, false);
        VQ_TRY(2, 4, false);
    }
#undef VQ_TRY
    return hipErrorInvalidValue;
}

template <int D>
hipError_t launch_sub(const AttendArgs &a, const AttendPlan &p, int sub, dim3 grid, hipStream_t stream) {
    return sub == 2 ? launch_rows<D, 2>(a, p, grid, stream) : sub == 4 ? launch_rows<D, 4>(a, p, grid, stream) : launch_rows<D, 8>(a, p, grid, stream);
}

}  // namespace

hipError_t VQ_CACHE_ATTEND(const AttendArgs &a, const AttendPlan &p, int dim, int sub, dim3 grid, hipStream_t stream) {
    switch (dim) {
        case 32: return launch_sub<32>(a, p, sub, grid, stream);
        case 64: return launch_sub<64>(a, p, sub, grid, stream);
        case 96: return launch_sub<96>(a, p, sub, grid, stream);
        case 128: return launch_sub<128>(a, p, sub, grid, stream);
        case 192: return launch_sub<192>(a, p, sub, grid, stream);
        default: return launch_sub<256>(a, p, sub, grid, stream);
    }
}
