// vq_cache_search.hip -- nearest codewords of float sub-vectors: vq_cache_write, and the search and sums of vq_cache_lbg_accum (vq_cache.h).
//
// A code is the argmin of a squared distance summed in fp64, the lowest codeword of equal ones.  It is found in three steps, each of
// which hands on what it cannot decide:
//   1. Scores 1/2 |c|^2 - x.c of 32 vectors against 32 codewords at a time, v_mfma 32x32x16 bf16.  Numbers of wider types go in as two or three
//      bf16 pieces each, and 1/2 |c|^2 as three further terms against ones, so a score comes out of the matrix unit whole.  A lane keeps the two
//      least of the minima over groups of 8 codewords, the group's number in the low bits.  With B = 1/2 max |c|^2 + |x| max |c|, a
//      score is off by 2^-18.5 B (bf16, 4 numbers) to 2^-16.7 B (fp32, 8 numbers): additions in fp32, dropped pieces, the group's number.
//      A second-best group more than twice that behind (GAP) holds no nearest codeword.
//   2. The 8 codewords of the best group by direct differences in fp32, each sum off by less than 2^-19 of itself.
//   3. Vectors that either step leaves open (close calls, ties, values beyond fp32's range, what is not finite) are searched by the whole wave
//      in fp64, by the definition: one in 600 to 900 where vectors and codewords are of one size (counted with these bounds on the CPU).
//
// A wave keeps its part's 256 codewords in registers as the operand of step 1 and streams its tokens past them.
//
// What it reaches (8 heads, 128 dims in parts of 4, 256 codewords, bf16): 16384 tokens' keys and values written in 113 us, an iteration
// on 32768 vectors a head in 172 us: 75 and 49 G sub-vectors/s, 19 and 12 T distances/s.  Bound by the VALU, busy for 90% of the cycles; of
// 436 operations on 64 sub-vectors, 224 take the least of the scores (7 for 8 of them; the matrix unit is busy a quarter of the time), 88
// are step 2's, 20 step 3's.  A write of a few tokens is 7 us of latency: codewords, operand, one turn.
// The same by parts of 2 and 8: written in 324 and 74 us, trained in 326 and 137; in fp16, whose numbers are two pieces a side, four terms and an
// operand that has to be moved, written in 345, 151 and 108 and trained in 340, 222 and 172; trained on fp32 in 366, 264 and 215.
// Groups of 16 in step 1 would save 48 operations there and cost 88 in step 2; vectors 32 at a time took 155 and 211 us.
#include "vq_cache_internal.h"

namespace {

template <typename V> constexpr int PIECES = 3;
template <> constexpr int PIECES<_Float16> = 2;
template <> constexpr int PIECES<__bf16> = 1;

// The products of pieces that step 1 takes: (vector's piece, codeword's piece), those below 2^-24 of the whole left out.
struct Terms {
    int n, x[6], c[6];
};
constexpr Terms terms_of(int xp, int cp) {
    Terms t = {0, {}, {}};
    for (int i = 0; i < xp; ++i)
        for (int j = 0; j < cp; ++j)
            if (i + j < 3) t.x[t.n] = i, t.c[t.n] = j, ++t.n;
    return t;
}

constexpr int SEARCH_WAVES = 8;
constexpr float FAR_SCORE = 1e38f, FAR_NUMBER = 1e18f, BOUND_MOST = 1e30f, SIZE_MOST = 1e34f;
// Rows past K lie at FAR_NUMBER: a vector within SIZE_MOST (1e17 long) and codewords within BOUND_MOST (1.5e15) are nearer to each other.
constexpr float SUM_SCALE = 16777216.0f;       // lifts fp32's smallest numbers into bf16's normal range
constexpr float COUNTED = 0x1p100f;            // training leaves out what is larger
constexpr float NEAR = 0x1p126f;               // vectors shorter than 2^63 are added by products: 1024 of them, times SUM_SCALE, stay inside fp32
// Training's sums.  Products add up so many vectors at a time in fp32, in a step of 32 vectors for each piece of their numbers, each off by a step
// (2^-23 of the sum so far) at most; what they give goes into LDS by an addition whose error is kept and goes on with the next products.  Equal
// numbers err the same way in every step, so a sum is off by up to 2^-17 of its numbers' sizes (32 steps by 1 or 2 pieces, or 8 by 3);
// added over the whole chunk in one go, 4096 fp32 copies of a number gave a mean up to 162 * 2^-24 off, now 6.  Costs 1 to 3% of an iteration.
constexpr int fold_after(int pieces) { return pieces == 1 ? 1024 : pieces == 2 ? 512 : 256; }      // vectors

__device__ inline uint32_t bf16_bits(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }

// v = sum of P bf16 pieces (to 2^-8P of itself; exact for a type of 8P bits).
template <int P> __device__ inline void split(float v, uint32_t (&piece)[P]) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
        piece[i] = bf16_bits(v);
        v -= __builtin_bit_cast(float, piece[i] << 16);
    }
}

template <typename V, int N> struct alignas(N * sizeof(V) < 16 ? N * sizeof(V) : 16) Numbers {
    V v[N];
};

// a and b: what lanes l and l + 32 found for the lower vectors and for the upper ones.  To each lane, both findings about its own.
__device__ inline void to_owners(float &a, float &b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), false, false);
    const uint32_t first = r[0], second = r[1];
    a = __builtin_bit_cast(float, first);
    b = __builtin_bit_cast(float, second);
}

// The least of all lanes' numbers, in all.
template <int CONTROL, int ROWS> __device__ inline uint32_t min_with(uint32_t v) {      // (a lane that the control names no other for: with itself)
    return min(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CONTROL, ROWS, 0xf, false));
}
__device__ inline uint32_t wave_min(uint32_t v) {
    v = min_with<0x111, 0xf>(v);     // one, two, four and eight lanes to the right inside a row of 16
    v = min_with<0x112, 0xf>(v);
    v = min_with<0x114, 0xf>(v);
    v = min_with<0x118, 0xf>(v);
    v = min_with<0x142, 0xa>(v);     // the last lane of a row to all of the next, for the second and the fourth
    v = min_with<0x143, 0xc>(v);     // lane 31 to the upper half
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// All ones in each half of `labels` that equals that of `row`, zeros in the other.
__device__ inline uint32_t equal_halves(uint32_t labels, uint32_t row) {
    const u16x2 one = {1, 1};
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(u16x2, labels ^ row), one) - one);
}

// The lesser of two finite scores, without the canonicalisation that fminf of unknown bits brings.
__device__ inline float least(float a, float b) { return __builtin_amdgcn_fmed3f(-FAR_SCORE * 3.0f, a, b); }

// Where codeword k starts in a wave's table in LDS: 16 rows and a pad, so that the same rows of different groups, which is what the lanes
// ask for at once in step 2, lie in different banks.
template <int SUB> __device__ constexpr int row_at(int k) { return k * SUB + (k >> 4) * (SUB < 4 ? 2 : 4); }

// T: the vectors' type, C: the codebook's; NT: groups of 32 codewords.
template <typename T, typename C, int SUB, int NT, bool TRAIN>
__global__ __launch_bounds__(SEARCH_WAVES * 64) void k_cache_search(const SearchArgs a) {
    constexpr int XP = PIECES<T>, CP = PIECES<C>, H2 = SUB / 2;
    constexpr Terms TM = terms_of(XP, CP);
    constexpr int PAIRS = TM.n * H2 + 2, NM = (PAIRS * 2 + 15) / 16;     // slots in pairs; the last two hold the norm
    // Where a vector's slots fit into one half of the operand, the codewords stand in both: a lane of the upper half then
    // gives its own vector's numbers there, and none have to be moved.
    constexpr bool TWICE = PAIRS <= 4;
    __shared__ __align__(16) float s_tab[SEARCH_WAVES][row_at<SUB>(NT * 32)];
    __shared__ __align__(16) uint16_t s_hi[TRAIN ? SEARCH_WAVES : 1][64], s_lo[TRAIN ? SEARCH_WAVES : 1][64];
    __shared__ __align__(16) uint16_t s_x[TRAIN ? SEARCH_WAVES : 1][XP][SUB][64];
    __shared__ f32x4 s_sum[TRAIN ? SEARCH_WAVES : 1][SUB][64];            // a lane's own sums: see fold_after
    const int lane = threadIdx.x & 63, col = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int which = blockIdx.z, parts = a.dim / SUB, per = parts / a.pw;
    const int h = blockIdx.x / per, m = blockIdx.x % per * a.pw + wave % a.pw;
    const int chunk = blockIdx.y * (SEARCH_WAVES / a.pw) + wave / a.pw;
    const int64_t begin = (int64_t)chunk * a.chunk;
    const int64_t end = begin + a.chunk < a.tokens ? begin + a.chunk : a.tokens;
    if (begin >= end && !TRAIN) return;
    float *tab = s_tab[wave];
    const C *cb = static_cast<const C *>(a.cb[which]) + (a.cb_heads == 1 ? 0 : (int64_t)h * a.K * a.dim) + m * SUB;
    const T *x0 = static_cast<const T *>(a.x[which]) + h * a.head_stride[which] + m * SUB;

    const int64_t slots = a.pages * a.page, page_bytes = (int64_t)a.heads * a.page * parts;
    uint8_t *codes = which == 0 ? a.k_codes + (int64_t)h * a.page * parts + m : a.v_codes + ((int64_t)h * parts + m) * a.page;

    // See above: twice what a score may be off by, in steps of 2^-23 B.  Additions (a step each, whichever way the unit rounds), the group's
    // number, dropped pieces, the norm's own sum; two steps for B, which is rounded too.
    constexpr float GAP = 2 * (TM.n * SUB + 3 + 16 + 2 + SUB / 2 + 2) * 0x1p-23f;

    // the codewords: operand of step 1, and in fp32 for steps 2 and 3; rows past K lie far away
    u32x4 A[NT][NM];
    float reach = 0.0f;                                                   // max |c|^2, infinite if any codeword is not finite
    Numbers<C, SUB> raws[NT];                                             // all loads first: a call on a few tokens is their latency
#pragma unroll
    for (int t = 0; t < NT; ++t) raws[t] = *reinterpret_cast<const Numbers<C, SUB> *>(cb + (int64_t)(t * 32 + col < a.K ? t * 32 + col : a.K - 1) * a.dim);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int k = t * 32 + col;
        const Numbers<C, SUB> raw = raws[t];
        float c[SUB], norm = 0.0f;
        uint32_t cp[CP][H2];
#pragma unroll
        for (int e = 0; e < SUB; ++e) {
            c[e] = k < a.K ? (float)raw.v[e] : 0.0f;
            norm += c[e] * c[e];
        }
        reach = fmaxf(reach, norm < INFINITY ? norm : INFINITY);
#pragma unroll
        for (int i = 0; i < H2; ++i) {
            uint32_t p0[CP], p1[CP];
            split<CP>(-c[2 * i], p0);
            split<CP>(-c[2 * i + 1], p1);
#pragma unroll
            for (int p = 0; p < CP; ++p) cp[p][i] = p0[p] | p1[p] << 16;
        }
        uint32_t np[3];
        split<3>(k < a.K ? 0.5f * norm : FAR_SCORE, np);
        auto pair = [&](int s) -> uint32_t {
            return s < TM.n * H2 ? cp[TM.c[s / H2]][s % H2] : s == TM.n * H2 ? np[0] | np[1] << 16 : s == TM.n * H2 + 1 ? np[2] : 0u;
        };
#pragma unroll
        for (int n = 0; n < NM; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) A[t][n][j] = hh && !TWICE ? pair(8 * n + 4 + j) : pair(8 * n + j);
        if (hh == 0)
#pragma unroll
            for (int e = 0; e < SUB; ++e) tab[row_at<SUB>(k) + e] = k < a.K ? c[e] : FAR_NUMBER;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) reach = fmaxf(reach, __shfl_xor(reach, o));
    const float far = __builtin_amdgcn_sqrtf(reach);
    // A vector longer than this is left to step 3: 2^19 times as long as any codeword, its distances may be equal in fp64 where step 1 can tell them
    // apart, and then the lowest number is asked for.  (Up to there, what step 1 tells apart differs by 2^-36 |x|^2 or more, fp64 sums
    // by 2^-47 at most.  Step 2 leaves nearly all of those open by itself, but not in a group of one codeword.)
    const float size_most = a.K > 1 ? fminf(SIZE_MOST, reach * 0x1p38f) : SIZE_MOST;

    f32x4 sum[TRAIN ? SUB + 1 : 1];
    double away = 0.0;
    int counted = 0;
    if constexpr (TRAIN)
#pragma unroll
        for (int e = 0; e <= SUB; ++e) {
            sum[e] = (f32x4){0, 0, 0, 0};
            if (e < SUB) s_sum[wave][e][lane] = sum[e];
        }
    // v into sum[e], exactly: the rounded sum to LDS, what is missing stays behind
    auto put = [&](int e, f32x4 v) {
        const f32x4 had = s_sum[wave][e][lane], now = had + v, added = now - had;
        s_sum[wave][e][lane] = now;
        __builtin_amdgcn_sched_barrier(0);                        // (one after the other: few registers)
        return (had - (now - added)) + (v - added);
    };

    auto fetch = [&](int64_t t) -> Numbers<T, SUB> {                      // past the end: the last token again
        t = t < end ? t : end - 1;
        return *reinterpret_cast<const Numbers<T, SUB> *>(x0 + t * a.token_stride[which]);
    };
    Numbers<T, SUB> next;
    if (begin < end) next = fetch(begin + lane);
    for (int64_t t0 = begin; t0 < end; t0 += 64) {
        // A lane has a vector of its own.  Step 1 takes the lower 32 lanes' and then the upper 32 lanes', the rest all 64.
        const Numbers<T, SUB> raw = next;
        if (t0 + 64 < end) next = fetch(t0 + 64 + lane);
        const int64_t token = t0 + lane;
        int64_t slot = -1;
        if constexpr (!TRAIN) slot = a.slots[token < end ? token : end - 1];
        float x[SUB], size = 0.0f;
        uint32_t xp[XP][H2];
#pragma unroll
        for (int e = 0; e < SUB; ++e) {
            x[e] = (float)raw.v[e];
            size += x[e] * x[e];
        }
#pragma unroll
        for (int i = 0; i < H2; ++i) {
            uint32_t p0[XP], p1[XP];
            split<XP>(x[2 * i], p0);
            split<XP>(x[2 * i + 1], p1);
#pragma unroll
            for (int p = 0; p < XP; ++p) xp[p][i] = p0[p] | p1[p] << 16;
        }
        auto pair = [](int s, uint32_t const (&of)[XP][H2]) -> uint32_t {
            return s < TM.n * H2 ? of[TM.x[s / H2]][s % H2] : s == TM.n * H2 ? 0x3f803f80u : s == TM.n * H2 + 1 ? 0x3f80u : 0u;
        };
        // step 1
        float m1[2], m2[2];
        m1[0] = m1[1] = m2[0] = m2[1] = FAR_SCORE * 3.0f;
        auto score = [&](int half, int t, u32x4 const (&B)[NM]) {
            f32x16 s = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int n = 0; n < NM; ++n)
                s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, A[t][n]), __builtin_bit_cast(bf16x8, B[n]), s, 0, 0, 0);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                float v = FAR_SCORE * 3.0f;
#pragma unroll
                for (int i = 0; i < 8; i += 2) v = fminf(fminf(v, s[8 * q + i]), s[8 * q + i + 1]);
                const float key = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, v) & ~15u) | (uint32_t)(2 * t + q));
                m2[half] = __builtin_amdgcn_fmed3f(m1[half], m2[half], key);
                m1[half] = least(m1[half], key);
            }
        };
        if constexpr (TWICE) {
            u32x4 B[2][NM];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t own = pair(j, xp);
                B[0][0][j] = hh ? 0u : own, B[1][0][j] = hh ? own : 0u;
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) score(0, t, B[0]), score(1, t, B[1]);
        } else {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t of[XP][H2];
#pragma unroll
                for (int p = 0; p < XP; ++p)
#pragma unroll
                    for (int i = 0; i < H2; ++i) of[p][i] = __builtin_amdgcn_permlane32_swap(xp[p][i], xp[p][i], false, false)[half];
                u32x4 B[NM];
#pragma unroll
                for (int n = 0; n < NM; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j) B[n][j] = hh ? pair(8 * n + 4 + j, of) : pair(8 * n + j, of);
#pragma unroll
                for (int t = 0; t < NT; ++t) score(half, t, B);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        float l1 = m1[0], h1 = m1[1], l2 = m2[0], h2 = m2[1];
        to_owners(l1, h1);
        to_owners(l2, h2);
        const bool upper = h1 < l1;
        const float best = upper ? h1 : l1, second = least(upper ? l1 : h1, least(l2, h2));
        const float bound = 0.5f * reach + __builtin_amdgcn_sqrtf(size) * far;
        bool open = !(second - best > bound * GAP + 1e-36f) || !(bound < BOUND_MOST) || !(size < size_most);
        const int group = __builtin_bit_cast(uint32_t, best) & (2 * NT - 1);      // (a score beyond fp32 names any)

        // step 2: rows k0 to k0 + 3 and k0 + 8 to k0 + 11
        const int k0 = group * 16 + 4 * (int)upper, at0 = row_at<SUB>(group * 16) + (upper ? 4 * SUB : 0);
        float d1 = FAR_SCORE * 3.0f, d2 = FAR_SCORE * 3.0f;               // (what is not finite here is open already)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float d = 0.0f;
#pragma unroll
            for (int e = 0; e < SUB; ++e) {
                const float v = x[e] - tab[at0 + (j + (j & 4)) * SUB + e];
                d = __builtin_fmaf(v, v, d);
            }
            const float key = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, d) & ~7u) | j);
            d2 = __builtin_amdgcn_fmed3f(d1, d2, key);
            d1 = least(d1, key);
        }
        open = open || !(d2 > d1 * 1.00000763f + 1e-36f);
        const int nth = __builtin_bit_cast(uint32_t, d1) & 7u;
        int code = k0 + nth + (nth & 4);

        // step 3
        uint64_t todo = __ballot(open && token < end);
        while (todo) {
            const int v = __builtin_ctzll(todo);
            todo &= todo - 1;
            double y[SUB];
#pragma unroll
            for (int e = 0; e < SUB; ++e) y[e] = (double)__builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x[e]), v));
            double d = INFINITY;
            uint32_t k_best = 256;
#pragma unroll 2
            for (int k = lane; k < NT * 32; k += 64) {
                double f = 0.0;
#pragma unroll
                for (int e = 0; e < SUB; ++e) {
                    const double w = y[e] - (double)tab[row_at<SUB>(k) + e];
                    f += w * w;
                }
                if (k < a.K && f < d) d = f, k_best = k;
            }
            // distances are not negative: their bits are in their order, the upper halves first
            const uint64_t bits = __builtin_bit_cast(uint64_t, d);
            const uint32_t high = wave_min((uint32_t)(bits >> 32));
            uint32_t low = (uint32_t)(bits >> 32) == high ? (uint32_t)bits : ~0u;
            const uint32_t lowest = wave_min(low);
            const uint32_t k_least = wave_min((uint32_t)(bits >> 32) == high && low == lowest ? k_best : 256u);
            if (lane == v) code = k_least < 256u ? (int)k_least : 0;
        }

        if constexpr (!TRAIN) {
            if (token < end && slot >= 0 && slot < slots) {
                const int64_t p = a.page_shift >= 0 ? slot >> a.page_shift : slot / a.page;
                const int o = (int)(slot - p * a.page);
                codes[p * page_bytes + (which == 0 ? o * parts : o)] = (uint8_t)code;
            }
        } else {
            const bool near = token < end && size < NEAR;
            bool fine = near;                                             // it counts; of longer ones (and of NaN) those do whose numbers all are small enough
            if (__builtin_expect(__any(token < end && !near), 0)) {
                fine = token < end;
#pragma unroll
                for (int e = 0; e < SUB; ++e) fine = fine && fabsf(x[e]) < COUNTED;
            }
            // sums by products with the one-hot numbers of the codewords: number = 16 hi + lo, and
            // sum[hi][lo] = sum over vectors of (x where its hi is this row) * (1 where its lo is this column)
            counted += __popcll(__ballot(fine));
            if (fine) {
                double f = 0.0;
#pragma unroll
                for (int e = 0; e < SUB; ++e) {
                    const double w = (double)x[e] - (double)tab[row_at<SUB>(code) + e];
                    f += w * w;
                }
                away += f <= INFINITY ? f : INFINITY;
            }
            s_hi[wave][lane] = near ? (uint16_t)(code >> 4) : (uint16_t)0xffff;
            s_lo[wave][lane] = (uint16_t)(code & 15);
#pragma unroll
            for (int e = 0; e < SUB; ++e) {
                uint32_t piece[XP];
                split<XP>(x[e] * SUM_SCALE, piece);
#pragma unroll
                for (int p = 0; p < XP; ++p) s_x[wave][p][e][lane] = (uint16_t)piece[p];
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            const uint32_t row = (lane & 15) * 0x10001u;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int first = 32 * half + 8 * (lane >> 4);
                u32x4 member = *reinterpret_cast<const u32x4 *>(&s_hi[wave][first]), lows = *reinterpret_cast<const u32x4 *>(&s_lo[wave][first]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    member[j] = equal_halves(member[j], row);
                    lows[j] = equal_halves(lows[j], row) & 0x3f803f80u;
                }
                const bf16x8 lo8 = __builtin_bit_cast(bf16x8, lows);
#pragma unroll
                for (int p = XP - 1; p >= 0; --p)                         // (the smallest pieces first)
#pragma unroll
                    for (int e = 0; e < SUB; ++e) {
                        const u32x4 of = *reinterpret_cast<const u32x4 *>(&s_x[wave][p][e][first]) & member;
                        sum[e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, of), lo8, sum[e], 0, 0, 0);
                    }
                const u32x4 ones = member & 0x3f803f80u;
                sum[SUB] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, ones), lo8, sum[SUB], 0, 0, 0);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if ((t0 - begin) % fold_after(XP) == fold_after(XP) - 64)
#pragma unroll
                for (int e = 0; e < SUB; ++e) sum[e] = put(e, sum[e] * (1.0f / SUM_SCALE)) * SUM_SCALE;
            // longer vectors one by one, by the lane that holds their codeword
            for (uint64_t todo = __ballot(fine && !near); todo; todo &= todo - 1) {
                const int v = __builtin_ctzll(todo), c = __builtin_amdgcn_readlane(code, v);
                f32x4 one = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < 4; ++i) one[i] = lane == (c >> 6 << 4 | (c & 15)) && (c >> 4 & 3) == i ? 1.0f : 0.0f;
#pragma unroll
                for (int e = 0; e < SUB; ++e)
                    sum[e] += put(e, one * __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x[e]), v))) * SUM_SCALE;
                sum[SUB] += one;
            }
        }
    }
    if constexpr (TRAIN) {
        const int64_t place = (int64_t)chunk * a.heads * parts + h * parts + m;
#pragma unroll
        for (int e = 0; e <= SUB; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                a.part_sums[(place * (SUB + 1) + e) * 256 + (4 * (lane >> 4) + i) * 16 + (lane & 15)] =
                    e < SUB ? s_sum[wave][e < SUB ? e : 0][lane][i] + sum[e][i] * (1.0f / SUM_SCALE) : sum[e][i];
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) away += __shfl_xor(away, o);
        if (lane == 0) a.part_dist[place] = make_double2(away, (double)counted);
    }
}

// Adds the chunks' sums, in fp64 and in an order that follows from the sizes.  A workgroup takes C = 1 << shift codewords of a head and part;
// its 1024 threads are C codewords by 1024 / C shares of the chunks.  Reads (sub + 1) KB a chunk once; where a new codebook is asked for it
// also divides, and the sums are not stored.  Bound by latency and by the chunks' sums coming back (64 groups of 32 chunks, 19 MB: 8.4 us): C
// falls, to a cache line's 32, until there are workgroups for all compute units or a thread has one chunk (parts of 4, 16 groups of 470
// chunks: 39.7 us for the iteration with 256 codewords to a workgroup, 26.2 so; 12 groups, parts of 8, 146 chunks: 46.6, 32.2, and with
// 16 codewords 37.3).
constexpr int GATHER_THREADS = 1024;
__device__ inline double wave_sum(double v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    return v;
}
template <int SUB>
__global__ __launch_bounds__(GATHER_THREADS) void k_lbg_gather(const float *__restrict__ part_sums, const double2 *__restrict__ part_dist, int chunks,
                                                               int shift, const LbgOut out) {
    __shared__ double s_sum[SUB + 1][GATHER_THREADS], s_away[GATHER_THREADS / 64], s_n[GATHER_THREADS / 64];
    const int tid = threadIdx.x, parts = out.dim / SUB, h = blockIdx.x / parts, m = blockIdx.x % parts;
    const int k = (blockIdx.y << shift) + (tid & ((1 << shift) - 1)), side = tid >> shift, sides = GATHER_THREADS >> shift;
    const int64_t groups = (int64_t)out.heads * parts;
    double sum[SUB + 1];
#pragma unroll
    for (int e = 0; e <= SUB; ++e) sum[e] = 0.0;
#pragma unroll 4
    for (int c = side; c < chunks; c += sides) {
        const float *p = part_sums + (c * groups + blockIdx.x) * ((SUB + 1) * 256) + k;
#pragma unroll
        for (int e = 0; e <= SUB; ++e) sum[e] += (double)p[e * 256];
    }
#pragma unroll
    for (int e = 0; e <= SUB; ++e) s_sum[e][tid] = sum[e];
    if (blockIdx.y == 0) {
        double away = 0.0, n = 0.0;
        for (int c = tid; c < chunks; c += GATHER_THREADS) {
            const double2 d = part_dist[c * groups + blockIdx.x];
            away += d.x, n += d.y;
        }
        away = wave_sum(away), n = wave_sum(n);
        if ((tid & 63) == 0) s_away[tid >> 6] = away, s_n[tid >> 6] = n;
    }
    __syncthreads();
    for (int o = sides / 2; o; o >>= 1) {
        if (side < o)
#pragma unroll
            for (int e = 0; e <= SUB; ++e) s_sum[e][tid] += s_sum[e][tid + (o << shift)];
        __syncthreads();
    }
    if (side == 0 && k < out.K) {
        const double n = s_sum[SUB][tid];
        const int64_t at = ((int64_t)h * out.K + k) * out.dim + m * SUB;
        out.counts[(int64_t)blockIdx.x * out.K + k] = (int64_t)n;
#pragma unroll
        for (int e = 0; e < SUB; ++e) {
            const double s = s_sum[e][tid];
            if (out.cb_new) out.cb_new[at + e] = n > 0.0 ? (float)(s / n) : out.cb_old[at + e];
            else out.sums[at + e] = s;
        }
    }
    if (blockIdx.y == 0 && tid == 0) {
        double away = 0.0, n = 0.0;
        for (int w = 0; w < GATHER_THREADS / 64; ++w) away += s_away[w], n += s_n[w];
        out.dist[blockIdx.x] = out.cb_new ? (n > 0.0 ? away / n : 0.0) : away;
    }
}

template <typename T, typename C, int SUB, bool TRAIN>
void launch_sub(const SearchArgs &a, dim3 grid, hipStream_t stream) {
    const dim3 block(SEARCH_WAVES * 64);
    if (a.K <= 64) hipLaunchKernelGGL((k_cache_search<T, C, SUB, 2, TRAIN>), grid, block, 0, stream, a);
    else if (a.K <= 128) hipLaunchKernelGGL((k_cache_search<T, C, SUB, 4, TRAIN>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((k_cache_search<T, C, SUB, 8, TRAIN>), grid, block, 0, stream, a);
}

template <typename T, typename C, bool TRAIN>
void launch(const SearchArgs &a, int sub, dim3 grid, hipStream_t stream) {
    if (sub == 2) launch_sub<T, C, 2, TRAIN>(a, grid, stream);
    else if (sub == 4) launch_sub<T, C, 4, TRAIN>(a, grid, stream);
    else launch_sub<T, C, 8, TRAIN>(a, grid, stream);
}

}  // namespace

SearchPlan vq_internal_search_plan(int64_t tokens, int heads, int dim, int sub, int both) {
    constexpr int CUS = 256;
    SearchPlan p;
    const int parts = dim / sub;
    p.pw = parts % 8 ? 4 : 8;
    const int64_t side = SEARCH_WAVES / p.pw;                             // token ranges side by side in one workgroup
    const int64_t base = (int64_t)heads * (parts / p.pw) * both;
    // A workgroup takes 8 parts, or 4 where they do not come by eights (dims of 96 by 8); two workgroups for each compute unit, or one in
    // training by parts of 8, whose registers and LDS leave no room for two (8192 vectors, 4 heads: 46 us; in two rounds 54).  A write is spread as
    // thinly as turns of 64 tokens allow (256 tokens: 7.8 us; turns of 128 9.4).  A training chunk of fewer than 128 costs more to gather
    // than it saves (1000 vectors, 4 heads: 19.4 us; of 64 20.1, of 256 23.1), and none is longer than 4096: its sums are fp32.
    const int fewest = both == 2 ? 64 : 128, longest = both == 2 ? 1 << 24 : 4096;
    const int64_t most = (tokens + fewest * side - 1) / (fewest * side), least = (tokens + longest * side - 1) / (longest * side);
    int64_t n = ((both == 2 || sub < 8 ? 2 : 1) * CUS + base - 1) / base;
    n = n < most ? n : most;
    n = n > least ? n : least;
    p.chunk = (int)(((tokens + n * side - 1) / (n * side) + 63) / 64 * 64);
    p.blocks = (int)((tokens + p.chunk * side - 1) / (p.chunk * side));
    p.chunks = (int)(p.blocks * side);
    return p;
}

hipError_t vq_internal_search(const SearchArgs &a, int sub, int dtype, bool train, int blocks, hipStream_t stream) {
    const dim3 grid(a.heads * (a.dim / sub / a.pw), blocks, train ? 1 : 2);
    if (train) {
        if (dtype == VQ_F32) launch<float, float, true>(a, sub, grid, stream);
        else if (dtype == VQ_BF16) launch<__bf16, float, true>(a, sub, grid, stream);
        else launch<_Float16, float, true>(a, sub, grid, stream);
    } else {
        if (dtype == VQ_BF16) launch<__bf16, __bf16, false>(a, sub, grid, stream);
        else launch<_Float16, _Float16, false>(a, sub, grid, stream);
    }
    return hipGetLastError();
}

hipError_t vq_internal_lbg_gather(const SearchArgs &a, int sub, int chunks, const LbgOut &out, hipStream_t stream) {
    const int groups = a.heads * (a.dim / sub);
    int shift = 8;
    auto across = [&]() { return (out.K + (1 << shift) - 1) >> shift; };
    while (shift > 5 && (out.K <= 1 << (shift - 1) || (groups * across() < 256 && chunks > GATHER_THREADS >> shift))) --shift;
    const dim3 grid(groups, across()), block(GATHER_THREADS);
    if (sub == 2) hipLaunchKernelGGL(k_lbg_gather<2>, grid, block, 0, stream, a.part_sums, a.part_dist, chunks, shift, out);
    else if (sub == 4) hipLaunchKernelGGL(k_lbg_gather<4>, grid, block, 0, stream, a.part_sums, a.part_dist, chunks, shift, out);
    else hipLaunchKernelGGL(k_lbg_gather<8>, grid, block, 0, stream, a.part_sums, a.part_dist, chunks, shift, out);
    return hipGetLastError();
}
