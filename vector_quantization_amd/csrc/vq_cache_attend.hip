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
// Softmax in base 2 with a running maximum per row that is only moved once a score exceeds it by 8 (weights stay
// below 2^8, sums are fp32), so that most tiles need neither a reduction across lanes nor a rescaling.  Weights are rounded to the cache's type
// for the second product (half a step, as the values themselves are of that type); the sum of weights takes them unrounded.

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

// NB consecutive bytes from an address that is a multiple of the largest power of two in NB (4 at most).
template <int NB> __device__ inline void load_bytes(uint32_t *w, const uint8_t *p) {
    if constexpr (NB % 16 == 0) {
#pragma unroll
        for (int i = 0; i < NB / 16; ++i) {
            const u32x4 v = *reinterpret_cast<const u32x4 *>(p + 16 * i);
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    } else if constexpr (NB % 8 == 0) {
#pragma unroll
        for (int i = 0; i < NB / 8; ++i) {
            const u32x2 v = *reinterpret_cast<const u32x2 *>(p + 8 * i);
            w[2 * i] = v.x, w[2 * i + 1] = v.y;
        }
    } else if constexpr (NB % 4 == 0) {
#pragma unroll
        for (int i = 0; i < NB / 4; ++i) w[i] = *reinterpret_cast<const uint32_t *>(p + 4 * i);
    } else if constexpr (NB % 2 == 0) {
#pragma unroll
        for (int i = 0; i < (NB + 3) / 4; ++i) {
            w[i] = *reinterpret_cast<const uint16_t *>(p + 4 * i);
            if (4 * i + 2 < NB) w[i] |= (uint32_t)*reinterpret_cast<const uint16_t *>(p + 4 * i + 2) << 16;
        }
    } else {
        w[0] = 0;
#pragma unroll
        for (int i = 0; i < NB; ++i) w[0] |= (uint32_t)p[i] << (8 * i);
    }
}

// Look-ups name LDS by its byte offset: the kernel has no other LDS, so s_mem lies at 0, and an address is what the code and
// the lane make of it without a base to be added each time.
template <typename V> __device__ inline V lds(uint32_t at) { return *(const __attribute__((address_space(3))) V *)at; }

__device__ inline float wave_any_max(float v) {          // the maximum over the four lanes of one row
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}

// 8 numbers of a finished row, place = row * q_heads + head: v against the maximum `most` (base 2) and the sum of weights.
template <typename T>
__device__ inline void store_row(const AttendArgs &a, int64_t place, int D, int c, f32x4 v0, f32x4 v1, float most, float sum) {
    const float over = sum > 0.0f ? 1.0f / sum : 0.0f;
    *reinterpret_cast<u32x4 *>(static_cast<T *>(a.out) + place * D + c * 8) =
        (u32x4){pack2<T>(v0[0] * over, v0[1] * over), pack2<T>(v0[2] * over, v0[3] * over),
                pack2<T>(v1[0] * over, v1[1] * over), pack2<T>(v1[2] * over, v1[3] * over)};
    if (c == 0 && a.lse) a.lse[place] = sum > 0.0f ? most * 0.69314718055994531f + logf(sum) : -INFINITY;
}

// The tiles that the rows of one item see: rows tile * RB * 16 on of a sequence, whose row i sees tokens 0 .. n_kv - n_q + i.
template <int RB> __device__ inline int tiles_of(int tile, int n_q, int n_kv, int group) {
    const int n_rows = n_q * group, past = (tile + 1) * RB * 16;
    const int end = n_kv - n_q + ((past < n_rows ? past : n_rows) - 1) / group + 1;
    return end < 0 ? 0 : (end + TILE - 1) / TILE;
}
// What an item counts in the division of the work: its tiles, and one where it has none but zeros to be written.
template <int RB> __device__ inline int cost_of(int tile, int n_q, int n_kv, int group) {
    const int n = tiles_of<RB>(tile, n_q, n_kv, group);
    return n < 1 ? 1 : n;
}

// One head's work is all its items side by side, (sequence, tile of rows) after (sequence, tile of rows), cut into as many equal
// ranges of tiles as there are workgroups: causal and ragged lengths are balanced by themselves, and a workgroup stages its tables once.
// A range may begin and end inside an item.  Such an item's parts go to the workspace (`slots`, two a workgroup: the part that begins
// an item and the part that does not), and the workgroup that holds its beginning notes it for k_cache_join.
template <typename T, int D, int SUB, int RB, int NW, bool VLDS>
__global__ __launch_bounds__(NW * 64) void k_cache_attend(const AttendArgs a) {
    constexpr int M = D / SUB, KS = D / 32, NB = M / 4, KW = (NB + 3) / 4;
    constexpr int E = value_chunk(D, SUB), U = D / (16 * E), ROWS = RB * 16;
    extern __shared__ __align__(16) uint8_t s_mem[];
    if ((uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)s_mem != 0) return;      // (never: see lds())
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = blockIdx.x, group = a.q_heads / a.heads;
    const int Kp = a.Kp, kstride = key_stride(Kp, SUB);
    const int k_at = VLDS ? Kp * D * 2 : 0;                       // the value table comes first: see look-ups
    const int64_t cb0 = a.cb_heads == 1 ? 0 : (int64_t)h * a.K * D;
    const T *k_cb = static_cast<const T *>(a.cb[0]) + cb0, *v_cb = static_cast<const T *>(a.cb[1]) + cb0;
    const int page16 = a.page >> 4;
    const uint32_t fold = (uint32_t)(Kp - 1) * 0x01010101u;     // keeps codes of no codeword inside the tables
    const int64_t page_bytes = (int64_t)a.heads * a.page * M;
    const int64_t head_at = (int64_t)h * a.page * M;
    const uint32_t k_lane = r * M + g * NB;
    uint32_t v_lane[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v_lane[u] = ((u * 16 + r) * E / SUB) * a.page + 4 * g;

    // this workgroup's range; every wave works it out by itself, 64 sequences at a time
    auto cost_of_sequence = [&](int b) -> int64_t {
        if (b >= a.seqs) return 0;
        int64_t first;
        int n_q, n_kv;
        sequence(a, b, first, n_q, n_kv);
        const int tiles = (n_q * group + ROWS - 1) / ROWS;
        int64_t sum = 0;
        for (int t = 0; t < tiles; ++t) sum += cost_of<RB>(t, n_q, n_kv, group);
        return sum;
    };
    auto running = [&](int64_t v) -> int64_t {                    // sum over the lanes up to this one
        for (int o = 1; o < 64; o <<= 1) {
            const int64_t up = __shfl_up(v, o);
            if (lane >= o) v += up;
        }
        return v;
    };
    const int64_t mine = cost_of_sequence(lane);
    int64_t all = __shfl(running(mine), 63);
    for (int b0 = 64; b0 < a.seqs; b0 += 64) all += __shfl(running(cost_of_sequence(b0 + lane)), 63);
    int64_t parts = all / a.least_tiles;
    parts = parts < 1 ? 1 : parts > (int64_t)gridDim.y ? (int64_t)gridDim.y : parts;
    const int me = h * gridDim.y + blockIdx.y;
    const int64_t begin = all * blockIdx.y / parts, past = all * (blockIdx.y + 1) / parts;
    if ((int64_t)blockIdx.y >= parts || begin >= past) {
        if (a.parts > 1 && threadIdx.x == 0) a.notes[me] = AttendNote{-1, 0, 0, 0};
        return;
    }
    int b = 0;
    int64_t skip = begin;                                         // tiles of the work before the range, from sequence b on
    for (int b0 = 0; b0 < a.seqs; b0 += 64) {
        const int64_t sum = running(b0 == 0 ? mine : cost_of_sequence(b0 + lane)), whole = __shfl(sum, 63);
        if (skip < whole) {
            const int at = __builtin_ctzll(__ballot(sum > skip));
            b = b0 + at;
            if (at > 0) skip -= __shfl(sum, at - 1);
            break;
        }
        skip -= whole;
    }
    b = __builtin_amdgcn_readfirstlane(b);
    int tile = 0;
    int64_t left = past - begin, now = begin - skip;              // now: where item (b, tile) begins

    // codebooks -> LDS, 16 bytes at a time, several loads under way at once; rows past K are zeros
    constexpr int BATCH = 4;
    for (int i0 = threadIdx.x; i0 < Kp * (D / 8); i0 += BATCH * NW * 64) {
        u32x4 kv[BATCH], vv[BATCH];
#pragma unroll
        for (int x = 0; x < BATCH; ++x) {
            const int i = i0 + x * NW * 64;
            kv[x] = vv[x] = (u32x4){0, 0, 0, 0};
            if (i < a.K * (D / 8)) {
                kv[x] = *reinterpret_cast<const u32x4 *>(k_cb + (int64_t)i * 8);
                if constexpr (VLDS) vv[x] = *reinterpret_cast<const u32x4 *>(v_cb + (int64_t)i * 8);
            }
        }
#pragma unroll
        for (int x = 0; x < BATCH; ++x) {
            const int i = i0 + x * NW * 64, k = i / (D / 8), c = i % (D / 8);
            if (i >= Kp * (D / 8)) continue;
            if constexpr (SUB == 8) {
                *reinterpret_cast<u32x4 *>(s_mem + k_at + c * kstride + k * 16) = kv[x];
            } else if constexpr (SUB == 4) {
                *reinterpret_cast<u32x2 *>(s_mem + k_at + (2 * c) * kstride + k * 8) = kv[x].xy;
                *reinterpret_cast<u32x2 *>(s_mem + k_at + (2 * c + 1) * kstride + k * 8) = kv[x].zw;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) *reinterpret_cast<uint32_t *>(s_mem + k_at + (4 * c + j) * kstride + k * 4) = kv[x][j];
            }
            if constexpr (VLDS) *reinterpret_cast<u32x4 *>(s_mem + i * 16) = vv[x];
        }
    }
    __syncthreads();

    AttendNote note = {-1, 0, 0, 0};
    while (left > 0 && b < a.seqs) {
        int64_t first;
        int n_q, n_kv;
        sequence(a, b, first, n_q, n_kv);
        const int n_rows = n_q * group;
        if (tile * ROWS >= n_rows) {
            ++b;
            tile = 0;
            continue;
        }
        const int tiles = tiles_of<RB>(tile, n_q, n_kv, group), cost = tiles < 1 ? 1 : tiles;
        if (skip >= cost) {
            skip -= cost;
            now += cost;
            ++tile;
            continue;
        }
        const int take = (int)(left < cost - skip ? left : cost - skip);
        const int lo = (int)skip < tiles ? (int)skip : tiles, hi = (int)skip + take < tiles ? (int)skip + take : tiles;
        const bool whole_item = take == cost;
        const int32_t *table = a.table + (int64_t)b * a.width;
        const int row0 = tile * ROWS, rows_here = n_rows - row0 < ROWS ? n_rows - row0 : ROWS;
        const int back = n_kv - n_q;                              // row i sees tokens 0 .. back + i
        const int all_see = back + row0 / group;                  // every row of the item sees tokens up to here

        u32x4 q[RB][KS];
        int sees[RB];
        f32x4 o[RB][U][E];
        float top[RB], total[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int row = rb * 16 + r < rows_here ? row0 + rb * 16 + r : row0;
            const int i = row / group, head = h * group + row % group;
            const T *p = static_cast<const T *>(a.q) + (first + i) * a.q_token_stride + head * a.q_head_stride + g * (D / 4);
            sees[rb] = back + i;
#pragma unroll
            for (int s = 0; s < KS; ++s) q[rb][s] = *reinterpret_cast<const u32x4 *>(p + 8 * s) ^ a.flip;
            top[rb] = -INFINITY;
            total[rb] = 0.0f;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < E; ++e) o[rb][u][e] = (f32x4){0, 0, 0, 0};
        }

        // A wave's tiles: lo + wave, then every NW-th.  Codes are fetched AHEAD tiles before their use, page numbers one tile before their codes.
        // Loads come back in the order of their issue, so a turn asks for page numbers first: the next turn's wait
        // for them then leaves this turn's codes under way.
        constexpr int AHEAD = 2;
        int t = lo + wave;
        int pi = 2 * t / page16, off = 2 * t % page16, tp = t;   // page and 16-token group of the next page numbers to be fetched, and their tile
        const int step_p = 2 * NW / page16, step_o = 2 * NW % page16;
        int raw[2][2], at16[2][2], pages_of[AHEAD][2];           // page numbers and groups in two sets, taken in turn; a group < 0 is not there
        uint32_t kc[AHEAD][2][KW], vc[AHEAD][2][U];
        auto fetch_pages = [&](int set) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                int x = pi, y = off + s;
                if (y >= page16) x += 1, y = 0;
                const bool in = tp * TILE + 16 * s < n_kv && tp < hi;
                raw[set][s] = table[in ? x : 0];
                at16[set][s] = in ? y : -1;
            }
            pi += step_p;
            off += step_o;
            tp += NW;
            if (off >= page16) pi += 1, off -= page16;
        };
        auto fetch = [&](int slot, int set) {
            fetch_pages(1 - set);
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int n = __builtin_amdgcn_readfirstlane(raw[set][s]), y = __builtin_amdgcn_readfirstlane(at16[set][s]);
                const bool there = y >= 0 && n >= 0 && n < a.pages;
                const int group16 = there ? y * 16 : 0;
                const int64_t base = (there ? n : 0) * page_bytes + head_at;
                pages_of[slot][s] = there ? n : -1;
                const uint8_t *k_from = a.codes[0] + (base + group16 * M), *v_from = a.codes[1] + (base + group16);
                load_bytes<NB>(kc[slot][s], k_from + k_lane);
#pragma unroll
                for (int u = 0; u < U; ++u) vc[slot][s][u] = *reinterpret_cast<const uint32_t *>(v_from + v_lane[u]);
            }
        };
        static_assert(AHEAD == 2, "a turn's slot of codes is also its set of page numbers");
        if (t < hi) {
            fetch_pages(0);
            fetch(0, 0);
            fetch(1, 1);
        }
        auto turn = [&](int slot) {
            uint32_t k_now[2][KW], v_now[2][U];
            const int pg_now[2] = {pages_of[slot][0], pages_of[slot][1]};
#pragma unroll
            for (int s = 0; s < 2; ++s) {
#pragma unroll
                for (int i = 0; i < KW; ++i) k_now[s][i] = kc[slot][s][i] & fold;
#pragma unroll
                for (int u = 0; u < U; ++u) v_now[s][u] = vc[slot][s][u] & fold;
            }
            fetch(slot, slot);                                   // (past the end: page 0, not looked at)
            // Look-ups.  With few waves all of a tile's go first, so that they pass through LDS one behind the other; with many, the waves
            // hide each other's and registers count for more.
            constexpr bool FIRST = NW <= 8 && D <= 128;
            auto look_k = [&](int s, int ks) -> u32x4 {
                u32x4 x;
#pragma unroll
                for (int j = 0; j < 8 / SUB; ++j) {
                    const int n = ks * (8 / SUB) + j;            // the lane's n-th part, g * NB + n of the vector
                    const uint32_t code = (k_now[s][n / 4] >> (8 * (n % 4))) & 255u;
                    const uint32_t at = k_at + g * NB * kstride + n * kstride + code * (SUB * 2);
                    if constexpr (SUB == 8) x = lds<u32x4>(at);
                    else if constexpr (SUB == 4) {
                        const u32x2 v = lds<u32x2>(at);
                        x[2 * j] = v.x, x[2 * j + 1] = v.y;
                    } else x[j] = lds<uint32_t>(at);
                }
                return x;
            };
            auto look_v = [&](int u, uint32_t (&x)[8][E / 2]) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    uint32_t at;
                    if constexpr (VLDS && D == 128) {
                        // a row has 256 bytes: the code is the second byte of the address, put there with the first in one go
                        at = __builtin_amdgcn_perm(v_now[j / 4][u], (uint32_t)(r * E * 2), 0x0c0c0000u | (4u + j % 4) << 8);
                    } else {
                        uint32_t code = (v_now[j / 4][u] >> (8 * (j % 4))) & 255u;
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
            f32x4 z[RB][2];
            uint32_t vx[FIRST ? U : 1][8][E / 2];
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) z[rb][0] = z[rb][1] = (f32x4){0, 0, 0, 0};
            if constexpr (FIRST) {
                u32x4 kx[2][KS];
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) kx[s][ks] = look_k(s, ks);
#pragma unroll
                for (int u = 0; u < U; ++u) look_v(u, vx[u]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int s = 0; s < 2; ++s)
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) z[rb][s] = mfma16<T>(kx[s][ks], q[rb][ks], z[rb][s]);
            } else {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const u32x4 x = look_k(s, ks);
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) z[rb][s] = mfma16<T>(x, q[rb][ks], z[rb][s]);
                    }
            }
            // weights
            u32x4 w[RB];
            const bool whole = pg_now[0] >= 0 && pg_now[1] >= 0 && t * TILE + TILE - 1 <= all_see;
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                if (!whole) {
#pragma unroll
                    for (int s = 0; s < 2; ++s)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (pg_now[s] < 0 || t * TILE + 16 * s + 4 * g + i > sees[rb]) z[rb][s][i] = -INFINITY;
                }
                float best = -INFINITY;
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) best = fmaxf(best, z[rb][s][i]);
                best *= a.scale2;
                if (__any(best > top[rb] + 8.0f)) {
                    const float now = fmaxf(top[rb], wave_any_max(best));
                    const float keep = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top[rb] - now);
                    top[rb] = now;
                    total[rb] *= keep;
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int e = 0; e < E; ++e) o[rb][u][e] *= keep;
                }
                const float base = top[rb] == -INFINITY ? 0.0f : -top[rb];
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) z[rb][s][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[rb][s][i], a.scale2, base));
                total[rb] += ((z[rb][0][0] + z[rb][0][1]) + (z[rb][0][2] + z[rb][0][3])) + ((z[rb][1][0] + z[rb][1][1]) + (z[rb][1][2] + z[rb][1][3]));
                w[rb] = (u32x4){pack2<T>(z[rb][0][0], z[rb][0][1]), pack2<T>(z[rb][0][2], z[rb][0][3]),
                                pack2<T>(z[rb][1][0], z[rb][1][1]), pack2<T>(z[rb][1][2], z[rb][1][3])};
            }
            // values: E numbers of 8 tokens, transposed to E operands of 8 tokens
#pragma unroll
            for (int u = 0; u < U; ++u) {
                uint32_t(&x)[8][E / 2] = vx[FIRST ? u : 0];
                if constexpr (!FIRST) look_v(u, x);
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
            t += NW;
        };
        __builtin_amdgcn_s_waitcnt(0x0f70);                       // all loads: inside the loop no wait is left but those of the codes
        while (t < hi) {
            turn(0);
            if (t >= hi) break;
            turn(1);
        }

        // Join the waves: maxima and sums first, then every wave's part against the common maximum, added in the waves' order, as many
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
        __syncthreads();
        float keep[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            float most = -INFINITY;
#pragma unroll 4
            for (int x = 0; x < NW; ++x) most = fmaxf(most, s_ml[x * ROWS + rb * 16 + r].x);
            keep[rb] = top[rb] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top[rb] - most);
        }
        constexpr int EACH = (ROWS * (D / 8) + NW * 64 - 1) / (NW * 64);       // pieces of 8 numbers a thread adds up
        f32x4 v0[EACH], v1[EACH];
#pragma unroll
        for (int n = 0; n < EACH; ++n) v0[n] = v1[n] = (f32x4){0, 0, 0, 0};
        const int at_once = a.join_rows / rows_here;
        for (int w0 = 0; w0 < NW; w0 += at_once) {
            if (wave >= w0 && wave < w0 + at_once)
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
                    if (rb * 16 + r < rows_here) {
                        float *p = s_o + ((wave - w0) * rows_here + rb * 16 + r) * (D + 4);
#pragma unroll
                        for (int u = 0; u < U; ++u)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
#pragma unroll
                                for (int e = 0; e < E; ++e) p[(u * 16 + 4 * g + i) * E + e] = o[rb][u][e][i] * keep[rb];
                    }
            __syncthreads();
#pragma unroll
            for (int n = 0; n < EACH; ++n) {
                const int i = threadIdx.x + n * NW * 64, x = i / (D / 8), c = i % (D / 8);
                if (x < rows_here)
                    for (int y = w0; y < w0 + at_once && y < NW; ++y) {
                        const float *p = s_o + ((y - w0) * rows_here + x) * (D + 4) + c * 8;
                        v0[n] += *reinterpret_cast<const f32x4 *>(p);
                        v1[n] += *reinterpret_cast<const f32x4 *>(p + 4);
                    }
            }
            __syncthreads();
        }
        const int slot = 2 * me + (skip == 0 ? 1 : 0);
#pragma unroll
        for (int n = 0; n < EACH; ++n) {
            const int i = threadIdx.x + n * NW * 64, x = i / (D / 8), c = i % (D / 8);
            if (x >= rows_here) continue;
            float most = -INFINITY, sum = 0.0f;
#pragma unroll 4
            for (int y = 0; y < NW; ++y) most = fmaxf(most, s_ml[y * ROWS + x].x);
#pragma unroll 4
            for (int y = 0; y < NW; ++y) {
                const float2 ml = s_ml[y * ROWS + x];
                sum += ml.x == -INFINITY ? 0.0f : ml.y * __builtin_amdgcn_exp2f(ml.x - most);
            }
            if (whole_item) {
                const int row = row0 + x;
                store_row<T>(a, (first + row / group) * a.q_heads + h * group + row % group, D, c, v0[n], v1[n], most, sum);
            } else {
                float *p = a.part_o + ((int64_t)slot * ROWS + x) * D + c * 8;
                *reinterpret_cast<f32x4 *>(p) = v0[n];
                *reinterpret_cast<f32x4 *>(p + 4) = v1[n];
                if (c == 0) a.part_ml[(int64_t)slot * ROWS + x] = make_float2(most, sum);
            }
        }
        if (!whole_item && skip == 0) note = AttendNote{b, tile, (int)(((now + cost) * parts + all - 1) / all) - 1, 0};
        __syncthreads();                                          // the next item's sums go to the same place

        left -= take;
        now += cost;
        skip = 0;
        ++tile;
    }
    if (a.parts > 1 && threadIdx.x == 0) a.notes[me] = note;
}

// Joins an item's parts: the one of the workgroup that noted it, then the others in order.
template <typename T, int D, int RB>
__global__ __launch_bounds__(256) void k_cache_join(const AttendArgs a) {
    constexpr int ROWS = RB * 16;
    const int h = blockIdx.x, me = h * gridDim.y + blockIdx.y, group = a.q_heads / a.heads;
    const AttendNote note = a.notes[me];
    if (note.seq < 0) return;
    int64_t first;
    int n_q, n_kv;
    sequence(a, note.seq, first, n_q, n_kv);
    const int pieces = note.last - (int)blockIdx.y + 1;
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
    if (p.lds > 48 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)p.lds);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(kernel, grid, dim3(NW * 64), p.lds, stream, a);
    if (a.parts > 1) hipLaunchKernelGGL((k_cache_join<T, D, RB>), grid, dim3(256), 0, stream, a);
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
