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

#ifndef VQ_RB
#define VQ_RB 4
#define VQ_NW 4
#endif

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

__device__ inline float wave_any_max(float v) {          // the maximum over the four lanes of one row
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}

template <typename T, int D, int SUB, int RB, int NW, bool VLDS>
__global__ __launch_bounds__(NW * 64) void k_cache_attend(const AttendArgs a) {
    constexpr int M = D / SUB, KS = D / 32, NB = M / 4, KW = (NB + 3) / 4;
    constexpr int E = value_chunk(D, SUB), U = D / (16 * E);
    extern __shared__ __align__(16) uint8_t s_mem[];
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = blockIdx.x, b = blockIdx.z;
    const int group = a.q_heads / a.heads;
    int64_t first;
    int n_q, n_kv;
    sequence(a, b, first, n_q, n_kv);
    const int64_t n_rows = (int64_t)n_q * group;
    const int row_tiles = (int)((n_rows + RB * 16 - 1) / (RB * 16));
    const int64_t items = (int64_t)row_tiles * a.splits;
    const int Kp = a.Kp, kstride = key_stride(Kp, SUB);
    const int v_at = (M * kstride + 15) / 16 * 16;
    const int64_t cb0 = a.cb_heads == 1 ? 0 : (int64_t)h * a.K * D;
    const T *k_cb = static_cast<const T *>(a.cb[0]) + cb0, *v_cb = static_cast<const T *>(a.cb[1]) + cb0;
    const int32_t *table = a.table + (int64_t)b * a.width;
    const int page16 = a.page >> 4;
    const uint32_t fold = (uint32_t)(Kp - 1) * 0x01010101u;     // keeps codes of no codeword inside the tables
    const int64_t page_bytes = (int64_t)a.heads * a.page * M;
    const uint8_t *kc0 = a.codes[0] + (int64_t)h * a.page * M + r * M + g * NB;
    const uint8_t *vc0 = a.codes[1] + (int64_t)h * a.page * M + 4 * g;

    for (int64_t item = blockIdx.y; item < items; item += gridDim.y) {
        // the rows that see most come first
        const int tile = row_tiles - 1 - (int)(item / a.splits), split = (int)(item % a.splits);
        const int64_t row0 = (int64_t)tile * RB * 16;
        const int64_t last_row = (row0 + RB * 16 < n_rows ? row0 + RB * 16 : n_rows) - 1;
        const int back = n_kv - n_q;                            // row i sees tokens 0 .. back + i
        const int all_see = back + (int)(row0 / group);         // every row of the tile sees tokens up to here
        int end = back + (int)(last_row / group) + 1;
        end = end < 0 ? 0 : end;
        const int tiles = (end + TILE - 1) / TILE;
        const int lo = split * a.split_tiles < tiles ? split * a.split_tiles : tiles;
        const int hi = split == a.splits - 1 ? tiles : (lo + a.split_tiles < tiles ? lo + a.split_tiles : tiles);

        if (lo < hi) {
            // codebooks -> LDS, 16 bytes at a time; rows past K are zeros
            for (int i = threadIdx.x; i < Kp * (D / 8); i += NW * 64) {
                const int k = i / (D / 8), c = i % (D / 8);
                u32x4 kv = {0, 0, 0, 0}, vv = {0, 0, 0, 0};
                if (k < a.K) {
                    kv = *reinterpret_cast<const u32x4 *>(k_cb + (int64_t)k * D + c * 8);
                    if constexpr (VLDS) vv = *reinterpret_cast<const u32x4 *>(v_cb + (int64_t)k * D + c * 8);
                }
                if constexpr (SUB == 8) {
                    *reinterpret_cast<u32x4 *>(s_mem + c * kstride + k * 16) = kv;
                } else if constexpr (SUB == 4) {
                    *reinterpret_cast<u32x2 *>(s_mem + (2 * c) * kstride + k * 8) = kv.xy;
                    *reinterpret_cast<u32x2 *>(s_mem + (2 * c + 1) * kstride + k * 8) = kv.zw;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) *reinterpret_cast<uint32_t *>(s_mem + (4 * c + j) * kstride + k * 4) = kv[j];
                }
                if constexpr (VLDS) *reinterpret_cast<u32x4 *>(s_mem + v_at + k * (D * 2) + c * 16) = vv;
            }
        }
        __syncthreads();

        u32x4 q[RB][KS];
        int sees[RB];
        f32x4 o[RB][U][E];
        float top[RB], total[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int64_t row = row0 + rb * 16 + r;
            const bool have = row < n_rows;
            const int i = (int)((have ? row : row0) / group), head = h * group + (int)((have ? row : row0) % group);
            const T *p = static_cast<const T *>(a.q) + (first + i) * a.q_token_stride + head * a.q_head_stride + g * (D / 4);
            sees[rb] = back + i;
#pragma unroll
            for (int s = 0; s < KS; ++s) q[rb][s] = *reinterpret_cast<const u32x4 *>(p + 8 * s);
            top[rb] = -INFINITY;
            total[rb] = 0.0f;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < E; ++e) o[rb][u][e] = (f32x4){0, 0, 0, 0};
        }

        // a wave's tiles: lo + wave, then every NW-th; page numbers are fetched two tiles ahead, codes one
        int t = lo + wave;
        int pi = 2 * t / page16, off = 2 * t % page16;          // page and 16-token group of the tile's first half
        const int step_p = 2 * NW / page16, step_o = 2 * NW % page16;
        int pg[2], at16[2];
        uint32_t kc[2][KW], vc[2][U];
        auto fetch_pages = [&](int tt, int (&p)[2], int (&o16)[2]) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                int x = pi, y = off + s;
                if (y >= page16) x += 1, y = 0;
                const bool in = tt * TILE + 16 * s < n_kv;
                int n = in ? table[x] : -1;
                p[s] = (n >= 0 && n < a.pages) ? n : -1;
                o16[s] = in ? y : 0;
            }
            pi += step_p;
            off += step_o;
            if (off >= page16) pi += 1, off -= page16;
        };
        auto fetch_codes = [&](const int (&p)[2], const int (&o16)[2]) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int64_t base = (p[s] < 0 ? 0 : p[s]) * page_bytes;
                load_bytes<NB>(kc[s], kc0 + base + (int64_t)o16[s] * 16 * M);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    vc[s][u] = *reinterpret_cast<const uint32_t *>(vc0 + base + (int64_t)((u * 16 + r) * E / SUB) * a.page + o16[s] * 16);
            }
        };
        int pg_next[2], at_next[2];
        if (t < hi) {
            fetch_pages(t, pg, at16);
            fetch_codes(pg, at16);
            fetch_pages(t + NW, pg_next, at_next);
        }
        for (; t < hi; t += NW) {
            uint32_t k_now[2][KW], v_now[2][U];
            const int pg_now[2] = {pg[0], pg[1]};
#pragma unroll
            for (int s = 0; s < 2; ++s) {
#pragma unroll
                for (int i = 0; i < KW; ++i) k_now[s][i] = kc[s][i] & fold;
#pragma unroll
                for (int u = 0; u < U; ++u) v_now[s][u] = vc[s][u] & fold;
            }
            if (t + NW < hi) {
                pg[0] = pg_next[0], pg[1] = pg_next[1], at16[0] = at_next[0], at16[1] = at_next[1];
                fetch_codes(pg, at16);
                fetch_pages(t + 2 * NW, pg_next, at_next);
            }
            // scores
            f32x4 z[RB][2];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) z[rb][s] = (f32x4){0, 0, 0, 0};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    u32x4 x;
#pragma unroll
                    for (int j = 0; j < 8 / SUB; ++j) {
                        const int n = ks * (8 / SUB) + j;        // the lane's n-th part, g * NB + n of the vector
                        const uint32_t code = (k_now[s][n / 4] >> (8 * (n % 4))) & 255u;
                        const uint8_t *p = s_mem + g * NB * kstride + n * kstride + code * (SUB * 2);
                        if constexpr (SUB == 8) x = *reinterpret_cast<const u32x4 *>(p);
                        else if constexpr (SUB == 4) {
                            const u32x2 v = *reinterpret_cast<const u32x2 *>(p);
                            x[2 * j] = v.x, x[2 * j + 1] = v.y;
                        } else x[j] = *reinterpret_cast<const uint32_t *>(p);
                    }
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) z[rb][s] = mfma16<T>(x, q[rb][ks], z[rb][s]);
                }
            }
            // weights
            u32x4 w[RB];
            const bool whole = pg_now[0] >= 0 && pg_now[1] >= 0 && t * TILE + TILE - 1 <= all_see;
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                float best = -INFINITY;
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float v = z[rb][s][i] * a.scale2;
                        if (!whole && (pg_now[s] < 0 || t * TILE + 16 * s + 4 * g + i > sees[rb])) v = -INFINITY;
                        z[rb][s][i] = v;
                        best = fmaxf(best, v);
                    }
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
                const float base = top[rb] == -INFINITY ? 0.0f : top[rb];
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        z[rb][s][i] = __builtin_amdgcn_exp2f(z[rb][s][i] - base);
                        total[rb] += z[rb][s][i];
                    }
                w[rb] = (u32x4){pack2<T>(z[rb][0][0], z[rb][0][1]), pack2<T>(z[rb][0][2], z[rb][0][3]),
                                pack2<T>(z[rb][1][0], z[rb][1][1]), pack2<T>(z[rb][1][2], z[rb][1][3])};
            }
            // values: E numbers of 8 tokens, transposed to E operands of 8 tokens
#pragma unroll
            for (int u = 0; u < U; ++u) {
                uint32_t x[8][E / 2];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    uint32_t code = (v_now[j / 4][u] >> (8 * (j % 4))) & 255u;
                    if constexpr (!VLDS) code = code < (uint32_t)a.K ? code : (uint32_t)a.K - 1;
                    const uint8_t *p = VLDS ? s_mem + v_at + code * (D * 2) + (u * 16 + r) * E * 2
                                            : reinterpret_cast<const uint8_t *>(v_cb) + code * (D * 2) + (u * 16 + r) * E * 2;
                    if constexpr (E == 8) {
                        const u32x4 v = *reinterpret_cast<const u32x4 *>(p);
                        x[j][0] = v.x, x[j][1] = v.y, x[j][2] = v.z, x[j][3] = v.w;
                    } else if constexpr (E == 4) {
                        const u32x2 v = *reinterpret_cast<const u32x2 *>(p);
                        x[j][0] = v.x, x[j][1] = v.y;
                    } else x[j][0] = *reinterpret_cast<const uint32_t *>(p);
                }
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
        }

        // join the waves: maxima and sums first, then every wave's part against the common maximum, added in the waves' order
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            total[rb] += __shfl_xor(total[rb], 16);
            total[rb] += __shfl_xor(total[rb], 32);
        }
        __syncthreads();                                         // the tables are done with
        float *s_o = reinterpret_cast<float *>(s_mem);
        float2 *s_ml = reinterpret_cast<float2 *>(s_mem + (size_t)NW * RB * 16 * (D + 4) * 4);
        if (g == 0)
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) s_ml[wave * RB * 16 + rb * 16 + r] = make_float2(top[rb], total[rb]);
        __syncthreads();
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            float most = -INFINITY;
#pragma unroll
            for (int x = 0; x < NW; ++x) most = fmaxf(most, s_ml[x * RB * 16 + rb * 16 + r].x);
            const float keep = top[rb] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top[rb] - most);
            float *p = s_o + (wave * RB * 16 + rb * 16 + r) * (D + 4);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < E; ++e) p[(u * 16 + 4 * g + i) * E + e] = o[rb][u][e][i] * keep;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < RB * 16 * (D / 8); i += NW * 64) {
            const int x = i / (D / 8), c = i % (D / 8);
            const int64_t row = row0 + x;
            if (row >= n_rows) continue;
            float most = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int y = 0; y < NW; ++y) most = fmaxf(most, s_ml[y * RB * 16 + x].x);
            f32x4 v0 = {0, 0, 0, 0}, v1 = {0, 0, 0, 0};
#pragma unroll
            for (int y = 0; y < NW; ++y) {
                const float2 ml = s_ml[y * RB * 16 + x];
                sum += ml.x == -INFINITY ? 0.0f : ml.y * __builtin_amdgcn_exp2f(ml.x - most);
                const float *p = s_o + (y * RB * 16 + x) * (D + 4) + c * 8;
                v0 += *reinterpret_cast<const f32x4 *>(p);
                v1 += *reinterpret_cast<const f32x4 *>(p + 4);
            }
            const int64_t place = (first + row / group) * a.q_heads + h * group + row % group;
            if (a.splits > 1) {
                float *p = a.part_o + ((int64_t)split * a.rows * a.q_heads + place) * D + c * 8;
                *reinterpret_cast<f32x4 *>(p) = v0;
                *reinterpret_cast<f32x4 *>(p + 4) = v1;
                if (c == 0) a.part_ml[(int64_t)split * a.rows * a.q_heads + place] = make_float2(most, sum);
            } else {
                const float over = sum > 0.0f ? 1.0f / sum : 0.0f;
                *reinterpret_cast<u32x4 *>(static_cast<T *>(a.out) + place * D + c * 8) =
                    (u32x4){pack2<T>(v0[0] * over, v0[1] * over), pack2<T>(v0[2] * over, v0[3] * over),
                            pack2<T>(v1[0] * over, v1[1] * over), pack2<T>(v1[2] * over, v1[3] * over)};
                if (c == 0 && a.lse) a.lse[place] = sum > 0.0f ? most * 0.69314718055994531f + logf(sum) : -INFINITY;
            }
        }
        __syncthreads();
    }
}

// Joins the pieces of the context: one thread for 8 numbers of a row.
template <typename T>
__global__ __launch_bounds__(256) void k_cache_join(const AttendArgs a, int D) {
    int64_t begin = a.starts[0], end = a.starts[a.seqs];
    begin = begin < 0 ? 0 : begin;
    end = end > a.rows ? a.rows : end;
    const int64_t all = a.rows * a.q_heads;
    const int chunks = D / 8;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all * chunks; i += (int64_t)gridDim.x * 256) {
        const int64_t place = i / chunks;
        const int c = (int)(i % chunks);
        if (place / a.q_heads < begin || place / a.q_heads >= end) continue;
        float most = -INFINITY, sum = 0.0f;
        for (int s = 0; s < a.splits; ++s) most = fmaxf(most, a.part_ml[s * all + place].x);
        f32x4 v0 = {0, 0, 0, 0}, v1 = {0, 0, 0, 0};
        for (int s = 0; s < a.splits; ++s) {
            const float2 ml = a.part_ml[s * all + place];
            if (ml.x == -INFINITY) continue;
            const float keep = __builtin_amdgcn_exp2f(ml.x - most);
            const float *p = a.part_o + (s * all + place) * D + c * 8;
            sum += ml.y * keep;
            v0 += *reinterpret_cast<const f32x4 *>(p) * keep;
            v1 += *reinterpret_cast<const f32x4 *>(p + 4) * keep;
        }
        const float over = sum > 0.0f ? 1.0f / sum : 0.0f;
        *reinterpret_cast<u32x4 *>(static_cast<T *>(a.out) + place * D + c * 8) =
            (u32x4){pack2<T>(v0[0] * over, v0[1] * over), pack2<T>(v0[2] * over, v0[3] * over),
                    pack2<T>(v1[0] * over, v1[1] * over), pack2<T>(v1[2] * over, v1[3] * over)};
        if (c == 0 && a.lse) a.lse[place] = sum > 0.0f ? most * 0.69314718055994531f + logf(sum) : -INFINITY;
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
    if (a.splits > 1) {
        const int64_t blocks = (a.rows * a.q_heads * (D / 8) + 255) / 256;
        hipLaunchKernelGGL(k_cache_join<T>, dim3((unsigned)(blocks > 65536 ? 65536 : blocks)), dim3(256), 0, stream, a, D);
    }
    return hipGetLastError();
}

template <int D, int SUB>
hipError_t launch_rows(const AttendArgs &a, const AttendPlan &p, dim3 grid, hipStream_t stream) {
#define VQ_TRY(RB, NW, VLDS) \
    if (p.rb == RB && p.nw == NW && p.values_in_lds == VLDS) return launch<D, SUB, RB, NW, VLDS>(a, p, grid, stream)
    VQ_TRY(1, 8, true);
    if constexpr (D >= 192) {
        VQ_TRY(1, 8, false);
        VQ_TRY(2, 4, false);
        VQ_TRY(2, 4, true);
    } else {
        VQ_TRY(VQ_RB, VQ_NW, true);
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
