// vq_cache.hip -- HIP kernels (gfx950 / CDNA4) and C ABI of the vector-quantised key-value cache (vq_cache.h).
#include <stdarg.h>
#include <stdio.h>
#include <type_traits>

#include "vq_cache_internal.h"


namespace {

int fail(int code, const char *fmt, ...) {
    char text[400];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof(text), fmt, ap);
    va_end(ap);
    return vq_internal_fail(code, text);
}

#define LAUNCH_CHECK(name)                                                                         \
    do {                                                                                           \
        hipError_t e_ = hipGetLastError();                                                         \
        if (e_ != hipSuccess) return fail(VQ_E_HIP, "launch of %s failed: %s", name, hipGetErrorString(e_)); \
    } while (0)

// ------------------------------------------------------------------------------------------------
// kernels
// ------------------------------------------------------------------------------------------------

struct ReadArgs {
    const int64_t *slots;
    int64_t tokens, pages;
    const void *cb[2];
    int cb_heads, heads, K;
    int page, page_shift;              // page = 1 << page_shift, or page_shift < 0
    int chunk;                         // tokens a workgroup takes
    const uint8_t *codes[2];
    void *out[2];
};

// Codes -> vectors.  Bound by the writes: 65536 tokens of 8 heads and 128 dims, 268 MB of vectors out of 34 MB of codes, take 54 us, 5.6 TB/s;
// a copy reaches 5.0.  A few tokens are 4 us of latency.  A thread writes 16 bytes, 8 numbers of 8 / SUB codewords; neighbouring threads
// write neighbouring ones.

// The 16 bytes that N codes stand for, at place c of a vector.
template <int D, int SUB> __device__ inline u32x4 expand(const uint8_t *book, uint32_t codes, int K, int c) {
    u32x4 v;
#pragma unroll
    for (int j = 0; j < 8 / SUB; ++j) {
        const int code = codes >> (8 * j) & 255u, k = code < K ? code : K - 1;
        const uint8_t *w = book + k * (D * 2) + c * 16 + j * (SUB * 2);
        if constexpr (SUB == 8) v = *reinterpret_cast<const u32x4 *>(w);
        else if constexpr (SUB == 4) {
            const u32x2 x = *reinterpret_cast<const u32x2 *>(w);
            v[2 * j] = x.x, v[2 * j + 1] = x.y;
        } else v[j] = *reinterpret_cast<const uint32_t *>(w);
    }
    return v;
}
// Where the codes of a slot lie: the head's first byte of its page, and its place in the page.  A slot outside the cache: false.
__device__ inline bool locate(const ReadArgs &a, int64_t slot, int64_t page_bytes, int64_t &from, int &o) {
    if (slot < 0 || slot >= a.pages * a.page) return false;
    const int64_t p = a.page_shift >= 0 ? slot >> a.page_shift : slot / a.page;
    from = p * page_bytes;
    o = (int)(slot - p * a.page);
    return true;
}

// A few tokens: everything comes out of the caches.
template <int D, int SUB>
__global__ __launch_bounds__(512) void k_cache_read_few(const ReadArgs a) {
    constexpr int M = D / SUB, CH = D / 8, N = 8 / SUB;
    const int h = blockIdx.x, which = blockIdx.z;
    const uint8_t *book = static_cast<const uint8_t *>(a.cb[which]) + (a.cb_heads == 1 ? 0 : (int64_t)h * a.K * D * 2);
    const int64_t begin = (int64_t)blockIdx.y * a.chunk, end = begin + a.chunk < a.tokens ? begin + a.chunk : a.tokens;
    const uint8_t *codes = a.codes[which] + (int64_t)h * a.page * M;
    uint8_t *out = static_cast<uint8_t *>(a.out[which]);
    for (int64_t i = begin * CH + threadIdx.x; i < end * CH; i += 512) {
        const int c = (int)(i % CH);
        int64_t from;
        int o;
        u32x4 v = {0, 0, 0, 0};
        if (locate(a, a.slots[i / CH], (int64_t)a.heads * a.page * M, from, o)) {
            uint32_t w = 0;
#pragma unroll
            for (int j = 0; j < N; ++j)
                w |= (uint32_t)codes[from + (which == 0 ? (int64_t)o * M + c * N + j : (int64_t)(c * N + j) * a.page + o)] << (8 * j);
            v = expand<D, SUB>(book, w, a.K, c);
        }
        *reinterpret_cast<u32x4 *>(out + (i / CH * a.heads + h) * (D * 2) + c * 16) = v;
    }
}

// Many: a workgroup holds one head's codebook in LDS (both cache types have 2 bytes a number) and expands `chunk` tokens, READ_TOKENS at a
// time.  Their codes pass through LDS, where those of the next are put once they have come, so that they are fetched the way they lie: a
// key's side by side, of the values one part of neighbouring tokens.  (Fetched as they are used, by threads of neighbouring parts,
// the values' bytes came out of 16 lines a load, and reading the values took 85 us where the keys took 50.)
constexpr int READ_TOKENS = 128;
constexpr int read_row(int M) { return M + 4; }           // a token's codes in LDS, padded: the stores of one part go to different banks
template <int D, int SUB, bool PAST>                      // PAST: the vectors are stored past the caches
__global__ __launch_bounds__(512) void k_cache_read(const ReadArgs a) {
    constexpr int M = D / SUB, CH = D / 8, N = 8 / SUB, ROW = read_row(M);
    constexpr int WORDS = READ_TOKENS * M / 4, EACH_K = (WORDS + 511) / 512, EACH_V = M / 4;     // fetches a thread: words of keys' codes, values' bytes
    extern __shared__ __align__(16) uint8_t s_book[];
    uint8_t *s_codes = s_book + (size_t)a.K * D * 2;
    uint8_t *s_there = s_codes + READ_TOKENS * ROW;
    const int h = blockIdx.x, which = blockIdx.z;
    const uint8_t *book = static_cast<const uint8_t *>(a.cb[which]) + (a.cb_heads == 1 ? 0 : (int64_t)h * a.K * D * 2);
    for (int i = threadIdx.x; i < a.K * CH; i += 512) reinterpret_cast<u32x4 *>(s_book)[i] = reinterpret_cast<const u32x4 *>(book)[i];
    const int64_t begin = (int64_t)blockIdx.y * a.chunk, end = begin + a.chunk < a.tokens ? begin + a.chunk : a.tokens;
    const int64_t page_bytes = (int64_t)a.heads * a.page * M;
    const uint8_t *codes = a.codes[which] + (int64_t)h * a.page * M;
    uint8_t *out = static_cast<uint8_t *>(a.out[which]);

    auto find = [&](int64_t token, int64_t &from, int &o) -> bool { return token < end && locate(a, a.slots[token], page_bytes, from, o); };
    auto work = [&](auto keys) {                                  // (both sides' loops apart: each with its own registers)
        constexpr bool KEYS = decltype(keys)::value;
        constexpr int EACH = KEYS ? EACH_K : EACH_V;
        uint32_t got[EACH];
        bool there[KEYS ? EACH : 1];
        auto fetch = [&](int64_t t0) {
            int64_t from = 0;
            int o = 0;
            if constexpr (KEYS) {
#pragma unroll
                for (int n = 0; n < EACH; ++n) {
                    const int i = threadIdx.x + n * 512;
                    got[n] = 0;
                    there[n] = i < WORDS && find(t0 + i / (M / 4), from, o);
                    if (there[n]) got[n] = *reinterpret_cast<const uint32_t *>(codes + from + (int64_t)o * M + i % (M / 4) * 4);
                }
            } else {
                there[0] = find(t0 + threadIdx.x % READ_TOKENS, from, o);
#pragma unroll
                for (int n = 0; n < EACH; ++n) {
                    got[n] = 0;
                    if (there[0]) got[n] = codes[from + (int64_t)(threadIdx.x / READ_TOKENS + 4 * n) * a.page + o];
                }
            }
        };
        auto put = [&]() {
            if constexpr (KEYS) {
#pragma unroll
                for (int n = 0; n < EACH; ++n) {
                    const int i = threadIdx.x + n * 512, t = i / (M / 4), w = i % (M / 4);
                    if (i >= WORDS) continue;
                    *reinterpret_cast<uint32_t *>(s_codes + t * ROW + w * 4) = got[n];
                    if (w == 0) s_there[t] = there[n];
                }
            } else {
                const int t = threadIdx.x % READ_TOKENS, m = threadIdx.x / READ_TOKENS;
#pragma unroll
                for (int n = 0; n < EACH; ++n) s_codes[t * ROW + m + 4 * n] = (uint8_t)got[n];
                if (m == 0) s_there[t] = there[0];
            }
        };
        fetch(begin);
        for (int64_t t0 = begin; t0 < end; t0 += READ_TOKENS) {
            put();
            __syncthreads();
            if (t0 + READ_TOKENS < end) fetch(t0 + READ_TOKENS);
            const int here = end - t0 < READ_TOKENS ? (int)(end - t0) : READ_TOKENS;
#pragma unroll 4
            for (int i = threadIdx.x; i < here * CH; i += 512) {
                const int t = i / CH, c = i % CH;
                const uint8_t *q = s_codes + t * ROW + c * N;
                uint32_t w;
                if constexpr (N == 1) w = *q;
                else if constexpr (N == 2) w = *reinterpret_cast<const uint16_t *>(q);
                else w = *reinterpret_cast<const uint32_t *>(q);
                u32x4 v = expand<D, SUB>(s_book, w, a.K, c);
                if (!s_there[t]) v = (u32x4){0, 0, 0, 0};
                u32x4 *to = reinterpret_cast<u32x4 *>(out + ((t0 + t) * a.heads + h) * (D * 2) + c * 16);
                if constexpr (PAST) __builtin_nontemporal_store(v, to);
                else *to = v;
            }
            __syncthreads();
        }
    };
    if (which == 0) work(std::true_type{});
    else work(std::false_type{});
}

template <int D, int SUB, bool PAST> hipError_t launch_read_many(const ReadArgs &a, dim3 grid, hipStream_t stream) {
    const size_t lds = (size_t)a.K * D * 2 + READ_TOKENS * (read_row(D / SUB) + 1);
    static_assert(256 * D * 2 + READ_TOKENS * (read_row(D / SUB) + 1) <= LDS_MOST, "codebook and codes fit into LDS");
    static std::atomic<uint64_t> allowed{0};
    const hipError_t e = vq_internal_allow_lds(reinterpret_cast<const void *>(k_cache_read<D, SUB, PAST>), allowed);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((k_cache_read<D, SUB, PAST>), grid, dim3(512), lds, stream, a);
    return hipGetLastError();
}

template <int D, int SUB> hipError_t launch_read(const ReadArgs &a, hipStream_t stream) {
    // A codebook goes to LDS where a workgroup's look-ups are worth the staging; those of a few tokens, and few of 16 bytes, go to the caches.
    // (8 heads, 256 codewords, from the caches and through LDS, us: 128 dims by 4: 4.2 and 4.1 at 64 tokens, 10.8 and 7.5 at 4096; 256
    // dims by 2: 2.9 and 5.4 at one token, 9.4 and 6.4 at 64; 2 heads, 256 dims by 8: 4.7 and 5.0 at 64, 6.1 and 6.5 at 4096.)
    const dim3 grid(a.heads, (unsigned)((a.tokens + a.chunk - 1) / a.chunk), 2);
    // What the last cache (256 MB) can keep for whoever reads it next is left there; more is stored past it.  Read and then added up by another
    // kernel, 128 MiB of vectors took 56 us with the caches and 59 past them, 160 MiB 86 and 79, 192 MiB 108 and 90, 512 MiB 314 and
    // 303 (by itself the read of 256 MiB takes 80 and 54).
    const bool past = a.tokens * a.heads * D * 4 > (int64_t)144 << 20;
    if ((a.tokens < a.chunk ? a.tokens : a.chunk) * (16 / SUB) >= a.K)
        return past ? launch_read_many<D, SUB, true>(a, grid, stream) : launch_read_many<D, SUB, false>(a, grid, stream);
    hipLaunchKernelGGL((k_cache_read_few<D, SUB>), grid, dim3(512), 0, stream, a);
    return hipGetLastError();
}

template <int D> hipError_t launch_read(const ReadArgs &a, int sub, hipStream_t stream) {
    return sub == 2 ? launch_read<D, 2>(a, stream) : sub == 4 ? launch_read<D, 4>(a, stream) : launch_read<D, 8>(a, stream);
}

// The closing half by itself: a workgroup for each head and part, a thread for each codeword.
__global__ __launch_bounds__(256) void k_lbg_close(const double *sums, const int64_t *counts, const double *dist, const float *cb_old, int dim,
                                                   int sub, int K, float *cb_new, double *mean_dist) {
    __shared__ int64_t s_n[256];
    const int parts = dim / sub, h = blockIdx.x / parts, m = blockIdx.x % parts, k = threadIdx.x;
    const int64_t n = k < K ? counts[(int64_t)blockIdx.x * K + k] : 0;
    s_n[k] = n;
    __syncthreads();
    for (int o = 128; o; o >>= 1) {
        if (k < o) s_n[k] += s_n[k + o];
        __syncthreads();
    }
    if (k == 0) mean_dist[blockIdx.x] = s_n[0] > 0 ? dist[blockIdx.x] / (double)s_n[0] : 0.0;
    if (k >= K) return;
    const int64_t at = ((int64_t)h * K + k) * dim + m * sub;
    for (int e = 0; e < sub; ++e) cb_new[at + e] = n > 0 ? (float)(sums[at + e] / (double)n) : cb_old[at + e];
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
int check_shape(int heads, int dim, int sub, int K) {
    if (heads <= 0) return fail(VQ_E_INVALID, "need heads > 0 (got %d)", heads);
    if (heads > 1024) return fail(VQ_E_UNSUPPORTED, "heads=%d: at most 1024", heads);
    if (dim != 32 && dim != 64 && dim != 96 && dim != 128 && dim != 192 && dim != 256)
        return fail(VQ_E_UNSUPPORTED, "dim=%d: 32, 64, 96, 128, 192 or 256", dim);
    if (sub != 2 && sub != 4 && sub != 8) return fail(VQ_E_UNSUPPORTED, "sub=%d: 2, 4 or 8", sub);
    if (K < 1 || K > 256) return fail(VQ_E_UNSUPPORTED, "K=%d: a code is one byte, 1 to 256 codewords", K);
    return VQ_OK;
}

int check_cache(const void *k_codes, const void *v_codes, const void *k_cb, const void *v_cb, int cb_heads, int heads,
                int64_t pages, int page, int dtype) {
    if (!k_codes || !v_codes || !k_cb || !v_cb) return fail(VQ_E_INVALID, "null pointer");
    if (((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_cb | (uintptr_t)v_cb) & 15)
        return fail(VQ_E_INVALID, "codes and codebooks must start at multiples of 16 bytes");
    if (cb_heads != 1 && cb_heads != heads) return fail(VQ_E_INVALID, "cb_heads=%d: 1 or heads (%d)", cb_heads, heads);
    if (pages <= 0 || pages > 0x7fffffff) return fail(VQ_E_INVALID, "need 0 < pages < 2^31");
    if (page <= 0 || page > (1 << 20)) return fail(VQ_E_INVALID, "need 0 < page <= 2^20 (got %d)", page);
    if (page % 16) return fail(VQ_E_UNSUPPORTED, "page=%d: a multiple of 16", page);
    if (dtype != VQ_BF16 && dtype != VQ_F16) return fail(VQ_E_UNSUPPORTED, "cache vectors are VQ_BF16 or VQ_F16");
    return VQ_OK;
}

// Vectors are read 16 bytes at a time: both strides have to keep that alignment.
int check_vectors(const char *name, const void *p, int64_t token_stride, int64_t head_stride, int64_t size) {
    if (!p) return fail(VQ_E_INVALID, "null pointer");
    if (((uintptr_t)p & 15) || (token_stride * size) % 16 || (head_stride * size) % 16)
        return fail(VQ_E_INVALID, "the vectors of %s must start at multiples of 16 bytes", name);
    return VQ_OK;
}

int64_t at_most(int64_t n, int64_t most) { return n < most ? n : most; }

// How many rows a workgroup takes at a time and how many workgroups a head gets.  Host arithmetic on sizes alone.
struct Attention {
    AttendPlan p;
    int parts, join_at, join_rows, seq_at;
    bool split;
    size_t slots, ws;
};
Attention plan_attention(int q_heads, int heads, int dim, int sub, int K, int seqs, int64_t max_q, int64_t max_kv) {
    constexpr int CUS = 256;
    Attention r;
    const int Kp = dim <= 128 ? 256 : rows_padded(K), group = q_heads / heads;      // (as k_cache_attend lays out its tables)
    const int64_t per_seq = at_most(max_q, 0x3fffffff) * group;
    // Behind the tables lie the waves' maxima and sums, 16 rows of at least one wave, and the workgroup's range.  More than 16 rows a sequence
    // go 32 at a time, so that a look-up serves twice the products; the value table fits beside them wherever it does beside 16.
    // (16 sequences of 20000 tokens, 4 rows: 53 us by 16 rows, 62 by 32; of 4000 tokens, 32 rows: 34 and 31; a chunk of 8192 rows on 16384
    // tokens: 1081 and 673.)
    const size_t keys = key_bytes(Kp, dim, sub), values = (size_t)Kp * dim * 2, row = (size_t)(dim + 4) * 4;
    auto waves = [&](int rb) { return rb == 2 && dim >= 192 ? 4 : 8; };
    auto fits = [&](int rb, size_t tables) { return tables + (size_t)waves(rb) * rb * 16 * 8 + 16 * row + SEQ_BYTES <= LDS_MOST; };
    r.p.rb = per_seq <= 16 ? 1 : 2;
    r.p.nw = waves(r.p.rb);
    r.p.values_in_lds = fits(r.p.rb, keys + values);
    const int rows = r.p.rb * 16;
    const size_t ml = (size_t)r.p.nw * rows * 8, tables = keys + (r.p.values_in_lds ? values : 0);
    const size_t room = (LDS_MOST - SEQ_BYTES - tables - ml) / row, most = (size_t)r.p.nw * rows;      // (room >= 16: it fits)
    r.join_at = (int)tables;
    r.join_rows = (int)(room < most ? room : most);
    r.seq_at = (int)(tables + ml + r.join_rows * row);
    r.p.lds = r.seq_at + SEQ_BYTES;
    // a head has at most so many items and tiles, by the caller's word
    const int64_t items = at_most(at_most((per_seq + rows - 1) / rows, 0x3fffffff) * seqs, 0x3fffffff);
    const int64_t tiles = items * ((at_most(max_kv, 0x7fffffff) + TILE - 1) / TILE);
    const int64_t wanted = parts_wanted(tiles, items);
    int64_t parts = (CUS + heads - 1) / heads;
    if (parts * heads > CUS && parts > 1) --parts;
    const bool whole = items <= parts && tiles <= items * WHOLE_TILES;
    parts = whole ? items : parts < wanted ? parts : wanted;
    r.parts = (int)(parts < 1 ? 1 : parts);
    r.split = !whole && r.parts > 1;
    r.slots = r.split ? (size_t)2 * heads * r.parts : 0;
    r.ws = r.slots * (rows * ((size_t)dim * 4 + 8)) + r.slots / 2 * sizeof(AttendNote);
    return r;
}

int lbg(const void *x, int64_t token_stride, int64_t head_stride, int64_t tokens, const float *cb, int sub, int dtype, const LbgOut &out,
        void *ws, size_t ws_bytes, void *stream) {
    const int heads = out.heads, dim = out.dim, K = out.K;
    int rc = check_shape(heads, dim, sub, K);
    if (rc) return rc;
    if (dtype != VQ_F32 && dtype != VQ_BF16 && dtype != VQ_F16) return fail(VQ_E_UNSUPPORTED, "dtype=%d", dtype);
    if (tokens < 1) return fail(VQ_E_INVALID, "need tokens >= 1");
    if (tokens > 0x7fffffff) return fail(VQ_E_UNSUPPORTED, "tokens below 2^31");
    if (!cb || !out.counts || !out.dist) return fail(VQ_E_INVALID, "null pointer");
    if ((uintptr_t)cb & 15) return fail(VQ_E_INVALID, "the codebook must start at a multiple of 16 bytes");
    if ((rc = check_vectors("x", x, token_stride, head_stride, dtype == VQ_F32 ? 4 : 2))) return rc;
    const SearchPlan p = vq_internal_search_plan(tokens, heads, dim, sub, 1);
    if (p.blocks > 65535) return fail(VQ_E_UNSUPPORTED, "tokens=%lld: at most 65535 chunks of 4096 in one call", (long long)tokens);
    const size_t need = vq_cache_lbg_ws_bytes(tokens, heads, dim, sub, K);
    if (!ws || ws_bytes < need) return fail(VQ_E_WORKSPACE, "workspace of %zu bytes, %zu needed", ws ? ws_bytes : 0, need);
    if ((uintptr_t)ws & 15) return fail(VQ_E_INVALID, "the workspace must start at a multiple of 16 bytes");
    hipStream_t st = static_cast<hipStream_t>(stream);
    double2 *part_dist = static_cast<double2 *>(ws);
    float *part_sums = reinterpret_cast<float *>(part_dist + (int64_t)p.chunks * heads * (dim / sub));
    const SearchArgs a = {{x, x}, {token_stride, token_stride}, {head_stride, head_stride}, {cb, cb}, tokens, heads, heads, dim, K, p.pw, p.chunk,
                          nullptr, 0, 0, 0, nullptr, nullptr, part_sums, part_dist};
    hipError_t e = vq_internal_search(a, sub, dtype, true, p.blocks, st);
    if (e == hipSuccess) e = vq_internal_lbg_gather(a, sub, p.chunks, out, st);
    if (e != hipSuccess) return fail(VQ_E_HIP, "launch of k_cache_search failed: %s", hipGetErrorString(e));
    return VQ_OK;
}

}  // namespace

hipError_t vq_internal_allow_lds(const void *kernel, std::atomic<uint64_t> &allowed) {
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return e;
    const uint64_t bit = device < 64 ? 1ull << device : 0;        // (further devices are asked every time)
    if (allowed.load(std::memory_order_acquire) & bit) return hipSuccess;
    e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS_MOST);
    if (e == hipSuccess) allowed.fetch_or(bit, std::memory_order_release);
    return e;
}

extern "C" {

int vq_cache_write(const void *k, int64_t k_token_stride, int64_t k_head_stride, const void *v, int64_t v_token_stride,
                   int64_t v_head_stride, const int64_t *slots, int64_t tokens, const void *k_cb, const void *v_cb, int cb_heads,
                   int heads, int dim, int sub, int K, int dtype, uint8_t *k_codes, uint8_t *v_codes, int64_t pages, int page,
                   void *stream) {
    int rc = check_shape(heads, dim, sub, K);
    if (rc) return rc;
    if ((rc = check_cache(k_codes, v_codes, k_cb, v_cb, cb_heads, heads, pages, page, dtype))) return rc;
    if (tokens < 0) return fail(VQ_E_INVALID, "need tokens >= 0");
    if (tokens > 0x7fffffff) return fail(VQ_E_UNSUPPORTED, "tokens below 2^31");
    if (tokens == 0) return VQ_OK;
    if (!slots) return fail(VQ_E_INVALID, "null pointer");
    if ((rc = check_vectors("k", k, k_token_stride, k_head_stride, 2))) return rc;
    if ((rc = check_vectors("v", v, v_token_stride, v_head_stride, 2))) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const SearchPlan p = vq_internal_search_plan(tokens, heads, dim, sub, 2);
    const SearchArgs a = {{k, v}, {k_token_stride, v_token_stride}, {k_head_stride, v_head_stride}, {k_cb, v_cb}, tokens, cb_heads, heads, dim, K,
                          p.pw, p.chunk, slots, pages, page, page & (page - 1) ? -1 : __builtin_ctz(page), k_codes, v_codes, nullptr, nullptr};
    const hipError_t e = vq_internal_search(a, sub, dtype, false, p.blocks, st);
    if (e != hipSuccess) return fail(VQ_E_HIP, "launch of k_cache_search failed: %s", hipGetErrorString(e));
    return VQ_OK;
}

int vq_cache_read(const int64_t *slots, int64_t tokens, const void *k_cb, const void *v_cb, int cb_heads, int heads, int dim,
                  int sub, int K, int dtype, const uint8_t *k_codes, const uint8_t *v_codes, int64_t pages, int page, void *k_out,
                  void *v_out, void *stream) {
    int rc = check_shape(heads, dim, sub, K);
    if (rc) return rc;
    if ((rc = check_cache(k_codes, v_codes, k_cb, v_cb, cb_heads, heads, pages, page, dtype))) return rc;
    if (tokens < 0) return fail(VQ_E_INVALID, "need tokens >= 0");
    if (tokens > 0x7fffffff) return fail(VQ_E_UNSUPPORTED, "tokens below 2^31");
    if (tokens == 0) return VQ_OK;
    if (!slots) return fail(VQ_E_INVALID, "null pointer");
    if ((rc = check_vectors("k_out", k_out, dim, dim, 2))) return rc;
    if ((rc = check_vectors("v_out", v_out, dim, dim, 2))) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    // two workgroups for each compute unit, of 64 tokens at least
    int64_t chunk = (tokens * heads * 2 + 511) / 512;
    chunk = chunk < 64 ? 64 : chunk;
    if ((tokens + chunk - 1) / chunk > 65535) chunk = (tokens + 65534) / 65535;
    const ReadArgs a = {slots, tokens, pages, {k_cb, v_cb}, cb_heads, heads, K, page, page & (page - 1) ? -1 : __builtin_ctz(page), (int)chunk,
                        {k_codes, v_codes}, {k_out, v_out}};
    hipError_t e;
    switch (dim) {
        case 32: e = launch_read<32>(a, sub, st); break;
        case 64: e = launch_read<64>(a, sub, st); break;
        case 96: e = launch_read<96>(a, sub, st); break;
        case 128: e = launch_read<128>(a, sub, st); break;
        case 192: e = launch_read<192>(a, sub, st); break;
        default: e = launch_read<256>(a, sub, st); break;
    }
    if (e != hipSuccess) return fail(VQ_E_HIP, "launch of k_cache_read failed: %s", hipGetErrorString(e));
    return VQ_OK;
}

size_t vq_cache_attention_ws_bytes(int64_t rows, int q_heads, int heads, int dim, int sub, int K, int seqs, int64_t max_q,
                                   int64_t max_kv) {
    if (rows <= 0 || q_heads <= 0 || q_heads > 4096 || seqs <= 0 || max_q < 1 || max_kv < 1 || check_shape(heads, dim, sub, K) ||
        q_heads % heads)
        return 0;
    return plan_attention(q_heads, heads, dim, sub, K, seqs, max_q, max_kv).ws;
}

int vq_cache_attention(const void *q, int64_t q_token_stride, int64_t q_head_stride, int64_t rows, int q_heads, const void *k_cb,
                       const void *v_cb, int cb_heads, int heads, int dim, int sub, int K, int dtype, const uint8_t *k_codes,
                       const uint8_t *v_codes, int64_t pages, int page, const int32_t *table, int seqs, int width,
                       const int32_t *kv_lens, const int32_t *starts, int64_t max_q, int64_t max_kv, double scale, void *out,
                       float *lse, void *ws, size_t ws_bytes, void *stream) {
    int rc = check_shape(heads, dim, sub, K);
    if (rc) return rc;
    if ((rc = check_cache(k_codes, v_codes, k_cb, v_cb, cb_heads, heads, pages, page, dtype))) return rc;
    if (q_heads <= 0 || q_heads % heads) return fail(VQ_E_INVALID, "q_heads=%d: a positive multiple of heads (%d)", q_heads, heads);
    if (q_heads > 4096) return fail(VQ_E_UNSUPPORTED, "q_heads=%d: at most 4096", q_heads);
    if (rows < 0 || seqs < 0 || width < 0) return fail(VQ_E_INVALID, "need rows, seqs and width >= 0");
    if (rows > 0x3fffffff || rows * (q_heads / heads) > 0x3fffffff || (int64_t)width * page > 0x7fffffff)
        return fail(VQ_E_UNSUPPORTED, "rows * q_heads / heads below 2^30, width * page below 2^31");
    if (max_q < 1 || max_kv < 1) return fail(VQ_E_INVALID, "need max_q and max_kv >= 1");
    if (!(fabs(scale) < 1e38)) return fail(VQ_E_INVALID, "scale must be finite and below 1e38 in size");
    if (rows == 0 || seqs == 0) return VQ_OK;
    if (seqs > 65535) return fail(VQ_E_UNSUPPORTED, "seqs=%d: at most 65535", seqs);
    if ((!table && width > 0) || !kv_lens || !starts) return fail(VQ_E_INVALID, "null pointer");
    if ((rc = check_vectors("q", q, q_token_stride, q_head_stride, 2))) return rc;
    if ((rc = check_vectors("out", out, dim, dim, 2))) return rc;
    const Attention r = plan_attention(q_heads, heads, dim, sub, K, seqs, max_q, max_kv);
    if (r.ws > 0 && (!ws || ws_bytes < r.ws)) return fail(VQ_E_WORKSPACE, "workspace of %zu bytes, %zu needed", ws ? ws_bytes : 0, r.ws);
    if (r.ws > 0 && ((uintptr_t)ws & 15)) return fail(VQ_E_INVALID, "the workspace must start at a multiple of 16 bytes");
    float *part_o = static_cast<float *>(ws);
    float2 *part_ml = reinterpret_cast<float2 *>(part_o + r.slots * r.p.rb * 16 * dim);
    AttendArgs a = {q, q_token_stride, q_head_stride, rows, q_heads, {k_cb, v_cb}, cb_heads, heads, K, rows_padded(K), {k_codes, v_codes}, pages,
                    page, table, seqs, width, kv_lens, starts, (float)fmax(fabs(scale) * 1.4426950408889634, 1e-45), scale < 0 ? 0x80008000u : 0u,
                    out, lse, r.split, r.join_at, r.join_rows, r.seq_at, part_o, part_ml,
                    reinterpret_cast<AttendNote *>(part_ml + r.slots * r.p.rb * 16)};
    const dim3 grid(heads, r.parts);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const hipError_t e = (dtype == VQ_BF16 ? vq_internal_attend_bf16 : vq_internal_attend_f16)(a, r.p, dim, sub, grid, st);
    if (e != hipSuccess) return fail(VQ_E_HIP, "launch of k_cache_attend failed: %s", hipGetErrorString(e));
    return VQ_OK;
}

size_t vq_cache_lbg_ws_bytes(int64_t tokens, int heads, int dim, int sub, int K) {
    if (tokens <= 0 || tokens > 0x7fffffff || check_shape(heads, dim, sub, K)) return 0;
    const SearchPlan p = vq_internal_search_plan(tokens, heads, dim, sub, 1);
    return (size_t)p.chunks * heads * (dim / sub) * ((sub + 1) * 256 * 4 + 16);
}

int vq_cache_lbg_accum(const void *x, int64_t token_stride, int64_t head_stride, int64_t tokens, const float *cb, int heads, int dim,
                       int sub, int K, int dtype, double *sums, int64_t *counts, double *dist, void *ws, size_t ws_bytes,
                       void *stream) {
    if (!sums) return fail(VQ_E_INVALID, "null pointer");
    return lbg(x, token_stride, head_stride, tokens, cb, sub, dtype, {heads, dim, K, sums, counts, dist, cb, nullptr}, ws, ws_bytes, stream);
}

int vq_cache_lbg_iterate(const void *x, int64_t token_stride, int64_t head_stride, int64_t tokens, const float *cb, int heads, int dim,
                         int sub, int K, int dtype, float *cb_new, int64_t *counts, double *mean_dist, void *ws, size_t ws_bytes,
                         void *stream) {
    if (!cb_new) return fail(VQ_E_INVALID, "null pointer");
    return lbg(x, token_stride, head_stride, tokens, cb, sub, dtype, {heads, dim, K, nullptr, counts, mean_dist, cb, cb_new}, ws, ws_bytes, stream);
}

int vq_cache_lbg_finish(const double *sums, const int64_t *counts, const double *dist, const float *cb_old, int heads, int dim,
                        int sub, int K, float *cb_new, double *mean_dist, void *stream) {
    int rc = check_shape(heads, dim, sub, K);
    if (rc) return rc;
    if (!sums || !counts || !dist || !cb_old || !cb_new || !mean_dist) return fail(VQ_E_INVALID, "null pointer");
    hipLaunchKernelGGL(k_lbg_close, dim3(heads * (dim / sub)), dim3(256), 0, static_cast<hipStream_t>(stream), sums, counts, dist, cb_old, dim, sub,
                       K, cb_new, mean_dist);
    LAUNCH_CHECK("k_lbg_close");
    return VQ_OK;
}

}  // extern "C"
