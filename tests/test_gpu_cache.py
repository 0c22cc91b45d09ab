"""The vector-quantised key-value cache (HipEngine.cache_*, train_cache_codebooks) against its definitions in 64 bits, computed on the CPU."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}     # half a step, relative


@pytest.fixture(scope="module")
def eng():
    from vector_quantization_amd import HipEngine
    return HipEngine(DEV)


# ---- definitions ------------------------------------------------------------------------------------------------------

def codes64(x, cb, sub):
    """x (T, H, D), cb (1 or H, K, D) -> (codes (T, H, M), least squared distances): left-to-right fp64 sums, strictly less wins."""
    T, H, D = x.shape
    K = cb.shape[1]
    xs, cs = x.double().numpy().reshape(T, H, D // sub, sub), cb.double().expand(H, -1, -1).numpy().reshape(H, K, D // sub, sub)
    best = np.full((T, H, D // sub), np.inf)
    code = np.zeros((T, H, D // sub), np.int64)
    with np.errstate(all="ignore"):
        for k in range(K):
            d = np.zeros_like(best)
            for e in range(sub):
                t = xs[..., e] - cs[None, :, k, :, e]
                d = d + t * t
            less = d < best
            best[less] = d[less]
            code[less] = k
    return code, best


def vectors64(codes, cb, sub):
    """codes (n, M) of one head and its codebook (K, D) -> (n, D)."""
    K, D = cb.shape
    c = cb.double().reshape(K, -1, sub)
    return c[codes.long().clamp(max=K - 1), torch.arange(D // sub)].reshape(-1, D)


def attention64(q, k_cb, v_cb, k_codes, v_codes, table, kv_lens, starts, sub, scale):
    """(out, lse, sum of p |v|, bound on the error of a score); rows of no sequence are NaN in out."""
    rows, Hq, D = q.shape
    pages, H, page, _ = k_codes.shape
    out = torch.full((rows, Hq, D), math.nan, dtype=torch.float64)
    lse = torch.full((rows, Hq), math.nan, dtype=torch.float64)
    size = torch.zeros((rows, Hq, D), dtype=torch.float64)
    slip = torch.zeros((rows, Hq, 1), dtype=torch.float64)
    for b in range(len(kv_lens)):
        s, e = int(starts[b]), int(starts[b + 1])
        n = min(int(kv_lens[b]), table.shape[1] * page)
        j = torch.arange(n)
        p = table[b].long()[j // page]
        there = (p >= 0) & (p < pages)
        p = p.clamp(0, pages - 1)
        for h in range(H):
            kd = vectors64(k_codes[p, h, j % page], k_cb[h % k_cb.shape[0]], sub)
            vd = vectors64(v_codes[p, h, :, j % page], v_cb[h % v_cb.shape[0]], sub)
            for g in range(h * Hq // H, (h + 1) * Hq // H):
                for r in range(s, e):
                    see = there & (j <= n - (e - s) + (r - s))
                    if not see.any():
                        out[r, g], lse[r, g] = 0.0, -math.inf
                        continue
                    z = (kd[see] @ q[r, g].double()) * scale
                    w = torch.softmax(z, 0)
                    out[r, g], lse[r, g] = w @ vd[see], torch.logsumexp(z, 0)
                    size[r, g] = w @ vd[see].abs()
                    # fp32 products and sums of D terms, the score's own rounding, the base-2 argument and the exponential
                    slip[r, g] = 2.0 ** -23 * ((D + 8) * (kd[see].abs() @ q[r, g].double().abs()).max() * abs(scale) + 4 * z.abs().max() + 4)
    return out, lse, size, slip


def check_attention(got, lse, ref, n):
    out, ref_lse, size, slip = ref
    have = ~out[..., 0].isnan()
    half = HALF[got.dtype]
    got, lse = got.cpu().double(), lse.cpu().double()
    assert torch.equal(lse[have].isinf(), ref_lse[have].isinf())
    # the weights are rounded once to the cache's type and the result once; sums of n terms in fp32
    tol = half * (1 + half) * (out.abs() + size) + (2 * slip + (n + 8) * 2.0 ** -23) * size
    assert ((got - out).abs() <= tol)[have].all(), float(((got - out).abs() / tol)[have].nan_to_num().max())
    fine = have & ~ref_lse.isinf()
    tol = slip[..., 0] + (n + 8) * 2.0 ** -23 + 2.0 ** -21 * ref_lse.abs()
    assert ((lse - ref_lse).abs() <= tol)[fine].all()


def data(seed, shape, dtype):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen)
    return (x + 0.5 * x.roll(1, -1)).to(dtype)


def random_codes(seed, pages, H, page, M, K):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randint(0, K, (pages, H, page, M), generator=gen).to(torch.uint8),
            torch.randint(0, K, (pages, H, M, page), generator=gen).to(torch.uint8))


# ---- write and read -----------------------------------------------------------------------------------------------------

WRITE = [
    # tokens, heads, dim, sub, K, page, dtype
    (1, 1, 32, 2, 256, 16, torch.bfloat16), (1, 8, 128, 4, 256, 64, torch.bfloat16), (17, 3, 64, 8, 100, 16, torch.float16),
    (33, 2, 96, 4, 255, 48, torch.bfloat16), (64, 2, 128, 8, 17, 16, torch.bfloat16), (65, 1, 192, 2, 33, 32, torch.float16),
    (200, 2, 256, 4, 256, 128, torch.float16), (300, 1, 128, 4, 1, 64, torch.bfloat16), (129, 5, 64, 2, 2, 16, torch.bfloat16),
    (1000, 2, 128, 4, 256, 64, torch.bfloat16), (700, 2, 32, 8, 16, 16, torch.float16), (513, 1, 256, 8, 256, 32, torch.bfloat16),
    (140, 1, 96, 8, 31, 16, torch.bfloat16), (90, 2, 192, 8, 256, 16, torch.bfloat16), (90, 1, 96, 2, 256, 16, torch.float16),
]


@pytest.mark.parametrize("T,H,D,sub,K,page,dtype", WRITE)
def test_write_and_read(eng, T, H, D, sub, K, page, dtype):
    k, v = data(1, (T, H, D), dtype), data(2, (T, H, D), dtype)
    k_cb, v_cb = data(3, (H, K, D), dtype), data(4, (H, K, D), dtype)
    if K > 6:
        k_cb[:, K - 2] = k_cb[:, 3]                                      # equal codewords: the lower number wins
        v_cb[:, 5] = 0.0
    k[T // 2] = 0.5 * (k_cb[:, 0].float() + k_cb[:, K - 1].float()).to(dtype)  # near the middle of two codewords
    pages = -(-T // page) + 2
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(5))[:T]
    if T > 20:
        slots[3], slots[7], slots[11] = -1, pages * page, -(1 << 60)
    kc, vc = random_codes(6, pages, H, page, D // sub, 256)
    ref_k, ref_v = kc.clone(), vc.clone()
    keep = (slots >= 0) & (slots < pages * page)
    p, o = slots[keep] // page, slots[keep] % page
    ref_k[p, :, o] = torch.from_numpy(codes64(k, k_cb, sub)[0]).to(torch.uint8)[keep]
    ref_v[p, :, :, o] = torch.from_numpy(codes64(v, v_cb, sub)[0]).to(torch.uint8)[keep]
    d_kc, d_vc = kc.to(DEV), vc.to(DEV)
    args = [t.to(DEV) for t in (k, v, slots, k_cb, v_cb)]
    eng.cache_write(*args, d_kc, d_vc)
    assert torch.equal(d_kc.cpu(), ref_k)
    assert torch.equal(d_vc.cpu(), ref_v)
    got_k, got_v = eng.cache_read(args[2], args[3], args[4], d_kc, d_vc)
    for h in range(H):
        want_k = torch.zeros((T, D), dtype=torch.float64)
        want_v = torch.zeros((T, D), dtype=torch.float64)
        want_k[keep] = vectors64(ref_k[p, h, o], k_cb[h], sub)
        want_v[keep] = vectors64(ref_v[p, h, :, o], v_cb[h], sub)
        assert torch.equal(got_k[:, h].cpu().double(), want_k)
        assert torch.equal(got_v[:, h].cpu().double(), want_v)


LONG_READ = [
    (5001, 16, 32, 8, 256, 16, torch.bfloat16), (9000, 8, 64, 2, 100, 48, torch.float16), (8500, 8, 96, 8, 255, 16, torch.bfloat16),
    (8449, 8, 96, 2, 256, 64, torch.float16), (9001, 8, 128, 4, 256, 64, torch.bfloat16), (9000, 8, 192, 2, 7, 16, torch.float16),
    (8300, 8, 256, 2, 256, 16, torch.bfloat16), (20001, 8, 256, 4, 256, 128, torch.bfloat16), (5001, 16, 64, 4, 16, 32, torch.float16),
]


@pytest.mark.parametrize("T,H,D,sub,K,page,dtype", LONG_READ)
def test_long_read(eng, T, H, D, sub, K, page, dtype):
    """Reads that keep the codebook in LDS, several turns of a workgroup, the last one ragged; codes of no codeword, slots of no page, one slot twice."""
    M, pages = D // sub, -(-T // page) + 2
    kc, vc = (t.to(DEV) for t in random_codes(6, pages, H, page, M, 256))
    cbs = [data(s, (H, K, D), dtype).to(DEV) for s in (3, 4)]
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(5))[:T]
    slots[T // 2:] = slots[T // 2:].sort()[0]                            # half of them in order, as a prompt lies
    slots[3], slots[7], slots[T - 1], slots[130] = -1, pages * page, -(1 << 60), slots[129]
    slots = slots.to(DEV)
    keep = (slots >= 0) & (slots < pages * page)
    p, o = torch.where(keep, slots, 0) // page, torch.where(keep, slots, 0) % page
    h, m = torch.arange(H, device=DEV)[:, None], torch.arange(M, device=DEV)
    got = eng.cache_read(slots, *cbs, kc, vc)
    for x, codes, cb in zip(got, (kc[p, :, o], vc[p, :, :, o]), cbs):
        want = cb.reshape(H, K, M, sub)[h, codes.long().clamp(max=K - 1), m].reshape(T, H, D)
        assert torch.equal(x, torch.where(keep[:, None, None], want, 0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", ["grid", "huge", "tiny", "nonfinite", "far codeword", "bad codebook", "close", "offset"])
def test_write_hard_values(eng, dtype, case):
    """Values at which a search in less than 64 bits goes astray: exact ties, overflow, denormals, what is not finite."""
    T, H, D, sub, K = 130, 1, 64, 4, 256
    top = torch.finfo(dtype).max
    gen = torch.Generator().manual_seed(9)
    x, cb = data(7, (T, H, D), dtype), data(8, (H, K, D), dtype)
    if case == "grid":                                                   # whole numbers: ties everywhere
        x = torch.randint(-3, 4, (T, H, D), generator=gen).to(dtype)
        cb = torch.randint(-2, 3, (H, K, D), generator=gen).to(dtype)
    elif case == "huge":
        x, cb = (x.float() * (top / 16)).to(dtype), (cb.float() * (top / 16)).to(dtype)
    elif case == "tiny":
        small = torch.finfo(dtype).tiny
        x, cb = (x.float() * small / 4).to(dtype), (cb.float() * small / 4).to(dtype)
    elif case == "nonfinite":
        x[3, 0, 5], x[4, 0, 7], x[5, 0, 0] = math.nan, math.inf, -math.inf
        x[6] = math.nan
    elif case == "far codeword":
        cb[:, 7], cb[:, 9] = top, -top
    elif case == "bad codebook":
        cb[:, 0], cb[:, 5], cb[:, 9] = math.nan, math.inf, -math.inf
        cb[:, 11, 3] = math.nan
    elif case == "close":                                                # all codewords within a step or two of one point
        cb = (1.0 + torch.randint(0, 3, (H, K, D), generator=gen) * torch.finfo(dtype).eps).to(dtype)
        x = (1.0 + torch.randint(-2, 5, (T, H, D), generator=gen) * torch.finfo(dtype).eps).to(dtype)
    elif case == "offset":                                               # far from the origin against their spread
        x, cb = (x.float() + 200).to(dtype), (cb.float() + 200).to(dtype)
    kc, vc = eng.cache_buffers(9, 16, H, D, sub)
    slots = torch.arange(T, device=DEV)
    eng.cache_write(x.to(DEV), x.flip(0).to(DEV), slots, cb.to(DEV), cb.flip(1).to(DEV), kc, vc)
    assert torch.equal(kc.cpu().transpose(1, 2).reshape(144, H, D // sub)[:T].long(), torch.from_numpy(codes64(x, cb, sub)[0]))
    assert torch.equal(vc.cpu().permute(0, 3, 1, 2).reshape(144, H, D // sub)[:T].long(), torch.from_numpy(codes64(x.flip(0), cb.flip(1), sub)[0]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [1, 7, 100, 255])
def test_large_vectors_keep_to_the_codewords_there_are(eng, K, dtype):
    """Vectors of numbers near 1e18, and far larger and smaller ones, beside a codebook that does not fill its tile."""
    T, H, D, sub = 96, 1, 32, 4
    x = (data(7, (T, H, D), torch.float32) * (10.0 ** torch.arange(10, 34).repeat_interleave(4)).reshape(T, 1, 1)).to(dtype)
    x[32:36] = torch.tensor([1e18, -1e18, 0.9e18, 1.1e18]).to(dtype).reshape(4, 1, 1)
    cb = torch.zeros((H, K, D)) if K == 1 else data(8, (H, K, D), torch.float32)
    code = torch.from_numpy(codes64(x, cb.to(dtype), sub)[0])
    if dtype != torch.float32:
        kc, vc = eng.cache_buffers(6, 16, H, D, sub)
        eng.cache_write(x.to(DEV), x.to(DEV), torch.arange(T, device=DEV), cb.to(dtype).to(DEV), cb.to(dtype).to(DEV), kc, vc)
        assert torch.equal(kc.cpu().transpose(1, 2).reshape(T, H, D // sub).long(), code)
        assert torch.equal(vc.cpu().permute(0, 3, 1, 2).reshape(T, H, D // sub).long(), code)
    code = torch.from_numpy(codes64(x, cb, sub)[0])
    counted = (x.double().abs() < 2.0 ** 100).reshape(T, H, -1, sub).all(-1)
    assert not counted.all() and counted.any()
    _, counts, dist = eng.cache_lbg_accum(x.to(DEV), cb.to(DEV), sub)
    for m in range(D // sub):
        assert torch.equal(counts[0, m].cpu(), torch.bincount(code[:, 0, m][counted[:, 0, m]], minlength=K))
    assert dist.isfinite().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [1, 40, 100])
def test_products_beyond_fp32(eng, K, dtype):
    """Vectors and codewords of 1e20, whose products fp32 does not hold."""
    T, H, D, sub = 70, 2, 32, 8
    x, cb = data(7, (T, H, D), torch.float32).mul(1e20).to(dtype), data(8, (H, K, D), torch.float32) * 1e20
    if dtype != torch.float32:
        half = cb.to(dtype)
        kc, vc = eng.cache_buffers(5, 16, H, D, sub)
        eng.cache_write(x.to(DEV), x.to(DEV), torch.arange(T, device=DEV), half.to(DEV), half.to(DEV), kc, vc)
        assert torch.equal(kc.cpu().transpose(1, 2).reshape(80, H, D // sub)[:T].long(), torch.from_numpy(codes64(x, half, sub)[0]))
    sums, counts, dist = eng.cache_lbg_accum(x.to(DEV), cb.to(DEV), sub)
    new, mean = eng.cache_lbg_finish(sums, counts, dist, cb.to(DEV))
    check_training(x, cb, sub, sums, counts, dist, new, mean)


def test_write_strides_and_shared_codebook(eng):
    """Keys and values inside one larger tensor, copies where their vectors do not start at multiples of 16 bytes, one codebook for all heads."""
    T, H, D, sub, K, page = 77, 4, 64, 4, 256, 16
    qkv = data(1, (T, 3 * H, D), torch.bfloat16).to(DEV)
    cb = data(3, (1, K, D), torch.bfloat16).to(DEV)
    k, v = qkv[:, H:2 * H], qkv[:, 2 * H:]
    slots = torch.arange(T, device=DEV)
    kc, vc = eng.cache_buffers(5, page, H, D, sub)
    eng.cache_write(k, v, slots, cb, cb, kc, vc)
    want = torch.from_numpy(codes64(k.cpu(), cb.cpu(), sub)[0])
    assert torch.equal(kc.cpu().transpose(1, 2).reshape(-1, H, D // sub)[:T].long(), want)
    odd = torch.zeros((T, H, D + 1), dtype=torch.bfloat16, device=DEV)
    odd[..., 1:] = k
    turned = v.permute(2, 1, 0).contiguous().permute(2, 1, 0)
    kc2, vc2 = eng.cache_buffers(5, page, H, D, sub)
    eng.cache_write(odd[..., 1:], turned, slots, cb, cb, kc2, vc2)
    assert torch.equal(kc, kc2) and torch.equal(vc, vc2)
    got_k, got_v = eng.cache_read(slots[::2], cb, cb, kc, vc)                       # a strided list of slots
    assert torch.equal(got_k.cpu().double(), torch.stack([vectors64(want[::2, h], cb[0].cpu(), sub) for h in range(H)], 1))
    one = k[:1].expand(T, H, D)                                                     # a broadcast input
    eng.cache_write(one, one, slots, cb, cb, kc2, vc2)
    assert (kc2.transpose(1, 2).reshape(-1, H, D // sub)[:T] == kc[0, :, 0]).all()


def test_write_same_slot_twice(eng):
    """Each code of a slot that two tokens name is that of either; nothing else is touched."""
    T, H, D, sub, K = 40, 2, 64, 4, 64
    k = data(1, (T, H, D), torch.bfloat16)
    cb = data(3, (H, K, D), torch.bfloat16)
    kc, vc = eng.cache_buffers(2, 16, H, D, sub)
    eng.cache_write(k.to(DEV), k.to(DEV), torch.full((T,), 5, device=DEV), cb.to(DEV), cb.to(DEV), kc, vc)
    want = torch.from_numpy(codes64(k, cb, sub)[0])
    assert (want == kc.cpu()[0, :, 5].long()).any(0).all() and (want == vc.cpu()[0, :, :, 5].long()).any(0).all()
    kc[0, :, 5], vc[0, :, :, 5] = 0, 0
    assert not kc.any() and not vc.any()


# ---- attention ----------------------------------------------------------------------------------------------------------

ATTEND = [
    # new tokens, lengths, q_heads, heads, dim, sub, K, page, dtype
    ([1], [1], 1, 1, 32, 2, 256, 16, torch.bfloat16),
    ([1], [33], 8, 2, 128, 4, 256, 64, torch.bfloat16),
    ([1, 1, 1, 1], [500, 1, 17, 256], 8, 8, 128, 4, 256, 16, torch.bfloat16),
    ([1, 1], [2000, 700], 16, 1, 64, 8, 200, 32, torch.float16),
    ([1, 1], [300, 90], 40, 2, 128, 8, 256, 16, torch.bfloat16),
    ([5, 0, 3, 2, 17], [5, 40, 100, 0, 29], 6, 2, 64, 4, 256, 16, torch.float16),
    ([4, 9], [2, 3], 4, 4, 64, 2, 256, 16, torch.bfloat16),             # more new tokens than there are: rows that see nothing
    ([70], [70], 4, 2, 96, 4, 100, 48, torch.bfloat16),
    ([33, 80], [450, 81], 14, 2, 128, 2, 256, 128, torch.float16),
    ([40], [300], 3, 3, 192, 4, 256, 16, torch.bfloat16),
    ([20, 1], [130, 64], 8, 2, 256, 8, 256, 32, torch.bfloat16),
    ([20, 1], [130, 64], 8, 2, 256, 4, 128, 32, torch.float16),
    ([1, 3], [130, 64], 5, 1, 96, 8, 3, 16, torch.bfloat16),
    ([130], [600], 2, 1, 32, 8, 16, 16, torch.float16),
    ([200], [201], 8, 1, 64, 2, 256, 16, torch.bfloat16),
    ([2, 50], [700, 333], 4, 2, 192, 2, 40, 64, torch.float16),
]


def attention_case(n_q, n_kv, Hq, H, D, sub, K, page, dtype, seed=0, spare_rows=0):
    B, width = len(n_q), max(1, -(-max(n_kv) // page))
    pages = sum(-(-n // page) for n in n_kv) + 2
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    table = torch.full((B, width), -7, dtype=torch.int32)
    at = 0
    for b, n in enumerate(n_kv):
        use = -(-n // page)
        table[b, :use] = order[at:at + use]
        at += use
    q = data(seed + 1, (sum(n_q) + spare_rows, Hq, D), dtype)
    k_cb, v_cb = data(seed + 2, (H, K, D), dtype), data(seed + 3, (H, K, D), dtype)
    kc, vc = random_codes(seed + 4, pages, H, page, D // sub, K)
    starts = torch.tensor([0] + list(np.cumsum(n_q)), dtype=torch.int32)
    return q, k_cb, v_cb, kc, vc, table, torch.tensor(n_kv, dtype=torch.int32), starts


@pytest.mark.parametrize("n_q,n_kv,Hq,H,D,sub,K,page,dtype", ATTEND)
def test_attention(eng, n_q, n_kv, Hq, H, D, sub, K, page, dtype):
    case = attention_case(n_q, n_kv, Hq, H, D, sub, K, page, dtype)
    out, lse = eng.cache_attention(*[t.to(DEV) for t in case], max(n_q), max_kv=max(1, max(n_kv)), want_lse=True)
    ref = attention64(*case, sub, 1.0 / math.sqrt(D))
    check_attention(out, lse, ref, max(n_kv))


def test_attention_peaked_and_large_scores(eng):
    """Scores of several hundred, one token that holds nearly all the weight, a scale of one's own, a negative one."""
    args = ([1, 30], [300, 140], 4, 2, 64, 4, 256, 16, torch.bfloat16)
    for scale in (4.0, -3.0, 0.0):
        case = list(attention_case(*args, seed=20))
        case[0] = case[0] * 8
        out, lse = eng.cache_attention(*[t.to(DEV) for t in case], 30, scale=scale, want_lse=True)
        check_attention(out, lse, attention64(*case, 4, scale), 300)


@pytest.mark.parametrize("n_q,n_kv", [([1, 1], [40, 700]), ([30, 3], [300, 60])])
def test_attention_nan_stays_in_its_row(eng, n_q, n_kv):
    """A query that is no number gives a row and a logarithm that are none, and leaves the rows beside it as they are."""
    case = list(attention_case(n_q, n_kv, 4, 2, 64, 4, 256, 16, torch.bfloat16, seed=25))
    clean = eng.cache_attention(*[t.to(DEV) for t in case], max(n_q), want_lse=True)
    case[0][1, 2, 5] = math.nan
    out, lse = eng.cache_attention(*[t.to(DEV) for t in case], max(n_q), want_lse=True)
    bad = torch.zeros((sum(n_q), 4), dtype=torch.bool, device=DEV)
    bad[1, 2] = True
    assert out[bad].isnan().all() and torch.equal(lse.isnan(), bad)
    check_attention(out[~bad], lse[~bad], [t.reshape(bad.shape + t.shape[2:])[~bad.cpu()] for t in attention64(*case, 4, 0.125)], max(n_kv))
    assert clean[0].isfinite().all()


def test_attention_rows_of_no_sequence_bad_pages_and_codes(eng):
    """Rows behind the last sequence stay; pages outside the cache are not seen; what lies behind a sequence's end (codes of no codeword,
    page numbers of no page) does not matter; lengths past the table are cut to it."""
    for n_q, n_kv in (([3, 1], [100, 40]), ([1, 1], [100, 40]), ([40, 2], [100, 40])):
        q, k_cb, v_cb, kc, vc, table, kv_lens, starts = attention_case(n_q, n_kv, 4, 2, 64, 4, 100, 16, torch.bfloat16, seed=30, spare_rows=9)
        table[0, 2], table[1, 1] = 1 << 30, -5
        last = int(table[0, 6])
        kc[last, :, 4:], vc[last, :, :, 4:] = 255, 254                    # tokens 100 on
        q[sum(n_q):] = math.nan
        spare = torch.full_like(q, 7.0).to(DEV)
        case = (q, k_cb, v_cb, kc, vc, table, kv_lens, starts)
        out, lse = eng.cache_attention(*[t.to(DEV) for t in case], max(n_q), out=spare, want_lse=True)
        assert out is spare and (out[sum(n_q):] == 7.0).all()
        check_attention(out, lse, attention64(*case, 4, 0.125), 100)
        far = kv_lens.clone()
        far[0] = 2 ** 31 - 1                                              # cut to the 112 tokens of the table
        kc[last, :, 4:], vc[last, :, :, 4:] = 1, 2
        case = (q, k_cb, v_cb, kc, vc, table, far, starts)
        out, lse = eng.cache_attention(*[t.to(DEV) for t in case], max(n_q), want_lse=True)
        check_attention(out, lse, attention64(*case, 4, 0.125), 112)


def test_attention_starts_out_of_order_stay_in_bounds(eng):
    """Starts that break their rule give rows of some sequence or none, and nothing is written outside the rows."""
    q, k_cb, v_cb, kc, vc, table, kv_lens, starts = attention_case([3, 4], [50, 60], 4, 2, 64, 4, 256, 16, torch.bfloat16, seed=40)
    for bad in ([-5, 3, 900], [3, 0, 7], [7, 7, 7], [0, 0, 0], [2 ** 31 - 1, 0, -2 ** 31]):
        starts = torch.tensor(bad, dtype=torch.int32)
        whole = torch.full((27, 4, 64), 3.0, dtype=torch.bfloat16, device=DEV)
        eng.cache_attention(*[t.to(DEV) for t in (q, k_cb, v_cb, kc, vc, table, kv_lens, starts)], 4, out=whole[10:17])
        assert (whole[:10] == 3.0).all() and (whole[17:] == 3.0).all() and whole.isfinite().all()


@pytest.mark.parametrize("max_q,max_kv", [(1, 1), (1, 100000), (5000, 1), (64, None)])
def test_attention_hints_do_not_change_results(eng, max_q, max_kv):
    args = ([1, 64, 3], [900, 333, 20], 8, 2, 128, 4, 256, 16, torch.bfloat16)
    case = attention_case(*args, seed=50)
    out, lse = eng.cache_attention(*[t.to(DEV) for t in case], max_q, max_kv=max_kv, want_lse=True)
    check_attention(out, lse, attention64(*case, 4, 1.0 / math.sqrt(128)), 900)


@pytest.mark.parametrize("max_q,max_kv", [(5, 200), (5, 100000), (1, 1), (5, 1600)])
@pytest.mark.parametrize("seqs,H", [(64, 8), (65, 2), (150, 1), (200, 8)])
def test_attention_many_sequences(eng, seqs, H, max_q, max_kv):
    """More sequences than a wave has lanes, some of no rows or no tokens, cut and uncut."""
    gen = torch.Generator().manual_seed(seqs)
    n_q, n_kv = (torch.randint(0, top, (seqs,), generator=gen).tolist() for top in (6, 201))
    n_q[0], n_q[-1], n_kv[-1] = 5, 1, 200
    case = attention_case(n_q, n_kv, 2 * H, H, 32, 8, 16, 16, torch.bfloat16, seed=seqs)
    out, lse = eng.cache_attention(*[t.to(DEV) for t in case], max_q, max_kv=max_kv, want_lse=True)
    check_attention(out, lse, attention64(*case, 8, 32 ** -0.5), max(n_kv))


@pytest.mark.parametrize("dtype,D,sub", [(torch.bfloat16, 32, 8), (torch.float16, 64, 4)])
def test_attention_many_row_tiles(eng, dtype, D, sub):
    """A sequence of more tiles of rows than a wave has lanes, between short ones."""
    case = attention_case([3, 1100, 0, 2], [90, 1250, 7, 400], 2, 1, D, sub, 64, 32, dtype, seed=77)
    out, lse = eng.cache_attention(*[t.to(DEV) for t in case], 1100, want_lse=True)
    check_attention(out, lse, attention64(*case, sub, D ** -0.5), 1250)


def test_attention_strided_q_shared_codebook_repeatable(eng):
    args = ([1, 20], [200, 95], 8, 4, 64, 4, 256, 16, torch.float16)
    q, k_cb, v_cb, *rest = attention_case(*args, seed=60)
    k_cb, v_cb = k_cb[:1].contiguous(), v_cb[:1].contiguous()
    wide = data(61, (21, 16, 64), torch.float16).to(DEV)
    rest_d = [t.to(DEV) for t in rest]
    out, lse = eng.cache_attention(wide[:, 4:12], k_cb.to(DEV), v_cb.to(DEV), *rest_d, 20, want_lse=True)
    check_attention(out, lse, attention64(wide[:, 4:12].cpu(), k_cb, v_cb, *rest, 4, 0.125), 200)
    again, lse2 = eng.cache_attention(wide[:, 4:12], k_cb.to(DEV), v_cb.to(DEV), *rest_d, 20, want_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    turned = wide[:, 4:12].permute(2, 0, 1).contiguous().permute(1, 2, 0)
    assert torch.equal(out, eng.cache_attention(turned, k_cb.to(DEV), v_cb.to(DEV), *rest_d, 20))


def test_attention_parts_join_by_lse(eng):
    """Attention over the two halves of a context, joined by their logarithms, is that over the whole."""
    q, k_cb, v_cb, kc, vc, table, kv_lens, starts = attention_case([1], [512], 4, 2, 64, 4, 256, 16, torch.bfloat16, seed=70)
    dev = [t.to(DEV) for t in (q, k_cb, v_cb, kc, vc)]
    s = starts.to(DEV)
    parts = []
    for cols in (table[:, :16], table[:, 16:]):
        o, l = eng.cache_attention(*dev, cols.contiguous().to(DEV), torch.tensor([256], dtype=torch.int32, device=DEV), s, 1, want_lse=True)
        parts.append((o.double(), l.double()))
    w = torch.softmax(torch.stack([l for _, l in parts]), 0)[..., None]
    joined = w[0] * parts[0][0] + w[1] * parts[1][0]
    ref, _, size, _ = attention64(q, k_cb, v_cb, kc, vc, table, kv_lens, starts, 4, 0.125)
    # each part carries its own two roundings, of weights and of the result
    assert ((joined.cpu() - ref).abs() <= 2.0 ** -8 * 2.1 * size).all()


def test_offsets_past_32_bits(eng):
    """A cache of more than 2^32 bytes of codes: the last pages are written, read and attended to."""
    H, D, sub, K, page = 8, 64, 2, 16, 1024
    pages = (1 << 32) // (H * page * (D // sub)) + 9
    kc = torch.zeros((pages, H, page, D // sub), dtype=torch.uint8, device=DEV)
    vc = torch.zeros((pages, H, D // sub, page), dtype=torch.uint8, device=DEV)
    T = 100
    k, v = data(1, (T, H, D), torch.bfloat16), data(2, (T, H, D), torch.bfloat16)
    cb = data(3, (H, K, D), torch.bfloat16)
    slots = torch.arange(T) + (pages - 1) * page + 20
    table = torch.tensor([[pages - 1]], dtype=torch.int32)
    eng.cache_write(k.to(DEV), v.to(DEV), slots.to(DEV), cb.to(DEV), cb.to(DEV), kc, vc)
    last_k, last_v = kc[-1:].cpu(), vc[-1:].cpu()
    assert torch.equal(last_k[0, :, 20:120].transpose(0, 1).long(), torch.from_numpy(codes64(k, cb, sub)[0]))
    assert torch.equal(last_v[0, :, :, 20:120].permute(2, 0, 1).long(), torch.from_numpy(codes64(v, cb, sub)[0]))
    got_k, _ = eng.cache_read(slots.to(DEV), cb.to(DEV), cb.to(DEV), kc, vc)
    assert torch.equal(got_k[:, 1].cpu().double(), vectors64(last_k[0, 1, 20:120], cb[1], sub))
    q = data(4, (2, H, D), torch.bfloat16)
    n_kv, starts = torch.tensor([121], dtype=torch.int32), torch.tensor([0, 2], dtype=torch.int32)
    out, lse = eng.cache_attention(q.to(DEV), cb.to(DEV), cb.to(DEV), kc, vc, table.to(DEV), n_kv.to(DEV), starts.to(DEV), 2, want_lse=True)
    check_attention(out, lse, attention64(q, cb, cb, last_k, last_v, torch.zeros_like(table), n_kv, starts, sub, 0.125), 121)
    del kc, vc
    torch.cuda.empty_cache()


# ---- training -----------------------------------------------------------------------------------------------------------

TRAIN = [
    # tokens, heads, dim, sub, K, dtype
    (1, 1, 32, 2, 256, torch.bfloat16), (31, 2, 64, 4, 16, torch.float32), (33, 1, 128, 8, 256, torch.bfloat16), (500, 3, 64, 4, 100, torch.float16),
    (700, 1, 96, 2, 33, torch.float32), (257, 2, 192, 8, 256, torch.float32), (2500, 1, 32, 4, 256, torch.bfloat16), (900, 2, 256, 8, 7, torch.float16),
    (5000, 1, 32, 8, 256, torch.float32), (300, 2, 96, 8, 256, torch.bfloat16), (30000, 1, 32, 8, 100, torch.float16), (20000, 1, 32, 2, 9, torch.float32), (300, 1, 96, 4, 1, torch.bfloat16), (4097, 1, 64, 2, 200, torch.float16),
]


def check_training(x, cb, sub, sums, counts, dist, new, mean):
    """Everything one iteration gives against 64 bits."""
    T, H, D = x.shape
    K = cb.shape[1]
    fine = x.double().reshape(T, H, D // sub, sub).isfinite().all(-1)
    code, least = codes64(x, cb, sub)
    code, least = torch.from_numpy(code), torch.from_numpy(least)
    for h in range(H):
        for m in range(D // sub):
            ok = fine[:, h, m]
            xs = x[ok, h, m * sub:(m + 1) * sub].double()
            c = code[ok, h, m]
            n = torch.bincount(c, minlength=K)
            assert torch.equal(counts[h, m].cpu(), n)
            want = torch.zeros((K, sub), dtype=torch.float64).index_add_(0, c, xs)
            size = torch.zeros((K, sub), dtype=torch.float64).index_add_(0, c, xs.abs())
            part = slice(m * sub, (m + 1) * sub)
            # partial sums of at most 4096 vectors in fp32, 32 of them in each step of the accumulation, joined in fp64
            tol = (4096 / 32 + 32) * 2.0 ** -23 * size
            assert bool(((sums[h, :, part].cpu() - want).abs() <= tol).all())
            centre = torch.where(n[:, None] > 0, want / n.clamp(min=1)[:, None], cb[h, :, part].double())
            # the division's result is rounded to fp32: half a step relative, or half of 2^-149 below 2^-126, where steps no longer shrink
            off = (new[h, :, part].cpu().double() - centre).abs()
            assert bool((off <= tol / n.clamp(min=1)[:, None] + 2.0 ** -24 * 1.001 * centre.abs() + 2.0 ** -150).all())
            far = least[ok, h, m]
            assert abs(float(dist[h, m]) - float(far.sum())) <= 1e-12 * float(far.sum())
            assert abs(float(mean[h, m]) - float(far.sum()) / max(1, int(ok.sum()))) <= 2e-12 * float(far.sum()) / max(1, int(ok.sum()))


@pytest.mark.parametrize("T,H,D,sub,K,dtype", TRAIN)
def test_training_iteration(eng, T, H, D, sub, K, dtype):
    x, cb = data(1, (T, H, D), dtype), data(2, (H, K, D), torch.float32)
    if K > 6:
        cb[:, K - 2] = cb[:, 3]
        cb[:, 4] = 1e6                                                   # without members
    sums, counts, dist = eng.cache_lbg_accum(x.to(DEV), cb.to(DEV), sub)
    new, mean = eng.cache_lbg_finish(sums, counts, dist, cb.to(DEV))
    check_training(x, cb, sub, sums, counts, dist, new, mean)
    if K > 6:
        assert torch.equal(new[:, 4].cpu(), cb[:, 4])
    new2, counts2, mean2 = eng.cache_lbg_iterate(x.to(DEV), cb.to(DEV), sub)
    assert torch.equal(new, new2) and torch.equal(counts, counts2) and torch.equal(mean, mean2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", ["grid", "nonfinite", "huge", "tiny", "close", "offset", "all bad"])
def test_training_hard_values(eng, dtype, case):
    T, H, D, sub, K = 200, 1, 64, 4, 64
    gen = torch.Generator().manual_seed(9)
    x, cb = data(7, (T, H, D), dtype), data(8, (H, K, D), torch.float32)
    if case == "grid":
        x = torch.randint(-3, 4, (T, H, D), generator=gen).to(dtype)
        cb = torch.randint(-2, 3, (H, K, D), generator=gen).float()
    elif case == "nonfinite":
        x[3, 0, 5], x[4, 0, 7], x[5, 0, 0] = math.nan, math.inf, -math.inf
        cb[:, 9], cb[:, 3, 2] = math.inf, math.nan
    elif case == "all bad":
        x[:] = math.nan
    elif case == "huge":
        size = 2.0 ** 90 if dtype != torch.float16 else 8000.0
        x, cb = (x.float() * size).to(dtype), cb * size
    elif case == "tiny":
        x, cb = (x.float() * 2.0 ** (-130 if dtype != torch.float16 else -20)).to(dtype), cb * 2.0 ** (-130 if dtype != torch.float16 else -20)
    elif case == "close":
        cb = 1.0 + torch.randint(0, 3, (H, K, D), generator=gen) * 2.0 ** -23
        x = (1.0 + torch.randint(-2, 5, (T, H, D), generator=gen) * torch.finfo(dtype).eps).to(dtype)
    elif case == "offset":
        x, cb = (x.float() + 200).to(dtype), cb + 200
    sums, counts, dist = eng.cache_lbg_accum(x.to(DEV), cb.to(DEV), sub)
    new, mean = eng.cache_lbg_finish(sums, counts, dist, cb.to(DEV))
    cb_ref = torch.where(cb.isnan(), cb, cb)
    if case == "nonfinite":
        assert torch.equal(new[:, 9].cpu(), cb[:, 9])                    # no member: stays, infinite
        new, cb_ref = new.clone(), cb_ref.clone()
        keep = cb.isfinite()
        new[~keep.to(DEV)] = 0.0
        sums_ref_cb = cb_ref.clone()
        code, _ = codes64(x, sums_ref_cb, sub)
        fine = x.double().reshape(T, H, D // sub, sub).isfinite().all(-1)
        for m in range(D // sub):
            c = torch.from_numpy(code[:, 0, m])[fine[:, 0, m]]
            assert torch.equal(counts[0, m].cpu(), torch.bincount(c, minlength=K))
        return
    check_training(x, cb_ref, sub, sums, counts, dist, new, mean)


def test_training_strides(eng):
    wide = data(1, (300, 6, 64), torch.bfloat16).to(DEV)
    cb = data(2, (2, 32, 64), torch.float32)
    x = wide[:, 2:4]
    sums, counts, dist = eng.cache_lbg_accum(x, cb.to(DEV), 4)
    new, mean = eng.cache_lbg_finish(sums, counts, dist, cb.to(DEV))
    check_training(x.cpu(), cb, 4, sums, counts, dist, new, mean)
    odd = torch.zeros((300, 2, 65), dtype=torch.bfloat16, device=DEV)
    odd[..., 1:] = x
    again = eng.cache_lbg_accum(odd[..., 1:], cb.to(DEV), 4)
    assert all(torch.equal(a, b) for a, b in zip(again, (sums, counts, dist)))
    none = eng.cache_lbg_accum(x[:0], cb.to(DEV), 4)
    assert not any(t.any() for t in none)
    half = [eng.cache_lbg_accum(part, cb.to(DEV), 4) for part in (x[:111], x[111:])]     # shards' results add up
    assert torch.equal(half[0][1] + half[1][1], counts)
    assert (half[0][0] + half[1][0] - sums).abs().max() <= 1e-3


def test_train_codebooks(eng):
    """Eight tight clouds a part are found; the distortion of each stage falls; k that is no power of two is rounded up."""
    from vector_quantization_amd import train_cache_codebooks
    gen = torch.Generator().manual_seed(3)
    T, H, D, sub = 4000, 2, 32, 4
    centres = torch.randn((H, 8, D), generator=gen) * 4
    pick = torch.randint(0, 8, (T, H, D // sub), generator=gen)
    x = torch.stack([centres[h].reshape(8, D // sub, sub)[pick[:, h], torch.arange(D // sub)].reshape(T, D) for h in range(H)], 1)
    x = (x + 0.01 * torch.randn(x.shape, generator=gen)).to(torch.bfloat16).to(DEV)
    res = train_cache_codebooks(eng, x, 7, sub, log=None)
    assert res.codebook.shape == (H, 8, D) and res.codebook.isfinite().all() and len(res.iters_per_stage) == 3
    ends = np.cumsum(res.iters_per_stage) - 1
    assert res.distortions[ends[0]] > res.distortions[ends[1]] > res.distortions[ends[2]]
    assert train_cache_codebooks(eng, x[:1], 1, sub, log=None).codebook.shape == (H, 1, D)
    with pytest.raises(ValueError, match="cannot exceed"):
        train_cache_codebooks(eng, x[:4], 8, sub, log=None)


# ---- together, on streams and in graphs -----------------------------------------------------------------------------------

def serving_state(eng, dtype=torch.bfloat16):
    from vector_quantization_amd import train_cache_codebooks
    H, D, sub, K, page = 2, 64, 4, 64, 16
    sample = data(1, (2000, H, D), dtype).to(DEV)
    k_cb = train_cache_codebooks(eng, sample, K, sub, log=None, max_iterations=10).codebook.to(dtype)
    v_cb = train_cache_codebooks(eng, sample.flip(0).contiguous(), K, sub, log=None, max_iterations=10).codebook.to(dtype)
    kc, vc = eng.cache_buffers(40, page, H, D, sub)
    return H, D, sub, page, k_cb, v_cb, kc, vc


def test_prompt_then_steps(eng):
    """Trained codebooks; two prompts written and attended to, then single tokens, against attention over the vectors read back."""
    H, D, sub, page, k_cb, v_cb, kc, vc = serving_state(eng)
    Hq, lens = 6, [100, 37]
    table = torch.randperm(40, generator=torch.Generator().manual_seed(5))[:20].reshape(2, 10).to(torch.int32).to(DEV)

    def slots(b, first, n):
        j = torch.arange(first, first + n, device=DEV)
        return table[b].long()[j // page] * page + j % page

    def step(n_q, seed):
        rows = sum(n_q)
        k, v, q = (data(seed + i, (rows, h, D), torch.bfloat16).to(DEV) for i, h in enumerate((H, H, Hq)))
        s = torch.cat([slots(b, lens[b] - n, n) for b, n in enumerate(n_q)])
        eng.cache_write(k, v, s, k_cb, v_cb, kc, vc)
        starts = torch.tensor([0] + list(np.cumsum(n_q)), dtype=torch.int32, device=DEV)
        kv = torch.tensor(lens, dtype=torch.int32, device=DEV)
        out, lse = eng.cache_attention(q, k_cb, v_cb, kc, vc, table, kv, starts, max(n_q), want_lse=True)
        for b, n in enumerate(n_q):
            kd, vd = (t.cpu().double() for t in eng.cache_read(slots(b, 0, lens[b]), k_cb, v_cb, kc, vc))
            r0 = int(starts[b])
            for g in range(Hq):
                z = q[r0:r0 + n, g].cpu().double() @ kd[:, g // 3].T / 8.0
                z = z.masked_fill(torch.arange(lens[b]) > lens[b] - n + torch.arange(n)[:, None], -math.inf)
                ref = torch.softmax(z, 1) @ vd[:, g // 3]
                size = torch.softmax(z, 1) @ vd[:, g // 3].abs()
                assert ((out[r0:r0 + n, g].cpu().double() - ref).abs() <= 2.0 ** -8 * (ref.abs() + 1.1 * size)).all()
                assert ((lse[r0:r0 + n, g].cpu().double() - torch.logsumexp(z, 1)).abs() <= 1e-4).all()

    step(lens, 10)
    for i in range(3):
        lens[0] += 1
        lens[1] += 1
        step([1, 1], 20 + 3 * i)


def test_other_stream_and_current_device_stream(eng):
    """Calls go to the current stream, behind what is on it."""
    H, D, sub, page, k_cb, v_cb, kc, vc = serving_state(eng)
    x = data(3, (600, H, D), torch.bfloat16)
    side = torch.cuda.Stream()
    slots = torch.arange(600, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        a = torch.zeros((4096, 4096), device=DEV)
        for _ in range(20):
            a = a @ a                                                    # keeps the stream busy
        k = x.to(DEV, non_blocking=True) + a[0, 0].to(torch.bfloat16)
        eng.cache_write(k, k, slots, k_cb, v_cb, kc, vc)
        got, _ = eng.cache_read(slots, k_cb, v_cb, kc, vc)
    side.synchronize()
    code = torch.from_numpy(codes64(x, k_cb.cpu(), sub)[0])
    assert torch.equal(got[:, 0].cpu().double(), vectors64(code[:, 0], k_cb[0].cpu(), sub))


def test_graphs(eng):
    """A serving step and a training iteration captured into two graphs, replayed in turn with eager work between, new inputs and lengths each time."""
    H, D, sub, page, k_cb, v_cb, kc, vc = serving_state(eng)
    Hq = 8
    table = torch.arange(40, dtype=torch.int32, device=DEV).reshape(2, 20)
    k, v, q = (torch.zeros((2, h, D), dtype=torch.bfloat16, device=DEV) for h in (H, H, Hq))
    slots = torch.zeros(2, dtype=torch.int64, device=DEV)
    kv = torch.ones(2, dtype=torch.int32, device=DEV)
    starts = torch.arange(3, dtype=torch.int32, device=DEV)
    x = torch.zeros((900, H, D), dtype=torch.bfloat16, device=DEV)
    cb = k_cb.float()

    def serve():
        eng.cache_write(k, v, slots, k_cb, v_cb, kc, vc)
        return eng.cache_attention(q, k_cb, v_cb, kc, vc, table, kv, starts, 1, want_lse=True)

    def train():
        return eng.cache_lbg_iterate(x, cb, sub)

    graphs = []
    for fn in (serve, train):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            fn()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = fn()
        graphs.append((g, out))
    first = [data(100 + i, (318, H, D), torch.bfloat16).to(DEV) for i in range(2)]
    for b in range(2):
        eng.cache_write(first[b], first[b], table[b].long().repeat_interleave(page)[:318] * page + torch.arange(318, device=DEV) % page,
                        k_cb, v_cb, kc, vc)
    for i, lens in enumerate(([300, 17], [301, 18], [40, 319], [1, 1])):
        k.copy_(data(10 * i, (2, H, D), torch.bfloat16))
        v.copy_(data(10 * i + 1, (2, H, D), torch.bfloat16))
        q.copy_(data(10 * i + 2, (2, Hq, D), torch.bfloat16))
        x.copy_(data(10 * i + 3, (900, H, D), torch.bfloat16))
        kv.copy_(torch.tensor(lens, dtype=torch.int32))
        slots.copy_(torch.tensor([int(table[b, (n - 1) // page]) * page + (n - 1) % page for b, n in enumerate(lens)]))
        graphs[0][0].replay()
        graphs[1][0].replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in graphs[0][1]] + [t.clone() for t in graphs[1][1]]
        codes = kc.clone(), vc.clone()
        want = list(serve()) + list(train())
        assert torch.equal(codes[0], kc) and torch.equal(codes[1], vc)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_empty_calls(eng):
    H, D, sub, page, k_cb, v_cb, kc, vc = serving_state(eng)
    none = torch.zeros((0, H, D), dtype=torch.bfloat16, device=DEV)
    before = kc.clone()
    eng.cache_write(none, none, torch.zeros(0, dtype=torch.int64, device=DEV), k_cb, v_cb, kc, vc)
    assert torch.equal(kc, before)
    got = eng.cache_read(torch.zeros(0, dtype=torch.int64, device=DEV), k_cb, v_cb, kc, vc)
    assert got[0].shape == (0, H, D)
    z = torch.zeros(0, dtype=torch.int32, device=DEV)
    out, lse = eng.cache_attention(none, k_cb, v_cb, kc, vc, torch.zeros((0, 4), dtype=torch.int32, device=DEV), z,
                                   torch.zeros(1, dtype=torch.int32, device=DEV), 1, want_lse=True)
    assert out.shape == (0, H, D) and lse.shape == (0, H)
    q = torch.ones((3, H, D), dtype=torch.bfloat16, device=DEV)               # a table of no pages: no token is seen
    out, lse = eng.cache_attention(q, k_cb, v_cb, kc, vc, torch.zeros((1, 0), dtype=torch.int32, device=DEV),
                                   torch.tensor([50], dtype=torch.int32, device=DEV), torch.tensor([0, 3], dtype=torch.int32, device=DEV), 3, want_lse=True)
    assert not out.any() and (lse == -math.inf).all()
