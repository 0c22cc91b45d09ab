"""Values and shapes at which the cache operators (HipEngine.cache_*) could go astray, each for itself, against their definitions in 64 bits."""
import math

import numpy as np
import pytest
import torch

from test_gpu_cache import DEV, HALF, attention64, attention_case, check_attention, check_training, codes64, data, vectors64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    from vector_quantization_amd import HipEngine
    return HipEngine(DEV)


# ---- attention ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,hint", [(1, 1), (1, None), (20, 1)])
@pytest.mark.parametrize("where", ["first", "last", "by turns"])
@pytest.mark.parametrize("nats", [17.5, 19.0, 24.0, 26.0])
def test_attention_where_one_token_takes_all_and_gives_nothing(eng, dtype, rows, hint, where, nats):
    """Tokens whose values are zero hold all but e^-nats of the weight, so the result is what the others add: their weights may not vanish.
    A hint of one token leaves all the work to one workgroup, in which one wave meets the heavy token and an eighth of the others."""
    n, D, sub, K, page = 20000, 64, 4, 32, 64
    q, k_cb, v_cb, kc, vc, table, kv_lens, starts = attention_case([rows], [n], 2, 1, D, sub, K, page, dtype, seed=80)
    q[:] = 0.25
    k_cb[:] = ((1 - nats / 16) + (torch.arange(K) - 16) / 512)[:, None].to(dtype)
    k_cb[:, 0] = 1.0                                                     # its score is 16, the others' lie about `nats` below
    v_cb[:] = (1e4 + 1e4 * torch.rand((1, K, D), generator=torch.Generator().manual_seed(81))).to(dtype)
    v_cb[:, 0] = 0.0
    kc.clamp_(min=1), vc.clamp_(min=1)
    j = torch.arange(n)
    heavy = {"first": j == 5, "last": j == n - 30, "by turns": j // 256 % 2 == 0}[where]      # (256: a tile for each of eight waves)
    at, off = table[0].long()[j[heavy] // page], j[heavy] % page
    kc[at, :, off], vc[at, :, :, off] = 0, 0
    case = (q, k_cb, v_cb, kc, vc, table, kv_lens, starts)
    out, lse = eng.cache_attention(*[t.to(DEV) for t in case], hint or rows, max_kv=hint, scale=1.0, want_lse=True)
    ref, ref_lse, size, slip = attention64(*case, sub, 1.0)
    half = HALF[dtype]
    # as check_attention; results below fp16's normal numbers are off by half of 2^-24; and the 31 tokens beside the heavy one in its tile have weights
    # that are off by 2^-33 of its own at most (half of 2^-24, where its own is 2^8 or more)
    tol = half * (1 + half) * (ref.abs() + size) + (2 * slip + (n + 8) * 2.0 ** -23) * size + 2.0 ** -25 + 31 * 2.0 ** -33 * v_cb.max().double()
    assert (tol <= 0.25 * ref).any() or where == "by turns"
    off = (out.cpu().double() - ref).abs()
    assert (off <= tol).all(), float((off / ref).max())
    assert ((lse.cpu().double() - ref_lse).abs() <= slip[..., 0] + (n + 8) * 2.0 ** -23 + 2.0 ** -21 * ref_lse.abs()).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_levels_far_apart(eng, dtype):
    """Tiles whose scores fall and rise by up to a thousand: maxima move both ways, nothing overflows, only what is too small to be seen is lost."""
    n, D, sub, K, page = 3000, 64, 4, 64, 64
    q, k_cb, v_cb, kc, vc, table, kv_lens, starts = attention_case([3], [n], 2, 1, D, sub, K, page, dtype, seed=85)
    q[:] = 0.25
    level = torch.randint(0, K, (n,), generator=torch.Generator().manual_seed(86))
    level = level[torch.arange(n) // 32 * 32]                            # one level to a tile
    k_cb[:] = (torch.arange(K) - K / 2)[:, None].to(dtype)
    kc[table[0].long()[torch.arange(n) // page], :, torch.arange(n) % page] = level[:, None, None].to(torch.uint8)
    for scale in (1.0, 0.25, 1 / 64):
        case = (q, k_cb, v_cb, kc, vc, table, kv_lens, starts)
        out, lse = eng.cache_attention(*[t.to(DEV) for t in case], 1, max_kv=1, scale=scale, want_lse=True)
        check_attention(out, lse, attention64(*case, sub, scale), n)


@pytest.mark.parametrize("dtype,size", [(torch.float16, 2e4), (torch.bfloat16, 2e4), (torch.bfloat16, 1e8), (torch.bfloat16, 1e15)])
@pytest.mark.parametrize("n_q,n_kv", [([1, 1], [700, 90]), ([20, 40], [300, 64])])
def test_attention_scores_whose_steps_are_large(eng, dtype, size, n_q, n_kv):
    """Scores of 10^10 and more, where neighbouring fp32 numbers are far apart: the largest takes all, and its value comes back as it is."""
    D, sub, K = 64, 4, 256
    case = list(attention_case(n_q, n_kv, 4, 2, D, sub, K, 16, dtype, seed=90))
    case[0], case[1] = (case[0].float().clamp(-3, 3) * size).to(dtype), (case[1].float().clamp(-3, 3) * size).to(dtype)
    ref, ref_lse, _, slip = attention64(*case, sub, 1.0)
    # rows whose two largest scores could change places are left out: their weights are 0 and 1 to the last bit everywhere else
    out, lse = eng.cache_attention(*[t.to(DEV) for t in case], max(n_q), scale=1.0, want_lse=True)
    out, lse = out.cpu().double(), lse.cpu().double()
    assert out.isfinite().all() and lse.isfinite().all()
    assert ((lse - ref_lse).abs() <= slip[..., 0] + 2.0 ** -21 * ref_lse.abs()).all()
    q, k_cb, _, kc, _, table, kv_lens, starts = case
    sure = torch.zeros(out.shape[:2], dtype=torch.bool)
    for b in range(len(n_q)):
        j = torch.arange(n_kv[b])
        for h in range(2):
            kd = vectors64(kc[table[b].long()[j // 16], h, j % 16], k_cb[h], sub)
            for r in range(int(starts[b]), int(starts[b + 1])):
                see = j <= n_kv[b] - int(starts[b + 1]) + r
                for g in (2 * h, 2 * h + 1):
                    z = (kd[see] @ q[r, g].double()).sort(descending=True)[0]
                    sure[r, g] = len(z) == 1 or z[0] - z[1] > 2 * slip[r, g, 0] + 200
    assert sure.float().mean() > 0.9
    assert torch.equal(out[sure], ref[sure])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n_q,n_kv", [([1, 1], [40, 700]), ([30, 3], [300, 60])])
def test_attention_infinite_scores(eng, dtype, n_q, n_kv):
    """A row with scores of plus infinity is none, with scores of minus infinity alone sees nothing;
    the rows beside it stay as they are."""
    case = list(attention_case(n_q, n_kv, 4, 2, 64, 4, 256, 16, dtype, seed=87))
    q, k_cb = case[:2]
    k_cb[:, :, 5] = k_cb[:, :, 5].abs() + 0.5
    clean = [t.cpu() for t in eng.cache_attention(*[t.to(DEV) for t in case], max(n_q), want_lse=True)]
    q[1, 0, 5], q[1, 3, 5] = math.inf, -math.inf
    out, lse = (t.cpu() for t in eng.cache_attention(*[t.to(DEV) for t in case], max(n_q), want_lse=True))
    assert out[1, 0].isnan().all() and lse[1, 0].isnan()
    assert not out[1, 3].any() and lse[1, 3] == -math.inf
    rest = torch.ones(out.shape[:2], dtype=torch.bool)
    rest[1, 0] = rest[1, 3] = False
    half = HALF[dtype]
    assert out[rest].isfinite().all() and lse[rest].isfinite().all()
    # the same sums, against references that may have moved at other tiles
    assert ((out.double() - clean[0].double())[rest].abs() <= 4 * half * case[2].abs().max().double()).all()
    assert ((lse.double() - clean[1].double())[rest].abs() <= 2.0 ** -18 * (1 + clean[1].double().abs())[rest]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,rows", [(64, 1), (128, 40), (192, 1), (256, 20)])
def test_attention_of_one_token_is_its_value(eng, dtype, D, rows):
    """A row that sees one token, or one 80 nats above the others, gives that token's value as it is, whatever the score."""
    sub, K = 4, 64
    case = list(attention_case([1, rows], [1, rows], 4, 2, D, sub, K, 16, dtype, seed=88))
    q, k_cb, v_cb, kc, vc, table, kv_lens, starts = case
    ref = attention64(*case, sub, 0.37)[0]
    out = eng.cache_attention(*[t.to(DEV) for t in case], rows, scale=0.37).cpu().double()
    assert torch.equal(out[:2], ref[:2])                                 # each sequence's first row
    k_cb[:, 0], q[:] = 2.0, 1.0 + torch.rand(q.shape, generator=torch.Generator().manual_seed(89)).to(dtype)
    k_cb[:, 1:] = -k_cb[:, 1:].abs()
    kc.clamp_(min=1)
    page, at = int(table[1, 0]), 0
    kc[page, :, at] = 0                                                  # every row of the second sequence sees its first token
    ref, _, size, _ = attention64(*case, sub, 1.0)
    out = eng.cache_attention(*[t.to(DEV) for t in case], rows, scale=1.0).cpu().double()
    value = torch.stack([vectors64(vc[page, g // 2, :, at][None], v_cb[g // 2], sub)[0] for g in range(4)])
    assert (ref[1:] - value).abs().max() < 1e-20
    assert torch.equal(out[1:], value.expand(rows, 4, D))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 12])
def test_attention_of_the_largest_values(eng, dtype, rows):
    """A mean of the type's largest numbers is none larger, though weights whose rounding is all upwards make it one by a step."""
    n, D, sub, K = 32, 64, 4, 64
    q, k_cb, v_cb, kc, vc, table, kv_lens, starts = attention_case([rows], [n], 4, 2, D, sub, K, 16, dtype, seed=91)
    q[:], k_cb[:], kc[:] = 0.25, 0.0, 1
    k_cb[:, 0] = 1.0                                                     # one token's score is 16, the others' 0; one wave takes them all
    kc[int(table[0, 0]), :, 3] = 0
    v_cb[:] = torch.finfo(dtype).max * (1 if dtype == torch.float16 else 2.0 ** -20)     # (fp32's sums hold 2^20 of the latter)
    v_cb[:, :, ::2] *= -1
    weight = 0.5 + 1.05 * HALF[dtype] / 2                                # of the others: a little above the middle of two neighbours
    case = (q, k_cb, v_cb, kc, vc, table, kv_lens, starts)
    scale = -math.log(weight) / 16
    out, lse = eng.cache_attention(*[t.to(DEV) for t in case], rows, scale=scale, want_lse=True)
    assert out.isfinite().all()
    check_attention(out, lse, attention64(*case, sub, scale), n)


@pytest.mark.parametrize("scale", [3e-38, -2e-39, 1e-44])
def test_attention_tiny_scale(eng, scale):
    """A scale near or below fp32's smallest normal number is taken as it is."""
    case = list(attention_case([1, 20], [300, 95], 4, 2, 64, 4, 256, 16, torch.bfloat16, seed=95))
    case[0], case[1] = (case[0].float() * 1e18).to(torch.bfloat16), (case[1].float() * 1e18).to(torch.bfloat16)
    out, lse = eng.cache_attention(*[t.to(DEV) for t in case], 20, scale=scale, want_lse=True)
    check_attention(out, lse, attention64(*case, 4, scale), 300)


WIDE = [
    # new tokens, lengths, q_heads, heads, dim, sub, K, page, dtype: single tokens, sixteen rows a head at most; 192 and 256 dims
    ([1, 1], [700, 90], 4, 2, 192, 2, 40, 64, torch.float16), ([1, 1], [2500, 90], 4, 2, 192, 4, 128, 16, torch.bfloat16),
    ([1, 1], [333, 1], 8, 2, 192, 8, 100, 16, torch.bfloat16), ([1, 2], [1700, 64], 8, 1, 192, 8, 128, 48, torch.float16),
    ([1, 1], [700, 90], 4, 2, 192, 2, 256, 64, torch.bfloat16), ([1, 1], [2500, 90], 4, 2, 192, 4, 256, 16, torch.float16),
    ([1, 1], [333, 1], 8, 2, 192, 8, 255, 16, torch.float16), ([1, 1], [3000, 3000], 8, 2, 192, 8, 129, 32, torch.bfloat16),
    ([1, 1], [700, 90], 4, 2, 256, 2, 40, 64, torch.float16), ([1, 1], [2500, 90], 4, 2, 256, 4, 128, 16, torch.bfloat16),
    ([1, 1], [333, 1], 8, 2, 256, 8, 100, 16, torch.bfloat16), ([1, 2], [1700, 64], 8, 1, 256, 8, 128, 48, torch.float16),
    ([1, 1], [700, 90], 4, 2, 256, 2, 256, 64, torch.bfloat16), ([1, 1], [2500, 90], 4, 2, 256, 4, 256, 16, torch.float16),
    ([1, 1], [333, 1], 8, 2, 256, 8, 255, 16, torch.float16), ([1, 1], [3000, 3000], 8, 2, 256, 8, 129, 32, torch.bfloat16),
    ([1, 1], [700, 90], 4, 2, 192, 2, 64, 64, torch.bfloat16), ([1, 1], [1700, 90], 4, 2, 192, 2, 200, 64, torch.float16),
    ([1, 1], [700, 90], 4, 2, 192, 4, 64, 64, torch.float16), ([1, 1], [1700, 90], 4, 2, 192, 4, 200, 64, torch.bfloat16),
    ([1, 1], [700, 90], 4, 2, 256, 2, 64, 64, torch.bfloat16), ([1, 1], [1700, 90], 4, 2, 256, 2, 200, 64, torch.float16),
    ([1, 1], [700, 90], 4, 2, 256, 4, 64, 64, torch.float16), ([1, 1], [1700, 90], 4, 2, 256, 4, 200, 64, torch.bfloat16),
    # many rows: what is looked up in the caches and what is not, by the pairs of dims and parts that no other test has
    ([40, 3], [300, 64], 4, 2, 192, 8, 256, 16, torch.bfloat16), ([40, 3], [300, 64], 4, 2, 192, 8, 16, 16, torch.float16),
    ([40, 3], [300, 64], 4, 2, 256, 2, 256, 16, torch.float16), ([40, 3], [300, 64], 4, 2, 256, 2, 33, 16, torch.bfloat16),
    ([1, 40], [300, 64], 4, 2, 32, 4, 256, 16, torch.bfloat16), ([1, 1], [300, 2000], 4, 2, 32, 4, 100, 16, torch.float16),
    ([1, 40], [300, 64], 4, 2, 96, 2, 256, 16, torch.float16), ([1, 1], [300, 2000], 4, 2, 96, 2, 100, 16, torch.bfloat16),
]


@pytest.mark.parametrize("hint", [None, 1])
@pytest.mark.parametrize("n_q,n_kv,Hq,H,D,sub,K,page,dtype", WIDE)
def test_attention_wide(eng, n_q, n_kv, Hq, H, D, sub, K, page, dtype, hint):
    """(hint: with what the table holds the longer sequences are cut between workgroups; with one token none is.)"""
    case = attention_case(n_q, n_kv, Hq, H, D, sub, K, page, dtype, seed=D + sub)
    out, lse = eng.cache_attention(*[t.to(DEV) for t in case], max(n_q), max_kv=hint, want_lse=True)
    check_attention(out, lse, attention64(*case, sub, 1.0 / math.sqrt(D)), max(n_kv))


@pytest.mark.parametrize("n_q,n_kv,Hq,H,D,sub,K,dtype", [
    ([1], [501], 32, 8, 128, 4, 256, torch.bfloat16), ([1] * 16, [2000 + 700 * i for i in range(16)], 32, 8, 128, 4, 256, torch.bfloat16),
    ([61, 1, 30, 2, 7], [3001, 900, 1400, 0, 2000], 6, 2, 64, 8, 200, torch.float16), ([600], [4000], 32, 8, 128, 4, 256, torch.bfloat16)])
def test_attention_repeats_itself(eng, n_q, n_kv, Hq, H, D, sub, K, dtype):
    """The same call gives the same bits, other calls between."""
    case = [t.to(DEV) for t in attention_case(n_q, n_kv, Hq, H, D, sub, K, 16, dtype, seed=97)]
    first = eng.cache_attention(*case, max(n_q), want_lse=True)
    for i in range(4):
        other = torch.empty(1 << (16 + 2 * i), device=DEV).fill_(math.nan)          # what the allocator hands out next holds something else
        del other
        again = eng.cache_attention(*case, max(n_q), want_lse=True)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_attention_longest_context(eng):
    """The longest length there is, 2^31 - 16 tokens, by a table that names one page again and again."""
    D, sub, K, page, width = 32, 8, 16, 16, (1 << 27) - 1
    q, k_cb, v_cb, kc, vc, table, kv_lens, starts = attention_case([1], [16], 1, 1, D, sub, K, page, torch.bfloat16, seed=99)
    ref, ref_lse, size, slip = attention64(q, k_cb, v_cb, kc, vc, table, kv_lens, starts, sub, D ** -0.5)
    long = torch.full((1, width), int(table[0, 0]), dtype=torch.int32, device=DEV)
    lens = torch.tensor([2 ** 31 - 1], dtype=torch.int32, device=DEV)
    out, lse = eng.cache_attention(*[t.to(DEV) for t in (q, k_cb, v_cb, kc, vc)], long, lens, starts.to(DEV), 1, want_lse=True)
    # a lane adds 2^31 / (256 workgroups * 8 waves * 32) = 2^15 times; all those additions may err the same way
    adds = 2.0 ** 15 * 1.1 * 2.0 ** -23
    assert ((out.cpu().double() - ref).abs() <= 2.0 ** -8 * 1.01 * (ref.abs() + size) + (2 * slip + 2 * adds) * size).all()
    assert ((lse.cpu().double() - ref_lse - math.log(width)).abs() <= slip[..., 0] + adds + 2.0 ** -21 * 30).all()


# ---- search and training ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("sub", [2, 4, 8])
@pytest.mark.parametrize("K", [2, 5, 17, 20, 21, 33, 37, 256])
def test_codewords_too_small_to_tell_apart(eng, K, sub):
    """Codewords of 10^-19 to 10^-12 of the vectors' size: where the sums of 64 bits are equal, the lowest number wins."""
    T, H, D = 600, 1, 64
    x = data(7, (T, H, D), torch.bfloat16)
    x = (x.float() * 10.0 ** (torch.arange(T) % 8).float().reshape(T, 1, 1)).to(torch.bfloat16)
    cb = (data(8, (H, K, D), torch.float32) * 1e-12).to(torch.bfloat16)
    code, _ = codes64(x, cb, sub)
    assert len(np.unique(code)) > 1
    kc, vc = eng.cache_buffers(38, 16, H, D, sub)
    eng.cache_write(x.to(DEV), x.to(DEV), torch.arange(T, device=DEV), cb.to(DEV), cb.to(DEV), kc, vc)
    assert torch.equal(kc.cpu().transpose(1, 2).reshape(608, H, D // sub)[:T].long(), torch.from_numpy(code))
    assert torch.equal(vc.cpu().permute(0, 3, 1, 2).reshape(608, H, D // sub)[:T].long(), torch.from_numpy(code))
    _, counts, _ = eng.cache_lbg_accum(x.to(DEV), cb.float().to(DEV), sub)
    for m in range(D // sub):
        assert torch.equal(counts[0, m].cpu(), torch.bincount(torch.from_numpy(code[:, 0, m]), minlength=K))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,D,sub", [(8, 256, 2), (8, 256, 4), (8, 256, 8)])
@pytest.mark.parametrize("value", [math.pi, 0.1, -1234.567])
def test_training_mean_of_equal_vectors(eng, dtype, H, D, sub, value):
    """Whole chunks of 4096 equal vectors: their mean is that vector within the roundings of 256 of them."""
    T = 4096 * {2: 4, 4: 8, 8: 8}[sub] + 40
    x = torch.full((1, 1, 1), value, dtype=dtype, device=DEV).expand(T, H, D).contiguous()
    x[:, 1] *= 1.5
    cb = torch.full((H, 3, D), 1e4, device=DEV)
    cb[:, 1] = value
    sums, counts, _ = eng.cache_lbg_accum(x, cb, sub)
    assert (counts[:, :, 1] == T).all()
    want = x[0].double()
    # Products of three pieces add up 256 numbers in 8 steps of 32: 24 additions, each off by 2^-23 of a partial sum at most (half of all, on average),
    # all the same way.  What they add up to is added exactly, rounded once to fp32 and joined in fp64.
    off = float(((sums[:, 1] / T - want).abs() / want.abs()).max())
    assert off <= (2 * 3 * 4.5 + 1) * 2.0 ** -24, off * 2 ** 24
    new, _, _ = eng.cache_lbg_iterate(x, cb, sub)
    assert float(((new[:, 1].double() - want).abs() / want.abs()).max()) <= (2 * 3 * 4.5 + 2) * 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sub", [2, 4, 8])
def test_training_sums_of_the_largest_numbers(eng, dtype, sub):
    """Numbers just below 2^100: hundreds of them in one cluster add up to more than 2^106."""
    T, H, D, K = 1500, 1, 64, 7
    x = data(7, (T, H, D), torch.float32)
    x = x.sign() * (0.5 + 0.49 * x.abs().clamp(max=1.0))
    big = torch.arange(T) % 3 == 0
    x = torch.where(big[:, None, None], x * 2.0 ** 100, x).to(dtype)
    cb = data(8, (H, K, D), torch.float32)
    cb[:, 3], cb[:, 5] = 2.0 ** 99, -2.0 ** 99
    sums, counts, dist = eng.cache_lbg_accum(x.to(DEV), cb.to(DEV), sub)
    assert sums.isfinite().all() and float(sums.abs().max()) > 2.0 ** 104
    new, mean = eng.cache_lbg_finish(sums, counts, dist, cb.to(DEV))
    check_training(x, cb, sub, sums, counts, dist, new, mean)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_training_beside_what_is_not_finite(eng, dtype):
    """Vectors and codewords that are not finite, everything that an iteration gives: they are left out, or stay as they were."""
    T, H, D, sub, K = 200, 1, 64, 4, 64
    x, cb = data(7, (T, H, D), dtype), data(8, (H, K, D), torch.float32)
    x[3, 0, 5], x[4, 0, 7], x[5, 0, 0] = math.nan, math.inf, -math.inf
    cb[:, 9], cb[:, 3, 2] = math.inf, math.nan
    code, least = codes64(x, cb, sub)
    fine = x.double().reshape(T, H, D // sub, sub).isfinite().all(-1)
    sums, counts, dist = (t.cpu() for t in eng.cache_lbg_accum(x.to(DEV), cb.to(DEV), sub))
    new, mean = (t.cpu() for t in eng.cache_lbg_finish(sums.to(DEV), counts.to(DEV), dist.to(DEV), cb.to(DEV)))
    new2, counts2, mean2 = (t.cpu() for t in eng.cache_lbg_iterate(x.to(DEV), cb.to(DEV), sub))
    assert torch.equal(counts, counts2) and torch.equal(mean, mean2) and torch.equal(new.nan_to_num(7.0), new2.nan_to_num(7.0))
    for m in range(D // sub):
        ok, part = fine[:, 0, m], slice(m * sub, (m + 1) * sub)
        xs, c = x[ok, 0, part].double(), torch.from_numpy(code[:, 0, m])[ok]
        n = torch.bincount(c, minlength=K)
        assert torch.equal(counts[0, m], n)
        want, size = (torch.zeros((K, sub), dtype=torch.float64).index_add_(0, c, t) for t in (xs, xs.abs()))
        tol = 32 * 2.0 ** -23 * size
        assert ((sums[0, :, part] - want).abs() <= tol).all()
        far = torch.from_numpy(least[:, 0, m])[ok].sum()
        assert abs(float(dist[0, m] - far)) <= 1e-12 * float(far) and abs(float(mean[0, m] - far / int(ok.sum()))) <= 2e-12 * float(far) / int(ok.sum())
        has = n > 0
        centre = want[has] / n[has, None]
        assert ((new[0, has, part].double() - centre).abs() <= tol[has] / n[has, None] + 2.0 ** -24 * 1.001 * centre.abs()).all()
        assert torch.equal(new[0, ~has, part].nan_to_num(7.0), cb[0, ~has, part].nan_to_num(7.0))


class HalvesOnly:
    """An engine of the two halves alone."""

    def __init__(self, eng):
        self.device, self.cache_lbg_accum, self.cache_lbg_finish = eng.device, eng.cache_lbg_accum, eng.cache_lbg_finish


def test_whole_training_by_one_call_an_iteration(eng, monkeypatch):
    """A process by itself trains by cache_lbg_iterate, bit for bit as by the two halves."""
    from vector_quantization_amd import train_cache_codebooks
    x = data(5, (3000, 3, 64), torch.bfloat16).to(DEV)
    halves = train_cache_codebooks(HalvesOnly(eng), x, 32, 4, log=None, max_iterations=20)
    monkeypatch.setattr(eng, "cache_lbg_accum", lambda *a: pytest.fail("the halves were called"), raising=False)
    one = train_cache_codebooks(eng, x, 32, 4, log=None, max_iterations=20)
    assert torch.equal(one.codebook, halves.codebook)
    assert one.distortions == halves.distortions and one.iters_per_stage == halves.iters_per_stage
