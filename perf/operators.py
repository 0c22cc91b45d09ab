"""The vector-quantised key-value cache: what is timed, on which sizes, and the operators' plain forms.

A cache entry of one token and one head is a vector of `dim` numbers, cut into dim / sub sub-vectors; each is stored as the
number (one byte) of its nearest codeword in squared distance.  A codebook is (heads, K, dim): its row k holds codeword k of
every sub-vector side by side.  Key codes lie as (pages, heads, page, dim / sub), value codes as (pages, heads, dim / sub, page).

  write      quantises new keys and values and puts their codes into the cache's slots
  read       the vectors that the codes of given slots stand for
  attention  causal attention of packed sequences' newest tokens over the paged cache, with the logarithm of each row's sum
  train      one LBG iteration of float codebooks: nearest codewords, their members' means and counts, the mean distortion
"""
import math
import random

import numpy as np
import torch

own = False
DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_engine = None


def listed():
    return [
        # one token for each of eight sequences in a serving step: the latency of a call
        {"name": "write step", "op": "write", "tokens": 8, "heads": 8, "dim": 128, "sub": 4, "K": 256, "page": 64, "dtype": "bf16"},
        # an odd prompt, half precision, small heads, a codebook of no power of two
        {"name": "write odd", "op": "write", "tokens": 1237, "heads": 3, "dim": 64, "sub": 2, "K": 100, "page": 16, "dtype": "fp16"},
        # a long prompt
        {"name": "write prompt", "op": "write", "tokens": 16384, "heads": 8, "dim": 128, "sub": 4, "K": 256, "page": 64, "dtype": "bf16"},
        # a few entries taken back out
        {"name": "read few", "op": "read", "tokens": 77, "heads": 4, "dim": 96, "sub": 2, "K": 256, "page": 16, "dtype": "fp16"},
        # a whole prompt's cache taken back out
        {"name": "read prompt", "op": "read", "tokens": 65536, "heads": 8, "dim": 128, "sub": 4, "K": 256, "page": 64, "dtype": "bf16"},
        # one sequence, one new token, a short history
        {"name": "step short", "op": "attention", "kind": "step", "seqs": 1, "max_q": 1, "max_kv": 501, "q_heads": 32, "heads": 8,
         "dim": 128, "sub": 4, "K": 256, "page": 64, "dtype": "bf16"},
        # a serving step: one new token for each of sixteen sequences with long histories
        {"name": "step batch", "op": "attention", "kind": "step", "seqs": 16, "max_q": 1, "max_kv": 32768, "q_heads": 32, "heads": 8,
         "dim": 128, "sub": 4, "K": 256, "page": 64, "dtype": "bf16"},
        # a mixed step of ragged chunks, odd groups, one sequence without history
        {"name": "mixed ragged", "op": "attention", "kind": "mixed", "seqs": 7, "max_q": 61, "max_kv": 3001, "q_heads": 6, "heads": 2,
         "dim": 64, "sub": 8, "K": 200, "page": 16, "dtype": "fp16"},
        # a chunk of a long prompt over what came before it
        {"name": "chunk", "op": "attention", "kind": "chunk", "seqs": 1, "max_q": 2048, "max_kv": 16384, "q_heads": 32, "heads": 8,
         "dim": 128, "sub": 4, "K": 256, "page": 64, "dtype": "bf16"},
        # a small calibration set in 32 bits
        {"name": "train small", "op": "train", "tokens": 1500, "heads": 2, "dim": 64, "sub": 4, "K": 64, "dtype": "fp32"},
        # sub-vectors of eight
        {"name": "train wide", "op": "train", "tokens": 8192, "heads": 4, "dim": 128, "sub": 8, "K": 256, "dtype": "fp16"},
        # a calibration set of a whole layer
        {"name": "train layer", "op": "train", "tokens": 32768, "heads": 8, "dim": 128, "sub": 4, "K": 256, "dtype": "bf16"},
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["write", "read", "attention", "attention", "train"])
    case = {"op": op, "heads": rng.randint(1, 8), "dim": rng.choice([32, 64, 64, 96, 128, 128, 128, 192, 256]), "sub": rng.choice([2, 4, 8]),
            "K": rng.choice([256, 256, rng.randint(16, 255)]), "dtype": rng.choice(["bf16", "bf16", "fp16"])}
    if op == "train":
        case["dtype"] = rng.choice(["bf16", "fp16", "fp32"])
        case["tokens"] = _spread(rng, 300, 32768)
    elif op == "attention":
        case["page"] = rng.choice([16, 32, 48, 64, 128, 256])
        case["kind"] = rng.choice(["step", "step", "chunk", "mixed"])
        case["q_heads"] = case["heads"] * rng.choice([1, 2, 3, 4, 5, 7, 8])
        case["seqs"] = 1 if case["kind"] == "chunk" else _spread(rng, 1, 32)
        case["max_q"] = 1 if case["kind"] == "step" else _spread(rng, 2, 2048 if case["kind"] == "chunk" else 256)
        case["max_kv"] = _spread(rng, 17, 32768)
        while case["seqs"] * case["max_kv"] * case["heads"] * case["dim"] > 16 * 32768 * 8 * 128 or \
                case["seqs"] * case["max_q"] * case["q_heads"] * case["max_kv"] > 2048 * 32 * 16384:
            case["max_kv"] = case["max_kv"] * 2 // 3
        case["max_q"] = min(case["max_q"], case["max_kv"])
    else:
        case["page"] = rng.choice([16, 32, 48, 64, 128, 256])
        case["tokens"] = _spread(rng, 1, 16384 if op == "write" else 65536)
    if op in ("write", "train"):
        while case["tokens"] * case["heads"] * (case["dim"] // case["sub"]) * case["K"] > (1 << 30):
            case["tokens"] = case["tokens"] * 2 // 3
    if op == "read":
        while case["tokens"] * case["heads"] * case["dim"] > (1 << 26):
            case["tokens"] = case["tokens"] * 2 // 3
    return case


def _lengths(case):
    """New tokens and history (the new ones among it) of each sequence; they follow from the case alone."""
    r = random.Random("%(kind)s %(seqs)d %(max_q)d %(max_kv)d" % case)
    n_q, n_kv = [], []
    for b in range(case["seqs"]):
        kv = case["max_kv"] if b == 0 else r.randint(max(1, case["max_kv"] // 4), case["max_kv"])
        q = case["max_q"] if b == 0 or case["kind"] == "step" else r.randint(0, case["max_q"])
        if case["kind"] == "mixed" and b == 3:
            kv, q = 0, min(2, case["max_q"])          # rows that see nothing
        n_q.append(q if kv == 0 else min(q, kv))
        n_kv.append(kv)
    return n_q, n_kv


def _mixed_vectors(shape, mix, gen):
    """Vectors whose neighbouring elements are correlated and whose sizes differ from element to element, as a projection's outputs are."""
    x = torch.randn(shape, generator=gen, device=DEVICE)
    x = x + 0.5 * x.roll(1, -1)
    return x * mix


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    rng = np.random.default_rng(int(seed))
    heads, dim, sub, K = case["heads"], case["dim"], case["sub"], case["K"]
    dtype = DTYPES[case["dtype"]]
    parts = dim // sub
    s = {"case": case, "sub": sub}
    mix = torch.rand((heads, 1, dim), generator=gen, device=DEVICE) + 0.5
    books = [0.9 * _mixed_vectors((heads, K, dim), mix, gen) for _ in range(2)]
    if case["op"] == "train":
        s["cb"] = books[0]
        s["x"] = _mixed_vectors((case["tokens"], heads, dim), mix[:, 0], gen).to(dtype)
        return s
    s["k_cb"], s["v_cb"] = books[0].to(dtype), books[1].to(dtype)
    page = case["page"]
    if case["op"] == "attention":
        n_q, n_kv = _lengths(case)
        width = -(-max(1, max(n_kv)) // page)
        pages = sum(-(-n // page) for n in n_kv) + 3
        order = rng.permutation(pages)
        table = np.zeros((case["seqs"], width), np.int32)
        at = 0
        for b, n in enumerate(n_kv):
            use = -(-n // page)
            table[b, :use] = order[at:at + use]
            at += use
        s["table"] = torch.from_numpy(table).to(DEVICE)
        s["n_kv"] = torch.tensor(n_kv, dtype=torch.int32, device=DEVICE)
        s["starts"] = torch.tensor(np.concatenate([[0], np.cumsum(n_q)]), dtype=torch.int32, device=DEVICE)
        s["max_q"], s["max_kv"] = max(n_q), max(n_kv)
        s["q"] = torch.randn((sum(n_q), case["q_heads"], dim), generator=gen, device=DEVICE).to(dtype)
    else:
        tokens = case["tokens"]
        pages = -(-tokens // page) + 2
        order = rng.permutation(pages)
        at = np.arange(tokens, dtype=np.int64)
        slots = order[at // page].astype(np.int64) * page + at % page
        if case["op"] == "write":
            if tokens >= 100:
                slots[rng.integers(0, tokens, 5)] = -1           # padding: tokens that are not stored
            s["k"] = _mixed_vectors((tokens, heads, dim), mix[:, 0], gen).to(dtype)
            s["v"] = _mixed_vectors((tokens, heads, dim), mix[:, 0], gen).to(dtype)
        s["slots"] = torch.from_numpy(slots).to(DEVICE)
    s["k_codes"] = torch.randint(0, K, (pages, heads, page, parts), generator=gen, device=DEVICE, dtype=torch.uint8)
    s["v_codes"] = torch.randint(0, K, (pages, heads, parts, page), generator=gen, device=DEVICE, dtype=torch.uint8)
    return s


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    global _engine
    if _engine is None:
        from vector_quantization_amd import HipEngine
        _engine = HipEngine(DEVICE)
    op = s["case"]["op"]
    if op == "write":
        _engine.cache_write(s["k"], s["v"], s["slots"], s["k_cb"], s["v_cb"], s["k_codes"], s["v_codes"])
        return s["k_codes"], s["v_codes"]
    if op == "read":
        return _engine.cache_read(s["slots"], s["k_cb"], s["v_cb"], s["k_codes"], s["v_codes"])
    if op == "attention":
        return _engine.cache_attention(s["q"], s["k_cb"], s["v_cb"], s["k_codes"], s["v_codes"], s["table"], s["n_kv"], s["starts"],
                                       s["max_q"], max_kv=s["max_kv"], want_lse=True)
    return _engine.cache_lbg_iterate(s["x"], s["cb"], s["sub"])


# ---- the plain forms ----------------------------------------------------------------------------------------------------

def _nearest(x, cb, sub):
    """(heads, parts, tokens) numbers of the nearest codewords, in 64 bits: which is nearest hangs on the last bits where two are close."""
    tokens, heads, dim = x.shape
    parts = dim // sub
    xs = x.double().reshape(tokens, heads, parts, sub).permute(1, 2, 0, 3).reshape(heads * parts, tokens, sub)
    cs = cb.double().reshape(heads, -1, parts, sub).permute(0, 2, 1, 3).reshape(heads * parts, -1, sub)
    score = (0.5 * cs * cs).sum(-1)[:, None, :] - torch.matmul(xs, cs.transpose(1, 2).contiguous())
    return score.argmin(-1).reshape(heads, parts, tokens)


def _looked_up(codes, cb, sub):
    """codes (..., heads, n, parts) -> the vectors (..., heads, n, dim) in 32 bits."""
    heads, K, dim = cb.shape
    parts = dim // sub
    c = cb.float().reshape(heads, K, parts, sub)
    h = torch.arange(heads, device=codes.device)[:, None, None]
    m = torch.arange(parts, device=codes.device)
    return c[h, codes.long(), m].flatten(-2)


def _plain(s):
    op, sub = s["case"]["op"], s["sub"]
    if op == "train":
        return _plain_train(s["x"], s["cb"], sub)
    if op == "attention":
        return _plain_attention(s)
    page, slots = s["case"]["page"], s["slots"]
    if op == "write":
        k, v = _nearest(s["k"], s["k_cb"], sub), _nearest(s["v"], s["v_cb"], sub)
        # a token without a slot rewrites the first slot of the last token that has one, with what that token writes there
        use = torch.where(slots >= 0, torch.arange(slots.numel(), device=slots.device), -1)
        use = torch.where(use >= 0, use, use.amax())
        slots, k, v = slots[use], k[:, :, use], v[:, :, use]
        s["k_codes"][slots // page, :, slots % page] = k.permute(2, 0, 1).to(torch.uint8)
        s["v_codes"][slots // page, :, :, slots % page] = v.permute(2, 0, 1).to(torch.uint8)
        return s["k_codes"], s["v_codes"]
    kc = s["k_codes"][slots // page, :, slots % page]
    vc = s["v_codes"][slots // page, :, :, slots % page]
    dtype = s["k_cb"].dtype
    return tuple(_looked_up(c[:, :, None], cb, sub)[:, :, 0].to(dtype) for c, cb in ((kc, s["k_cb"]), (vc, s["v_cb"])))


def _plain_attention(s):
    sub, q, starts, n_kv = s["sub"], s["q"], s["starts"].long(), s["n_kv"].long()
    heads, K, dim = s["k_cb"].shape
    rows, q_heads = q.shape[:2]
    seqs, group = n_kv.numel(), q_heads // heads
    table = s["table"].long()
    k = _looked_up(s["k_codes"][table].permute(0, 2, 1, 3, 4).flatten(2, 3), s["k_cb"], sub)
    v = _looked_up(s["v_codes"][table].permute(0, 2, 1, 4, 3).flatten(2, 3), s["v_cb"], sub)
    length = k.shape[2]
    step = torch.arange(s["max_q"], device=q.device)
    n_q = starts[1:] - starts[:-1]
    at = (starts[:-1, None] + step).clamp(max=rows - 1)
    qp = q.float()[at].reshape(seqs, s["max_q"], heads, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, heads, -1, dim)
    score = torch.matmul(qp, k.transpose(-1, -2).contiguous()) / math.sqrt(dim)
    last = (n_kv - n_q)[:, None] + step
    sees = torch.arange(length, device=q.device) <= last[:, :, None]
    sees &= (torch.arange(length, device=q.device) < n_kv[:, None])[:, None]
    score = score.masked_fill(~sees.repeat_interleave(group, 1)[:, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = (score - top).exp()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / total.clamp(min=1e-30)
    lse = torch.where(total > 0, top + total.clamp(min=1e-30).log(), -math.inf)[..., 0]
    row = torch.arange(rows, device=q.device)
    seq = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    out = out.reshape(seqs, heads, s["max_q"], group, dim).transpose(1, 2)[seq, row - starts[seq]]
    lse = lse.reshape(seqs, heads, s["max_q"], group).transpose(1, 2)[seq, row - starts[seq]]
    return out.reshape(rows, q_heads, dim).to(q.dtype), lse.reshape(rows, q_heads)


def _plain_train(x, cb, sub):
    tokens, heads, dim = x.shape
    K, parts = cb.shape[1], dim // sub
    codes = _nearest(x, cb, sub)
    near = codes.permute(2, 0, 1)                                      # (tokens, heads, parts)
    at = ((torch.arange(heads, device=x.device)[:, None] * parts + torch.arange(parts, device=x.device)) * K + near).flatten()
    xs = x.double().reshape(-1, sub)
    old = cb.double().reshape(heads, K, parts, sub).transpose(1, 2).reshape(-1, sub)
    counts = torch.zeros(heads * parts * K, dtype=torch.int64, device=x.device).index_add_(0, at, torch.ones_like(at))
    sums = torch.zeros_like(old).index_add_(0, at, xs)
    new = torch.where(counts[:, None] > 0, sums / counts.clamp(min=1)[:, None], old)
    off = (xs - old[at]).square().sum(-1).reshape(tokens, heads, parts).mean(0)
    new = new.reshape(heads, parts, K, sub).transpose(1, 2).reshape(heads, K, dim)
    return new.float(), counts.reshape(heads, parts, K), off


# ---- what a pass cannot do without --------------------------------------------------------------------------------------

def work(case):
    heads, dim, K, parts = case["heads"], case["dim"], case["K"], case["dim"] // case["sub"]
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "train":
        n = case["tokens"] * heads
        return {"bytes": n * dim * size + heads * K * (2 * dim * 4 + parts * 8) + heads * parts * 8, "flops": n * (2 * dim * K + 4 * dim)}
    books = 2 * heads * K * dim * size
    if case["op"] == "attention":
        n_q, n_kv = _lengths(case)
        rows = sum(n_q) * case["q_heads"]
        seen = sum(sum(max(0, kv - q + i + 1) for i in range(q)) for q, kv in zip(n_q, n_kv))
        moved = sum(kv for q, kv in zip(n_q, n_kv) if q) * heads * parts * 2
        return {"bytes": moved + books + rows * (2 * dim * size + 4), "flops": 4 * dim * case["q_heads"] * seen}
    n = case["tokens"] * heads
    both = 2 * (n * dim * size + n * parts) + books + case["tokens"] * 8
    return {"bytes": both, "flops": 4 * n * dim * K if case["op"] == "write" else 0}


# ---- the definitions in 64 bits, written apart from the above -------------------------------------------------------------

def _codes64(x, cb, sub):
    """(tokens, heads, parts): the codeword of the least sum of squares, the lowest number of equal ones."""
    tokens, heads, dim = x.shape
    K = cb.shape[1]
    out = torch.empty((tokens, heads, dim // sub), dtype=torch.int64, device=x.device)
    for h in range(heads):
        xh, ch = x[:, h].double().reshape(tokens, -1, sub), cb[h].double().reshape(K, -1, sub)
        far = torch.zeros((tokens, K, dim // sub), dtype=torch.float64, device=x.device)
        for e in range(sub):
            far += (xh[:, None, :, e] - ch[None, :, :, e]) ** 2
        out[:, h] = far.argmin(1)
    return out


def _vectors64(codes, cb, sub):
    """codes (n, parts) of one head, cb (K, dim) -> (n, dim)."""
    K, dim = cb.shape
    picked = torch.stack([cb.double().reshape(K, -1, sub)[codes[:, m].long(), m] for m in range(dim // sub)], 1)
    return picked.reshape(codes.shape[0], dim)


def exact(case, seed):
    s = prepare(case, seed)
    sub = s["sub"]
    if case["op"] == "train":
        x, cb = s["x"], s["cb"]
        codes = _codes64(x, cb, sub)
        tokens, heads, dim = x.shape
        K, parts = cb.shape[1], dim // sub
        new, counts = cb.double().clone(), torch.zeros((heads, parts, K), dtype=torch.int64, device=x.device)
        off = torch.zeros((heads, parts), dtype=torch.float64, device=x.device)
        for h in range(heads):
            for m in range(parts):
                xs, c = x[:, h, m * sub:(m + 1) * sub].double(), codes[:, h, m]
                member = torch.nn.functional.one_hot(c, K).double()
                counts[h, m] = member.sum(0).long()
                mean = member.T.contiguous() @ xs / counts[h, m].clamp(min=1)[:, None]
                new[h, :, m * sub:(m + 1) * sub] = torch.where(counts[h, m][:, None] > 0, mean, new[h, :, m * sub:(m + 1) * sub])
                off[h, m] = ((xs - cb[h, :, m * sub:(m + 1) * sub].double()[c]) ** 2).sum(1).mean()
        return new, counts, off
    if case["op"] == "write":
        kept = (s["slots"] >= 0).nonzero()[:, 0]
        p, o = s["slots"][kept] // case["page"], s["slots"][kept] % case["page"]
        kc, vc = _codes64(s["k"][kept], s["k_cb"], sub), _codes64(s["v"][kept], s["v_cb"], sub)
        for h in range(case["heads"]):
            s["k_codes"][p, h, o] = kc[:, h].to(torch.uint8)
            s["v_codes"][p, h, :, o] = vc[:, h].to(torch.uint8)
        return s["k_codes"], s["v_codes"]
    if case["op"] == "read":
        p, o = s["slots"] // case["page"], s["slots"] % case["page"]
        k = torch.stack([_vectors64(s["k_codes"][p, h, o], s["k_cb"][h], sub) for h in range(case["heads"])], 1)
        v = torch.stack([_vectors64(s["v_codes"][p, h, :, o], s["v_cb"][h], sub) for h in range(case["heads"])], 1)
        return k, v
    n_q, n_kv = _lengths(case)
    q, heads, page = s["q"].double(), case["heads"], case["page"]
    group = case["q_heads"] // heads
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    start = 0
    for b, (nq, nkv) in enumerate(zip(n_q, n_kv)):
        rows, start = slice(start, start + nq), start + nq
        if nq == 0 or nkv == 0:
            continue
        j = torch.arange(nkv, device=q.device)
        p, o = s["table"][b].long()[j // page], j % page
        hidden = j[None, :] > nkv - nq + torch.arange(nq, device=q.device)[:, None]
        for h in range(heads):
            kd = _vectors64(s["k_codes"][p, h, o], s["k_cb"][h], sub)
            vd = _vectors64(s["v_codes"][p, h, :, o], s["v_cb"][h], sub)
            for g in range(h * group, (h + 1) * group):
                z = (q[rows, g] @ kd.T.contiguous() * _scale(kd)).masked_fill(hidden, -math.inf)
                lse[rows, g] = torch.logsumexp(z, 1)
                out[rows, g] = torch.softmax(z, 1) @ vd
    return out, lse


def _scale(k):
    return 1.0 / math.sqrt(k.shape[-1])
