"""The vector-quantised key-value cache: HipEngine's cache_* methods and the training of their codebooks.

The image path's three steps (LBG training VQ_Full.py:60-98, encode :120-126, decode :153-169) for the keys and
values of attention.  The vector of one token and one head, dim numbers, is cut into parts = dim / sub sub-vectors,
each stored as one byte: the number of its nearest codeword in squared distance.

    codebook   (heads, K, dim), or (1, K, dim) for all heads; row k holds codeword k of every sub-vector side by side
    k_codes    (pages, heads, page, parts) uint8
    v_codes    (pages, heads, parts, page) uint8
    slot       page number * page + place in the page

dim is 32, 64, 96, 128, 192 or 256, sub 2, 4 or 8, K 1 to 256, page a multiple of 16.  At dim = 128, sub = 4 a token
takes 32 bytes a head for its key and 32 for its value, an eighth of bfloat16.

The methods launch on the engine's device and its current stream, allocate what they return (and their workspace)
from torch's allocator and wait for nothing, so they may be captured into a graph.  None of them is differentiable:
they refuse tensors that require a gradient.
"""
import ctypes
import math

import torch

from ._lib import lib, check, VQ_BF16, VQ_F16, VQ_F32

_DTYPES = {torch.float32: VQ_F32, torch.bfloat16: VQ_BF16, torch.float16: VQ_F16}


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else ctypes.c_void_p(0)


# ---- checks of arguments: shapes, types and devices only, nothing is read from the GPU ------------------------------

def _tensor(name, t, device, dtypes, dims):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the engine on {device}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} has dtype {t.dtype}, expected {' or '.join(str(d) for d in dtypes)}")
    if t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions, got shape {tuple(t.shape)}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient: the cache operators are not differentiable")
    return t


def _whole(name, t):
    if not t.is_contiguous() or t.data_ptr() % 16:
        raise ValueError(f"{name} must be contiguous and start at a multiple of 16 bytes")
    return t


def _vectors(t):
    """t as the kernels read it: each vector's numbers side by side from a multiple of 16 bytes.  Anything else is copied."""
    size = t.element_size()
    if t.numel() == 0 or (t.stride(2) == 1 and t.data_ptr() % 16 == 0 and t.stride(0) * size % 16 == 0 and t.stride(1) * size % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _books(t, multiple=16):
    return t if t.is_contiguous() and t.data_ptr() % multiple == 0 else t.clone(memory_format=torch.contiguous_format)


def cache_shape(k_cb, v_cb, k_codes, v_codes, device):
    """Checks codebooks and code buffers against each other; returns (heads, dim, sub, K, pages, page)."""
    _tensor("k_cb", k_cb, device, (torch.bfloat16, torch.float16), 3)
    _tensor("v_cb", v_cb, device, (k_cb.dtype,), 3)
    _whole("k_codes", _tensor("k_codes", k_codes, device, (torch.uint8,), 4))
    _whole("v_codes", _tensor("v_codes", v_codes, device, (torch.uint8,), 4))
    pages, heads, page, parts = k_codes.shape
    if 0 in k_codes.shape:
        raise ValueError(f"k_codes must not be empty, got shape {tuple(k_codes.shape)}")
    if tuple(v_codes.shape) != (pages, heads, parts, page):
        raise ValueError(f"v_codes must have shape {(pages, heads, parts, page)} (k_codes: {tuple(k_codes.shape)}), got {tuple(v_codes.shape)}")
    if k_cb.shape != v_cb.shape or k_cb.shape[0] not in (1, heads) or 0 in k_cb.shape:
        raise ValueError(f"codebooks must be (1 or {heads}, K, dim) of one shape, got {tuple(k_cb.shape)} and {tuple(v_cb.shape)}")
    K, dim = k_cb.shape[1:]
    if dim % parts:
        raise ValueError(f"vectors of {dim} numbers cannot be cut into the {parts} codes of a cache entry")
    return heads, dim, dim // parts, K, pages, page


def check_vectors(name, t, tokens, heads, dim, dtype, device):
    _tensor(name, t, device, (dtype,), 3)
    if tokens is not None and t.shape[0] != tokens or t.shape[1] != heads or t.shape[2] != dim:
        raise ValueError(f"{name} must have shape {('tokens' if tokens is None else tokens, heads, dim)}, got {tuple(t.shape)}")
    return _vectors(t)


def check_ints(name, t, dtype, shape, device):
    _tensor(name, t, device, (dtype,), len(shape))
    if any(s is not None and s != n for s, n in zip(shape, t.shape)):
        raise ValueError(f"{name} must have shape {tuple('any' if s is None else s for s in shape)}, got {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


class CacheOps:
    """The vector-quantised key-value cache on one device (mixed into HipEngine)."""

    def cache_buffers(self, pages, page, heads, dim, sub):
        """Empty (k_codes, v_codes) for pages * page tokens."""
        if min(pages, page, heads, dim, sub) < 1 or dim % sub or page % 16:
            raise ValueError(f"need positive sizes, dim a multiple of sub and page of 16, got pages={pages}, page={page}, heads={heads}, "
                             f"dim={dim}, sub={sub}")
        parts = dim // sub
        return (torch.zeros((pages, heads, page, parts), dtype=torch.uint8, device=self.device),
                torch.zeros((pages, heads, parts, page), dtype=torch.uint8, device=self.device))

    def cache_write(self, k, v, slots, k_cb, v_cb, k_codes, v_codes):
        """Quantises k and v (tokens, heads, dim) and stores the codes at slots (tokens, int64); a slot outside the cache
        (-1, say) stores nothing.  Slots should be distinct: of two tokens with one slot, each code is that of either."""
        heads, dim, sub, K, pages, page = cache_shape(k_cb, v_cb, k_codes, v_codes, self.device)
        slots = check_ints("slots", slots, torch.int64, (None,), self.device)
        tokens = slots.shape[0]
        k = check_vectors("k", k, tokens, heads, dim, k_cb.dtype, self.device)
        v = check_vectors("v", v, tokens, heads, dim, k_cb.dtype, self.device)
        if tokens == 0:
            return
        k_cb, v_cb = _books(k_cb), _books(v_cb)
        with torch.cuda.device(self.device):
            check(lib.vq_cache_write(_ptr(k), k.stride(0), k.stride(1), _ptr(v), v.stride(0), v.stride(1), _ptr(slots), tokens,
                                     _ptr(k_cb), _ptr(v_cb), k_cb.shape[0], heads, dim, sub, K, _DTYPES[k_cb.dtype], _ptr(k_codes),
                                     _ptr(v_codes), pages, page, self._stream()), "vq_cache_write")

    def cache_read(self, slots, k_cb, v_cb, k_codes, v_codes):
        """The keys and values that the codes at slots stand for: two tensors (tokens, heads, dim) of the codebooks'
        dtype.  A slot outside the cache reads as zeros."""
        heads, dim, sub, K, pages, page = cache_shape(k_cb, v_cb, k_codes, v_codes, self.device)
        slots = check_ints("slots", slots, torch.int64, (None,), self.device)
        tokens = slots.shape[0]
        k_cb, v_cb = _books(k_cb), _books(v_cb)
        k, v = (torch.empty((tokens, heads, dim), dtype=k_cb.dtype, device=self.device) for _ in range(2))
        if tokens:
            with torch.cuda.device(self.device):
                check(lib.vq_cache_read(_ptr(slots), tokens, _ptr(k_cb), _ptr(v_cb), k_cb.shape[0], heads, dim, sub, K, _DTYPES[k_cb.dtype],
                                        _ptr(k_codes), _ptr(v_codes), pages, page, _ptr(k), _ptr(v), self._stream()), "vq_cache_read")
        return k, v

    def cache_attention(self, q, k_cb, v_cb, k_codes, v_codes, table, kv_lens, starts, max_q, max_kv=None, scale=None, out=None,
                        want_lse=False):
        """Causal attention of packed sequences' newest tokens over the cache.

        q (rows, q_heads, dim): sequence b owns rows starts[b] to starts[b + 1] (starts: int32, one more than sequences)
        and the first kv_lens[b] (int32) tokens of the pages table[b] (int32, (sequences, width)); its rows are the newest
        of those tokens, whose keys and values are in the cache already.  Query head h reads cache head
        h // (q_heads / heads).  A row that sees no token gets zeros (and a logarithm of minus infinity); rows of no
        sequence are left as they were in `out`, and are undefined where the call allocates it.
        max_q, max_kv: the longest of the sequences' rows and lengths, as the host knows them; they shape the launch only
        (max_kv None: what the table can hold).  scale: 1 / sqrt(dim) if None.
        Returns out (rows, q_heads, dim), with want_lse also the natural logarithm of each row's sum of exponentials
        (rows, q_heads) float32, by which results over parts of a context are joined."""
        heads, dim, sub, K, pages, page = cache_shape(k_cb, v_cb, k_codes, v_codes, self.device)
        _tensor("q", q, self.device, (k_cb.dtype,), 3)
        rows, q_heads = q.shape[:2]
        if q.shape[2] != dim or q_heads == 0 or q_heads % heads:
            raise ValueError(f"q must have shape (rows, a multiple of {heads}, {dim}), got {tuple(q.shape)}")
        kv_lens = check_ints("kv_lens", kv_lens, torch.int32, (None,), self.device)
        seqs = kv_lens.shape[0]
        starts = check_ints("starts", starts, torch.int32, (seqs + 1,), self.device)
        table = check_ints("table", table, torch.int32, (seqs, None), self.device)
        width = table.shape[1]
        if out is None:
            out = torch.empty((rows, q_heads, dim), dtype=q.dtype, device=self.device)
        else:
            _whole("out", _tensor("out", out, self.device, (q.dtype,), 3))
            if out.shape != q.shape:
                raise ValueError(f"out must have shape {tuple(q.shape)}, got {tuple(out.shape)}")
        lse = torch.empty((rows, q_heads), dtype=torch.float32, device=self.device) if want_lse else None
        if rows and seqs:
            q, k_cb, v_cb = _vectors(q), _books(k_cb), _books(v_cb)
            scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
            max_q = int(max_q)
            max_kv = max(1, width * page) if max_kv is None else int(max_kv)
            need = lib.vq_cache_attention_ws_bytes(rows, q_heads, heads, dim, sub, K, seqs, max_q, max_kv)
            ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
            with torch.cuda.device(self.device):
                check(lib.vq_cache_attention(_ptr(q), q.stride(0), q.stride(1), rows, q_heads, _ptr(k_cb), _ptr(v_cb), k_cb.shape[0], heads,
                                             dim, sub, K, _DTYPES[q.dtype], _ptr(k_codes), _ptr(v_codes), pages, page, _ptr(table), seqs,
                                             width, _ptr(kv_lens), _ptr(starts), max_q, max_kv, scale, _ptr(out), _ptr(lse), _ptr(ws), need,
                                             self._stream()), "vq_cache_attention")
        return (out, lse) if want_lse else out

    def cache_lbg_accum(self, x, cb, sub):
        """The accumulating half of an LBG iteration of float codebooks cb (heads, K, dim) float32 over the vectors
        x (tokens, heads, dim): for each codeword the sum (heads, K, dim) float64 and number (heads, parts, K) int64 of the
        sub-vectors nearest to it, and the sum of their squared distances (heads, parts) float64.  A sub-vector of numbers
        that are not all finite is left out.  Shards' results are added."""
        _tensor("cb", cb, self.device, (torch.float32,), 3)
        _tensor("x", x, self.device, tuple(_DTYPES), 3)
        heads, K, dim = cb.shape
        check_vectors("x", x, None, heads, dim, x.dtype, self.device)
        if 0 in cb.shape or sub < 1 or dim % sub:
            raise ValueError(f"codebook of shape {tuple(cb.shape)} cannot be cut into sub-vectors of {sub}")
        tokens, parts = x.shape[0], dim // sub
        make = torch.empty if tokens else torch.zeros
        sums = make((heads, K, dim), dtype=torch.float64, device=self.device)
        counts = make((heads, parts, K), dtype=torch.int64, device=self.device)
        dist = make((heads, parts), dtype=torch.float64, device=self.device)
        if tokens:
            x, cb = _vectors(x), _books(cb)
            need = lib.vq_cache_lbg_ws_bytes(tokens, heads, dim, sub, K)
            ws = torch.empty(need, dtype=torch.uint8, device=self.device)
            with torch.cuda.device(self.device):
                check(lib.vq_cache_lbg_accum(_ptr(x), x.stride(0), x.stride(1), tokens, _ptr(cb), heads, dim, sub, K, _DTYPES[x.dtype],
                                             _ptr(sums), _ptr(counts), _ptr(dist), _ptr(ws), need, self._stream()), "vq_cache_lbg_accum")
        return sums, counts, dist

    def cache_lbg_finish(self, sums, counts, dist, cb):
        """The closing half: (new codebook, mean squared distance (heads, parts)); a codeword without members stays."""
        _tensor("cb", cb, self.device, (torch.float32,), 3)
        heads, K, dim = cb.shape
        _tensor("dist", dist, self.device, (torch.float64,), 2)
        parts = dist.shape[1]
        _tensor("sums", sums, self.device, (torch.float64,), 3)
        _tensor("counts", counts, self.device, (torch.int64,), 3)
        if 0 in cb.shape or parts < 1 or dim % parts or dist.shape[0] != heads or sums.shape != cb.shape or \
                tuple(counts.shape) != (heads, parts, K):
            raise ValueError(f"shapes do not belong together: sums {tuple(sums.shape)}, counts {tuple(counts.shape)}, dist {tuple(dist.shape)}, "
                             f"cb {tuple(cb.shape)}")
        sums, counts, dist, cb = (t.contiguous() for t in (sums, counts, dist, cb))
        new, mean = torch.empty_like(cb), torch.empty_like(dist)
        with torch.cuda.device(self.device):
            check(lib.vq_cache_lbg_finish(_ptr(sums), _ptr(counts), _ptr(dist), _ptr(cb), heads, dim, dim // parts, K, _ptr(new), _ptr(mean),
                                          self._stream()), "vq_cache_lbg_finish")
        return new, mean

    def cache_lbg_iterate(self, x, cb, sub):
        """One LBG iteration of the float codebooks cb (heads, K, dim) over the vectors x (tokens, heads, dim): returns (new
        codebook, members (heads, parts, K), mean squared distance to the old codewords (heads, parts))."""
        sums, counts, dist = self.cache_lbg_accum(x, cb, sub)
        new, mean = self.cache_lbg_finish(sums, counts, dist, cb)
        return new, counts, mean


def _added_over_ranks(sums, counts, dist, group):
    """The ranks' three results added in rank order, so that every rank holds the same bits."""
    import torch.distributed as dist_
    from .lbg import _all_gather_into
    world = dist_.get_world_size(group=group)
    out = []
    for t in (sums, counts, dist):
        parts = _all_gather_into(t.reshape(-1), world, group)
        total = parts[0].clone()
        for r in range(1, world):
            total += parts[r]
        out.append(total.reshape(t.shape))
    return out


def train_cache_codebooks(engine, x, k, sub, epsilon=0.01, threshold=0.001, max_iterations=100, group=None, log=print):
    """Trains the codebooks of a key or value cache by LBG: the split schedule and stop rule of VQ_Full.py:60-98 for every
    head and part side by side, in squared distance.

    x (tokens, heads, dim): sample vectors on the engine's device, of any of the three float types; this rank's share where
    `group` names a process group.  A split replaces every codeword c by c + e and c - e, e being epsilon times the root
    of its part's mean squared distance per number (the reference scales c, which cannot part codewords near
    zero).  A stage ends once the total distortion changes by less than `threshold` of itself.
    Returns an LBGResult whose codebook is (heads, K, dim) float32, K the next power of two from k; the cache takes it
    rounded to its own dtype."""
    from .lbg import LBGResult
    if not 1 <= k <= 256:
        raise ValueError(f"k={k}: a code is one byte, 1 to 256 codewords")
    if x.dim() != 3:
        raise ValueError(f"x must have shape (tokens, heads, dim), got {tuple(x.shape)}")
    tokens, heads, dim = x.shape
    if sub < 1 or dim % sub:
        raise ValueError(f"vectors of {dim} numbers cannot be cut into sub-vectors of {sub}")

    def iterate(cb):
        part = engine.cache_lbg_accum(x, cb, sub)
        if group is not None:
            part = _added_over_ranks(*part, group)
        new, mean = engine.cache_lbg_finish(*part, cb)
        return new, part[1], mean

    # the one centroid first: the mean of all vectors, then their spread around it
    cb, counts, _ = iterate(torch.zeros((heads, 1, dim), dtype=torch.float32, device=engine.device))
    if int(counts.sum(-1).min().item()) < k:
        raise ValueError(f"Invalid quantization level k={k}: cannot exceed the number of vectors ({int(counts.sum(-1).min().item())}).")
    _, _, mean = iterate(cb)
    iters, conv, distortions = [], [], []
    while cb.shape[1] < k:
        step = (epsilon * (mean / sub).sqrt()).float().repeat_interleave(sub, 1)[:, None]
        cb = torch.cat([cb + step, cb - step], 1)
        prev, done, conv_i = float("inf"), 0, -1
        for i in range(max_iterations):
            cb, _, mean = iterate(cb)
            distortion = float(mean.sum().item())
            distortions.append(distortion)
            done += 1
            if prev != float("inf") and (distortion == prev or abs(prev - distortion) < threshold * prev):
                conv_i = i
                if log is not None:
                    log(f"Converged at iter {i}, distortion={distortion:.3f}")
                break
            prev = distortion
        iters.append(done)
        conv.append(conv_i)
    return LBGResult(cb, iters, conv, distortions)
