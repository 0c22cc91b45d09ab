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
they refuse tensors that require a gradient or carry a tangent.
"""
import math
from types import SimpleNamespace

import torch
from torch.autograd import forward_ad

from ._lib import lib, check, VQ_BF16, VQ_F16, VQ_F32

_DTYPES = {torch.float32: VQ_F32, torch.bfloat16: VQ_BF16, torch.float16: VQ_F16}


# where torch counts its levels of forward-mode derivatives: -1 outside of them all, where no tensor carries a tangent
_levels = forward_ad if hasattr(forward_ad, "_current_level") else SimpleNamespace(_current_level=0)


# ---- checks of arguments: shapes, types and devices only, nothing is read from the GPU.  They run on every call, so what
# is right passes in one expression and only what is not is looked at again for its message. ------------------------------

def _tensor(name, t, device, dtypes, dims):
    if (isinstance(t, torch.Tensor) and t.dtype in dtypes and t.dim() == dims and t.device == device and not t.requires_grad and
            _levels._current_level < 0):
        return t
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
    if t.is_floating_point() and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} carries a tangent: the cache operators are not differentiable")
    return t


def _whole(name, t):
    if not t.is_contiguous() or t.data_ptr() % 16:
        raise ValueError(f"{name} must be contiguous and start at a multiple of 16 bytes")
    return t


def _vectors(t):
    """t as the kernels read it: each vector's numbers side by side from a multiple of 16 bytes.  Anything else is copied."""
    token, head, one = t.stride()
    if one == 1 and (token | head) * t.element_size() % 16 == 0 and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _books(t):
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


_HALVES = (torch.bfloat16, torch.float16)
_BYTES = (torch.uint8,)
_INT32 = (torch.int32,)
_INT64 = (torch.int64,)
_FLOATS = tuple(_DTYPES)
_F32 = (torch.float32,)
_F64 = (torch.float64,)


def cache_shape(k_cb, v_cb, k_codes, v_codes, device):
    """Checks codebooks and code buffers against each other; returns (heads, dim, sub, K, pages, page)."""
    try:
        dtype = k_cb.dtype
        right = (dtype in _HALVES and v_cb.dtype is dtype and k_codes.dtype is torch.uint8 and v_codes.dtype is torch.uint8 and
                 k_cb.device == device and v_cb.device == device and k_codes.device == device and v_codes.device == device and
                 k_cb.dim() == 3 and k_codes.dim() == 4 and not (k_cb.requires_grad or v_cb.requires_grad or _levels._current_level >= 0) and
                 k_codes.is_contiguous() and v_codes.is_contiguous() and not (k_codes.data_ptr() | v_codes.data_ptr()) % 16)
    except AttributeError:
        right = False
    if not right:
        _tensor("k_cb", k_cb, device, _HALVES, 3)
        _tensor("v_cb", v_cb, device, (k_cb.dtype,), 3)
        _whole("k_codes", _tensor("k_codes", k_codes, device, _BYTES, 4))
        _whole("v_codes", _tensor("v_codes", v_codes, device, _BYTES, 4))
    pages, heads, page, parts = k_codes.shape
    books, K, dim = k_cb.shape
    if not (pages and heads and page and parts):
        raise ValueError(f"k_codes must not be empty, got shape {tuple(k_codes.shape)}")
    if v_codes.shape != (pages, heads, parts, page):
        raise ValueError(f"v_codes must have shape {(pages, heads, parts, page)} (k_codes: {tuple(k_codes.shape)}), got {tuple(v_codes.shape)}")
    if k_cb.shape != v_cb.shape or books not in (1, heads) or not (K and dim):
        raise ValueError(f"codebooks must be (1 or {heads}, K, dim) of one shape, got {tuple(k_cb.shape)} and {tuple(v_cb.shape)}")
    if dim % parts:
        raise ValueError(f"vectors of {dim} numbers cannot be cut into the {parts} codes of a cache entry")
    return heads, dim, dim // parts, K, pages, page


def _ints(name, t, dtypes, dims, device):
    if not (isinstance(t, torch.Tensor) and t.dtype in dtypes and t.dim() == dims and t.device == device):
        _tensor(name, t, device, dtypes, dims)
    return t if t.is_contiguous() else t.contiguous()


def _sized(name, t, shape):
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    return t


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

    def _launch(self, name, *args):
        """Calls the library on the engine's device and its current stream."""
        stream = self._stream()
        if torch.cuda.current_device() == self.device.index:
            check(getattr(lib, name)(*args, stream), name)
        else:
            with torch.cuda.device(self.device):
                check(getattr(lib, name)(*args, stream), name)

    def cache_write(self, k, v, slots, k_cb, v_cb, k_codes, v_codes):
        """Quantises k and v (tokens, heads, dim) and stores the codes at slots (tokens, int64); a slot outside the cache
        (-1, say) stores nothing.  Slots should be distinct: of two tokens with one slot, each code is that of either."""
        device = self.device
        heads, dim, sub, K, pages, page = cache_shape(k_cb, v_cb, k_codes, v_codes, device)
        slots = _ints("slots", slots, _INT64, 1, device)
        tokens = slots.shape[0]
        dtypes, shape = (k_cb.dtype,), (tokens, heads, dim)
        _sized("k", _tensor("k", k, device, dtypes, 3), shape)
        _sized("v", _tensor("v", v, device, dtypes, 3), shape)
        if tokens == 0:
            return
        k, v, k_cb, v_cb = _vectors(k), _vectors(v), _books(k_cb), _books(v_cb)
        self._launch("vq_cache_write", k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), slots.data_ptr(),
                     tokens, k_cb.data_ptr(), v_cb.data_ptr(), k_cb.shape[0], heads, dim, sub, K, _DTYPES[k_cb.dtype], k_codes.data_ptr(),
                     v_codes.data_ptr(), pages, page)

    def cache_read(self, slots, k_cb, v_cb, k_codes, v_codes):
        """The keys and values that the codes at slots stand for: two tensors (tokens, heads, dim) of the codebooks'
        dtype.  A slot outside the cache reads as zeros."""
        device = self.device
        heads, dim, sub, K, pages, page = cache_shape(k_cb, v_cb, k_codes, v_codes, device)
        slots = _ints("slots", slots, _INT64, 1, device)
        tokens = slots.shape[0]
        k_cb, v_cb = _books(k_cb), _books(v_cb)
        k = torch.empty(tokens, heads, dim, dtype=k_cb.dtype, device=device)       # (sizes one by one: the shorter way through torch)
        v = torch.empty_like(k)
        if tokens:
            self._launch("vq_cache_read", slots.data_ptr(), tokens, k_cb.data_ptr(), v_cb.data_ptr(), k_cb.shape[0], heads, dim, sub, K,
                         _DTYPES[k_cb.dtype], k_codes.data_ptr(), v_codes.data_ptr(), pages, page, k.data_ptr(), v.data_ptr())
        return k, v

    def cache_attention(self, q, k_cb, v_cb, k_codes, v_codes, table, kv_lens, starts, max_q, max_kv=None, scale=None, out=None,
                        want_lse=False):
        """Causal attention of packed sequences' newest tokens over the cache.

        q (rows, q_heads, dim): sequence b owns rows starts[b] to starts[b + 1] (starts: int32, one more than sequences)
        and the first kv_lens[b] (int32) tokens of the pages table[b] (int32, (sequences, width)); its rows are the newest
        of those tokens, whose keys and values are in the cache already.  Query head h reads cache head
        h // (q_heads / heads).  A row that sees no token gets zeros (and a logarithm of minus infinity); rows of no
        sequence are left as they were in `out`, and are undefined in what the call allocates.  `out` overlaps no other argument.
        max_q, max_kv: the longest of the sequences' rows and lengths, as the host knows them; they shape the launch only
        (max_kv None: what the table can hold).  scale: 1 / sqrt(dim) if None.
        Returns out (rows, q_heads, dim), with want_lse also the natural logarithm of each row's sum of exponentials
        (rows, q_heads) float32, by which results over parts of a context are joined."""
        device = self.device
        heads, dim, sub, K, pages, page = cache_shape(k_cb, v_cb, k_codes, v_codes, device)
        dtype = k_cb.dtype
        _tensor("q", q, device, (dtype,), 3)
        rows, q_heads, q_dim = q.shape
        if q_dim != dim or q_heads == 0 or q_heads % heads:
            raise ValueError(f"q must have shape (rows, a multiple of {heads}, {dim}), got {tuple(q.shape)}")
        kv_lens = _ints("kv_lens", kv_lens, _INT32, 1, device)
        seqs = kv_lens.shape[0]
        starts = _sized("starts", _ints("starts", starts, _INT32, 1, device), (seqs + 1,))
        table = _ints("table", table, _INT32, 2, device)
        width = table.shape[1]
        _sized("table", table, (seqs, width))
        if out is None:
            out = torch.empty_like(q) if q.is_contiguous() else torch.empty(rows, q_heads, dim, dtype=dtype, device=device)
        else:
            _sized("out", _whole("out", _tensor("out", out, device, (dtype,), 3)), (rows, q_heads, dim))
        lse = torch.empty(rows, q_heads, dtype=torch.float32, device=device) if want_lse else None
        if rows and seqs:
            q, k_cb, v_cb = _vectors(q), _books(k_cb), _books(v_cb)
            scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
            max_q = int(max_q)
            max_kv = max(1, width * page) if max_kv is None else int(max_kv)
            need = lib.vq_cache_attention_ws_bytes(rows, q_heads, heads, dim, sub, K, seqs, max_q, max_kv)
            ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
            self._launch("vq_cache_attention", q.data_ptr(), q.stride(0), q.stride(1), rows, q_heads, k_cb.data_ptr(), v_cb.data_ptr(),
                         k_cb.shape[0], heads, dim, sub, K, _DTYPES[dtype], k_codes.data_ptr(), v_codes.data_ptr(), pages, page,
                         table.data_ptr(), seqs, width, kv_lens.data_ptr(), starts.data_ptr(), max_q, max_kv, scale, out.data_ptr(),
                         lse.data_ptr() if want_lse else None, ws.data_ptr() if need else None, need)
        return (out, lse) if want_lse else out

    def _lbg_arguments(self, x, cb, sub):
        device = self.device
        _tensor("cb", cb, device, _F32, 3)
        _tensor("x", x, device, _FLOATS, 3)
        heads, K, dim = cb.shape
        tokens = x.shape[0]
        _sized("x", x, (tokens, heads, dim))
        if not (heads and K and dim) or sub < 1 or dim % sub:
            raise ValueError(f"codebook of shape {tuple(cb.shape)} cannot be cut into sub-vectors of {sub}")
        return tokens, heads, K, dim, dim // sub

    def cache_lbg_accum(self, x, cb, sub):
        """The accumulating half of an LBG iteration of float codebooks cb (heads, K, dim) float32 over the vectors
        x (tokens, heads, dim): for each codeword the sum (heads, K, dim) float64 and number (heads, parts, K) int64 of the
        sub-vectors nearest to it, and the sum of their squared distances (heads, parts) float64.  A sub-vector of
        which a number is 2^100 or more in size, or NaN, is left out.  Shards' results are added."""
        device = self.device
        tokens, heads, K, dim, parts = self._lbg_arguments(x, cb, sub)
        make = torch.empty if tokens else torch.zeros
        sums = make((heads, K, dim), dtype=torch.float64, device=device)
        counts = make((heads, parts, K), dtype=torch.int64, device=device)
        dist = make((heads, parts), dtype=torch.float64, device=device)
        if tokens:
            x, cb = _vectors(x), _books(cb)
            need = lib.vq_cache_lbg_ws_bytes(tokens, heads, dim, sub, K)
            ws = torch.empty(need, dtype=torch.uint8, device=device)
            self._launch("vq_cache_lbg_accum", x.data_ptr(), x.stride(0), x.stride(1), tokens, cb.data_ptr(), heads, dim, sub, K, _DTYPES[x.dtype],
                         sums.data_ptr(), counts.data_ptr(), dist.data_ptr(), ws.data_ptr(), need)
        return sums, counts, dist

    def cache_lbg_finish(self, sums, counts, dist, cb):
        """The closing half: (new codebook, mean squared distance (heads, parts)); a codeword without members stays."""
        device = self.device
        _tensor("cb", cb, device, _F32, 3)
        heads, K, dim = cb.shape
        _tensor("dist", dist, device, _F64, 2)
        parts = dist.shape[1]
        _tensor("sums", sums, device, _F64, 3)
        _tensor("counts", counts, device, _INT64, 3)
        if not (heads and K and dim) or parts < 1 or dim % parts or dist.shape[0] != heads or sums.shape != cb.shape or \
                counts.shape != (heads, parts, K):
            raise ValueError(f"shapes do not belong together: sums {tuple(sums.shape)}, counts {tuple(counts.shape)}, dist {tuple(dist.shape)}, "
                             f"cb {tuple(cb.shape)}")
        sums, counts, dist, cb = (t.contiguous() for t in (sums, counts, dist, cb))
        new, mean = torch.empty_like(cb), torch.empty_like(dist)
        self._launch("vq_cache_lbg_finish", sums.data_ptr(), counts.data_ptr(), dist.data_ptr(), cb.data_ptr(), heads, dim, dim // parts, K,
                     new.data_ptr(), mean.data_ptr())
        return new, mean

    def cache_lbg_iterate(self, x, cb, sub):
        """One LBG iteration of the float codebooks cb (heads, K, dim) float32 over the vectors x (tokens, heads, dim): both
        halves in one.  Returns (new codebook, members (heads, parts, K), mean squared distance to the old codewords
        (heads, parts))."""
        device = self.device
        tokens, heads, K, dim, parts = self._lbg_arguments(x, cb, sub)
        if tokens == 0:
            sums, counts, dist = self.cache_lbg_accum(x, cb, sub)
            new, mean = self.cache_lbg_finish(sums, counts, dist, cb)
            return new, counts, mean
        x, cb = _vectors(x), _books(cb)
        new = torch.empty(heads, K, dim, dtype=torch.float32, device=device)
        counts = torch.empty(heads, parts, K, dtype=torch.int64, device=device)
        mean = torch.empty(heads, parts, dtype=torch.float64, device=device)
        need = lib.vq_cache_lbg_ws_bytes(tokens, heads, dim, sub, K)
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        self._launch("vq_cache_lbg_iterate", x.data_ptr(), x.stride(0), x.stride(1), tokens, cb.data_ptr(), heads, dim, sub, K, _DTYPES[x.dtype],
                     new.data_ptr(), counts.data_ptr(), mean.data_ptr(), ws.data_ptr(), need)
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
    `group` names a process group, whose results are added between the two halves of an iteration; a process by itself runs
    both in one (cache_lbg_iterate), with the same bits.  A split replaces every codeword c by c + e and c - e, e being epsilon times the root
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

    whole = getattr(engine, "cache_lbg_iterate", None) if group is None else None     # (an engine may have the halves alone)

    def iterate(cb):
        if whole is not None:
            return whole(x, cb, sub)
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
