"""The cache operators' checks of arguments: they come before any GPU work, so they run on a CPU-only machine."""
import contextlib
import ctypes
import os
import re

import pytest
import torch

from vector_quantization_amd import _lib, train_cache_codebooks
from vector_quantization_amd.cache import CacheOps

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = ctypes.c_void_p(4096)


class CpuEngine(CacheOps):
    """The methods on host tensors; a call that gets as far as the library is reported."""
    device = torch.device("cpu")

    def _stream(self):
        raise AssertionError("reached the launch")


@pytest.fixture
def eng(monkeypatch):
    monkeypatch.setattr(torch.cuda, "device", lambda *_a: contextlib.nullcontext())
    return CpuEngine()


def test_header_binding_and_exports_agree():
    text = open(os.path.join(ROOT, "include", "vq_cache.h")).read()
    names = sorted(set(re.findall(r"\b(vq_cache_[a-z0-9_]+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S))))
    assert names == sorted(_lib.CACHE_SIGNATURES)
    lib = ctypes.CDLL(_lib.library_path())
    for name in names:
        assert hasattr(lib, name)
    assert not hasattr(lib, "vq_internal_fail")


def write(**kw):
    a = dict(k=P, kt=1024, kh=128, v=P, vt=1024, vh=128, slots=P, tokens=4, k_cb=P, v_cb=P, cb_heads=8, heads=8, dim=128, sub=4, K=256,
             dtype=_lib.VQ_BF16, kc=P, vc=P, pages=4, page=16)
    a.update(kw)
    return _lib.lib.vq_cache_write(*a.values(), None)


@pytest.mark.parametrize("kw,rc,text", [
    (dict(dim=80), _lib.VQ_E_UNSUPPORTED, "dim=80"), (dict(sub=3), _lib.VQ_E_UNSUPPORTED, "sub=3"), (dict(K=257), _lib.VQ_E_UNSUPPORTED, "K=257"),
    (dict(K=0), _lib.VQ_E_UNSUPPORTED, "K=0"), (dict(heads=0), _lib.VQ_E_INVALID, "heads"), (dict(heads=2000, cb_heads=1), _lib.VQ_E_UNSUPPORTED, "heads"),
    (dict(cb_heads=3), _lib.VQ_E_INVALID, "cb_heads=3"), (dict(page=24), _lib.VQ_E_UNSUPPORTED, "page=24"), (dict(page=0), _lib.VQ_E_INVALID, "page"),
    (dict(pages=0), _lib.VQ_E_INVALID, "pages"), (dict(pages=1 << 31), _lib.VQ_E_INVALID, "pages"), (dict(dtype=_lib.VQ_F32), _lib.VQ_E_UNSUPPORTED, "VQ_BF16"),
    (dict(dtype=9), _lib.VQ_E_UNSUPPORTED, "VQ_BF16"), (dict(k=None), _lib.VQ_E_INVALID, "null"), (dict(slots=None), _lib.VQ_E_INVALID, "null"),
    (dict(kc=None), _lib.VQ_E_INVALID, "null"), (dict(vc=ctypes.c_void_p(4104)), _lib.VQ_E_INVALID, "16 bytes"), (dict(tokens=-1), _lib.VQ_E_INVALID, "tokens"),
    (dict(kt=1025), _lib.VQ_E_INVALID, "vectors of k"), (dict(vh=12), _lib.VQ_E_INVALID, "vectors of v"), (dict(v=ctypes.c_void_p(4098)), _lib.VQ_E_INVALID, "vectors of v"),
])
def test_write_refuses(kw, rc, text):
    assert write(**kw) == rc and text in _lib.last_error()


def test_write_of_nothing_is_fine():
    assert write(tokens=0, k=None, v=None, slots=None) == _lib.VQ_OK


def test_read_refuses():
    f = _lib.lib.vq_cache_read
    ok = [P, 4, P, P, 8, 8, 128, 4, 256, _lib.VQ_F16, P, P, 4, 16, P, P]
    for at, value, rc in ((0, None, _lib.VQ_E_INVALID), (1, -1, _lib.VQ_E_INVALID), (6, 100, _lib.VQ_E_UNSUPPORTED), (9, 0, _lib.VQ_E_UNSUPPORTED),
                          (14, None, _lib.VQ_E_INVALID), (15, ctypes.c_void_p(4100), _lib.VQ_E_INVALID), (13, 8, _lib.VQ_E_UNSUPPORTED)):
        args = list(ok)
        args[at] = value
        assert f(*args, None) == rc


def attend(**kw):
    a = dict(q=P, qt=4096, qh=128, rows=10, q_heads=32, k_cb=P, v_cb=P, cb_heads=8, heads=8, dim=128, sub=4, K=256, dtype=_lib.VQ_BF16, kc=P, vc=P,
             pages=4, page=16, table=P, seqs=2, width=4, kv_lens=P, starts=P, max_q=1, max_kv=64, scale=0.1, out=P, lse=P, ws=P, ws_bytes=1 << 40)
    a.update(kw)
    return _lib.lib.vq_cache_attention(*a.values(), None)


@pytest.mark.parametrize("kw,rc,text", [
    (dict(q_heads=12), _lib.VQ_E_INVALID, "q_heads=12"), (dict(q_heads=0), _lib.VQ_E_INVALID, "q_heads"), (dict(q_heads=8192), _lib.VQ_E_UNSUPPORTED, "q_heads"),
    (dict(rows=-1), _lib.VQ_E_INVALID, "rows"), (dict(rows=1 << 31), _lib.VQ_E_UNSUPPORTED, "2^31"), (dict(width=1 << 28), _lib.VQ_E_UNSUPPORTED, "2^31"),
    (dict(max_q=0), _lib.VQ_E_INVALID, "max_q"), (dict(max_kv=0), _lib.VQ_E_INVALID, "max_kv"), (dict(scale=float("nan")), _lib.VQ_E_INVALID, "scale"),
    (dict(scale=float("inf")), _lib.VQ_E_INVALID, "scale"), (dict(seqs=70000), _lib.VQ_E_UNSUPPORTED, "seqs"), (dict(table=None), _lib.VQ_E_INVALID, "null"),
    (dict(kv_lens=None), _lib.VQ_E_INVALID, "null"), (dict(starts=None), _lib.VQ_E_INVALID, "null"), (dict(q=None), _lib.VQ_E_INVALID, "null"),
    (dict(out=None), _lib.VQ_E_INVALID, "null"), (dict(qt=4097), _lib.VQ_E_INVALID, "vectors of q"), (dict(dim=48), _lib.VQ_E_UNSUPPORTED, "dim=48"),
    (dict(dtype=_lib.VQ_F32), _lib.VQ_E_UNSUPPORTED, "VQ_BF16"), (dict(page=40), _lib.VQ_E_UNSUPPORTED, "page=40"),
])
def test_attention_refuses(kw, rc, text):
    assert attend(**kw) == rc and text in _lib.last_error()


def test_attention_refuses_a_small_workspace():
    need = _lib.lib.vq_cache_attention_ws_bytes(1, 32, 8, 128, 4, 256, 1, 1, 1 << 16)
    if need:
        assert attend(rows=1, seqs=1, max_kv=1 << 16, ws_bytes=need - 1) == _lib.VQ_E_WORKSPACE
        assert attend(rows=1, seqs=1, max_kv=1 << 16, ws=None) == _lib.VQ_E_WORKSPACE


def test_lbg_refuses():
    lib = _lib.lib
    need = lib.vq_cache_lbg_ws_bytes(100, 2, 64, 4, 16)
    assert need > 0 and lib.vq_cache_lbg_ws_bytes(0, 2, 64, 4, 16) == 0
    ok = [P, 128, 64, 100, P, 2, 64, 4, 16, _lib.VQ_F32, P, P, P, P, need]
    for at, value, rc in ((0, None, _lib.VQ_E_INVALID), (1, 130, _lib.VQ_E_INVALID), (3, 0, _lib.VQ_E_INVALID), (3, 1 << 31, _lib.VQ_E_UNSUPPORTED), (4, None, _lib.VQ_E_INVALID),
                          (6, 65, _lib.VQ_E_UNSUPPORTED), (9, 7, _lib.VQ_E_UNSUPPORTED), (10, None, _lib.VQ_E_INVALID), (13, None, _lib.VQ_E_WORKSPACE),
                          (14, need - 1, _lib.VQ_E_WORKSPACE), (13, ctypes.c_void_p(4100), _lib.VQ_E_INVALID)):
        args = list(ok)
        args[at] = value
        assert lib.vq_cache_lbg_accum(*args, None) == rc, at
    assert lib.vq_cache_lbg_finish(P, P, None, P, 2, 64, 4, 16, P, P, None) == _lib.VQ_E_INVALID


def parts(dtype=torch.bfloat16, heads=2, dim=64, sub=4, K=16, pages=3, page=32):
    return [torch.zeros((heads, K, dim), dtype=dtype), torch.zeros((heads, K, dim), dtype=dtype),
            torch.zeros((pages, heads, page, dim // sub), dtype=torch.uint8), torch.zeros((pages, heads, dim // sub, page), dtype=torch.uint8)]


def test_engine_refuses_what_does_not_fit(eng):
    k_cb, v_cb, kc, vc = parts()
    x, slots = torch.zeros((5, 2, 64), dtype=torch.bfloat16), torch.zeros(5, dtype=torch.int64)
    for bad in ((x[:4], x, slots), (x, x[:, :1], slots), (x, x.float(), slots), (x, x[..., :32], slots), (x, x, slots.int()), (x, x, slots[None]), (x[0], x, slots)):
        with pytest.raises(ValueError):
            eng.cache_write(*bad, k_cb, v_cb, kc, vc)
    for bad in ((k_cb, v_cb[:, :8], kc, vc), (k_cb.float(), v_cb.float(), kc, vc), (k_cb, v_cb.half(), kc, vc), (k_cb, v_cb, kc, kc), (k_cb, v_cb, kc.int(), vc),
                (k_cb, v_cb, kc.transpose(1, 2), vc), (k_cb, v_cb, kc[:0], vc[:0]), (k_cb[..., :60], v_cb[..., :60], kc, vc), (k_cb[:0], v_cb[:0], kc, vc)):
        with pytest.raises(ValueError):
            eng.cache_write(x, x, slots, *bad)
        with pytest.raises(ValueError):
            eng.cache_read(slots, *bad)
    with pytest.raises(TypeError):
        eng.cache_write(x, x, [1, 2], k_cb, v_cb, kc, vc)
    with pytest.raises(ValueError, match="is on meta"):
        eng.cache_write(x.to("meta"), x, slots, k_cb, v_cb, kc, vc)
    with pytest.raises(ValueError, match="not differentiable"):
        eng.cache_write(x.clone().requires_grad_(), x, slots, k_cb, v_cb, kc, vc)
    with pytest.raises(ValueError):
        eng.cache_buffers(4, 24, 2, 64, 4)
    for t in eng.cache_buffers(4, 16, 2, 64, 4):
        assert not t.any()
    with pytest.raises(AssertionError, match="reached the launch"):
        eng.cache_write(x, x, slots, k_cb, v_cb, kc, vc)


def test_engine_attention_refuses_what_does_not_fit(eng):
    books = parts()
    q = torch.zeros((5, 4, 64), dtype=torch.bfloat16)
    table, lens, starts = torch.zeros((2, 3), dtype=torch.int32), torch.ones(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for bad in ((q[:, :3], table, lens, starts), (q[..., :32], table, lens, starts), (q.half(), table, lens, starts), (q, table[:1], lens, starts),
                (q, table, lens.long(), starts), (q, table, lens, starts[:2]), (q, table.long(), lens, starts), (q[0], table, lens, starts)):
        with pytest.raises(ValueError):
            eng.cache_attention(bad[0], *books, *bad[1:], 3)
    with pytest.raises(ValueError, match="out must"):
        eng.cache_attention(q, *books, table, lens, starts, 3, out=torch.zeros((4, 4, 64), dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="contiguous"):
        eng.cache_attention(q, *books, table, lens, starts, 3, out=torch.zeros((4, 5, 64), dtype=torch.bfloat16).transpose(0, 1))
    with pytest.raises(AssertionError, match="reached the launch"):
        eng.cache_attention(q, *books, table, lens, starts, 3)


def test_engine_lbg_refuses_what_does_not_fit(eng):
    x, cb = torch.zeros((9, 2, 64)), torch.zeros((2, 16, 64))
    for bad in ((x.double(), cb, 4), (x, cb.half(), 4), (x[:, :1], cb, 4), (x, cb, 5), (x, cb, 0), (x[0], cb, 4), (x, cb[:, :0], 4)):
        with pytest.raises(ValueError):
            eng.cache_lbg_accum(*bad)
    sums, counts, dist = eng.cache_lbg_accum(x[:0], cb, 4)
    assert sums.shape == cb.shape and counts.shape == (2, 16, 16) and dist.shape == (2, 16) and not sums.any()
    for bad in ((sums[:1], counts, dist, cb), (sums, counts[:, :8], dist, cb), (sums, counts, dist[:, :5], cb), (sums.float(), counts, dist, cb)):
        with pytest.raises(ValueError):
            eng.cache_lbg_finish(*bad)
    with pytest.raises(ValueError, match="k=300"):
        train_cache_codebooks(eng, x, 300, 4)
    with pytest.raises(ValueError, match="cut into"):
        train_cache_codebooks(eng, x, 4, 5)


# ---- training over several processes ---------------------------------------------------------------------------------

class HostEngine:
    """cache_lbg_accum / cache_lbg_finish by their definitions, on the host."""
    device = torch.device("cpu")

    def cache_lbg_accum(self, x, cb, sub):
        T, H, D = x.shape
        K, M = cb.shape[1], D // sub
        xs, cs = x.double().reshape(T, H, M, sub), cb.double().reshape(H, K, M, sub)
        d = (xs[:, :, None] - cs[None]).square().sum(-1)                  # (T, H, K, M)
        least, code = d.min(2)
        hot = torch.nn.functional.one_hot(code, K).double()                # (T, H, M, K)
        sums = torch.einsum("thmk,thme->hkme", hot, xs).reshape(H, K, D)
        return sums, hot.sum(0).long(), least.sum(0)

    def cache_lbg_finish(self, sums, counts, dist, cb):
        H, K, D = cb.shape
        M = counts.shape[1]
        n = counts.permute(0, 2, 1).repeat_interleave(D // M, 2).double()
        return torch.where(n > 0, sums / n.clamp(min=1), cb.double()).float(), dist / counts.sum(-1).clamp(min=1)


def clouds():
    g = torch.Generator().manual_seed(1)
    return torch.randn((301, 2, 16), generator=g) + 4 * torch.randint(-1, 2, (301, 2, 16), generator=g)


def _rank(rank, world, port, out):
    import torch.distributed as dist
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=world)
    x = clouds()
    mine = x[:113] if rank == 0 else x[113:]
    res = train_cache_codebooks(HostEngine(), mine, 8, 4, group=dist.group.WORLD, log=None)
    torch.save((res.codebook, res.iters_per_stage, res.distortions), f"{out}/{rank}.pt")
    dist.destroy_process_group()


def test_training_over_two_processes(tmp_path):
    """Shards of unequal size train what one process trains on all vectors; both ranks end with the same bits."""
    import socket
    import torch.multiprocessing as mp
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.start_processes(_rank, args=(2, port, str(tmp_path)), nprocs=2, start_method="spawn")
    (cb0, it0, d0), (cb1, it1, d1) = (torch.load(tmp_path / f"{r}.pt", weights_only=True) for r in range(2))
    one = train_cache_codebooks(HostEngine(), clouds(), 8, 4, log=None)
    assert torch.equal(cb0, cb1) and it0 == it1 and d0 == d1
    assert it0 == one.iters_per_stage and len(one.distortions) == sum(it0)
    assert one.codebook.shape == (2, 8, 16)
    # sums of 301 numbers in fp64 in two orders: the same to 301 * 2^-53 of their size, then one rounding to fp32 and its like in each iteration
    assert (cb0 - one.codebook).abs().max() <= 2.0 ** -22 * one.codebook.abs().max()
    assert one.distortions[-1] < one.distortions[0]


def test_training_log_and_stop_rule():
    lines = []
    res = train_cache_codebooks(HostEngine(), clouds(), 4, 4, log=lines.append)
    assert len(lines) == 2 and all(line.startswith("Converged at iter") for line in lines)
    assert res.converged_iter == [n - 1 for n in res.iters_per_stage]
    short = train_cache_codebooks(HostEngine(), clouds(), 4, 4, log=None, max_iterations=1)
    assert short.iters_per_stage == [1, 1] and short.converged_iter == [-1, -1]
    flat = train_cache_codebooks(HostEngine(), torch.ones(9, 1, 16), 4, 4, log=None)      # no spread: nothing to part, nothing diverges
    assert torch.equal(flat.codebook, torch.ones(1, 4, 16)) and flat.distortions[-1] == 0.0


def test_training_by_whole_iterations():
    """An engine that runs an iteration in one call is trained by it, and by the halves where a group's results are added."""
    class Whole(HostEngine):
        calls = 0

        def cache_lbg_iterate(self, x, cb, sub):
            self.calls += 1
            part = HostEngine.cache_lbg_accum(self, x, cb, sub)
            new, mean = HostEngine.cache_lbg_finish(self, *part, cb)
            return new, part[1], mean

        def cache_lbg_accum(self, *_a):
            raise AssertionError("the halves were called")

    eng = Whole()
    one, halves = (train_cache_codebooks(e, clouds(), 8, 4, log=None) for e in (eng, HostEngine()))
    assert torch.equal(one.codebook, halves.codebook) and one.distortions == halves.distortions
    assert eng.calls == 2 + sum(one.iters_per_stage)
    with pytest.raises(ValueError, match="cannot exceed"):
        train_cache_codebooks(eng, clouds()[:4], 8, 4, log=None)


def test_tangents_are_refused(eng):
    """Forward-mode derivatives would be lost without a word; tensors without one pass also where others may carry one."""
    from torch.autograd import forward_ad
    k_cb, v_cb, kc, vc = parts()
    x, slots = torch.zeros((5, 2, 64), dtype=torch.bfloat16), torch.zeros(5, dtype=torch.int64)
    table, lens, starts = torch.zeros((2, 3), dtype=torch.int32), torch.ones(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    f, cb = torch.zeros((9, 2, 64)), torch.zeros((2, 16, 64))
    sums, counts, dist = eng.cache_lbg_accum(f[:0], cb, 4)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: eng.cache_write(dual(x), x, slots, k_cb, v_cb, kc, vc), lambda: eng.cache_write(x, dual(x), slots, k_cb, v_cb, kc, vc),
                     lambda: eng.cache_write(x, x, slots, dual(k_cb), v_cb, kc, vc), lambda: eng.cache_read(slots, k_cb, dual(v_cb), kc, vc),
                     lambda: eng.cache_attention(dual(x), k_cb, v_cb, kc, vc, table, lens, starts, 3),
                     lambda: eng.cache_attention(x, k_cb, v_cb, kc, vc, table, lens, starts, 3, out=dual(x)),
                     lambda: eng.cache_lbg_accum(dual(f), cb, 4), lambda: eng.cache_lbg_iterate(f, dual(cb), 4),
                     lambda: eng.cache_lbg_finish(dual(sums), counts, dist, cb), lambda: eng.cache_lbg_finish(sums, counts, dual(dist), cb)):
            with pytest.raises(ValueError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                call()
        with pytest.raises(AssertionError, match="reached the launch"):
            eng.cache_write(x, x, slots, k_cb, v_cb, kc, vc)
        with torch.no_grad(), pytest.raises(AssertionError, match="reached the launch"):
            eng.cache_write(x.clone().requires_grad_(), x, slots, k_cb, v_cb, kc, vc)


@pytest.mark.parametrize("seqs,max_q,max_kv,dim,sub,K", [(1, 1, 1 << 16, 128, 4, 256), (16, 1, 20000, 64, 8, 200), (1, 2048, 16384, 256, 2, 256), (3, 40, 5000, 192, 4, 64)])
def test_attention_workspace_is_asked_for_and_checked(seqs, max_q, max_kv, dim, sub, K):
    """Where a head's work is cut there has to be a workspace, of the size that is named and in its place."""
    kw = dict(rows=seqs * max_q, seqs=seqs, max_q=max_q, max_kv=max_kv, dim=dim, sub=sub, K=K, qt=32 * dim, qh=dim)
    need = _lib.lib.vq_cache_attention_ws_bytes(seqs * max_q, 32, 8, dim, sub, K, seqs, max_q, max_kv)
    assert need > 0
    assert attend(**kw, ws_bytes=need - 1) == _lib.VQ_E_WORKSPACE and str(need) in _lib.last_error()
    assert attend(**kw, ws=None) == _lib.VQ_E_WORKSPACE
    assert attend(**kw, ws=ctypes.c_void_p(4100), ws_bytes=need) == _lib.VQ_E_INVALID and "16 bytes" in _lib.last_error()
    assert _lib.lib.vq_cache_attention_ws_bytes(1, 32, 8, dim, sub, K, 1, 1, 64) == 0      # a short sequence is not cut
