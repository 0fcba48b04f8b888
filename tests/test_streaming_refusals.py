"""Argument checks of the masked and paged attention and of the cache that need no GPU, the key intervals of the masks, and
the oracle of the cache."""
from __future__ import annotations

import ctypes
import importlib

import numpy as np
import pytest
import torch


def test_masked_attention_refusals(pkg):
    q = torch.zeros(1, 4, 3, 64)
    k = torch.zeros(1, 2, 5, 64)
    f = pkg.masked_attention
    with pytest.raises(ValueError, match="head_dim=64"):
        f(q[..., :32], k[..., :32], k[..., :32])
    with pytest.raises(ValueError, match="batch, heads"):
        f(q[0], k, k)
    with pytest.raises(ValueError, match="incompatible"):
        f(q, torch.zeros(1, 3, 5, 64), torch.zeros(1, 3, 5, 64))
    with pytest.raises(ValueError, match="incompatible"):
        f(q, k, k[:, :, :4])
    with pytest.raises(ValueError, match="one dtype"):
        f(q, k.half(), k.half())
    with pytest.raises(ValueError, match="unsupported dtype"):
        f(q.double(), k.double(), k.double())
    for cap in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="softcap"):
            f(q, k, k, softcap=cap)
    for scale in (0.0, -0.1, float("inf")):
        with pytest.raises(ValueError, match="scale"):
            f(q, k, k, scale=scale)
    with pytest.raises(ValueError, match="distance_slope"):
        f(q, k, k, distance_slope=torch.zeros(2))
    with pytest.raises(ValueError, match="positions are used"):
        f(q, k, k, key_position=torch.zeros(5))
    with pytest.raises(ValueError, match="key_range"):
        f(q, k, k, key_range=torch.zeros(3, 2))
    with pytest.raises(ValueError, match="key_range"):
        f(q, k, k, key_range=torch.zeros(2, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="out must"):
        f(q, k, k, out=torch.zeros(1, 4, 2, 64))
    with pytest.raises(RuntimeError, match="CUDA"):
        f(q, k, k)


def test_cache_refusals(pkg):
    with pytest.raises(RuntimeError, match="CUDA"):
        pkg.PagedCache.empty(1, 4, 4, device="cpu")
    with pytest.raises(ValueError, match="pages hold"):
        pkg.PagedCache.empty(1, 4, 4, page_size=48, device="cpu")
    with pytest.raises(ValueError, match="at least 1"):
        pkg.PagedCache.empty(0, 4, 4, device="cpu")
    k = torch.zeros(4, 16, 2, 64)
    ints = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    make = pkg.PagedCache
    with pytest.raises(ValueError, match="cache pools"):
        make(torch.zeros(4, 24, 2, 64), k, None, ints(1, 2), ints(1), ints(4))
    with pytest.raises(ValueError, match="one shape"):
        make(k, k.half(), None, ints(1, 2), ints(1), ints(4))
    with pytest.raises(ValueError, match="log_mass"):
        make(k, k, torch.zeros(4, 8), ints(1, 2), ints(1), ints(4))
    with pytest.raises(ValueError, match="table"):
        make(k, k, None, ints(1, 2), ints(2), ints(4))
    with pytest.raises(ValueError, match="int32"):
        make(k, k, None, ints(1, 2).long(), ints(1), ints(4))
    with pytest.raises(ValueError, match="contiguous"):
        make(k, torch.zeros(4, 16, 64, 2).transpose(2, 3), None, ints(1, 2), ints(1), ints(4))


def test_c_entry_points_refuse_bad_arguments(pkg):
    lib, C = pkg.load_library(), pkg._clib
    s = (ctypes.c_int64 * 3)(64, 64, 64)
    mods = C.ScoreMods(scale=0.125)
    dense = lambda dt=1, q=16, B=1, H=4, Hkv=2, Nq=3, Nk=5, D=64, st=s, m=mods: lib.vb200_masked_attention(  # noqa: E731
        dt, q, 16, 16, 16, B, H, Hkv, Nq, Nk, D, st, s, s, s, m, None, 0, None)
    for kw, word in ((dict(dt=7), b"dtype"), (dict(D=32), b"head_dim"), (dict(Hkv=3), b"sizes"), (dict(Nk=0), b"sizes"),
                     (dict(Nk=1 << 31), b"range"), (dict(q=None), b"null"), (dict(q=8), b"aligned"),
                     (dict(st=(ctypes.c_int64 * 3)(64, 64, 60)), b"aligned"), (dict(m=C.ScoreMods(scale=float("nan"))), b"scale"),
                     (dict(m=C.ScoreMods(scale=1.0, softcap=-1.0)), b"softcap"), (dict(m=None), b"mods")):
        assert dense(**kw) == C.EINVAL and word in lib.vb200_last_error(), (kw, lib.vb200_last_error())
    assert dense(Nq=0) == 0
    cache = lambda **k: C.CacheHandle(**dict(dict(k=16, v=16, table=16, length=16, references=16, pages=4, page_size=16,  # noqa: E731
                                                  kv_heads=2, slots=2, max_pages=4), **k))
    two = (ctypes.c_int64 * 2)(64, 64)
    paged = lambda c, H=4, rows=2, n=1, q=16, seq=16: lib.vb200_paged_attention(1, q, 16, rows, H, 64, two, two, c, seq, 16, n, 1,  # noqa: E731
                                                                               mods, None, 0, None)
    for c, kw, word in ((cache(page_size=24), {}, b"pages of"), (cache(), dict(H=3), b"multiple"), (cache(pages=0), {}, b"range"),
                        (cache(k=None), {}, b"null"), (cache(), dict(q=None), b"null"), (cache(), dict(n=3, seq=None), b"slots"),
                        (cache(k=24), {}, b"aligned")):
        assert paged(c, **kw) == C.EINVAL and word in lib.vb200_last_error(), (kw, lib.vb200_last_error())
    assert paged(cache(), n=0) == 0 and paged(cache(), rows=0) == 0
    size = lib.vb200_cache_append_workspace_size(1, 2, 4)
    app = lambda c, ws=16, size=size, mass=None, k=16: lib.vb200_cache_append(c, 1, 16, 16, 1, k, 16, mass, 2, two, two, ws, size, None)  # noqa: E731
    for c, kw, word in ((cache(page_size=8), {}, b"pages of"), (cache(), dict(size=16), b"workspace"), (cache(), dict(mass=16), b"log-mass"),
                        (cache(), dict(k=24), b"aligned"), (cache(references=None), {}, b"null")):
        assert app(c, **kw) == C.EINVAL and word in lib.vb200_last_error(), (kw, lib.vb200_last_error())
    assert lib.vb200_cache_fork(cache(), 1, 16, None, 1, 16, 1 << 20, None) == C.EINVAL
    assert lib.vb200_cache_fork(cache(), 1, 16, 16, 1, 16, 4, None) == C.EINVAL
    assert lib.vb200_cache_free(cache(), 1, None, 1, None) == C.EINVAL
    assert lib.vb200_cache_compact(cache(), 1, None, 16, 1 << 20, None) == C.EINVAL
    assert lib.vb200_cache_compact(cache(), 1, 16, 16, 4, None) == C.EINVAL


def test_attention_ranges(pkg):
    f = pkg.attention_ranges
    assert f(3).tolist() == [[0, 3]] * 3 and f(0).shape == (0, 2)
    assert f(2, 4, step=1).tolist() == [[0, 3], [0, 4]]
    assert f(5, step=2).tolist() == [[0, 2], [0, 2], [0, 4], [0, 4], [0, 5]]
    docs = torch.tensor([0, 2, 2, 5])
    assert f(5, documents=docs).tolist() == [[0, 2], [0, 2], [2, 5], [2, 5], [2, 5]]
    assert f(5, documents=docs, step=1, prefix=2).tolist() == [[0, 2], [0, 2], [2, 4], [2, 4], [2, 5]]
    assert f(4, step=1, window=2).tolist() == [[0, 1], [0, 2], [1, 3], [2, 4]]
    assert f(4, documents=torch.tensor([0, 2, 4]), window=1).tolist() == [[0, 2], [1, 2], [2, 4], [3, 4]]
    for bad in (dict(keys=1), dict(step=0), dict(window=0), dict(prefix=-1), dict(documents=torch.tensor([0])),
                dict(documents=torch.zeros(3))):
        with pytest.raises(ValueError):
            f(2, **bad)


def test_oracle_against_plain_softmax(oracle):
    rng = np.random.default_rng(0)
    q, k, v = rng.standard_normal((3, 1, 2, 6, 64))
    out, _ = oracle.streaming.masked_attention(q, k, v)
    ref = torch.softmax(torch.from_numpy(q @ k.swapaxes(-1, -2) / 8), -1).numpy() @ v
    assert np.abs(out - ref).max() < 1e-12


def test_oracle_cache_keeps_tokens(oracle):
    """Appends, forks and compactions leave every slot's tokens what was written, and the references what the tables hold."""
    rng = np.random.default_rng(1)
    c = oracle.streaming.Cache(np.zeros((20, 4, 1, 2)), np.zeros((20, 4, 1, 2)), np.zeros((20, 4)), np.full((3, 10), -1), [0] * 3, [0] * 20)
    want = {0: [], 1: [], 2: []}
    for _ in range(200):
        what = rng.integers(4)
        a, b = rng.integers(0, 3, 2)
        if what == 0:
            n = int(rng.integers(1, 6))
            x = rng.standard_normal((n, 1, 2))
            if c.append([a], [0, n], x, -x, x[:, 0, 0]):
                want[a] = want[a] + list(x)
        elif what == 1:
            c.fork([a], [b])
            want[b] = list(want[a])
        elif what == 2:
            c.free([a])
            want[a] = []
        else:
            used = c.compact()
            assert used == sum(r > 0 for r in c.refs) and all(r == 0 for r in c.refs[used:])
        for s in range(3):
            k, v, m = c.tokens(s)
            assert len(k) == len(want[s]) and all((x == y).all() for x, y in zip(k, want[s])) and (v == -k).all()
        count = np.bincount([p for row in c.held for p in row], minlength=20)
        assert count.tolist() == c.refs


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_oracle_bound_is_narrow(oracle, dtype):
    """Over long keys the bound stays a few roundings of the output: values that are missing from it, one tile's of 127 keys, are
    outside."""
    rng = np.random.default_rng(2)
    n = 8000
    q, k = rng.standard_normal((1, 1, 3, 64)), rng.standard_normal((1, 1, n, 64))
    v = np.abs(rng.standard_normal((1, 1, n, 64)))
    out, bound = oracle.streaming.masked_attention(q, k, v, dtype=dtype)
    assert (bound < 3 * 2 * oracle.streaming.EPS_HALF[dtype] * out).all()
    less = v.copy()
    less[:, :, :127] = 0
    lost, _ = oracle.streaming.masked_attention(q, k, less, dtype=dtype)
    assert (np.abs(lost - out) > bound).all()
    bias = np.full(n, -14.0)
    bias[9] = 12.0
    v[0, 0, 9] = 0  # the output is what keys 26 nats below the top add up to
    out, bound = oracle.streaming.masked_attention(q, k, v, bias, dtype=dtype)
    # at most two roundings of the whole, the result's step, and what the other roundings take as above
    assert (bound <= (2 + 3 * 2 * oracle.streaming.EPS_HALF[dtype]) * out + 2.0 ** -25).all()


def _bytes(t):
    at = torch.zeros(1, dtype=torch.int64) + t.data_ptr()
    for s, n in zip(t.stride(), t.shape):
        at = (at[:, None] + s * t.element_size() * torch.arange(n)).flatten()
    return {int(x) + i for x in at for i in range(t.element_size())}


def test_shared_memory_is_seen(pkg):
    """Against the sets of bytes, over views of one buffer."""
    share = importlib.import_module(pkg.__name__ + ".streaming")._share_memory
    rng = np.random.default_rng(7)
    base = torch.zeros(600, dtype=torch.bfloat16)
    found = 0
    for _ in range(600):
        views = []
        for _ in range(2):
            while True:
                shape, stride = rng.integers(1, 5, 3).tolist(), rng.choice([0, 1, 2, 4, 7, 8, 16, 24, 48], 3).tolist()
                first, last = int(rng.integers(0, 120)), sum(s * (n - 1) for s, n in zip(stride, shape))
                if first + last < 600:
                    break
            views.append(base.as_strided(shape, stride, first))
        want = bool(_bytes(views[0]) & _bytes(views[1]))
        assert share(*views) == want, [(v.shape, v.stride(), v.storage_offset()) for v in views]
        found += want
    assert 100 < found < 500


def test_outputs_that_share_memory(pkg):
    """Refused where an output has a byte of an input, taken where views of one buffer lie side by side."""
    f = pkg.masked_attention
    buf = torch.zeros(1, 9, 4, 2, 64)  # tokens of q | k | v | out
    q, k, v, out = (buf[:, :, i].transpose(1, 2) for i in range(4))
    heads = torch.zeros(1, 8, 9, 64)   # heads of q | k | v | out
    tokens = torch.zeros(1, 2, 36, 64)  # every head: tokens of q | k | v | out
    for x in ((q, k, v, out), heads.chunk(4, 1), tokens.chunk(4, 2)):
        with pytest.raises(RuntimeError, match="CUDA"):  # as far as a call comes without one
            f(*x[:3], out=x[3])
        for i in range(3):
            with pytest.raises(ValueError, match="share memory"):
                f(*x[:3], out=x[i])
    rows = torch.zeros(1, 2, 10, 64)
    for a, b in ((rows[:, :, :9], rows[:, :, 1:]), (rows[:, :, 1:], rows[:, :, :9])):
        with pytest.raises(ValueError, match="share memory"):
            f(a, k, v, out=b)
        with pytest.raises(ValueError, match="share memory"):
            f(q, a, v, out=b)
        with pytest.raises(ValueError, match="share memory"):
            f(q, k, a, out=b)
    with pytest.raises(ValueError, match="share memory"):
        f(q, k, v, log_key_mass=rows.view(-1)[-9:], out=rows[:, :, 1:])


def test_derivatives_are_refused(pkg):
    refuse = importlib.import_module(pkg.__name__ + ".streaming")._refuse_gradients
    t = torch.zeros(2)
    refuse("call", t, None)
    with pytest.raises(RuntimeError, match="no backward"):
        refuse("call", t, torch.zeros(2, requires_grad=True))
    with torch.no_grad():
        refuse("call", torch.zeros(2, requires_grad=True))
    with torch.autograd.forward_ad.dual_level():
        refuse("call", t, None)
        dual = torch.autograd.forward_ad.make_dual(t, torch.ones(2))
        with pytest.raises(RuntimeError, match="forward-mode"):
            refuse("call", t, dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            refuse("call", dual)


def test_integers_beyond_32_bits(pkg):
    """Slots and offsets that int32 does not hold are refused on the host; nothing wraps round to another slot."""
    f = importlib.import_module(pkg.__name__ + ".streaming")._int_vector
    cpu = torch.device("cpu")
    for good in ([1, 2], [], range(3), np.array([1, -5]), torch.tensor([2 ** 31 - 1, -2 ** 31]), torch.tensor([1, 7], dtype=torch.uint32),
                 torch.tensor([3], dtype=torch.uint8)):
        assert f("sequence", good, cpu).tolist() == [int(x) for x in good] and f("sequence", good, cpu).dtype == torch.int32
    for bad in ([2 ** 32], [0, 2 ** 31], [-2 ** 31 - 1], torch.tensor([2 ** 40]), torch.tensor([2 ** 32 - 1], dtype=torch.uint32),
                torch.tensor([2 ** 63 + 1], dtype=torch.uint64), torch.zeros(2, dtype=torch.complex64), torch.zeros(2, dtype=torch.bool)):
        with pytest.raises(ValueError, match="sequence"):
            f("sequence", bad, cpu)
    with pytest.raises(ValueError, match="2\\^31"):
        pkg.attention_ranges(1, 2 ** 31)


def test_scales_that_overflow_are_refused(pkg):
    """A scale is held with a factor log2(e): the largest finite ones would become infinite, and every result NaN."""
    lib, C = pkg.load_library(), pkg._clib
    s = (ctypes.c_int64 * 3)(64, 64, 64)
    two = (ctypes.c_int64 * 2)(64, 64)
    cache = C.CacheHandle(k=16, v=16, table=16, length=16, references=16, pages=4, page_size=16, kv_heads=2, slots=2, max_pages=4)
    for mods in (C.ScoreMods(scale=3e38), C.ScoreMods(scale=3e38, softcap=1e-3)):
        assert lib.vb200_masked_attention(1, 16, 16, 16, 16, 1, 4, 2, 3, 5, 64, s, s, s, s, mods, None, 0, None) == C.EINVAL
        assert b"out of range" in lib.vb200_last_error()
        assert lib.vb200_paged_attention(1, 16, 16, 2, 4, 64, two, two, cache, 16, 16, 1, 1, mods, None, 0, None) == C.EINVAL
        assert b"out of range" in lib.vb200_last_error()


def test_oracle_bound_of_a_growing_bias(oracle):
    """A distance bias of either sign rounds by its size: a negative slope takes nothing from the bound."""
    rng = np.random.default_rng(3)
    q, k, v = np.zeros((1, 1, 4, 64)), rng.standard_normal((1, 1, 900, 64)), rng.standard_normal((1, 1, 900, 64))
    out, bound = oracle.streaming.masked_attention(q, k, v, slope=[-2.0])
    # the keys that count lie 890 tokens away and more: their bias and the row's maximum, each 1,780, round 8 times
    assert (bound > 2 * 8 * 2.0 ** -24 * 1700 * np.abs(out)).all()
