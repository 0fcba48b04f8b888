"""The paged cache and the attention over it on the GPU, against the oracle's token-by-token cache and 64-bit attention."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import TORCH_DTYPE, to_np

pytestmark = pytest.mark.gpu


def pair(pkg, oracle, device, slots=4, pages=24, max_pages=10, page=16, heads=2, dtype="bf16", masses=True):
    """A cache on the device and the oracle's, both empty."""
    cache = pkg.PagedCache.empty(slots, pages, max_pages, page_size=page, heads=heads, dtype=TORCH_DTYPE[dtype], masses=masses,
                                 device=device)
    ref = oracle.streaming.Cache(np.zeros((pages, page, heads, 64), np.float32), np.zeros((pages, page, heads, 64), np.float32),
                                 np.zeros((pages, page), np.float32) if masses else None, np.full((slots, max_pages), -1), [0] * slots,
                                 [0] * pages)
    return cache, ref


def tokens(rng, n, heads, dtype, oracle):
    k, v = (oracle.round_to(rng.standard_normal((n, heads, 64)).astype(np.float32), dtype) for _ in range(2))
    return k, v, np.log(rng.integers(1, 9, n)).astype(np.float32)


def same(cache, ref):
    """Bookkeeping and every byte of the pools."""
    assert to_np(cache.table).astype(int).tolist() == ref.table().tolist()
    assert cache.length.tolist() == ref.length
    assert cache.references.tolist() == ref.refs
    assert np.array_equal(to_np(cache.k), ref.k) and np.array_equal(to_np(cache.v), ref.v)
    if ref.mass is not None:
        assert np.array_equal(to_np(cache.log_mass), ref.mass)


def append(cache, ref, device, dtype, rng, oracle, sequence, counts, behind=0, masses=True):
    """Appends on both; ``behind`` rows lie behind the last sequence's."""
    off = np.concatenate([[0], np.cumsum(counts)]).astype(int).tolist()
    k, v, m = tokens(rng, off[-1] + behind, ref.k.shape[2], dtype, oracle)
    t = lambda x: torch.from_numpy(x).to(device=device, dtype=TORCH_DTYPE[dtype])  # noqa: E731
    cache.append(torch.tensor(sequence, device=device), torch.tensor(off, device=device), t(k), t(v),
                 torch.from_numpy(m).to(device) if masses and ref.mass is not None else None)
    return ref.append(sequence, off, k, v, m if masses and ref.mass is not None else None)


@pytest.mark.parametrize("dtype,page,heads,masses", [("bf16", 16, 2, True), ("f16", 32, 1, False), ("f32", 64, 3, True), ("bf16", 128, 16, True)])
def test_operations_in_a_row(pkg, oracle, cuda_device, dtype, page, heads, masses):
    """Random appends (ragged, with empty chunks), forks, frees and compactions, all state compared after each."""
    rng = np.random.default_rng(page)
    cache, ref = pair(pkg, oracle, cuda_device, slots=5, pages=30, max_pages=9, page=page, heads=heads, dtype=dtype, masses=masses)
    done = 0
    for _ in range(60):
        what = rng.integers(5)
        some = rng.permutation(5)[:rng.integers(1, 5)].tolist()
        if what <= 1:
            done += append(cache, ref, cuda_device, dtype, rng, oracle, some, rng.integers(0, 2 * page, len(some)),
                           behind=int(rng.integers(3)), masses=bool(rng.integers(2)))
        elif what == 2:
            to = rng.integers(0, 5, len(some)).tolist()
            cache.fork(some, to)
            ref.fork(some, to)
        elif what == 3:
            cache.free(torch.tensor(some[:2], device=cuda_device))
            ref.free(some[:2])
        else:
            used = cache.compact()
            assert int(used) == ref.compact()
        same(cache, ref)
        pkg.device_error_flags()  # a pool that was full is part of the test
    assert done > 5


def test_append_all_or_nothing(pkg, oracle, cuda_device):
    rng = np.random.default_rng(0)
    cache, ref = pair(pkg, oracle, cuda_device, slots=3, pages=6, max_pages=4)
    assert append(cache, ref, cuda_device, "bf16", rng, oracle, [0, 1], [40, 20])  # 3 + 2 pages
    same(cache, ref)
    assert pkg.device_error_flags() == 0
    assert not append(cache, ref, cuda_device, "bf16", rng, oracle, [1, 2], [5, 17])  # one page is left, two are asked for
    same(cache, ref)
    assert pkg.device_error_flags() == 4
    assert not append(cache, ref, cuda_device, "bf16", rng, oracle, [0, 1], [25, 1])  # slot 0 would need a fifth page
    same(cache, ref)
    assert pkg.device_error_flags() == 4
    assert append(cache, ref, cuda_device, "bf16", rng, oracle, [0, 1], [24, 12])  # exactly full
    same(cache, ref)
    assert pkg.device_error_flags() == 0


def test_bad_indices_are_left_out(pkg, oracle, cuda_device):
    rng = np.random.default_rng(1)
    cache, ref = pair(pkg, oracle, cuda_device)
    append(cache, ref, cuda_device, "bf16", rng, oracle, [1, 4, -1, 0, 1], [5, 3, 2, 20, 7])  # out of range, named twice
    same(cache, ref)
    assert pkg.device_error_flags() == 2
    t = lambda *x: torch.tensor(x, device=cuda_device, dtype=torch.int32)  # noqa: E731
    k = torch.zeros(8, 2, 64, device=cuda_device, dtype=torch.bfloat16)
    for off in ((0, 5, 3), (0, 4, 9), (-1, 2, 4)):  # descending, beyond the rows, before them
        cache.append(t(0, 2), t(*off), k, k)
        same(cache, ref)
        assert pkg.device_error_flags() == 2
    cache.fork([1, 7, 0], [2, 1, -3])
    ref.fork([1, 7, 0], [2, 1, -3])
    same(cache, ref)
    assert pkg.device_error_flags() == 2
    cache.free([9, -1, 1, 1])
    ref.free([9, -1, 1])
    same(cache, ref)
    assert pkg.device_error_flags() == 2


def test_forks_of_forks(pkg, oracle, cuda_device):
    """Swaps, chains, one target twice, a slot onto itself; then every branch writes its own last page."""
    rng = np.random.default_rng(2)
    cache, ref = pair(pkg, oracle, cuda_device, pages=40)
    append(cache, ref, cuda_device, "bf16", rng, oracle, [0, 1, 2], [20, 37, 16])
    for a, b in (([0, 1], [1, 0]), ([0, 1, 2], [1, 2, 3]), ([0, 1], [3, 3]), ([2, 2, 0], [2, 0, 2]), ([3], [3])):
        cache.fork(a, b)
        ref.fork(a, b)
        same(cache, ref)
    append(cache, ref, cuda_device, "bf16", rng, oracle, [3, 0, 2, 1], [1, 1, 30, 0])
    same(cache, ref)
    cache.free([0, 1, 2, 3])
    ref.free([0, 1, 2, 3])
    same(cache, ref)
    assert int(cache.references.abs().sum()) == 0 and pkg.device_error_flags() == 0


def test_empty_calls(pkg, oracle, cuda_device):
    cache, ref = pair(pkg, oracle, cuda_device)
    k = torch.zeros(0, 2, 64, device=cuda_device, dtype=torch.bfloat16)
    cache.append([], [0], k, k)
    cache.append([1], [0, 0], k, k)
    cache.fork([], [])
    cache.fork([1], [2])
    cache.free([])
    assert int(cache.compact()) == 0
    same(cache, ref)
    assert pkg.device_error_flags() == 0


def test_many_sequences_and_pages(pkg, oracle, cuda_device):
    """More sequences than the bookkeeping block has threads, more pages than it scans in a round."""
    rng = np.random.default_rng(3)
    cache, ref = pair(pkg, oracle, cuda_device, slots=1500, pages=9000, max_pages=8, heads=1)
    order = rng.permutation(1500).tolist()
    assert append(cache, ref, cuda_device, "bf16", rng, oracle, order, rng.integers(0, 60, 1500))
    same(cache, ref)
    gone = rng.permutation(1500)[:700].tolist()
    cache.free(gone)
    ref.free(gone)
    assert append(cache, ref, cuda_device, "bf16", rng, oracle, order[:900], rng.integers(0, 30, 900))
    same(cache, ref)
    cache.fork(list(range(700)), list(range(750, 1450)))
    ref.fork(list(range(700)), list(range(750, 1450)))
    same(cache, ref)
    assert int(cache.compact()) == ref.compact()
    same(cache, ref)
    assert pkg.device_error_flags() == 0


# ---------------------------------------------------------------- attention over the cache

def filled(pkg, oracle, device, dtype, page, heads, lengths, seed=0, masses=True):
    """Slots of these lengths on scattered pages (other slots freed in between), pools around them full of NaN."""
    rng = np.random.default_rng(seed)
    need = sum(-(-n // page) for n in lengths)
    cache, ref = pair(pkg, oracle, device, slots=2 * len(lengths), pages=2 * need + 3, max_pages=max(-(-max(lengths) // page), 1) + 1,
                      page=page, heads=heads, dtype=dtype, masses=masses)
    cache.k.fill_(float("nan")), cache.v.fill_(float("nan"))
    if masses:
        cache.log_mass.fill_(float("nan"))
    n = len(lengths)
    every = [int(x) for pair_ in zip(range(n), range(n, 2 * n)) for x in pair_]
    append(cache, ref, device, dtype, rng, oracle, every, [max(1, x // 2) for x in lengths for _ in range(2)])
    cache.free(list(range(n, 2 * n)))
    ref.free(list(range(n, 2 * n)))
    append(cache, ref, device, dtype, rng, oracle, list(range(n)), [x - max(1, x // 2) if x else 0 for x in lengths])
    return rng, cache, ref


def attend(pkg, oracle, device, dtype, cache, ref, rng, sequence, counts, heads, causal=True, ranges=None, q_scale=2.0, behind=0, **kw):
    td = TORCH_DTYPE[dtype]
    off = np.concatenate([[0], np.cumsum(counts)]).astype(int)
    q = oracle.round_to((rng.standard_normal((off[-1] + behind, heads, 64)) * q_scale).astype(np.float32), dtype)
    slope = kw.pop("slope", None)
    out = torch.full(q.shape, 7.0, device=device, dtype=td)
    dev = lambda x, t=torch.int32: None if x is None else torch.as_tensor(np.asarray(x)).to(device=device, dtype=t)  # noqa: E731
    got = pkg.paged_attention(dev(q, td), cache, dev(sequence), dev(off), causal=causal, key_range=dev(ranges),
                              distance_slope=dev(slope, torch.float32), out=out, **kw)
    assert got is out
    got = to_np(out)
    for i, s in enumerate(sequence):
        k, v, m = ref.tokens(s)
        n, L = counts[i], ref.length[s]
        if ranges is not None:
            r = np.asarray(ranges)[off[i]:off[i + 1]]
        else:
            end = np.arange(L - n + 1, L + 1) if causal else np.full(n, L)
            r = np.stack([np.zeros(n, int), end], 1)
        want, bound = oracle.streaming.masked_attention(q[None, off[i]:off[i + 1]].swapaxes(1, 2), k[None].swapaxes(1, 2), v[None].swapaxes(1, 2),
                                                        m, r, slope=slope, qpos=np.arange(L - n, L), dtype=dtype, **kw)
        part = got[off[i]:off[i + 1]].swapaxes(0, 1)[None]
        assert np.isfinite(part).all()
        over = np.abs(part - want) - bound
        assert over.max(initial=-1) <= 0, f"sequence {i}: off by {over.max():.3e} more than the bound"
    assert (got[off[-1]:] == 7).all()  # rows behind the last sequence are left as they were
    assert pkg.device_error_flags() == 0
    return got


CHUNKS = [  # lengths, new rows
    ([1], [1]),
    ([300], [1]),
    ([5, 700, 64, 128, 129], [1, 1, 1, 1, 1]),
    ([33, 260, 700], [33, 17, 1]),
    ([400, 1, 530], [300, 1, 257]),
    ([200, 77], [0, 77]),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("case", range(len(CHUNKS)))
def test_paged(pkg, oracle, cuda_device, dtype, page, case):
    lengths, counts = CHUNKS[case]
    rng, cache, ref = filled(pkg, oracle, cuda_device, dtype, page, 2, lengths, seed=case)
    order = rng.permutation(len(lengths)).tolist()
    attend(pkg, oracle, cuda_device, dtype, cache, ref, rng, order, [counts[i] for i in order], 4, causal=case % 2 == 0, behind=case % 3)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("counts", [[1, 2, 1], [150, 40, 3]])
def test_paged_scores(pkg, oracle, cuda_device, dtype, counts):
    rng, cache, ref = filled(pkg, oracle, cuda_device, dtype, 32, 2, [500, 333, 90])
    slope = np.array([0.5, 0.1, 0.02, 0.004, 0.001, 0.0], np.float32)
    attend(pkg, oracle, cuda_device, dtype, cache, ref, rng, [2, 0, 1], counts[::-1], 6, softcap=15.0, slope=slope, scale=0.2)
    rng, cache, ref = filled(pkg, oracle, cuda_device, dtype, 32, 2, [500, 333, 90], masses=False)
    attend(pkg, oracle, cuda_device, dtype, cache, ref, rng, [0, 1, 2], counts, 2)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("counts", [[2, 1], [200, 130]])
def test_paged_ranges(pkg, oracle, cuda_device, dtype, counts):
    """Frames in causal order, windows, and rows that see nothing, given as key intervals."""
    rng, cache, ref = filled(pkg, oracle, cuda_device, dtype, 16, 2, [420, 300])
    n = sum(counts)
    r = np.sort(rng.integers(-3, 430, (n, 2)), axis=1)
    r[::5] = 100
    r[1::7] = [290, 999]
    for i in range(n):  # the oracle's intervals are inside the slot, as the kernels clip them
        L = 420 if i < counts[0] else 300
        r[i] = np.clip(r[i], 0, L)
    got = attend(pkg, oracle, cuda_device, dtype, cache, ref, rng, [0, 1], counts, 2, ranges=r)
    empty = np.nonzero(r[:, 1] <= r[:, 0])[0]
    assert len(empty) and (got[empty] == 0).all()


def test_padded_batch_and_empty_slots(pkg, oracle, cuda_device):
    """Empty sequences between others, an empty slot with a row, rows behind the last sequence."""
    rng, cache, ref = filled(pkg, oracle, cuda_device, "bf16", 16, 2, [50, 20, 30])
    attend(pkg, oracle, cuda_device, "bf16", cache, ref, rng, [0, 4, 1, 2, 0], [0, 1, 2, 0, 1], 2, causal=False, behind=9)
    attend(pkg, oracle, cuda_device, "bf16", cache, ref, rng, [4, 0, 1, 2], [40, 50, 0, 30], 2, causal=False, behind=200)


@pytest.mark.parametrize("rows", [3, 90])
def test_bad_pages_and_slots_are_reported(pkg, oracle, cuda_device, rows):
    """Page numbers outside the pool, slots and offsets out of range: an error bit, no access, the other sequences right."""
    rng, cache, ref = filled(pkg, oracle, cuda_device, "bf16", 16, 2, [100, 120, 140])
    good = cache.table.clone()
    q = torch.randn(3 * rows, 2, 64, device=cuda_device).bfloat16()
    off = torch.tensor([0, rows, 2 * rows, 3 * rows], device=cuda_device, dtype=torch.int32)
    want = pkg.paged_attention(q, cache, [0, 1, 2], off)
    assert pkg.device_error_flags() == 0
    for bad in (-1, cache.k.shape[0], 2 ** 31 - 1):
        cache.table[1, 2] = bad
        got = pkg.paged_attention(q, cache, [0, 1, 2], off)
        assert pkg.device_error_flags() == 2
        assert torch.equal(got[:rows], want[:rows]) and torch.equal(got[2 * rows:], want[2 * rows:])
    cache.table.copy_(good)
    got = pkg.paged_attention(q, cache, [0, 99, 2], off)
    assert pkg.device_error_flags() == 2
    assert torch.equal(got[:rows], want[:rows]) and torch.equal(got[2 * rows:], want[2 * rows:])
    bad_off = off.clone()
    bad_off[3] = 3 * rows + 5
    got = pkg.paged_attention(q, cache, [0, 1, 2], bad_off)
    assert pkg.device_error_flags() == 2 and torch.equal(got[:2 * rows], want[:2 * rows])
    cache.length[2] = 10 ** 6  # longer than its table row: read no further than the row
    pkg.paged_attention(q, cache, [0, 1, 2], off)
    assert pkg.device_error_flags() == 2


@pytest.mark.parametrize("rows", [1, 40])
def test_pool_beyond_32_bits(pkg, oracle, cuda_device, rows):
    """Pools of more than 2^31 elements: pages at the far end are written, copied, moved and read."""
    page, heads, pages = 128, 16, 17000  # 2.2e9 elements
    cache = pkg.PagedCache.empty(3, pages, 8, page_size=page, heads=heads, device=cuda_device)
    cache.references[: pages - 12] = 1  # all but the last pages are taken
    rng = np.random.default_rng(5)
    k, v, m = tokens(rng, 300, heads, "bf16", oracle)
    t = lambda x: torch.from_numpy(x).to(cuda_device, torch.bfloat16)  # noqa: E731
    cache.append([0], [0, 290], t(k[:290]), t(v[:290]), torch.from_numpy(m[:290]).to(cuda_device))
    cache.fork([0], [1])
    cache.append([1], [0, 10], t(k[290:]), t(v[290:]), torch.from_numpy(m[290:]).to(cuda_device))
    assert cache.table[1, :3].tolist() == [pages - 12, pages - 11, pages - 9]
    q = oracle.round_to(rng.standard_normal((rows, heads, 64)).astype(np.float32), "bf16")
    end = np.arange(300 - rows + 1, 301)
    want, bound = oracle.streaming.masked_attention(q[None].swapaxes(1, 2), k[None].swapaxes(1, 2), v[None].swapaxes(1, 2), m,
                                                    np.stack([0 * end, end], 1), dtype="bf16")
    for far in (True, False):
        got = to_np(pkg.paged_attention(t(q), cache, [1], [0, rows])).swapaxes(0, 1)[None]
        assert (np.abs(got - want) <= bound).all()
        if far:
            cache.references[: pages - 12] = 0
        assert int(cache.compact()) == 4  # moves the far pages to the front
        assert int(cache.table.max()) == 3
    assert pkg.device_error_flags() == 0


def test_streamed_step_in_a_graph(pkg, oracle, cuda_device):
    """Append, attention, fork and free recorded once and replayed: the same state and bits as eager calls."""
    g = torch.Generator(device=cuda_device).manual_seed(3)
    make = lambda: pkg.PagedCache.empty(3, 60, 12, page_size=16, heads=2, device=cuda_device)  # noqa: E731
    seq = torch.tensor([0, 1], device=cuda_device, dtype=torch.int32)
    off = torch.tensor([0, 7, 30], device=cuda_device, dtype=torch.int32)
    two, zero = torch.tensor([2], device=cuda_device, dtype=torch.int32), torch.tensor([0], device=cuda_device, dtype=torch.int32)
    x = torch.empty(30, 3, 2, 64, device=cuda_device, dtype=torch.bfloat16)

    def step(cache):
        cache.append(seq, off, x[:, 1], x[:, 2])
        cache.fork(zero, two)
        return pkg.paged_attention(x[:, 0], cache, seq, off)

    inputs = [torch.randn(30, 3, 2, 64, generator=g, device=cuda_device).bfloat16() for _ in range(4)]
    eager, graphed = make(), make()
    x.copy_(inputs[0])
    step(make())  # warm up
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(graphed)
    graphed.table.fill_(-1), graphed.length.zero_(), graphed.references.zero_()
    for t in inputs:
        x.copy_(t)
        graph.replay()
        want = step(eager)
        assert torch.equal(out, want)
        for name in ("k", "v", "log_mass", "table", "length", "references"):
            assert torch.equal(getattr(eager, name), getattr(graphed, name)), name
    assert pkg.device_error_flags() == 0


def test_refusals_on_the_gpu(pkg, cuda_device):
    cache = pkg.PagedCache.empty(2, 4, 4, page_size=16, heads=2, masses=False, device=cuda_device)
    z = lambda *s, dt=torch.bfloat16: torch.zeros(s, device=cuda_device, dtype=dt)  # noqa: E731
    with pytest.raises(ValueError, match="k and v must"):
        cache.append([0], [0, 1], z(1, 3, 64), z(1, 3, 64))
    with pytest.raises(ValueError, match="cache holds"):
        cache.append([0], [0, 1], z(1, 2, 64).half(), z(1, 2, 64).half())
    with pytest.raises(ValueError, match="log-masses"):
        cache.append([0], [0, 1], z(1, 2, 64), z(1, 2, 64), z(1))
    with pytest.raises(ValueError, match="offsets"):
        cache.append([0], [0, 1, 1], z(1, 2, 64), z(1, 2, 64))
    with pytest.raises(ValueError, match="sequence"):
        cache.free(torch.zeros(1, device=cuda_device))
    with pytest.raises(ValueError, match="target"):
        cache.fork([0], [0, 1])
    with pytest.raises(RuntimeError, match="no backward"):
        cache.append([0], [0, 1], z(1, 2, 64).requires_grad_(), z(1, 2, 64))
    f = pkg.paged_attention
    with pytest.raises(ValueError, match="no multiple"):
        f(z(1, 3, 64), cache, [0], [0, 1])
    with pytest.raises(ValueError, match="q must be"):
        f(z(1, 2, 32), cache, [0], [0, 1])
    with pytest.raises(ValueError, match="cache holds"):
        f(z(1, 2, 64).float(), cache, [0], [0, 1])
    with pytest.raises(ValueError, match="key_range"):
        f(z(1, 2, 64), cache, [0], [0, 1], key_range=z(1, 2))
    with pytest.raises(ValueError, match="softcap"):
        f(z(1, 2, 64), cache, [0], [0, 1], softcap=-2.0)
    with pytest.raises(ValueError, match="distance_slope"):
        f(z(1, 2, 64), cache, [0], [0, 1], distance_slope=z(3))
    with pytest.raises(RuntimeError, match="no backward"):
        f(z(1, 2, 64).requires_grad_(), cache, [0], [0, 1])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("softcap", [None, 5.0])
def test_paged_distance_over_whole_tiles(pkg, oracle, cuda_device, causal, softcap):
    """Chunks longer than a query tile over a past whose tiles are taken last to first, the last of them filled in part."""
    rng = np.random.default_rng(33)
    cache, ref = pair(pkg, oracle, cuda_device, slots=2, pages=120, max_pages=60, page=32, heads=2)
    append(cache, ref, cuda_device, "bf16", rng, oracle, [0, 1], [1203, 650])
    append(cache, ref, cuda_device, "bf16", rng, oracle, [0, 1], [290, 150])
    q = oracle.round_to(rng.standard_normal((440, 4, 64)).astype(np.float32), "bf16")
    slope = np.array([0.003, 0.5, 2.0, 0.0], np.float32)
    out = pkg.paged_attention(torch.from_numpy(q).to(cuda_device, torch.bfloat16), cache, [0, 1], [0, 290, 440], causal=causal,
                              softcap=softcap, distance_slope=torch.from_numpy(slope).to(cuda_device))
    for s, (a, b) in enumerate(((0, 290), (290, 440))):
        L, n = ref.length[s], b - a
        rows = [ref.held[s][j // 32] * 32 + j % 32 for j in range(L)]
        k, v, m = (t.reshape(-1, *t.shape[2:])[rows] for t in (ref.k, ref.v, ref.mass))
        seen = np.array([[0, L - n + i + 1 if causal else L] for i in range(n)])
        want, bound = oracle.streaming.masked_attention(q[a:b].transpose(1, 0, 2)[None], k.transpose(1, 0, 2)[None], v.transpose(1, 0, 2)[None],
                                                        m, seen, softcap=softcap, slope=slope, dtype="bf16")
        off = np.abs(to_np(out[a:b]).transpose(1, 0, 2) - want[0]) - bound[0]
        assert off.max() <= 0, off.max()
    assert pkg.device_error_flags() == 0


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,counts,heads,kv_heads,page", [
    ([700, 1100], [300, 300], 37, 1, 16),    # 148 row blocks that run whole: the last, partly filled key tile is the 6th and the 9th
    ([700, 1100], [300, 300], 37, 1, 64),
    ([1700, 2100], [300, 300], 37, 1, 64),   # the 14th and the 17th
    ([1700, 2100], [300, 300], 37, 1, 16),
    ([5900], [1041], 4, 4, 16),              # 20 blocks in 7 parts each: the 7th of its part
    ([5900], [1041], 8, 2, 64),              # 40 in 3: the 16th
    ([9273], [1041], 4, 2, 64),              # 20 in 7: the 11th
])
@pytest.mark.parametrize("stale", [float("nan"), 100.0])
def test_last_tile_without_masses(pkg, oracle, cuda_device, dtype, causal, lengths, counts, heads, kv_heads, page, stale):
    """Long streams in a cache without masses: every value of every tile takes part, what lies behind the last key does not.
    All values are positive, so a tile's missing values are more than the bound allows."""
    rng = np.random.default_rng(sum(lengths) + page)
    cache, ref = pair(pkg, oracle, cuda_device, slots=len(lengths), pages=sum(-(-n // page) for n in lengths), heads=kv_heads,
                      max_pages=-(-max(lengths) // page) + 1, page=page, dtype=dtype, masses=False)
    cache.k.fill_(stale), cache.v.fill_(stale)
    n = sum(lengths)
    k, v = (oracle.round_to(f(rng.standard_normal((n, kv_heads, 64))).astype(np.float32), dtype) for f in (np.array, np.abs))
    off = np.concatenate([[0], np.cumsum(lengths)]).tolist()
    order = list(range(len(lengths)))
    t = lambda x: torch.from_numpy(x).to(cuda_device, TORCH_DTYPE[dtype])  # noqa: E731
    cache.append(order, off, t(k), t(v))
    assert ref.append(order, off, k, v)
    attend(pkg, oracle, cuda_device, dtype, cache, ref, rng, order, counts, heads, causal=causal, q_scale=1.0)


def test_outputs_in_the_cache_are_refused(pkg, cuda_device):
    cache = pkg.PagedCache.empty(2, 4, 4, page_size=16, heads=2, device=cuda_device)
    x = torch.zeros(3, 3, 2, 64, device=cuda_device, dtype=torch.bfloat16)
    seq, off = (torch.tensor(t, device=cuda_device, dtype=torch.int32) for t in ([0], [0, 2]))
    q = x[:2, 0]
    for bad in (x[1:, 0], cache.k[1, :2], cache.v[3, 5:7], q):
        with pytest.raises(ValueError, match="share memory"):
            pkg.paged_attention(q, cache, seq, off, out=bad)
    assert pkg.paged_attention(q, cache, seq, off, out=x[:2, 2]).data_ptr() == x[0, 2].data_ptr()
    assert pkg.device_error_flags() == 0


def test_derivatives_are_refused(pkg, cuda_device):
    cache = pkg.PagedCache.empty(2, 4, 4, page_size=16, heads=2, device=cuda_device)
    x = torch.zeros(1, 2, 64, device=cuda_device, dtype=torch.bfloat16)
    dense = torch.zeros(1, 2, 5, 64, device=cuda_device)
    ad = torch.autograd.forward_ad
    with ad.dual_level():
        dual = ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: cache.append([0], [0, 1], dual, x), lambda: pkg.paged_attention(dual, cache, [0], [0, 1]),
                     lambda: pkg.masked_attention(dense, ad.make_dual(dense, dense), dense)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
    assert cache.length.tolist() == [0, 0]
    cache.v.requires_grad_()
    for call in (lambda: cache.append([0], [0, 1], x, x), lambda: pkg.paged_attention(x, cache, [0], [0, 1])):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
    with torch.no_grad():
        cache.append([0], [0, 1], x, x)
    assert cache.length.tolist() == [1, 0] and pkg.device_error_flags() == 0


def test_integers_beyond_32_bits(pkg, oracle, cuda_device):
    """On the device they name no slot and no row: an error bit, and the cache as it was."""
    rng, cache, ref = filled(pkg, oracle, cuda_device, "bf16", 16, 2, [20, 30])
    t = lambda *x: torch.tensor(x, device=cuda_device)  # noqa: E731
    k = torch.zeros(4, 2, 64, device=cuda_device, dtype=torch.bfloat16)
    before = cache.length.clone(), cache.table.clone()
    for call in (lambda: cache.append(t(2 ** 32), t(0, 4), k, k), lambda: cache.append(t(0), t(2 ** 32, 2 ** 32 + 4), k, k),
                 lambda: cache.fork(t(2 ** 32 + 1), t(2)), lambda: cache.fork(t(1), t(2 ** 33 + 2)), lambda: cache.free(t(-2 ** 32))):
        call()
        assert pkg.device_error_flags() == 2
        assert torch.equal(cache.length, before[0]) and torch.equal(cache.table, before[1])
    out = torch.full((4, 2, 64), 7.0, device=cuda_device, dtype=torch.bfloat16)
    pkg.paged_attention(k, cache, t(2 ** 32), t(0, 4), out=out)
    pkg.paged_attention(k, cache, t(0), t(2 ** 32, 2 ** 32 + 4), out=out)
    assert pkg.device_error_flags() == 2 and bool((out == 7).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,rows", [(4, 300), (2, 3)])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("softcap,dist,mass", [(None, False, False), (8.0, True, True), (None, True, True), (30.0, False, True)])
def test_rows_beside_hidden_values(pkg, oracle, cuda_device, dtype, heads, rows, paged, softcap, dist, mass):
    """Every row's tiles hold values that are NaN and hidden from it, so every row is computed a second time: intervals from one
    key to 900, in a dense tensor and over pages, with all that changes a score."""
    n, td = 1000, TORCH_DTYPE[dtype]
    rng = np.random.default_rng(rows + heads)
    k, v, m = tokens(rng, n, 2, dtype, oracle)
    m[::17] = -np.inf
    hide = np.ones(n, bool)
    hide[40:940] = False
    k[hide], v[hide] = np.nan, np.nan
    r = np.sort(rng.integers(40, 940, (rows, 2)), 1).astype(np.int32)
    r[::5] = [40, 940]
    r[1::7, 1] = r[1::7, 0] + 1
    q = oracle.round_to((rng.standard_normal((rows, heads, 64)) * 2).astype(np.float32), dtype)
    slope = (2.0 ** -np.arange(1, heads + 1)).astype(np.float32) if dist else None
    m = m if mass else None
    t = lambda x, d=td: None if x is None else torch.from_numpy(np.ascontiguousarray(x)).to(cuda_device, d)  # noqa: E731
    kw = dict(key_range=t(r, torch.int32), softcap=softcap, distance_slope=t(slope, torch.float32))
    if paged:
        cache = pkg.PagedCache.empty(2, 70, 65, page_size=16, heads=2, dtype=td, masses=mass, device=cuda_device)
        cache.append([1], [0, n], t(k), t(v), t(m, torch.float32))
        got = pkg.paged_attention(t(q), cache, [1], [0, rows], **kw).transpose(0, 1)[None]
    else:
        dense = lambda x: t(x.swapaxes(0, 1)[None])  # noqa: E731
        got = pkg.masked_attention(dense(q), dense(k), dense(v), t(m, torch.float32), **kw)
    want, bound = oracle.streaming.masked_attention(*(x[None].swapaxes(1, 2) for x in (q, np.where(hide[:, None, None], 0, k), np.where(hide[:, None, None], 0, v))),
                                                    m, r, softcap=softcap, slope=slope, dtype=dtype)
    got = to_np(got)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= bound).all(), (np.abs(got - want) - bound).max()
    assert pkg.device_error_flags() == 0
