"""The global-attention block with a mask and over a paged cache, as a user runs it: merged frames, forked and freed streams,
a recorded step.  Everything around the attention is taken from the module's own operators (whose results have tests of their
own and repeat bit for bit), the attention itself from the oracle in 64 bits with its bound; the output projection is the
identity, exact in every type."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import TORCH_DTYPE, to_np

pytestmark = pytest.mark.gpu

DIM, HEADS, FRAME, SPECIAL = 256, 4, 90, 5


def block(pkg, device, dtype, seed=0):
    m = pkg.GlobalAttention(DIM, HEADS, device=device, dtype=TORCH_DTYPE[dtype])
    rng = np.random.default_rng(seed)
    with torch.no_grad():
        for p in m.parameters():
            p.copy_(torch.from_numpy(rng.standard_normal(p.shape).astype(np.float32) * (0.1 if p.ndim > 1 else 0.5)))
        m.proj.weight.copy_(torch.eye(DIM))
        m.proj.bias.zero_()
    return m


def merge_plan(pkg, oracle, device, frames, kept, seed, preserve=False, special=False):
    rng = np.random.default_rng(seed)
    N = frames * FRAME
    special_ids = np.concatenate([np.arange(f * FRAME, f * FRAME + SPECIAL) for f in range(frames)])
    others = np.setdiff1d(np.arange(N), special_ids)
    keep = np.sort(np.concatenate([special_ids, rng.choice(others, kept - special_ids.size, replace=False)]))
    src = np.setdiff1d(np.arange(N), keep)
    parent = np.stack([rng.choice(kept, 4, replace=False) for _ in src])
    w = rng.dirichlet(np.ones(4), size=src.size).astype(np.float32)
    t = lambda a, dt=torch.long: torch.as_tensor(a, device=device, dtype=dt)  # noqa: E731
    norm = t(oracle.normalizer(parent, w, kept), torch.float32).view(1, -1, 1)
    return pkg.WeightedBilinearTokenPlan(
        keep=t(keep)[None], source_original=t(src)[None], source_parent_compact=t(parent)[None],
        source_pool_weights=t(w, torch.float32)[None], source_restore_weights=t(w, torch.float32)[None], original_tokens=N,
        normalizer=norm, preserve_queries=preserve, preserve_destination_keys=preserve, dense_special_queries=special,
        special_query_original=t(special_ids), special_query_compact=t(np.searchsorted(keep, special_ids)),
        key_log_mass=norm[..., 0].log())


def compact(pkg, m, qkv, plan):
    """q, k, v [rows, H, 64] of the plan's attention, and q, k, v of the clip, all from the framework's own operators."""
    ab = __import__("importlib").import_module(pkg.__name__ + ".attention_block")
    dense = ab._dense_rows(qkv, HEADS, m.q_norm, m.k_norm)
    if plan is None:
        rows = dense
    elif ab._fused_ok(qkv, plan, m.q_norm, m.k_norm):
        rows = [t[None] for t in ab._compact_rows_fused(qkv[0], plan, m.q_norm, m.k_norm)]
    else:
        rows = ab._compact_rows(*dense, plan)
    return [to_np(t.reshape(t.shape[1], HEADS, 64)) for t in rows], dense


def close(got, ref, bound):
    """got [rows, H, 64] or [rows, DIM] against ref and bound [H, rows, 64]."""
    got = to_np(got).astype(np.float64).reshape(-1, HEADS, 64).transpose(1, 0, 2)
    off = np.abs(got - ref) - bound
    assert np.isfinite(got).all() and off.max() <= 0, (off.max(), np.abs(got - ref).max())


def attend(oracle, q, k, v, mass, dtype, ranges=None, **mods):
    heads_first = lambda t: np.asarray(t).transpose(1, 0, 2)[None]  # noqa: E731
    o, b = oracle.streaming.masked_attention(heads_first(q), heads_first(k), heads_first(v), mass, ranges, dtype=dtype, **mods)
    return o[0], b[0]


MASKS = {
    "frames in order": dict(step=FRAME),
    "two clips": dict(documents=[0, 2 * FRAME, 4 * FRAME], step=FRAME, prefix=SPECIAL),
    "window": dict(step=1, window=100),
    "score changes": dict(step=FRAME, softcap=5.0, slope=True),
    "positions": dict(slope=True, position=True),
}


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["none", "compact", "preserve"])
@pytest.mark.parametrize("name", list(MASKS))
def test_forward_with_a_mask(pkg, oracle, cuda_device, name, kind, dtype):
    spec = dict(MASKS[name])
    frames, kept = 4, 131
    N = frames * FRAME
    rng = np.random.default_rng(3)
    m = block(pkg, cuda_device, dtype)
    plan = None if kind == "none" else merge_plan(pkg, oracle, cuda_device, frames, kept, 4, preserve=kind == "preserve")
    x = torch.from_numpy(rng.standard_normal((1, N, DIM)).astype(np.float32)).to(cuda_device, TORCH_DTYPE[dtype])
    softcap, slope = spec.pop("softcap", None), np.array([0.02, 0.01, 0.0, 0.3], np.float32) if spec.pop("slope", False) else None
    position = (np.arange(N, dtype=np.float32) // FRAME) if spec.pop("position", False) else None
    if "documents" in spec:
        spec["documents"] = torch.tensor(spec["documents"], device=cuda_device)
    ranges = pkg.attention_ranges(N, device=cuda_device, **spec) if spec else None
    t = lambda a: None if a is None else torch.from_numpy(a).to(cuda_device)  # noqa: E731
    mask = pkg.AttentionMask(key_range=ranges, softcap=softcap, distance_slope=t(slope), position=t(position))
    with torch.no_grad():
        y = m(x, plan, mask)
        qkv = m.qkv_projection(x)
        (q, k, v), _ = compact(pkg, m, qkv, plan)
    keep = np.arange(N) if plan is None else to_np(plan.keep[0]).astype(int)
    at = keep if kind == "compact" else np.arange(N)  # the clip's token of every query row
    place = np.arange(N, dtype=np.float32) if position is None else position
    seen = None
    if ranges is not None:  # compact keys whose kept token lies in the row's interval, counted one by one
        own = to_np(ranges).astype(int)[at]
        seen = np.array([[(keep < b).sum(), (keep < e).sum()] for b, e in own])
    mass = None if plan is None else to_np(plan.key_log_mass[0])
    ref, bound = attend(oracle, q, k, v, mass, dtype, seen, softcap=softcap, slope=slope, qpos=place[at], kpos=place[keep])
    close(y[0][torch.from_numpy(at).to(cuda_device)], ref, bound)  # restore copies the rows of kept tokens
    assert pkg.device_error_flags() == 0


def test_mask_with_dense_special_queries(pkg, oracle, cuda_device):
    """Special queries attend over the dense keys under the clip's own intervals, the other rows over the merged ones."""
    N = 3 * FRAME
    m = block(pkg, cuda_device, "bf16")
    plan = merge_plan(pkg, oracle, cuda_device, 3, 99, 5, special=True)
    x = torch.randn(1, N, DIM, generator=torch.Generator().manual_seed(0)).to(cuda_device, torch.bfloat16)
    ranges = pkg.attention_ranges(N, step=FRAME, device=cuda_device)
    with torch.no_grad():
        y = m(x, plan, pkg.AttentionMask(key_range=ranges))
        qkv = m.qkv_projection(x)
        fn = __import__("importlib").import_module(pkg.__name__ + ".ops").head_layernorm
        ln = [(n.weight.detach().float(), n.bias.detach().float()) for n in (m.q_norm, m.k_norm)]
        special = plan.special_query_original
        q = to_np(fn(qkv[0][special][:, :DIM].contiguous(), *ln[0])).reshape(-1, HEADS, 64)
        k = to_np(fn(qkv[0][:, DIM:2 * DIM], *ln[1])).reshape(N, HEADS, 64)
        v = to_np(qkv[0][:, 2 * DIM:]).reshape(N, HEADS, 64)
    ref, bound = attend(oracle, q, k, v, None, "bf16", to_np(ranges).astype(int)[to_np(special).astype(int)])
    close(y[0][special], ref, bound)


def test_forward_batch_with_own_intervals(pkg, oracle, cuda_device):
    rng = np.random.default_rng(8)
    m = block(pkg, cuda_device, "f32")
    x = torch.from_numpy(rng.standard_normal((2, 60, DIM)).astype(np.float32)).to(cuda_device)
    ranges = torch.stack([pkg.attention_ranges(60, step=20), pkg.attention_ranges(60, step=1)]).to(cuda_device)
    with torch.no_grad():
        y = m(x, mask=pkg.AttentionMask(key_range=ranges))
        for b in range(2):
            (q, k, v), _ = compact(pkg, m, m.qkv_projection(x)[b:b + 1], None)
            ref, bound = attend(oracle, q, k, v, None, "f32", to_np(ranges[b]).astype(int))
            close(y[b], ref, bound)


@pytest.mark.parametrize("dtype,page", [("bf16", 16), ("f16", 64), ("f32", 32)])
def test_streams_of_merged_frames(pkg, oracle, cuda_device, dtype, page):
    """Two streams of merged frames; one is forked and both branches go on, the other is freed, the pool is compacted
    in between: every step against the oracle over all that the stream has seen."""
    m = block(pkg, cuda_device, dtype)
    cache = pkg.PagedCache.empty(3, 80, 40, page_size=page, heads=HEADS, dtype=TORCH_DTYPE[dtype], device=cuda_device)
    gen = torch.Generator().manual_seed(1)
    seen = {}

    def step(slot, frames, kept, seed, preserve=False):
        plan = merge_plan(pkg, oracle, cuda_device, frames, kept, seed, preserve=preserve) if kept else None
        x = torch.randn(1, frames * FRAME if kept else frames, DIM, generator=gen).to(cuda_device, TORCH_DTYPE[dtype])
        with torch.no_grad():
            y = m.stream(x, cache, torch.tensor([slot], device=cuda_device), token_plan=plan)
            (q, k, v), _ = compact(pkg, m, m.qkv_projection(x), plan)
        mass = to_np(plan.key_log_mass[0]) if kept else np.zeros(len(k), np.float32)
        old = seen.get(slot)
        seen[slot] = [k, v, mass] if old is None else [np.concatenate(ab) for ab in zip(old, (k, v, mass))]
        ref, bound = attend(oracle, q, *seen[slot], dtype)
        close(y[0] if preserve or not kept else y[0][plan.keep[0]], ref, bound)
        assert y.shape == x.shape and cache.length[slot].item() == len(seen[slot][0])

    step(0, 2, 70, 10)
    step(1, 1, 33, 11)
    step(0, 1, 40, 12, preserve=True)
    cache.fork([0], [2])
    seen[2] = seen[0]
    step(2, 1, 31, 13)
    step(0, 1, 0, 14)  # one token as it is
    cache.free([1])
    del seen[1]
    used = cache.compact()
    shared = len(seen[0][0]) // page
    assert shared <= int(used) <= -(-len(seen[0][0]) // page) + -(-len(seen[2][0]) // page)
    step(2, 7, 0, 15)
    step(1, 1, 45, 16)
    step(0, 2, 55, 17)
    assert pkg.device_error_flags() == 0


def test_streams_side_by_side(pkg, oracle, cuda_device):
    """Ragged chunks of three streams in one call, token by token and with a cap."""
    m = block(pkg, cuda_device, "bf16")
    cache = pkg.PagedCache.empty(4, 20, 8, page_size=16, heads=HEADS, device=cuda_device)
    gen = torch.Generator().manual_seed(2)
    slots, seen = [3, 0, 2], {s: None for s in (3, 0, 2)}
    for counts in ([20, 1, 33], [1, 1, 1], [0, 17, 5]):
        cut = np.concatenate([[0], np.cumsum(counts)]).tolist()
        x = torch.randn(1, cut[-1], DIM, generator=gen).to(cuda_device, torch.bfloat16)
        with torch.no_grad():
            y = m.stream(x, cache, slots, cut, causal=True, softcap=3.0)
            (q, k, v), _ = compact(pkg, m, m.qkv_projection(x), None)
        for i, s in enumerate(slots):
            a, b = cut[i], cut[i + 1]
            seen[s] = (k[a:b], v[a:b]) if seen[s] is None else tuple(np.concatenate(t) for t in zip(seen[s], (k[a:b], v[a:b])))
            L = len(seen[s][0])
            if b > a:
                ref, bound = attend(oracle, q[a:b], *seen[s], None, "bf16", np.array([[0, L - (b - a) + j + 1] for j in range(b - a)]),
                                    softcap=3.0)
                close(y[0, a:b], ref, bound)
    assert pkg.device_error_flags() == 0


def test_recorded_stream_step(pkg, oracle, cuda_device):
    """A frame's step recorded once and replayed for every new frame gives the eager step's rows and cache."""
    m = block(pkg, cuda_device, "bf16")
    plan = merge_plan(pkg, oracle, cuda_device, 1, 40, 20)
    make = lambda: pkg.PagedCache.empty(1, 40, 40, page_size=16, heads=HEADS, device=cuda_device)  # noqa: E731
    cache, other = make(), make()
    slot = torch.zeros(1, device=cuda_device, dtype=torch.int32)
    x = torch.zeros(1, FRAME, DIM, device=cuda_device, dtype=torch.bfloat16)
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad(), torch.cuda.stream(side):
        m.stream(x, cache, slot, token_plan=plan)  # warm up, then empty again
        cache.free(slot)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        y = m.stream(x, cache, slot, token_plan=plan)
    gen = torch.Generator().manual_seed(3)
    for f in range(6):
        new = torch.randn(1, FRAME, DIM, generator=gen).to(cuda_device, torch.bfloat16)
        x.copy_(new)
        graph.replay()
        with torch.no_grad():
            ref = m.stream(new, other, slot, token_plan=plan)
        assert torch.equal(y, ref) and cache.length.item() == other.length.item() == 40 * (f + 1)
    for a, b in ((cache.k, other.k), (cache.v, other.v), (cache.table, other.table), (cache.references, other.references)):
        assert torch.equal(a[:15], b[:15])
    assert pkg.device_error_flags() == 0


def test_copies_of_a_cache(pkg, oracle, cuda_device):
    """A deep copy owns its pages: both go on by themselves."""
    rng = np.random.default_rng(9)
    cache = pkg.PagedCache.empty(2, 6, 3, page_size=16, heads=HEADS, device=cuda_device)
    t = lambda n: torch.from_numpy(rng.standard_normal((n, HEADS, 64)).astype(np.float32)).to(cuda_device, torch.bfloat16)  # noqa: E731
    k = t(20)
    cache.append([0], [0, 20], k, k)
    other = __import__("copy").deepcopy(cache)
    cache.free([0])
    cache.append([1], [0, 40], t(40), t(40))
    q = t(1)
    ref, bound = attend(oracle, to_np(q), to_np(k), to_np(k), None, "bf16")
    close(pkg.paged_attention(q, other, [0], [0, 1]), ref, bound)
    assert other.length.tolist() == [20, 0] and cache.length.tolist() == [0, 40] and pkg.device_error_flags() == 0
    with pytest.raises(AttributeError):
        cache.k = other.k


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_hard_merged_clips_and_streams(pkg, oracle, cuda_device, dtype):
    """A hard-merge plan has no masses: two clips under one mask (a batch), and one clip streamed."""
    rng = np.random.default_rng(12)
    N, kept = 2 * FRAME, 60
    m = block(pkg, cuda_device, dtype)
    keep = np.stack([np.sort(rng.choice(N, kept, replace=False)) for _ in range(2)])
    inverse = rng.integers(0, kept, (2, N))
    for b in range(2):
        inverse[b, keep[b]] = np.arange(kept)
    t = lambda a: torch.from_numpy(a).to(cuda_device)  # noqa: E731
    plan = pkg.TokenPlan(t(keep), t(inverse), N)
    one = pkg.TokenPlan(t(keep[:1]), t(inverse[:1]), N)
    x = t(rng.standard_normal((2, N, DIM)).astype(np.float32)).to(TORCH_DTYPE[dtype])
    ranges = pkg.attention_ranges(N, step=FRAME, device=cuda_device)
    ab = __import__("importlib").import_module(pkg.__name__ + ".attention_block")
    cache = pkg.PagedCache.empty(1, 10, 10, page_size=16, heads=HEADS, dtype=TORCH_DTYPE[dtype], masses=False, device=cuda_device)
    with torch.no_grad():
        y = m(x, plan, pkg.AttentionMask(key_range=ranges))
        rows = ab._compact_rows(*ab._dense_rows(m.qkv_projection(x), HEADS, m.q_norm, m.k_norm), plan)
        z = m.stream(x[:1], cache, [0], token_plan=one)
        single = ab._compact_rows(*ab._dense_rows(m.qkv_projection(x[:1]), HEADS, m.q_norm, m.k_norm), one)
    for b in range(2):
        own = to_np(ranges).astype(int)[keep[b]]
        seen = np.array([[(keep[b] < lo).sum(), (keep[b] < hi).sum()] for lo, hi in own])
        q, k, v = (to_np(r[b]).reshape(kept, HEADS, 64) for r in rows)
        ref, bound = attend(oracle, q, k, v, None, dtype, seen)
        close(y[b][t(keep[b])], ref, bound)
    q, k, v = (to_np(r[0]).reshape(kept, HEADS, 64) for r in single)
    ref, bound = attend(oracle, q, k, v, None, dtype)
    close(z[0][t(keep[0])], ref, bound)
    assert cache.length.item() == kept and pkg.device_error_flags() == 0


def test_rows_outside_the_chunks(pkg, oracle, cuda_device):
    """A padded batch: rows before the first chunk and behind the last are those of a row without keys, whatever memory they got."""
    m = block(pkg, cuda_device, "bf16")
    cache = pkg.PagedCache.empty(3, 20, 8, page_size=16, heads=HEADS, device=cuda_device)
    n, cut = 300, [4, 20, 20, 50]
    x = torch.randn(1, n, DIM, generator=torch.Generator().manual_seed(4)).to(cuda_device, torch.bfloat16)
    with torch.no_grad():
        for _ in range(3):
            stale = [torch.full((n, HEADS, 64), float("nan"), device=cuda_device, dtype=torch.bfloat16) for _ in range(8)]
            del stale
            y = m.stream(x, cache, [2, 1, 0], cut, causal=True)
            empty = m.proj(torch.zeros(1, DIM, device=cuda_device, dtype=torch.bfloat16))
            outside = torch.cat([y[0, :4], y[0, 50:]])
            assert torch.equal(outside, empty.expand_as(outside)) and bool(torch.isfinite(y).all())
    assert cache.length.tolist() == [90, 0, 48] and pkg.device_error_flags() == 0
