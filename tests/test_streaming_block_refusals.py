"""Argument checks of the block's mask and of its streamed form, and the merged places of a mask; no GPU."""
from __future__ import annotations

import numpy as np
import pytest
import torch


def test_mask_refusals(pkg):
    m = pkg.GlobalAttention(128, 2)
    x = torch.zeros(1, 6, 128)
    ints = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    for bad in (ints(5, 2), ints(2, 6, 2), ints(6), torch.zeros(6, 2), torch.zeros(6, 2, dtype=torch.int64)):
        with pytest.raises(ValueError, match="key_range"):
            m(x, mask=pkg.AttentionMask(key_range=bad))
    with pytest.raises(ValueError, match="position"):
        m(x, mask=pkg.AttentionMask(position=torch.zeros(6)))
    with pytest.raises(ValueError, match="position"):
        m(x, mask=pkg.AttentionMask(position=torch.zeros(5), distance_slope=torch.zeros(2)))
    with pytest.raises(ValueError, match="distance_slope"):
        m(x, mask=pkg.AttentionMask(distance_slope=torch.zeros(3)))
    with pytest.raises(ValueError, match="softcap"):
        m(x, mask=pkg.AttentionMask(softcap=-1.0))


def test_mask_at_merged_tokens(pkg):
    """Intervals, counted by hand, and positions of rows and keys that stand at some tokens of the clip."""
    rng = np.random.default_rng(0)
    N = 40
    keep = np.stack([np.sort(rng.choice(N, 9, replace=False)) for _ in range(2)])
    rows = np.stack([rng.choice(N, 5) for _ in range(2)])
    pos = torch.from_numpy(rng.standard_normal(N).astype(np.float32))
    t = torch.from_numpy
    for kr in (pkg.attention_ranges(N, step=7, window=12), torch.stack([pkg.attention_ranges(N, step=1), pkg.attention_ranges(N, step=10)])):
        mask = pkg.AttentionMask(key_range=kr, distance_slope=torch.zeros(2), position=pos)
        got = mask._scores(t(rows), t(keep))
        dense = mask._scores(t(rows), None)
        for b in range(2):
            own = (kr[b] if kr.ndim == 3 else kr).numpy()[rows[b]]
            assert dense["key_range"][b].tolist() == own.tolist() and dense["key_position"] is pos
            assert got["key_range"][b].tolist() == [[(keep[b] < lo).sum(), (keep[b] < hi).sum()] for lo, hi in own]
            assert got["key_range"].dtype == torch.int32
            assert torch.equal(got["key_position"][b], pos[t(keep[b])]) and torch.equal(got["query_position"][b], pos[t(rows[b])])
    got = pkg.AttentionMask(distance_slope=torch.zeros(2))._scores(t(rows), t(keep))
    assert got["query_position"].tolist() == rows.tolist() and got["key_position"].tolist() == keep.tolist() and "key_range" not in got


def test_stream_refusals(pkg):
    m = pkg.GlobalAttention(128, 2)
    x = torch.zeros(1, 6, 128)

    class Plan:
        dense_special_queries = True

    with pytest.raises(ValueError, match="x must be"):
        m.stream(x[0], None, [0])
    with pytest.raises(ValueError, match="x must be"):
        m.stream(x.expand(2, -1, -1), None, [0])
    with pytest.raises(ValueError, match="offsets are needed"):
        m.stream(x, None, [0, 1])
    with pytest.raises(ValueError, match="dense special"):
        m.stream(x, None, [0], token_plan=Plan())
    Plan.dense_special_queries = False
    with pytest.raises(ValueError, match="one stream"):
        m.stream(x, None, [0, 1], token_plan=Plan())
    with pytest.raises(ValueError, match="one stream"):
        m.stream(x, None, [0], token_plan=Plan(), causal=True)
    with pytest.raises(ValueError, match="one chunk"):
        m.stream(x, None, [0], [0, 6], token_plan=Plan())


def test_output_refusals(pkg):
    q = torch.zeros(1, 4, 3, 64)
    with pytest.raises(ValueError, match="broadcast"):
        pkg.masked_attention(q, q, q, out=torch.zeros(1, 1, 1, 64).expand(1, 4, 3, 64))
    for i in range(3):
        x = [torch.zeros(1, 4, 3, 64) for _ in range(3)]
        with pytest.raises(ValueError, match="share memory"):
            pkg.masked_attention(*x, out=x[i])


def test_a_refused_stream_step_leaves_the_cache(pkg):
    """What the attention would refuse after the append is refused before it."""
    m = pkg.GlobalAttention(128, 2)

    class Cache:
        k = torch.zeros(4, 16, 2, 64)

        def append(self, *args):
            raise AssertionError("the cache was written")

    x = torch.zeros(1, 6, 128)
    for cap in (0.0, -1.0, float("nan")):
        with torch.no_grad(), pytest.raises(ValueError, match="softcap"):
            m.stream(x, Cache(), [0], softcap=cap)
    m.requires_grad_(False)
    m.q_norm.weight.requires_grad_()  # the queries alone require a gradient
    with pytest.raises(RuntimeError, match="no backward"):
        m.stream(x, Cache(), [0])
