"""Masked attention on the GPU against its definition in 64 bits (``oracle.streaming``): types, head layouts, masks that
leave rows empty, caps, distances, biases, strides, values that must not reach a row, graphs and streams.

The tolerance of every element is the oracle's bound, counted from the roundings that the kernels make."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import TORCH_DTYPE, to_np

pytestmark = pytest.mark.gpu


def make(seed, B, H, Hkv, Nq, Nk, dtype, oracle, q_scale=2.0):
    rng = np.random.default_rng(seed)
    q = rng.standard_normal((B, H, Nq, 64)).astype(np.float32) * q_scale
    k = rng.standard_normal((B, Hkv, Nk, 64)).astype(np.float32)
    v = rng.standard_normal((B, Hkv, Nk, 64)).astype(np.float32)
    return rng, *(oracle.round_to(t, dtype) for t in (q, k, v))


def gpu(t, device, dtype=None):
    return None if t is None else torch.from_numpy(np.ascontiguousarray(t)).to(device=device, dtype=dtype)


def check(got, ref, bound):
    got = to_np(got) if isinstance(got, torch.Tensor) else got
    over = np.abs(got - ref) - bound
    assert np.isfinite(got).all(), f"{np.sum(~np.isfinite(got))} values are not finite"
    assert over.max(initial=-1.0) <= 0, f"{np.sum(over > 0)} values off by up to {over.max():.3e} more than their bound"


def run(pkg, oracle, device, dtype, q, k, v, bias=None, ranges=None, slope=None, qpos=None, kpos=None, **kw):
    td = TORCH_DTYPE[dtype]
    out = pkg.masked_attention(gpu(q, device, td), gpu(k, device, td), gpu(v, device, td), gpu(bias, device),
                               key_range=gpu(ranges, device), distance_slope=gpu(slope, device), query_position=gpu(qpos, device),
                               key_position=gpu(kpos, device), **kw)
    assert out.dtype == td and out.shape == q.shape
    ref, bound = oracle.streaming.masked_attention(q, k, v, bias, ranges, slope=slope, qpos=qpos, kpos=kpos, dtype=dtype, **kw)
    check(out, ref, bound)
    assert pkg.device_error_flags() == 0
    return out


SHAPES = [  # B, H, Hkv, Nq, Nk
    (1, 1, 1, 1, 1),
    (1, 4, 1, 2, 7),      # eight row x head pairs over a few keys
    (2, 2, 2, 1, 1000),   # single rows, keys split
    (1, 6, 2, 9, 129),
    (2, 4, 2, 130, 257),  # a second query tile with two rows, ragged tails
    (1, 3, 3, 300, 300),
    (1, 2, 1, 17, 1041),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_plain(pkg, oracle, cuda_device, dtype, shape):
    _, q, k, v = make(sum(shape), *shape, dtype, oracle)
    run(pkg, oracle, cuda_device, dtype, q, k, v)


MASKS = {
    "causal": dict(step=1),
    "frames": dict(step=17),
    "documents": dict(documents=[0, 5, 5, 140, 141, 333]),
    "document frames prefix": dict(documents=[0, 100, 333], step=30, prefix=7),
    "prefix": dict(step=1, prefix=130),
    "window": dict(step=1, window=3),
    "window of a document": dict(documents=[0, 128, 333], window=150),
}


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("mask", sorted(MASKS))
@pytest.mark.parametrize("queries", [333, 5])
def test_masks(pkg, oracle, cuda_device, dtype, mask, queries):
    spec = dict(MASKS[mask])
    if "documents" in spec:
        spec["documents"] = torch.tensor(spec["documents"], device=cuda_device)
    ranges = pkg.attention_ranges(queries, 333, device=cuda_device, **spec).cpu().numpy()
    rng, q, k, v = make(3, 1, 4, 2, queries, 333, dtype, oracle)
    mass = np.log(rng.integers(1, 50, 333)).astype(np.float32)
    run(pkg, oracle, cuda_device, dtype, q, k, v, mass, ranges)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("queries", [200, 3])
def test_empty_and_odd_ranges(pkg, oracle, cuda_device, dtype, queries):
    """Rows that see nothing, ranges beyond the keys, reversed ones, a hole between the rows' keys, per batch entry."""
    rng, q, k, v = make(4, 2, 2, 2, queries, 700, dtype, oracle)
    r = np.sort(rng.integers(-5, 720, (2, queries, 2)), axis=2).astype(np.int32)
    r[:, ::7] = 50
    r[:, 1::11] = [300, 20]
    r[:, 2::13] = [690, 5000]
    r[0, queries // 2:] = [600, 640]
    out = run(pkg, oracle, cuda_device, dtype, q, k, v, None, r)
    empty = torch.from_numpy(np.minimum(r[..., 1], 700) <= np.maximum(r[..., 0], 0)).to(cuda_device)
    assert bool(empty.any()) and bool((out.transpose(1, 2)[empty] == 0).all())
    r[:] = 5
    out = run(pkg, oracle, cuda_device, dtype, q, k, v, None, r)  # no row sees a key
    assert (out == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("queries", [180, 2])
@pytest.mark.parametrize("softcap,dist,mass", [(20.0, False, False), (None, True, False), (5.0, True, True), (100.0, False, True)])
def test_scores(pkg, oracle, cuda_device, dtype, queries, softcap, dist, mass):
    rng, q, k, v = make(5, 2, 4, 4, queries, 400, dtype, oracle, q_scale=6.0)
    bias = np.log(rng.integers(1, 50, (2, 400))).astype(np.float32) if mass else None
    slope = np.array([0.5, 0.25, 0.01, -0.003], np.float32) if dist else None
    kpos = np.sort(rng.uniform(0, 60, (2, 400))).astype(np.float32) if dist and mass else None
    qpos = rng.uniform(0, 60, queries).astype(np.float32) if dist and mass else None
    r = pkg.attention_ranges(queries, 400, step=1, device=cuda_device).cpu().numpy()
    run(pkg, oracle, cuda_device, dtype, q, k, v, bias, r, slope=slope, qpos=qpos, kpos=kpos, softcap=softcap, scale=0.2)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("queries", [150, 2])
def test_extreme_biases(pkg, oracle, cuda_device, dtype, queries):
    """Masses of zero (bias -inf) hide a key; the type's lowest value outweighs every score but not another such key."""
    rng, q, k, v = make(6, 3, 2, 2, queries, 300, dtype, oracle)
    bias = np.zeros((3, 300), np.float32)
    bias[0, ::2] = -np.inf
    bias[0, 1::4] = np.finfo(np.float32).min
    bias[1] = np.finfo(np.float32).min
    bias[2] = -np.inf
    v[2] = np.nan
    v[0, :, ::2] = np.nan
    k[0, :, ::4] = np.inf
    out = run(pkg, oracle, cuda_device, dtype, q, k, v, bias)
    assert (out[2] == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("queries", [150, 2])
@pytest.mark.parametrize("softcap", [None, 30.0])
def test_mask_constants(pkg, oracle, cuda_device, dtype, queries, softcap):
    """Large biases that programs use as masks, alone in a row and beside others, and rows that only see such keys."""
    rng, q, k, v = make(14, 1, 2, 2, queries, 260, dtype, oracle)
    bias = rng.choice([0.0, -1e4, -1e9, -7600.0, -3e38, -np.inf, 2.0], 260).astype(np.float32)
    bias[:130] = -1e4 - np.arange(130) / 8
    bias[20:40] = -1e9
    bias[40:60] = -2e30
    r = np.stack([rng.integers(0, 60, queries), rng.integers(60, 261, queries)], 1).astype(np.int32)
    r[::3] = [20, 40]
    r[1::5] = [30, 60]
    run(pkg, oracle, cuda_device, dtype, q, k, v, bias, r, softcap=softcap)
    bias[200], bias[7] = 3e38, 1e33
    run(pkg, oracle, cuda_device, dtype, q, k, v, bias, r, softcap=softcap)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("softcap", [0.01, 1.0, 4.0, 9.0, 400.0, 1e5, 1e12])
def test_caps_of_any_size(pkg, oracle, cuda_device, dtype, softcap):
    _, q, k, v = make(15, 1, 2, 2, 140, 200, dtype, oracle, q_scale=8.0)
    run(pkg, oracle, cuda_device, dtype, q, k, v, softcap=softcap)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("queries", [333, 4])
def test_hidden_values_do_not_reach_a_row(pkg, oracle, cuda_device, dtype, queries):
    """NaN and infinities in keys and values that a row does not see, in the tiles that it reads."""
    docs = torch.tensor([0, 20, 150, 151, 333], device=cuda_device)
    r = pkg.attention_ranges(queries, 333, documents=docs, step=1, device=cuda_device).cpu().numpy()
    _, q, k, v = make(7, 1, 2, 2, queries, 333, dtype, oracle)
    clean = run(pkg, oracle, cuda_device, dtype, q, k, v, None, r)
    td = TORCH_DTYPE[dtype]
    bad_k, bad_v = k.copy(), v.copy()
    bad_k[:, :, 332], bad_v[:, :, 332] = np.nan, np.inf   # the last key: only the last row sees it
    bad_v[:, 0, 25, 3] = -np.inf                            # a key of document 1: its rows from 25 on see it
    bad_k[:, 1, 7] = np.inf
    got = pkg.masked_attention(gpu(q, cuda_device, td), gpu(bad_k, cuda_device, td), gpu(bad_v, cuda_device, td),
                               key_range=gpu(r, cuda_device))
    sees = np.zeros((1, 2, queries), bool)
    for h, j in ((0, 332), (1, 332), (0, 25), (1, 7)):
        sees[0, h] |= (r[:, 0] <= j) & (j < r[:, 1])
    sees = torch.from_numpy(sees).to(cuda_device)
    same = (got == clean).all(-1) | sees
    assert bool(same.all()) or torch.allclose(got[~sees].float(), clean[~sees].float(), rtol=2.0 ** -7, atol=2.0 ** -8)
    assert bool(torch.isfinite(got[~sees]).all()) and not bool(torch.isfinite(got[sees]).all(-1).any())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("queries", [300, 4])
def test_hidden_values_of_any_size(pkg, oracle, cuda_device, dtype, queries):
    """Hidden keys and values near the largest finite number, beside rows whose scores are far below zero."""
    r = pkg.attention_ranges(queries, 300, step=1, window=40, device=cuda_device).cpu().numpy()
    rng, q, k, v = make(12, 1, 2, 2, queries, 300, dtype, oracle)
    bias = np.where(np.arange(300) % 3 == 0, -np.inf, -300.0).astype(np.float32)
    v[:, :, ::3] = 3e38
    k[:, :, ::6] = 3e38
    run(pkg, oracle, cuda_device, dtype, q, k, v, bias, r)
    first = 300 - queries
    r[:] = [0, first + 1]
    r[1:, 1] = first  # only the first row sees the key at its own place
    v[:, :, first] = 3e38
    bias[first] = -np.inf if dtype == "f32" else 0.0
    out = run(pkg, oracle, cuda_device, dtype, q[:, :, 1:], k, v, bias, r[1:]) if queries > 4 else None
    assert out is None or bool((out.abs() < 100).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_strides(pkg, oracle, cuda_device, dtype):
    """Views of a packed q | k | v buffer, a broadcast batch of keys, rows that are not 16-byte aligned, a given output."""
    td = TORCH_DTYPE[dtype]
    rng = np.random.default_rng(8)
    x = oracle.round_to(rng.standard_normal((2, 150, 3 * 4 * 64)).astype(np.float32), dtype)
    t = gpu(x, cuda_device, td).view(2, 150, 3, 4, 64)
    q, k, v = (t[:, :, i].transpose(1, 2) for i in range(3))
    npy = [to_np(y) for y in (q, k, v)]
    ref, bound = oracle.streaming.masked_attention(*npy, dtype=dtype)
    buf = torch.full((2, 152, 4, 64), 7.0, device=cuda_device, dtype=td)
    out = buf[:, 1:151].transpose(1, 2)
    assert pkg.masked_attention(q, k, v, out=out) is out
    check(out, ref, bound)
    assert bool((buf[:, 0] == 7).all()) and bool((buf[:, 151] == 7).all())  # what lies beside is left as it was
    kb, vb = k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1)
    ref, bound = oracle.streaming.masked_attention(npy[0], npy[1][[0, 0]], npy[2][[0, 0]], dtype=dtype)
    check(pkg.masked_attention(q, kb, vb), ref, bound)
    odd = torch.empty(2 * 4 * 150 * 65, device=cuda_device, dtype=td)[1:1 + 2 * 4 * 150 * 64].view(2, 4, 150, 64)
    odd.copy_(q)
    ref, bound = oracle.streaming.masked_attention(*npy, dtype=dtype)
    check(pkg.masked_attention(odd, k, v), ref, bound)


@pytest.mark.parametrize("dtype,queries", [("bf16", 40), ("bf16", 2), ("f32", 2)])
def test_offsets_beyond_32_bits(pkg, oracle, cuda_device, dtype, queries):
    """Keys whose rows lie more than 2^32 bytes (and elements) apart."""
    td = TORCH_DTYPE[dtype]
    Nk, stride = 200, (1 << 32) // 192 // 64 * 64
    base = torch.zeros(Nk * stride + 64, device=cuda_device, dtype=td)
    _, q, k, v = make(9, 1, 1, 1, queries, Nk, dtype, oracle)
    kk = base.as_strided((1, 1, Nk, 64), (0, 0, stride, 1))
    kk.copy_(gpu(k, cuda_device, td))
    ref, bound = oracle.streaming.masked_attention(q, k, v, dtype=dtype)
    check(pkg.masked_attention(gpu(q, cuda_device, td), kk, gpu(v, cuda_device, td)), ref, bound)
    check(pkg.masked_attention(gpu(q, cuda_device, td), gpu(k, cuda_device, td), kk), *oracle.streaming.masked_attention(q, k, k, dtype=dtype))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_no_rows_and_no_keys(pkg, cuda_device, dtype):
    td = TORCH_DTYPE[dtype]
    z = lambda *s: torch.ones(s, device=cuda_device, dtype=td)  # noqa: E731
    assert pkg.masked_attention(z(1, 2, 0, 64), z(1, 2, 5, 64), z(1, 2, 5, 64)).shape == (1, 2, 0, 64)
    assert bool((pkg.masked_attention(z(1, 2, 3, 64), z(1, 2, 0, 64), z(1, 2, 0, 64)) == 0).all())
    assert pkg.masked_attention(z(0, 2, 3, 64), z(0, 2, 5, 64), z(0, 2, 5, 64)).numel() == 0


@pytest.mark.parametrize("queries", [300, 3])
def test_repeatable_graph_and_stream(pkg, cuda_device, queries):
    """The same bits from a second call, from a replayed graph with refilled inputs, from another stream and from two
    graphs replayed at once."""
    g = torch.Generator(device=cuda_device).manual_seed(1)
    new = lambda n: torch.randn(1, 4, n, 64, generator=g, device=cuda_device).bfloat16()  # noqa: E731
    q, k, v = new(queries), new(900), new(900)
    mass = torch.rand(900, generator=g, device=cuda_device)
    r = pkg.attention_ranges(queries, 900, step=64, device=cuda_device)
    call = lambda: pkg.masked_attention(q, k, v, mass, key_range=r, softcap=30.0)  # noqa: E731
    a, b = call(), call()
    assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, c)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call())
        graphs.append(graph)
    q.copy_(new(queries))
    k.copy_(new(900))
    ref = call()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(3):
            graphs[0].replay()
    for _ in range(3):
        graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], ref) and torch.equal(outs[1], ref)
    assert pkg.device_error_flags() == 0


def test_refusals_on_the_gpu(pkg, cuda_device):
    q = torch.zeros(1, 2, 4, 64, device=cuda_device, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no backward"):
        pkg.masked_attention(q.clone().requires_grad_(), q, q)
    with torch.no_grad():
        pkg.masked_attention(q.clone().requires_grad_(), q, q)
    with pytest.raises(ValueError, match="tensors are on"):
        pkg.masked_attention(q, q, q, torch.zeros(4))
    with pytest.raises(ValueError, match="out must"):
        pkg.masked_attention(q, q, q, out=torch.empty(1, 2, 4, 65, device=cuda_device, dtype=torch.bfloat16)[..., :64])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("softcap", [None, 4.0])
@pytest.mark.parametrize("mask", [None, dict(step=1), dict(step=200, window=500)])
def test_distance_over_whole_tiles(pkg, oracle, cuda_device, dtype, softcap, mask):
    """Tiles whose keys all lie before, behind or among the rows' positions, flat to steep slopes and one that grows with
    the distance, with a bias that hides keys and one that nearly does."""
    slope = np.array([0.0, 1e-4, 0.02, 0.7, 3.0, 40.0, -0.01, 0.2], np.float32)
    rng, q, k, v = make(31, 1, 8, 4, 700, 1100, dtype, oracle, q_scale=1.0)
    bias = np.log(rng.integers(1, 9, 1100)).astype(np.float32)
    bias[[3, 500, 1099]] = -np.inf
    bias[[4, 501, 1098]] = np.finfo(np.float32).min
    ranges = None if mask is None else to_np(pkg.attention_ranges(700, 1100, **mask)).astype(np.int32)
    for b in (bias, None):
        run(pkg, oracle, cuda_device, dtype, q, k, v, b, ranges, slope=slope, softcap=softcap)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("softcap", [None, 3.0, 60.0])
@pytest.mark.parametrize("growth", [0.02, -0.02, 0.3])
def test_maxima_that_keep_growing(pkg, oracle, cuda_device, dtype, softcap, growth):
    """Scores that rise (or fall) along the keys by far more than the running maximum leaves room for, in steps of one row or
    of all, so that parts of a tile, the first or the last, have to be taken again."""
    rng, q, k, v = make(32, 1, 2, 2, 256, 1000, dtype, oracle, q_scale=1.0)
    lift = np.arange(1000, dtype=np.float32) * growth
    q[..., 0], k[..., 0] = 8.0, oracle.round_to(lift % 50 if growth == 0.3 else lift, dtype)
    q[:, :, 5::7, 0] = 0.0  # rows whose scores do not rise
    run(pkg, oracle, cuda_device, dtype, q, k, v, softcap=softcap)
    bias = oracle.round_to(rng.standard_normal(1000).astype(np.float32) * 9, "f32")
    run(pkg, oracle, cuda_device, dtype, q, k, v, bias, softcap=softcap)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("what", ["far below", "nan", "massless"])
def test_keys_that_the_polynomial_does_not_take(pkg, oracle, cuda_device, dtype, what):
    """Keys in tiles that every row sees whole, one in each place of a tile: scores far below the maximum, NaN (whose rows are
    NaN, and only those), mass 0."""
    rng, q, k, v = make(41, 1, 2, 1, 300, 1024, dtype, oracle, q_scale=1.0)
    odd = 256 + 129 * np.arange(5)  # tiles 2 to 6, other places of the tile
    odd = np.concatenate([odd + i for i in range(0, 24, 3)])
    bias = np.zeros(1024, np.float32)
    if what == "far below":
        bias[odd] = -150.0
    elif what == "massless":
        bias[odd] = -np.inf
    else:
        k[0, 0, odd[::9]] = np.nan
        ranges = np.tile(np.array([[0, 1024]], np.int32), (300, 1))
        ranges[:7, 1] = 256  # these rows do not see them
        out = pkg.masked_attention(*(gpu(t, cuda_device, TORCH_DTYPE[dtype]) for t in (q, k, v)), key_range=gpu(ranges, cuda_device))
        out = to_np(out)
        assert np.isnan(out[:, :, 7:]).all()
        ref, bound = oracle.streaming.masked_attention(q[:, :, :7], k[:, :, :256], v[:, :, :256], dtype=dtype)
        check(out[:, :, :7], ref, bound)
        return
    run(pkg, oracle, cuda_device, dtype, q, k, v, bias)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,queries", [(2, 300), (1, 2)])
@pytest.mark.parametrize("top", [[0], [20000], [32927], range(5, 32928, 144)], ids=["first", "inside", "last", "many"])
@pytest.mark.parametrize("depth", [12.0, 13.0, 14.5])
@pytest.mark.parametrize("softcap", [None, 60.0])
def test_small_probabilities_add_up(pkg, oracle, cuda_device, dtype, heads, queries, top, depth, softcap):
    """Keys that stand 12 to 14.5 nats above the other ones of 32,928, which have one score, so that their probabilities round the
    same way.  The high keys' values are 0, so the output is what the small probabilities add up to.

    Tolerance, relative to the output (all values are positive): each probability and the result are rounded once, 2 * eps / 2 and 1%
    for the second order; the exponential may be a polynomial (2^-13), and the sum that it is divided by too; scores are sums of one
    product and zeros, at most 16 long and rounded 16 times; sums of n terms round at most n / 16 + 128 times.  Besides, fp16
    rounds to its step 2^-24: with the largest probability kept above 2^3, each of at most four roundings takes 2^-25 / 2^3 of it
    from a key's."""
    n, top = 32928, list(top)
    q, k = np.zeros((1, heads, queries, 64), np.float32), np.zeros((1, 1, n, 64), np.float32)
    q[..., 0] = 8.0
    k[0, 0, :, 0] = -depth
    k[0, 0, top, 0] = 0.0
    v = oracle.round_to((np.abs(np.random.default_rng(queries).standard_normal((1, 1, n, 64))) + 0.5).astype(np.float32), dtype)
    v[0, 0, top] = 0.0
    td = TORCH_DTYPE[dtype]
    got = to_np(pkg.masked_attention(*(gpu(t, cuda_device, td) for t in (q, k, v)), softcap=softcap))
    x = k[0, 0, :, 0].astype(np.float64)
    x = x if softcap is None else softcap * np.tanh(x / softcap)
    p = np.exp(x) / np.exp(x).sum()
    want = p @ v[0, 0].astype(np.float64)
    half, u = oracle.streaming.EPS_HALF[dtype], 2.0 ** -24
    rel = 2.02 * half + 2 * (2.0 ** -13 + 16 * 16 * u + (n / 16 + 128) * u + (0 if softcap is None else softcap * 2.0 ** -21))
    # the result's own smallest step: 2^-25
    step = 4 * 2.0 ** -28 * p.max() * v[0, 0].sum(0) + 2.0 ** -25 if dtype == "f16" else 0.0
    assert (np.abs(got - want) <= rel * want + step).all(), np.abs(got / want - 1).max()
    assert pkg.device_error_flags() == 0


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("queries", [300, 2])
@pytest.mark.parametrize("scale", [1e-30, 1e-5, 2.0 ** -9, 1 / 64, 0.125])
@pytest.mark.parametrize("dist", [False, True])
def test_biases_at_any_scale(pkg, oracle, cuda_device, dtype, queries, scale, dist):
    """Biases and distances of ordinary size beside products of any scale: bias / scale leaves the range of fp16 and of bf16."""
    rng, q, k, v = make(51, 1, 2, 2, queries, 400, dtype, oracle)
    bias = rng.choice([0.0, -0.7, -1.3, 1.0, -30.0], 400).astype(np.float32)
    slope = np.array([0.01, 0.3], np.float32) if dist else None
    run(pkg, oracle, cuda_device, dtype, q, k, v, bias, slope=slope, scale=scale)
    if dist:
        run(pkg, oracle, cuda_device, dtype, q, k, v, slope=slope, scale=scale)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("queries", [300, 2])
@pytest.mark.parametrize("size", [160.0, 248.0, 504.0])
def test_biases_that_products_outweigh(pkg, oracle, cuda_device, dtype, queries, size):
    """Keys whose products with the queries are as large as their bias is low (3,200 to 31,752 nats), beside keys without either."""
    rng, q, k, v = make(52, 1, 2, 2, queries, 400, dtype, oracle, q_scale=1.0)
    bias = np.zeros(400, np.float32)
    q[..., 0] = size
    k[..., 0] = 0.0
    k[:, :, 7::50, 0] = size
    bias[7::50] = -size * size / 8 + rng.uniform(-2, 2, 8)
    run(pkg, oracle, cuda_device, dtype, q, k, v, bias)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("mass", [False, True])
def test_parts_without_keys(pkg, oracle, cuda_device, dtype, mass):
    """A block in parts whose rows see a few keys at both ends, so that the parts in between have no tile and reach the
    joining at once: the same bits every time, and right."""
    rng, q, k, v = make(61, 1, 4, 4, 256, 9000, dtype, oracle)
    bias = np.log(rng.integers(1, 9, 9000)).astype(np.float32) if mass else None
    r = np.zeros((256, 2), np.int32)
    r[:128] = np.sort(rng.integers(0, 130, (128, 2)), 1)
    r[128:] = np.sort(rng.integers(8800, 9001, (128, 2)), 1)
    first = run(pkg, oracle, cuda_device, dtype, q, k, v, bias, r)
    td = TORCH_DTYPE[dtype]
    args = [gpu(t, cuda_device, td) for t in (q, k, v)]
    b, kr = gpu(bias, cuda_device), gpu(r, cuda_device)
    outs = [pkg.masked_attention(*args, b, key_range=kr) for _ in range(200)]
    assert all(torch.equal(o, first) for o in outs) and pkg.device_error_flags() == 0


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("queries", [300, 2])
@pytest.mark.parametrize("softcap", [50.0, 3e3, 3e4, 1e5, 1e6, 1e9, 1e30])
def test_scores_far_below_the_cap(pkg, oracle, cuda_device, dtype, queries, softcap):
    """A cap that scores hardly reach, down to one that changes nothing, leaves them their bits."""
    rng, q, k, v = make(71, 1, 2, 2, queries, 300, dtype, oracle)
    run(pkg, oracle, cuda_device, dtype, q, k, v, softcap=softcap)
    run(pkg, oracle, cuda_device, dtype, q, k, v, np.log(rng.integers(1, 9, 300)).astype(np.float32), softcap=softcap)
    k[0, 0, 5], k[0, 1, 200] = np.nan, np.nan  # exact_row: the rows that do not see these keys
    r = np.tile(np.array([[6, 200]], np.int32), (queries, 1))
    v[0, 0, 5], v[0, 1, 200] = np.nan, np.nan
    run(pkg, oracle, cuda_device, dtype, q, k, v, None, r, softcap=softcap)


@pytest.mark.parametrize("dtype,queries,page", [("bf16", 600, 0), ("f16", 600, 0), ("bf16", 3, 0), ("f32", 3, 0), ("bf16", 600, 64), ("f16", 2, 128)])
@pytest.mark.parametrize("softcap", [None, 20.0])
def test_distances_beyond_24_bits(pkg, oracle, cuda_device, dtype, queries, page, softcap):
    """More than 2^24 keys, dense and paged: the distances among the last tokens are whole numbers that fp32 positions of the
    sequence do not hold."""
    td, near = TORCH_DTYPE[dtype], 1800
    n = (1 << 24) + (1 << 20) + 3
    k, v = (torch.zeros(1, 1, -(-n // 128) * 128, 64, device=cuda_device, dtype=td) for _ in range(2))
    rng, qn, kn, vn = make(81, 1, 1, 1, queries, near, dtype, oracle, q_scale=1.0)
    k[:, :, n - near:n], v[:, :, n - near:n] = gpu(kn, cuda_device, td), gpu(vn, cuda_device, td)
    first = near - queries + np.arange(queries)
    r = np.stack([np.maximum(first - 900, 0), first + 1], 1).astype(np.int32)
    r[::3, 1] = near  # keys behind the row too
    slope = np.array([0.75], np.float32)
    q, kr, sl = gpu(qn, cuda_device, td), gpu(r + (n - near), cuda_device, torch.int32), gpu(slope, cuda_device)
    if page:
        pools = [t.view(-1, page, 1, 64) for t in (k, v)]
        pages = pools[0].shape[0]
        ints = lambda x: x.to(device=cuda_device, dtype=torch.int32)  # noqa: E731
        cache = pkg.PagedCache(*pools, None, ints(torch.arange(pages).view(1, pages)), ints(torch.tensor([n])), ints(torch.ones(pages)))
        out = pkg.paged_attention(q[0].transpose(0, 1), cache, [0], [0, queries], key_range=kr, distance_slope=sl, softcap=softcap)
        out = out.transpose(0, 1)[None]
    else:
        out = pkg.masked_attention(q, k[:, :, :n], v[:, :, :n], key_range=kr, distance_slope=sl, softcap=softcap)
    check(out, *oracle.streaming.masked_attention(qn, kn, vn, None, r, slope=slope, softcap=softcap, dtype=dtype))
    assert pkg.device_error_flags() == 0
