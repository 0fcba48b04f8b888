"""Global-attention block with a token plan, on the B200 operators.

``GlobalAttention`` holds the parameters of the reference's ``SelfAttention`` as used by the
aggregator's global blocks (vggt_omega/models/layers/attention.py:210-241 with qkv_bias,
proj_bias, mask_k_bias and use_qk_norm, as vggt_omega/models/aggregator.py:96-110 builds them)
and runs ``forward(x, token_plan=...)`` with the reference's semantics
(attention.py:264-314, 328-439):

    qkv = qkv(x)  (cuBLAS)  ->  q/k LayerNorm over the head dim
    compact:  compact-query plans compact Q, K and V; query-preserving plans keep all
              queries, physical keys (compact_key) and pooled values
    mass-bias attention over the compact keys with bias key_log_mass  (tcgen05 kernel)
    dense special queries: exact attention of the camera / register queries over the dense
              K/V (the same kernel without bias), written over their compact rows
    proj  (cuBLAS)  ->  restore  (top-4 gather kernel)

Tensors stay token-major throughout: Q/K/V are [B, T, H, 64] views of the qkv buffer and
the attention output is written token-major, so no transposes are materialised.

Two forms go beyond the reference, whose clip is there as a whole (no counterpart):

* ``mask=`` of ``forward`` and ``compute_attention``: an ``AttentionMask`` over the clip's tokens (frames in causal order,
  several clips in one sequence, windows, capped scores, a distance bias), carried over to the merged tokens of the plan;
* ``GlobalAttention.stream``: frames that arrive one after the other, merged, appended to a ``PagedCache`` and attended
  over all that the cache holds of their stream.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn.functional as F
from torch import nn

from .ops import head_layernorm, mass_bias_attention, row_gather
from .streaming import PagedCache, _positive, _refuse_gradients, masked_attention, paged_attention
from .token_plan import WeightedBilinearTokenPlan

__all__ = ["AttentionMask", "GlobalAttention", "compute_attention"]


@dataclass(frozen=True, eq=False)
class AttentionMask:
    """What a block's rows see and how their scores change, over the tokens of the clip (``attention_ranges`` makes the
    intervals, ``masked_attention`` says what the fields do).  With a token plan a merged token stands at the place of the
    token that it keeps: it is seen where that one is, and distances are those of the kept tokens.  (What a kept token
    pooled from others goes with it.)  The plan's kept tokens must ascend, as the planners make them.  Inference only: a masked
    call refuses inputs that require a gradient while gradients are recorded."""

    key_range: torch.Tensor | None = None       # int32 [N, 2] or [B, N, 2]
    softcap: float | None = None
    distance_slope: torch.Tensor | None = None  # [H]
    position: torch.Tensor | None = None        # [N] or [B, N]; by default the token index

    def _scores(self, rows: torch.Tensor | None, keys: torch.Tensor | None) -> dict:
        """Arguments of ``masked_attention`` for the query rows and keys that stand at the clip's tokens ``rows`` and
        ``keys`` ([B, .], ascending keys; None: every token, as its own key, and with ``rows`` None its own row)."""
        args = dict(softcap=self.softcap, distance_slope=self.distance_slope)
        if self.key_range is not None:
            kr = self.key_range
            if rows is not None:
                kr = kr.expand(rows.shape[0], *kr.shape[-2:]).gather(1, rows.unsqueeze(-1).expand(-1, -1, 2))
                if keys is not None:
                    kr = torch.searchsorted(keys.contiguous(), kr.flatten(1).to(keys.dtype)).view(kr.shape)
            args["key_range"] = kr.to(torch.int32)
        if self.distance_slope is not None:
            for name, at in (("query_position", rows), ("key_position", keys)):
                if at is None:
                    args[name] = self.position
                elif self.position is None:
                    args[name] = at.to(torch.float32)
                else:
                    args[name] = self.position.expand(at.shape[0], self.position.shape[-1]).gather(1, at)
        return args

    def _check(self, batch: int, tokens: int) -> None:
        kr, pos = self.key_range, self.position
        if kr is not None and (kr.dtype != torch.int32 or kr.shape not in ((tokens, 2), (batch, tokens, 2))):
            raise ValueError(f"mask: key_range must be int32 [{tokens}, 2] or [{batch}, {tokens}, 2]")
        if pos is not None and (self.distance_slope is None or pos.shape not in ((tokens,), (batch, tokens))):
            raise ValueError(f"mask: position must be [{tokens}] or [{batch}, {tokens}] and goes with distance_slope")


def _attend(q, k, v, log_key_mass, mask: AttentionMask | None, rows=None, keys=None) -> torch.Tensor:
    """The attention of a block: ``mass_bias_attention``, or with a mask ``masked_attention`` over the same inputs."""
    if mask is None:
        return mass_bias_attention(q, k, v, log_key_mass)
    dtype = q.dtype
    if dtype == torch.float32 and torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") == torch.bfloat16:
        dtype = torch.bfloat16  # as mass_bias_attention does
    bias = None if log_key_mass is None else log_key_mass.reshape(-1)
    return masked_attention(q.to(dtype), k.to(dtype), v.to(dtype), bias, **mask._scores(rows, keys))


def _places(token_plan) -> tuple[torch.Tensor, torch.Tensor]:
    """The clip's tokens at which the query rows and the compact keys of a plan stand, [B, .]."""
    keys = token_plan.keep.to(torch.int64)
    if getattr(token_plan, "preserve_queries", False):
        return torch.arange(token_plan.original_tokens, device=keys.device).expand(keys.shape[0], -1), keys
    rows = getattr(token_plan, "query_keep", None)
    return (keys if rows is None else rows.to(torch.int64)), keys


def _bhtd(x: torch.Tensor, heads: int) -> torch.Tensor:
    """[B, T, C] -> [B, H, T, d] view."""
    B, T, C = x.shape
    return x.view(B, T, heads, C // heads).transpose(1, 2)


def _ln_params(q_norm, k_norm):
    if q_norm is None or k_norm is None:
        return None, None, 1e-5
    w = torch.stack([q_norm.weight.detach(), k_norm.weight.detach()]).float()
    b = torch.stack([q_norm.bias.detach(), k_norm.bias.detach()]).float()
    return w, b, float(q_norm.eps)


def _fused_ok(qkv: torch.Tensor, token_plan, q_norm, k_norm) -> bool:
    """The one-kernel LayerNorm + Q||K||V compaction applies to 16-bit qkv buffers with a
    WeightedBilinearTokenPlan without a separate query plan."""
    if not isinstance(token_plan, WeightedBilinearTokenPlan) or token_plan.query_keep is not None:
        return False
    if qkv.dtype not in (torch.bfloat16, torch.float16) or qkv.shape[0] != 1 or (qkv.shape[2] // 3) % 256:
        return False
    if (q_norm is None) != (k_norm is None):
        return False
    return q_norm is None or (q_norm.elementwise_affine and tuple(q_norm.normalized_shape) == (64,))


def _compact_rows_fused(x, plan, q_norm, k_norm):
    """q, k, v [rows, C] of the compact attention (views of one buffer) from the rows x [N, 3C] of a qkv buffer."""
    C = x.shape[1] // 3
    lw, lb, eps = _ln_params(q_norm, k_norm)
    preserve = plan.preserve_queries
    if preserve:
        mask = 0b100 | (0 if plan.preserve_destination_keys else 0b010)
    else:
        mask = 0b111
    packed = plan.compact_qkv(x, lw, lb, eps, pool_mask=mask)  # [M, 3C]
    q = packed[:, :C]
    if preserve:
        q = head_layernorm(x[:, :C], lw[0], lb[0], eps) if lw is not None else x[:, :C]
    return q, packed[:, C:2 * C], packed[:, 2 * C:]


def _compute_attention_fused(qkv, num_heads, plan, q_norm, k_norm, mask=None):
    B, N, C3 = qkv.shape
    C = C3 // 3
    x = qkv[0]
    preserve = plan.preserve_queries
    view = lambda t, T: t.view(1, T, num_heads, C // num_heads).transpose(1, 2)
    q, k, v = _compact_rows_fused(x, plan, q_norm, k_norm)
    rows, keys = (None, None) if mask is None else _places(plan)
    o = _attend(view(q, q.shape[0]), view(k, k.shape[0]), view(v, k.shape[0]), plan.key_log_mass, mask, rows, keys)
    if plan.dense_special_queries:
        lw, lb, eps = _ln_params(q_norm, k_norm)
        original, out_index = plan.special_query_original, (
            plan.special_query_original if preserve else plan.special_query_compact)
        if original is None or out_index is None:
            raise RuntimeError("dense-special attention plan has no special-token mapping")
        qs = row_gather(x[:, :C], original)
        if lw is not None:
            qs = head_layernorm(qs, lw[0], lb[0], eps)
            kd = head_layernorm(x[:, C:2 * C], lw[1], lb[1], eps)
        else:
            kd = x[:, C:2 * C]
        exact = _attend(view(qs, qs.shape[0]), view(kd, N), view(x[:, 2 * C:], N), None, mask,
                        original.reshape(1, -1).to(torch.int64))
        o.index_copy_(2, out_index, exact)
    return o.transpose(1, 2).reshape(B, o.shape[2], C)


def compute_attention(qkv: torch.Tensor, num_heads: int, token_plan, q_norm: nn.Module | None = None,
                      k_norm: nn.Module | None = None, mask: AttentionMask | None = None) -> torch.Tensor:
    """Attention part of SelfAttention.compute_attention (attention.py:328-439) for a global
    block with a token plan; returns [B, Nq, C] (Nq = compact query count or N).

    16-bit qkv buffers with a WeightedBilinearTokenPlan take the fused path: one kernel
    LayerNorms q/k per head and compacts Q||K||V (``vb200_compact_qkv``).  Other inputs
    (fp32, hard-merge TokenPlan, separate query plans) compose the individual operators.

    ``mask``: rows see and weigh the keys as it says (the log-masses are then added in fp32)."""
    if mask is not None:
        mask._check(*qkv.shape[:2])
    if token_plan is not None and _fused_ok(qkv, token_plan, q_norm, k_norm):
        return _compute_attention_fused(qkv, num_heads, token_plan, q_norm, k_norm, mask)
    B, N, C3 = qkv.shape
    C = C3 // 3
    dense_q, dense_k, dense_v = _dense_rows(qkv, num_heads, q_norm, k_norm)
    if token_plan is None:
        x = _attend(dense_q.transpose(1, 2), dense_k.transpose(1, 2), dense_v.transpose(1, 2), None, mask)
        return x.transpose(1, 2).reshape(B, N, C)
    qc, kc, vc = _compact_rows(dense_q, dense_k, dense_v, token_plan)
    bias = getattr(token_plan, "key_log_mass", None)  # None: plain softmax attention
    rows, keys = (None, None) if mask is None else _places(token_plan)
    x = _attend(_bhtd(qc, num_heads), _bhtd(kc, num_heads), _bhtd(vc, num_heads), bias, mask, rows, keys)
    if getattr(token_plan, "dense_special_queries", False):
        original = token_plan.special_query_original
        out_index = original if getattr(token_plan, "preserve_queries", False) else token_plan.special_query_compact
        if original is None or out_index is None:
            raise RuntimeError("dense-special attention plan has no special-token mapping")
        exact = _attend(dense_q.index_select(1, original).transpose(1, 2), dense_k.transpose(1, 2),
                        dense_v.transpose(1, 2), None, mask, original.reshape(1, -1).to(torch.int64).expand(B, -1))
        x.index_copy_(2, out_index, exact.to(x.dtype))
    return x.transpose(1, 2).reshape(B, x.shape[2], C)


def _dense_rows(qkv, num_heads, q_norm, k_norm):
    """q, k, v [B, N, H, hd] of a qkv buffer, q and k normalised."""
    B, N, C3 = qkv.shape
    q, k, v = qkv.view(B, N, 3, num_heads, C3 // 3 // num_heads).unbind(2)  # [B, N, H, hd] views
    if q_norm is not None:
        q = q_norm(q)
    if k_norm is not None:
        k = k_norm(k)
    return q, k, v


def _compact_rows(q, k, v, token_plan):
    """q, k, v [B, rows, C] of the compact attention, one operator each."""
    flat = lambda t: t.reshape(t.shape[0], t.shape[1], t.shape[2] * t.shape[3])
    if getattr(token_plan, "preserve_queries", False):
        key = token_plan.compact_key(flat(k)) if hasattr(token_plan, "compact_key") else token_plan.compact(flat(k))
        return flat(q), key, token_plan.compact(flat(v))
    qc = token_plan.compact_query(flat(q)) if hasattr(token_plan, "compact_query") else token_plan.compact(flat(q))
    return qc, token_plan.compact(flat(k)), token_plan.compact(flat(v))


class GlobalAttention(nn.Module):
    """Parameters and forward of a global-block SelfAttention (dim, heads, qkv / proj bias,
    masked k bias, q/k LayerNorm)."""

    def __init__(self, dim: int, num_heads: int, qkv_bias: bool = True, proj_bias: bool = True,
                 mask_k_bias: bool = True, use_qk_norm: bool = True, device=None, dtype=None) -> None:
        super().__init__()
        self.num_heads = num_heads
        head_dim = dim // num_heads
        factory = dict(device=device, dtype=dtype)
        self.qkv = nn.Linear(dim, dim * 3, bias=qkv_bias, **factory)
        self.proj = nn.Linear(dim, dim, bias=proj_bias, **factory)
        self.use_qk_norm = use_qk_norm
        self.q_norm = nn.LayerNorm(head_dim, eps=1e-5, **factory) if use_qk_norm else None
        self.k_norm = nn.LayerNorm(head_dim, eps=1e-5, **factory) if use_qk_norm else None
        mask = torch.ones(dim * 3, device=device, dtype=dtype or torch.float32)
        if mask_k_bias:
            mask[dim: 2 * dim] = 0
        self.register_buffer("bias_mask", mask)

    def load_reference_state(self, state: dict) -> None:
        """Load a state dict of the reference SelfAttention (names qkv.*, proj.*, q_norm.*,
        k_norm.*, qkv.bias_mask)."""
        own = {k: v for k, v in state.items() if k != "qkv.bias_mask"}
        self.load_state_dict({**own, "bias_mask": state.get("qkv.bias_mask", self.bias_mask)}, strict=True)

    def _masked_qkv_bias(self):
        """qkv bias with the key part zeroed (the reference's LinearKMaskedBias,
        layers/attention.py:195-207), cached until either tensor is modified in place (torch's
        version counters), so a step does not recompute it."""
        b = self.qkv.bias
        if b is None:
            return None
        key = (b.data_ptr(), b._version, self.bias_mask.data_ptr(), self.bias_mask._version, b.dtype)
        cached = getattr(self, "_bias_cache", None)
        if cached is None or cached[0] != key:
            cached = (key, b * self.bias_mask.to(b.dtype))
            self._bias_cache = cached
        return cached[1]

    def qkv_projection(self, x: torch.Tensor) -> torch.Tensor:
        return F.linear(x, self.qkv.weight, self._masked_qkv_bias())

    def _qkv(self, x: torch.Tensor, token_plan) -> torch.Tensor:
        qkv = getattr(token_plan, "precomputed_qkv", None)
        return self.qkv_projection(x) if qkv is None else qkv

    def forward(self, x: torch.Tensor, token_plan=None, mask: AttentionMask | None = None) -> torch.Tensor:
        qkv = self._qkv(x, token_plan)
        attn = compute_attention(qkv, self.num_heads, token_plan, self.q_norm, self.k_norm, mask)
        y = self.proj(attn)
        if token_plan is None:
            return y
        return token_plan.restore(y)

    def stream(self, x: torch.Tensor, cache: PagedCache, sequence, offsets=None, token_plan=None, *, causal: bool = False,
               softcap: float | None = None) -> torch.Tensor:
        """The block over frames that arrive one after the other: the keys, values and masses of ``x`` go behind what slot
        ``sequence[i]`` of the cache holds, and its rows attend over all of it.  Inference only (no gradients).

        x [1, N, C]: chunks offsets[i] .. offsets[i + 1] of rows of the streams ``sequence``; offsets may be left out for one
        stream.  Rows see the past and their whole chunk, or with ``causal`` no later token.  With a token plan, x is the
        new frames of one stream, merged among themselves: the cache takes its merged keys with their masses.
        Special queries of a plan attend over merged keys here (the past is kept in that form only), so plans with
        ``dense_special_queries`` are refused, as is ``causal`` with a plan.  Returns [1, N, C]; rows outside every chunk (a padded
        batch) come out as rows without keys do.

        A pool without room for the chunks leaves the cache as it was and shows in ``device_error_flags()`` (bit 2); the
        rows then attend over the past alone, and with ``causal``, as if its last tokens were theirs, over part of it."""
        if x.ndim != 3 or x.shape[0] != 1:
            raise ValueError("stream: x must be [1, tokens, channels]")
        streams = len(sequence)
        if token_plan is not None:
            if streams != 1 or causal:
                raise ValueError("stream: a token plan merges the frames of one stream, which all see one another")
            if getattr(token_plan, "dense_special_queries", False):
                raise ValueError("stream: the cache holds merged keys only, dense special queries cannot be served")
            if offsets is not None:
                raise ValueError("stream: with a token plan all rows are one chunk")
        elif offsets is None and streams != 1:
            raise ValueError("stream: offsets are needed for several streams")
        _positive("softcap", softcap)  # what the attention would refuse is refused before the cache takes anything
        qkv = self._qkv(x, token_plan)
        log_mass = None
        if token_plan is None:
            q, k, v = (t[0] for t in _dense_rows(qkv, self.num_heads, self.q_norm, self.k_norm))
        else:
            if _fused_ok(qkv, token_plan, self.q_norm, self.k_norm):
                rows = _compact_rows_fused(qkv[0], token_plan, self.q_norm, self.k_norm)
            else:
                rows = (t[0] for t in _compact_rows(*_dense_rows(qkv, self.num_heads, self.q_norm, self.k_norm), token_plan))
            q, k, v = (t.view(t.shape[0], self.num_heads, -1) for t in rows)
            log_mass = getattr(token_plan, "key_log_mass", None)
            log_mass = None if log_mass is None else log_mass.reshape(-1)
        q, k, v = (t.to(cache.k.dtype) for t in (q, k, v))  # LayerNorm gives fp32 under autocast
        _refuse_gradients("stream", q, k, v, log_mass)
        # made on the device, so that the step can be recorded into a graph
        chunk = lambda n: torch.arange(2, device=x.device, dtype=torch.int32) * n if offsets is None else offsets
        cache.append(sequence, chunk(k.shape[0]), k, v, log_mass)
        out = None if offsets is None else q.new_zeros(q.shape)  # the attention leaves rows outside the chunks as they are
        attn = paged_attention(q, cache, sequence, chunk(q.shape[0]), causal=causal, softcap=softcap, out=out)
        y = self.proj(attn.reshape(1, attn.shape[0], -1).to(qkv.dtype))
        return y if token_plan is None else token_plan.restore(y)
