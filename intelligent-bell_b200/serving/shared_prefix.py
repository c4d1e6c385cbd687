"""Decoding a batch behind one restored prefix.

The injector restores a prompt chunk that many requests share into a ``SpecDynamicCache``;
``SharedPrefixCache`` is what the batch decodes from: that prefix once, each sequence's own
tokens behind it, and per layer one call that turns the new queries and keys by their
positions (the keys straight into their cache slots), attends over both and, if asked, adds up
the weight that each own token was given, by which :meth:`SharedPrefixCache.evict` cuts the
own caches.  No counterpart in the reference (its model attends by itself).
"""

from __future__ import annotations

import torch

from ..kernels.attention import accumulate_attention_weights, shared_prefix_attention
from ..kernels.restore import DEFAULT_THETA
from ..kernels.rotary import RopeScaling, apply_rotary
from .kv_injector import SpecDynamicCache


class SharedPrefixCache:
    """``batch`` sequences behind the tokens of ``prefix`` (batch 1; its keys already turned).

    Args:
        prefix: a cache of batch 1, as ``MultiLayerKVInjector`` fills it.
        batch: sequences that share it.
        capacity: own tokens a layer to make room for at first.
        theta, rotary_dim, interleaved, scaling: of the rotary positions, see :func:`apply_rotary`;
            the prefix's tokens are at positions 0 to P - 1.
        track_weights: add up attention weights for :meth:`evict`.
    """

    def __init__(self, prefix: SpecDynamicCache, batch: int, capacity: int = 0, *,
                 theta: float = DEFAULT_THETA, rotary_dim: int | None = None, interleaved: bool = False,
                 scaling: RopeScaling | None = None, track_weights: bool = False) -> None:
        if batch < 1:
            raise ValueError(f"batch must be at least 1, got {batch}")
        self.prefix, self.batch = prefix, int(batch)
        self.own = SpecDynamicCache(capacity)
        self.theta, self.rotary_dim = float(theta), rotary_dim
        self.interleaved, self.scaling = bool(interleaved), scaling
        self.track_weights = bool(track_weights)
        self._scores: list[torch.Tensor | None] = []

    def prefix_views(self, layer_idx: int) -> tuple[torch.Tensor, torch.Tensor] | tuple[None, None]:
        """Token-major ``[P, H, D]`` views of the prefix layer (None, None: it has none)."""
        if self.prefix.get_seq_length(layer_idx) == 0:
            return None, None
        k, v = self.prefix[layer_idx]
        if k.shape[0] != 1:
            raise ValueError(f"the prefix must have batch 1, layer {layer_idx} has {k.shape[0]}")
        return k[0].transpose(0, 1), v[0].transpose(0, 1)

    def get_seq_length(self, layer_idx: int = 0) -> int:
        """Tokens that a new query of the layer sees: the prefix's and the own ones kept."""
        return self.prefix.get_seq_length(layer_idx) + self.own.get_seq_length(layer_idx)

    def next_position(self, layer_idx: int = 0) -> int:
        """Position of the layer's next token: behind the prefix and every own token so far, evicted
        ones included, truncated ones not."""
        return self.get_seq_length(layer_idx) + self.own.evicted_tokens(layer_idx)

    def scores(self, layer_idx: int) -> torch.Tensor:
        """float32 ``[B, H, own length]`` accumulated weights of the layer's own tokens."""
        if not self.track_weights:
            raise RuntimeError("weights are not tracked: give track_weights=True")
        return self._scores[layer_idx][..., :self.own.get_seq_length(layer_idx)]

    def attend(self, layer_idx: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
               scale: float | None = None) -> torch.Tensor:
        """Append the step's tokens and attend: q ``[B, Hq, n, D]``, k and v ``[B, H, n, D]``, not yet
        turned; returns ``[B, Hq, n, D]``.  Query j sees the prefix, the own tokens kept and the
        step's tokens up to its own."""
        if q.ndim != 4 or k.ndim != 4 or v.shape != k.shape:
            raise ValueError(f"q, k, v must be [B, H, n, D], got {tuple(q.shape)}, {tuple(k.shape)}, "
                             f"{tuple(v.shape)}")
        b, hq, n, d = q.shape
        if b != self.batch or k.shape[0] != b or k.shape[2] != n or k.shape[3] != d:
            raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} do not fit a batch of {self.batch}")
        if v.dtype != k.dtype or v.device != k.device:
            raise ValueError(f"v is {v.dtype} on {v.device}, k {k.dtype} on {k.device}")
        h = k.shape[1]
        while len(self._scores) <= layer_idx:
            self._scores.append(None)
        self.own.reserve(layer_idx, n, batch=b, heads=h, head_dim=d, dtype=k.dtype, device=k.device)
        k_slot, v_slot = self.own.append_slots(layer_idx, n)
        turned = torch.empty((b, n, hq, d), dtype=q.dtype, device=q.device)
        apply_rotary(q, k, self.next_position(layer_idx), theta=self.theta, rotary_dim=self.rotary_dim,
                     interleaved=self.interleaved, scaling=self.scaling, q_out=turned.transpose(1, 2),
                     k_out=k_slot)
        v_slot.copy_(v)
        start = self.own.get_seq_length(layer_idx)
        k_own, v_own = (x.transpose(1, 2) for x in self.own.views_with(layer_idx, n))
        k_pre, v_pre = self.prefix_views(layer_idx)
        turned = turned.view(b * n, hq, d)
        out, lse = shared_prefix_attention(turned, k_pre, v_pre, k_own, v_own, scale=scale)
        if self.track_weights:
            scores = self._room_for_scores(layer_idx, start, start + n, h, k.device)
            accumulate_attention_weights(turned, k_own, lse, scores, scale=scale)
        # nothing was refused: the step's tokens are the cache's
        self.own.commit(layer_idx, n)
        return out.view(b, n, hq, d).transpose(1, 2)

    def evict(self, budget: int, *, keep_first: int = 0, keep_recent: int = 0) -> None:
        """Cut every layer's own caches to ``budget`` tokens, see :func:`evict_tokens`.  Kept keys
        stay turned by the positions they had, and new tokens go on from :meth:`next_position`."""
        if not self.track_weights:
            raise RuntimeError("weights are not tracked: give track_weights=True")
        for layer in range(len(self.own)):
            if self.own.get_seq_length(layer):
                self.own.evict(layer, self._scores[layer], budget, keep_first=keep_first,
                               keep_recent=keep_recent)

    def _room_for_scores(self, layer_idx: int, start: int, end: int, heads: int,
                         device: torch.device) -> torch.Tensor:
        """The layer's scores up to ``end``, those of the tokens from ``start`` on zero."""
        have = self._scores[layer_idx]
        if have is None or have.shape[2] < end:
            room = torch.zeros((self.batch, heads, max(end, 2 * start, 16)), dtype=torch.float32, device=device)
            if have is not None:
                room[..., :start] = have[..., :start]
            self._scores[layer_idx] = have = room
        else:
            have[..., start:end] = 0
        return have[..., :end]
