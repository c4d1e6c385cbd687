"""Decoding a batch behind one restored prefix.

The injector restores a prompt chunk that many requests share into a ``SpecDynamicCache``;
``SharedPrefixCache`` is what the batch decodes from: that prefix once, each sequence's own
tokens behind it, and per layer one call that turns the new queries and keys by their
positions (the keys straight into their cache slots), attends over both and, if asked, adds up
the weight that each own token was given, by which :meth:`SharedPrefixCache.evict` cuts the
own caches.  No counterpart in the reference (its model attends by itself).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from ..kernels.attention import accumulate_attention_weights, shared_prefix_attention
from ..kernels.restore import DEFAULT_THETA
from ..kernels.rotary import RopeScaling, apply_rotary
from .kv_injector import SpecDynamicCache


@dataclass
class _Step:
    """A layer's last step, as far as taking it back needs it."""

    start: int  # own tokens before it
    n: int
    evicted: int  # own tokens evicted before it
    before: torch.Tensor  # the scores before it
    queries: torch.Tensor | None  # turned, [B, n, Hq, D]; None: more than MAX_DRAFT tokens
    lse: torch.Tensor | None
    scale: float | None


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

    MAX_DRAFT = 64  # tokens of a step whose queries are kept, so that truncate can take a part of it back

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
        self._spare: list[torch.Tensor | None] = []  # room for the next step's
        self._last: list[_Step | None] = []

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
            self._spare.append(None)
            self._last.append(None)
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
            before, after = self._room_for_scores(layer_idx, start, start + n, h, k.device)
            end = start + n
            accumulate_attention_weights(turned, k_own, lse, before[..., :end], scale=scale, out=after[..., :end])
            draft = n <= self.MAX_DRAFT
            self._scores[layer_idx], self._spare[layer_idx] = after, before
            self._last[layer_idx] = _Step(start, n, self.own.evicted_tokens(layer_idx), before,
                                          turned.view(b, n, hq, d) if draft else None,
                                          lse.view(b, n, hq) if draft else None, scale)
        # nothing was refused: the step's tokens are the cache's
        self.own.commit(layer_idx, n)
        return out.view(b, n, hq, d).transpose(1, 2)

    def truncate(self, max_seq_len: int) -> None:
        """Drop the newest own tokens (a draft's rejected ones) so that no layer holds more than
        ``max_seq_len`` tokens, the prefix's among them; the next token goes on from there.

        Tracked weights become those of the accepted tokens alone.  For that a layer can be cut back to
        where its last step began, and into that step if it had at most ``MAX_DRAFT`` tokens; no token
        from before the last eviction can be dropped.  What cannot be cut is refused before anything is."""
        cuts = []
        for layer in range(len(self.own)):
            size, own = self.prefix.get_seq_length(layer), self.own.get_seq_length(layer)
            if size + own <= max_seq_len:
                continue
            left = int(max_seq_len) - size
            if left < 0:
                raise ValueError(f"max_seq_len {max_seq_len} would cut the prefix of {size} tokens")
            if self.track_weights:
                last = self._last_step(layer)
                if last is None or left < last.start:
                    raise ValueError(f"layer {layer} can be cut back to {own if last is None else last.start} own "
                                     f"tokens (where its last step began or its last eviction ended), not to {left}")
                if last.queries is None and left > last.start:
                    raise ValueError(f"a step of {last.n} tokens can be taken back as a whole only "
                                     f"(up to {self.MAX_DRAFT} in part)")
            elif self.own.evicted_tokens(layer):
                raise ValueError(f"tokens of layer {layer} were evicted: without tracked weights none can be dropped")
            cuts.append((layer, left))
        for layer, left in cuts:
            last, n = self._last_step(layer), 0
            if last is not None:
                n = left - last.start
                after = self._spare[layer] = self._scores[layer]
                self._scores[layer], self._last[layer] = last.before, None
            if n:
                queries, lse = last.queries[:, :n].contiguous(), last.lse[:, :n].contiguous()
                k_own = self.own[layer][0][:, :, :left].transpose(1, 2)
                accumulate_attention_weights(queries.view(-1, *queries.shape[2:]), k_own,
                                             lse.view(-1, lse.shape[2]), last.before[..., :left], scale=last.scale,
                                             out=after[..., :left])
                self._scores[layer], self._spare[layer] = after, last.before
                self._last[layer] = _Step(last.start, n, last.evicted, last.before, queries, lse, last.scale)
            self.own.truncate_layer(layer, left)

    def _last_step(self, layer_idx: int) -> _Step | None:
        """The layer's last step, unless its tokens have been moved since."""
        last = self._last[layer_idx] if layer_idx < len(self._last) else None
        return None if last is None or last.evicted != self.own.evicted_tokens(layer_idx) else last

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
                         device: torch.device) -> tuple[torch.Tensor, torch.Tensor]:
        """The layer's scores, those of the tokens from ``start`` to ``end`` zero, and room for the next."""
        have, spare = self._scores[layer_idx], self._spare[layer_idx]
        if have is None or have.shape[2] < end:
            room = torch.zeros((self.batch, heads, max(end, 2 * start, 16)), dtype=torch.float32, device=device)
            if have is not None:
                room[..., :start] = have[..., :start]
            self._scores[layer_idx] = have = room
        else:
            have[..., start:end] = 0
        if spare is None or spare.shape[2] < end:
            self._spare[layer_idx] = spare = torch.empty_like(have)
        return have, spare
