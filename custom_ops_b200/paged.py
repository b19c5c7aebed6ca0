"""A paged key/value cache for decoding, over the operators of the paged group, and the angles of rotary
positions.  The reference has no counterpart.

    cache = PagedCache(layers=32, num_pages=4096, page_size=16, heads_k=8, head_dim=128,
                       max_requests=64, max_length=8192)
    freqs, mscale = rotary_frequencies(128, base=10000.0)

    slots, positions, cu = cache.extend(new_lens, num_tokens)          # once per step
    for layer in range(32):                                            # q (T, H, d), k, v (T, Hk, d)
        q = cache.append(layer, q, k, v, slots, positions, freqs, mscale=mscale)
        out = cache.attend(layer, q)                                   # a step of one token per request
    cache.release(rows)                                                # pages of finished requests

Nothing here synchronises: after one step outside a capture, a step may be captured into a CUDA graph and replayed.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import ops

__all__ = ["PagedCache", "rotary_frequencies"]


def rotary_frequencies(rot_dim: int, base: float = 10000.0, *, scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: Optional[int] = None, fast: float = 32.0, slow: float = 1.0, device=None):
    """``(freqs, mscale)`` for ``ops.rotary`` and ``ops.rotary_append``: ``rot_dim / 2`` angles per position,
    ``base ** (-2i / rot_dim)`` in float64, and the factor for the turned pairs.

    ``scaling`` stretches them for contexts ``factor`` times longer than a model was trained on:
    ``"linear"``   all angles divided by ``factor``;
    ``"base"``     the base raised to ``base * factor ** (rot_dim / (rot_dim - 2))``: the slowest pair is divided by
                   ``factor``, the fastest stays (published as "NTK-aware" scaling);
    ``"by_parts"`` pairs that turn at least ``fast`` times within ``original_length`` positions stay, those that
                   turn at most ``slow`` times are divided by ``factor``, linearly in between by the pair's
                   index, from the last that turns ``fast`` times to the first that turns no more than ``slow``
                   times, also where these lie outside the head's pairs; ``mscale`` is ``0.1 * log(factor) + 1``
                   ("NTK-by-parts" with YaRN's factor; Peng et al., 2023, arXiv:2309.00071.  Forms of it that move
                   the ends of the ramp onto the head's first and last pair differ where these would lie outside).
    """
    if rot_dim < 2 or rot_dim % 2 != 0:
        raise ValueError("rot_dim must be even and at least 2")
    if not (base > 1.0 and math.isfinite(base)) or not (factor >= 1.0 and math.isfinite(factor)):
        raise ValueError("base must be above 1 and factor at least 1")
    if scaling not in (None, "linear", "base", "by_parts"):
        raise ValueError(f"scaling must be None, 'linear', 'base' or 'by_parts', got {scaling!r}")
    if scaling == "base":
        if rot_dim == 2:
            raise ValueError("scaling='base' needs more than one pair")
        base = base * factor ** (rot_dim / (rot_dim - 2))
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    freqs = base ** (-i / rot_dim)
    mscale = 1.0
    if scaling == "linear":
        freqs = freqs / factor
    if scaling == "by_parts":
        if original_length is None or original_length <= 0 or not 0.0 < slow < fast:
            raise ValueError("scaling='by_parts' needs original_length > 0 and 0 < slow < fast")

        def pair_that_turns(times):          # its (fractional) index
            return rot_dim * math.log(original_length / (times * 2 * math.pi)) / (2 * math.log(base))

        lo, hi = math.floor(pair_that_turns(fast)), math.ceil(pair_that_turns(slow))
        ramp = ((i / 2 - lo) / max(hi - lo, 1)).clamp(0.0, 1.0)
        freqs = freqs * (1.0 - ramp) + freqs / factor * ramp
        mscale = 0.1 * math.log(factor) + 1.0
    return freqs.to(device if device is not None else "cuda"), mscale


class PagedCache:
    """Keys and values of up to ``max_requests`` requests in pages of ``page_size`` tokens, for every layer.

    ``k``, ``v`` are ``(layers, num_pages, heads_k, page_size, head_dim)``; one block table serves all layers.
    Page 0 is never given out.  Request ``b`` is row ``b`` of ``block_table`` and ``seq_lens``."""

    def __init__(self, *, layers: int, num_pages: int, page_size: int, heads_k: int, head_dim: int, max_requests: int,
                 max_length: int, dtype: torch.dtype = torch.bfloat16, device=None):
        if min(layers, page_size, heads_k, max_requests, max_length) < 1 or num_pages < 2:
            raise ValueError("layers, page_size, heads_k, max_requests and max_length must be at least 1, num_pages 2")
        if head_dim not in (64, 128):
            raise ValueError("Only head_dim=64 or head_dim=128 is supported")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("dtype must be torch.bfloat16 or torch.float16")
        device = torch.device("cuda" if device is None else device)
        shape = (layers, num_pages, heads_k, page_size, head_dim)
        self.page_size = page_size
        self.k = torch.empty(shape, dtype=dtype, device=device)
        self.v = torch.empty(shape, dtype=dtype, device=device)
        i32 = dict(dtype=torch.int32, device=device)
        self.block_table = torch.zeros((max_requests, -(-max_length // page_size)), **i32)
        self.seq_lens = torch.zeros((max_requests,), **i32)
        self.free_pages = torch.arange(1, num_pages, **i32)
        self.free_head = torch.zeros((1,), **i32)

    def extend(self, new_lens: torch.Tensor, num_tokens: int):
        """Room for ``new_lens[b]`` more tokens of every request (int32 ``(max_requests,)``; 0 for rows without
        one); ``num_tokens`` is the number of packed tokens, padding included.  Returns ``(slots, positions, cu)``
        of ``ops.paged_extend_``; a request whose tokens have slot -1 found no room and keeps its length."""
        return ops.paged_extend_(self.block_table, self.seq_lens, new_lens, self.free_pages, self.free_head,
                                 self.page_size, num_tokens)

    def append(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
               positions: Optional[torch.Tensor] = None, freqs: Optional[torch.Tensor] = None, *,
               interleaved: bool = False, mscale: float = 1.0) -> torch.Tensor:
        """Writes the packed new tokens' keys and values; with ``freqs`` q and k are turned first.  Returns q."""
        if freqs is None:
            ops.paged_append(k, v, slots, self.k[layer], self.v[layer])
            return q
        if positions is None:
            raise ValueError("rotary positions need `positions`")
        return ops.rotary_append(q, k, v, positions, slots, self.k[layer], self.v[layer], freqs,
                                 interleaved=interleaved, mscale=mscale)

    def attend(self, layer: int, q: torch.Tensor, *, return_lse: bool = False, **score):
        """Attention of one token per row - the newest of every request, q ``(max_requests, H, d)`` - over what
        the layer holds; ``score``: scale, window, softcap, slopes of ``ops.paged_attention``."""
        call = ops.paged_attention_lse if return_lse else ops.paged_attention
        return call(q, self.k[layer], self.v[layer], self.block_table, self.seq_lens, **score)

    def shrink(self, keep_lens: torch.Tensor) -> None:
        """Shortens every request to at most ``keep_lens`` tokens and frees the pages behind that."""
        ops.paged_shrink_(self.block_table, self.seq_lens, keep_lens, self.free_pages, self.free_head, self.page_size)

    def release(self, rows: torch.Tensor) -> None:
        """Frees all pages of the requests in ``rows``: an index or boolean tensor on the device, or a list (which is
        copied there)."""
        keep = self.seq_lens.clone()
        keep[rows] = 0
        self.shrink(keep)
