"""A KV cache of 4.5 bits a value, the attention that reads it and the eviction that keeps it short.

    cache = Kv4Cache.new(batch, max_seq, n_kv_heads, head_dim, device, track_weights=True)
    kv4_append_(k, v, cache)                                   # a prompt's keys (rotated) and values
    out = kv4_decode_attention_(qkv, cache, n_q_heads, lengths)    # one new token a sequence; then lengths += 1
    lengths = kv4_evict_(cache, lengths, keep=2048, recent=128)    # the slots that attention has weighed most

A value is `scale * code`: 32 neighbouring dims of a key or value share a bf16 scale, their largest magnitude over 7, and a
code is an integer in [-7, 7], the nearest (halves to the smaller magnitude).  At head_dim 128 a slot takes 144 bytes
instead of 512.  Keys are stored as they are attended to, rotated.  Sequences have lengths of their own: `lengths` is an
int32 tensor [batch] on the cache's GPU that the kernels read when they run, so a captured CUDA graph serves every step.

Calls are ordered by their stream and share nothing: scratch comes from the caching allocator, call by call.  No upstream
counterpart.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from .._ext import C
from ..errors import SymmMemError
from ..utils.trace import traced

_TILE = 64      # the kernels take slots in tiles of this many


class Kv4Cache:
    """The tensors of a 4-bit cache: codes uint8 [batch, kv heads, slots, head_dim / 2], two a byte, scales bfloat16
    [batch, kv heads, slots, head_dim / 32], and `weights` float32 [batch, kv heads, slots] or None: the attention
    weight that each slot has had in decode steps, summed over the query heads that share the kv head.  `slots` is a
    multiple of 64, of which `max_seq` are used.  The order of a row's codes is the kernels' own (`kv4_read` gives values)."""

    def __init__(self, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor, v_scales: torch.Tensor,
                 weights: Optional[torch.Tensor] = None, max_seq: Optional[int] = None):
        self.max_seq = int(k_codes.shape[2] if max_seq is None else max_seq)
        C.kv4_check(k_codes, k_scales, v_codes, v_scales, weights, self.max_seq)
        self.k_codes, self.k_scales, self.v_codes, self.v_scales, self.weights = k_codes, k_scales, v_codes, v_scales, weights

    @staticmethod
    def new(batch: int, max_seq: int, n_kv_heads: int, head_dim: int, device, track_weights: bool = False) -> "Kv4Cache":
        """An empty cache (every value zero)."""
        if head_dim not in (64, 128):
            raise SymmMemError("head_dim must be 64 or 128")
        if batch < 0 or max_seq < 1 or n_kv_heads < 1:
            raise SymmMemError("need batch >= 0, max_seq >= 1 and n_kv_heads >= 1")
        slots = -(-max_seq // _TILE) * _TILE

        def part(width, dtype):
            return torch.zeros(batch, n_kv_heads, slots, width, dtype=dtype, device=device)

        weights = torch.zeros(batch, n_kv_heads, slots, dtype=torch.float32, device=device) if track_weights else None
        return Kv4Cache(part(head_dim // 2, torch.uint8).fill_(0x88), part(head_dim // 32, torch.bfloat16),
                        part(head_dim // 2, torch.uint8).fill_(0x88), part(head_dim // 32, torch.bfloat16), weights, max_seq)

    @property
    def batch(self) -> int:
        return self.k_codes.shape[0]

    @property
    def n_kv_heads(self) -> int:
        return self.k_codes.shape[1]

    @property
    def slots(self) -> int:
        return self.k_codes.shape[2]

    @property
    def head_dim(self) -> int:
        return 2 * self.k_codes.shape[3]

    def reset(self) -> None:
        """Every value zero, every weight zero."""
        for codes, scales in ((self.k_codes, self.k_scales), (self.v_codes, self.v_scales)):
            codes.fill_(0x88)
            scales.zero_()
        if self.weights is not None:
            self.weights.zero_()


@traced("smr.kv4_append_")
def kv4_append_(k: torch.Tensor, v: torch.Tensor, cache: Kv4Cache, start: Union[int, torch.Tensor] = 0,
                counts: Optional[torch.Tensor] = None) -> Kv4Cache:
    """Keys and values `k`, `v` [batch, tokens, kv heads, head_dim] bfloat16 into slots `start`, `start + 1`, ... of their
    sequences.  `k` and `v` may be views of a projection's output (any strides that keep a row contiguous and on 16 bytes).
    `start`: an int, or an int32 tensor [batch]; `counts` (int32 [batch]): a padded batch, sequence b has only its first
    `counts[b]` tokens.  A sequence whose `start` in a tensor is outside
    `[0, max_seq)` is idle, tokens behind `max_seq` are dropped, and no other slot changes.  A group of
    32 dims that holds an infinity or a NaN reads back as NaN.  A written slot's weight starts from zero."""
    on_device = isinstance(start, torch.Tensor)
    C.kv4_append(k, v, cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales, cache.weights, cache.max_seq,
                 0 if on_device else start, start if on_device else None, counts)
    return cache


@traced("smr.kv4_read")
def kv4_read(cache: Kv4Cache, n: Optional[int] = None):
    """`(k, v)`, each [batch, n, kv heads, head_dim] bfloat16: what slots `[0, n)` (all `max_seq` without `n`) stand for,
    rounded to bfloat16; for the attention of a prompt's next chunk, or to go back to a cache of 16 bits."""
    return C.kv4_read(cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales, cache.max_seq,
                      cache.max_seq if n is None else n)


@traced("smr.kv4_decode_attention_")
def kv4_decode_attention_(qkv: torch.Tensor, cache: Kv4Cache, n_q_heads: int, lengths: Union[int, torch.Tensor],
                          out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one decode step over a 4-bit cache.  `qkv` [batch, (hq + 2 hkv) * head_dim] holds the new token's queries
    and keys, rotated (`rope_axes_`, `rope_`), and its values; it is not modified.  Sequence b has `lengths[b]` tokens in
    the cache: the new key and value are quantised into slot `lengths[b]` (hence the trailing underscore; the caller
    advances `lengths`), and `out[b] = softmax(q . K / sqrt(head_dim)) V` over slots `0 .. lengths[b]` per query head (head h
    reads kv head h // (hq / hkv)), the new token as it is stored.  A cache with `weights` has each slot's attention weight,
    summed over the query heads of its kv head, added to them; the new slot starts from zero.

    `lengths`: an int32 tensor [batch], or an int for all.  A sequence whose length is negative, or `max_seq` and more, is
    idle: its output row is zero and its cache is left alone.  `head_dim` is 64 or 128, hq / hkv at most 8, batch at most
    1024.  A NaN or an infinity in a row of q, K or V shows in the outputs and weights that read it, and in no others; a query
    with a magnitude of 2^118 or more counts as one, and so does a score beyond fp32.

    Scores, maxima, sums and weights are fp32.  A probability times the scale of a value's group is rounded to fp16 on its way into
    the weighted sum: 2^-11 of itself at most while it is at least 2^-29 of the largest probability times the largest scale in 64
    slots, for values between 2^-56 and 2^100.  Smaller products lose bits, and below 2^-40 they count as zero."""
    on_device = isinstance(lengths, torch.Tensor)
    return C.kv4_decode_attention(qkv, cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales, cache.weights,
                                  cache.max_seq, n_q_heads, 0 if on_device else lengths, lengths if on_device else None, out)


@traced("smr.kv4_evict_")
def kv4_evict_(cache: Kv4Cache, lengths: torch.Tensor, keep: int, recent: int = 0) -> torch.Tensor:
    """Cuts sequences of more than `keep` tokens to `keep` slots, for every kv head by its own weights: the last `recent`
    slots stay, and of the others those with the most accumulated attention weight (equal weights: the lower slot; NaN counts
    as an infinity).  The slots that stay move down to `0 .. keep - 1` in their order, with their weights; what is behind
    them is left as it was.  Returns the new lengths, `min(lengths, keep)`; sequences that are short enough, idle (negative) or
    of an impossible length (above `max_seq`) do not change."""
    if cache.weights is None:
        raise SymmMemError("eviction needs a cache that tracks weights")
    return C.kv4_evict(cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales, cache.weights, cache.max_seq, lengths, keep,
                       recent)
