"""What the 4-bit cache's operators refuse, and the arithmetic of their codes; no GPU."""
import numpy as np
import pytest
import torch

import kv4_reference as ref
from symm_mem_recipes_b200 import ops
from symm_mem_recipes_b200.errors import SymmMemError

BF16 = torch.bfloat16


def parts(batch=2, hkv=2, slots=128, dim=128, weights=False):
    w = torch.zeros(batch, hkv, slots) if weights else None
    return dict(k_codes=torch.zeros(batch, hkv, slots, dim // 2, dtype=torch.uint8),
                k_scales=torch.zeros(batch, hkv, slots, dim // 32, dtype=BF16),
                v_codes=torch.zeros(batch, hkv, slots, dim // 2, dtype=torch.uint8),
                v_scales=torch.zeros(batch, hkv, slots, dim // 32, dtype=BF16), weights=w)


class Fake:
    """A cache whose tensors are on the CPU: refused at the last check, after the one that a test is about."""

    def __init__(self, max_seq=100, **kw):
        self.__dict__.update(parts(**kw))
        self.max_seq = max_seq


def refused(words, fn, *args, **kw):
    with pytest.raises(SymmMemError, match=words):
        fn(*args, **kw)


@pytest.mark.parametrize("change, words", [
    (dict(k_codes=torch.zeros(2, 2, 128, 48, dtype=torch.uint8)), "head_dim of 64 or 128"),
    (dict(k_codes=torch.zeros(2, 2, 128, 64, dtype=torch.int8)), "uint8"),
    (dict(v_codes=torch.zeros(2, 2, 64, 64, dtype=torch.uint8)), "v_codes"),
    (dict(k_scales=torch.zeros(2, 2, 128, 4)), "scales must be bfloat16"),
    (dict(v_scales=torch.zeros(2, 2, 128, 2, dtype=BF16)), "scales must be bfloat16"),
    (dict(weights=torch.zeros(2, 2, 64)), "weights"),
    (dict(weights=torch.zeros(2, 2, 128, dtype=torch.float64)), "weights"),
    (dict(k_codes=torch.zeros(2, 2, 128, 128, dtype=torch.uint8)[..., ::2]), "contiguous"),
    (dict(max_seq=129), "max_seq"),
    (dict(), "on a GPU"),
])
def test_cache_refuses(change, words):
    refused(words, ops.Kv4Cache, **{**parts(), **change})


def test_cache_refuses_odd_slots_and_shared_memory():
    refused("multiple of 64", ops.Kv4Cache, **parts(slots=100))
    p = parts()
    p["v_codes"] = p["k_codes"]
    refused("share memory", ops.Kv4Cache, **p)


def test_cache_refuses_no_heads():
    none = {name: t[:, :0] for name, t in parts(weights=True).items()}
    refused("at least one kv head", ops.Kv4Cache, **none)


def test_new_refuses():
    for bad in (dict(head_dim=96), dict(max_seq=0), dict(n_kv_heads=0), dict(batch=-1)):
        refused("need|head_dim", ops.Kv4Cache.new, **{**dict(batch=1, max_seq=4, n_kv_heads=1, head_dim=64, device="cpu"), **bad})


def test_append_refuses():
    k = torch.zeros(2, 5, 2, 128, dtype=BF16)
    ok = Fake()
    refused("cache's sizes", ops.kv4_append_, k, k[:, :4], ok)
    refused("cache's sizes", ops.kv4_append_, k[:1], k[:1], ok)
    refused("cache's sizes", ops.kv4_append_, k[..., :64], k[..., :64], ok)
    refused("bfloat16", ops.kv4_append_, k.float(), k.float(), ok)
    wide = torch.zeros(2, 5, 2, 256, dtype=BF16)[..., ::2]
    refused("contiguous", ops.kv4_append_, wide, wide, ok)
    odd = torch.zeros(2, 5, 2, 132, dtype=BF16)[..., :128]
    refused("16 bytes", ops.kv4_append_, odd, odd, ok)
    shifted = torch.zeros(2 * 5 * 2 * 128 + 1, dtype=BF16)[1:].view(2, 5, 2, 128)
    refused("16 bytes", ops.kv4_append_, shifted, shifted, ok)
    refused("outside", ops.kv4_append_, k, k, ok, 96)
    refused("outside", ops.kv4_append_, k, k, ok, -1)
    refused("start", ops.kv4_append_, k, k, ok, torch.zeros(1, dtype=torch.int32))
    refused("start", ops.kv4_append_, k, k, ok, torch.zeros(2, dtype=torch.int64))
    refused("counts", ops.kv4_append_, k, k, ok, 0, torch.zeros(2))
    refused("on a GPU", ops.kv4_append_, k, k, ok, 95)


def test_read_refuses():
    refused("101 slots", ops.kv4_read, Fake(), 101)
    refused("-1 slots", ops.kv4_read, Fake(), -1)
    refused("on a GPU", ops.kv4_read, Fake())


def test_decode_attention_refuses():
    qkv, ok = torch.zeros(2, (8 + 4) * 128, dtype=BF16), Fake()
    lengths = torch.zeros(2, dtype=torch.int32)
    attend = ops.kv4_decode_attention_
    refused("bfloat16", attend, qkv.float(), ok, 8, lengths)
    refused("hq / hkv", attend, qkv, ok, 7, lengths)
    refused("hq / hkv", attend, torch.zeros(2, (18 + 4) * 128, dtype=BF16), ok, 18, lengths)
    refused("hq / hkv", attend, qkv, ok, 0, lengths)
    refused("cache's sizes", attend, qkv[:1], ok, 8, lengths)
    refused("cache's sizes", attend, qkv[:, :-8], ok, 8, lengths)
    refused("16 bytes", attend, torch.zeros(2, 12 * 128 + 4, dtype=BF16)[:, :12 * 128], ok, 8, lengths)
    refused("lengths", attend, qkv, ok, 8, lengths.long())
    refused("lengths", attend, qkv, ok, 8, lengths[:1])
    refused("outside", attend, qkv, ok, 8, 100)
    refused("outside", attend, qkv, ok, 8, -1)
    refused("out must be", attend, qkv, ok, 8, lengths, torch.zeros(2, 8 * 128))
    refused("out must not", attend, qkv, ok, 8, lengths, qkv.view(-1)[:2 * 8 * 128].view(2, 8 * 128))
    refused("1024", attend, torch.zeros(1025, 12 * 64, dtype=BF16), Fake(batch=1025, slots=64, dim=64, max_seq=64), 8, 0)
    refused("on a GPU", attend, qkv, ok, 8, lengths)


def test_evict_refuses():
    lengths = torch.zeros(2, dtype=torch.int32)
    refused("tracks weights", ops.kv4_evict_, Fake(), lengths, 10)
    ok = Fake(weights=True)
    refused("keep must", ops.kv4_evict_, ok, lengths, 0)
    refused("keep must", ops.kv4_evict_, ok, lengths, 101)
    refused("recent", ops.kv4_evict_, ok, lengths, 10, 11)
    refused("recent", ops.kv4_evict_, ok, lengths, 10, -1)
    refused("lengths", ops.kv4_evict_, ok, lengths.long(), 10)
    refused("on a GPU", ops.kv4_evict_, ok, lengths, 10)


def test_rope_axes_refuses():
    x, pos = torch.zeros(6, 256, dtype=BF16), torch.zeros(3, 6, dtype=torch.int32)
    rope = ops.rope_axes_
    refused("bfloat16", rope, x.float(), 2, 128, pos, (16, 24, 24), 1e4)
    refused("head_dim", rope, x, 2, 96, pos, (16, 24, 24), 1e4)
    refused("row length", rope, x, 3, 128, pos, (16, 24, 24), 1e4)
    refused("row length", rope, x, -1, 128, pos, (16, 24, 24), 1e4)
    refused("theta", rope, x, 2, 128, pos, (16, 24, 24), 1.0)
    refused("theta", rope, x, 2, 128, pos, (16, 24, 24), float("nan"))
    refused("add up", rope, x, 2, 128, pos, (16, 24, 25), 1e4)
    refused("number of pairs", rope, x, 2, 128, pos, (-16, 40, 40), 1e4)
    refused("sections", rope, x, 2, 128, pos, (), 1e4)
    refused("positions", rope, x, 2, 128, pos.long(), (16, 24, 24), 1e4)
    refused("positions", rope, x, 2, 128, pos[:2], (16, 24, 24), 1e4)
    refused("positions", rope, x, 2, 128, pos[0], (32, 32), 1e4)
    refused("along the tokens", rope, x, 2, 128, torch.zeros(3, 12, dtype=torch.int32)[:, ::2], (16, 24, 24), 1e4)
    refused("must not overlap", rope, torch.zeros(256, dtype=BF16).expand(6, 256), 2, 128, pos, (16, 24, 24), 1e4)
    refused("16 bytes", rope, torch.zeros(6, 260, dtype=BF16)[:, :256], 2, 128, pos, (16, 24, 24), 1e4)
    refused("on a GPU", rope, x, 2, 128, pos, (16, 24, 24), 1e4)


def test_packing_round_trip():
    codes = torch.randint(-7, 8, (3, 128), generator=torch.Generator().manual_seed(0)).double()
    for dim in (64, 128):
        for is_key in (True, False):
            c = codes[:, :dim]
            assert torch.equal(ref.unpack(ref.pack(c, is_key), is_key), c)
            assert len(set(ref.pack(torch.eye(dim).double(), is_key).argmax(-1).tolist())) == dim // 2


def test_nibbles_are_those_of_the_exact_quotient():
    """rint(x * (1 / s) * (1 - 2^-14)) in fp32 against ceil(x / s - 1/2) in integers, for every pair of bf16 significands
    and every ratio of exponents that gives a code of 0 to 7."""
    f = np.float32
    m = np.arange(128, 256)
    ms, mx = np.meshgrid(m, m, indexing="ij")
    for shift in range(-3, 4):                                   # x = mx * 2^shift against s = ms
        x, s = mx.astype(f) * f(2.0 ** shift), ms.astype(f)
        keep = x <= 7.03 * s
        inv = (f(1) / s) * f(0.99993896484375)
        got = np.minimum(np.rint(x * inv), 7)
        num, den = mx * 2 ** (shift + 3), ms * 8                 # ceil(num / den - 1/2) = ceil((2 num - den) / (2 den))
        want = np.minimum(-((den - 2 * num) // (2 * den)), 7)
        assert np.array_equal(got[keep].astype(int), want[keep])


def test_cut_heads_are_joined_whole():
    """Every tile of every head reaches the output once, however the list of tiles falls on warps and CTAs."""
    import random

    from symm_mem_recipes_b200._ext import C
    assert C.check_kv4_cuts([], 3) == 0 and C.check_kv4_cuts([0, 0], 3) == 0
    assert C.check_kv4_cuts([2048] * 8, 296) == 0 and C.check_kv4_cuts([1] * 2400, 296) == 0 and C.check_kv4_cuts([9000], 296) == 0
    for seed in range(4000):
        rng = random.Random(seed)
        heads = [rng.choice((0, 1, 1, 2, 3, rng.randint(1, 40))) for _ in range(rng.randint(1, 14))]
        assert C.check_kv4_cuts(heads, rng.randint(1, 7)) == 0, (seed, heads)


def test_stack_refuses_positions_that_are_none():
    """A step over 4-bit caches takes positions of 32 bits; refused before anything is written."""
    from symm_mem_recipes_b200.models.llama_tp_layer import LlamaTPStack

    class Sequences:
        positions = torch.full((3,), 7, dtype=torch.int32)

        def step(self, x):
            return x + 1

    stack = LlamaTPStack.__new__(LlamaTPStack)
    stack.sequences = Sequences()
    for pos in (-1, 2 ** 31, 2 ** 31 + 5, -2 ** 40):
        with pytest.raises(ValueError, match="position"):
            stack.decode_step(torch.zeros(1), pos)
    assert stack.sequences.positions.tolist() == [7] * 3
    assert stack.decode_step(torch.zeros(1), 2 ** 31 - 1).item() == 1 and stack.sequences.positions.tolist() == [2 ** 31 - 1] * 3
    assert stack.decode_step(torch.zeros(1)).item() == 1


def test_eviction_right_after_a_prompt_warns(monkeypatch):
    """No step has weighed the prompt's slots: all but the recent ones would stay by their age."""
    import warnings

    from symm_mem_recipes_b200.models.llama_tp_layer import Kv4Sequences
    cuts = []
    monkeypatch.setattr(ops, "kv4_evict_", lambda cache, lengths, keep, recent: cuts.append((cache, keep, recent)) or lengths.clamp(max=keep))
    seq = Kv4Sequences.__new__(Kv4Sequences)
    seq.caches, seq.graph, seq.lengths, seq.positions = ["a", "b"], None, torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    seq._run = lambda x: x
    seq.begin(50)
    with pytest.warns(UserWarning, match="no step since the prompt"):
        seq.evict(30, recent=4)
    assert cuts == [("a", 30, 4), ("b", 30, 4)] and seq.lengths.tolist() == [30, 30] and seq.positions.tolist() == [50, 50]
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        seq.evict(20, recent=20)
        seq.step(torch.zeros(1))
        seq.evict(10)
        seq.begin(60)
        seq.step(torch.zeros(1))
        seq.evict(10, recent=3)
    assert seq.lengths.tolist() == [10, 10]


def kernels_of(name):
    """(name, body) of the __global__ functions of a kernel file, comments taken out."""
    import pathlib
    import re
    root = pathlib.Path(ops.__file__).resolve().parent.parent / "csrc" / "kernels"
    text = re.sub(r"//[^\n]*", "", (root / name).read_text())
    out = []
    for m in re.finditer(r"__global__[^;{]*?(\w+)\((?:const\b|int\b|\w+\s+\w+)[^{;]*\)\s*\{", text):
        depth, end = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        out.append((m.group(1), text[m.end():end]))
    return text, out


@pytest.mark.parametrize("name", ["kv4_attention.cu", "kv4_cache.cu", "rope_axes.cu"])
def test_inputs_are_loaded_coherently(name):
    """The kernels start under the one in front, which may still write their inputs: no load by the read-only path."""
    text, kernels = kernels_of(name)
    assert len(kernels) >= 1 and all("pdl_wait()" in body for _, body in kernels)
    assert "ld_16_nc" not in text and "ld.global.nc" not in text and "__ldg" not in text and "__restrict__" not in text


@pytest.mark.parametrize("name", ["kv4_attention.cu", "kv4_cache.cu", "rope_axes.cu"])
def test_nothing_is_read_before_the_wait(name):
    """Lengths, positions and caches belong to the kernels in front until pdl_wait has returned, and every CTA calls it: what
    stands in front of it uses the launch's arguments alone."""
    for kernel, body in kernels_of(name)[1]:
        before = body[:body.index("pdl_wait()")]
        for word in ("tiles_of", "length_of", "lengths[", "pos[", "positions[", "ld_16", "return", "ws."):
            assert word not in before, (kernel, word)
