"""Decode attention over a 4-bit cache where the list of tiles is cut among warps (two launches), many tiles a warp: the shapes
that a server's batches have, which fill the warps' rings many times over and cut heads between CTAs.

Tolerances, beside those of the scores and of roundings (`off` and the terms of 2^-8, 2^-11 and 2^-10.9, as derived in the file of the
single operators): a warp adds at most T = ceil(tiles / warps) tiles of one head in a chain.  The weighted sum has four MMAs a tile, each of which
loses 2^-18.4 sum p s, p and s probabilities and value scales: 4 T 2^-18.4 sum p s.  The sum of the probabilities takes 8 T fp32
additions in a lane, 3 over lanes, 4 over warps, and one for each of P pieces: relative 2^-24 each, and so do the pieces' values.  A
piece or chain is rescaled once a tile and once a piece at most by an exponential that is off by 2^-22; numerator and sum share that
factor, the accumulated weights see it once for the sum."""
import math

import pytest
import torch

import kv4_reference as ref
from symm_mem_recipes_b200 import ops
from test_gpu_kv4 import copy_of, filled, gen, int32, normal, put, same

pytestmark = pytest.mark.gpu


def rows_of(cache, b, n):
    """Keys and values of a sequence's first n slots, [kv heads, n, D] in 64 bits."""
    return (ref.values(ref.unpack(cache.k_codes[b, :, :n], True), cache.k_scales[b, :, :n]),
            ref.values(ref.unpack(cache.v_codes[b, :, :n], False), cache.v_scales[b, :, :n]))


def check(cache, before, qkv, g, lengths, out):
    hkv, dim = cache.n_kv_heads, cache.head_dim
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    warps = 4 * min(2 * sms, -(-cache.batch * hkv * (cache.slots // 64) // 4))
    tiles = hkv * sum(n // 64 + 1 for n in lengths if 0 <= n < cache.max_seq)
    chain = -(-tiles // warps)
    assert chain >= 8                                    # what this file is about
    q, k, v = qkv.split((g * hkv * dim, hkv * dim, hkv * dim), dim=1)
    want = copy_of(before)
    for b, n in enumerate(lengths):
        if not 0 <= n < cache.max_seq:
            assert not out[b].any()
            continue
        put(want, b, n, k[b].view(hkv, dim), v[b].view(hkv, dim))
        keys, values = rows_of(want, b, n + 1)
        pieces = (n // 64 + 1) // (4 * max(1, tiles // warps)) + 3
        adds = (8 * chain + 7 + pieces) * 2.0 ** -24
        for h in range(hkv):
            queries = q[b].view(hkv, g, dim)[h].double()
            o, p, room, a = ref.attend(queries, keys[h], values[h])
            group_scale = want.k_scales[b, h, :n + 1].double().sum(-1).max() / math.sqrt(dim)
            off = 2 * 2.0 ** -18 * a + 2 * 2.0 ** -10.9 * float(queries.abs().max() * group_scale) + 2.0 ** -19
            ps = (p @ want.v_scales[b, h, :n + 1].double()).repeat_interleave(32, dim=1)
            err = (out[b].view(hkv, g, dim)[h].double() - o).abs()
            tol = 2.0 ** -8 * o.abs() + (2.0 ** -11 + off + 2 * adds) * room + (2.0 ** -10.9 + 4 * chain * 2.0 ** -18.4) * ps
            assert bool((err <= tol).all()), (b, h, n, float((err / tol).max()))
            if cache.weights is not None:
                old = want.weights[b, h, :n + 1].double()
                old[n] = 0
                w = old + p.sum(0)
                err = (cache.weights[b, h, :n + 1].double() - w).abs()
                tol = 2.0 ** -22 * w + (off + adds + (chain + pieces) * 2.0 ** -22) * p.sum(0)
                assert bool((err <= tol).all()), (b, h, n, float((err / tol).max()))
                want.weights[b, h, :n + 1] = cache.weights[b, h, :n + 1]
    assert same(cache, want)


@pytest.mark.parametrize("batch, hkv, g, dim, max_seq, least, weights", [
    # more query heads than a joining CTA each would have room for: one CTA joins all of a kv head's
    (32, 8, 8, 128, 16384, 0, False),
    (50, 8, 3, 64, 8192, 0, True),
    (40, 6, 5, 128, 8000, 0, False),
    (80, 4, 8, 128, 6000, 0, True),
    (80, 4, 4, 64, 6000, 100, False),
    # a joining CTA a query head
    (2, 8, 5, 64, 131000, 90000, False),
    (1, 8, 7, 128, 130000, 129999, True),
    (3, 4, 1, 128, 70000, 60000, False),
    (3, 2, 2, 64, 120000, 110000, True),
])
def test_decode_attention_over_long_lists(batch, hkv, g, dim, max_seq, least, weights):
    cache = filled(200, batch, max_seq, hkv, dim, weights)
    lengths = torch.randint(least, max_seq, (batch,), generator=gen(201), device="cuda").tolist()
    if batch > 4:
        lengths[batch // 2] = -1                         # idle ones, between the others and at both ends
        lengths[0] = max_seq
        lengths[1], lengths[2], lengths[3] = 0, max_seq - 1, 63
        lengths[-1] = -5
    before = copy_of(cache)
    qkv = normal(202, batch, (g + 2) * hkv * dim, std=1.5)
    out = ops.kv4_decode_attention_(qkv, cache, g * hkv, int32(lengths))
    check(cache, before, qkv, g, lengths, out)
    again = copy_of(before)
    assert torch.equal(ops.kv4_decode_attention_(qkv, again, g * hkv, int32(lengths)), out) and same(again, cache)


@pytest.mark.parametrize("dim, weights", [(64, True), (128, False)])
def test_nan_in_long_lists_stays_where_it_is(dim, weights):
    """A NaN in one key of a head that many CTAs share shows in that head's outputs and weights and in no others."""
    batch, hkv, g, max_seq = 2, 8, 4, 70000
    cache = filled(210, batch, max_seq, hkv, dim, weights)
    clean = copy_of(cache)
    lengths = int32([69000, 65432])
    qkv = normal(211, batch, (g + 2) * hkv * dim)
    cache.k_scales[0, 3, 40000, 0] = math.nan
    cache.v_scales[1, 7, 60000, 1] = math.nan            # dims 32..63
    want = ops.kv4_decode_attention_(qkv, clean, g * hkv, lengths).view(batch, hkv, g, dim)
    got = ops.kv4_decode_attention_(qkv, cache, g * hkv, lengths).view(batch, hkv, g, dim)
    bad = torch.isnan(got)
    assert bad[0, 3].all() and bad[1, 7, :, 32:64].all() and int(bad.sum()) == g * dim + g * 32
    assert torch.equal(got[~bad], want[~bad])
    if weights:
        lost = torch.isnan(cache.weights)
        assert lost[0, 3, :69001].all() and int(lost.sum()) == 69001
        assert torch.equal(cache.weights[~lost], clean.weights[~lost])


def test_long_lists_in_graphs_side_by_side():
    """Two captured graphs of one shape replayed on two streams at once: each has scratch of its own."""
    caches = [filled(220 + 10 * i, 6, 20000, 8, 64, True) for i in range(2)]
    qs = [normal(240 + i, 6, 6 * 8 * 64) for i in range(2)]
    lengths = [int32([19999, 0, -1, 15000, 18000, 17000]), int32([5, 19000, 19998, -1, 20000, 16000])]
    want, graphs, outs = [], [], []
    for cache, q, n in zip(caches, qs, lengths):
        c = copy_of(cache)
        want.append((ops.kv4_decode_attention_(q, c, 32, n), c))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.kv4_decode_attention_(q, cache, 32, n))
        graphs.append(g)
    torch.cuda.synchronize()
    for g in graphs:
        with torch.cuda.stream(torch.cuda.Stream()):
            g.replay()
    torch.cuda.synchronize()
    for (o, c), got, cache in zip(want, outs, caches):
        assert torch.equal(o, got) and same(c, cache)


@pytest.mark.parametrize("weights", [False, True])
def test_a_list_without_tiles(weights):
    """All sequences idle, in the form of two launches: rows of zeros, nothing else touched; then one of them goes on."""
    batch, hkv, g, dim = 80, 8, 2, 128
    cache = filled(230, batch, 128, hkv, dim, weights)
    before = copy_of(cache)
    qkv = normal(231, batch, (g + 2) * hkv * dim)
    lengths = [(-1, 128, -2 ** 31, 2 ** 31 - 1)[b % 4] for b in range(batch)]
    out = torch.full((batch, g * hkv * dim), 3.0, dtype=torch.bfloat16, device="cuda")
    assert not ops.kv4_decode_attention_(qkv, cache, g * hkv, int32(lengths), out=out).any() and same(cache, before)
    lengths[77] = 0
    out = ops.kv4_decode_attention_(qkv, cache, g * hkv, int32(lengths))
    put(before, 77, 0, *(qkv[77].view(-1, hkv, dim)[i] for i in (g, g + 1)))
    if weights:
        before.weights[77, :, 0] = g
    v = ref.values(ref.unpack(before.v_codes[77, :, 0], False), before.v_scales[77, :, 0]).repeat_interleave(g, dim=0)
    assert not out[:77].any() and not out[78:].any() and same(cache, before)
    # one slot of probability 1: the scale in fp16 (8 bits of 11, exact), sums cut at 2^-10.9 s and 2^-18.4 15 s, the result in bf16
    tol = 2.0 ** -8 * v.abs() + (2.0 ** -10.9 + 4 * 2.0 ** -18.4) * before.v_scales[77, :, 0].double().repeat_interleave(32, dim=1).repeat_interleave(g, dim=0)
    assert bool(((out[77].view(hkv * g, dim).double() - v).abs() <= tol).all())
