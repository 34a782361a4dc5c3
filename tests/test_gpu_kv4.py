"""The 4-bit cache's operators on a GPU against their definitions in 64 bits.

Tolerances.  A rounding to bf16 is off by 2^-8 of the result at most.  Codes and scales are exact.  The rotation's
sine and cosine are off by 2^-21.1 (the intrinsic's bound on [-pi, pi]) and 2^-21.3 for the fp32 angle, together under 2^-20,
and three fp32 roundings add 3 * 2^-24: 2^-19.5 (|x| + |y|) covers both.  A score is a sum of head_dim <= 128 fp32 products in
at most 64 dependent steps: off by 2^-18 A, A the largest sum |q k| / sqrt(D), and so is p relative to itself, twice
(numerator and sum), with 2^-20 for the exponential; the probabilities may be rounded to fp16 (2^-11) on their way into the
weighted sum, which adds 2^-18 of sum p |v| for its own steps.

Both sums may be taken over nibbles n = c + 8 in [1, 15] by tensor cores, with 8 sum(q s) or 8 sum(p s) taken off.  An MMA adds 17
numbers, each cut at 2^-24 of twice the largest nominal product or of the accumulator.  Products: a nibble may be a subnormal of
bf16 (nominal 2^-126, unit 2^-133) or one of fp16 (2^-14, unit 2^-22): 17 * 2^-24 * 2^8 = 2^-11.9 of the largest |q| s, two MMAs a
group of 32 dims, so 2^-10.9 max|q| sum_g s / sqrt(D) in a score; 17 * 2^-24 * 2^9 = 2^-10.9 of p s, and the largest p s
of each MMA add up to no more than sum p s.  Accumulators: k of them in a chain lose k * 2^-23 of the total, 15 sum p s, and of 8
sum p s: k * 2^-18.4 sum p s.  A warp has four such MMAs a tile of 64 slots and goes on to a second tile once the work has more
tiles than warps: k = 8 for up to 512 tiles in all and 8 more for every further 512 is no less."""
import math

import pytest
import torch

import kv4_reference as ref
from symm_mem_recipes_b200 import ops

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(seed, *shape, std=1.0):
    return (torch.randn(*shape, generator=gen(seed), device="cuda") * std).to(BF16)


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def filled(seed, batch, max_seq, hkv, dim, weights=False):
    """A cache whose every slot holds something, the unused ones too."""
    cache = ops.Kv4Cache.new(batch, max_seq, hkv, dim, "cuda", track_weights=weights)
    for i, (codes, scales) in enumerate(((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales))):
        c = torch.randint(-7, 8, (batch, hkv, cache.slots, dim), generator=gen(seed + i), device="cuda")
        codes.copy_(ref.pack(c, i == 0))
        scales.copy_(torch.rand(scales.shape, generator=gen(seed + 2 + i), device="cuda") * 0.3 + 0.02)
    if weights:
        cache.weights.copy_(torch.rand(cache.weights.shape, generator=gen(seed + 4), device="cuda") * 3)
    return cache


def copy_of(cache):
    w = cache.weights.clone() if cache.weights is not None else None
    return ops.Kv4Cache(cache.k_codes.clone(), cache.k_scales.clone(), cache.v_codes.clone(), cache.v_scales.clone(), w,
                        max_seq=cache.max_seq)


def same(a, b):
    """Every byte of two caches."""
    for name in ("k_codes", "k_scales", "v_codes", "v_scales", "weights"):
        x, y = getattr(a, name), getattr(b, name)
        if x is not None and not torch.equal(x.view(torch.uint8), y.view(torch.uint8)):
            return False
    return True


def put(cache, b, slot, k, v):
    """The rows [hkv, D] of one slot by the definition."""
    for i, (x, codes, scales) in enumerate(((k, cache.k_codes, cache.k_scales), (v, cache.v_codes, cache.v_scales))):
        c, s = ref.quantise(x)
        codes[b, :, slot] = ref.pack(c, i == 0)
        scales[b, :, slot] = s


def content(cache, b, h, n):
    return (ref.values(ref.unpack(cache.k_codes[b, h, :n], True), cache.k_scales[b, h, :n]),
            ref.values(ref.unpack(cache.v_codes[b, h, :n], False), cache.v_scales[b, h, :n]))


# ---- rotation ----

@pytest.mark.parametrize("tokens, hq, hkv, dim, sections, interleaved, inverse", [
    (1, 8, 1, 128, (16, 24, 24), False, False),
    (37, 8, 1, 128, (16, 24, 24), True, False),
    (130, 64, 8, 128, (24, 20, 20), True, True),
    (1021, 4, 1, 64, (8, 12, 12), True, False),
    (65, 3, 3, 64, (32,), False, True),
    (9, 1, 1, 64, (0, 31, 1), False, False),
    (18, 2, 1, 128, (1,) * 8 + (7,) * 8, True, False),
])
def test_rope_axes(tokens, hq, hkv, dim, sections, interleaved, inverse):
    x = normal(1, tokens, (hq + 2 * hkv) * dim)
    pos = torch.randint(-(1 << 27), 1 << 27, (len(sections), tokens), generator=gen(2), device="cuda").int()
    pos[:, ::2] %= 5000
    theta = 500000.0
    # 64-bit angles of positions up to 2^27 are good to about 2^27 * 2^-52 = 2^-25
    want = ref.rope_axes(x, hq + hkv, dim, pos, sections, theta, interleaved, inverse)
    got = x.clone()
    assert ops.rope_axes_(got, hq + hkv, dim, pos, sections, theta, interleaved, inverse) is got
    heads = x[:, :(hq + hkv) * dim].double().abs().unflatten(1, (hq + hkv, 2, dim // 2))
    room = (heads[:, :, 0] + heads[:, :, 1])[:, :, None].expand_as(heads).reshape(tokens, -1)
    err = (got.double() - want)[:, :(hq + hkv) * dim].abs()
    assert bool((err <= 2.0 ** -8 * want[:, :(hq + hkv) * dim].abs() + 2.0 ** -19.5 * room).all())
    assert torch.equal(got[:, (hq + hkv) * dim:], x[:, (hq + hkv) * dim:])


def test_rope_axes_equal_positions_is_rope():
    """Text: the axes agree, and small positions give what `rope_` gives, up to one bf16 step of either rounding."""
    x = normal(3, 64, 5 * 128)
    a, b = x.clone(), x.clone()
    pos = torch.arange(7, 71, device="cuda").int().expand(3, 64)
    ops.rope_axes_(a, 4, 128, pos, (16, 24, 24), 500000.0)
    ops.rope_(b, 4, 128, 64, 500000.0, pos0=7)
    assert bool(((a.double() - b.double()).abs() <= 2.0 ** -7 * b.double().abs() + 2.0 ** -14).all())


def test_rope_axes_strided_rows_and_empty():
    wide = normal(4, 11, 4 * 64 + 64)
    rows = wide[:, 32:32 + 4 * 64]
    pos = torch.arange(11, device="cuda").int()
    want = rows.contiguous()
    ops.rope_axes_(want, 3, 64, pos, (32,), 1e4)
    before = wide.clone()
    ops.rope_axes_(rows, 3, 64, pos, (32,), 1e4)
    assert torch.equal(rows, want)
    assert torch.equal(wide[:, :32], before[:, :32]) and torch.equal(wide[:, 288:], before[:, 288:])
    ops.rope_axes_(wide[:0, :256], 3, 64, pos[:0], (32,), 1e4)
    ops.rope_axes_(want, 0, 64, pos, (32,), 1e4)


def test_rope_axes_inverse_is_the_gradient():
    """d/dx <w, R x> = R^T w, the rotation back; against differences in 64 bits of the definition, and of the call."""
    tokens, dim, sections = 5, 64, (8, 12, 12)
    pos = torch.randint(0, 9000, (3, tokens), generator=gen(5), device="cuda").int()
    x, w = normal(6, tokens, dim), normal(7, tokens, dim)
    grad = ops.rope_axes_(w.clone(), 1, dim, pos, sections, 1e4, interleaved=True, inverse=True).double()
    for i in range(0, dim, 5):
        step = torch.zeros(tokens, dim, dtype=torch.float64, device="cuda")
        step[:, i] = 0.5
        up = ref.rope_axes(x.double() + step, 1, dim, pos, sections, 1e4, True)
        down = ref.rope_axes(x.double() - step, 1, dim, pos, sections, 1e4, True)
        diff = ((up - down) * w.double()).sum(1)                  # the map is linear: exact up to 64-bit rounding
        pair = w.double()[:, i % 32].abs() + w.double()[:, i % 32 + 32].abs()
        assert bool(((grad[:, i] - diff).abs() <= 2.0 ** -8 * diff.abs() + 2.0 ** -19.5 * pair).all())


# ---- rows in and out ----

@pytest.mark.parametrize("dim, hkv", [(64, 1), (64, 3), (128, 1), (128, 8)])
@pytest.mark.parametrize("tokens, start, counts", [(1, [0, 63], None), (5, [60, 3], [5, 0]), (77, [0, 51], [70, 77])])
def test_append_and_read(dim, hkv, tokens, start, counts):
    cache = filled(10, 2, 130, hkv, dim, weights=True)
    want = copy_of(cache)
    qkv = normal(11, 2, tokens, 3 * hkv * dim, std=3.0)
    k, v = (qkv[..., i * hkv * dim:(i + 1) * hkv * dim].unflatten(2, (hkv, dim)) for i in (1, 2))
    for b in range(2):
        for t in range(tokens if counts is None else counts[b]):
            put(want, b, start[b] + t, k[b, t], v[b, t])
            want.weights[b, :, start[b] + t] = 0
    got = ops.kv4_append_(k, v, cache, int32(start), counts=None if counts is None else int32(counts))
    assert got is cache and same(cache, want)
    for n in (0, 1, 130):
        rk, rv = ops.kv4_read(cache, n)
        assert rk.shape == rv.shape == (2, n, hkv, dim)
        for b in range(2):
            for h in range(hkv):
                wk, wv = content(want, b, h, n)
                assert torch.equal(rk[b, :, h], wk.to(BF16)) and torch.equal(rv[b, :, h], wv.to(BF16))
    assert ops.kv4_read(cache)[0].shape[1] == 130


def test_append_values_of_every_kind():
    """Zeros, halves between two codes, tiny and huge groups, infinities and NaN, each group by itself."""
    row = normal(12, 1, 8, 1, 128)
    row[0, 0, 0, :32] = 0
    row[0, 1, 0, :32] = torch.arange(32, device="cuda").to(BF16) / 4 - 3.5       # scale bf16(0.6) and halves of it
    row[0, 2, 0, :32] = torch.tensor([7.0] + [0.5, 1.5, -2.5, 6.5, -6.5, 3.0, -0.5] * 4 + [0.0] * 3, device="cuda").to(BF16)
    row[0, 3, 0, 5] = math.inf
    row[0, 4, 0, 40] = math.nan
    row[0, 5, 0, 64:96] = 2.0 ** -110
    row[0, 5, 0, 96:] = 2.0 ** -99
    row[0, 6, 0, :64] = 3.0e38
    row[0, 7, 0, 33] = -math.inf
    cache = ops.Kv4Cache.new(1, 8, 1, 128, "cuda")
    ops.kv4_append_(row, -row, cache)
    for t in range(8):
        ck, sk = ref.quantise(row[0, t])
        cv, sv = ref.quantise(-row[0, t])
        assert torch.equal(cache.k_codes[0, :, t], ref.pack(ck, True)), t
        assert torch.equal(cache.v_codes[0, :, t], ref.pack(cv, False)), t
        assert torch.equal(cache.k_scales[0, :, t].nan_to_num(-1), sk.nan_to_num(-1)), t
        assert torch.equal(cache.v_scales[0, :, t].nan_to_num(-1), sv.nan_to_num(-1)), t
    k, _ = ops.kv4_read(cache, 8)
    nan = torch.isnan(k[0, :, 0]).unflatten(1, (4, 32)).all(-1)
    assert torch.isnan(k).sum().item() == nan.sum().item() * 32
    assert nan.nonzero().tolist() == [[3, 0], [4, 1], [7, 1]]


def test_append_from_an_int_and_unlike_strides():
    """One start for all; keys contiguous, values a transposed view."""
    cache, want = filled(16, 2, 90, 3, 128, weights=True), None
    want = copy_of(cache)
    k, v = normal(17, 2, 4, 3, 128), normal(18, 2, 3, 4, 128).transpose(1, 2)
    for b in range(2):
        for t in range(4):
            put(want, b, 86 + t, k[b, t], v[b, t])
            want.weights[b, :, 86 + t] = 0
    ops.kv4_append_(k, v, cache, 86)
    assert same(cache, want)


def test_append_outside_is_skipped():
    """A start from the device that leaves the cache writes only what is inside."""
    cache = filled(13, 4, 70, 2, 64)
    want = copy_of(cache)
    k, v = normal(14, 4, 6, 2, 64), normal(15, 4, 6, 2, 64)
    start = [66, -3, 70, 2147483647]
    for t in range(4):
        put(want, 0, 66 + t, k[0, t], v[0, t])
    ops.kv4_append_(k, v, cache, int32(start))
    assert same(cache, want)
    ops.kv4_append_(k[:, :0], v[:, :0], cache)
    assert same(cache, want)


def test_append_more_tokens_than_an_int_counts():
    """One row, broadcast over 2^31 + 3 tokens: what fits is written, the rest dropped."""
    cache = filled(16, 1, 70, 1, 64)
    want = copy_of(cache)
    k, v = normal(17, 1, 1, 1, 64), normal(18, 1, 1, 1, 64)
    for t in range(66, 70):
        put(want, 0, t, k[0, 0], v[0, 0])
    ops.kv4_append_(k.expand(1, 2 ** 31 + 3, 1, 64), v.expand(1, 2 ** 31 + 3, 1, 64), cache, int32([66]))
    assert same(cache, want)


# ---- attention ----

def check_attention(cache, qkv, hq, lengths, out, before):
    """`out` and `cache` after the call against `before`, the cache ahead of it."""
    tiles = sum(n // 64 + 1 for n in lengths if 0 <= n < cache.max_seq) * cache.n_kv_heads
    chain = 8 * (1 + tiles // 512)
    batch, hkv, dim, g = cache.batch, cache.n_kv_heads, cache.head_dim, hq // cache.n_kv_heads
    want = copy_of(before)
    q, k, v = qkv.split((hq * dim, hkv * dim, hkv * dim), dim=1)
    for b in range(batch):
        n = lengths[b]
        if not 0 <= n < cache.max_seq:
            assert not out[b].any()
            continue
        put(want, b, n, k[b].view(hkv, dim), v[b].view(hkv, dim))
        for h in range(hkv):
            keys, values = content(want, b, h, n + 1)
            o, p, room, a = ref.attend(q[b].view(hkv, g, dim)[h].double(), keys, values)
            group_scale = want.k_scales[b, h, :n + 1].double().sum(-1).max() / math.sqrt(dim)
            off = 2 * 2.0 ** -18 * a + 2 * 2.0 ** -10.9 * float(q[b].view(hkv, g, dim)[h].abs().max() * group_scale) + 2.0 ** -19
            err = (out[b].view(hkv, g, dim)[h].double() - o).abs()
            ps = (p @ want.v_scales[b, h, :n + 1].double()).repeat_interleave(32, dim=1)
            tol = 2.0 ** -8 * o.abs() + (2.0 ** -11 + 2.0 ** -18 + off) * room + (2.0 ** -10.9 + chain * 2.0 ** -18.4) * ps + 1e-30
            assert bool((err <= tol).all()), (b, h, n, float((err / tol).max()))
            if cache.weights is not None:
                old = want.weights[b, h, :n + 1].double()
                old[n] = 0
                w = old + p.sum(0)
                err = (cache.weights[b, h, :n + 1].double() - w).abs()
                tol = 2.0 ** -22 * w + off * p.sum(0)
                assert bool((err <= tol).all()), (b, h, n, float((err / tol).max()))
                want.weights[b, h, :n + 1] = cache.weights[b, h, :n + 1]
    assert same(cache, want)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("hkv, g", [(1, 8), (2, 1), (3, 5), (8, 2)])
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("lengths", [[0], [1], [62, 63, 64, 65], [129, -1, 299, 300, 0, 17, 2000000000]])
def test_decode_attention(dim, hkv, g, weights, lengths):
    cache = filled(20, len(lengths), 300, hkv, dim, weights)
    before = copy_of(cache)
    qkv = normal(21, len(lengths), (g + 2) * hkv * dim, std=2.0)
    given = qkv.clone()
    out = ops.kv4_decode_attention_(qkv, cache, g * hkv, int32(lengths))
    check_attention(cache, qkv, g * hkv, lengths, out, before)
    assert torch.equal(qkv, given)


@pytest.mark.parametrize("batch, hkv, g, dim, max_seq, least", [
    (1, 1, 8, 128, 20011, 20010), (2, 2, 4, 128, 9001, 1), (40, 2, 3, 64, 700, 0), (300, 1, 2, 64, 100, 0), (1, 8, 8, 64, 33000, 32000),
    (160, 1, 8, 128, 130, -9), (75, 2, 5, 128, 320, -40), (19, 8, 1, 64, 1000, 0), (3, 3, 7, 128, 5000, 0), (33, 2, 8, 128, 2048, 0),
    (1024, 1, 4, 64, 64, -20), (1000, 1, 1, 128, 200, -50),
])
def test_decode_attention_long_and_many(batch, hkv, g, dim, max_seq, least):
    """Contexts over many tiles and CTAs, batches over many warps, ragged lengths."""
    cache = filled(22, batch, max_seq, hkv, dim, weights=True)
    before = copy_of(cache)
    qkv = normal(23, batch, (g + 2) * hkv * dim)
    lengths = torch.randint(least, max_seq, (batch,), generator=gen(24), device="cuda").tolist()
    out = ops.kv4_decode_attention_(qkv, cache, g * hkv, int32(lengths))
    check_attention(cache, qkv, g * hkv, lengths, out, before)


def test_decode_attention_int_length_out_and_strides():
    cache = filled(25, 2, 150, 2, 128)
    before = copy_of(cache)
    wide = normal(26, 2, (8 + 4) * 128 + 64)
    qkv = wide[:, 64:]
    out = torch.empty(2, 8 * 128, dtype=BF16, device="cuda")
    assert ops.kv4_decode_attention_(qkv, cache, 8, 149, out=out) is out
    check_attention(cache, qkv, 8, [149, 149], out, before)


def test_decode_attention_scales_of_all_sizes():
    """Value scales over 60 binades, the largest last; a key that wins by far: the sum keeps what each key contributes."""
    cache = filled(27, 1, 260, 1, 128, weights=True)
    n = 250
    cache.v_scales[0, 0, :n] = (2.0 ** torch.linspace(-30, 30, n, device="cuda"))[:, None].to(BF16)
    before = copy_of(cache)
    qkv = normal(28, 1, 10 * 128, std=0.3)
    out = ops.kv4_decode_attention_(qkv, cache, 8, int32([n]))
    check_attention(cache, qkv, 8, [n], out, before)
    cache = copy_of(before)
    cache.k_codes[0, 0, 3] = ref.pack(ref.quantise(qkv[0, :128].clone())[0], True)
    cache.k_scales[0, 0, 3] = 40.0              # slot 3, whose values are 2^-29 of the largest, takes all of query 0
    before = copy_of(cache)
    out = ops.kv4_decode_attention_(qkv, cache, 8, int32([n]))
    check_attention(cache, qkv, 8, [n], out, before)


def test_decode_attention_zero_values():
    cache = ops.Kv4Cache.new(2, 100, 1, 64, "cuda", track_weights=True)
    qkv = torch.zeros(2, 6 * 64, dtype=BF16, device="cuda")
    out = ops.kv4_decode_attention_(qkv, cache, 4, int32([0, 70]))
    assert not out.any()
    assert cache.weights[0, 0, 0].item() == 4.0
    assert bool(((cache.weights[1, 0, :71] - 4 / 71).abs() <= 2.0 ** -20).all()) and not cache.weights[1, 0, 71:].any()


def test_decode_attention_large_queries():
    """A query of 2^117 is a number, over keys of zero the mean of the values; one of 2^118 counts as an infinity."""
    cache = filled(31, 1, 100, 1, 64)
    cache.k_scales.zero_()
    before = copy_of(cache)
    qkv = normal(32, 1, 6 * 64)
    qkv[0, 4 * 64:5 * 64] = 0
    qkv[0, 64 + 5] = 2.0 ** 117
    qkv[0, 2 * 64 + 5] = -2.0 ** 118
    out = ops.kv4_decode_attention_(qkv, cache, 4, int32([90])).view(4, 64)
    assert torch.isnan(out[2]).all() and int(torch.isnan(out).sum()) == 64
    calm = normal(32, 1, 6 * 64)
    calm[0, 4 * 64:5 * 64] = 0
    cache = copy_of(before)
    want = ops.kv4_decode_attention_(calm, cache, 4, int32([90]))
    check_attention(cache, calm, 4, [90], want, before)
    want = want.view(4, 64)
    assert torch.equal(out[[0, 1, 3]], want[[0, 1, 3]])      # all scores are zero either way


def test_decode_attention_nan_stays_where_it_is():
    """NaN behind the last slot is not read; in a visible row it shows in what reads it and nowhere else."""
    cache = filled(29, 2, 200, 2, 128, weights=True)
    clean = copy_of(cache)
    qkv = normal(30, 2, 8 * 128)
    for scales in (cache.k_scales, cache.v_scales):
        scales[0, :, 101:] = math.nan
        scales[1, :, 151:] = math.inf
    want = ops.kv4_decode_attention_(qkv, clean, 4, int32([100, 150]))
    got = ops.kv4_decode_attention_(qkv, cache, 4, int32([100, 150]))
    assert torch.equal(got, want) and torch.equal(cache.weights, clean.weights)
    cache.v_scales[0, 1, 50, 2] = math.nan        # dims 64..95 of head 1's values
    cache.k_scales[1, 0, 9, 1] = math.nan         # a key of head 0
    got = ops.kv4_decode_attention_(qkv, cache, 4, int32([100, 150])).view(2, 2, 2, 128)
    want = want.view(2, 2, 2, 128)
    bad = torch.isnan(got)
    assert bad[0, 1, :, 64:96].all() and bad[1, 0].all() and int(bad.sum()) == 2 * 32 + 2 * 128
    assert torch.equal(got[~bad], want[~bad])
    qkv[0, 128 + 7] = math.nan                    # query head 1 of sequence 0
    got = ops.kv4_decode_attention_(qkv, clean, 4, int32([100, 150])).view(2, 4, 128)
    bad = torch.isnan(got)
    assert bad[0, 1].all() and int(bad.sum()) == 128
    assert torch.isnan(clean.weights[0, 0, :101]).all() and not torch.isnan(clean.weights[0, 1]).any()


def test_decode_attention_is_repeatable():
    """The same call gives the same bits, whatever ran before it."""
    cache = filled(31, 5, 3000, 2, 128, weights=True)
    qkv, lengths = normal(32, 5, 12 * 128), int32([2999, 100, 1500, 0, 2222])
    first = copy_of(cache)
    want = ops.kv4_decode_attention_(qkv, first, 8, lengths)
    for _ in range(3):
        again = copy_of(cache)
        got = ops.kv4_decode_attention_(qkv, again, 8, lengths)
        assert torch.equal(got, want) and same(again, first)


def test_decode_attention_on_two_streams_and_in_graphs():
    """Two calls at once and two captured graphs: each has scratch of its own; lengths are read at replay."""
    a, b = filled(33, 4, 5000, 2, 128, True), filled(34, 3, 4000, 1, 64, True)
    qa, qb = normal(35, 4, 12 * 128), normal(36, 3, 10 * 64)
    la, lb = int32([4000, 10, 4999, 77]), int32([3999, 2000, 5])
    ca, cb = copy_of(a), copy_of(b)
    wa, wb = ops.kv4_decode_attention_(qa, ca, 8, la), ops.kv4_decode_attention_(qb, cb, 8, lb)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    xa, xb = copy_of(a), copy_of(b)
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        oa = ops.kv4_decode_attention_(qa, xa, 8, la)
    with torch.cuda.stream(s2):
        ob = ops.kv4_decode_attention_(qb, xb, 8, lb)
    torch.cuda.synchronize()
    assert torch.equal(oa, wa) and torch.equal(ob, wb) and same(xa, ca) and same(xb, cb)
    graphs, outs, caches, lens = [], [], [copy_of(a), copy_of(b)], [la.clone().zero_(), lb.clone().zero_()]
    for cache, q, hq, n in zip(caches, (qa, qb), (8, 8), lens):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.kv4_decode_attention_(q, cache, hq, n))
        graphs.append(g)
    lens[0].copy_(la)
    lens[1].copy_(lb)
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        graphs[0].replay()
    with torch.cuda.stream(s2):
        graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], wa) and torch.equal(outs[1], wb) and same(caches[0], ca) and same(caches[1], cb)


def test_first_calls_in_a_capture():
    """A process whose first calls are captured: what is looked up once is looked up then."""
    import subprocess
    import sys
    code = """
import torch
from symm_mem_recipes_b200 import ops
cache = ops.Kv4Cache.new(3, 5000, 2, 128, "cuda", track_weights=True)
x, n = torch.randn(3, 12 * 128, device="cuda").bfloat16(), torch.tensor([4000, 0, 77], dtype=torch.int32, device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    ops.rope_axes_(x, 10, 128, n, (64,), 1e4)
    out = ops.kv4_decode_attention_(x, cache, 8, n)
    new = ops.kv4_evict_(cache, n + 1, 50)
y = x.clone()
g.replay()
torch.cuda.synchronize()
fresh = ops.Kv4Cache.new(3, 5000, 2, 128, "cuda", track_weights=True)
ops.rope_axes_(y, 10, 128, n, (64,), 1e4)
want = ops.kv4_decode_attention_(y, fresh, 8, n)
assert torch.equal(x, y) and torch.equal(out, want) and new.tolist() == [50, 1, 50]
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=200)


def test_offsets_beyond_32_bits():
    """A cache whose codes pass 4 GB: the last sequence's rows are written, attended and evicted at their own place."""
    batch, hkv, slots, dim = 17, 8, 1 << 19, 128
    free, _ = torch.cuda.mem_get_info()
    if free < 30 << 30:
        pytest.skip("needs 30 GB")
    cache = ops.Kv4Cache.new(batch, slots, hkv, dim, "cuda", track_weights=True)
    assert cache.k_codes.numel() > 1 << 32
    n, b = 900, batch - 1
    k, v = normal(37, 1, n, hkv, dim), normal(38, 1, n, hkv, dim)
    small = ops.Kv4Cache.new(1, 1024, hkv, dim, "cuda", track_weights=True)
    ops.kv4_append_(k, v, small)
    wide = torch.zeros(batch, n, hkv, dim, dtype=BF16, device="cuda")
    counts = [0] * b + [n]
    wide_v = wide.clone()
    wide[b], wide_v[b] = k[0], v[0]
    ops.kv4_append_(wide, wide_v, cache, 0, counts=int32(counts))
    qkv = normal(39, 1, 10 * hkv * dim)
    all_qkv = qkv.expand(batch, -1).contiguous()
    lengths = [-1] * b + [n]
    got = ops.kv4_decode_attention_(all_qkv, cache, 8 * hkv, int32(lengths))
    before = ops.Kv4Cache.new(1, 1024, hkv, dim, "cuda", track_weights=True)
    ops.kv4_append_(k, v, before)
    last = ops.Kv4Cache(cache.k_codes[b:, :, :1024].contiguous(), cache.k_scales[b:, :, :1024].contiguous(),
                        cache.v_codes[b:, :, :1024].contiguous(), cache.v_scales[b:, :, :1024].contiguous(),
                        cache.weights[b:, :, :1024].contiguous())
    check_attention(last, qkv, 8 * hkv, [n], got[b:], before)
    assert not got[:b].any()
    ops.kv4_decode_attention_(qkv, small, 8 * hkv, int32([n]))
    small.weights.copy_(last.weights)
    ops.kv4_evict_(small, int32([n + 1]), 300, recent=7)
    new = ops.kv4_evict_(cache, int32([-1] * b + [n + 1]), 300, recent=7)
    assert new.tolist() == [-1] * b + [300]
    for name in ("k_codes", "k_scales", "v_codes", "v_scales", "weights"):
        assert torch.equal(getattr(cache, name)[b, :, :300], getattr(small, name)[0, :, :300]), name


# ---- eviction ----

def check_evict(cache, lengths, keep, recent):
    want = copy_of(cache)
    for b, n in enumerate(lengths):
        for h in range(cache.n_kv_heads):
            if not keep < n <= cache.max_seq:
                continue
            stay = torch.tensor(ref.evict_order(cache.weights[b, h], n, keep, recent), device="cuda")
            for name in ("k_codes", "k_scales", "v_codes", "v_scales", "weights"):
                getattr(want, name)[b, h, :keep] = getattr(cache, name)[b, h, stay]
    new = ops.kv4_evict_(cache, int32(lengths), keep, recent)
    assert new.tolist() == [n if n > cache.max_seq else min(n, keep) for n in lengths]
    assert same(cache, want)


@pytest.mark.parametrize("dim, hkv", [(64, 1), (128, 3)])
@pytest.mark.parametrize("max_seq, lengths, keep, recent", [
    (70, [70, 1, 0, -1, 71, 33], 32, 5), (2, [2], 1, 0), (2, [2], 1, 1), (300, [300, 299], 299, 299), (300, [300, 250], 7, 0),
    (6001, [6001, 5000, 4097], 4096, 100), (40001, [40001], 2500, 64), (131072, [131072, 100000], 60000, 1)])
def test_evict(dim, hkv, max_seq, lengths, keep, recent):
    check_evict(filled(40, len(lengths), max_seq, hkv, dim, weights=True), lengths, keep, recent)


def test_evict_ties_and_odd_weights():
    """Equal weights go to the lower slot; zeros of both signs are equal; infinities and NaN are the heaviest."""
    cache = filled(41, 6, 3000, 1, 64, weights=True)
    w = cache.weights[:, 0]
    w[0].fill_(0.25)
    w[1] = torch.randint(0, 3, (cache.slots,), generator=gen(42), device="cuda").float()
    w[2].zero_()
    w[2, ::2] = -0.0
    w[3, ::7] = math.inf
    w[3, 1::7] = math.nan
    w[4].neg_()
    w[5] = 2.0 ** -torch.arange(cache.slots, device="cuda").float().remainder(149)
    check_evict(cache, [3000, 2999, 2000, 3000, 2500, 3000], 1000, 10)


def test_evict_in_a_graph_and_beside_another():
    a, b = filled(43, 2, 9000, 2, 128, True), filled(44, 3, 500, 1, 64, True)
    la, lb = int32([9000, 8000]), int32([500, 400, 300])
    wa, wb = copy_of(a), copy_of(b)
    ops.kv4_evict_(wa, la, 1000, 50)
    ops.kv4_evict_(wb, lb, 350, 50)
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    na, nb = la.clone().zero_(), lb.clone().zero_()
    with torch.cuda.graph(ga):
        oa = ops.kv4_evict_(a, na, 1000, 50)
    with torch.cuda.graph(gb):
        ob = ops.kv4_evict_(b, nb, 350, 50)
    na.copy_(la)
    nb.copy_(lb)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        ga.replay()
    with torch.cuda.stream(s2):
        gb.replay()
    torch.cuda.synchronize()
    assert oa.tolist() == [1000, 1000] and ob.tolist() == [350, 350, 300]
    assert same(a, wa) and same(b, wb)


# ---- a run of them together ----

@pytest.mark.parametrize("hkv, g, dim", [(1, 8, 128), (2, 2, 64)])
def test_serving_run(hkv, g, dim):
    """Ragged prompts, a chunk behind them, decode steps with positions of their own, eviction, more steps; against a cache
    kept by the definitions."""
    batch, hq, max_seq, theta = 3, hkv * g, 200, 500000.0
    heads, sections = hq + 2 * hkv, (dim // 8, dim // 8, dim // 4)
    cache = ops.Kv4Cache.new(batch, max_seq, hkv, dim, "cuda", track_weights=True)
    counts = [50, 7, 33]
    qkv = normal(50, batch * 50, heads * dim)
    pos = torch.randint(0, 300, (3, batch * 50), generator=gen(51), device="cuda").int()
    ops.rope_axes_(qkv, hq + hkv, dim, pos, sections, theta)
    k, v = (qkv.view(batch, 50, heads, dim)[:, :, i:i + hkv] for i in (hq, hq + hkv))
    ops.kv4_append_(k, v, cache, 0, counts=int32(counts))
    ops.kv4_append_(k[:, :9], v[:, :9], cache, int32(counts))
    rk, _ = ops.kv4_read(cache, 16)
    assert torch.equal(rk[1, 7:14], rk[1, :7])
    lengths, seen = int32([n + 9 for n in counts]), int32([n + 9 for n in counts])
    for step in range(12):
        before = copy_of(cache)
        x = normal(60 + step, batch, heads * dim)
        ops.rope_axes_(x, hq + hkv, dim, seen, (dim // 2,), theta)
        out = ops.kv4_decode_attention_(x, cache, hq, lengths)
        check_attention(cache, x, hq, lengths.tolist(), out, before)
        lengths += 1
        seen += 1
        if step == 7:
            check_evict(cache, lengths.tolist(), 40, 8)
            lengths = lengths.clamp(max=40)


@pytest.mark.parametrize("batch, hkv, max_seq", [(3, 2, 700), (160, 1, 300), (2, 4, 21000)])
def test_steps_back_to_back_are_the_steps_one_by_one(batch, hkv, max_seq):
    """Launches that start under their predecessors: a chain of steps without a pause gives the bits of one with pauses."""
    g, dim, keep = 4, 128, max_seq // 3
    results = []
    for pause in (True, False):
        cache = filled(91, batch, max_seq, hkv, dim, weights=True)
        lengths = torch.randint(0, max_seq - 10, (batch,), generator=gen(92), device="cuda").int()
        outs = []
        for step in range(8):
            x = normal(93 + step, batch, (g + 2) * hkv * dim)
            if pause:
                torch.cuda.synchronize()
            ops.rope_axes_(x, (g + 1) * hkv, dim, lengths, (64,), 1e4)
            if pause:
                torch.cuda.synchronize()
            outs.append(ops.kv4_decode_attention_(x, cache, g * hkv, lengths))
            if pause:
                torch.cuda.synchronize()
            lengths = lengths + 1
            if step % 3 == 2:
                lengths = ops.kv4_evict_(cache, lengths, keep, recent=5)
            if pause:
                torch.cuda.synchronize()
            k, v = ops.kv4_read(cache, 33)
            ops.kv4_append_(v[:, :2], k[:, 3:5], cache, 7)
        results.append((torch.stack(outs), cache))
    torch.cuda.synchronize()
    assert torch.equal(results[0][0], results[1][0]) and same(results[0][1], results[1][1])


@pytest.mark.parametrize("batch, hkv, max_seq", [(9, 8, 9000), (2, 4, 21000)])
def test_evict_then_decode_with_nothing_between(batch, hkv, max_seq):
    """Lengths that an eviction has just written, straight into a decode step of two launches, five times over: the bits of
    the same calls with pauses."""
    g, dim = 5, 128
    xs = [normal(101 + i, batch, (g + 2) * hkv * dim) for i in range(5)]
    full = torch.randint(max_seq - 200, max_seq + 1, (batch,), generator=gen(100), device="cuda").int()
    full[0] = -1
    if batch > 2:
        full[1] = 17
    results = []
    for pause in (True, False):
        cache = filled(102, batch, max_seq, hkv, dim, weights=True)
        lengths, outs, news = full.clone(), [], []
        torch.cuda.synchronize()
        for i, x in enumerate(xs):
            lengths = ops.kv4_evict_(cache, lengths, max_seq - 300 - 1500 * i, recent=5)
            if pause:
                torch.cuda.synchronize()
            outs.append(ops.kv4_decode_attention_(x, cache, g * hkv, lengths))
            news.append(lengths)
            if pause:
                torch.cuda.synchronize()
        results.append((torch.stack(outs), torch.stack(news), cache))
    torch.cuda.synchronize()
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    assert same(results[0][2], results[1][2])
    assert results[0][1][-1].max().item() == max_seq - 6300


# ---- the layer and the stack ----

def stack_of(**kw):
    from symm_mem_recipes_b200.models.llama_tp_layer import LlamaTPConfig, LlamaTPStack
    cfg = LlamaTPConfig(hidden=512, n_heads=8, n_kv_heads=2, head_dim=64, ffn=512)
    return LlamaTPStack(cfg, 2, torch.device("cuda", torch.cuda.current_device()), batch=3, max_seq=96, seed=3, **kw)


def test_stack_with_a_4_bit_cache():
    """A prompt and steps through two layers: the graph's steps are the eager ones, a step is what its ops make of it one by one,
    and the prompt's rows are in the caches as `kv4_append_` puts them there."""
    from symm_mem_recipes_b200.models.llama_tp_layer import new_kv_caches
    graph, eager = stack_of(kv_bits=4, track_weights=True), stack_of(kv_bits=4, track_weights=True, use_graph=False)
    plain = stack_of(use_graph=False)
    x = normal(70, 3 * 40, 512, std=0.5)
    y = graph.prefill(x, 40)
    assert torch.equal(y, eager.prefill(x, 40)) and torch.equal(y, plain.prefill(x, 40))
    for cache, (kc, vc) in zip(graph.caches, plain.caches):
        want = ops.Kv4Cache.new(3, 96, 2, 64, "cuda", track_weights=True)
        ops.kv4_append_(kc[:, :40], vc[:, :40], want)
        assert same(cache, want)
    assert graph.sequences.lengths.tolist() == [40] * 3
    far = 0.0
    for step in range(6):
        x = normal(80 + step, 3, 512, std=0.5)
        manual = [copy_of(c) for c in eager.caches]
        lengths, positions = eager.sequences.lengths.clone(), eager.sequences.positions.clone()
        a, b = graph.decode_step(x).clone(), eager.decode_step(x)
        assert torch.equal(a, b)
        h = x
        for lyr, cache in zip(eager.layers, manual):
            qkv = ops.gemv(ops.rms_norm(h, lyr.norm1, lyr.cfg.eps), lyr.w_qkv, weights_nk=True)
            ops.rope_axes_(qkv, lyr.hq + lyr.hkv, 64, positions, (32,), lyr.cfg.rope_theta)
            out = ops.kv4_decode_attention_(qkv, cache, lyr.hq, lengths)
            h2, x1 = ops.rms_norm(lyr._row_parallel_decode(out, "o", True), lyr.norm2, lyr.cfg.eps, residual=h)
            h = x1 + lyr._row_parallel_decode(ops.silu_mul(ops.gemv(h2, lyr.w_gate_up, weights_nk=True)), "down", True)
        assert torch.equal(h, b) and all(same(m, c) for m, c in zip(manual, eager.caches))
        assert torch.isfinite(a).all()
        ref16 = plain.decode_step(x, 40 + step)
        far = max(far, float((a.double() - ref16.double()).norm() / ref16.double().norm()))
    assert far < 1.0        # four bits instead of sixteen, not another function
    graph.evict(30, recent=4)
    assert graph.sequences.lengths.tolist() == [30] * 3 and graph.sequences.positions.tolist() == [46] * 3
    graph.sequences.lengths[1] = -1
    before = [copy_of(c) for c in graph.caches]
    y = graph.decode_step(normal(90, 3, 512, std=0.5))
    assert torch.isfinite(y).all() and graph.sequences.lengths.tolist() == [31, -1, 31]
    assert graph.sequences.positions.tolist() == [47, 46, 47]
    for was, now in zip(before, graph.caches):
        assert torch.equal(was.k_codes[1], now.k_codes[1]) and torch.equal(was.weights[1], now.weights[1])
    graph.reset()
    assert not graph.caches[0].weights.any() and graph.sequences.lengths.tolist() == [0] * 3
    assert len(new_kv_caches(plain.layers, 1, 4)) == 2


def test_stack_of_full_caches():
    """A sequence that has filled its caches waits, unchanged, until they are cut."""
    stack = stack_of(kv_bits=4, track_weights=True)
    stack.prefill(normal(91, 3 * 90, 512, std=0.5), 90)
    stack.sequences.lengths[1] = stack.sequences.positions[1] = 95
    for step in range(3):
        stack.decode_step(normal(92 + step, 3, 512, std=0.5))
    assert stack.sequences.lengths.tolist() == [93, 96, 93] and stack.sequences.positions.tolist() == [93, 96, 93]
    stack.evict(40, recent=8)
    before = [copy_of(c) for c in stack.caches]
    stack.decode_step(normal(95, 3, 512, std=0.5))
    assert stack.sequences.lengths.tolist() == [41] * 3 and stack.sequences.positions.tolist() == [94, 97, 94]
    for was, now in zip(before, stack.caches):
        assert not torch.equal(was.k_codes[1, :, 40], now.k_codes[1, :, 40])


def test_stack_refuses():
    with pytest.raises(ValueError, match="kv_bits"):
        stack_of(kv_bits=8)
    with pytest.raises(ValueError, match="4-bit"):
        stack_of(track_weights=True)
    plain = stack_of(use_graph=False)
    with pytest.raises(ValueError, match="kv_bits=4"):
        plain.evict(3)
    with pytest.raises(ValueError, match="position"):
        plain.decode_step(torch.zeros(3, 512, dtype=BF16, device="cuda"))
    with pytest.raises(ValueError, match="Kv4Cache of this batch"):
        plain.layers[0].forward(normal(1, 3 * 8, 512), 3, 8, kv_cache=ops.Kv4Cache.new(2, 96, 2, 64, "cuda"))
