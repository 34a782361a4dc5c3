"""The operators of a 4-bit KV cache, by which their speed is judged on one GPU.

A decoder layer that serves from a cache of 4.5 bits a value makes four kinds of calls: queries and keys are rotated by
positions of their own (`rope_axes_`), a chunk of a prompt goes into the cache and what is there comes back for the chunk's
attention (`kv4_append_`, `kv4_read`), a new token of every sequence is appended and attends (`kv4_decode_attention_`), and
a cache that has grown keeps its heaviest slots (`kv4_evict_`).  Head counts and widths are those of the package's layer
configurations, whole or as one rank's share.

The cache: uint8 codes [batch, kv heads, slots, D / 2], two values a byte, and bf16 scales [batch, kv heads, slots, D / 32],
one for 32 neighbouring dims; a value is scale * (nibble - 8).  Dim d has g = d / 32.  A key row is four parts of D / 8 bytes,
part c = d % 32 / 8, in it four bytes a group, low nibble first; a value row is eight parts of D / 16 bytes, part
r = d % 32 / 4, in it two bytes a group.
"""
import math
import random

import torch

own = False

_TILE = 64      # slots are allocated in tiles of 64
_THETA = 500000.0


def listed():
    return [
        # one new token of four sequences in a rank's share at TP8, positions of three axes: pure call latency
        {"name": "rope_decode_b4", "kind": "rope", "tokens": 4, "hq": 8, "hkv": 1, "dim": 128, "axes": 3, "interleaved": False,
         "inverse": False},
        # the narrow layer, an odd number of tokens, axes dealt in turn, rotated back
        {"name": "rope_back_1021", "kind": "rope", "tokens": 1021, "hq": 4, "hkv": 1, "dim": 64, "axes": 2, "interleaved": True,
         "inverse": True},
        # a prompt of images and text through the whole layer's heads
        {"name": "rope_prompt_8192", "kind": "rope", "tokens": 8192, "hq": 64, "hkv": 8, "dim": 128, "axes": 3,
         "interleaved": True, "inverse": False},
        # a few tokens a sequence behind a short prompt, the narrow heads
        {"name": "append_4x5", "kind": "append", "batch": 4, "tokens": 5, "before": 60, "hkv": 1, "dim": 64, "max_seq": 128},
        # an odd chunk of two prompts behind what is there, of which all comes back
        {"name": "append_2x509", "kind": "append", "batch": 2, "tokens": 509, "before": 1500, "hkv": 8, "dim": 128,
         "max_seq": 2048},
        # one long prompt at once, the whole layer's kv heads
        {"name": "append_1x16384", "kind": "append", "batch": 1, "tokens": 16384, "before": 0, "hkv": 8, "dim": 128,
         "max_seq": 16384},
        # one short sequence of a rank's share at TP8: pure call latency
        {"name": "attend_b1_200", "kind": "attend", "batch": 1, "hkv": 1, "group": 8, "dim": 128, "max_seq": 200, "least": 1.0,
         "idle": 0, "weights": False},
        # a full batch at TP8 with one idle row, weights kept for eviction
        {"name": "attend_b16_8192", "kind": "attend", "batch": 16, "hkv": 1, "group": 8, "dim": 128, "max_seq": 8192,
         "least": 0.3, "idle": 1, "weights": True},
        # one very long context, the whole layer, weights kept
        {"name": "attend_b1_131072", "kind": "attend", "batch": 1, "hkv": 8, "group": 8, "dim": 128, "max_seq": 131072,
         "least": 1.0, "idle": 0, "weights": True},
        # a large batch of ragged contexts, the whole layer
        {"name": "attend_b32_16384", "kind": "attend", "batch": 32, "hkv": 8, "group": 8, "dim": 128, "max_seq": 16384,
         "least": 0.4, "idle": 0, "weights": False},
        # a cache that grew by 64 slots goes back to its budget, the narrow heads
        {"name": "evict_b4_to_448", "kind": "evict", "batch": 4, "hkv": 1, "dim": 64, "max_seq": 512, "least": 1.0, "keep": 448,
         "recent": 32},
        # long prompts cut down to what decoding reads
        {"name": "evict_b8_to_4096", "kind": "evict", "batch": 8, "hkv": 8, "dim": 128, "max_seq": 32768, "least": 0.1,
         "keep": 4096, "recent": 256},
    ]


def _log_int(rng, lo, hi):
    """An integer in [lo, hi], uniform in its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("rope", "append", "attend", "attend", "evict"))
    dim = rng.choice((64, 128, 128))
    hkv = rng.choice((1, 2, 4, 8))
    if kind == "rope":
        group = rng.choice((1, 4, 8))
        return {"kind": kind, "tokens": _log_int(rng, 1, 8192), "hq": hkv * group, "hkv": hkv, "dim": dim,
                "axes": rng.randint(1, 3), "interleaved": rng.random() < 0.5, "inverse": rng.random() < 0.3}
    if kind == "append":
        batch = _log_int(rng, 1, 16)
        tokens, before = _log_int(rng, 1, 8192 // batch), rng.choice((0, rng.randint(1, 8192 // batch)))
        return {"kind": kind, "batch": batch, "tokens": tokens, "before": before, "hkv": hkv, "dim": dim,
                "max_seq": tokens + before + rng.randint(0, 100)}
    batch = _log_int(rng, 1, 32)
    if kind == "attend":
        return {"kind": kind, "batch": batch, "hkv": hkv, "group": rng.randint(1, 8), "dim": dim,
                "max_seq": _log_int(rng, 33, min(131072, 2_800_000 // (batch * hkv))), "least": rng.choice((0.0, 0.3, 1.0)),
                "idle": rng.choice((0, 0, batch // 4)), "weights": rng.random() < 0.5}
    max_seq = _log_int(rng, 65, min(65536, 2_000_000 // (batch * hkv)))
    keep = rng.randint(max_seq // 16, max_seq - 1)
    return {"kind": kind, "batch": batch, "hkv": hkv, "dim": dim, "max_seq": max_seq, "least": rng.choice((0.1, 1.0)),
            "keep": keep, "recent": rng.randint(0, min(keep, 256))}


def _lengths(case):
    """Tokens in the cache before the call: from `least` of the slots up to all but one of them; -1 for an idle row."""
    b, s = case["batch"], case["max_seq"]
    got = [max(0, int(s * (case["least"] + (1 - case["least"]) * (i + 1) / b)) - 1) for i in range(b)]
    return [-1 if i < case.get("idle", 0) else n for i, n in enumerate(got)]


def _sections(dim, axes):
    half = dim // 2
    return (half,) if axes == 1 else (half // 2, half // 2) if axes == 2 else (half // 4, half * 3 // 8, half * 3 // 8)


def _axis_of_pair(sections, interleaved):
    """The axis whose position turns pair i: axis after axis, or dealt in turn until an axis has its share."""
    dealt = [(k if interleaved else 0, a) for a, share in enumerate(sections) for k in range(share)]
    return [a for _, a in sorted(dealt)]


def _normal(gen, *shape, std=1.0):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.bfloat16).mul_(std)


def _cache(gen, batch, hkv, max_seq, dim, weights):
    """A cache that has been written: bell-shaped codes, scales that differ from row to row, weights of many steps."""
    slots = -(-max_seq // _TILE) * _TILE
    bell = torch.tensor([-7, -5, -4, -3, -2, -2, -1, 0, 0, 1, 2, 2, 3, 4, 5, 7], device="cuda") + 8
    pairs = (bell[:, None] * 16 + bell[None, :]).reshape(256).to(torch.uint8)
    state = {"max_seq": max_seq}
    for name, mean in (("k", 0.3), ("v", 0.2)):
        random_bytes = torch.randint(0, 256, (batch, hkv, slots, dim // 2), generator=gen, device="cuda", dtype=torch.uint8)
        for at in range(0, slots, 8192):     # an index is eight times a byte
            random_bytes[:, :, at:at + 8192] = pairs[random_bytes[:, :, at:at + 8192].int()]
        state[name + "_codes"] = random_bytes
        rows = torch.randn(batch, hkv, slots, 1, generator=gen, device="cuda")
        groups = torch.randn(batch, hkv, slots, dim // 32, generator=gen, device="cuda")
        state[name + "_scales"] = (mean * torch.exp(0.3 * rows + 0.2 * groups)).bfloat16()
    state["weights"] = torch.rand(batch, hkv, slots, generator=gen, device="cuda").log_().neg_() if weights else None
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dim, hkv = case["kind"], case["dim"], case["hkv"]

    def int32(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    if kind == "rope":
        tokens, hq, sections = case["tokens"], case["hq"], _sections(dim, case["axes"])
        first = torch.randint(0, 200000, (1, 1), generator=gen, device="cuda")       # deep into a conversation
        place = torch.randint(0, 64, (case["axes"], tokens), generator=gen, device="cuda")     # row and column of a patch
        place[0] = torch.arange(tokens, device="cuda")
        axis = torch.tensor(_axis_of_pair(sections, case["interleaved"]), device="cuda")
        return {"kind": kind, "qkv": _normal(gen, tokens, (hq + 2 * hkv) * dim), "n_heads": hq + hkv, "dim": dim,
                "positions": (first + place).int(), "sections": sections, "axis": axis, "interleaved": case["interleaved"],
                "inverse": case["inverse"]}
    batch = case["batch"]
    if kind == "append":
        tokens, before = case["tokens"], case["before"]
        qkv = _normal(gen, batch, tokens, 3 * hkv * dim)
        qkv[..., 5::dim] *= 6                                                        # a dim that stands out, as in keys
        k, v = qkv[..., hkv * dim:2 * hkv * dim], qkv[..., 2 * hkv * dim:]           # views of the projection's output
        turn = random.Random(seed)
        return {"kind": kind, **_cache(gen, batch, hkv, case["max_seq"], dim, False),
                "k": k.unflatten(2, (hkv, dim)), "v": v.unflatten(2, (hkv, dim)),
                "start": int32([max(0, before - turn.randint(0, 40)) for _ in range(batch)]),
                "counts": int32([tokens - turn.randint(0, tokens // 8) for _ in range(batch)]), "read": tokens + before}
    lengths = _lengths(case)
    random.Random(seed).shuffle(lengths)
    state = {"kind": kind, **_cache(gen, batch, hkv, case["max_seq"], dim, case.get("weights", True)),
             "lengths": int32([max(n, 0) if kind == "evict" else n for n in lengths])}
    if kind == "attend":
        hq = hkv * case["group"]
        state.update(qkv=_normal(gen, batch, (hq + 2 * hkv) * dim), hq=hq)
        state["qkv"][:, :hq * dim] *= 2
        return state
    state.update(keep=case["keep"], recent=case["recent"])
    return state


# ---- plain forms ----

def _values(codes, scales, is_key):
    """fp32 values of rows [..., D / 2] of codes and [..., D / 32] of scales."""
    groups = scales.shape[-1]
    both = torch.stack((codes & 15, codes >> 4), dim=-1)
    if is_key:      # (c, g, byte, nibble) -> (g, c, byte, nibble)
        both = both.unflatten(-2, (4, groups, 4)).transpose(-4, -3)
    else:           # (r, g, byte, nibble) -> (g, r, byte, nibble)
        both = both.unflatten(-2, (8, groups, 2)).transpose(-4, -3)
    values = both.flatten(-3).float().sub_(8).mul_(scales.float().unsqueeze(-1))
    return values.flatten(-2)


def _quantised(x, is_key):
    """Codes and scales of bf16 rows [..., D]: scale = bf16(largest / 7), the nearest code, halves to the smaller one."""
    groups = x.float().unflatten(-1, (-1, 32))
    largest = groups.abs().amax(-1)
    scales = torch.where(largest < 2.0 ** -100, 0.0, largest / 7).bfloat16()
    scales = torch.where(torch.isfinite(largest), scales, float("nan"))
    steps = torch.ceil(groups.abs() / scales.float().unsqueeze(-1) - 0.5).nan_to_num(0.0, 0.0, 0.0)
    nibbles = (torch.sign(groups).nan_to_num(0.0) * steps + 8).to(torch.uint8)
    parts = nibbles.unflatten(-1, (4, 4, 2) if is_key else (8, 2, 2)).transpose(-4, -3)
    return (parts[..., 0] | (parts[..., 1] << 4)).flatten(-3), scales


def _plain_rope(s):
    half, heads = s["dim"] // 2, s["n_heads"]
    frequency = _THETA ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    angle = s["positions"][s["axis"]].t().double() * frequency           # far positions: 32 bits would lose the angle
    if s["inverse"]:
        angle = -angle
    cos, sin = angle.cos().float().unsqueeze(1), angle.sin().float().unsqueeze(1)
    part = s["qkv"][:, :heads * s["dim"]].unflatten(1, (heads, s["dim"]))
    x, y = part.float().split(half, dim=2)
    part.copy_(torch.cat((x * cos - y * sin, y * cos + x * sin), dim=2))
    return s["qkv"]


def _plain_append(s):
    batch, tokens = s["k"].shape[:2]
    rows = torch.arange(batch, device="cuda")[:, None]
    slots = s["start"][:, None] + torch.arange(tokens, device="cuda")
    written = (torch.arange(tokens, device="cuda") < s["counts"][:, None])[..., None, None]
    k, k_scale = _quantised(s["k"], True)
    v, v_scale = _quantised(s["v"], False)
    s["k_codes"][rows, :, slots] = torch.where(written, k, s["k_codes"][rows, :, slots])
    s["v_codes"][rows, :, slots] = torch.where(written, v, s["v_codes"][rows, :, slots])
    s["k_scales"][rows, :, slots] = torch.where(written, k_scale, s["k_scales"][rows, :, slots])
    s["v_scales"][rows, :, slots] = torch.where(written, v_scale, s["v_scales"][rows, :, slots])
    n = s["read"]
    k = _values(s["k_codes"][:, :, :n], s["k_scales"][:, :, :n], True).transpose(1, 2).bfloat16()
    v = _values(s["v_codes"][:, :, :n], s["v_scales"][:, :, :n], False).transpose(1, 2).bfloat16()
    return {"k": k.contiguous(), "v": v.contiguous()}


def _plain_attend(s):
    batch, hkv, slots, dim = *s["k_codes"].shape[:3], 2 * s["k_codes"].shape[3]
    q, k, v = s["qkv"].split((s["hq"] * dim, hkv * dim, hkv * dim), dim=1)
    lengths = s["lengths"].long()
    active = lengths >= 0
    rows, at = torch.arange(batch, device="cuda"), lengths.clamp_min(0)
    for name, new in (("k", k), ("v", v)):
        codes, scales = _quantised(new.unflatten(1, (hkv, dim)), name == "k")
        on = active[:, None, None]
        s[name + "_codes"][rows, :, at] = torch.where(on, codes, s[name + "_codes"][rows, :, at])
        s[name + "_scales"][rows, :, at] = torch.where(on, scales, s[name + "_scales"][rows, :, at])
    seen = torch.arange(slots, device="cuda") <= lengths[:, None]
    q = q.unflatten(1, (hkv, -1, dim)).float()
    score = (q @ _values(s["k_codes"], s["k_scales"], True).transpose(2, 3)) / math.sqrt(dim)
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(active[:, None, None, None], top, 0.0))
    p = e / e.sum(-1, keepdim=True).clamp_min(1e-30)
    values = _values(s["v_codes"], s["v_scales"], False).masked_fill(~seen[:, None, :, None], 0.0)
    out = (p @ values).bfloat16().flatten(1)
    if s["weights"] is not None:
        new = (torch.arange(slots, device="cuda") == lengths[:, None])[:, None]
        s["weights"].copy_(torch.where(new, 0.0, s["weights"]) + p.sum(2))
    return out


def _plain_evict(s):
    batch, hkv, slots = s["weights"].shape
    slot, lengths = torch.arange(slots, device="cuda"), s["lengths"][:, None, None]
    worth = torch.where(slot >= lengths - s["recent"], math.inf, s["weights"])
    worth = torch.where(slot < lengths, worth, -math.inf)
    kept = torch.sort(worth, dim=-1, descending=True, stable=True).indices[..., :s["keep"]].sort(-1).values
    for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
        rows = s[name].gather(2, kept.unsqueeze(-1).expand(-1, -1, -1, s[name].shape[3]))
        s[name][:, :, :s["keep"]] = rows
    s["weights"][:, :, :s["keep"]] = s["weights"].gather(2, kept)
    return s["lengths"].clamp_max(s["keep"])


# ---- the package's calls ----

def _handle(s):
    """The cache that a program makes once and keeps."""
    if "cache" not in s:
        from symm_mem_recipes_b200.ops import Kv4Cache
        s["cache"] = Kv4Cache(s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"], s["weights"], max_seq=s["max_seq"])
    return s["cache"]


def _own_run(s):
    from symm_mem_recipes_b200 import ops
    kind = s["kind"]
    if kind == "rope":
        return ops.rope_axes_(s["qkv"], s["n_heads"], s["dim"], s["positions"], s["sections"], _THETA,
                              interleaved=s["interleaved"], inverse=s["inverse"])
    cache = _handle(s)
    if kind == "append":
        ops.kv4_append_(s["k"], s["v"], cache, s["start"], counts=s["counts"])
        k, v = ops.kv4_read(cache, s["read"])
        return {"k": k, "v": v}
    if kind == "attend":
        return ops.kv4_decode_attention_(s["qkv"], cache, s["hq"], s["lengths"])
    return ops.kv4_evict_(cache, s["lengths"], s["keep"], recent=s["recent"])


def run(state):
    """One pass.  What a call updates in place comes back with its result; codes are exact, so they come as they are stored."""
    if own:
        out = _own_run(state)
    else:
        out = {"rope": _plain_rope, "append": _plain_append, "attend": _plain_attend, "evict": _plain_evict}[state["kind"]](state)
    if state["kind"] in ("rope", "append"):
        return out
    return {"out": out, "weights": state["weights"],
            **{name: state[name] for name in ("k_codes", "k_scales", "v_codes", "v_scales")}}


def work(case):
    kind, dim, hkv = case["kind"], case["dim"], case["hkv"]
    row = 2 * (dim // 2 + dim // 16)         # a slot's key and value with their scales
    if kind == "rope":
        rotated = case["tokens"] * (case["hq"] + hkv) * dim
        return {"bytes": 4 * rotated + 4 * case["tokens"] * case["axes"], "flops": 3 * rotated}
    if kind == "append":
        new, read = (case["batch"] * hkv * n for n in (case["tokens"], case["tokens"] + case["before"]))
        return {"bytes": (new + read) * (4 * dim + row), "flops": 4 * dim * (new + read)}
    lengths = [n for n in _lengths(case) if n >= 0]
    if kind == "attend":
        seen = hkv * (sum(lengths) + len(lengths))
        hq = hkv * case["group"]
        return {"bytes": seen * (row + (8 if case["weights"] else 0)) + 2 * case["batch"] * dim * (2 * hq + 2 * hkv),
                "flops": 4 * seen * case["group"] * dim}
    cut = [n for n in lengths if n > case["keep"]]
    return {"bytes": hkv * (4 * sum(cut) + len(cut) * case["keep"] * 2 * (row + 4)), "flops": hkv * sum(cut)}


# ---- the definitions in 64 bits ----

def _exact_rope(s):
    tokens, heads, dim = s["qkv"].shape[0], s["n_heads"], s["dim"]
    out = s["qkv"].double()
    x = out[:, :heads * dim].clone().reshape(tokens, heads, 2, dim // 2)
    for i in range(dim // 2):
        angle = s["positions"][int(s["axis"][i])].double() * math.exp(-math.log(_THETA) * 2 * i / dim)
        turn = torch.polar(torch.ones_like(angle), -angle if s["inverse"] else angle)[:, None]
        z = torch.complex(x[:, :, 0, i], x[:, :, 1, i]) * turn
        x[:, :, 0, i], x[:, :, 1, i] = z.real, z.imag
    out[:, :heads * dim] = x.reshape(tokens, heads * dim)
    return out


def _dims(dim, is_key):
    """(byte, high nibble) of every dim of a row."""
    if is_key:
        return [(d % 32 // 8 * (dim // 8) + d // 32 * 4 + d % 8 // 2, d % 2) for d in range(dim)]
    return [(d % 32 // 4 * (dim // 16) + d // 32 * 2 + d % 4 // 2, d % 2) for d in range(dim)]


def _exact_rows(codes, scales, is_key):
    """Values in 64 bits of codes [n, D / 2] and scales [n, D / 32], dim by dim."""
    dim = 2 * codes.shape[1]
    out = torch.empty(codes.shape[0], dim, dtype=torch.float64, device=codes.device)
    for d, (byte, high) in enumerate(_dims(dim, is_key)):
        nibble = torch.div(codes[:, byte], 16, rounding_mode="floor") if high else codes[:, byte] % 16
        out[:, d] = (nibble.double() - 8) * scales[:, d // 32].double()
    return out


def _exact_round_trip(x):
    """bf16 rows [n, D] as their codes and scales stand for them, in 64 bits; and the scales."""
    x = x.double().reshape(x.shape[0], -1, 32)
    scale = (x.abs().max(-1).values / 7).to(torch.bfloat16).double()
    step = scale.unsqueeze(-1)
    code = torch.floor(x.abs() / step)                       # then one more where that is nearer
    code = code + (x.abs() - code * step > (code + 1) * step - x.abs())
    return (torch.copysign(code, x) * step).flatten(1), scale


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "rope":
        return _exact_rope(s)
    batch, hkv = s["k_codes"].shape[:2]
    pairs = [(b, h) for b in range(batch) for h in range(hkv)]
    if kind == "append":
        n, got = s["read"], {}
        for name in ("k", "v"):
            out = torch.empty(batch, n, hkv, case["dim"], dtype=torch.float64, device="cuda")
            for b, h in pairs:
                out[b, :, h] = _exact_rows(s[name + "_codes"][b, h, :n], s[name + "_scales"][b, h, :n], name == "k")
                first, count = int(s["start"][b]), int(s["counts"][b])
                out[b, first:first + count, h] = _exact_round_trip(s[name][b, :count, h])[0]
            got[name] = out
        return got
    scales = {name: s[name].double() for name in ("k_scales", "v_scales")}
    weights = s["weights"].double() if s["weights"] is not None else None
    out = None
    if kind == "attend":
        dim, hq = case["dim"], s["hq"]
        out = torch.zeros(batch, hq * dim, dtype=torch.float64, device="cuda")
        fresh = s["qkv"][:, hq * dim:].reshape(batch, 2, hkv, dim)
        for b, h in pairs:
            n, g = int(s["lengths"][b]), case["group"]
            if n < 0:
                continue
            rows = []
            for j, name in enumerate(("k", "v")):
                new, scale = _exact_round_trip(fresh[b, j, h][None])
                old = _exact_rows(s[name + "_codes"][b, h, :n], s[name + "_scales"][b, h, :n], name == "k")
                rows.append(torch.cat((old, new)))
                scales[name + "_scales"][b, h, n] = scale[0]
            q = s["qkv"][b, h * g * dim:(h + 1) * g * dim].double().reshape(g, dim)
            p = torch.softmax(q @ rows[0].t() * dim ** -0.5, dim=-1)
            out[b, h * g * dim:(h + 1) * g * dim] = (p @ rows[1]).flatten()
            if weights is not None:
                weights[b, h, n] = 0
                weights[b, h, :n + 1] += p.sum(0)
    else:
        for b, h in pairs:
            n, keep = int(s["lengths"][b]), s["keep"]
            if n <= keep:
                continue
            old = max(0, n - s["recent"])
            w = s["weights"][b, h, :old].tolist()
            order = sorted(range(old), key=lambda i: (-w[i], i))[:keep - (n - old)]
            kept = torch.tensor(sorted(order) + list(range(old, n)), device="cuda")
            weights[b, h, :keep] = weights[b, h, kept]
            for name in scales:
                scales[name][b, h, :keep] = scales[name][b, h, kept]
    return {"out": out, "weights": weights, "k_codes": None, "v_codes": None, **scales}
