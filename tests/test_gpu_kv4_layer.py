"""The decoder layer's step over a 4-bit cache against the layer in 64 bits, computed from the weights and from what the cache
stands for; alone and over two ranks.

Tolerances.  The step rounds to bf16 twelve times on the way to the layer's change y - x (norm twice, projections, rotation, attention,
activation; scores see the queries' and the key's rounding); each is off by 2^-8 of its vector at most, and random weights carry
relative errors of vectors over as they are.  The two sums of the residual stream are rounded relative to themselves, |x| and the change
together: in all 2^-8 (12 + 2 (|x| + |change|) / |change|) of the change's norm, sequence by sequence.  The new token's row is within
half a code of the key and value that it should be, whose own rounding errors are 2^-8 of the sums of absolute products behind a
pair of dims (the norm's rounding), and three roundings of 2^-8 more."""
import pytest
import torch
import torch.distributed as dist

import kv4_reference as ref
from symm_mem_recipes_b200.utils.testing import spawn_ranks

pytestmark = pytest.mark.gpu


def _sum_over_ranks(t):
    if dist.is_initialized():
        dist.all_reduce(t)
    return t


def _norm(x, w, eps):
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w.double()


def _layer_in_64_bits(lyr, cache, x, lengths, positions, attention=True, head_of=lambda h, hkv, g: h // g):
    """The change of a step, after which `cache` is given, and how far the new rows are from what they should be (in tolerances)."""
    cfg, hq, hkv, dim = lyr.cfg, lyr.hq, lyr.hkv, lyr.cfg.head_dim
    x = x.double()
    h1 = _norm(x, lyr.norm1, cfg.eps)
    w = lyr.w_qkv.double()
    qkv = ref.rope_axes(h1 @ w.t(), hq + hkv, dim, positions, (dim // 2,), cfg.rope_theta)
    room = (h1.abs() @ w.abs().t()).unflatten(1, (-1, 2, dim // 2)).sum(2, keepdim=True).expand(-1, -1, 2, -1).flatten(1)
    pair = qkv.abs().unflatten(1, (-1, 2, dim // 2)).sum(2, keepdim=True).expand(-1, -1, 2, -1).flatten(1)
    attn, worst = torch.zeros(x.shape[0], hq * dim, dtype=torch.float64, device=x.device), 0.0
    for b, n in enumerate(lengths):
        rows = []
        for i, (codes, scales) in enumerate(((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales))):
            got = ref.values(ref.unpack(codes[b, :, :n + 1], i == 0), scales[b, :, :n + 1])
            part = slice((hq + i * hkv) * dim, (hq + (i + 1) * hkv) * dim)
            step = scales[b, :, n].double().repeat_interleave(32, dim=1)
            tol = 0.5 * step + (2.0 ** -8 * room + 3 * 2.0 ** -8 * pair)[b, part].view(hkv, dim) * 1.02
            worst = max(worst, float(((got[:, n] - qkv[b, part].view(hkv, dim)).abs() / tol).max()))
            rows.append(got)
        for h in range(hq):
            kv = head_of(h, hkv, hq // hkv)
            p = torch.softmax(rows[0][kv] @ qkv[b, h * dim:(h + 1) * dim] / dim ** 0.5, dim=0)
            attn[b, h * dim:(h + 1) * dim] = p @ rows[1][kv]
    x1 = x + _sum_over_ranks(attn @ lyr.w_o.double().t()) * attention
    gate, up = (_norm(x1, lyr.norm2, cfg.eps) @ lyr.w_gate_up.double().t()).split(lyr.ffn_local, dim=1)
    y = x1 + _sum_over_ranks((torch.nn.functional.silu(gate) * up) @ lyr.w_down.double().t())
    return y - x, worst


def _off(got, want):
    return (got - want).norm(dim=1) / want.norm(dim=1)


def _worker(rank, world_size):
    from symm_mem_recipes_b200.models.llama_tp_layer import LlamaTPConfig, LlamaTPStack
    from symm_mem_recipes_b200.parallel import symm_mem

    dev = torch.device("cuda", rank)
    cfg = LlamaTPConfig(hidden=512, n_heads=8 * world_size, n_kv_heads=2 * world_size, head_dim=64, ffn=512 * world_size)
    batch, prompt = 4, 40
    eager, graph = (LlamaTPStack(cfg, 2, dev, batch, max_seq=96, seed=7, kv_bits=4, track_weights=True, use_graph=g)
                    for g in (False, True))
    assert graph.graph is not None and eager.graph is None
    for stack in (eager, graph):
        for lyr in stack.layers:                     # attention that tells its slots apart and moves the stream
            for w, part, by in ((lyr.w_qkv, slice(0, lyr.hq * 64), 8), (lyr.w_o, slice(None), 16)):
                w[part] *= by
            if lyr.w_o_t is not None:
                lyr.w_o_t.copy_(lyr.w_o.t())
    g = torch.Generator().manual_seed(4)             # the same activations on every rank
    x = (torch.randn(batch * prompt, cfg.hidden, generator=g) * 0.5).to(torch.bfloat16).to(dev)
    rows = batch * prompt // world_size
    for stack in (eager, graph):
        stack.prefill(x[rank * rows:(rank + 1) * rows].contiguous(), prompt)
        symm_mem.check_status(dev)
        stack.sequences.lengths.copy_(torch.tensor([40, 23, 31, 40]))          # as if some had been cut
        stack.sequences.positions.copy_(torch.tensor([40, 64, 37, 40]))
    failures = []
    for step in range(3):
        x = (torch.randn(batch, cfg.hidden, generator=g) * 0.5).to(torch.bfloat16).to(dev)
        lengths, positions = eager.sequences.lengths.clone(), eager.sequences.positions.clone()
        h = x
        for i, (lyr, cache) in enumerate(zip(eager.layers, eager.caches)):
            y = lyr.decode_kv4(h, cache, lengths, positions)
            symm_mem.check_status(dev)
            change, rows_off = _layer_in_64_bits(lyr, cache, h, lengths.tolist(), positions)
            size, ratio = change.norm(dim=1), h.double().norm(dim=1)
            tol = 2.0 ** -8 * (12 + 2 * (ratio + size) / size)
            off = _off(y.double() - h.double(), change)
            if not bool((off <= tol).all()):
                failures.append(f"step {step}, layer {i}: off by {off.tolist()}, allowed {tol.tolist()}")
            if not rows_off <= 1:
                failures.append(f"step {step}, layer {i}: the new rows are {rows_off} tolerances off")
            # what would be a mistake is far outside: another position, no attention, heads that read others' keys
            other, rows_other = _layer_in_64_bits(lyr, cache, h, lengths.tolist(), lengths)
            none = _layer_in_64_bits(lyr, cache, h, lengths.tolist(), positions, attention=False)[0]
            mixed = _layer_in_64_bits(lyr, cache, h, lengths.tolist(), positions, head_of=lambda h, hkv, g: h % hkv)[0]
            if not (rows_other > 2 and float((_off(other, change) / tol)[1]) > 2 and bool((_off(none, change) > 2 * tol).all()) and
                    bool((_off(mixed, change) > 2 * tol).all())):
                failures.append(f"step {step}, layer {i}: a mistake would not show")
            h = y
        eager.sequences.lengths += 1
        eager.sequences.positions += 1
        got = graph.decode_step(x)
        symm_mem.check_status(dev)
        size = h.double().norm(dim=1)
        if not bool(((got.double() - h.double()).norm(dim=1) <= 2.0 ** -7 * 28 * size).all()):      # both within 14 roundings
            failures.append(f"step {step}: the graph's step is not the eager one")
        if not (torch.equal(graph.sequences.lengths, eager.sequences.lengths) and
                torch.equal(graph.sequences.positions, eager.sequences.positions)):
            failures.append(f"step {step}: lengths or positions")
    torch.cuda.synchronize()
    del graph
    assert not failures, failures


def test_layer_over_a_4_bit_cache_world_of_one():
    torch.cuda.set_device(0)
    _worker(0, 1)


@pytest.mark.multigpu(2)
def test_layer_over_a_4_bit_cache_2gpu():
    spawn_ranks(_worker, 2, "nccl")


def test_tensor_parallel_prefill_into_a_4_bit_cache():
    """`forward_tp` leaves in a 4-bit cache what `kv4_append_` makes of its 16-bit keys and values."""
    from symm_mem_recipes_b200 import ops
    from symm_mem_recipes_b200.models.llama_tp_layer import LlamaTPConfig, LlamaTPDecoderLayer

    dev = torch.device("cuda", 0)
    torch.cuda.set_device(0)
    cfg = LlamaTPConfig.tiny(1)
    for fused_glue in (True, False):
        layer = LlamaTPDecoderLayer(cfg, dev, seed=3, fused_glue=fused_glue)
        x = (torch.randn(2 * 33, cfg.hidden, generator=torch.Generator().manual_seed(1)) * 0.5).to(torch.bfloat16).to(dev)
        kv = tuple(torch.zeros(2, 33, layer.hkv, cfg.head_dim, dtype=torch.bfloat16, device=dev) for _ in range(2))
        cache, want = (ops.Kv4Cache.new(2, 50, layer.hkv, cfg.head_dim, dev, track_weights=True) for _ in range(2))
        y = layer.forward_tp(x, 2, 33, kv_cache=kv)
        assert torch.equal(layer.forward_tp(x, 2, 33, kv_cache=cache), y)
        ops.kv4_append_(*kv, want)
        for name in ("k_codes", "k_scales", "v_codes", "v_scales", "weights"):
            assert torch.equal(getattr(cache, name), getattr(want, name)), name
        with pytest.raises(ValueError, match="Kv4Cache of this batch"):
            layer.forward_tp(x, 2, 33, kv_cache=ops.Kv4Cache.new(2, 32, layer.hkv, cfg.head_dim, dev))
