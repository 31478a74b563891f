"""Projections, rotary positions, cache and attention one behind the other, as a layer runs them: every step's cache and result against the
formulas in 64 bits, evaluated on what the layer's own projections gave."""
import math

import pytest

pytestmark = pytest.mark.gpu

HIDDEN = 512
BASE = 1e6


def _job(rt, tensor, n, k, offset):
    from qwen38_metal_b200 import MappedQ4AffineJob

    w, s, b = rt.alloc_shard(n * (k // 2) + offset), rt.alloc_shard(n * (k // 64) * 2 + offset), rt.alloc_shard(n * (k // 64) * 2 + offset)
    job = MappedQ4AffineJob(w, offset, s, offset, b, offset, n, offset % 4 == 0)
    rt.synth_q4(9091, tensor, 0.05, 0, n, k, job)
    return job


def _layer(rt, fmt, heads, kv_heads, dim, sequences, per, page, rotary_dim, tokens):
    from qwen38_metal_b200 import AttentionLayer

    shapes = ((heads * dim, HIDDEN), (kv_heads * dim, HIDDEN), (kv_heads * dim, HIDDEN), (HIDDEN, heads * dim))
    jobs = [_job(rt, i, n, k, 2 if i == 1 else 0) for i, (n, k) in enumerate(shapes)]
    return AttentionLayer(rt, *jobs, HIDDEN, heads, kv_heads, dim, sequences, per, page, fmt, rotary_dim, BASE, None, tokens)


def _share(layer, other):
    """`other` continues what `layer` has begun."""
    for name in ("pools", "scales", "table", "lengths", "cache", "pages"):
        setattr(other, name, getattr(layer, name))


class _Twin:
    """The same cache for the 64-bit forms of attention_helpers, and every key and value that a step has brought."""

    def __init__(self, layer):
        from attention_helpers import Cache

        self.view = Cache.__new__(Cache)
        self.view.fmt, self.view.kv_heads, self.view.dim, self.view.page = layer.cache.format, layer.kv_heads, layer.head_dim, layer.cache.page_tokens
        self.view.table, self.view.pools, self.view.scales = layer.table, layer.pools, layer.scales

    def check(self, rt, layer, x):
        import torch

        from attention_helpers import TOP, attention64, rounded, turned64
        from qwen38_metal_b200 import rotary_frequencies

        rt.device_status()
        freq, factor = rotary_frequencies(layer.rotary_dim_of_test, BASE)
        positions, tokens = layer.positions, layer.tokens
        rows = torch.nonzero(positions >= 0).flatten()
        sequence = (rows // tokens).int()
        # the cache holds the keys turned and the values, each within a step of its type: half a step of codes (one where the largest is
        # involved: its scale is rounded too), or 2^-8 of a bf16 value, and the keys what turning in 32 bits is off by, 2^-21 of the pair
        for side, raw in ((0, layer.keys), (1, layer.values)):
            given = raw[rows].double().view(len(rows), layer.kv_heads, layer.head_dim)
            size = torch.zeros_like(given)
            if side == 0:
                given, size = turned64(given, positions[rows], freq, factor, "half")
            held = self.view.held(side, sequence, positions[rows])[0]
            top = given.abs().amax(-1, keepdim=True)
            if self.view.fmt == "int8":
                room = top * (0.5 / 127 + 2.0 ** -20)
            elif self.view.fmt == "e4m3":
                room = given.abs() * 2.0 ** -4 + top * (2.0 ** -10 / TOP["e4m3"] + 2.0 ** -18)
            else:
                room = given.abs() * 2.0 ** -8 + 2.0 ** -20 * top
            assert bool(((held - given).abs() <= room + 2.0 ** -21 * size).all())
        # queries are turned in place: they are checked by the next lines' inputs being the layer's own
        lengths = layer.lengths.tolist()
        ref, bound = attention64(self.view, lengths, layer.queries.view(-1, layer.heads, layer.head_dim), tokens, layer.scale)
        off = (layer.attended.view_as(ref).double() - ref).abs()
        assert bool((off <= rounded(bound, ref, "bf16")).all())
        out = torch.empty_like(layer.out)
        from qwen38_metal_b200 import capi

        rt.matmul_batch_device(layer.attended.data_ptr(), capi.Q4B_BF16, len(out), layer.heads * layer.head_dim, [layer.o], [out.data_ptr()])
        rt.device_status()
        assert torch.equal(out, layer.out)


@pytest.mark.parametrize("fmt,heads,kv_heads,dim,page,rotary_dim", [("int8", 24, 4, 256, 16, 64), ("e4m3", 8, 2, 128, 64, 128), ("bf16", 6, 2, 64, 32, 32)])
def test_prompts_then_tokens_then_drafts(runtime, fmt, heads, kv_heads, dim, page, rotary_dim):
    import torch

    from qwen38_metal_b200 import capi

    gen = torch.Generator(device="cuda").manual_seed(5)
    sequences, per = 3, -(-96 // page)
    prompt = _layer(runtime, fmt, heads, kv_heads, dim, sequences, per, page, rotary_dim, 16)
    prompt.table.copy_(torch.randperm(sequences * per, generator=torch.Generator().manual_seed(2)).view(sequences, per))
    step = _layer(runtime, fmt, heads, kv_heads, dim, sequences, per, page, rotary_dim, 1)
    draft = _layer(runtime, fmt, heads, kv_heads, dim, sequences, per, page, rotary_dim, 4)
    for other in (step, draft):
        _share(prompt, other)
    for layer in (prompt, step, draft):
        layer.rotary_dim_of_test = rotary_dim
    try:
        x = {layer: torch.randn(sequences * layer.tokens, HIDDEN, generator=gen, device="cuda").to(torch.bfloat16) for layer in (prompt, step, draft)}
        twin = _Twin(prompt)

        def run(layer, new=None):
            layer.advance(new)
            torch.cuda.synchronize()
            layer.forward(x[layer].data_ptr())
            raw = layer.queries
            twin.check(runtime, layer, x[layer])
            return raw

        # prompts of 35, 16 and 0 tokens, sixteen at a time; the queries' turn is checked here
        for new in ([16, 16, 0], [16, 0, 0], [3, 0, 0]):
            run(prompt, torch.tensor(new, dtype=torch.int32, device="cuda"))
        assert prompt.lengths.tolist() == [35, 16, 0] and bool((prompt.attended.view(3, 16, -1)[2] == 0).all())
        given = torch.empty_like(prompt.queries)
        runtime.matmul_batch_device(x[prompt].data_ptr(), capi.Q4B_BF16, len(given), HIDDEN, [prompt.q], [given.data_ptr()])
        runtime.device_status()
        from attention_helpers import turned64
        from qwen38_metal_b200 import rotary_frequencies

        freq, factor = rotary_frequencies(rotary_dim, BASE)
        ref, size = turned64(given.view(-1, heads, dim), prompt.positions, freq, factor, "half")
        padded = prompt.positions < 0
        off = (prompt.queries.view_as(ref).double() - ref).abs() - 2.0 ** -21 * size - 1e-30
        assert bool((off[~padded] <= 0).all())
        # single tokens: the first steps eagerly, the rest as replays of one captured step
        for _ in range(2):
            run(step)
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step.forward(x[step].data_ptr(), stream.cuda_stream)
        for i in range(14):
            x[step].copy_(torch.randn(sequences, HIDDEN, generator=gen, device="cuda").to(torch.bfloat16))
            step.advance()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            if i % 5 == 0 or i == 13:
                twin.check(runtime, step, x[step])
        assert step.lengths.tolist() == [51, 32, 16]
        # the same step eagerly, with nothing between the five launches, gives the same bits
        first = [step.attended.clone(), step.out.clone()]
        for _ in range(3):
            step.attended.fill_(math.nan)
            step.forward(x[step].data_ptr())
            runtime.device_status()
            assert torch.equal(step.attended, first[0]) and torch.equal(step.out, first[1])
        # four draft tokens of each, of which two are kept: the next four are written over the others
        run(draft)
        draft.lengths -= 2
        run(draft)
        assert draft.lengths.tolist() == [57, 38, 22]
    finally:
        for layer in (prompt, step, draft):
            layer.close()


def test_wrong_projections_are_refused(runtime):
    from qwen38_metal_b200 import AttentionLayer, Q4RuntimeError

    q, o = _job(runtime, 0, 128, HIDDEN, 0), _job(runtime, 1, HIDDEN, 128, 0)
    kv = _job(runtime, 2, 64, HIDDEN, 0)
    for jobs, fmt in (((q, kv, q, o), "int8"), ((kv, kv, kv, o), "int8"), ((q, kv, kv, q), "int8"), ((q, kv, kv, o), "int4")):
        with pytest.raises(Q4RuntimeError):
            AttentionLayer(runtime, *jobs, HIDDEN, 2, 1, 64, 1, 1, cache_format=fmt)
    for more in (dict(tokens=0), dict(tokens=17), dict(sequences=0), dict(page_tokens=24)):
        with pytest.raises(Q4RuntimeError):
            AttentionLayer(runtime, q, kv, kv, o, HIDDEN, 2, 1, 64, **{"sequences": 1, "pages_per_sequence": 1, "page_tokens": 16, **more})
