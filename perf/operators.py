"""Performance cases of the attention operators that stand between a layer's Q/K/V projections and its output projection.

A case is a dict of plain values. `kind` names the operator:

    rotary      CudaRuntime.rotary_device       rotary positions of the queries, out of place
    cache       CudaRuntime.kv_write_device     new keys and values quantised into a paged cache (keys rotated on the way if
                CudaRuntime.kv_read_device      `rotary_dim` is not 0), and the same tokens read back
    attention   CudaRuntime.attention_device    one new token, or a few draft tokens, of every sequence over its paged cache

`heads` query heads, `kv_heads` key and value heads of `dim` values; `format` is what the cache holds (bf16, or int8 or e4m3
codes with a scale for each token and head); `page` tokens per page. Heads of 256 values with 24 query and 4 key heads, 64 of
the 256 values rotated, pages of int8 codes and contexts of up to 262144 tokens are those of the benchmark's model; the others
are generic. Where `own` is false the operators are computed in their plain form.
"""
import math

import numpy as np
import torch

own = False

_LAST = {}  # the runtime of this process, created once as a serving program does


def _runtime():
    if "rt" not in _LAST:
        from qwen38_metal_b200 import CudaRuntime

        _LAST["rt"] = CudaRuntime(0)
    return _LAST["rt"]


# ---- cases ----------------------------------------------------------------------------------------------------------


def _rotary(name, tokens, heads, dim, rotary_dim, layout, scaling, first, x, out):
    return {"name": name, "kind": "rotary", "tokens": tokens, "heads": heads, "dim": dim, "rotary_dim": rotary_dim,
            "layout": layout, "scaling": scaling, "first": first, "x": x, "out": out}


def _cache(name, sequences, tokens, past, kv_heads, dim, fmt, page, x, out, rotary_dim=0):
    return {"name": name, "kind": "cache", "sequences": sequences, "tokens": tokens, "past": past, "kv_heads": kv_heads,
            "dim": dim, "format": fmt, "page": page, "x": x, "out": out, "rotary_dim": rotary_dim}


def _attention(name, sequences, shortest, longest, drafts, heads, kv_heads, dim, fmt, page, x, out):
    return {"name": name, "kind": "attention", "sequences": sequences, "shortest": shortest, "longest": longest,
            "drafts": drafts, "heads": heads, "kv_heads": kv_heads, "dim": dim, "format": fmt, "page": page, "x": x,
            "out": out}


def listed():
    return [
        # the queries of one decode token, as the projection leaves them: the smallest call
        _rotary("rotary_decode", 1, 24, 256, 64, "half", "none", 8191, "f32", "bf16"),
        # the queries of a prompt block
        _rotary("rotary_prompt", 2048, 24, 256, 64, "half", "none", 0, "f32", "bf16"),
        # a prompt chunk of odd length far into a context that was stretched four times, whole heads, neighbouring pairs
        _rotary("rotary_far", 777, 32, 128, 128, "interleaved", "yarn", 200001, "bf16", "bf16"),
        # one decode step of sixteen requests: keys rotated, quantised and appended
        _cache("cache_append", 16, 16, 5000, 4, 256, "int8", 16, "f32", "bf16", 64),
        # a prompt block of one request, written and taken back in full precision
        _cache("cache_prompt_int8", 1, 4096, 4099, 4, 256, "int8", 16, "f32", "f32"),
        # prompts of five requests in one call, 8-bit floating point, large pages
        _cache("cache_prompts_e4m3", 5, 3005, 129, 8, 128, "e4m3", 64, "bf16", "bf16"),
        # the first decode steps of a chat: latency
        _attention("attention_start", 1, 37, 37, 1, 24, 4, 256, "int8", 16, "f32", "bf16"),
        # one request in the middle of a context
        _attention("attention_8k", 1, 8200, 8200, 1, 24, 4, 256, "int8", 16, "f32", "bf16"),
        # a serving batch of very different lengths
        _attention("attention_lanes", 32, 500, 8000, 1, 24, 4, 256, "int8", 16, "f32", "bf16"),
        # one request at the model's full context
        _attention("attention_long", 1, 262144, 262144, 1, 24, 4, 256, "int8", 16, "f32", "bf16"),
        # four draft tokens of four requests verified at once over an unquantised cache
        _attention("attention_verify", 4, 9001, 20011, 4, 24, 4, 256, "bf16", 16, "bf16", "f32"),
        # a large batch with smaller heads, 8-bit floating point, large pages: the largest call
        _attention("attention_many", 128, 3100, 5100, 1, 32, 8, 128, "e4m3", 64, "bf16", "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def _one(rng):
    kind = rng.choices(("rotary", "cache", "attention"), (25, 30, 45))[0]
    dim = rng.choice((64, 80, 128, 128, 192, 256, 256))
    x, out = rng.choice(("f32", "f32", "bf16")), rng.choice(("bf16", "bf16", "f32"))
    if kind == "rotary":
        rotary_dim = dim if rng.random() < 0.5 else 2 * rng.randint(4, dim // 2)
        scaling = rng.choice(("none", "linear", "ntk", "yarn"))
        case = _rotary("", _log_int(rng, 1, 8192), rng.choice((1, 4, 8, 15, 24, 32)), dim, rotary_dim,
                       rng.choice(("half", "interleaved")), scaling, _log_int(rng, 1, 1 << 20) - 1, x, out)
    elif kind == "cache":
        sequences = _log_int(rng, 1, 64)
        tokens = sequences if rng.random() < 0.4 else max(sequences, _log_int(rng, 2, 8192))
        # (rotated keys differ in their last bits between two ways to compute them, and a code on a border with them: bf16)
        rotary_dim = rng.choice((0, 0, dim, 16 * rng.randint(1, dim // 16)))
        case = _cache("", sequences, tokens, _log_int(rng, 1, 20000) - 1, rng.choice((1, 2, 4, 8)), dim,
                      rng.choice(("int8", "int8", "e4m3", "bf16")), rng.choice((16, 16, 32, 48, 64, 256)), x,
                      "bf16" if rotary_dim else out, rotary_dim)
    else:
        longest = _log_int(rng, 1, 262144)
        kv_heads = rng.choice((1, 2, 4, 8))
        case = _attention("", _log_int(rng, 1, 256), max(1, round(longest * rng.uniform(0.1, 1))), longest,
                          rng.choice((1, 1, 1, 2, 4, 7)), kv_heads * rng.choice((1, 2, 4, 6, 8, 12)), kv_heads, dim,
                          rng.choice(("int8", "int8", "e4m3", "bf16")), rng.choice((16, 16, 32, 48, 64, 256)), x, out)
    del case["name"]
    return case


def _padded_bytes(case):
    """The plain form's fp32 copies of keys and values, padded to the longest sequence."""
    if case["kind"] != "attention":
        return 0
    return case["sequences"] * case["longest"] * case["kv_heads"] * case["dim"] * 8


def draw(rng):
    """One more case of the same ranges: sizes spread over their logarithm, no larger than the largest listed one."""
    cases = listed()
    most, most_padded = max(_cost(c) for c in cases), max(_padded_bytes(c) for c in cases)
    while True:
        case = _one(rng)
        if _cost(case) <= most and _padded_bytes(case) <= most_padded:
            return case


# ---- inputs ---------------------------------------------------------------------------------------------------------


def _spread(count, lo, hi):
    """`count` lengths from lo to hi in no order, the same for every seed: they are part of the case."""
    return [lo + (i * 40503 + 12345) % 65536 * (hi - lo) // 65535 for i in range(count)]


def _lengths(case):
    return [max(n, case["drafts"]) for n in _spread(case["sequences"], case["shortest"], case["longest"])]


def _new_tokens(case):
    """How many of the call's tokens each sequence gets: as even as it goes, the first ones more."""
    each, more = divmod(case["tokens"], case["sequences"])
    return [each + (s < more) for s in range(case["sequences"])]


_DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16}
_POOL = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn, "bf16": torch.bfloat16}
_BASE, _STRETCH, _TRAINED = 10000000.0, 4.0, 65536  # rotary base; stretched contexts: factor and original length


class State:
    pass


def _frequencies(rotary_dim, scaling):
    """Radians per token of every pair, and the factor on cosine and sine, in 64 bits."""
    i = np.arange(0, rotary_dim, 2, dtype=np.float64)
    if scaling == "linear":
        return _BASE ** (-i / rotary_dim) / _STRETCH, 1.0
    if scaling == "ntk":
        base = _BASE * _STRETCH ** (rotary_dim / (rotary_dim - 2)) if rotary_dim > 2 else _BASE
        return base ** (-i / rotary_dim), 1.0
    f = _BASE ** (-i / rotary_dim)
    if scaling == "none":
        return f, 1.0
    # pairs that turn more than 32 times in the trained length keep their frequency, those that turn less than once are stretched
    edge = lambda turns: rotary_dim * math.log(_TRAINED / (turns * 2 * math.pi)) / (2 * math.log(_BASE))  # noqa: E731
    low, high = max(math.floor(edge(32.0)), 0), min(math.ceil(edge(1.0)), rotary_dim - 1)
    ramp = np.clip((i / 2 - low) / max(high - low, 1e-3), 0.0, 1.0)
    return f / _STRETCH * ramp + f * (1 - ramp), 0.1 * math.log(_STRETCH) + 1.0


def _scaling_of(case):
    return case.get("scaling", "none")


def prepare(case, seed):
    st = State()
    st.case = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    st.stream = torch.cuda.current_stream().cuda_stream
    dim, x, out = case["dim"], _DTYPE[case["x"]], _DTYPE[case["out"]]
    if case.get("rotary_dim"):
        freq, st.factor = _frequencies(case["rotary_dim"], _scaling_of(case))
        st.freq = torch.tensor(freq, device="cuda")
    if case["kind"] == "rotary":
        st.q = randn(case["tokens"], case["heads"], dim).to(x)
        st.positions = case["first"] + torch.arange(case["tokens"], dtype=torch.int32, device="cuda")
        st.out = torch.zeros(case["tokens"], case["heads"], dim, dtype=out, device="cuda")
    else:
        page = case["page"]
        if case["kind"] == "cache":
            new = _new_tokens(case)
            past = _spread(case["sequences"], case["past"] // 2, case["past"])
            ends = [p + n for p, n in zip(past, new)]
            st.positions = i32([p + i for p, n in zip(past, new) for i in range(n)])
            st.sequences = i32([s for s, n in enumerate(new) for _ in range(n)])
            # keys differ in size from channel to channel, as projections make them
            wide = torch.exp(0.5 * randn(case["kv_heads"], dim))
            st.k = (randn(case["tokens"], case["kv_heads"], dim) * wide).to(x)
            st.v = randn(case["tokens"], case["kv_heads"], dim).to(x)
            st.k_out = torch.zeros(st.k.shape, dtype=out, device="cuda")
            st.v_out = torch.zeros(st.v.shape, dtype=out, device="cuda")
        else:
            ends = _lengths(case)
            st.lengths = i32(ends)
            st.q = (2.0 * randn(case["sequences"] * case["drafts"], case["heads"], dim)).to(x)
            st.out = torch.zeros(st.q.shape, dtype=out, device="cuda")
            st.scale = dim ** -0.5
        per = (max(ends) + page - 1) // page
        used = [(n + page - 1) // page for n in ends]
        pages = sum(used) + 3
        # pages as a server hands them out after a while: in no order; entries behind a sequence's last page are 0
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        inside = torch.arange(per, device="cuda")[None, :] < i32(used)[:, None]
        at = torch.arange(per, device="cuda")[None, :] + (torch.cumsum(i32(used), 0) - i32(used))[:, None]
        st.table = torch.where(inside, order[torch.where(inside, at, 0)], 0).to(torch.int32)
        shape = (pages, case["kv_heads"], page)
        st.scales = [torch.ones(0, device="cuda")] * 2
        if case["kind"] == "cache":
            st.pools = [torch.zeros(*shape, dim, dtype=torch.uint8, device="cuda").view(torch.int8).to(torch.bfloat16)
                        if case["format"] == "bf16" else
                        torch.zeros(*shape, dim, dtype=torch.uint8, device="cuda").view(_POOL[case["format"]])
                        for _ in range(2)]
            if case["format"] != "bf16":
                st.scales = [torch.zeros(shape, device="cuda") for _ in range(2)]
        else:
            st.pools = []
            for _ in range(2):
                z = randn(*shape, dim)
                if case["format"] == "int8":
                    z = z.mul_(36.0).round_().clamp_(-127, 127)
                elif case["format"] == "e4m3":
                    z = z.mul_(127.0).clamp_(-448, 448)
                st.pools.append(z.to(_POOL[case["format"]]))
                del z
            if case["format"] != "bf16":
                unit = 1 / 36.0 if case["format"] == "int8" else 1 / 127.0
                st.scales = [unit * (0.5 + torch.rand(shape, generator=gen, device="cuda")) for _ in range(2)]
    if own:
        _handles(st, case)
    return st


def _handles(st, case):
    """What a serving program keeps: the runtime, the rotary frequencies, and where the cache and its page table are."""
    from qwen38_metal_b200 import KvCache, KvTable, capi

    st.rt = _runtime()
    kind = {"f32": capi.Q4B_F32, "bf16": capi.Q4B_BF16}
    st.x_kind, st.out_kind = kind[case["x"]], kind[case["out"]]
    st.rotary = None
    if case.get("rotary_dim"):
        scaling = None
        if _scaling_of(case) != "none":
            scaling = {"kind": _scaling_of(case), "factor": _STRETCH, "original_length": _TRAINED}
        st.rotary = st.rt.rotary_create(case["rotary_dim"], base=_BASE, layout=case.get("layout", "half"), scaling=scaling)
    if case["kind"] != "rotary":
        scaled = case["format"] != "bf16"
        st.kv = KvCache(format=case["format"], kv_heads=case["kv_heads"], head_dim=case["dim"], page_tokens=case["page"],
                        pages=st.pools[0].shape[0], k=st.pools[0].data_ptr(), v=st.pools[1].data_ptr(),
                        k_scales=st.scales[0].data_ptr() if scaled else 0, v_scales=st.scales[1].data_ptr() if scaled else 0)
        st.pages = KvTable(pages=st.table.data_ptr(), sequences=st.table.shape[0], pages_per_sequence=st.table.shape[1])


# ---- one pass -------------------------------------------------------------------------------------------------------


def _run_own(st):
    case, rt = st.case, st.rt
    dim = case["dim"]
    if case["kind"] == "rotary":
        width = case["heads"] * dim
        rt.rotary_device(st.rotary, st.q.data_ptr(), st.x_kind, width, case["tokens"], case["heads"], dim,
                         st.positions.data_ptr(), st.out.data_ptr(), st.out_kind, width, st.stream)
        return st.out
    if case["kind"] == "cache":
        width = case["kv_heads"] * dim
        rt.kv_write_device(st.kv, st.pages, st.positions.data_ptr(), st.sequences.data_ptr(), case["tokens"],
                           st.k.data_ptr(), width, st.v.data_ptr(), width, st.x_kind, st.rotary, st.stream)
        rt.kv_read_device(st.kv, st.pages, st.positions.data_ptr(), st.sequences.data_ptr(), case["tokens"],
                          st.k_out.data_ptr(), width, st.v_out.data_ptr(), width, st.out_kind, st.stream)
        return {"k": st.k_out, "v": st.v_out}
    width = case["heads"] * dim
    rt.attention_device(st.kv, st.pages, st.lengths.data_ptr(), st.q.data_ptr(), st.x_kind, width, case["heads"],
                        case["drafts"], st.scale, st.out.data_ptr(), st.out_kind, width, st.stream)
    return st.out


def _rotated(x, positions, freq, factor, rotary_dim, layout):
    """x [tokens][heads][dim] in 32 bits, rotated; the angles of far positions in 64."""
    angle = positions.double()[:, None] * freq
    c, s = (factor * torch.cos(angle)).float()[:, None, :], (factor * torch.sin(angle)).float()[:, None, :]
    y = x.clone()
    if layout == "half":
        a, b = x[..., :rotary_dim // 2], x[..., rotary_dim // 2:rotary_dim]
        y[..., :rotary_dim // 2], y[..., rotary_dim // 2:rotary_dim] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., 0:rotary_dim:2], x[..., 1:rotary_dim:2]
        y[..., 0:rotary_dim:2], y[..., 1:rotary_dim:2] = a * c - b * s, b * c + a * s
    return y


def _quantised(x, fmt):
    """Codes and scales of x [tokens][heads][dim]: one scale for each token and head. Quotients next to a border in 64 bits."""
    if fmt == "bf16":
        return x.to(torch.bfloat16), None
    scale = x.abs().amax(-1) / torch.full((), 127.0 if fmt == "int8" else 448.0, device=x.device)
    quotient = torch.where(scale[..., None] > 0, x.double() / scale.double()[..., None], 0.0)
    if fmt == "int8":
        return quotient.round().clamp(-127, 127).to(torch.int8), scale
    step = torch.ldexp(torch.ones_like(quotient), torch.frexp(quotient.abs().clamp(min=2.0 ** -6))[1] - 4)
    return ((quotient / step).round() * step).clamp(-448, 448).to(torch.float8_e4m3fn), scale


def _run_plain(st):
    case = st.case
    out = _DTYPE[case["out"]]
    if case["kind"] == "rotary":
        st.out.copy_(_rotated(st.q.float(), st.positions, st.freq, st.factor, case["rotary_dim"], case["layout"]))
        return st.out
    if case["kind"] == "cache":
        page = st.table[st.sequences.long(), (st.positions // case["page"]).long()].long()
        place = (st.positions % case["page"]).long()
        k = st.k.float()
        if case["rotary_dim"]:
            k = _rotated(k, st.positions, st.freq, st.factor, case["rotary_dim"], "half")
        kc, ks = _quantised(k, case["format"])
        vc, vs = _quantised(st.v.float(), case["format"])
        raw = torch.int16 if case["format"] == "bf16" else torch.uint8
        kp, vp = st.pools
        kp.view(raw)[page, :, place] = kc.view(raw)
        vp.view(raw)[page, :, place] = vc.view(raw)
        if ks is not None:
            st.scales[0][page, :, place] = ks
            st.scales[1][page, :, place] = vs
        k_back = kp.view(raw)[page, :, place].view(kp.dtype).float()
        v_back = vp.view(raw)[page, :, place].view(vp.dtype).float()
        if ks is not None:
            k_back = k_back * st.scales[0][page, :, place][..., None]
            v_back = v_back * st.scales[1][page, :, place][..., None]
        return {"k": k_back.to(out), "v": v_back.to(out)}
    seqs, drafts, kvh, dim = case["sequences"], case["drafts"], case["kv_heads"], case["dim"]
    group = case["heads"] // kvh
    table = st.table.long()

    def whole(pool, scales):  # [sequences][kv heads][padded length][dim] in 32 bits
        raw = pool.view(torch.int16 if case["format"] == "bf16" else torch.uint8)[table].view(pool.dtype).float()
        if case["format"] != "bf16":
            raw = raw * scales[table][..., None]
        return raw.permute(0, 2, 1, 3, 4).reshape(seqs, kvh, -1, dim)

    q = st.q.float().view(seqs, drafts, kvh, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, kvh, drafts * group, dim)
    score = torch.matmul(q, whole(st.pools[0], st.scales[0]).transpose(2, 3)) * st.scale
    at = torch.arange(score.shape[-1], device="cuda")
    last = st.lengths[:, None] - drafts + torch.arange(drafts, device="cuda")[None, :]  # [sequences][drafts]
    seen = (at <= last[..., None]).repeat_interleave(group, 1)[:, None]  # [sequences][1][rows][padded length]
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(score - torch.where(top == -math.inf, 0.0, top)), 0.0)
    total = p.sum(-1, keepdim=True)
    v = torch.where((at < st.lengths[:, None])[:, None, :, None], whole(st.pools[1], st.scales[1]), 0.0)
    o = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    o = o.view(seqs, kvh, drafts, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs * drafts, case["heads"], dim)
    st.out.copy_(o)
    return st.out


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# ---- the same from the definition, in 64 bits -----------------------------------------------------------------------


def _turn64(x, positions, freq, factor, rotary_dim, layout):
    z = x.double()
    half = rotary_dim // 2
    first = list(range(half)) if layout == "half" else list(range(0, rotary_dim, 2))
    second = [i + half for i in first] if layout == "half" else [i + 1 for i in first]
    # a pair is a complex number, turned by its angle
    pair = torch.complex(z[..., first], z[..., second])
    angle = torch.outer(positions.double(), freq)
    pair = pair * torch.polar(torch.full_like(angle, factor), angle)[:, None, :]
    z = z.clone()
    z[..., first], z[..., second] = pair.real, pair.imag
    return z


def _held64(x, fmt):
    """What a cache row stands for, from x in 64 bits. The scale is a 32-bit number; a code is the nearest one."""
    if fmt == "bf16":
        return x.float().to(torch.bfloat16).double()
    top = 127.0 if fmt == "int8" else 448.0
    scale = (x.abs().amax(-1, keepdim=True).float().double() / top).float().double()
    if fmt == "int8":
        codes = torch.arange(-127, 128, device=x.device, dtype=torch.float64)
    else:
        every = torch.arange(256, device=x.device, dtype=torch.int32).to(torch.uint8).view(torch.float8_e4m3fn).double()
        codes = torch.unique(every[~every.isnan()])
    ratio = x / scale
    upper = torch.searchsorted(codes, ratio.contiguous()).clamp(1, len(codes) - 1)
    lo, hi = codes[upper - 1], codes[upper]
    even = (upper - 1 - len(codes) // 2) % 2 == 0  # codes count outwards from zero: every other one ends in an even digit
    code = torch.where((ratio - lo < hi - ratio) | ((ratio - lo == hi - ratio) & even), lo, hi)
    return code * scale


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "rotary":
        return _turn64(st.q, st.positions, st.freq, st.factor, case["rotary_dim"], case["layout"])
    if case["kind"] == "cache":
        k = st.k.double()
        if case["rotary_dim"]:
            k = _turn64(st.k, st.positions, st.freq, st.factor, case["rotary_dim"], "half")
        return {"k": _held64(k, case["format"]), "v": _held64(st.v.double(), case["format"])}
    result = torch.zeros(st.q.shape, dtype=torch.float64, device="cuda")
    group, drafts = case["heads"] // case["kv_heads"], case["drafts"]
    for s, n in enumerate(_lengths(case)):
        rows = st.table[s, :(n + case["page"] - 1) // case["page"]].long()
        for h in range(case["kv_heads"]):
            held = []
            for pool, scales in zip(st.pools, st.scales):
                z = pool.view(torch.int16 if case["format"] == "bf16" else torch.uint8)[rows, h].view(pool.dtype).double()
                if case["format"] != "bf16":
                    z = z * scales[rows, h].double()[..., None]
                held.append(z.reshape(-1, case["dim"])[:n])
            for i in range(drafts):
                seen = n - drafts + i + 1
                q = st.q[s * drafts + i, h * group:(h + 1) * group].double()
                weight = torch.softmax(q @ held[0][:seen].T * st.scale, -1)
                result[s * drafts + i, h * group:(h + 1) * group] = weight @ held[1][:seen]
    return result


# ---- work -----------------------------------------------------------------------------------------------------------


def work(case):
    """Inputs read once, outputs written once: a cache row is its codes and its scale."""
    size = {"f32": 4, "bf16": 2, "int8": 1, "e4m3": 1}
    x, out = size[case["x"]], size[case["out"]]
    if case["kind"] == "rotary":
        values = case["tokens"] * case["heads"] * case["dim"]
        turned = case["tokens"] * case["heads"] * case["rotary_dim"]
        return {"bytes": values * (x + out) + 4 * case["tokens"], "flops": 3 * turned}
    row = case["dim"] * size[case["format"]] + (0 if case["format"] == "bf16" else 4)
    if case["kind"] == "cache":
        rows = 2 * case["tokens"] * case["kv_heads"]
        return {"bytes": rows * (case["dim"] * (x + out) + 2 * row) + 16 * case["tokens"], "flops": 4 * rows * case["dim"]}
    lengths = _lengths(case)
    held = 2 * case["kv_heads"] * row * sum(lengths)
    io = case["sequences"] * case["drafts"] * case["heads"] * case["dim"] * (x + out)
    pairs = sum(n - case["drafts"] + i + 1 for n in lengths for i in range(case["drafts"]))
    return {"bytes": held + io + 4 * case["sequences"], "flops": 4 * pairs * case["heads"] * case["dim"]}


def _cost(case):
    w = work(case)
    return w["bytes"] / 6.5e12 + w["flops"] / 1.6e15
