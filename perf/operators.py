"""The paged 8-bit key/value cache: what its two operators are timed and compared on, and their plain forms.

``ops.kv_append`` rotates the keys of new tokens by their positions and writes keys and values into pages as e4m3 codes with a
power-of-two scale for each (page, head); the queries of the same tokens are rotated beside them.  ``ops.fa_paged`` is the
attention of the new tokens over the cache.  Sizes are those of this repository's own configurations (heads 32/8, 64/8, 12, 16;
head_dim 64 and 128) or generic ones.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_HEADS = ((32, 8), (64, 8), (16, 16), (12, 12), (28, 4), (8, 1))
_MIN_EXP, _MAX_EXP = -100, 119  # of a scale: e4m3 times the scale stays a normal bf16 and finite


# ------------------------------------------------------------------------------------------------------------------------
# the cases
# ------------------------------------------------------------------------------------------------------------------------
def _case(op, B, n, ragged, cached, Hq, Hkv, D, page, dtype, layout="bhsd", lse=False):
    """B sequences with up to ``cached`` tokens in the cache and n new ones each (ragged: 1 to n)."""
    return dict(op=op, B=B, n=n, ragged=ragged, cached=cached, Hq=Hq, Hkv=Hkv, D=D, page=page, dtype=dtype, layout=layout, lse=lse)


def listed():
    return [
        # one token for one sequence: what a single user waits for
        _case("append", 1, 1, False, 1000, 32, 8, 128, 64, "bf16") | {"name": "append B1 one token"},
        # a decode step of a full batch
        _case("append", 64, 1, False, 1500, 32, 8, 128, 64, "bf16") | {"name": "append B64 one token"},
        # prompts of 2048 tokens
        _case("append", 4, 2048, False, 0, 32, 8, 128, 64, "bf16") | {"name": "append B4 prompts"},
        # a batch of prompts of many lengths behind a shared beginning, heads of 64, small pages
        _case("append", 24, 301, True, 130, 12, 12, 64, 16, "fp16", "bshd") | {"name": "append B24 ragged D64"},
        # a short conversation, one token: latency
        _case("attend", 1, 1, False, 1000, 32, 8, 128, 64, "bf16") | {"name": "attend B1 one token"},
        # a decode step of a full batch
        _case("attend", 64, 1, False, 4095, 32, 8, 128, 64, "bf16") | {"name": "attend B64 one token"},
        # few long contexts, wide groups
        _case("attend", 3, 1, False, 60011, 64, 8, 128, 128, "bf16", lse=True) | {"name": "attend B3 long"},
        # heads of 64 without groups, small pages, token-major pages
        _case("attend", 40, 1, False, 1777, 12, 12, 64, 16, "fp16", "bshd") | {"name": "attend B40 one token D64"},
        # several proposed tokens are checked at once
        _case("attend", 24, 4, False, 3001, 32, 8, 128, 32, "bf16") | {"name": "attend B24 four tokens"},
        # prompts in chunks: 2048 new tokens behind 6144
        _case("attend", 2, 2048, False, 6144, 32, 8, 128, 64, "bf16", lse=True) | {"name": "attend B2 chunks"},
        # a prompt on itself, heads of 64
        _case("attend", 4, 1024, False, 0, 16, 16, 64, 64, "fp16") | {"name": "attend B4 prompts D64"},
        # prompts of many lengths, single tokens among them
        _case("attend", 16, 400, True, 1500, 28, 4, 128, 64, "bf16", "bshd") | {"name": "attend B16 ragged"},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    while True:
        op = rng.choice(("append", "attend"))
        Hq, Hkv = rng.choice(_HEADS)
        D, page = rng.choice((64, 128)), rng.choice((16, 32, 64, 128))
        kind = rng.choice(("one", "few", "prompt"))
        n = {"one": 1, "few": rng.randint(2, 8), "prompt": _log(rng, 9, 2048)}[kind]
        cached = rng.choice((0, _log(rng, 1, 60000), _log(rng, 1, 60000)))
        case = _case(op, _log(rng, 1, 128), n, n > 1 and rng.random() < 0.5, cached, Hq, Hkv, D, page, rng.choice(("bf16", "fp16")),
                     rng.choice(("bhsd", "bshd")), op == "attend" and rng.random() < 0.5)
        longest, tokens = max(_plan(case)[1]), sum(_plan(case)[0])
        # the padded scores, keys and values of the plain form, and the tokens of an append, stay within the largest listed cases
        if op == "attend" and case["B"] * Hq * n * longest <= 2 * 32 * 2048 * 8192 and case["B"] * longest * Hkv * D <= 64 * 4096 * 8 * 128 \
                and work(case)["flops"] <= 4.8e11:
            return case
        if op == "append" and tokens * (Hq + 2 * Hkv) * D <= 8192 * 48 * 128 and case["B"] * (longest + page) * Hkv * D <= 128 << 20:
            return case


def _plan(case):
    """New tokens and lengths (new tokens included) of the sequences."""
    spread = case["cached"] // 2 + 1
    new = [1 + (b * 7919 + 211) % case["n"] if case["ragged"] else case["n"] for b in range(case["B"])]
    return new, [m + case["cached"] - (b * 104729) % spread for b, m in enumerate(new)]


def work(case):
    new, lens = _plan(case)
    Hq, Hkv, D, tokens = case["Hq"], case["Hkv"], case["D"], sum(new)
    if case["op"] == "append":
        pages = sum((end - 1) // case["page"] - (end - m) // case["page"] + 1 for m, end in zip(new, lens))
        return {"bytes": tokens * D * (4 * Hq + 6 * Hkv + 4) + pages * (Hkv * 8 + 4), "flops": tokens * (Hq + Hkv) * D * 3}
    visible = sum(m * end - m * (m - 1) // 2 for m, end in zip(new, lens))
    pages = sum(-(-end // case["page"]) for end in lens)
    return {"bytes": 2 * sum(lens) * Hkv * D + 4 * tokens * Hq * D + pages * (Hkv * 8 + 4) + (4 * tokens * Hq if case["lse"] else 0),
            "flops": 4 * visible * Hq * D}


def prepare(case, seed):
    dev, dtype = torch.device("cuda"), _DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    new, lens = _plan(case)
    B, Hq, Hkv, D, page = case["B"], case["Hq"], case["Hkv"], case["D"], case["page"]
    tokens, columns = sum(new), -(-max(lens) // page) + 1
    count = B * columns + 3

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    def cache():  # codes whose largest is near the end of e4m3, as a scale by blocks leaves them
        shape = (count, Hkv, page, D) if case["layout"] == "bhsd" else (count, page, Hkv, D)
        codes = (normal(*shape) * 90.0).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
        return codes, torch.exp2(torch.randint(-8, -5, (count, Hkv), device=dev, generator=g).float())

    k_pages, k_scale = cache()
    v_pages, v_scale = cache()
    packed = normal(tokens, Hq + 2 * Hkv, D).to(dtype)  # one projection's output: q, k and v are views of it
    state = dict(case=case, q=packed[:, :Hq], k=packed[:, Hq:Hq + Hkv], v=packed[:, Hq + Hkv:], k_pages=k_pages, v_pages=v_pages,
                 k_scale=k_scale, v_scale=v_scale, max_tokens=max(new))
    state["page_table"] = torch.randperm(count, device=dev, generator=g)[:B * columns].reshape(B, columns).to(torch.int32)
    state["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    ends = torch.tensor([0] + new, dtype=torch.int32, device=dev).cumsum(0).to(torch.int32)
    state["starts"] = ends if case["ragged"] else None  # None: every sequence has as many
    if case["op"] == "append":
        angles = torch.arange(max(lens) + 1, dtype=torch.float64, device=dev)[:, None] \
            * 10000.0 ** (torch.arange(D // 2, dtype=torch.float64, device=dev) * (-2.0 / D))
        state["rope"] = (angles.cos().float(), angles.sin().float())
    return state


def run(state):
    case = state["case"]
    if own:
        from heddle_b200 import ops

        pages = ops.KvPages(state["k_pages"], state["v_pages"], state["k_scale"], state["v_scale"], case["layout"])
        if case["op"] == "append":
            q = ops.kv_append(state["k"], state["v"], pages, state["page_table"], state["seq_lens"], starts=state["starts"],
                              rope=state["rope"], q=state["q"])
            return [q, state["k_pages"], state["v_pages"], state["k_scale"], state["v_scale"]]
        return ops.fa_paged(state["q"], pages, state["page_table"], state["seq_lens"], starts=state["starts"],
                            max_tokens=state["max_tokens"], return_lse=case["lse"])
    return _plain_append(state) if case["op"] == "append" else _plain_attend(state)


# ------------------------------------------------------------------------------------------------------------------------
# the plain forms
# ------------------------------------------------------------------------------------------------------------------------
def _by_token(state):
    """Sequence, place in it and position in the cache of every new token."""
    lens, tokens = state["seq_lens"].long(), state["q"].shape[0]
    starts = state["starts"]
    starts = torch.arange(lens.numel() + 1, device=lens.device) * (tokens // lens.numel()) if starts is None else starts.long()
    t = torch.arange(tokens, device=lens.device)
    seq = (t[:, None] >= starts[None, 1:]).sum(1)
    place = t - starts[seq]
    return seq, place, lens[seq] - (starts[1:] - starts[:-1])[seq] + place


def _turned(x, cos, sin):
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _written(pages, scale, x, page, slot, begun, earlier, layout):
    """Codes of x [tokens, heads, D] into the pages, scales of the pages kept up.  Each sequence's first page ``begun`` holds
    ``earlier`` tokens already (0: the page starts here, and what it held does not count)."""
    by_slot = pages if layout == "bshd" else pages.transpose(1, 2)  # [pages, page_size, heads, D]
    mantissa, exponent = torch.frexp(x.abs().amax(-1))
    need = torch.ldexp(torch.ones_like(mantissa), (exponent - 9 + (mantissa > 0.875)).clamp(_MIN_EXP, _MAX_EXP))
    need = torch.where(mantissa == 0, torch.full_like(need, 2.0 ** _MIN_EXP), need)
    old = scale[begun]  # [sequences, heads]
    scale[page] = 0.0
    scale[begun] = torch.where((earlier > 0)[:, None], old, torch.zeros_like(old))
    scale.scatter_reduce_(0, page[:, None].expand_as(need), need, "amax")
    codes = by_slot[begun].float()  # [sequences, page_size, heads, D]
    held = torch.arange(by_slot.shape[1], device=x.device)[None, :] < earlier[:, None]
    again = torch.where(held[:, :, None, None], codes * (old / scale[begun])[:, None, :, None], codes)
    by_slot.view(torch.uint8)[begun] = again.to(torch.float8_e4m3fn).view(torch.uint8)
    by_slot.view(torch.uint8)[page, slot] = (x / scale[page][:, :, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_append(state):
    seq, place, position = _by_token(state)
    size, layout, table = state["case"]["page"], state["case"]["layout"], state["page_table"].long()
    page, slot = table[seq, position // size], position % size
    old = torch.zeros_like(state["seq_lens"], dtype=torch.long).scatter_reduce_(0, seq, position - place, "amax")  # tokens held before
    begun = table.gather(1, (old // size)[:, None])[:, 0]
    cos, sin = (t[position][:, None] for t in state["rope"])
    _written(state["k_pages"], state["k_scale"], _turned(state["k"], cos, sin), page, slot, begun, old % size, layout)
    _written(state["v_pages"], state["v_scale"], state["v"].float(), page, slot, begun, old % size, layout)
    return [_turned(state["q"], cos, sin).to(state["q"].dtype), state["k_pages"], state["v_pages"], state["k_scale"], state["v_scale"]]


def _plain_attend(state):
    case, q, table = state["case"], state["q"], state["page_table"].long()
    seq, place, position = _by_token(state)
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    B, n = case["B"], state["max_tokens"]

    def dense(pages, scale):  # [B, heads, keys, D]
        by_head = pages if case["layout"] == "bhsd" else pages.transpose(1, 2)
        return (by_head[table].float() * scale[table][..., None, None]).transpose(1, 2).flatten(2, 3)

    keys = torch.arange(table.shape[1] * case["page"], device=q.device)
    inside = keys[None, :] < state["seq_lens"][:, None]  # [B, keys]
    padded = torch.zeros(B, n, Hq, D, device=q.device)
    padded[seq, place] = q.float()
    last = torch.full((B, n), -1, device=q.device)
    last[seq, place] = position
    seen = ((keys <= last[..., None]) & inside[:, None])[:, None, :, None]  # [B, 1, n, 1, keys]
    rows = padded.reshape(B, n, Hkv, Hq // Hkv, D).transpose(1, 2).flatten(2, 3)  # [B, Hkv, n * group, D]
    s = (rows @ dense(state["k_pages"], state["k_scale"]).transpose(-1, -2)) / math.sqrt(D)
    s = s.reshape(B, Hkv, n, Hq // Hkv, -1).masked_fill_(~seen, -math.inf).flatten(2, 3)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    v = dense(state["v_pages"], state["v_scale"]).masked_fill_(~inside[:, None, :, None], 0.0)
    o = (p @ v) / torch.where(total > 0, total, torch.ones_like(total))
    lse = top + total.log()

    def packed(x):  # [B, Hkv, n * group, C] -> [tokens, Hq, C]
        return x.reshape(B, Hkv, n, Hq // Hkv, -1).transpose(1, 2)[seq, place].flatten(1, 2)

    o = packed(o).to(q.dtype)
    return (o, packed(lse)[..., 0].contiguous()) if case["lse"] else o


# ------------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ------------------------------------------------------------------------------------------------------------------------
def _e4m3(x):
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))).clamp_min(-6.0) - 3.0)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def exact(case, seed):
    state = prepare(case, seed)
    new, lens = _plan(case)
    Hq, Hkv, D, size = case["Hq"], case["Hkv"], case["D"], case["page"]
    heads_first = case["layout"] == "bhsd"
    table, at = state["page_table"].tolist(), 0
    if case["op"] == "append":
        i = torch.arange(D // 2, device="cuda")
        q = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda")
        k = torch.empty(state["k"].shape, dtype=torch.float64, device="cuda")
        caches = [[state[name + "_pages"].double(), state[name + "_scale"].double()] for name in "kv"]
        for b, (m, end) in enumerate(zip(new, lens)):
            cos, sin = (t.double()[end - m:end][:, None] for t in state["rope"])
            for x, y in ((state["q"], q), (state["k"], k)):
                x = x[at:at + m].double()
                y[at:at + m, :, :D // 2] = x[..., i] * cos - x[..., i + D // 2] * sin
                y[at:at + m, :, D // 2:] = x[..., i + D // 2] * cos + x[..., i] * sin
            for block in range((end - m) // size, (end - 1) // size + 1):
                low, high = max(end - m, block * size), min(end, (block + 1) * size)
                p, a, z = table[b][block], low - block * size, high - block * size
                for (codes, scales), x in zip(caches, (k, state["v"])):
                    x = x[at + low - (end - m):at + high - (end - m)].double()  # [tokens, heads, D]
                    cells = codes[p].transpose(0, 1) if heads_first else codes[p]  # [slots, heads, D]
                    s = torch.exp2(torch.ceil(torch.log2(x.abs().amax((0, 2)) / 448.0)).clamp(_MIN_EXP, _MAX_EXP))
                    if a > 0:
                        s = torch.maximum(s, scales[p])
                        cells[:a] = _e4m3(cells[:a] * (scales[p] / s)[:, None])
                    cells[a:z] = _e4m3(x / s[:, None])
                    scales[p] = s
            at += m
        return [q, caches[0][0], caches[1][0], caches[0][1], caches[1][1]]
    out = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(state["q"].shape[:2], dtype=torch.float64, device="cuda")
    for b, (m, end) in enumerate(zip(new, lens)):
        ids = state["page_table"][b, :-(-end // size)].long()
        k, v = (((state[name + "_pages"][ids] if heads_first else state[name + "_pages"][ids].transpose(1, 2)).double()
                 * state[name + "_scale"][ids].double()[..., None, None]).transpose(0, 1).reshape(Hkv, -1, D)[:, :end] for name in "kv")
        hidden = torch.arange(end, device="cuda")[None, :] > torch.arange(end - m, end, device="cuda")[:, None]
        for h in range(Hq):
            kv = h // (Hq // Hkv)
            s = (state["q"][at:at + m, h].double() @ k[kv].T) * D ** -0.5
            s[hidden] = -math.inf
            lse[at:at + m, h] = torch.logsumexp(s, -1)
            out[at:at + m, h] = torch.softmax(s, -1) @ v[kv]
        at += m
    return (out, lse) if case["lse"] else out
