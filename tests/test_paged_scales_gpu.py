"""The paged attention over pages whose scales are far apart, and rows that see few of them, against the formulas in 64 bits."""
import math

import pytest
import torch

from test_paged_gpu import DT, _cache, _clean, _gen, _ints

pytestmark = pytest.mark.gpu

FEW = dict(B=5, Hkv=2, group=2)    # the rows kernel, whatever the number of tokens up to 64
WIDE = dict(B=10, Hkv=16, group=1)  # the tiles kernel, one block an item
LONG = dict(B=4, Hkv=8, group=4)    # the tiles kernel, keys of an item over several blocks (of long tables)


def _reference(q, pages, table, lens, new, causal, floor):
    """(O, LSE, tolerances of both) in fp64.  ``floor``: P is kept as a multiple of 2^-24 of what O is held in, so that every key's weight may be
    off by 2^-25 of that; O is held in 2^-8 of a unit which is at most 2^9 times the largest product of a visible key's weight and its
    value scale: 2^-24 of that product, for all keys together sum |code| 2^-24 (floor 24).  Where all scales are alike the unit is the scale: 2^-33."""
    T, Hq, D = q.shape
    by_head = [(t if pages.layout == "bhsd" else t.transpose(1, 2)) for t in (pages.k, pages.v)]
    size, Hkv = by_head[0].shape[2], by_head[0].shape[1]
    group, eps = Hq // Hkv, torch.finfo(q.dtype).eps / 2
    out, tol = (torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device) for _ in range(2))
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64, device=q.device)
    lse_tol = torch.zeros_like(lse)
    row = 0
    for b, (n, length) in enumerate(zip(new, lens)):
        ids = table[b, :-(-length // size)].long()
        there = ((ids >= 0) & (ids < pages.k.shape[0])).repeat_interleave(size)[:length]
        ids = torch.where((ids >= 0) & (ids < pages.k.shape[0]), ids, 0)
        k, v = (by_head[w][ids].to(torch.float32).double().transpose(0, 1).reshape(Hkv, -1, D)[:, :length] for w in (0, 1))
        ks, vs = (s[ids].double().T.repeat_interleave(size, 1)[:, :length] for s in (pages.k_scale, pages.v_scale))
        pos = torch.arange(length - n, length, device=q.device)
        visible = there[None] & ((torch.arange(length, device=q.device)[None] <= pos[:, None]) | (not causal))  # [n, length]
        for h in range(Hkv):
            x = q[row:row + n, h * group:(h + 1) * group].double()
            kd, vd = k[h] * ks[h][:, None], v[h] * vs[h][:, None]
            seen = visible[:, None]
            s = torch.where(seen, x @ kd.T * D ** -0.5, -math.inf)  # [n, group, length]
            top = s.amax(-1, keepdim=True)
            some = top > -math.inf
            top = torch.where(some, top, 0.0)
            p = torch.exp(s - top)
            total = torch.where(some, p.sum(-1, keepdim=True), 1.0)
            o = p @ vd / total
            # a score: D products and sums in fp32.  The exponent of a weight, x f + (8 - m + w) in base 2, where w is log2 of the value scale relative to
            # another one and m a score plus such a logarithm: three roundings of fp32, each off by 2^-24 of a number of at most
            # 1.45 (|s| + |top|) + span + 8, which moves the weight by ln 2 of that.  3 ln 2 2^-24 (1.45 (|s| + |top|) + span + 8) is less
            # than (|s| + |top| + span) 2^-22 and the 2^-19 below
            present = vs[h][there & (vs[h] > 0)].log2()
            span = (present.max() - present.min()).item() if present.numel() else 0.0
            err = torch.where(seen, (x.abs() @ kd.abs().T) * (D ** -0.5 * D * 2.0 ** -23) + (s.abs() + top.abs() + span) * 2.0 ** -22, 0.0)
            at, heads = slice(row, row + n), slice(h * group, (h + 1) * group)
            out[at, heads] = o
            moved = ((p * err) @ vd.abs() + (p * err).sum(-1, keepdim=True) * o.abs()) / total
            lost = (seen.double() @ v[h].abs()) * (p * vs[h]).amax(-1, keepdim=True) * 2.0 ** -floor / total
            # P to fp16 is off by half a step (2^-11), exponentials and sums by 2^-19
            tol[at, heads] = o.abs() * eps * 1.01 + (2.0 ** -11 + 2.0 ** -19) * (p @ vd.abs()) / total + 1.1 * moved + lost
            lse[at, heads] = torch.where(some, top + torch.log(total), -math.inf)[..., 0]
            lse_tol[at, heads] = 1.1 * ((p * err).sum(-1) / total[..., 0]) + 2.0 ** -19 + lse[at, heads].abs().nan_to_num(posinf=0.0) * 2.0 ** -22
        row += n
    return out, lse, tol + torch.finfo(q.dtype).smallest_normal * eps, lse_tol


def _check(got, got_lse, ref):
    out, lse, tol, lse_tol = ref
    assert not torch.isnan(got).any() and not torch.isnan(got_lse).any()
    bad = (got.double() - out).abs() > tol
    assert not bad.any(), (int(bad.sum()), got[bad][:6], out[bad][:6], tol[bad][:6])
    empty = lse == -math.inf
    assert torch.equal(got_lse == -math.inf, empty)
    assert ((got_lse.double() - lse).abs() <= lse_tol)[~empty].all()


def _blocks(pages, table, which, exponents):
    """Scales of the sequences' blocks: 2^exponents(block, blocks)."""
    scale = (pages.k_scale, pages.v_scale)[which]
    for block in range(table.shape[1]):
        scale[table[:, block].long()] = 2.0 ** exponents(block, table.shape[1])


def _setting(kind, spread, pages, table, q, g):
    """Scales, keys and queries in which a page far above the others must not decide the result."""
    later = lambda block, blocks: -6 if block >= (blocks + 1) // 2 else -6 - spread  # noqa: E731
    if kind == "values behind the causal limit":
        _blocks(pages, table, 1, later)
    elif kind == "keys behind the causal limit":
        _blocks(pages, table, 0, later)
        q.mul_(2.0 ** min(spread, 12))  # fp16 holds that; scores of some size where the small keys alone are seen
    elif kind == "keys that a query has no part in":  # every third page, in the upper half of head_dim, where the queries are 0
        D = q.shape[2]
        _blocks(pages, table, 0, lambda block, blocks: -6 + spread if block % 3 == 1 else -6)
        for block in range(1, table.shape[1], 3):
            pages.k.view(torch.uint8)[table[:, block].long()[:, None, None], :, :, :D // 2] = 0
        q[..., D // 2:] = 0
    elif kind == "values seen with a low score":
        _blocks(pages, table, 0, lambda block, blocks: -6)
        _blocks(pages, table, 1, lambda block, blocks: -6 + spread if block % 4 == 2 else -6)
        one = torch.tensor([1.0, -448.0], device="cuda").to(torch.float8_e4m3fn).view(torch.uint8)
        pages.k.view(torch.uint8)[..., 0] = one[0]
        for block in range(2, table.shape[1], 4):  # weights of about 2^-spread
            pages.k.view(torch.uint8)[table[:, block].long(), ..., 0] = one[1]
        q[..., 0] = spread * math.log(2) * q.shape[2] ** 0.5 * 64 / 448
    else:  # steps that add up, and any
        if kind == "values in steps":
            _blocks(pages, table, 1, lambda block, blocks: -40 + (block * spread) // blocks)
        else:
            pages.v_scale.copy_(torch.exp2(torch.randint(-spread, 1, pages.v_scale.shape, device="cuda", generator=g).float()))
            pages.k_scale.copy_(torch.exp2(torch.randint(-spread // 2 - 3, -3, pages.k_scale.shape, device="cuda", generator=g).float()))


KINDS = ("values behind the causal limit", "keys behind the causal limit", "keys that a query has no part in", "values seen with a low score",
         "values in steps", "any")
CALLS = [  # form, new, length, page size, D, dtype, layout
    (FEW, 4, 18, 16, 128, "bf16", "bhsd"),
    (FEW, 3, 200, 16, 64, "fp16", "bshd"),
    (FEW, 1, 1000, 32, 128, "fp16", "bhsd"),
    (FEW, 60, 130, 16, 64, "bf16", "bhsd"),
    (WIDE, 128, 128, 16, 128, "bf16", "bhsd"),
    (WIDE, 100, 300, 32, 64, "fp16", "bshd"),
    (LONG, 70, 1500, 64, 128, "bf16", "bhsd"),
    (LONG, 64, 1100, 16, 64, "fp16", "bhsd"),
]


@pytest.mark.parametrize("spread", (9, 16, 25, 40))
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form,new,length,size,D,dtype,layout", CALLS)
def test_scales_far_apart(built_lib, form, new, length, size, D, dtype, layout, kind, spread):
    from heddle_b200 import ops
    g = _gen(191)
    B, Hkv, group = form["B"], form["Hkv"], form["group"]
    lens = [length - b for b in range(B)]
    lens = [max(n, new) for n in lens]
    pages, table = _cache(B, lens, size, Hkv, D, layout, g)
    q = (torch.randn(B * new, Hkv * group, D, device="cuda", generator=g)).to(DT[dtype])
    heads_first = pages if layout == "bhsd" else pages._replace(k=pages.k.transpose(1, 2), v=pages.v.transpose(1, 2))
    _setting(kind, spread, heads_first, table, q, g)
    out, lse = ops.fa_paged(q, pages, table, _ints(lens), return_lse=True)
    _clean()
    _check(out, lse, _reference(q, pages, table, lens, [new] * B, True, 24))


@pytest.mark.parametrize("form,new,length,size,D", ((FEW, 4, 100, 16, 128), (FEW, 2, 300, 32, 64), (WIDE, 100, 300, 16, 128), (LONG, 70, 1100, 32, 64)))
def test_scales_far_apart_among_pages_that_are_not_there(built_lib, form, new, length, size, D):
    """The same with pages of nobody's, value scales of 0, and sequences without keys; then with a NaN key and a NaN query."""
    from heddle_b200 import ops
    g = _gen(193)
    B, Hkv, group = form["B"], form["Hkv"], form["group"]
    lens = [length - 3 * b for b in range(B)]
    lens[1] = 0
    pages, table = _cache(B, lens, size, Hkv, D, "bhsd", g)
    q = torch.randn(B * new, Hkv * group, D, device="cuda", generator=g).bfloat16()
    _setting("any", 40, pages, table, q, g)
    for block in (1, 2, 5):
        table[0, block] = -1
        pages.v_scale[table[2, block].long()] = 0
    for block in range(128 // size, min(256 // size, table.shape[1] - 1)):  # all of a tile of 128 keys
        pages.v_scale[table[3, block].long()] = 0
    out, lse = ops.fa_paged(q, pages, table, _ints(lens), causal=False, return_lse=True)
    assert ops.cache_status() == 3 and ops.status_word() == 0  # a page outside of the cache, a sequence shorter than its rows
    live = torch.ones(B * new, dtype=torch.bool, device="cuda")
    live[new:2 * new] = False
    keep = [b for b in range(B) if b != 1]
    ref = _reference(q[live], pages, table[keep], [lens[b] for b in keep], [new] * (B - 1), False, 24)
    _check(out[live], lse[live], ref)
    assert (out[~live] == 0).all() and (lse[~live] == -math.inf).all()
    pages.k.view(torch.uint8)[table[2, 3].long(), Hkv - 1, size - 1] = 0x7F  # as kv_append stores a token with a NaN
    q[0, 0, 5] = math.nan
    sick = torch.zeros(B * new, Hkv * group, dtype=torch.bool, device="cuda")
    sick[0, 0] = True
    sick[2 * new:3 * new, (Hkv - 1) * group:] = True
    again, again_lse = ops.fa_paged(q, pages, table, _ints(lens), causal=False, return_lse=True)
    assert ops.cache_status() == 3 and ops.status_word() == 0
    assert torch.isnan(again[sick]).all() and torch.isnan(again_lse[sick]).all()
    assert torch.equal(again[~sick], out[~sick]) and torch.equal(again_lse[~sick], lse[~sick])


@pytest.mark.parametrize("D,dtype", ((64, "bf16"), (64, "fp16"), (128, "bf16"), (128, "fp16")))
def test_many_small_weights_beside_a_large_one(built_lib, D, dtype):
    """A key with nearly all of the weight and a value of zero; 20000 others with 2^-24.5 of it each make the result.  As many sequences and
    heads as there are blocks, all of the same pages, so that the large weight has its share of them in its own part."""
    from heddle_b200 import ops
    g = _gen(197)
    B, n, size, Hkv, group = 60, 20000, 128, 8, 4
    pages, table = _cache(1, [n], size, Hkv, D, "bhsd", g)
    pages.k.zero_()
    pages.k_scale.fill_(2.0 ** -6)
    pages.v_scale.fill_(2.0 ** -6)
    pages.v.copy_((torch.rand(pages.v.shape, device="cuda", generator=g) * 300 + 100).to(torch.float8_e4m3fn))
    first = int(table[0, 7])
    pages.k[first, :, 11, 0] = 256.0
    pages.v.view(torch.uint8)[first, :, 11] = 0
    q = torch.zeros(1, Hkv, group, D, device="cuda", dtype=DT[dtype])
    q[..., 0] = torch.tensor([24.5, 23.6, 24.9, 20.3], device="cuda") * math.log(2) * D ** 0.5 / 4
    q = q.flatten(1, 2)
    out, lse = ops.fa_paged(q.expand(B, -1, -1).contiguous(), pages, table.expand(B, -1).contiguous(), _ints([n] * B), return_lse=True)
    _clean()
    ref = _reference(q, pages, table, [n], [1], True, 33)
    for b in range(B):
        _check(out[b:b + 1], lse[b:b + 1], ref)


@pytest.mark.parametrize("form,new", ((FEW, 1), (FEW, 40), (WIDE, 128), (LONG, 70)))
def test_queries_that_are_not_finite_and_see_nothing(built_lib, form, new):
    """A row without a visible key is 0 whatever its query holds: a sequence without tokens, rows in front of the first one."""
    from heddle_b200 import ops
    g = _gen(199)
    B, Hkv, group = form["B"], form["Hkv"], form["group"]
    lens = [1000 - 11 * b for b in range(B)]
    lens[0], lens[2] = 0, new // 2
    pages, table = _cache(B, lens, 32, Hkv, 64, "bhsd", g)
    q = torch.randn(B * new, Hkv * group, 64, device="cuda", generator=g).bfloat16()
    blind = torch.zeros(B * new, dtype=torch.bool, device="cuda")
    blind[:new] = blind[2 * new:3 * new - new // 2] = True
    want, want_lse = ops.fa_paged(q, pages, table, _ints(lens), return_lse=True)
    q[blind, :, 3], q[blind, 0, 5] = math.nan, math.inf
    out, lse = ops.fa_paged(q, pages, table, _ints(lens), return_lse=True)
    assert ops.cache_status() == 2 and ops.status_word() == 0
    assert (out[blind] == 0).all() and (lse[blind] == -math.inf).all()
    assert torch.equal(out[~blind], want[~blind]) and torch.equal(lse[~blind], want_lse[~blind])


@pytest.mark.parametrize("form,new,length,size,D,dtype,layout", CALLS)
@pytest.mark.parametrize("where", ("first", "last", "between"))
def test_pages_of_zeros(built_lib, form, new, length, size, D, dtype, layout, where):
    """Values of zero, as kv_append stores them, with the smallest scale there is, beside ordinary ones with scales of 2^-6 and 1."""
    from heddle_b200 import ops
    g = _gen(241)
    B, Hkv, group = form["B"], form["Hkv"], form["group"]
    lens = [max(length - b, new) for b in range(B)]
    pages, table = _cache(B, lens, size, Hkv, D, layout, g)
    columns = table.shape[1]
    blocks = {"first": range((columns + 1) // 2), "last": range(columns // 2, columns), "between": range(columns // 3, columns, 3)}[where]
    _blocks(pages, table, 1, lambda block, _: -100 if block in blocks else -6 if block % 2 else 0)
    for block in blocks:
        pages.v.view(torch.uint8)[table[:, block].long()] = 0
    q = torch.randn(B * new, Hkv * group, D, device="cuda", generator=g).to(DT[dtype])
    out, lse = ops.fa_paged(q, pages, table, _ints(lens), return_lse=True)
    _clean()
    _check(out, lse, _reference(q, pages, table, lens, [new] * B, True, 24))
