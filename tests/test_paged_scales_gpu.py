"""The paged attention over pages whose scales are far apart, and rows that see few of them, against the formulas in 64 bits."""
import math

import pytest
import torch

from test_paged_gpu import DT, _cache, _clean, _gen, _ints

pytestmark = pytest.mark.gpu

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
            # a score: D products and sums in fp32, and x f - m in fp32 (base 2)
            err = torch.where(seen, (x.abs() @ kd.abs().T) * (D ** -0.5 * D * 2.0 ** -23) + (s.abs() + top.abs()) * 2.0 ** -22, 0.0)
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
