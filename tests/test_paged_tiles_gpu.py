"""Paged attention of prompts where its tiles kernel takes them: enough (sequence, KV head) pairs, or keys, for the limit of rows to be low.
The same edges as in test_paged_gpu.py."""
import math

import pytest
import torch

from oracle import paged_oracle as P
from test_paged_gpu import DT, _cache, _clean, _close, _gen, _ints

pytestmark = pytest.mark.gpu

CASES = [  # new, lens, page size, Hkv, group, D, dtype, layout, ragged call, causal
    # one block an item
    ([70] * 10, [70 + 31 * b for b in range(10)], 16, 16, 1, 128, "bf16", "bhsd", False, True),
    ([33] * 10, [128 + b for b in range(10)], 32, 16, 3, 64, "fp16", "bshd", False, True),
    ([90] * 10, [200 + 9 * b for b in range(10)], 128, 16, 1, 64, "bf16", "bhsd", False, False),
    ([20, 100, 0, 1, 65, 64, 90, 3, 80, 70], [20, 600, 9, 300, 65, 500, 128, 200, 1000, 71], 64, 16, 4, 128, "fp16", "bhsd", True, True),
    # keys of an item over several blocks: parts that no row of a tile of rows sees, items with fewer tiles than parts
    ([64] * 4, [2000, 1500, 64, 777], 64, 8, 4, 128, "bf16", "bshd", False, True),
    ([256] * 2, [1500, 256], 32, 4, 4, 64, "fp16", "bhsd", False, True),
    ([300, 1, 200], [1700, 900, 200], 16, 8, 4, 128, "bf16", "bhsd", True, True),
    ([130] * 3, [2000, 131, 900], 128, 8, 2, 64, "bf16", "bhsd", False, False),
]


@pytest.mark.parametrize("new,lens,size,Hkv,group,D,dtype,layout,ragged,causal", CASES)
def test_attend(built_lib, new, lens, size, Hkv, group, D, dtype, layout, ragged, causal):
    from heddle_b200 import ops
    g = _gen(71)
    pages, table = _cache(len(new), lens, size, Hkv, D, layout, g)
    live = sum(new)
    T = live + (2 if ragged else 0)
    q = (torch.randn(T, Hkv * group + 1, D, device="cuda", generator=g) * 2).to(DT[dtype])[:, 1:]
    starts = torch.tensor([0] + new).cumsum(0).int().cuda() if ragged else None
    out = torch.full((T, Hkv * group, D), 7.0, dtype=DT[dtype], device="cuda")
    got, lse = ops.fa_paged(q, pages, table, _ints(lens), starts=starts, max_tokens=max(new), causal=causal, return_lse=True, out=out)
    _clean()
    assert (out[live:] == 7.0).all()
    ref = P.attend(q[:live], P.Cache(pages), table.cpu(), lens, None if starts is None else starts.tolist(), causal)
    _close(got[:live], lse[:live], ref, dtype)


WIDE = (10, 16)  # sequences, KV heads: one block an item
LONG = (4, 8)    # several


@pytest.mark.parametrize("B,Hkv,scale", ((*WIDE, 1), (*LONG, 4)))
def test_stale_places_do_not_matter(built_lib, B, Hkv, scale):
    from heddle_b200 import ops
    g = _gen(73)
    new, lens, size = 70, [scale * (37 + 61 * b) + 70 for b in range(B)], 32
    pages, table = _cache(B, lens, size, Hkv, 128, "bhsd", g)
    q = torch.randn(B * new, Hkv * scale, 128, device="cuda", generator=g).bfloat16()
    first = ops.fa_paged(q, pages, table, _ints(lens), return_lse=True)
    for which in (pages.k, pages.v):
        codes = which.view(torch.uint8)
        used = torch.zeros(codes.shape[:3], dtype=torch.bool, device="cuda")
        for b, n in enumerate(lens):
            for block in range(-(-n // size)):
                used[int(table[b, block]), :, :min(size, n - block * size)] = True
        codes[~used] = 0x7F
    for b, n in enumerate(lens):
        for block in range(-(-n // size), table.shape[1]):
            pages.k_scale[int(table[b, block])] = math.nan
            table[b, block] = -7
    again = ops.fa_paged(q, pages, table, _ints(lens), return_lse=True)
    _clean()
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("B,Hkv,group,length", ((*WIDE, 1, 400), (*LONG, 4, 1500)))
def test_pages_that_are_not_there(built_lib, B, Hkv, group, length):
    from heddle_b200 import ops
    g = _gen(79)
    new, size, lens = 70, 16, [length - 13 * b for b in range(B)]
    pages, table = _cache(B, lens, size, Hkv, 128, "bhsd", g)
    for block in (1, 12, *range(16, 24)):
        table[0, block] = -1 if block % 2 else pages.k.shape[0] + block
    table[1, (lens[1] - 1) // size] = -1
    pages.k_scale[int(table[2, 5])] = 0
    q = torch.randn(B * new, Hkv * group, 128, device="cuda", generator=g).bfloat16()
    out, lse = ops.fa_paged(q, pages, table, _ints(lens), return_lse=True)
    assert ops.cache_status() == 1 and ops.status_word() == 0
    table[2, 5] = -1
    _close(out, lse, P.attend(q, P.Cache(pages), table.cpu(), lens), "bf16")


@pytest.mark.parametrize("B,Hkv,group,length", ((*WIDE, 1, 300), (*LONG, 4, 1500)))
def test_scales_and_rows_without_keys(built_lib, B, Hkv, group, length):
    """Value scales over 2^40, scores of hundreds, sequences that are empty or shorter than their rows."""
    from heddle_b200 import ops
    g = _gen(83)
    new, lens = 70, [length - 11 * b for b in range(B)]
    lens[1], lens[2] = 0, 30
    pages, table = _cache(B, lens, 16, Hkv, 128, "bhsd", g)
    pages.v_scale.copy_(torch.exp2(torch.randint(-30, 10, pages.v_scale.shape, device="cuda", generator=g).float()))
    pages.k_scale.copy_(torch.exp2(torch.randint(-12, -3, pages.k_scale.shape, device="cuda", generator=g).float()))
    q = (torch.randn(B * new, Hkv * group, 128, device="cuda", generator=g) * 4).half()
    q[0, 0] = 0
    out, lse = ops.fa_paged(q, pages, table, _ints(lens), return_lse=True)
    assert ops.cache_status() == 2 and ops.status_word() == 0
    assert (out[new:2 * new] == 0).all() and (lse[new:2 * new] == -math.inf).all() and (lse[2 * new:2 * new + 40] == -math.inf).all()
    _close(out, lse, P.attend(q, P.Cache(pages), table.cpu(), lens), "fp16")


@pytest.mark.parametrize("B,Hkv,group,length", ((*WIDE, 1, 300), (*LONG, 4, 1500)))
def test_what_is_not_finite_stays_alone(built_lib, B, Hkv, group, length):
    """A query with a NaN or infinity, and a token that kv_append stored as one: only the rows that see them are NaN."""
    from heddle_b200 import ops
    g = _gen(89)
    new, lens, Hq = 70, [length] * B, Hkv * group
    pages, table = _cache(B, lens, 32, Hkv, 64, "bhsd", g)
    q = torch.randn(B * new, Hq, 64, device="cuda", generator=g).bfloat16()
    ref = ops.fa_paged(q, pages, table, _ints(lens))
    q[5, 1, 3], q[new + 7, Hq - 1, 60] = math.nan, -math.inf
    before = ops.fa_paged(q, pages, table, _ints(lens))
    codes, place = pages.k.view(torch.uint8), length - 40  # as kv_append stores such a token
    codes[int(table[2, place // 32]), 3, place % 32] = 0x7F
    after = ops.fa_paged(q, pages, table, _ints(lens))
    _clean()
    sick = torch.zeros(B * new, Hq, dtype=torch.bool, device="cuda")
    sick[5, 1] = sick[new + 7, Hq - 1] = True
    assert torch.isnan(before[sick]).all() and torch.equal(before[~sick], ref[~sick])
    sees = torch.zeros_like(sick)
    sees[2 * new + new - 40:3 * new, 3 * group:4 * group] = True
    assert torch.isnan(after[sick | sees]).all() and torch.equal(after[~(sick | sees)], ref[~(sick | sees)])
