"""What the paged cache's kernels do with tables, lengths and starts that are wrong: what they write, what they leave, what they report."""
import pytest
import torch

from oracle import paged_oracle as P
from test_paged_gpu import _cache, _gen, _ints, _rope

pytestmark = pytest.mark.gpu


def _same(a, b):
    return all(torch.equal(torch.nan_to_num(x, nan=1e9), torch.nan_to_num(y, nan=1e9)) for x, y in zip(a.codes + a.scales, b.codes + b.scales))


DESCENDING = [  # starts, rows, tokens of each sequence, page size, Hkv
    ([0, 100, 0, 100], 100, 200, 16, 2),
    ([0, 3, 1, 4], 4, 50, 16, 1),
    ([0, 300, 299, 600], 600, 700, 64, 4),
    ([5, 4] + [6] * 299, 6, 40, 32, 2),   # more sequences than a block of the rows kernel has threads, the first one wrong
    ([0] * 299 + [70, 69], 70, 90, 32, 2),  # the last one
]


@pytest.mark.parametrize("starts,T,length,size,Hkv", DESCENDING)
def test_starts_that_descend(built_lib, starts, T, length, size, Hkv):
    """Nothing is written, neither to the cache nor to the outputs, and it is reported, by append too."""
    from heddle_b200 import ops
    g = _gen(211)
    B, D = len(starts) - 1, 64
    lens = [length] * B
    pages, table = _cache(B, lens, size, Hkv, D, "bhsd", g)
    before = P.Cache(pages)
    k, v, q = (torch.randn(T, H, D, device="cuda", generator=g).bfloat16() for H in (Hkv, Hkv, 2 * Hkv))
    ops.kv_append(k, v, pages, table, _ints(lens), starts=_ints(starts), rope=_rope(length, D), q=q)
    assert ops.cache_status() == 4
    assert _same(before, P.Cache(pages))
    for hint in (None, T, 1):
        out = torch.full_like(q, 7.0)
        ops.fa_paged(q, pages, table, _ints(lens), starts=_ints(starts), max_tokens=hint, out=out)
        assert ops.cache_status() == 4 and ops.status_word() == 0
        assert (out == 7.0).all()


@pytest.mark.parametrize("n,Hkv", ((2, 1), (150, 8)))
def test_starts_that_leave_the_rows(built_lib, n, Hkv):
    """They are taken as the nearest that do not: the first and last row."""
    from heddle_b200 import ops
    g = _gen(223)
    D, size, lens = 64, 16, [n + 40, n + 30, n + 33]
    pages, table = _cache(3, lens, size, Hkv, D, "bhsd", g)
    copy = pages._replace(**{name: getattr(pages, name).clone() for name in ("k", "v", "k_scale", "v_scale")})
    k, v, q = (torch.randn(3 * n, H, D, device="cuda", generator=g).bfloat16() for H in (Hkv, Hkv, 2 * Hkv))
    results = []
    for where, starts, status in ((pages, [0, n, 2 * n, 3 * n], 0), (copy, [-5, n, 2 * n, 1 << 30], 4)):
        turned = ops.kv_append(k, v, where, table, _ints(lens), starts=_ints(starts), q=q)
        assert ops.cache_status() == status
        results.append((turned, ops.fa_paged(turned, where, table, _ints(lens), starts=_ints(starts))))
        assert ops.cache_status() == status
    assert _same(P.Cache(pages), P.Cache(copy))
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])


OVERLONG = [  # new tokens, tokens that the lengths give the sequences, columns of the table, page size
    ([1, 1, 1], [49, 48, 200], 3, 16),
    ([5, 5], [66, 64], 2, 32),
    ([100, 30, 1], [150, 130, (1 << 31) - 1], 1, 128),
]


@pytest.mark.parametrize("rotate", (True, False))
@pytest.mark.parametrize("new,lens,columns,size", OVERLONG)
def test_append_behind_the_page_table(built_lib, new, lens, columns, size, rotate):
    """Tokens behind the last page of the table are left out; those in front of them keep their places and angles."""
    from heddle_b200 import ops
    g = _gen(227)
    B, Hkv, D = len(new), 2, 64
    pages, table = _cache(B, [columns * size] * B, size, Hkv, D, "bhsd", g)
    table = table[:, :columns].contiguous()
    k, v, q = (torch.randn(sum(new), H, D, device="cuda", generator=g).bfloat16() for H in (Hkv, Hkv, 4))
    starts, rope = torch.tensor([0] + new).cumsum(0).int().cuda(), _rope(250, D) if rotate else None
    want = P.Cache(pages)
    want.append(k, v, table.cpu(), lens, starts.tolist(), rope)
    turned = ops.kv_append(k, v, pages, table, _ints(lens), starts=starts, rope=rope, q=q)
    assert ops.cache_status() == (10 if rotate and max(lens) > 250 else 2)
    assert _same(want, P.Cache(pages))
    # the queries: as with a table that is long enough
    wide = torch.cat([table, torch.full((B, 8), -1, dtype=torch.int32, device="cuda")], 1).contiguous()
    again = ops.kv_append(k, v, pages, wide, _ints([min(n, 250) for n in lens]), starts=starts, rope=rope, q=q)
    ops.cache_status()
    for b in (b for b, n in enumerate(lens) if n <= 250):
        assert torch.equal(turned[starts[b]:starts[b + 1]], again[starts[b]:starts[b + 1]])


def test_reports_are_not_lost_while_others_are_read(built_lib):
    """One thread has two faults found, one after the other, again and again; another one reads all the time, and gets each."""
    import threading
    import time

    from heddle_b200 import ops
    pages, table = _cache(1, [16], 16, 1, 64, "bhsd", _gen(229))
    nowhere, q = torch.full_like(table, -1), torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda")
    fine, longer = _ints([16]), _ints([17 * table.shape[1]])
    torch.cuda.synchronize()
    reads, stop, failed = [], threading.Event(), []

    def reader():
        try:
            while not stop.is_set():
                reads.append(ops.cache_status())
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    thread = threading.Thread(target=reader)
    thread.start()
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            for n in range(1500):
                before = len(reads)
                ops.fa_paged(q, pages, nowhere, fine)   # a page outside of the cache
                for _ in range(n % 7):
                    time.sleep(0)
                ops.fa_paged(q, pages, table, longer)   # a length behind the table
                torch.cuda.current_stream().synchronize()
                got, until = 0, time.monotonic() + 2
                while got != 3 and time.monotonic() < until and not failed:
                    got = 0
                    for bits in reads[max(before - 1, 0):]:  # the last one may have begun before
                        got |= bits
                assert got == 3, (n, got)
                while len(reads) < before + 4 and time.monotonic() < until and not failed:  # nothing is left for the next pass
                    pass
    finally:
        stop.set()
        thread.join()
    assert not failed and set(reads) <= {0, 1, 2, 3}


@pytest.mark.parametrize("B,new,length,size,Hkv,group,D", ((3, 1, 300, 16, 2, 4, 128), (3, 7, 200, 64, 2, 4, 64), (10, 70, 300, 16, 16, 1, 128), (4, 64, 1500, 64, 8, 4, 64)))
@pytest.mark.parametrize("value_scale", (float("nan"), float("inf"), 2.0 ** 100, 0.0))
def test_a_page_whose_key_scale_is_zero_is_not_there(built_lib, B, new, length, size, Hkv, group, D, value_scale):
    """A page that nothing was written to yet: not seen, whatever its value scale is, and not reported."""
    from heddle_b200 import ops
    g = _gen(233)
    lens = [length - 5 * b for b in range(B)]
    pages, table = _cache(B, lens, size, Hkv, D, "bhsd", g)
    q = torch.randn(B * new, Hkv * group, D, device="cuda", generator=g).bfloat16()
    gone = [(0, 0), (0, 2), (1, 1), (1, (lens[1] - 1) // size), *((2, block) for block in range(128 // size))]
    for b, block in gone:
        pages.k_scale[int(table[b, block])] = 0
        pages.v_scale[int(table[b, block])] = value_scale
    out, lse = ops.fa_paged(q, pages, table, _ints(lens), return_lse=True)
    assert ops.cache_status() == 0 and ops.status_word() == 0
    for b, block in gone:
        table[b, block] = -1
    want, want_lse = ops.fa_paged(q, pages, table, _ints(lens), return_lse=True)
    assert ops.cache_status() == 1 and ops.status_word() == 0
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
