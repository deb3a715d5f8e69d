"""The paged 8-bit key/value cache on the GPU against the oracle in 64 bits: append, attention, and the two as a server runs them."""
import math

import pytest
import torch

from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _cache(B, lens, size, Hkv, D, layout, g, spare=2, filled=True):
    """Pages with random contents, a table of them in random order."""
    from heddle_b200 import ops
    columns = max(1, -(-max(max(lens), 1) // size))
    count = B * columns + spare
    pages = ops.kv_pages(count, size, Hkv, D, layout=layout)
    if filled:
        for codes, scale in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)):
            codes.copy_((torch.randn(codes.shape, device="cuda", generator=g) * 80).clamp(-448, 448).to(torch.float8_e4m3fn))
            scale.copy_(torch.exp2(torch.randint(-9, -4, scale.shape, device="cuda", generator=g).float()))
    table = torch.randperm(count, device="cuda", generator=g)[:B * columns].reshape(B, columns).to(torch.int32)
    return pages, table


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _rope(n, D):
    angle = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (torch.arange(D // 2, dtype=torch.float64) * (-2.0 / D))
    return angle.cos().float().cuda(), angle.sin().float().cuda()


def _clean():
    from heddle_b200 import ops
    torch.cuda.synchronize()
    assert ops.cache_status() == 0 and ops.status_word() == 0


# --------------------------------------------------------------------------------------------------------------------------
# append
# --------------------------------------------------------------------------------------------------------------------------
APPENDS = [  # new tokens of each sequence, tokens before, page size, Hkv, Hq, D, dtype, layout, ragged call
    ([1], [0], 16, 1, 1, 64, "bf16", "bhsd", False),
    ([1] * 5, [0, 15, 16, 17, 63], 16, 3, 6, 128, "bf16", "bhsd", False),
    ([1] * 3, [31, 64, 100], 32, 2, 2, 64, "fp16", "bshd", False),
    ([7] * 3, [0, 60, 125], 64, 2, 4, 128, "fp16", "bhsd", False),
    ([3, 0, 130, 1, 17], [5, 9, 0, 31, 127], 16, 2, 14, 128, "bf16", "bshd", True),
    ([200, 129], [100, 0], 128, 1, 2, 64, "bf16", "bhsd", True),
    ([33, 64, 1], [31, 0, 0], 64, 4, 4, 128, "bf16", "bhsd", True),
]


@pytest.mark.parametrize("new,before,size,Hkv,Hq,D,dtype,layout,ragged", APPENDS)
@pytest.mark.parametrize("rotate", (True, False))
def test_append(built_lib, new, before, size, Hkv, Hq, D, dtype, layout, ragged, rotate):
    from heddle_b200 import ops
    g = _gen(11)
    B, lens = len(new), [a + b for a, b in zip(new, before)]
    pages, table = _cache(B, lens, size, Hkv, D, layout, g)
    T = sum(new) + (3 if ragged else 0)  # rows of no sequence at the end
    packed = torch.randn(T, Hq + 2 * Hkv, D, device="cuda", generator=g).to(DT[dtype])
    packed[:, Hq:] *= torch.exp2(torch.randint(-6, 3, (T, 2 * Hkv, 1), device="cuda", generator=g).float()).to(DT[dtype])
    q, k, v = packed[:, :Hq], packed[:, Hq:Hq + Hkv], packed[:, Hq + Hkv:]
    starts = torch.tensor([0] + new).cumsum(0).int().cuda() if ragged else None
    rope = _rope(max(lens), D) if rotate else None
    want = P.Cache(pages)
    wrote = want.append(k, v, table.cpu(), lens, None if starts is None else starts.tolist(), rope)
    got_q = ops.kv_append(k, v, pages, table, _ints(lens), starts=starts, rope=rope, q=q)
    _clean()
    got = P.Cache(pages)
    for which in (0, 1):
        # the scales are powers of two of maxima that the oracle rounds as the kernel does: equal, and so is every code
        assert torch.equal(got.scales[which], want.scales[which])
        assert torch.equal(got.codes[which], want.codes[which])
    for (page, h, place), (x, y, fine) in wrote.items():
        assert fine
        for which, z in ((0, x), (1, y)):
            s = float(got.scales[which][page, h])
            # half a step of e4m3, whose smallest is 2^-9 of the scale
            assert ((got.codes[which][page, h, place] * s - z).abs() <= torch.maximum(z.abs() * 2.0 ** -4, torch.tensor(s * 2.0 ** -10))).all()
    # the queries: products and sum rounded to fp32 (three half steps of 2^-24 of their sizes), then to 16 bits
    for b, (row, n) in enumerate(P.spans(None if starts is None else starts.tolist(), T, lens)):
        for i in range(n):
            x = q[row + i].double().cpu()
            if rotate:
                cos, sin = (t[lens[b] - n + i].double().cpu() for t in rope)
                ref, size_of = P.rotated(x, cos, sin), P.rotated(x.abs(), cos.abs(), -sin.abs())
                size_of = torch.cat([size_of[:, :D // 2], P.rotated(x.abs(), cos.abs(), sin.abs())[:, D // 2:]], -1)
            else:
                ref, size_of = x, torch.zeros_like(x)
            tol = ref.abs() * (torch.finfo(DT[dtype]).eps / 2 * (1 + 2.0 ** -10)) + size_of * 2.0 ** -22 + torch.finfo(DT[dtype]).smallest_normal * 2.0 ** -10
            assert ((got_q[row + i].double().cpu() - ref).abs() <= tol).all()


def test_append_token_by_token_is_one_call_up_to_scales_that_grew(built_lib):
    """Values go in one by one; each code is the value to half a step of the scale it was rounded at last, plus half a step of those before."""
    from heddle_b200 import ops
    g = _gen(3)
    pages, table = _cache(1, [40], 16, 2, 64, "bhsd", g)
    k, v = (torch.randn(40, 2, 64, device="cuda", generator=g).bfloat16() * torch.exp2(torch.arange(40, device="cuda") / 4.0)[:, None, None].bfloat16()
            for _ in range(2))
    want = P.Cache(pages)
    for t in range(40):
        want.append(k[t:t + 1], v[t:t + 1], table.cpu(), [t + 1])
        ops.kv_append(k[t:t + 1], v[t:t + 1], pages, table, _ints([t + 1]))
    _clean()
    got = P.Cache(pages)
    for which in (0, 1):
        assert torch.equal(got.scales[which], want.scales[which]) and torch.equal(got.codes[which], want.codes[which])


def test_append_special_values(built_lib):
    """Zeros, the smallest and largest numbers, infinities and NaN."""
    from heddle_b200 import ops
    g = _gen(5)
    pages, table = _cache(6, [3] * 6, 16, 1, 64, "bhsd", g)
    k, v = (torch.randn(18, 1, 64, device="cuda", generator=g).bfloat16() for _ in range(2))
    k[0:3] = 0
    v[0:3] = 0
    k[3:6] *= 1e-38
    k[6:9] = 3.38e38 * k[6:9].sign()
    k[10, 0, 5] = math.inf
    v[13, 0, 63] = math.nan
    k[15, 0, 0], v[16, 0, 1] = -math.nan, -math.inf
    want = P.Cache(pages)
    want.append(k, v, table.cpu(), [3] * 6)
    ops.kv_append(k, v, pages, table, _ints([3] * 6))
    _clean()
    got = P.Cache(pages)
    for which in (0, 1):
        assert torch.equal(got.scales[which], want.scales[which])
        assert torch.equal(torch.nan_to_num(got.codes[which], nan=1000.0), torch.nan_to_num(want.codes[which], nan=1000.0))
    assert torch.isnan(got.codes[0][int(table[3, 0]), 0, 1]).all() and (got.codes[1][int(table[4, 0]), 0, 1] == 0).all()
    # a query that sees such a token is NaN, one that does not is not
    out = ops.fa_paged(torch.ones(18, 1, 64, device="cuda", dtype=torch.bfloat16), pages, table, _ints([3] * 6))
    _clean()
    assert torch.isnan(out).any(-1)[:, 0].tolist() == [False] * 10 + [True, True, False, True, True, True, True, True]


# --------------------------------------------------------------------------------------------------------------------------
# attention
# --------------------------------------------------------------------------------------------------------------------------
def _close(got, lse, ref, dtype):
    out, want_lse, mean, spread, score = ref
    eps = torch.finfo(DT[dtype]).eps / 2
    # P to fp16 (2^-12), a score off by `score` moves its weight and the sum by as much (twice), exponentials and sums 2^-20; what lies
    # 2^-23 below the largest value scale may be lost for every key
    tol = out.abs() * eps * 1.01 + (2.0 ** -12 + 2 * score[..., None] + 2.0 ** -19) * mean * (1 + 2.0 ** -6) + spread * 2.0 ** -22 + 1e-30
    tol += torch.finfo(DT[dtype]).smallest_normal * eps  # half a step of the subnormal numbers (fp16: 2^-25)
    got = got.cpu()
    bad = (got.double() - out).abs() > tol
    # a result from half a step beyond the type's largest number on is an infinity (fp16: 65504 + 16)
    largest = torch.finfo(DT[dtype]).max * (1 + eps / 2)
    bad &= ~((out.abs() + tol >= largest) & (got.double() == math.inf * out.sign()))
    assert not bad.any(), (got[bad][:8], out[bad][:8], tol[bad][:8])
    assert not torch.isnan(got).any()
    if lse is not None:
        lse = lse.double().cpu()
        empty = want_lse == -math.inf
        assert torch.equal(lse == -math.inf, empty)
        tol = score + want_lse.abs() * 2.0 ** -22 + 2.0 ** -19  # fp32 results of base-2 logarithms
        assert ((lse - want_lse).abs() <= tol)[~empty].all()


ATTENDS = [  # new, lens, page size, Hkv, group, D, dtype, layout, ragged call, causal
    ([1], [1], 16, 1, 1, 64, "bf16", "bhsd", False, True),
    ([1] * 4, [1, 31, 33, 700], 16, 2, 4, 128, "bf16", "bhsd", False, True),
    ([1] * 3, [129, 64, 2000], 64, 1, 8, 128, "fp16", "bshd", False, True),
    ([1] * 2, [1500, 5], 128, 3, 1, 64, "fp16", "bhsd", False, True),
    ([1] * 2, [300, 299], 32, 2, 17, 128, "bf16", "bhsd", False, True),
    ([4] * 3, [4, 100, 513], 32, 2, 4, 128, "bf16", "bshd", False, True),
    ([2] * 3, [2, 100, 513], 32, 2, 3, 64, "fp16", "bshd", False, True),
    ([5] * 2, [7, 90], 16, 2, 2, 64, "bf16", "bhsd", False, False),
    ([40, 0, 1, 77], [40, 12, 300, 130], 16, 2, 7, 128, "bf16", "bhsd", True, True),
    ([130, 3], [257, 3], 64, 1, 4, 64, "fp16", "bshd", True, True),
    ([60, 1], [200, 130], 32, 2, 2, 128, "fp16", "bhsd", True, False),
    ([260], [300], 64, 1, 2, 128, "bf16", "bhsd", True, True),
    # many rows: keys of an item over several SMs, rows that see none of some part, tiles that end with the keys, pages of every size
    ([128], [2000], 16, 1, 4, 128, "bf16", "bhsd", False, True),
    ([300], [300], 128, 2, 3, 64, "fp16", "bshd", False, True),
    ([256, 256], [1024, 1024], 64, 2, 1, 128, "fp16", "bhsd", False, True),
    ([129] * 3, [640, 641, 129], 32, 1, 5, 64, "bf16", "bshd", False, False),
    ([1, 400, 2, 90, 0, 33], [700, 900, 2, 1000, 50, 40], 64, 2, 4, 128, "bf16", "bshd", True, True),
    ([70] * 40, [70 + 9 * b for b in range(40)], 32, 4, 2, 64, "fp16", "bhsd", False, True),
]


@pytest.mark.parametrize("hint", (True, False))
@pytest.mark.parametrize("new,lens,size,Hkv,group,D,dtype,layout,ragged,causal", ATTENDS)
def test_attend(built_lib, new, lens, size, Hkv, group, D, dtype, layout, ragged, causal, hint):
    from heddle_b200 import ops
    g = _gen(7)
    pages, table = _cache(len(new), lens, size, Hkv, D, layout, g)
    T = sum(new) + (2 if ragged else 0)
    q = (torch.randn(T, Hkv * group + 1, D, device="cuda", generator=g) * 2).to(DT[dtype])[:, 1:]
    starts = torch.tensor([0] + new).cumsum(0).int().cuda() if ragged else None
    out = torch.full((T, Hkv * group, D), 7.0, dtype=DT[dtype], device="cuda")
    got, lse = ops.fa_paged(q, pages, table, _ints(lens), starts=starts, max_tokens=max(new) if hint else None, causal=causal, return_lse=True, out=out)
    _clean()
    assert got is out
    live = sum(new)
    assert (out[live:] == 7.0).all()
    cpu = P.attend(q[:live], P.Cache(pages), table.cpu(), lens, None if starts is None else starts.tolist(), causal)
    _close(got[:live], lse[:live], cpu, dtype)


def test_stale_places_and_pages_do_not_matter(built_lib):
    """What lies behind a sequence, in its last page, in pages of nobody and in the table's other entries, is never read as numbers."""
    from heddle_b200 import ops
    g = _gen(9)
    for new in (1, 20):
        lens, size = [37, 70, 21], 32
        pages, table = _cache(3, lens, size, 2, 128, "bhsd", g)
        table = torch.cat([table, torch.full((3, 2), -5, dtype=torch.int32, device="cuda")], 1).contiguous()
        table[0, 2], table[2, 1:3] = 1 << 30, -(1 << 31)
        q = torch.randn(3 * new, 8, 128, device="cuda", generator=g).bfloat16()
        first = ops.fa_paged(q, pages, table, _ints(lens), return_lse=True)
        for which in (pages.k, pages.v):
            codes = which.view(torch.uint8)
            used = torch.zeros(codes.shape[:3], dtype=torch.bool, device="cuda")
            for b, n in enumerate(lens):
                for block in range(-(-n // size)):
                    used[int(table[b, block]), :, :min(size, n - block * size)] = True
            codes[~used] = 0x7F
        unused = [p for p in range(pages.k.shape[0]) if p not in {int(table[b, i]) for b, n in enumerate(lens) for i in range(-(-n // size))}]
        pages.k_scale[unused], pages.v_scale[unused] = math.nan, math.inf
        again = ops.fa_paged(q, pages, table, _ints(lens), return_lse=True)
        _clean()
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("new", (1, 3, 50))
def test_rows_without_keys(built_lib, new):
    """Empty sequences, and (as the lengths say) queries in front of the first token."""
    from heddle_b200 import ops
    g = _gen(13)
    lens = [0, 5, 64]
    pages, table = _cache(3, lens, 16, 2, 64, "bhsd", g)
    q = torch.randn(3 * new, 4, 64, device="cuda", generator=g).half()
    out, lse = ops.fa_paged(q, pages, table, _ints(lens), return_lse=True)
    short = new > 0 and ops.cache_status()
    assert short == 2  # the first sequence has fewer tokens than rows
    _close(out, lse, P.attend(q, P.Cache(pages), table.cpu(), lens), "fp16")
    assert (out[:new] == 0).all() and (lse[:new] == -math.inf).all()


def test_what_the_device_finds_wrong(built_lib):
    from heddle_b200 import ops
    g = _gen(17)
    size, lens = 16, [40, 40]
    pages, table = _cache(2, lens, size, 1, 64, "bhsd", g)
    table[1, 1] = pages.k.shape[0]  # one behind the last page
    q = torch.randn(2, 2, 64, device="cuda", generator=g).half()
    out, lse = ops.fa_paged(q, pages, table, _ints(lens), return_lse=True)
    assert ops.cache_status() == 1 and ops.cache_status() == 0
    _close(out, lse, P.attend(q, P.Cache(pages), table.cpu(), lens), "fp16")  # its tokens are not there
    # a length behind the table row: taken as the row's
    out, lse = ops.fa_paged(q, pages, table[:, :1].contiguous(), _ints([1000, 16]), return_lse=True)
    assert ops.cache_status() == 2
    _close(out, lse, P.attend(q, P.Cache(pages), table[:, :1].cpu(), [16, 16]), "fp16")
    # starts that descend and leave the rows
    ops.fa_paged(q, pages, table[:, :1].contiguous(), _ints([16, 16]), starts=_ints([-3, 5, 1]))
    assert ops.cache_status() == 4
    # append: a page of nobody's is not written, nor a position behind the tables
    before = P.Cache(pages)
    k = torch.ones(2, 1, 64, device="cuda", dtype=torch.half)
    table[0, 2] = -1
    ops.kv_append(k, k, pages, table, _ints([40, 41]), rope=_rope(40, 64))
    assert ops.cache_status() == 9
    after = P.Cache(pages)
    assert all(torch.equal(x, y) for x, y in zip(before.codes + before.scales, after.codes + after.scales))
    _clean()


@pytest.mark.parametrize("new,group", ((100, 4), (200, 1)))
def test_pages_that_are_not_there_for_many_rows(built_lib, new, group):
    """The same with prompts: pages of nobody's and pages without scales within a tile of keys, in its last one, and a whole tile of them."""
    from heddle_b200 import ops
    g = _gen(41)
    size, lens = 16, [700, 333]
    pages, table = _cache(2, lens, size, 2, 128, "bhsd", g)
    for block in (1, 20, *range(24, 32), 43):
        table[0, block] = -1 if block % 2 else pages.k.shape[0] + block
    scaleless = int(table[1, 5])
    pages.k_scale[scaleless] = 0
    q = torch.randn(2 * new, 2 * group, 128, device="cuda", generator=g).bfloat16()
    out, lse = ops.fa_paged(q, pages, table, _ints(lens), return_lse=True)
    assert ops.cache_status() == 1 and ops.status_word() == 0
    table[1, 5] = -1  # a page whose key scale is 0 is not there either
    _close(out, lse, P.attend(q, P.Cache(pages), table.cpu(), lens), "bf16")


def test_scales_of_any_size_and_peaked_rows(built_lib):
    """Value scales that grow and shrink along a sequence by 2^30, scores up to hundreds: a row's result is still that of its own keys."""
    from heddle_b200 import ops
    g = _gen(19)
    lens, size = [500, 333], 16
    pages, table = _cache(2, lens, size, 2, 128, "bhsd", g)
    pages.v_scale.copy_(torch.exp2(torch.randint(-30, 10, pages.v_scale.shape, device="cuda", generator=g).float()))
    pages.k_scale.copy_(torch.exp2(torch.randint(-12, -3, pages.k_scale.shape, device="cuda", generator=g).float()))
    for new in (1, 30):
        q = (torch.randn(2 * new, 8, 128, device="cuda", generator=g) * 4).bfloat16()
        q[0, 0] = 0
        out, lse = ops.fa_paged(q, pages, table, _ints(lens), return_lse=True)
        _clean()
        _close(out, lse, P.attend(q, P.Cache(pages), table.cpu(), lens), "bf16")


def test_queries_that_are_not_finite_stay_alone(built_lib):
    from heddle_b200 import ops
    g = _gen(23)
    for new in (1, 40):
        pages, table = _cache(2, [100, 90], 32, 2, 64, "bhsd", g)
        q = torch.randn(2 * new, 6, 64, device="cuda", generator=g).bfloat16()
        ref = ops.fa_paged(q, pages, table, _ints([100, 90]))
        q[0, 1, 3], q[new, 5, 60] = math.nan, math.inf
        out = ops.fa_paged(q, pages, table, _ints([100, 90]))
        _clean()
        sick = torch.zeros(2 * new, 6, dtype=torch.bool, device="cuda")
        sick[0, 1] = sick[new, 5] = True
        assert torch.isnan(out[sick]).all() and torch.equal(out[~sick], ref[~sick])


# --------------------------------------------------------------------------------------------------------------------------
# as a server runs them
# --------------------------------------------------------------------------------------------------------------------------
def test_prompt_then_tokens(built_lib):
    """A ragged prompt, then decode steps captured once and replayed with other lengths, tokens and pages."""
    from heddle_b200 import ops
    g = _gen(29)
    B, Hq, Hkv, D, size, steps = 3, 8, 2, 128, 16, 20
    new = [37, 5, 64]
    top = [n + steps for n in new]
    pages, table = _cache(B, top, size, Hkv, D, "bhsd", g, filled=False)
    rope = _rope(max(top), D)

    def rows(n):
        return torch.randn(n, Hq + 2 * Hkv, D, device="cuda", generator=g).bfloat16()

    def split(x):
        return x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]

    want = P.Cache(pages)

    def check(x, lens, starts, q, out, lse):
        _, k, v = split(x)
        want.append(k, v, table.cpu(), lens, starts, rope)
        _close(out, lse, P.attend(q, want, table.cpu(), lens, starts), "bf16")

    starts = torch.tensor([0] + new).cumsum(0).int().cuda()
    x = rows(sum(new))
    q, k, v = split(x)
    q = ops.kv_append(k, v, pages, table, _ints(new), starts=starts, rope=rope, q=q)
    out, lse = ops.fa_paged(q, pages, table, _ints(new), starts=starts, max_tokens=64, return_lse=True)
    check(x, new, starts.tolist(), q, out, lse)

    lens = _ints(new)
    x = rows(B)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    saved = [t.clone() for t in pages[:4]]
    with torch.cuda.stream(side):
        lens.add_(1)
        q1 = ops.kv_append(*split(x)[1:], pages, table, lens, rope=rope, q=split(x)[0])
        ops.fa_paged(q1, pages, table, lens, return_lse=True)
        lens.sub_(1)
        for t, s in zip(pages[:4], saved):
            t.copy_(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            lens.add_(1)
            q1 = ops.kv_append(*split(x)[1:], pages, table, lens, rope=rope, q=split(x)[0])
            out, lse = ops.fa_paged(q1, pages, table, lens, return_lse=True)
    torch.cuda.current_stream().wait_stream(side)
    for step in range(steps):
        x.copy_(rows(B))
        graph.replay()
        torch.cuda.synchronize()
        check(x, [n + step + 1 for n in new], None, q1, out, lse)
    _clean()
    got = P.Cache(pages)
    for which in (0, 1):
        assert torch.equal(got.scales[which], want.scales[which]) and torch.equal(got.codes[which], want.codes[which])


def test_results_repeat_and_do_not_depend_on_the_stream(built_lib):
    from heddle_b200 import ops
    g = _gen(31)
    lens = [900, 20, 3000, 1, 450]
    pages, table = _cache(5, lens, 64, 4, 128, "bhsd", g)
    q = torch.randn(5, 16, 128, device="cuda", generator=g).bfloat16()
    n = _ints(lens)
    torch.cuda.synchronize()
    runs = [ops.fa_paged(q, pages, table, n, return_lse=True) for _ in range(3)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        with torch.cuda.stream(s):
            runs += [ops.fa_paged(q, pages, table, n, return_lse=True) for _ in range(3)]
    _clean()
    for out, lse in runs[1:]:
        assert torch.equal(out, runs[0][0]) and torch.equal(lse, runs[0][1])


def test_prompts_captured_and_replayed(built_lib):
    """A call of ragged prompts and single tokens is captured; lengths, starts and pages are others at its replays."""
    from heddle_b200 import ops
    g = _gen(43)
    B, T, size = 4, 300, 32
    pages, table = _cache(B, [900] * B, size, 2, 128, "bhsd", g)
    q = torch.randn(T, 8, 128, device="cuda", generator=g).bfloat16()
    lens, starts = _ints([900, 900, 900, 900]), _ints([0, 1, 250, 250, 300])
    out = torch.full_like(q, 3.0)
    call = lambda: ops.fa_paged(q, pages, table, lens, starts=starts, max_tokens=300, return_lse=True, out=out)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            _, lse = call()
    torch.cuda.current_stream().wait_stream(side)
    for new, n in (([1, 249, 0, 50], [900, 800, 0, 70]), ([100, 100, 99, 1], [100, 500, 129, 1]), ([1, 1, 1, 1], [33, 500, 128, 1]), ([0, 0, 300, 0], [5, 6, 640, 9])):
        order = torch.randperm(B, generator=torch.Generator().manual_seed(sum(n))).tolist()
        table.copy_(table[order].clone())
        lens.copy_(_ints(n))
        starts.copy_(torch.tensor([0] + new).cumsum(0).int())
        out.fill_(3.0)
        graph.replay()
        _clean()
        live = sum(new)
        assert (out[live:] == 3.0).all()
        _close(out[:live], lse[:live], P.attend(q[:live], P.Cache(pages), table.cpu(), n, starts.tolist()), "bf16")


def test_calls_on_two_streams_at_once(built_lib):
    from heddle_b200 import ops
    g = _gen(47)
    work = []
    for B, n, lens in ((3, 1, [2000, 100, 900]), (2, 150, [600, 150]), (5, 1, [700] * 5), (1, 300, [1500])):
        pages, table = _cache(B, lens, 64, 2, 128, "bhsd", g)
        q = torch.randn(B * n, 8, 128, device="cuda", generator=g).bfloat16()
        work.append((q, pages, table, _ints(lens)))
    alone = [ops.fa_paged(*w, return_lse=True) for w in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for _ in range(20):
        for w, s in zip(work, streams):
            with torch.cuda.stream(s):
                got.append(ops.fa_paged(*w, return_lse=True))
    _clean()
    for k, (out, lse) in enumerate(got):
        assert torch.equal(out, alone[k % 4][0]) and torch.equal(lse, alone[k % 4][1])


def test_sequences_share_a_prefix(built_lib):
    from heddle_b200 import ops
    g = _gen(37)
    pages, table = _cache(4, [200] * 4, 32, 2, 128, "bhsd", g)
    table[1:, :5] = table[0, :5]  # 160 tokens in common
    q = torch.randn(4, 8, 128, device="cuda", generator=g).bfloat16()
    lens = [200, 161, 160, 199]
    out, lse = ops.fa_paged(q, pages, table, _ints(lens), return_lse=True)
    _clean()
    _close(out, lse, P.attend(q, P.Cache(pages), table.cpu(), lens), "bf16")


def test_refusals_with_tensors(built_lib):
    from heddle_b200 import ops
    pages = ops.kv_pages(4, 16, 2, 64)
    table, lens = torch.zeros(2, 4, dtype=torch.int32, device="cuda"), _ints([1, 1])
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    for call in (lambda: ops.kv_append(x.float(), x.float(), pages, table, lens), lambda: ops.kv_append(x, x.half(), pages, table, lens),
                 lambda: ops.kv_append(x, x, pages, table, lens, q=x.half()), lambda: ops.fa_paged(x.float(), pages, table, lens)):
        with pytest.raises(TypeError):
            call()
    cos = torch.ones(8, 32, device="cuda")
    for call in (lambda: ops.kv_append(x[:, :1], x[:, :1], pages, table, lens), lambda: ops.kv_append(x, x[:1], pages, table, lens),
                 lambda: ops.kv_append(x, x, pages, table, lens, q=x[:1]), lambda: ops.kv_append(x, x, pages, table, lens, rope=(cos, cos[:, :16])),
                 lambda: ops.kv_append(x, x, pages, table, lens, rope=(cos[:, :16], cos[:, :16])),
                 lambda: ops.fa_paged(x[:, :, :32], pages, table, lens),
                 lambda: ops.fa_paged(x, pages, table, lens, out=x[:1]), lambda: ops.fa_paged(x, pages, table, lens, out=x.half())):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):
        ops.fa_paged(x, pages, table, lens.cpu())
    with pytest.raises(RuntimeError):
        ops.fa_paged(x[:, :1].expand(2, 3, 64).contiguous(), pages, table, lens)  # 3 heads over 2
    with pytest.raises(RuntimeError):
        ops.kv_append(x[:1].expand(3, 2, 64).contiguous(), x[:1].expand(3, 2, 64).contiguous(), pages, table, lens)  # 3 rows, 2 sequences
