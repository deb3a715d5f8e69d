"""The paged cache at the far ends: more sequences than a block has threads, and offsets that pass 32 bits."""
import pytest
import torch

from oracle import paged_oracle as P
from test_paged_gpu import DT, _cache, _clean, _close, _gen, _ints, _rope

pytestmark = pytest.mark.gpu

MANY = [  # sequences, rows of sequence b, tokens of it, page size, Hkv, group, D, ragged call, causal
    (129, lambda b: 1, lambda b: 1 + 5 * b % 67, 16, 2, 1, 64, False, True),
    (700, lambda b: 1, lambda b: 1 + 7 * b % 90, 32, 1, 4, 128, False, True),
    (300, lambda b: 3, lambda b: 3 + 11 * b % 50, 16, 1, 2, 64, False, True),
    (260, lambda b: b % 4, lambda b: 3 + 13 * b % 70, 64, 1, 4, 128, True, True),
    # the last sequences are the prompts; two kernels side by side
    (600, lambda b: 70 if b > 560 else b % 2, lambda b: 70 + b % 31, 16, 4, 2, 64, True, True),
    (530, lambda b: 140 if b % 90 == 5 else 1, lambda b: 140 + b % 60, 128, 2, 2, 128, True, False),
    (1100, lambda b: 33 if b >= 1040 else 0, lambda b: 33 + b % 9, 32, 4, 2, 64, True, True),
]


@pytest.mark.parametrize("B,rows,tokens,size,Hkv,group,D,ragged,causal", MANY)
def test_many_sequences(built_lib, B, rows, tokens, size, Hkv, group, D, ragged, causal):
    from heddle_b200 import ops
    g = _gen(131)
    new, lens = [rows(b) for b in range(B)], [tokens(b) for b in range(B)]
    T, Hq = sum(new), Hkv * group
    pages, table = _cache(B, lens, size, Hkv, D, "bhsd", g)
    rope = _rope(max(lens), D)
    k, v = (torch.randn(T, Hkv, D, device="cuda", generator=g).bfloat16() for _ in range(2))
    q = torch.randn(T, Hq, D, device="cuda", generator=g).bfloat16()
    starts = torch.tensor([0] + new).cumsum(0).int().cuda() if ragged else None
    at = None if starts is None else starts.tolist()
    want = P.Cache(pages)
    want.append(k, v, table.cpu(), lens, at, rope)
    q = ops.kv_append(k, v, pages, table, _ints(lens), starts=starts, rope=rope, q=q)
    out, lse = ops.fa_paged(q, pages, table, _ints(lens), starts=starts, max_tokens=max(new), causal=causal, return_lse=True)
    unhinted = ops.fa_paged(q, pages, table, _ints(lens), starts=starts, causal=causal)
    small = ops.fa_paged(q, pages, table, _ints(lens), starts=starts, max_tokens=1, causal=causal)
    _clean()
    got = P.Cache(pages)
    for which in (0, 1):
        assert torch.equal(got.scales[which], want.scales[which]) and torch.equal(got.codes[which], want.codes[which])
    ref = P.attend(q, want, table.cpu(), lens, at, causal)
    _close(out, lse, ref, "bf16")
    _close(unhinted, None, ref, "bf16")
    _close(small, None, ref, "bf16")


@pytest.mark.parametrize("layout", ("bhsd", "bshd"))
@pytest.mark.parametrize("B,new,length,Hkv,group", ((3, 1, 500, 8, 4), (3, 4, 500, 8, 4), (10, 70, 300, 8, 4), (2, 256, 1500, 8, 4)))
def test_pages_beyond_32_bits(built_lib, layout, B, new, length, Hkv, group):
    """The last pages of 5 GB of codes hold what the pages of a small cache hold: the same bits come out, and the same codes go in."""
    from heddle_b200 import ops
    g = _gen(137)
    size, D, count = 128, 128, 40000
    lens = [length - 9 * b for b in range(B)]
    small, table = _cache(B, lens, size, Hkv, D, layout, g)
    used = small.k.shape[0]
    large = ops.kv_pages(count, size, Hkv, D, layout=layout)
    assert (count - used) * Hkv * size * D > 2 ** 32
    for name in ("k", "v"):
        getattr(large, name).view(torch.uint8)[count - used:] = getattr(small, name).view(torch.uint8)
        getattr(large, name + "_scale")[count - used:] = getattr(small, name + "_scale")
    far = table + (count - used)
    k, v, q = (torch.randn(B * new, H, D, device="cuda", generator=g).bfloat16() for H in (Hkv, Hkv, Hkv * group))
    for pages, where in ((small, table), (large, far)):
        ops.kv_append(k, v, pages, where, _ints(lens))
    one = ops.fa_paged(q, small, table, _ints(lens), return_lse=True)
    two = ops.fa_paged(q, large, far, _ints(lens), return_lse=True)
    _clean()
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    for name in ("k", "v"):
        assert torch.equal(getattr(large, name).view(torch.uint8)[count - used:], getattr(small, name).view(torch.uint8))
        assert not getattr(large, name).view(torch.uint8)[:count - used].any()
        assert torch.equal(getattr(large, name + "_scale")[count - used:], getattr(small, name + "_scale"))


@pytest.mark.parametrize("Hkv,group,ragged", ((2, 1, False), (1, 64, False), (8, 4, True)))
def test_rows_beyond_32_bits(built_lib, Hkv, group, ragged):
    """Three tokens whose rows lie 1.2e9 elements apart, against the same rows side by side."""
    from heddle_b200 import ops
    g = _gen(139)
    D, step, T = 64, 1_200_000_000, 3
    Hq = Hkv * group
    lens = [90, 50] if ragged else [90, 50, 33]
    starts = _ints([0, 1, 3]) if ragged else None
    whole = torch.empty(2 * step + Hq * D, dtype=torch.bfloat16, device="cuda")
    rows = whole.as_strided((T, Hq, D), (step, D, 1))
    q = torch.randn(T, Hq, D, device="cuda", generator=g).bfloat16()
    rows.copy_(q)
    pages, table = _cache(len(lens), lens, 16, Hkv, D, "bhsd", g)
    k = rows[:, :Hkv]
    want = P.Cache(pages)
    want.append(k, k, table.cpu(), lens, None if starts is None else starts.tolist(), _rope(90, D))
    turned = ops.kv_append(q[:, :Hkv], q[:, :Hkv], pages, table, _ints(lens), starts=starts, rope=_rope(90, D), q=q)
    near = ops.fa_paged(turned, pages, table, _ints(lens), starts=starts)
    again = ops.kv_append(k, k, pages, table, _ints(lens), starts=starts, rope=_rope(90, D), q=rows)
    assert torch.equal(again, turned)
    rows.copy_(turned)
    far = torch.empty_like(whole).as_strided((T, Hq, D), (step, D, 1))
    got_far = ops.fa_paged(rows, pages, table, _ints(lens), starts=starts, out=far)
    _clean()
    got = P.Cache(pages)
    for which in (0, 1):
        assert torch.equal(got.scales[which], want.scales[which]) and torch.equal(got.codes[which], want.codes[which])
    assert got_far.data_ptr() == far.data_ptr() and torch.equal(far, near)


def test_one_step_of_a_large_batch_captured(built_lib):
    """More sequences than a block has threads, captured and replayed with lengths that moved on."""
    from heddle_b200 import ops
    g = _gen(149)
    B, Hkv, Hq, D, size = 200, 2, 4, 64, 16
    lens = [1 + 3 * b % 40 for b in range(B)]
    pages, table = _cache(B, [n + 4 for n in lens], size, Hkv, D, "bhsd", g)
    k, v = (torch.randn(B, Hkv, D, device="cuda", generator=g).bfloat16() for _ in range(2))
    q = torch.randn(B, Hq, D, device="cuda", generator=g).bfloat16()
    on_device, out = _ints(lens), torch.empty_like(q)

    def step():
        ops.kv_append(k, v, pages, table, on_device)
        ops.fa_paged(q, pages, table, on_device, out=out)
    want = P.Cache(pages)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    want.append(k, v, table.cpu(), lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for more in range(1, 4):
        on_device.add_(1)
        k.mul_(-1.0)
        graph.replay()
        torch.cuda.synchronize()
        now = [n + more for n in lens]
        want.append(k, v, table.cpu(), now)
        _close(out, None, P.attend(q, want, table.cpu(), now), "bf16")
    _clean()


@pytest.mark.parametrize("seed", range(24))
def test_drawn(built_lib, seed):
    """Batches of any mixture: items of one tile and of many in one run, sequences without rows or keys, heads in odd groups."""
    import random

    from heddle_b200 import ops
    rng, g = random.Random(seed), _gen(151 + seed)
    B, size, D = rng.choice((1, 3, 20, 150, 400)), rng.choice((16, 32, 64, 128)), rng.choice((64, 128))
    Hkv, group, dtype = rng.choice((1, 2, 5)), rng.choice((1, 3, 4, 8, 9)), rng.choice(("bf16", "fp16"))
    ragged, causal, layout = rng.random() < 0.6, rng.random() < 0.8, rng.choice(("bhsd", "bshd"))
    most, longest = rng.choice((1, 1, 4, 60 if B <= 20 else 2)), rng.choice((8, 70, 200, 900 if B <= 20 else 130))
    new = [rng.randint(0, most) for _ in range(B)] if ragged else [most] * B
    lens = [n + rng.randint(0, longest) for n in new]
    live = sum(new)
    T = live + (2 if ragged else 0)
    pages, table = _cache(B, lens, size, Hkv, D, layout, g)
    q = (torch.randn(T, Hkv * group, D, device="cuda", generator=g) * 2).to(DT[dtype])
    starts = torch.tensor([0] + new).cumsum(0).int().cuda() if ragged else None
    out = torch.full_like(q, 7.0)
    got, lse = ops.fa_paged(q, pages, table, _ints(lens), starts=starts, max_tokens=rng.choice((None, most)), causal=causal, return_lse=True, out=out)
    _clean()
    assert (out[live:] == 7.0).all()
    ref = P.attend(q[:live], P.Cache(pages), table.cpu(), lens, None if starts is None else starts.tolist(), causal)
    _close(got[:live], lse[:live], ref, dtype)


@pytest.mark.parametrize("B,new", ((5, 1), (5, 4), (10, 70), (2, 256)))
def test_rows_backwards(built_lib, B, new):
    """Tokens and heads from the last to the first, through the C interface: strides may be negative."""
    import ctypes as C

    from heddle_b200 import _lib, ops
    g = _gen(179)
    Hkv, Hq, D = 8, 16, 128
    T, lens = B * new, [300 + 17 * b for b in range(B)]
    pages, table = _cache(B, lens, 32, Hkv, D, "bhsd", g)
    q, seq_lens = torch.randn(T, Hq, D, device="cuda", generator=g).bfloat16(), _ints(lens)
    want = ops.fa_paged(q, pages, table, seq_lens)
    back, out = q.flip(0, 1).contiguous(), torch.zeros_like(q)
    last = 2 * D * (T * Hq - 1)  # bytes in front of the last head of the last token
    a = _lib.FaPagedArgs(ops._kv_cache("fa_paged", pages, table, seq_lens, None, q), back.data_ptr() + last, out.data_ptr() + last, None, -Hq * D, -D,
                         -Hq * D, -D, Hq, 0, 1, D ** -0.5, ops._DTYPES[q.dtype], torch.cuda.current_stream().cuda_stream)
    need = C.c_uint64(0)
    _lib.check(_lib.load().hb_fa_paged_workspace(C.byref(a), C.byref(need)))
    space = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    _lib.check(_lib.load().hb_fa_paged(C.byref(a), space.data_ptr(), need.value))
    _clean()
    assert torch.equal(out.flip(0, 1), want)
