"""The native host path of ``kv_append`` and ``fa_paged`` against the general path of ops.py: the same results, the same refusals."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _state(layout="bhsd", D=64, Hkv=2, Hq=4, new=2, B=2, dtype=BF):
    from heddle_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(5)
    pages = ops.kv_pages(8, 16, Hkv, D, layout=layout)
    for codes, scale in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)):
        codes.copy_((torch.randn(codes.shape, device="cuda", generator=g) * 80).to(torch.float8_e4m3fn))
        scale.fill_(2.0 ** -7)
    x = torch.randn(B * new, Hq + 2 * Hkv, D, device="cuda", generator=g).to(dtype)
    table = torch.randperm(8, device="cuda", generator=g)[:3 * B].reshape(B, 3).int()
    lens = torch.tensor([33, 20][:B], dtype=torch.int32, device="cuda")
    angle = torch.rand(48, D // 2, device="cuda", generator=g)
    return dict(q=x[:, :Hq], k=x[:, Hq:Hq + Hkv], v=x[:, Hq + Hkv:], pages=pages, table=table, lens=lens, rope=(angle.cos(), angle.sin()),
                starts=torch.tensor([0, 1, B * new][:B + 1], dtype=torch.int32, device="cuda"))


def _append(change=lambda s: s, **kw):
    def call(ops):
        s = change(_state(**kw))
        q = ops.kv_append(s["k"], s["v"], s["pages"], s["table"], s["lens"], starts=s.get("use_starts"), rope=s["rope"], q=s["q"])
        return (q, *s["pages"][:4])
    return call


def _attend(change=lambda s: s, args=None, **kw):
    def call(ops):
        s = change(_state(**kw))
        return ops.fa_paged(s["q"], s["pages"], s["table"], s["lens"], starts=s.get("use_starts"), **(args or {}))
    return call


def _set(**values):
    return lambda s: {**s, **{k: f(s) for k, f in values.items()}}


def _out(s_out):
    def call(ops):
        s = _state()
        out = s_out(s["q"])
        r = ops.fa_paged(s["q"], s["pages"], s["table"], s["lens"], out=out)
        assert r is out
        return r
    return call


FORMS = {  # name: (call, taken natively)
    "append": (_append(), True),
    "append bshd 128": (_append(layout="bshd", D=128), True),
    "append fp16, no rotation": (_append(_set(rope=lambda s: None), dtype=torch.float16), True),
    "append without queries": (_append(_set(q=lambda s: None)), True),
    "append starts": (_append(_set(use_starts=lambda s: s["starts"])), True),
    "append rows apart": (_append(_set(k=lambda s: s["k"].transpose(1, 2).contiguous().transpose(1, 2))), False),
    "append misaligned": (_append(_set(v=lambda s: torch.cat([s["v"].flatten(), s["v"].flatten()])[1:1 + s["v"].numel()].view(s["v"].shape))), False),
    "append 64-bit tables": (_append(_set(rope=lambda s: tuple(t.double() for t in s["rope"]))), False),
    "append misaligned tables": (_append(_set(rope=lambda s: tuple(torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape) for t in s["rope"]))), False),
    "append no rows": (_append(_set(k=lambda s: s["k"][:0], v=lambda s: s["v"][:0], q=lambda s: s["q"][:0])), False),
    "append other types": (_append(_set(v=lambda s: s["v"].half())), None),
    "append other heads": (_append(_set(k=lambda s: s["k"][:, :1], v=lambda s: s["v"][:, :1])), None),
    "append odd rows": (_append(_set(k=lambda s: s["k"][:3], v=lambda s: s["v"][:3], q=lambda s: s["q"][:3])), None),
    "append long table": (_append(_set(table=lambda s: s["table"].long())), None),
    "attend": (_attend(), True),
    "attend lse, scale, all keys": (_attend(args=dict(return_lse=True, softmax_scale=0.3, causal=False)), True),
    "attend starts": (_attend(_set(use_starts=lambda s: s["starts"]), args=dict(max_tokens=3)), True),
    "attend bshd 128 fp16": (_attend(layout="bshd", D=128, dtype=torch.float16), True),
    "attend out": (_out(lambda q: torch.empty(q.shape[0], 2 * q.shape[1], q.shape[2], dtype=q.dtype, device="cuda")[:, ::2]), True),
    "attend plain tuple": (_attend(_set(pages=lambda s: tuple(s["pages"]))), True),
    "attend rows apart": (_attend(_set(q=lambda s: s["q"].transpose(1, 2).contiguous().transpose(1, 2))), False),
    "attend no rows": (_attend(_set(q=lambda s: s["q"][:0])), False),
    "attend 3 heads": (_attend(_set(q=lambda s: s["q"][:, :3])), None),
    "attend bad layout": (_attend(_set(pages=lambda s: s["pages"]._replace(layout="sbhd"))), None),
    "attend fp32": (_attend(_set(q=lambda s: s["q"].float())), None),
    "attend scales of another shape": (_attend(_set(pages=lambda s: s["pages"]._replace(k_scale=s["pages"].k_scale.t().contiguous()))), None),
    "attend long lens": (_attend(_set(lens=lambda s: s["lens"].long())), None),
    "attend head_dim": (_attend(_set(q=lambda s: s["q"][..., :32])), None),
    "attend bad out": (_attend(args=dict(out=torch.empty(1))), None),
}


class _Spy:
    def __init__(self, native):
        self._native, self.taken = native, None

    def __getattr__(self, name):
        fn = getattr(self._native, name)

        def call(*args):
            self.taken = False
            r = fn(*args)
            self.taken = r is not NotImplemented
            return r
        return call


def _outcome(call, ops):
    try:
        r = call(ops)
    except Exception as e:  # noqa: BLE001  (a refusal is an outcome)
        return type(e), str(e)
    torch.cuda.synchronize()
    return r if isinstance(r, tuple) else (r,)


@pytest.mark.parametrize("form", list(FORMS))
def test_same_as_the_general_path(built_lib, monkeypatch, form):
    from heddle_b200 import _lib, ops
    call, taken = FORMS[form]
    spy = _Spy(_lib.native)
    monkeypatch.setattr(_lib, "native", spy)
    got = _outcome(call, ops)
    refused = isinstance(got[0], type)
    assert refused == (taken is None)
    if not refused:
        assert bool(spy.taken) == taken
    monkeypatch.setattr(_lib, "native", None)
    ref = _outcome(call, ops)
    assert len(got) == len(ref)
    for a, b in zip(got, ref):
        if isinstance(b, torch.Tensor):
            assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride() and a.device == b.device
            assert torch.equal(a.float(), b.float())
        else:
            assert a == b
    assert ops.status_word() == 0 and ops.cache_status() == 0
