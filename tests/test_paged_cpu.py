"""The paged cache's entry points without a GPU: layouts of the argument structs, what is refused before any CUDA call, the oracle."""
import ctypes
import math
import subprocess
from pathlib import Path

import pytest
import torch

from oracle import paged_oracle as P

ROOT = Path(__file__).resolve().parent.parent


def test_struct_layouts(built_lib, tmp_path):
    from heddle_b200 import _lib
    structs = {"hb_kv_cache": _lib.KvCache, "hb_kv_append_args": _lib.KvAppendArgs, "hb_fa_paged_args": _lib.FaPagedArgs}
    lines = [f'printf("%zu\\n", sizeof({name}));' for name in structs]
    lines += [f'printf("%zu\\n", offsetof({name}, {f}));' for name, cls in structs.items() for f, _ in cls._fields_]
    c = tmp_path / "t.c"
    c.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "heddle_b200.h"\nint main(void) {' + "\n".join(lines) + "return 0; }")
    subprocess.run(["gcc", "-std=c99", "-I", str(ROOT / "include"), str(c), "-o", str(tmp_path / "t")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout.split()]
    want = [ctypes.sizeof(cls) for cls in structs.values()] + [getattr(cls, f).offset for cls in structs.values() for f, _ in cls._fields_]
    assert got == want


def _cache(_lib, **over):
    c = _lib.KvCache(k=4096, v=4096, k_scale=4096, v_scale=4096, k_stride_p=8192, k_stride_h=1024, k_stride_s=128, v_stride_p=8192,
                     v_stride_h=1024, v_stride_s=128, num_pages=4, page_size=16, Hkv=2, D=128, page_table=4096, seq_lens=4096, starts=None,
                     table_stride=4, max_pages=4, B=2, T=2)
    for name, value in over.items():
        setattr(c, name, value)
    return c


def _append(_lib, cache=None, **over):
    a = _lib.KvAppendArgs(cache=_cache(_lib, **(cache or {})), k=4096, v=4096, k_stride_t=256, k_stride_h=128, v_stride_t=256, v_stride_h=128)
    for name, value in over.items():
        setattr(a, name, value)
    return a


def _attend(_lib, cache=None, **over):
    a = _lib.FaPagedArgs(cache=_cache(_lib, **(cache or {})), q=4096, o=4096, q_stride_t=512, q_stride_h=128, o_stride_t=512, o_stride_h=128, Hq=4)
    for name, value in over.items():
        setattr(a, name, value)
    return a


BAD_CACHE = [  # field, value, status
    (dict(D=96), "UNSUPPORTED"), (dict(page_size=24), "UNSUPPORTED"), (dict(page_size=0), "UNSUPPORTED"), (dict(Hkv=0), "BAD_ARG"),
    (dict(B=-1), "BAD_ARG"), (dict(T=-1), "BAD_ARG"), (dict(T=3), "BAD_ARG"), (dict(num_pages=-1), "BAD_ARG"), (dict(max_pages=-1), "BAD_ARG"),
    (dict(max_pages=1 << 28), "UNSUPPORTED"), (dict(k=None), "BAD_ARG"), (dict(v=None), "BAD_ARG"), (dict(k_scale=None), "BAD_ARG"),
    (dict(v_scale=None), "BAD_ARG"), (dict(page_table=None), "BAD_ARG"), (dict(seq_lens=None), "BAD_ARG"), (dict(k=4100), "ALIGN"),
    (dict(v_stride_s=120), "ALIGN"), (dict(k_stride_p=8), "ALIGN"), (dict(seq_lens=4098), "ALIGN"), (dict(starts=4097), "ALIGN"),
]


@pytest.mark.parametrize("fields,status", BAD_CACHE)
def test_bad_caches_are_refused(built_lib, fields, status):
    from heddle_b200 import _lib
    want = getattr(_lib, "HB_ERR_" + status)
    assert built_lib.hb_kv_append(ctypes.byref(_append(_lib, fields))) == want
    assert built_lib.hb_last_error().startswith(b"hb_kv_append: ")
    need = ctypes.c_uint64(7)
    assert built_lib.hb_fa_paged_workspace(ctypes.byref(_attend(_lib, fields)), ctypes.byref(need)) == want
    assert need.value == 0
    assert built_lib.hb_fa_paged(ctypes.byref(_attend(_lib, fields)), None, 0) == want
    assert built_lib.hb_last_error().startswith(b"hb_fa_paged: ")


def test_other_refusals(built_lib):
    from heddle_b200 import _lib
    append, attend = built_lib.hb_kv_append, lambda a: built_lib.hb_fa_paged(ctypes.byref(a), None, 0)
    assert append(None) == _lib.HB_ERR_BAD_ARG and built_lib.hb_fa_paged(None, None, 0) == _lib.HB_ERR_BAD_ARG
    assert built_lib.hb_fa_paged_workspace(ctypes.byref(_attend(_lib)), None) == _lib.HB_ERR_BAD_ARG
    assert built_lib.hb_cache_status(None) == _lib.HB_ERR_BAD_ARG
    for fields, status in ((dict(dtype=_lib.HB_FP8_E4M3), _lib.HB_ERR_UNSUPPORTED), (dict(rope_cos=4096), _lib.HB_ERR_BAD_ARG),
                           (dict(rope_cos=4096, rope_sin=4096, rope_len=-1), _lib.HB_ERR_BAD_ARG), (dict(q=4096, q_out=4096), _lib.HB_ERR_BAD_ARG),
                           (dict(k=None), _lib.HB_ERR_BAD_ARG), (dict(q=4096, Hq=4), _lib.HB_ERR_BAD_ARG), (dict(k=4104), _lib.HB_ERR_ALIGN),
                           (dict(v_stride_t=4), _lib.HB_ERR_ALIGN), (dict(q=4096, q_out=4100, Hq=4), _lib.HB_ERR_ALIGN)):
        assert append(ctypes.byref(_append(_lib, **fields))) == status, fields
    for fields, status in ((dict(dtype=_lib.HB_FP8_E4M3), _lib.HB_ERR_UNSUPPORTED), (dict(Hq=3), _lib.HB_ERR_BAD_ARG), (dict(Hq=0), _lib.HB_ERR_BAD_ARG),
                           (dict(q=None), _lib.HB_ERR_BAD_ARG), (dict(o=None), _lib.HB_ERR_BAD_ARG), (dict(o=4100), _lib.HB_ERR_ALIGN),
                           (dict(q_stride_h=4), _lib.HB_ERR_ALIGN), (dict(lse=4097), _lib.HB_ERR_ALIGN)):
        assert attend(_attend(_lib, **fields)) == status, fields
    assert attend(_attend(_lib, dict(T=1 << 30, B=1 << 30))) == _lib.HB_ERR_UNSUPPORTED  # T * Hq
    for empty in (dict(B=0, T=0), dict(T=0)):
        assert append(ctypes.byref(_append(_lib, empty))) == _lib.HB_OK and attend(_attend(_lib, empty)) == _lib.HB_OK


def test_tensors_are_checked(built_lib):
    from heddle_b200 import ops
    with pytest.raises(ValueError):
        ops.kv_pages(4, 24, 2, 128, device="cpu")
    with pytest.raises(ValueError):
        ops.kv_pages(4, 16, 2, 96, device="cpu")
    with pytest.raises(ValueError):
        ops.kv_pages(4, 16, 2, 64, layout="sbhd", device="cpu")
    pages = ops.kv_pages(4, 16, 2, 64, layout="bshd", device="cpu")
    assert pages.k.shape == (4, 16, 2, 64) and pages.k.dtype is torch.float8_e4m3fn and pages.k_scale.shape == (4, 2)
    x, table, lens = torch.zeros(2, 2, 64, dtype=torch.bfloat16), torch.zeros(2, 4, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.kv_append(x, x, pages, table, lens)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.fa_paged(x, pages, table, lens)
    # the checks of the tensors themselves, which do not ask for a device
    good = dict(pages=pages, page_table=table, seq_lens=lens, starts=None, x=x)
    assert ops._kv_cache("t", **good).Hkv == 2
    for bad, error in ((dict(pages=pages._replace(layout="sbhd")), ValueError), (dict(pages=pages._replace(v=pages.v[:, :8])), ValueError),
                       (dict(pages=pages._replace(k=pages.k.view(torch.uint8))), TypeError), (dict(page_table=table.long()), ValueError),
                       (dict(page_table=table[0]), ValueError), (dict(page_table=table.t().contiguous().t()), ValueError),
                       (dict(seq_lens=lens.long()), ValueError), (dict(seq_lens=lens[:1]), ValueError), (dict(starts=lens), ValueError),
                       (dict(pages=pages._replace(k_scale=pages.k_scale.double())), ValueError),
                       (dict(pages=pages._replace(v_scale=pages.v_scale[:, :1])), ValueError), (dict(x=x[..., :32]), ValueError),
                       (dict(x=x[0]), ValueError)):
        with pytest.raises(error):
            ops._kv_cache("t", **{**good, **bad})


def test_oracle_rounds_as_torch_does():
    x = torch.cat([torch.linspace(-448, 448, 20001, dtype=torch.float64), torch.linspace(-0.05, 0.05, 20001, dtype=torch.float64)])
    assert torch.equal(P.e4m3(x), x.float().double().to(torch.float8_e4m3fn).double()) or \
        (P.e4m3(x) != x.to(torch.float32).to(torch.float8_e4m3fn).double()).sum() == 0
    for largest in (1e-40, 2.0 ** -91, 1.0, 448.0, 448.0000001, 224.0, 1e30, 3.4e38):
        s = P.scale_of(largest)
        assert math.log2(s) == int(math.log2(s)) and (largest <= 448 * s or s == 2.0 ** 119) and (largest > 224 * s or s == 2.0 ** -100)
