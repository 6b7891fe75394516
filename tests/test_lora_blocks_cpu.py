"""CPU checks of the adapters and of attention over chosen blocks: layouts of the descriptors, and refusals, which come
before any device work, with their status and their name in the message."""
from __future__ import annotations

import ctypes
import subprocess

import pytest
import torch

from conftest import REPO


def test_lora_descriptor_layout_matches_c(tmp_path):
    import b2g

    fields = [f[0] for f in b2g.LoraDesc._fields_]
    lines = ['  printf("%zu\\n", sizeof(b2g_lora_desc));'] + [f'  printf("%zu\\n", offsetof(b2g_lora_desc, {f}));' for f in fields]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "b2g.h"\nint main(void){\n' + "\n".join(lines) + "\n  return 0;\n}\n")
    subprocess.run(["/usr/bin/gcc", "-I", str(REPO / "include"), "-I", "/usr/local/cuda/include", str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(b2g.LoraDesc)] + [getattr(b2g.LoraDesc, f).offset for f in fields]


def refused(lib, status, code, word):
    assert status == code and word in lib.b2g_last_error().decode(), (status, lib.b2g_last_error())


def lora_desc(**kw):
    import b2g

    d = b2g.LoraDesc(x=256, a=256, b=256, dtype=b2g.BF16, ldx=64, lda=64, a_stride=1024, ldb=16, b_stride=512, t=256, ldt=16, y=256,
                     out=256, y_dtype=b2g.BF16, ldy=32, ldo=32, rows=4, K=64, N=32, R=16, adapters=2, batch=2, cu=256, ids=None,
                     scale=None, gate=None, epilogue=b2g.EPI_NONE)
    for k, v in kw.items():
        setattr(d, k, v)
    return ctypes.byref(d)


BOTH = ((dict(rows=-1), 1, "negative"), (dict(dtype=7), 2, "BF16 or F16"), (dict(R=12), 2, "rank"), (dict(R=0), 2, "rank"),
        (dict(R=136), 2, "rank"), (dict(batch=65537), 2, "size"), (dict(cu=None), 1, "null"), (dict(t=None), 1, "null"),
        (dict(ldt=8), 1, "stride"), (dict(t=260), 2, "aligned"), (dict(ldt=18), 2, "aligned"))


def test_lora_down_refusals():
    import b2g

    lib = b2g.load()
    f = lib.b2g_lora_down
    refused(lib, f(None, None), 1, "b2g_lora_down: null")
    for kw, code, word in (*BOTH, (dict(K=60), 2, "K must"), (dict(K=0), 2, "K must"), (dict(x=None), 1, "null"), (dict(a=None), 1, "null"),
                           (dict(ldx=56), 1, "stride"), (dict(ldx=68), 2, "aligned"), (dict(a=264), 2, "aligned"),
                           (dict(lda=56), 1, "stride"), (dict(a_stride=1028), 2, "aligned")):
        refused(lib, f(lora_desc(**kw), None), code, word)
    assert f(lora_desc(rows=0, x=None, t=None), None) == 0 and f(lora_desc(batch=0, cu=None), None) == 0


def test_lora_up_refusals():
    import b2g

    lib = b2g.load()
    f = lib.b2g_lora_up
    refused(lib, f(None, None), 1, "b2g_lora_up: null")
    for kw, code, word in (*BOTH, (dict(y=None), 1, "null"), (dict(b=None), 1, "null"), (dict(out=None), 1, "null"),
                           (dict(y_dtype=b2g.F16), 2, "y must be"), (dict(epilogue=9), 2, "epilogue"),
                           (dict(epilogue=b2g.EPI_GATED_RESIDUAL), 1, "gate"), (dict(ldy=31), 1, "stride"),
                           (dict(ldo=31), 1, "stride"), (dict(ldb=8), 1, "stride"), (dict(ldb=20), 2, "aligned"), (dict(b=258), 2, "aligned"),
                           (dict(rows=2 ** 30, N=2 ** 20, ldy=2 ** 20, ldo=2 ** 20), 2, "size")):
        refused(lib, f(lora_desc(**kw), None), code, word)
    assert f(lora_desc(N=0, y=None, out=None, b=None), None) == 0 and f(lora_desc(rows=0), None) == 0


def packed(**kw):
    import b2g

    d = b2g.AttentionPackedDesc(q=256, k=256, v=256, out=256, dtype=b2g.BF16, ldq=256, hsq=128, ldk=256, hsk=128, ldv=256,
                                hsv=128, ldo=256, hso=128, total_q=8, total_k=8, batch=2, cu_q=256, cu_k=256, k_lens=None,
                                n_head=2, n_kv_head=2, d_head=128, scale=0.1, causal=0)
    for k, v in kw.items():
        setattr(d, k, v)
    return ctypes.byref(d)


def test_block_means_refusals():
    import b2g

    lib = b2g.load()
    f = lib.b2g_block_means
    refused(lib, f(None, None, 256, 3, None), 1, "b2g_block_means: null")
    for kw, code, word in ((dict(batch=-1), 1, "negative"), (dict(dtype=b2g.F32), 2, "BF16 or F16"), (dict(d_head=96), 2, "head dim"),
                           (dict(total_k=2 ** 30 + 1), 2, "size"), (dict(k=None), 1, "null"), (dict(cu_k=None), 1, "null"),
                           (dict(ldk=127), 1, "stride"), (dict(hsk=0), 1, "stride"), (dict(ldk=260), 2, "strides"),
                           (dict(k=264), 2, "aligned")):
        refused(lib, f(packed(**kw), None, 256, 3, None), code, word)
    refused(lib, f(packed(), None, 256, -1, None), 1, "negative")
    refused(lib, f(packed(), None, None, 3, None), 1, "null")
    refused(lib, f(packed(), None, 260, 3, None), 2, "aligned")
    assert f(packed(), None, None, 0, None) == 0 and f(packed(q=None, v=None, out=None, n_kv_head=0), None, 256, 3, None) == 0


def test_select_blocks_refusals():
    import b2g

    lib = b2g.load()
    f = lib.b2g_select_blocks
    refused(lib, f(None, 256, 3, 1, 0, 0, 256, 2, 1, None), 1, "b2g_select_blocks: null")
    for kw, code, word in ((dict(total_q=-1), 1, "negative"), (dict(n_head=3), 1, "multiple"), (dict(n_kv_head=0), 1, "multiple"),
                           (dict(q=None), 1, "null"), (dict(cu_q=None), 1, "null"), (dict(ldq=100), 1, "stride"),
                           (dict(hsq=132), 2, "strides"), (dict(q=257), 2, "aligned")):
        refused(lib, f(packed(**kw), 256, 3, 1, 0, 0, 256, 2, 1, None), code, word)
    for i, (code, word) in enumerate([(1, "negative")] * 4):
        args = [3, 1, 0, 0]
        args[i] = -1
        refused(lib, f(packed(), 256, *args, 256, 2, 1, None), code, word)
    refused(lib, f(packed(), None, 3, 1, 0, 0, 256, 2, 1, None), 1, "null")
    refused(lib, f(packed(), 256, 3, 1, 0, 0, None, 2, 1, None), 1, "null")
    refused(lib, f(packed(), 256, 3, 1, 0, 0, 256, 2, 257, None), 2, "2^20 keys")
    refused(lib, f(packed(), 260, 3, 1, 0, 0, 256, 2, 1, None), 2, "aligned")
    assert f(packed(), 256, 3, 1, 0, 0, 256, 0, 1, None) == 0


def test_attention_blocks_refusals():
    import b2g

    lib = b2g.load()
    f = lib.b2g_attention_blocks
    refused(lib, f(None, 256, 2, 1, None, 0, None), 1, "b2g_attention_blocks: null")
    for kw, code, word in ((dict(batch=-1), 1, "negative"), (dict(dtype=b2g.F32), 2, "BF16 or F16"), (dict(d_head=96), 2, "head dim"),
                           (dict(n_head=3), 1, "multiple"), (dict(scale=0.0), 1, "scale"), (dict(scale=float("nan")), 1, "scale"),
                           (dict(q=None), 1, "null"), (dict(v=None), 1, "null"), (dict(cu_k=None), 1, "null"),
                           (dict(ldv=260), 2, "strides"), (dict(out=264), 2, "aligned")):
        refused(lib, f(packed(**kw), 256, 2, 1, None, 0, None), code, word)
    refused(lib, f(packed(), 256, -2, 1, None, 0, None), 1, "negative")
    refused(lib, f(packed(), None, 2, 1, None, 0, None), 1, "null")
    refused(lib, f(packed(), 258, 2, 1, None, 0, None), 2, "aligned")
    assert f(packed(batch=0), 256, 2, 1, None, 0, None) == 0 and f(packed(total_q=0), None, 0, 0, None, 0, None) == 0


def test_python_refusals():
    """The wrappers check shapes and types before they touch the library."""
    import b2g

    half = dict(dtype=torch.bfloat16)
    x, a, b, y = torch.zeros(6, 64, **half), torch.zeros(2, 16, 64, **half), torch.zeros(2, 32, 16, **half), torch.zeros(6, 32, **half)
    cu, ids = torch.tensor([0, 4, 6], dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for args, kw, word in (((x[:, :56], a, b, y, cu), {}, "K mismatch"), ((x.float(), a, b, y, cu), {}, "BF16 or F16"),
                           ((x, a.half(), b, y, cu), {}, "of one type"), ((x, a, b[:1], y, cu), {}, "as many adapters"),
                           ((x, a, b[:, :, :8], y, cu), {}, "b must be"), ((x, a, b, y[:, :31], cu), {}, "y must be"),
                           ((x, a, b, y.half(), cu), {}, "y must be F32"), ((x, a, b, y, cu.long()), {}, "int32"),
                           ((x, a, b, y, cu), dict(ids=ids[:1]), "ids"), ((x, a, b, y, cu), dict(scale=torch.ones(3)), "scale"),
                           ((x, a, b, y, cu), dict(epilogue="relu"), "epilogue"), ((x, a, b, y, cu), dict(epilogue="gated_residual"), "gate"),
                           ((x, a, b, y, cu), dict(out=y.float()), "out must be"), ((x, a, b, y, cu), {}, "CUDA")):
        with pytest.raises(b2g.B2GError, match=word):
            b2g.lora(*args, **kw)
    with pytest.raises(b2g.B2GError, match="lora_down: out"):
        b2g.lora_down(x, a, cu, out=torch.zeros(6, 8))
    with pytest.raises(b2g.B2GError, match="lora_up: t must be"):
        b2g.lora_up(torch.zeros(6, 16, **half), b, y, cu)
    q, means = torch.zeros(6, 4, 64, **half), torch.zeros(2, 2, 64)
    k, chosen = torch.zeros(6, 2, 64, **half), torch.zeros(2, 2, 1, dtype=torch.int32)
    with pytest.raises(b2g.B2GError, match="block_means: k must"):
        b2g.block_means(k.float(), cu)
    with pytest.raises(b2g.B2GError, match="since needs"):
        b2g.block_means(k, cu, since=ids)
    with pytest.raises(b2g.B2GError, match="out must be"):
        b2g.block_means(k, cu, out=means.half())
    with pytest.raises(b2g.B2GError, match="means must be"):
        b2g.select_blocks(q, means.half(), cu, 3)
    with pytest.raises(b2g.B2GError, match="top must not"):
        b2g.select_blocks(q, means, cu, -1)
    with pytest.raises(b2g.B2GError, match="max_k must not"):
        b2g.select_blocks(q, means, cu, 1, max_k=-1)
    with pytest.raises(b2g.B2GError, match="chosen must be"):
        b2g.attention_blocks(q, k, k, chosen[:, :1], cu)
    with pytest.raises(b2g.B2GError, match="one head width"):
        b2g.attention_blocks(q, k, k.half(), chosen, cu)
