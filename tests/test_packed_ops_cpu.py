"""CPU checks of the packed-batch operators: the ctypes structs have the C layouts, and every refusal
comes before any device work, with its status and its name in the message."""
from __future__ import annotations

import ctypes
import subprocess

import pytest
import torch

from conftest import REPO


def test_descriptor_layouts_match_c(tmp_path):
    import b2g

    lines = []
    for name, cls in (("b2g_qk_norm_rope_desc", b2g.QkNormRopeDesc),
                      ("b2g_attention_packed_desc", b2g.AttentionPackedDesc)):
        lines.append(f'  printf("%zu\\n", sizeof({name}));')
        lines += [f'  printf("%zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "b2g.h"\nint main(void){\n' + "\n".join(lines) +
                   "\n  return 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["/usr/bin/gcc", "-I", str(REPO / "include"), "-I", "/usr/local/cuda/include", str(src), "-o",
                    str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for cls in (b2g.QkNormRopeDesc, b2g.AttentionPackedDesc):
        want.append(ctypes.sizeof(cls))
        want += [getattr(cls, f[0]).offset for f in cls._fields_]
    assert got == want


def refused(lib, status, code, word):
    assert status == code and word in lib.b2g_last_error().decode()


def test_quantize_s8_refusals():
    import b2g

    lib = b2g.load()
    f = lib.b2g_quantize_s8
    refused(lib, f(16, b2g.F32, -1, 8, 8, 16, 8, 16, None), 1, "negative")
    refused(lib, f(None, b2g.F32, 1, 8, 8, 16, 8, 16, None), 1, "null")
    refused(lib, f(16, b2g.F32, 2, 8, 7, 16, 8, 16, None), 1, "ld < cols")
    refused(lib, f(16, b2g.S8, 2, 8, 8, 16, 8, 16, None), 2, "F32, BF16 or F16")
    assert f(None, b2g.F32, 0, 8, 8, None, 8, None, None) == 0


def s8_desc(**kw):
    import b2g

    d = b2g.GemmDesc(M=4, N=8, K=32, a=256, a_dtype=b2g.S8, lda=32, b=256, b_dtype=b2g.S8, ldb=32, bias=None,
                     bias_dtype=b2g.F32, d=256, d_dtype=b2g.F32, ldd=8, epilogue=b2g.EPI_NONE, gate=None)
    for k, v in kw.items():
        setattr(d, k, v)
    return ctypes.byref(d)


def test_gemm_s8_refusals():
    import b2g

    lib = b2g.load()
    f = lib.b2g_gemm_s8
    refused(lib, f(None, 256, 256, None, 0, None), 1, "null")
    for kw, code, word in ((dict(M=-1), 1, "negative"), (dict(b_dtype=b2g.BF16), 2, "weights must be S8"),
                           (dict(a_dtype=b2g.E4M3), 2, "activations"), (dict(lda=31), 1, "lda/ldb"),
                           (dict(ldd=7), 1, "ldd"), (dict(a=None), 1, "null"), (dict(K=0), 2, "K must be"),
                           (dict(K=131072, lda=131072, ldb=131072), 2, "K must be"),
                           (dict(epilogue=9), 2, "epilogue"), (dict(epilogue=b2g.EPI_GATED_RESIDUAL), 1, "gate"),
                           (dict(d_dtype=b2g.S8), 2, "S8")):
        refused(lib, f(s8_desc(**kw), 256, 256, None, 0, None), code, word)
    refused(lib, f(s8_desc(), None, 256, None, 0, None), 1, "scales")
    refused(lib, f(s8_desc(), 256, None, None, 0, None), 1, "scales")
    assert f(s8_desc(M=0), None, None, None, 0, None) == 0
    assert lib.b2g_gemm_s8_workspace(3, 17, b2g.S8) == 0
    assert lib.b2g_gemm_s8_workspace(3, 17, b2g.BF16) >= 3 * 32 + 12
    refused(lib, lib.b2g_gemm(s8_desc(), None), 2, "b2g_gemm_s8")


def rope_desc(**kw):
    import b2g

    d = b2g.QkNormRopeDesc(q=256, k=256, dtype=b2g.BF16, q_out=256, k_out=256, out_dtype=b2g.BF16, ldq=256, hsq=128,
                           ldk=256, hsk=128, ldq_out=256, hsq_out=128, ldk_out=256, hsk_out=128, tokens=4, n_head=2,
                           n_kv_head=2, d_head=128, q_norm=None, k_norm=None, eps=1e-6, positions=256, ldp=3, n_axes=3,
                           axis_dim=(ctypes.c_int * 4)(16, 56, 56, 0), theta=10000.0, interleaved=1)
    for k, v in kw.items():
        setattr(d, k, (ctypes.c_int * 4)(*v) if k == "axis_dim" else v)
    return ctypes.byref(d)


def test_qk_norm_rope_refusals():
    import b2g

    lib = b2g.load()
    f = lib.b2g_qk_norm_rope
    refused(lib, f(None, None), 1, "null")
    for kw, code, word in ((dict(tokens=-1), 1, "negative"), (dict(d_head=127), 2, "d_head"), (dict(d_head=258), 2, "d_head"),
                           (dict(dtype=b2g.S8), 2, "inputs"), (dict(q=None), 1, "null"), (dict(k_out=None), 1, "null"),
                           (dict(n_axes=5), 1, "axes"), (dict(positions=None), 1, "axes"), (dict(ldp=2), 1, "axes"),
                           (dict(axis_dim=(16, 56, 58, 0)), 1, "axis widths"), (dict(axis_dim=(15, 56, 56, 0)), 1, "axis widths"),
                           (dict(theta=0.0), 1, "theta"), (dict(theta=float("nan")), 1, "theta"), (dict(eps=-1.0), 1, "eps")):
        refused(lib, f(rope_desc(**kw), None), code, word)
    assert f(rope_desc(tokens=0), None) == 0


def attn_desc(**kw):
    import b2g

    d = b2g.AttentionPackedDesc(q=256, k=256, v=256, out=256, dtype=b2g.BF16, ldq=256, hsq=128, ldk=256, hsk=128, ldv=256,
                                hsv=128, ldo=256, hso=128, total_q=8, total_k=8, batch=2, cu_q=256, cu_k=256, k_lens=None,
                                n_head=2, n_kv_head=2, d_head=128, scale=0.1, causal=0)
    for k, v in kw.items():
        setattr(d, k, v)
    return ctypes.byref(d)


def test_attention_packed_refusals():
    import b2g

    lib = b2g.load()
    f = lib.b2g_attention_packed
    refused(lib, f(None, None, 0, None), 1, "null")
    for kw, code, word in ((dict(batch=-1), 1, "negative"), (dict(dtype=b2g.F32), 2, "BF16 or F16"),
                           (dict(d_head=96), 2, "head dim"), (dict(n_head=3), 1, "multiple"), (dict(n_kv_head=0), 1, "multiple"),
                           (dict(scale=0.0), 1, "scale"), (dict(scale=float("inf")), 1, "scale"),
                           (dict(scale=float("nan")), 1, "scale"), (dict(total_k=2 ** 30 + 1), 2, "size"),
                           (dict(q=None), 1, "null"), (dict(cu_k=None), 1, "null"), (dict(ldq=127), 1, "stride"),
                           (dict(hsk=0), 1, "stride"), (dict(ldv=260), 2, "strides"), (dict(out=264), 2, "aligned")):
        refused(lib, f(attn_desc(**kw), None, 0, None), code, word)
    assert f(attn_desc(batch=0), None, 0, None) == 0 and f(attn_desc(total_q=0), None, 0, None) == 0


def test_python_refusals():
    """The wrappers check shapes and types before they touch the library."""
    import b2g

    x, w, s = torch.zeros(4, 32), torch.zeros(8, 32, dtype=torch.int8), torch.ones(8)
    with pytest.raises(b2g.B2GError, match="K mismatch"):
        b2g.gemm_s8(x[:, :16], w, s)
    with pytest.raises(b2g.B2GError, match="int8 wq"):
        b2g.gemm_s8(x, w.float(), s)
    with pytest.raises(b2g.B2GError, match="unit stride"):
        b2g.gemm_s8(torch.zeros(32, 4).T, w, s)
    with pytest.raises(b2g.B2GError, match="epilogue"):
        b2g.gemm_s8(x, w, s, epilogue="relu")
    with pytest.raises(b2g.B2GError, match="w_scale"):
        b2g.gemm_s8(x, w, s[:7], out=torch.zeros(4, 8))
    with pytest.raises(b2g.B2GError, match="quantize_s8"):
        b2g.quantize_s8(torch.zeros(3, dtype=torch.float32))
    q = torch.zeros(6, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(b2g.B2GError, match="positions"):
        b2g.qk_norm_rope(q, q, torch.zeros(6, 2), [16, 24, 24])
    with pytest.raises(b2g.B2GError, match="same tokens"):
        b2g.qk_norm_rope(q, q[:5], torch.zeros(6, 1), [64])
    cu = torch.tensor([0, 6], dtype=torch.int32)
    with pytest.raises(b2g.B2GError, match="int32"):
        b2g.attention_packed(q, q, q, cu.long())
    with pytest.raises(b2g.B2GError, match="one head width"):
        b2g.attention_packed(q, q, q.float(), cu)
    with pytest.raises(b2g.B2GError, match="k_lens"):
        b2g.attention_packed(q, q, q, cu, k_lens=cu)
