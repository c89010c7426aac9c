"""Stand-alone operators without a GPU: the Python descriptors have the C layout, and
calls that break a rule are refused before anything touches a device."""
import ctypes
import os
import subprocess

import pytest

import pkt_b200
from pkt_b200 import _lib

HEADER = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "include", "pkt_b200.h")
STRUCTS = {"pkt_layernorm_desc": _lib.LayerNormDesc, "pkt_fp8_quantize_desc": _lib.Fp8QuantizeDesc,
           "pkt_fp8_gemm_desc": _lib.Fp8GemmDesc, "pkt_adamw_tensor": _lib.AdamWTensor, "pkt_adamw_config": _lib.AdamWConfig}
BF16, F32, E4M3 = pkt_b200.DTYPE_BF16, pkt_b200.DTYPE_F32, pkt_b200.DTYPE_E4M3
P = 1 << 20  # an aligned address; never read, every call here fails first


def test_descriptors_have_the_c_layout(tmp_path):
    lines = []
    for name, cls in STRUCTS.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stdio.h>\n#include "{HEADER}"\nint main(void) {{\n' + "\n".join(lines) + "\nreturn 0; }\n")
    exe = tmp_path / "layout"
    subprocess.check_call(["gcc", "-o", str(exe), str(src)])
    got = dict(line.split() for line in subprocess.check_output([str(exe)], text=True).splitlines())
    for name, cls in STRUCTS.items():
        assert int(got[name]) == ctypes.sizeof(cls), name
        for f, _ in cls._fields_:
            assert int(got[f"{name}.{f}"]) == getattr(cls, f).offset, (name, f)


def refused(call, *words):
    with pytest.raises(pkt_b200.PktError) as e:
        call()
    assert e.value.code == _lib.PKT_ERR_ARGS, e.value
    for w in words:
        assert w in str(e.value), e.value


def ln(**kw):
    base = dict(rows=4, cols=64, dtype=BF16, param_dtype=F32, eps=1e-5, x=P, ldx=64, gamma=P, beta=P, y=P, ldy=64, mean=P,
                rstd=P, dy=P, lddy=64, dx=P, lddx=64, dgamma=P, dbeta=P, workspace=P, workspace_bytes=1 << 30)
    return pkt_b200.LayerNormDesc(**{**base, **kw})


@pytest.mark.parametrize("kw,word", [(dict(rows=-1), "rows"), (dict(cols=0), "columns"), (dict(dtype=E4M3), "dtype"),
                                     (dict(param_dtype=0), "param_dtype"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
                                     (dict(x=None), "x"), (dict(y=None), "y"), (dict(ldx=63), "stride"), (dict(ldy=63), "stride"),
                                     (dict(x=P + 1), "aligned"), (dict(gamma=P + 2), "gamma"), (dict(mean=P + 2), "mean")])
def test_layernorm_forward_refuses(kw, word):
    refused(lambda: pkt_b200.layernorm_forward(ln(**kw)), word)


@pytest.mark.parametrize("kw,word", [(dict(rows=-1), "rows"), (dict(dy=None), "dy"), (dict(x=None), "x"), (dict(lddy=8), "stride"),
                                     (dict(lddx=8), "stride"), (dict(mean=None), "mean"), (dict(rstd=None), "rstd"),
                                     (dict(dgamma=P + 1), "dgamma"), (dict(workspace=P + 1), "workspace")])
def test_layernorm_backward_refuses(kw, word):
    refused(lambda: pkt_b200.layernorm_backward(ln(**kw)), word)


def quant(**kw):
    base = dict(rows=4, cols=256, dtype=BF16, q_dtype=E4M3, block_rows=1, x=P, ldx=256, q=P, ldq=256, scale=P, ld_scale=4,
                qt=P, ldqt=16, scale_t=P, ld_scale_t=256)
    return pkt_b200.Fp8QuantizeDesc(**{**base, **kw})


@pytest.mark.parametrize("kw,word", [(dict(rows=-1), "-1"), (dict(dtype=E4M3), "dtype"), (dict(q_dtype=BF16), "q_dtype"),
                                     (dict(block_rows=64), "block_rows"), (dict(q=None, qt=None), "q or qt"), (dict(x=None), "x"),
                                     (dict(ldx=255), "stride"), (dict(q=P + 8), "16-byte"), (dict(ldq=264), "16"), (dict(ldq=240), "below"),
                                     (dict(scale=None), "scales"), (dict(ld_scale=3), "scales"), (dict(ldqt=0), "below"),
                                     (dict(qt=P + 4), "16-byte"), (dict(scale_t=None), "scales"), (dict(ld_scale_t=255), "scales")])
def test_quantize_refuses(kw, word):
    refused(lambda: pkt_b200.fp8_quantize(quant(**kw)), word)


def gemm(**kw):
    base = dict(M=8, N=16, K=256, a_dtype=E4M3, b_dtype=E4M3, a=P, lda=256, scale_a=P, ld_scale_a=8, a_block_rows=1, b=P, ldb=256,
                scale_b=P, ld_scale_b=1, b_block_rows=128, out=P, ldo=16, out_dtype=BF16)
    return pkt_b200.Fp8GemmDesc(**{**base, **kw})


@pytest.mark.parametrize("kw,word", [(dict(M=-1), "M=-1"), (dict(a_dtype=BF16), "a_dtype"), (dict(b_dtype=0), "b_dtype"),
                                     (dict(out_dtype=E4M3), "out_dtype"), (dict(a=P + 8), "16-byte"), (dict(lda=264), "16"),
                                     (dict(lda=240), "below"), (dict(b=None), "b "), (dict(scale_a=None), "scales"),
                                     (dict(ld_scale_a=7), "scale_a"), (dict(ld_scale_b=0), "scale_b"), (dict(a_block_rows=2), "block_rows"),
                                     (dict(b_block_rows=0), "block_rows"), (dict(out=None), "out"), (dict(ldo=15), "stride"),
                                     (dict(out=P + 1), "aligned")])
def test_gemm_refuses(kw, word):
    refused(lambda: pkt_b200.fp8_gemm(gemm(**kw)), word)


def test_null_arguments():
    L = _lib.load()
    for f in ("pkt_layernorm_forward", "pkt_layernorm_backward", "pkt_fp8_quantize", "pkt_fp8_gemm"):
        assert getattr(L, f)(None, None) == _lib.PKT_ERR_ARGS
    assert L.pkt_layernorm_backward_workspace(ln(), None) == _lib.PKT_ERR_ARGS
    assert L.pkt_ops_status(None) == _lib.PKT_ERR_ARGS
    assert L.pkt_adamw_create(0, None, None) == _lib.PKT_ERR_ARGS
    assert L.pkt_adamw_step(None, 1.0, 1.0, None, None) == _lib.PKT_ERR_ARGS
    assert L.pkt_adamw_set_grads(None, None, None) == _lib.PKT_ERR_ARGS
    assert L.pkt_adamw_set_step(None, 0, None) == _lib.PKT_ERR_ARGS
    assert L.pkt_adamw_get_step(None, None, None) == _lib.PKT_ERR_ARGS
    assert L.pkt_adamw_destroy(None) == _lib.PKT_OK


def test_empty_problems_need_no_memory():
    """Nothing to do: no pointer is looked at."""
    pkt_b200.layernorm_forward(ln(rows=0, x=None, y=None))
    pkt_b200.fp8_quantize(quant(rows=0))
    pkt_b200.fp8_quantize(quant(cols=0))
    pkt_b200.fp8_gemm(gemm(M=0))
    pkt_b200.fp8_gemm(gemm(N=0))


@pytest.mark.parametrize("kw", [dict(rows=2**31 - 1), dict(cols=2**31 - 100, ldx=2**31)])
def test_quantize_of_more_than_it_can_count(kw):
    with pytest.raises(pkt_b200.PktError, match="quantize of"):
        pkt_b200.fp8_quantize(quant(**kw))


@pytest.mark.parametrize("kw", [dict(M=2**31 - 1, ld_scale_a=2**31), dict(N=2**31 - 100, ldo=2**31, ld_scale_b=2**31)])
def test_gemm_of_more_than_it_can_count(kw):
    with pytest.raises(pkt_b200.PktError, match="fp8 gemm of"):
        pkt_b200.fp8_gemm(gemm(**kw))
