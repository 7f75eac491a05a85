"""Host-side checks of the decode step's operators (no GPU needed): what they
refuse, before any device work."""

from __future__ import annotations

import pytest
import torch

import fpv2


def _attention_args(**change):
    args = dict(q=torch.zeros(2, 8, 64, dtype=torch.bfloat16),
                k_pages=torch.zeros(6, 2, 16, 64, dtype=torch.bfloat16),
                v_pages=torch.zeros(6, 2, 16, 64, dtype=torch.bfloat16),
                page_table=torch.zeros(2, 3, dtype=torch.int32),
                lengths=torch.ones(2, dtype=torch.int32))
    args.update(change)
    return args


@pytest.mark.parametrize("change,message", [
    (dict(q=torch.zeros(8, 64, dtype=torch.bfloat16)), "q must have shape"),
    (dict(q=torch.zeros(2, 7, 64, dtype=torch.bfloat16)), "divisible by KV heads"),
    (dict(q=torch.zeros(2, 8, 64)), "share float16 or bfloat16"),
    (dict(q=torch.zeros(2, 8, 80, dtype=torch.bfloat16)), "head dimension"),
    (dict(q=torch.zeros(2, 8, 128, dtype=torch.bfloat16)), "head dimension"),
    (dict(k_pages=torch.zeros(2, 16, 64, dtype=torch.bfloat16)), "k_pages must have shape"),
    (dict(v_pages=torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16)), "same shape"),
    (dict(v_pages=torch.zeros(6, 2, 16, 64, dtype=torch.float16)), "share float16 or bfloat16"),
    (dict(k_pages=torch.zeros(6, 2, 16, 65, dtype=torch.bfloat16)[..., 1:]), "16-byte aligned"),
    (dict(page_table=torch.zeros(2, 3, dtype=torch.int64)), "page_table must be int32"),
    (dict(page_table=torch.zeros(3, 3, dtype=torch.int32)), "page_table must be int32"),
    (dict(page_table=torch.zeros(3, 2, dtype=torch.int32).T), "contiguous rows"),
    (dict(page_table=torch.zeros(2, 0, dtype=torch.int32)), "at least one page"),
    (dict(page_table=None, k_pages=torch.zeros(1, 2, 16, 64, dtype=torch.bfloat16),
          v_pages=torch.zeros(1, 2, 16, 64, dtype=torch.bfloat16)), "every sequence needs a page"),
    (dict(lengths=torch.ones(2, dtype=torch.int64)), "lengths must be"),
    (dict(lengths=torch.ones(3, dtype=torch.int32)), "lengths must be"),
    (dict(lengths=-1), "lengths must be"),
    (dict(window_tokens=0), "window_tokens"),
    (dict(window_tokens=1.5), "window_tokens"),
    (dict(sink_tokens=-1), "sink_tokens"),
    (dict(out=torch.zeros(2, 8, 64)), "out must be"),
    (dict(out=torch.zeros(2, 64, 8, dtype=torch.bfloat16).transpose(1, 2)), "out must be"),
])
def test_decode_attention_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        fpv2.decode_attention(**_attention_args(**change))


def test_decode_attention_refuses_cpu_tensors_and_gradients():
    with pytest.raises(RuntimeError, match="ROCm"):
        fpv2.decode_attention(**_attention_args())
    q = torch.zeros(2, 8, 64, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward"):
        fpv2.decode_attention(**_attention_args(q=q))


@pytest.mark.parametrize("cname,mirror", [("fpv2_decode_params", "DecodeParams"),
                                          ("fpv2_rope_pages_params", "RopePagesParams"),
                                          ("fpv2_sample_params", "SampleParams")])
def test_params_layouts_match_the_header(tmp_path, cname, mirror):
    """The ctypes mirrors, as gcc lays the header's structs out."""
    import ctypes
    import shutil
    import subprocess
    from pathlib import Path

    from fpv2 import _lib
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    cls = getattr(_lib, mirror)
    lines = ['#include <stddef.h>', '#include <stdio.h>', '#include "fpv2_decode.h"',
             "int main(void) {", f'  printf("%zu\\n", sizeof({cname}));']
    lines += [f'  printf("%zu\\n", offsetof({cname}, {name}));' for name, _ in cls._fields_]
    source, program = tmp_path / "layout.c", tmp_path / "layout"
    source.write_text("\n".join(lines + ["  return 0;", "}"]))
    include = Path(__file__).resolve().parents[1] / "include"
    subprocess.run([gcc, "-I", str(include), str(source), "-o", str(program)], check=True)
    got = [int(x) for x in subprocess.run([str(program)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    assert got == [ctypes.sizeof(cls)] + [getattr(cls, name).offset for name, _ in cls._fields_]


def _rope_args(**change):
    bf16 = torch.bfloat16
    args = dict(qkv=torch.zeros(3, 6 * 64, dtype=bf16), q_weight=torch.ones(64, dtype=bf16),
                k_weight=torch.ones(64, dtype=bf16), cos=torch.zeros(9, 32), sin=torch.zeros(9, 32),
                positions=torch.zeros(3, dtype=torch.int64), slots=torch.arange(3),
                k_pages=torch.zeros(2, 1, 16, 64, dtype=bf16),
                v_pages=torch.zeros(2, 1, 16, 64, dtype=bf16), query_heads=4)
    args.update(change)
    return args


@pytest.mark.parametrize("change,message", [
    (dict(qkv=torch.zeros(3, 6 * 64)), "qkv must be"),
    (dict(qkv=torch.zeros(3, 6, 64, dtype=torch.bfloat16)), "qkv must be"),
    (dict(qkv=torch.zeros(3, 7 * 64, dtype=torch.bfloat16)), "qkv rows must hold"),
    (dict(qkv=torch.zeros(3, 6 * 64, dtype=torch.float16)), "share a dtype"),
    (dict(query_heads=0), "query_heads"),
    (dict(query_heads=True), "query_heads"),
    (dict(q_weight=torch.ones(64)), "q_weight must be"),
    (dict(k_weight=torch.ones(32, dtype=torch.bfloat16)), "k_weight must be"),
    (dict(cos=torch.zeros(9, 32, dtype=torch.float64)), "cos must be"),
    (dict(sin=torch.zeros(8, 32)), "sin must be"),
    (dict(cos=torch.zeros(9, 28), sin=torch.zeros(9, 28)), "multiple of 8 angles"),
    (dict(cos=torch.zeros(9, 40), sin=torch.zeros(9, 40)), "half the head dimension"),
    (dict(cos=torch.zeros(0, 32), sin=torch.zeros(0, 32)), "cos and sin"),
    (dict(positions=torch.zeros(2, dtype=torch.int64)), "positions must be"),
    (dict(positions=torch.zeros(3)), "positions must be"),
    (dict(positions=-1), "positions must be"),
    (dict(slots=torch.zeros(6, dtype=torch.int64)[::2]), "slots must be"),
    (dict(slots=1.0), "slots must be"),
    (dict(k_pages=torch.zeros(2, 1, 16, 72, dtype=torch.bfloat16),
          v_pages=torch.zeros(2, 1, 16, 72, dtype=torch.bfloat16)), "multiple of 16"),
    (dict(v_pages=torch.zeros(2, 1, 64, 16, dtype=torch.bfloat16).transpose(2, 3)), "16-byte aligned"),
    (dict(out=torch.zeros(3, 4, 64)), "out must be"),
])
def test_rope_to_pages_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        fpv2.rope_to_pages(**_rope_args(**change))


def test_rope_to_pages_refuses_cpu_tensors_and_gradients():
    with pytest.raises(RuntimeError, match="ROCm"):
        fpv2.rope_to_pages(**_rope_args())
    weight = torch.ones(64, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward"):
        fpv2.rope_to_pages(**_rope_args(q_weight=weight))


def _linear_args(**change):
    bf16 = torch.bfloat16
    args = dict(x=torch.zeros(3, 128, dtype=bf16), packed=torch.zeros(10, 16, dtype=torch.int32),
                scales=torch.zeros(10, 2, dtype=bf16), biases=torch.zeros(10, 2, dtype=bf16))
    args.update(change)
    return args


@pytest.mark.parametrize("change,message", [
    (dict(x=torch.zeros(3, 128)), "x must be"),
    (dict(x=torch.zeros(3, 120, dtype=torch.bfloat16)), "as many columns"),
    (dict(packed=torch.zeros(10, 16)), "packed must be"),
    (dict(packed=torch.zeros(16, 10, dtype=torch.int32).T), "packed must have"),
    (dict(scales=torch.zeros(9, 2, dtype=torch.bfloat16)), "scales and biases must be"),
    (dict(scales=torch.zeros(10, 3, dtype=torch.bfloat16),
          biases=torch.zeros(10, 3, dtype=torch.bfloat16)), "groups must be"),
    (dict(scales=torch.zeros(10, 0, dtype=torch.bfloat16),
          biases=torch.zeros(10, 0, dtype=torch.bfloat16)), "groups must be"),
    (dict(scales=torch.zeros(10, 2), biases=torch.zeros(10, 2)), "share a dtype"),
    (dict(scales=torch.zeros(2, 10, dtype=torch.bfloat16).T), "scales must have"),
    (dict(biases=torch.zeros(10, 4, dtype=torch.bfloat16)[:, :2]), "biases must have"),
    (dict(out_dtype=torch.float16), "out_dtype"),
    (dict(out=torch.zeros(3, 9, dtype=torch.bfloat16)), "out must be"),
    (dict(out=torch.zeros(10, 3, dtype=torch.bfloat16).T), "out must be"),
    (dict(out=torch.zeros(1, 10, dtype=torch.bfloat16).expand(3, 10)), "out must be"),
])
def test_quantized_linear_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        fpv2.quantized_linear(**_linear_args(**change))


def test_quantized_linear_refuses_cpu_tensors_and_gradients():
    with pytest.raises(RuntimeError, match="ROCm"):
        fpv2.quantized_linear(**_linear_args())
    x = torch.zeros(3, 128, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward"):
        fpv2.quantized_linear(**_linear_args(x=x))


def test_quantize_weight_layout_and_refusals():
    w = torch.arange(32, dtype=torch.float32).remainder(16)[None]
    packed, scales, biases = fpv2.quantize_weight(w, group_size=32)
    assert [int(x) & 0xffffffff for x in packed[0]] == [0x76543210, 0xfedcba98] * 2
    assert scales.tolist() == [[1.0]] and biases.tolist() == [[0.0]]
    assert torch.equal(fpv2.dequantize_weight(packed, scales, biases), w)
    for bad in (dict(weight=torch.zeros(2, 100)), dict(weight=torch.zeros(2, 2, 64)),
                dict(weight=torch.zeros(2, 64, dtype=torch.int32)),
                dict(weight=torch.zeros(2, 48), group_size=16), dict(weight=torch.zeros(2, 0))):
        with pytest.raises(ValueError):
            fpv2.quantize_weight(**bad)


def _sample_args(**change):
    args = dict(logits=torch.zeros(3, 50), uniform=torch.zeros(3))
    args.update(change)
    return args


@pytest.mark.parametrize("change,message", [
    (dict(logits=torch.zeros(50)), "logits must be"),
    (dict(logits=torch.zeros(3, 50, dtype=torch.float64)), "logits must be"),
    (dict(logits=torch.zeros(3, 0)), "vocabulary must have"),
    (dict(logits=torch.zeros(1, 1).expand(3, (1 << 19) + 1)), "vocabulary must have"),
    (dict(uniform=torch.zeros(2)), "uniform must be"),
    (dict(uniform=torch.zeros(3, dtype=torch.float64)), "uniform must be"),
    (dict(uniform=torch.zeros(6)[::2]), "uniform must be"),
    (dict(temperature=-0.1), "temperature"),
    (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=float("inf")), "temperature"),
    (dict(temperature=torch.ones(2)), "temperature"),
    (dict(top_k=-1), "top_k"),
    (dict(top_k=2.0), "top_k"),
    (dict(top_k=torch.ones(3)), "top_k"),
    (dict(top_p=1.5), "top_p"),
    (dict(top_p=True), "top_p"),
    (dict(top_p=torch.ones(3, dtype=torch.float64)), "top_p"),
    (dict(min_p=-0.5), "min_p"),
    (dict(min_p="no"), "min_p"),
])
def test_sample_tokens_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        fpv2.sample_tokens(**_sample_args(**change))


def test_sample_tokens_refuses_cpu_tensors_and_gradients():
    with pytest.raises(RuntimeError, match="ROCm"):
        fpv2.sample_tokens(**_sample_args())
    with pytest.raises(RuntimeError, match="no backward"):
        fpv2.sample_tokens(**_sample_args(logits=torch.zeros(3, 50, requires_grad=True)))


def test_more_refusals():
    """Destinations that overlap themselves, indexes past 64 bits."""
    bf16 = torch.bfloat16
    for out in (torch.zeros(1, 8, 64, dtype=bf16).expand(2, 8, 64),
                torch.zeros(2, 1, 64, dtype=bf16).expand(2, 8, 64)):
        with pytest.raises(ValueError, match="out must be"):
            fpv2.decode_attention(**_attention_args(out=out))
    for out in (torch.zeros(1, 4, 64, dtype=bf16).expand(3, 4, 64),
                torch.zeros(3, 1, 64, dtype=bf16).expand(3, 4, 64)):
        with pytest.raises(ValueError, match="out must be"):
            fpv2.rope_to_pages(**_rope_args(out=out))
    for name in ("positions", "slots"):
        with pytest.raises(ValueError, match=name):
            fpv2.rope_to_pages(**_rope_args(**{name: 1 << 62}))


def test_rope_to_pages_refuses_caches_that_overlap():
    """Tokens' rows would be written over one another."""
    bf16 = torch.bfloat16
    k, v = (torch.zeros(2, 1, 16, 64, dtype=bf16) for _ in "kv")
    for name in ("k_pages", "v_pages"):
        for bad in (torch.zeros(1, 1, 16, 64, dtype=bf16).expand(2, 1, 16, 64),
                    torch.zeros(2, 1, 1, 64, dtype=bf16).expand(2, 1, 16, 64),
                    torch.zeros(2000, dtype=bf16).as_strided((2, 1, 16, 64), (1024, 1024, 8, 1))):
            with pytest.raises(ValueError, match="overlap"):
                fpv2.rope_to_pages(**_rope_args(**{"k_pages": k, "v_pages": v, name: bad}))


def test_c_entries_refuse_without_a_device():
    """Argument errors of the C entries come before any device call."""
    import ctypes

    from fpv2 import _lib
    if not _lib.LIB_PATH.exists():
        pytest.skip("libfpv2_hip.so not built (run __graft_entry__.build())")
    lib = _lib.load()

    def attention(**change):
        p = _lib.DecodeParams(batch=1, query_heads=4, kv_heads=2, head_dim=64, pages=3, page_size=16,
                              table_width=2, table_stride=2)
        for name, value in change.items():
            setattr(p, name, value)
        return lib.fpv2_decode_attention(8, 16, 16, 16, 16, 16, _lib.BF16, ctypes.byref(p), None, 0, None)

    for change in (dict(batch=-1), dict(kv_heads=0), dict(query_heads=5), dict(pages=0),
                   dict(page_size=0), dict(table_width=0), dict(window_tokens=-1), dict(sink_tokens=-2),
                   dict(length=-1), dict(page_size=1 << 30), dict(k_row_stride=4),
                   dict(table_stride=-1), dict()):
        assert attention(**change) == _lib.FPV2_ERR_ARGUMENT  # (the last: q is not aligned)
    assert attention(head_dim=80) == _lib.FPV2_ERR_UNSUPPORTED
    assert attention(batch=1 << 16) == _lib.FPV2_ERR_UNSUPPORTED
    assert attention(batch=0) == _lib.FPV2_OK
    assert lib.fpv2_decode_attention(0, 0, 0, 0, 0, 0, _lib.BF16, None, None, 0, None) == -1

    def rope(**change):
        p = _lib.RopePagesParams(tokens=2, query_heads=4, kv_heads=2, head_dim=64, rotary_half=32,
                                 table_rows=9, pages=3, page_size=16, qkv_row_stride=512,
                                 q_token_stride=256, q_head_stride=64)
        for name, value in change.items():
            setattr(p, name, value)
        return lib.fpv2_rope_to_pages(8, 16, 16, 16, 16, 16, 16, 16, 16, 16, _lib.F16,
                                      ctypes.byref(p), None)

    for change in (dict(tokens=-1), dict(kv_heads=0), dict(table_rows=0), dict(pages=0),
                   dict(pages=1 << 27, page_size=16), dict(position_bytes=2), dict(slot_bytes=1),
                   dict(qkv_row_stride=504), dict(q_head_stride=63), dict()):
        assert rope(**change) == _lib.FPV2_ERR_ARGUMENT
    for change in (dict(head_dim=72), dict(head_dim=528), dict(rotary_half=40), dict(rotary_half=12)):
        assert rope(**change) == _lib.FPV2_ERR_UNSUPPORTED
    assert rope(tokens=0) == _lib.FPV2_OK

    def linear(rows=2, n=32, k=128, group=64, xs=128, ps=16, ss=2, os=32, dtype=_lib.BF16,
               out_dtype=_lib.BF16, x=8):
        return lib.fpv2_quantized_linear(x, 16, 16, 16, 16, dtype, out_dtype, rows, n, k, group, xs, ps,
                                         ss, os, None)

    for change in (dict(rows=-1), dict(k=100), dict(k=0), dict(xs=120), dict(xs=130), dict(ps=14),
                   dict(ps=12), dict(ss=1), dict(os=31), dict(x=0), dict()):
        assert linear(**change) == _lib.FPV2_ERR_ARGUMENT
    for change in (dict(group=48), dict(dtype=_lib.F32), dict(out_dtype=_lib.F16)):
        assert linear(**change) == _lib.FPV2_ERR_UNSUPPORTED
    assert linear(rows=0) == _lib.FPV2_OK and linear(n=0) == _lib.FPV2_OK

    def sample(dtype=_lib.F32, logits=16, **change):
        p = _lib.SampleParams(batch=2, vocab=5000, logits_stride=5000, temperature=1.0, top_p=1.0)
        for name, value in change.items():
            setattr(p, name, value)
        return lib.fpv2_sample_tokens(logits, 16, dtype, ctypes.byref(p), 16, None, None, 0, None)

    for change in (dict(batch=-1), dict(batch=1 << 16), dict(vocab=0), dict(logits_stride=-1),
                   dict(logits=0), dict()):  # (the last: no workspace)
        assert sample(**change) == _lib.FPV2_ERR_ARGUMENT
    assert sample(vocab=(1 << 19) + 1) == _lib.FPV2_ERR_UNSUPPORTED
    assert sample(dtype=7) == _lib.FPV2_ERR_UNSUPPORTED
    assert sample(batch=0) == _lib.FPV2_OK
