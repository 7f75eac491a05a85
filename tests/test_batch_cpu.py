"""What the operators of ``fpv2.batch`` refuse, before any device work (no GPU needed), the layouts
of their C structures and what the C entries refuse."""

from __future__ import annotations

import ctypes

import pytest
import torch

import fpv2
from fpv2 import _lib

BF16, F16, F32, I8, I32, I64 = (torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.int32,
                                torch.int64)


def _shared_args(**change):
    args = dict(q=torch.zeros(2, 8, 64, dtype=BF16), prefix_k=torch.zeros(4, 2, 8, 64, dtype=BF16),
                prefix_v=torch.zeros(4, 2, 8, 64, dtype=BF16), prefix_table=torch.zeros(3, dtype=I32),
                prefix_length=torch.ones(1, dtype=I32), k_pages=torch.zeros(6, 2, 16, 64, dtype=BF16),
                v_pages=torch.zeros(6, 2, 16, 64, dtype=BF16), page_table=torch.zeros(2, 3, dtype=I32),
                lengths=torch.ones(2, dtype=I32))
    return {**args, **change}


def _pair(*shape, dtype=BF16):
    return [torch.zeros(*shape, dtype=dtype) for _ in "kv"]


def _prefix(k, v):
    return dict(prefix_k=k, prefix_v=v)


@pytest.mark.parametrize("change,message", [
    (dict(q=torch.zeros(8, 64, dtype=BF16)), "q must have shape"),
    (dict(q=torch.zeros(2, 7, 64, dtype=BF16)), "divisible by KV heads"),
    (dict(q=torch.zeros(2, 8, 64)), "share float16 or bfloat16"),
    (dict(q=torch.zeros(2, 8, 64, dtype=F16)), "share float16 or bfloat16"),
    (dict(q=torch.zeros(2, 8, 128, dtype=BF16)), "head dimension"),
    (_prefix(*_pair(4, 1, 8, 64)), "the prefix must have"),
    (_prefix(*_pair(4, 2, 8, 128)), "the prefix must have"),
    (_prefix(*_pair(4, 2, 8, 64, dtype=F16)), "share float16 or bfloat16"),
    (_prefix(torch.zeros(4, 2, 8, 64, dtype=BF16), torch.zeros(5, 2, 8, 64, dtype=BF16)), "same shape"),
    (_prefix(*_pair(0, 2, 8, 64)), "at least one row"),
    (_prefix(*(x[..., 1:] for x in _pair(4, 2, 8, 65))), "16-byte aligned"),
    (dict(prefix_table=torch.zeros(3, dtype=I64)), "prefix_table must be int32"),
    (dict(prefix_table=torch.zeros(1, 3, dtype=I32)), "prefix_table must be int32"),
    (dict(prefix_table=torch.zeros(0, dtype=I32)), "at least one page"),
    (dict(prefix_table=torch.zeros(6, dtype=I32)[::2]), "contiguous rows"),
    (dict(prefix_length=torch.ones(1, dtype=I64)), "prefix_length must be"),
    (dict(prefix_length=torch.ones(2, dtype=I32)), "prefix_length must be"),
    (dict(prefix_length=torch.tensor(1, dtype=I32)), "prefix_length must be"),
    (dict(prefix_length=-1), "prefix_length must be"),
    (dict(prefix_length=True), "prefix_length must be"),
    (dict(page_table=torch.zeros(3, 3, dtype=I32)), "page_table must be int32"),
    (dict(page_table=torch.zeros(2, 0, dtype=I32)), "at least one page"),
    (dict(page_table=None, k_pages=torch.zeros(1, 2, 16, 64, dtype=BF16),
          v_pages=torch.zeros(1, 2, 16, 64, dtype=BF16)), "every sequence needs a page"),
    (dict(lengths=torch.ones(2, dtype=I64)), "lengths must be"),
    (dict(lengths=1.0), "lengths must be"),
    (dict(out=torch.zeros(2, 8, 64)), "out must be"),
    (dict(out=torch.zeros(1, 8, 64, dtype=BF16).expand(2, 8, 64)), "out must be"),
])
def test_shared_prefix_attention_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        fpv2.shared_prefix_attention(**_shared_args(**change))


def test_shared_prefix_destinations():
    """In the queries' place, or apart from everything that is read."""
    args = _shared_args()
    for name in ("prefix_k", "prefix_v", "k_pages", "v_pages"):
        with pytest.raises(ValueError, match="share memory"):
            fpv2.shared_prefix_attention(**args, out=args[name].view(-1)[:1024].view(2, 8, 64))
    for name in ("page_table", "lengths", "prefix_table", "prefix_length"):
        memory = torch.zeros(4096, dtype=torch.uint8)
        table = memory[:4 * args[name].numel()].view(I32).view(args[name].shape)
        with pytest.raises(ValueError, match="share memory"):
            fpv2.shared_prefix_attention(**{**args, name: table}, out=memory[:2048].view(BF16).view(2, 8, 64))
    with pytest.raises(RuntimeError, match="ROCm"):
        fpv2.shared_prefix_attention(**args, out=args["q"])


def _cache_args(**change):
    args = dict(k_codes=torch.zeros(6, 2, 16, 64, dtype=I8), k_scales=torch.zeros(6, 2, 16),
                v_codes=torch.zeros(6, 2, 16, 64, dtype=I8), v_scales=torch.zeros(6, 2, 16))
    return {**args, **change}


def _write_args(**change):
    args = dict(k=torch.zeros(3, 2, 64, dtype=BF16), v=torch.zeros(3, 2, 64, dtype=BF16),
                slots=torch.arange(3), **_cache_args())
    return {**args, **change}


def _read_args(**change):
    return {**dict(page_table=torch.zeros(2, 3, dtype=I32), lengths=torch.ones(2, dtype=I32), **_cache_args()),
            **change}


def _attend_args(**change):
    return {**_read_args(q=torch.zeros(2, 8, 64, dtype=BF16)), **change}


CACHES = [
    (dict(k_codes=torch.zeros(6, 2, 16, 64, dtype=torch.uint8)), "k_codes must be int8"),
    (dict(v_codes=torch.zeros(2, 16, 64, dtype=I8)), "v_codes must be int8"),
    (dict(v_codes=torch.zeros(6, 2, 8, 64, dtype=I8)), "same shape"),
    (dict(k_scales=torch.zeros(6, 2, 16, 1)), "k_scales must be float32"),
    (dict(v_scales=torch.zeros(6, 2, 16, dtype=F16)), "v_scales must be float32"),
    (dict(k_codes=torch.zeros(6, 2, 16, 72, dtype=I8)[..., 8:]), "16-byte aligned"),
    (dict(k_codes=torch.zeros(6, 2, 64, 16, dtype=I8).transpose(2, 3)), "16-byte aligned"),
    (dict(k_codes=torch.zeros(0, 2, 16, 64, dtype=I8), v_codes=torch.zeros(0, 2, 16, 64, dtype=I8),
          k_scales=torch.zeros(0, 2, 16), v_scales=torch.zeros(0, 2, 16)), "at least one row"),
    (dict(k_codes=torch.zeros(6, 2, 16, 80, dtype=I8), v_codes=torch.zeros(6, 2, 16, 80, dtype=I8)),
     "head dimension"),
]


@pytest.mark.parametrize("change,message", CACHES)
def test_caches_of_codes_are_checked(change, message):
    for call, args in ((fpv2.quantize_to_pages, _write_args), (fpv2.dequantize_pages, _read_args),
                       (fpv2.quantized_decode_attention, _attend_args)):
        with pytest.raises(ValueError, match=message):
            call(**args(**change))


@pytest.mark.parametrize("change,message", [
    (dict(k=torch.zeros(3, 64, dtype=BF16)), "k must be"),
    (dict(k=torch.zeros(3, 1, 64, dtype=BF16)), "k must be"),
    (dict(v=torch.zeros(3, 2, 32, dtype=BF16)), "v must be"),
    (dict(v=torch.zeros(4, 2, 64, dtype=BF16)), "v must be"),
    (dict(k=torch.zeros(3, 2, 64)), "share float16 or bfloat16"),
    (dict(v=torch.zeros(3, 2, 64, dtype=F16)), "share float16 or bfloat16"),
    (dict(slots=torch.arange(2)), "slots must be"),
    (dict(slots=torch.arange(6)[::2]), "slots must be"),
    (dict(slots=torch.arange(3, dtype=torch.int16)), "slots must be"),
    (dict(slots=-1), "slots must be"),
    (dict(slots=1 << 62), "slots must be"),
])
def test_quantize_to_pages_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        fpv2.quantize_to_pages(**_write_args(**change))


def test_caches_whose_rows_share_memory_are_refused():
    memory = torch.zeros(1 << 16, dtype=I8)
    codes = memory[:6 * 2 * 16 * 64].view(6, 2, 16, 64)
    floats = torch.zeros(1 << 12)
    inside = memory[4096:4096 + 768].view(F32).view(6, 2, 16)
    for change in (dict(k_codes=codes[:1].expand(6, 2, 16, 64)),
                   dict(v_codes=codes[:, :, :1].expand(6, 2, 16, 64)),
                   dict(k_codes=codes, v_codes=codes),
                   dict(k_codes=codes, v_codes=memory[64:64 + 12288].view(6, 2, 16, 64)),
                   dict(k_codes=codes, v_scales=inside),
                   dict(k_scales=floats[:192].view(6, 2, 16), v_scales=floats[191:383].view(6, 2, 16)),
                   dict(v_scales=floats[:6].view(6, 1, 1).expand(6, 2, 16)),
                   dict(k_scales=floats.as_strided((6, 2, 16), (20, 10, 1)))):
        with pytest.raises(ValueError, match="overlap"):
            fpv2.quantize_to_pages(**_write_args(**change))
        with pytest.raises(RuntimeError, match="ROCm"):  # which only reads them
            fpv2.quantized_decode_attention(**_attend_args(**change))
    # keys beside values in one pool do not
    pool = torch.zeros(6, 16, 2, 2, 64, dtype=I8)
    scales = torch.zeros(6, 2, 16, 2)
    with pytest.raises(RuntimeError, match="ROCm"):
        fpv2.quantize_to_pages(**_write_args(
            k_codes=pool[:, :, 0].transpose(1, 2), v_codes=pool[:, :, 1].transpose(1, 2),
            k_scales=scales[..., 0], v_scales=scales[..., 1]))
    # what is written over what is read
    rows = memory[:768].view(BF16).view(3, 2, 64)
    slots = memory[:24].view(I64)
    for change in (dict(k=rows), dict(v=rows), dict(slots=slots)):
        with pytest.raises(ValueError, match="share memory"):
            fpv2.quantize_to_pages(**_write_args(k_codes=codes, **change))


@pytest.mark.parametrize("change,message", [
    (dict(page_table=torch.zeros(2, 3, dtype=I64)), "page_table must be int32"),
    (dict(page_table=torch.zeros(3, dtype=I32)), "page_table must be int32"),
    (dict(page_table=torch.zeros(2, 0, dtype=I32)), "at least one page"),
    (dict(page_table=torch.zeros(3, 2, dtype=I32).T, lengths=1), "contiguous rows"),
    (dict(page_table=None, lengths=torch.ones(7, dtype=I32)), "every sequence needs a page"),
    (dict(lengths=torch.ones(3, dtype=I32)), "lengths must be"),
    (dict(lengths=torch.ones(2, dtype=I64)), "lengths must be"),
    (dict(lengths=-1), "lengths must be"),
    (dict(tokens=-1), "tokens must be"),
    (dict(tokens=2.0), "tokens must be"),
    (dict(dtype=F32), "dtype must be"),
    (dict(out=tuple(_pair(2, 2, 48, 64, dtype=F32))), "out must be"),
    (dict(out=tuple(_pair(2, 2, 48, 64)), dtype=F16), "out must be"),
    (dict(out=tuple(_pair(2, 2, 48, 64)), tokens=47), "out must be"),
    (dict(out=tuple(_pair(1, 2, 48, 64))), "out must be"),
    (dict(out=tuple(x[..., 1:] for x in _pair(2, 2, 48, 65))), "out must be"),
    (dict(out=tuple(x.expand(2, 2, 48, 64) for x in _pair(1, 2, 48, 64))), "out must be"),
    (dict(out=tuple(x[0] for x in _pair(1, 2, 48, 64))), "out must be"),
    (dict(out=(torch.zeros(2, 2, 48, 64, dtype=BF16), torch.zeros(2, 2, 48, 64, dtype=F16))), "out must be"),
    (dict(out=_pair(2, 2, 48, 64)[:1] * 2), "share memory"),
])
def test_dequantize_pages_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        fpv2.dequantize_pages(**_read_args(**change))


def test_dequantize_destinations_apart():
    memory = torch.zeros(1 << 16, dtype=I8)
    codes = memory[:6 * 2 * 16 * 64].view(6, 2, 16, 64)
    out = (memory[4096:4096 + 2 * 12288].view(BF16).view(2, 2, 48, 64), torch.zeros(2, 2, 48, 64, dtype=BF16))
    for pair in (out, out[::-1]):
        with pytest.raises(ValueError, match="share memory"):
            fpv2.dequantize_pages(**_read_args(k_codes=codes), out=pair)
        with pytest.raises(RuntimeError, match="ROCm"):
            fpv2.dequantize_pages(**_read_args(), out=pair)


@pytest.mark.parametrize("change,message", [
    (dict(q=torch.zeros(8, 64, dtype=BF16)), "q must have shape"),
    (dict(q=torch.zeros(2, 7, 64, dtype=BF16)), "divisible by KV heads"),
    (dict(q=torch.zeros(2, 8, 64)), "float16 or bfloat16"),
    (dict(q=torch.zeros(2, 8, 128, dtype=BF16)), "head dimension"),
    (dict(page_table=torch.zeros(3, 3, dtype=I32)), "page_table must be int32"),
    (dict(page_table=None, q=torch.zeros(7, 8, 64, dtype=BF16), lengths=1), "every sequence needs a page"),
    (dict(lengths=torch.ones(3, dtype=I32)), "lengths must be"),
    (dict(window_tokens=0), "window_tokens"),
    (dict(sink_tokens=-1), "sink_tokens"),
    (dict(out=torch.zeros(2, 8, 64)), "out must be"),
])
def test_quantized_decode_attention_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        fpv2.quantized_decode_attention(**_attend_args(**change))


def test_quantized_decode_destinations():
    memory = torch.zeros(1 << 16, dtype=I8)
    codes = memory[:6 * 2 * 16 * 64].view(6, 2, 16, 64)
    with pytest.raises(ValueError, match="share memory"):
        fpv2.quantized_decode_attention(**_attend_args(v_codes=codes), out=memory[64:2112].view(BF16).view(2, 8, 64))
    args = _attend_args()
    with pytest.raises(RuntimeError, match="ROCm"):
        fpv2.quantized_decode_attention(**args, out=args["q"])


def _logprob_args(**change):
    return {**dict(logits=torch.zeros(3, 50), tokens=torch.zeros(3, dtype=I64)), **change}


@pytest.mark.parametrize("change,message", [
    (dict(logits=torch.zeros(50)), "logits must be"),
    (dict(logits=torch.zeros(3, 50, dtype=torch.float64)), "logits must be"),
    (dict(logits=torch.zeros(3, 0)), "vocabulary"),
    (dict(logits=torch.zeros(1, (1 << 19) + 1), tokens=torch.zeros(1, dtype=I64)), "vocabulary"),
    (dict(tokens=torch.zeros(2, dtype=I64)), "tokens must be"),
    (dict(tokens=torch.zeros(3)), "tokens must be"),
    (dict(tokens=torch.zeros(3, 1, dtype=I64)), "tokens must be"),
    (dict(tokens=torch.zeros(6, dtype=I64)[::2]), "tokens must be"),
    (dict(top=-1), "top must be"),
    (dict(top=33), "top must be"),
    (dict(top=2.0), "top must be"),
])
def test_token_logprobs_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        fpv2.token_logprobs(**_logprob_args(**change))


def test_cpu_tensors_gradients_and_tangents_are_refused():
    from torch.autograd import forward_ad
    calls = [(fpv2.shared_prefix_attention, _shared_args, ("q", "prefix_k", "v_pages")),
             (fpv2.quantize_to_pages, _write_args, ("k", "v", "k_scales")),
             (fpv2.dequantize_pages, _read_args, ("k_scales", "v_scales")),
             (fpv2.quantized_decode_attention, _attend_args, ("q", "v_scales")),
             (fpv2.token_logprobs, _logprob_args, ("logits",))]
    for call, args, names in calls:
        with pytest.raises(RuntimeError, match="ROCm"):
            call(**args())
        for name in names:
            x = args()[name].clone().requires_grad_()
            with pytest.raises(RuntimeError, match="no backward"):
                call(**args(**{name: x}))
            with torch.no_grad(), pytest.raises(RuntimeError, match="ROCm"):
                call(**args(**{name: x}))
            with forward_ad.dual_level(), pytest.raises(RuntimeError, match="derivative"):
                x = args()[name]
                call(**args(**{name: forward_ad.make_dual(x, torch.ones_like(x))}))


@pytest.mark.parametrize("cname,mirror", [
    ("fpv2_shared_prefix_params", "SharedPrefixParams"), ("fpv2_code_pages", "CodePages"),
    ("fpv2_quantize_params", "QuantizeParams"), ("fpv2_dequantize_params", "DequantizeParams"),
    ("fpv2_quantized_decode_params", "QuantizedDecodeParams"), ("fpv2_logprobs_params", "LogprobsParams")])
def test_params_layouts_match_the_header(tmp_path, cname, mirror):
    """The ctypes mirrors, as gcc lays the header's structs out."""
    import shutil
    import subprocess
    from pathlib import Path
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    cls = getattr(_lib, mirror)
    lines = ['#include <stddef.h>', '#include <stdio.h>', '#include "fpv2_batch.h"',
             "int main(void) {", f'  printf("%zu\\n", sizeof({cname}));']
    lines += [f'  printf("%zu\\n", offsetof({cname}, {name}));' for name, _ in cls._fields_]
    source, program = tmp_path / "layout.c", tmp_path / "layout"
    source.write_text("\n".join(lines + ["  return 0;", "}"]))
    include = Path(__file__).resolve().parents[1] / "include"
    subprocess.run([gcc, "-I", str(include), str(source), "-o", str(program)], check=True)
    got = [int(x) for x in subprocess.run([str(program)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    assert got == [ctypes.sizeof(cls)] + [getattr(cls, name).offset for name, _ in cls._fields_]


def _loaded():
    if not _lib.LIB_PATH.exists():
        pytest.skip("libfpv2_hip.so not built")
    return _lib.load()


def test_c_entries_refuse_before_any_launch():
    """Each refusal of the C entries, with its status and message."""
    lib = _loaded()

    def decode(**change):
        fields = dict(batch=2, query_heads=8, kv_heads=2, head_dim=64, pages=6, page_size=16, table_width=3,
                      table_stride=3, scale=1.0, q_batch_stride=512, q_head_stride=64, k_page_stride=2048,
                      k_head_stride=1024, k_row_stride=64, v_page_stride=2048, v_head_stride=1024,
                      v_row_stride=64, o_batch_stride=512, o_head_stride=64)
        return _lib.DecodeParams(**{**fields, **change})

    def refused(status, message, want=_lib.FPV2_ERR_ARGUMENT):
        assert status == want, (status, lib.fpv2_last_error())
        assert message in lib.fpv2_last_error(), lib.fpv2_last_error()

    def shared(own=None, pointers=(16,) * 10, work=1 << 40, dtype=_lib.BF16, **change):
        p = _lib.SharedPrefixParams(own or decode(), **{**dict(
            prefix_pages=4, prefix_page_size=8, prefix_table_width=3, pk_page_stride=1024, pk_head_stride=512,
            pk_row_stride=64, pv_page_stride=1024, pv_head_stride=512, pv_row_stride=64), **change})
        return lib.fpv2_shared_prefix_attention(*pointers, dtype, ctypes.byref(p), 16, work, None)

    refused(lib.fpv2_shared_prefix_attention(*(16,) * 10, _lib.BF16, None, 16, 1, None), b"null params")
    refused(shared(decode(query_heads=7)), b"divisible")
    refused(shared(decode(head_dim=80)), b"head_dim", _lib.FPV2_ERR_UNSUPPORTED)
    refused(shared(decode(window_tokens=4)), b"no window")
    refused(shared(prefix_pages=0), b"prefix's pages")
    refused(shared(prefix_table_width=1 << 29), b"2^30")
    refused(shared(prefix_length=-1), b"prefix_length")
    refused(shared(dtype=_lib.F32), b"dtype", _lib.FPV2_ERR_UNSUPPORTED)
    refused(shared(pointers=(0,) + (16,) * 9), b"null pointer")
    refused(shared(pointers=(16, 16, 16, None) + (16,) * 6), b"prefix table")
    refused(shared(pointers=(8,) + (16,) * 9), b"aligned")
    refused(shared(pk_row_stride=63), b"multiples of 8")
    refused(shared(decode(o_head_stride=-1)), b"output strides")
    refused(shared(work=16), b"workspace")
    assert shared(decode(batch=0)) == 0

    def codes(**change):
        fields = dict(kv_heads=2, head_dim=64, pages=6, page_size=16, k_page_stride=2048, k_head_stride=1024,
                      k_row_stride=64, v_page_stride=2048, v_head_stride=1024, v_row_stride=64,
                      ks_page_stride=32, ks_head_stride=16, ks_row_stride=1, vs_page_stride=32,
                      vs_head_stride=16, vs_row_stride=1)
        return _lib.CodePages(**{**fields, **change})

    def write(cache=None, pointers=(16,) * 7, dtype=_lib.BF16, **change):
        p = _lib.QuantizeParams(cache or codes(), **{**dict(
            tokens=3, slot_bytes=8, k_token_stride=128, k_head_stride=64, v_token_stride=128, v_head_stride=64),
            **change})
        return lib.fpv2_quantize_to_pages(*pointers, dtype, ctypes.byref(p), None)

    refused(lib.fpv2_quantize_to_pages(*(16,) * 7, _lib.BF16, None, None), b"null params")
    refused(write(codes(kv_heads=0)), b"kv_heads")
    refused(write(codes(head_dim=80)), b"head_dim", _lib.FPV2_ERR_UNSUPPORTED)
    refused(write(codes(page_size=0)), b"page_size")
    refused(write(codes(v_row_stride=72)), b"multiples of 16")
    refused(write(codes(ks_row_stride=-1)), b"strides of scales")
    refused(write(dtype=_lib.F32), b"dtype", _lib.FPV2_ERR_UNSUPPORTED)
    refused(write(tokens=-1), b"tokens")
    refused(write(tokens=1 << 31), b"tokens")
    refused(write(slot_bytes=2), b"slot_bytes")
    refused(write(slot_bytes=0, first_slot=-1), b"first_slot")
    refused(write(k_head_stride=4), b"multiples of 8")
    refused(write(pointers=(16, 16, 0, 16, 16, 16, 16)), b"null pointer")
    refused(write(pointers=(16, 16, 16, 24, 16, 16, 16)), b"aligned")
    assert write(tokens=0) == 0

    def read(cache=None, pointers=(16,) * 8, dtype=_lib.BF16, **change):
        p = _lib.DequantizeParams(cache or codes(), **{**dict(
            batch=2, table_width=3, table_stride=3, tokens=48, k_batch_stride=6144, k_head_stride=3136,
            k_row_stride=64, v_batch_stride=6144, v_head_stride=3136, v_row_stride=64), **change})
        return lib.fpv2_dequantize_pages(*pointers, dtype, ctypes.byref(p), None)

    refused(lib.fpv2_dequantize_pages(*(16,) * 8, _lib.BF16, None, None), b"null params")
    refused(read(codes(k_page_stride=8)), b"multiples of 16")
    refused(read(dtype=_lib.F32), b"dtype", _lib.FPV2_ERR_UNSUPPORTED)
    refused(read(batch=1 << 16), b"batch", _lib.FPV2_ERR_UNSUPPORTED)
    refused(read(table_width=0), b"table_width")
    refused(read(tokens=-1), b"tokens")
    refused(read(k_row_stride=4), b"multiples of 8")
    refused(read(pointers=(16,) * 7 + (0,)), b"null pointer")
    refused(read(pointers=(16,) * 4 + (None,) + (16,) * 3), b"one page")
    refused(read(pointers=(16,) * 7 + (24,)), b"aligned")
    assert read(tokens=0) == 0

    def attend(own=None, pointers=(16,) * 8, work=1 << 40, dtype=_lib.BF16, **change):
        p = _lib.QuantizedDecodeParams(own or decode(), **{**dict(
            ks_page_stride=32, ks_head_stride=16, ks_row_stride=1, vs_page_stride=32, vs_head_stride=16,
            vs_row_stride=1), **change})
        return lib.fpv2_quantized_decode_attention(*pointers, dtype, ctypes.byref(p), 16, work, None)

    refused(lib.fpv2_quantized_decode_attention(*(16,) * 8, _lib.BF16, None, 16, 1, None), b"null params")
    refused(attend(decode(head_dim=80)), b"head_dim", _lib.FPV2_ERR_UNSUPPORTED)
    refused(attend(dtype=_lib.F32), b"dtype", _lib.FPV2_ERR_UNSUPPORTED)
    refused(attend(decode(k_row_stride=72)), b"multiples of 16")
    refused(attend(decode(q_head_stride=12)), b"strides of q")
    refused(attend(vs_head_stride=-1), b"strides of scales")
    refused(attend(pointers=(0,) + (16,) * 7), b"null pointer")
    refused(attend(pointers=(16, 24) + (16,) * 6), b"aligned")
    refused(attend(pointers=(16,) * 5 + (None,) + (16,) * 2), b"one page")
    refused(attend(decode(table_width=300), work=16), b"workspace")
    assert attend(decode(batch=0)) == 0

    def logprobs(pointers=(16, 16), outs=(16,) * 4, work=1 << 40, dtype=_lib.F32, **change):
        p = _lib.LogprobsParams(**{**dict(rows=3, vocab=100_000, logits_stride=100_000, token_bytes=8, top=2),
                                   **change})
        return lib.fpv2_token_logprobs(*pointers, dtype, ctypes.byref(p), *outs, 16, work, None)

    refused(lib.fpv2_token_logprobs(16, 16, _lib.F32, None, *(16,) * 4, 16, 1, None), b"null params")
    refused(logprobs(rows=-1), b"rows")
    refused(logprobs(vocab=0), b"vocabulary", _lib.FPV2_ERR_UNSUPPORTED)
    refused(logprobs(vocab=(1 << 19) + 1), b"vocabulary", _lib.FPV2_ERR_UNSUPPORTED)
    refused(logprobs(logits_stride=-1), b"logits_stride")
    refused(logprobs(token_bytes=1), b"token_bytes")
    refused(logprobs(top=33), b"top")
    refused(logprobs(dtype=7), b"dtype", _lib.FPV2_ERR_UNSUPPORTED)
    refused(logprobs(pointers=(0, 16)), b"null pointer")
    refused(logprobs(outs=(16, 16, 0, 16)), b"null pointer")
    refused(logprobs(pointers=(18, 16)), b"aligned")
    refused(logprobs(work=16), b"workspace")
    assert logprobs(rows=0) == 0
