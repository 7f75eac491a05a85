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


def test_decode_params_layout_matches_the_header(tmp_path):
    """The ctypes mirror of fpv2_decode_params, as gcc lays the header's out."""
    import shutil
    import subprocess
    from pathlib import Path

    from fpv2 import _lib
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    lines = ['#include <stddef.h>', '#include <stdio.h>', '#include "fpv2_decode.h"',
             "int main(void) {", '  printf("%zu\\n", sizeof(fpv2_decode_params));']
    lines += [f'  printf("%zu\\n", offsetof(fpv2_decode_params, {name}));'
              for name, _ in _lib.DecodeParams._fields_]
    source, program = tmp_path / "layout.c", tmp_path / "layout"
    source.write_text("\n".join(lines + ["  return 0;", "}"]))
    include = Path(__file__).resolve().parents[1] / "include"
    subprocess.run([gcc, "-I", str(include), str(source), "-o", str(program)], check=True)
    got = [int(x) for x in subprocess.run([str(program)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    import ctypes
    assert got == [ctypes.sizeof(_lib.DecodeParams)] + [
        getattr(_lib.DecodeParams, name).offset for name, _ in _lib.DecodeParams._fields_]
