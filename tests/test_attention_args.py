"""Refusals of the attention entry points that need no GPU: handles, sizes, strides and pointers are checked on
the host before any CUDA call, and the Python layer checks its tensors first."""
import ctypes
import math

import pytest
import torch

from helios_b200 import _lib


def invalid(status, message, expect=_lib.G4Q_ERR_INVALID_ARGUMENT):
    assert status == expect, (status, _lib.last_error())
    assert message in _lib.last_error()


def test_handles_are_checked():
    L = _lib.load()
    bogus = ctypes.cast(ctypes.create_string_buffer(256), ctypes.c_void_p)
    for h, word in ((None, "non-null"), (bogus, "invalid")):
        invalid(L.g4q_rope_free(h), word)
        invalid(L.g4q_attn_free(h), word)
        invalid(L.g4q_qk_norm_rope(h, None, None, 1, None, None, None, 1e-6, None, None, None), word)
        invalid(L.g4q_kv_append(h, None, None, None, 1, None, None, 1e-6, 0, None, None, None, None), word)
        invalid(L.g4q_paged_attention(h, None, 1, None, None, 1.0, 0, None, None), word)


@pytest.mark.parametrize("head_dim,rotary,freqs,expect,message", [
    (96, 96, [1.0] * 48, _lib.G4Q_ERR_UNSUPPORTED_CONFIG, "head_dim must be"),
    (64, 24, [1.0] * 12, _lib.G4Q_ERR_UNSUPPORTED_CONFIG, "rotary_dim must be"),
    (64, 128, [1.0] * 64, _lib.G4Q_ERR_UNSUPPORTED_CONFIG, "rotary_dim must be"),
    (64, 0, [], _lib.G4Q_ERR_UNSUPPORTED_CONFIG, "rotary_dim must be"),
    (64, 16, [math.inf] * 8, _lib.G4Q_ERR_INVALID_ARGUMENT, "finite"),
    (64, 16, [math.nan] * 8, _lib.G4Q_ERR_INVALID_ARGUMENT, "finite"),
])
def test_rope_create_refuses(head_dim, rotary, freqs, expect, message):
    L = _lib.load()
    out = ctypes.c_void_p()
    arr = (ctypes.c_double * max(1, len(freqs)))(*freqs)
    invalid(L.g4q_rope_create(head_dim, rotary, arr, ctypes.byref(out)), message, expect)
    assert not out
    invalid(L.g4q_rope_create(64, 64, None, ctypes.byref(out)), "inv_freq")
    invalid(L.g4q_rope_create(64, 64, arr, None), "out must be non-null")


@pytest.mark.parametrize("hq,hk,d,expect,message", [
    (16, 8, 80, _lib.G4Q_ERR_UNSUPPORTED_CONFIG, "head_dim must be"),
    (16, 0, 64, _lib.G4Q_ERR_INVALID_ARGUMENT, "multiple of n_kv_heads"),
    (16, 5, 64, _lib.G4Q_ERR_INVALID_ARGUMENT, "multiple of n_kv_heads"),
    (4, 8, 64, _lib.G4Q_ERR_INVALID_ARGUMENT, "multiple of n_kv_heads"),
    (65, 1, 64, _lib.G4Q_ERR_UNSUPPORTED_CONFIG, "at most 64"),
])
def test_attn_create_refuses(hq, hk, d, expect, message):
    L = _lib.load()
    out = ctypes.c_void_p()
    invalid(L.g4q_attn_create(hq, hk, d, ctypes.byref(out)), message, expect)
    invalid(L.g4q_attn_create(16, 8, 64, None), "out must be non-null")


def test_python_layer_refuses_before_the_library():
    from helios_b200 import attention as A
    ops = _lib.torch_ops()
    cpu = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    for bad, word in ((cpu, "CUDA tensor"), (cpu.float(), "bfloat16"), (None, "torch tensor"), (3, "torch tensor")):
        with pytest.raises(ValueError, match=word):
            ops.paged_attention(0, 64, 0, 0, bad, 0, 0, 1.0, 0, None)
        with pytest.raises(ValueError, match=word):
            ops.qk_norm_rope(0, 64, 0, 0, bad, cpu, cpu, None, None, 1e-6, None, None)
        with pytest.raises(ValueError, match=word):
            ops.kv_append(0, 64, 0, 0, None, bad, cpu, 0, 0, None, None, 1e-6, 0, None)
    for window in (-1, 2 ** 31):
        with pytest.raises(ValueError, match="window"):
            ops.paged_attention(0, 64, 0, 0, cpu, 0, 0, 1.0, window, None)
    with pytest.raises(TypeError):
        ops.paged_attention(0, 64)
    with pytest.raises(TypeError):
        ops.paged_attention("x", 64, 0, 0, cpu, 0, 0, 1.0, 0, None)
    with pytest.raises(TypeError):
        ops.paged_attention(0, 64, 0, 0, cpu, 0, 0, "x", 0, None)
    with pytest.raises(OverflowError):
        ops.paged_attention(0, 64, 0, 0, cpu, 0, 0, 1.0, 2 ** 70, None)
    with pytest.raises(TypeError):
        ops.bind(0, 0, 0, None)
    with pytest.raises(ValueError, match="4-D bfloat16 CUDA"):
        A.PagedKVCache(torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16), torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="int32 CUDA"):
        A.PagedBatch(torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
                     torch.zeros(1, 1, dtype=torch.int32), max_q=1)
    with pytest.raises(ValueError, match="base"):
        A.Rope(64, base=0.0)
    with pytest.raises(ValueError, match="32 values"):
        A.Rope(64, inv_freq=[1.0])


def test_struct_layouts_match_the_header(tmp_path):
    """sizeof and offsetof of the public structs, from the C compiler against the ctypes binding."""
    import subprocess
    from conftest import ROOT
    structs = {"G4qHeadRows": _lib.G4qHeadRows, "G4qPagedCache": _lib.G4qPagedCache, "G4qPagedBatch": _lib.G4qPagedBatch}
    lines = []
    for n, s in structs.items():
        lines.append(f'printf("{n} %zu\\n", sizeof({n}));')
        lines += [f'printf("{n}.{f} %zu\\n", offsetof({n}, {f}));' for f, _ in s._fields_]
    src = tmp_path / "pins.c"
    src.write_text('#include <stdio.h>\n#include "g4q.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    exe = tmp_path / "pins"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for n, s in structs.items():
        assert int(got[n]) == ctypes.sizeof(s)
        for f, _ in s._fields_:
            assert int(got[f"{n}.{f}"]) == getattr(s, f).offset, (n, f)


def test_angle_reduction_on_the_host():
    """The fixed-point turns against 80-digit arithmetic: position * inv_freq / 2 pi modulo one turn."""
    from decimal import Decimal, getcontext
    getcontext().prec = 60
    two_pi = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494")
    for f in (1.0, 10000.0 ** (-2.0 / 256), 1e6 ** (-126 / 128), 3.9e-5, 7.25):
        turn = Decimal(f) / two_pi
        fixed = int((turn % 1) * 2 ** 64 + Decimal("0.5")) % 2 ** 64
        for pos in (0, 1, 16383, 262143, 2 ** 31 - 1, -5):
            got = (pos * fixed) % 2 ** 64 / 2.0 ** 64
            want = float((Decimal(pos) * turn) % 1) % 1.0
            assert min(abs(got - want), 1 - abs(got - want)) < 2.0 ** -32
