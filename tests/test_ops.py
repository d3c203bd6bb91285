"""The 8-bit operators' C entry points refuse what they cannot run
(include/vosk_amd_ops.h; no GPU: nothing is launched)."""
import ctypes as C
import os
import re
import subprocess

import pytest
import torch

from conftest import REPO

HDR = os.path.join(REPO, "include", "vosk_amd_ops.h")
P = 4096  # stands for a 16-byte aligned device address that is never read


@pytest.fixture(scope="module")
def lib():
    from vosk import ops
    return ops._c


def _err(lib):
    return lib.vamd_last_error().decode()


def test_header_is_plain_c_and_every_function_is_exported(lib):
    subprocess.run(["gcc", "-fsyntax-only", "-Wall", "-Werror", "-x", "c", HDR], check=True)
    names = set(re.findall(r"\b(vamd_op_\w+)\s*\(", open(HDR).read()))
    assert len(names) == 6
    assert not [n for n in names if not hasattr(lib, n)]


@pytest.mark.parametrize("k,want", [(1, 64), (64, 64), (65, 128), (1 << 17, 1 << 17), (0, -1), (-3, -1), ((1 << 17) + 1, -1)])
def test_code_bytes(lib, k, want):
    assert lib.vamd_op_code_bytes(k) == want


def test_workspace(lib):
    assert lib.vamd_op_linear_workspace(3, 65) == 3 * (128 + 4)
    assert lib.vamd_op_linear_workspace(0, 65) == 0
    assert lib.vamd_op_linear_workspace(-1, 65) < 0
    assert lib.vamd_op_linear_workspace(1, 0) < 0


ROWS = dict(device=0, stream=None, x=P, type=0, m=4, k=100, ldx=100, rows=None, count=None, cache_rows=4, codes=P, ldc=128, scales=P)


@pytest.mark.parametrize("change,what", [
    (dict(type=3), "element type"), (dict(m=-1), "rows"), (dict(k=0), "k has"), (dict(k=(1 << 17) + 1), "k has"),
    (dict(x=None), "null"), (dict(codes=None), "null"), (dict(scales=None), "null"), (dict(ldx=99), "overlap"),
    (dict(x=P + 2), "aligned"), (dict(codes=P + 8), "16-byte"), (dict(ldc=120), "16-byte"), (dict(ldc=64), "shorter"),
    (dict(cache_rows=3), "fewer"), (dict(rows=P, cache_rows=-1), "fewer"),
])
def test_quantize_rows_refuses(lib, change, what):
    assert lib.vamd_op_quantize_rows(*{**ROWS, **change}.values()) < 0
    assert what in _err(lib)


def test_nothing_to_do_is_no_error(lib):
    assert lib.vamd_op_quantize_rows(*{**ROWS, "m": 0}.values()) == 0
    assert lib.vamd_op_linear_int8(*{**LINEAR, "m": 0}.values()) == 0
    assert lib.vamd_op_linear_int8(*{**LINEAR, "n": 0}.values()) == 0


MAP = dict(device=0, stream=None, lengths=P, first=P, streams=2, table=P, ldt=3, pages=3, page=8, offsets=None, taps=2, step=1,
           low=None, high=None, clamp=1, starts=P, rows=P, cap=10)


@pytest.mark.parametrize("change,what", [
    (dict(streams=-1), "sizes"), (dict(cap=-1), "sizes"), (dict(cap=1 << 31), "sizes"), (dict(pages=0), "pages"),
    (dict(page=0), "pages"), (dict(pages=1 << 16, page=1 << 15), "pages"), (dict(taps=0), "offsets"), (dict(taps=17), "offsets"),
    (dict(offsets=0), "offsets"), (dict(step=0), "step"), (dict(starts=None), "null"), (dict(lengths=None), "null"),
    (dict(first=None), "null"), (dict(table=None), "null"), (dict(rows=None), "null"), (dict(ldt=2), "overlap"),
])
def test_frame_map_refuses(lib, change, what):
    offsets = (C.c_int * 17)(*range(17))
    a = {**MAP, "offsets": C.cast(offsets, C.c_void_p), **change}
    a["offsets"] = a["offsets"] or None
    assert lib.vamd_op_frame_map(*a.values()) < 0
    assert what in _err(lib)


LINEAR = dict(device=0, stream=None, codes=P, lda=128, scale=P, cache_rows=5, rows=P, taps=2, count=None, w=P, ldw=256,
              wscale=P, m=7, n=9, k=100, bias=None, relu=0, gain=None, shift=None, residual=None, ldr=0, residual_type=0,
              residual_scale=1.0, out=P, ldo=9, out_type=0)


@pytest.mark.parametrize("change,what", [
    (dict(m=-1), "sizes"), (dict(n=-1), "sizes"), (dict(k=0), "k has"), (dict(k=(1 << 17) + 1), "k has"), (dict(taps=0), "taps"),
    (dict(taps=17), "taps"), (dict(out_type=-1), "output type"), (dict(codes=None), "null"), (dict(scale=None), "null"),
    (dict(w=None), "null"), (dict(wscale=None), "null"), (dict(out=None), "null"), (dict(codes=P + 1), "16-byte"),
    (dict(lda=136), "16-byte"), (dict(w=P + 4), "16-byte"), (dict(ldw=264), "16-byte"), (dict(cache_rows=0), "shorter"),
    (dict(lda=64), "shorter"), (dict(ldw=128), "shorter"), (dict(rows=None), "row map"),
    (dict(rows=None, taps=1, cache_rows=6), "fewer"), (dict(gain=P), "together"), (dict(shift=P), "together"),
    (dict(ldo=8), "overlap"), (dict(out=P + 2), "aligned"), (dict(residual=P, residual_type=5), "residual type"),
    (dict(residual=P + 2), "residual is not aligned"),
])
def test_linear_int8_refuses(lib, change, what):
    assert lib.vamd_op_linear_int8(*{**LINEAR, **change}.values()) < 0
    assert what in _err(lib)


FLOAT = dict(device=0, stream=None, x=P, type=0, ldx=100, workspace=P, count=None, w=P, ldw=128, wscale=P, m=7, n=9, k=100,
             bias=None, relu=0, gain=None, shift=None, residual=None, ldr=0, residual_type=0, residual_scale=1.0, out=P, ldo=9,
             out_type=0)


@pytest.mark.parametrize("change,what", [
    (dict(k=0), "k has"), (dict(type=7), "element type"), (dict(x=None), "null"), (dict(ldx=50), "overlap"),
    (dict(workspace=None), "null"), (dict(workspace=P + 4), "16-byte"), (dict(ldw=64), "shorter"), (dict(m=-2), "rows"),
])
def test_linear_float_refuses(lib, change, what):
    assert lib.vamd_op_linear_float(*{**FLOAT, **change}.values()) < 0
    assert what in _err(lib)


def test_tensors_on_the_cpu_are_refused():
    from vosk import ops
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="GPU"):
        ops.quantize_rows(x)
    with pytest.raises(ValueError, match="GPU"):
        ops.linear_int8(x, x.to(torch.int8), x[:, 0])
    with pytest.raises(ValueError, match="GPU"):
        ops.frame_map(x[0].int(), x[0].int(), x.int(), 4, x.int())


def test_import_after_vosk_alone_names_the_cause():
    """Two HIP runtimes in one process: said at import, not found out at the first launch."""
    code = "import sys; sys.path.insert(0, %r); import vosk\ntry:\n  import vosk.ops\nexcept ImportError as e: print('SAID', e)" % (
        os.path.join(REPO, "vosk-api_amd"))
    out = subprocess.run(["python3", "-c", code], capture_output=True, text=True, check=True).stdout
    torch_has_its_own = os.path.exists(os.path.join(os.path.dirname(torch.__file__), "lib", "libamdhip64.so"))
    assert ("import torch before vosk" in out) == torch_has_its_own
