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


_p, _q, _i, _f = C.c_void_p, C.c_longlong, C.c_int, C.c_float


class Rows(C.Structure):
    _fields_ = [(n, _p) for n in "x rows from_ count codes scales".split()] + [(n, _q) for n in "m ldx cache_rows ldc ldrows ldfrom x_rows".split()] + \
        [(n, _i) for n in "type k".split()]


class Map(C.Structure):
    _fields_ = [(n, _p) for n in "lengths first table low high starts rows".split()] + [("ldt", _q), ("cap", _q)] + \
        [(n, _i) for n in "streams pages page page_stride frame_stride taps step clamp".split()] + [("offsets", _i * 16)]


class Linear(C.Structure):
    _fields_ = [(n, _p) for n in "codes scale rows count x workspace w wscale bias gain shift residual out out_to res_from".split()] + \
        [(n, _q) for n in "cache_rows lda ldx ldw ldr ldo ldrows ldout_to out_rows ldres_from res_rows".split()] + \
        [(n, _i) for n in "m n k taps relu x_type residual_type out_type".split()] + [("residual_scale", _f)]


def _call(lib, name, kind, **fields):
    return getattr(lib, name)(0, None, C.cast(C.pointer(kind(**fields)), C.c_char_p))


def test_header_is_plain_c_and_every_function_is_exported(lib, tmp_path):
    subprocess.run(["gcc", "-fsyntax-only", "-Wall", "-Werror", "-x", "c", HDR], check=True)
    names = set(re.findall(r"\b(vamd_op_\w+)\s*\(", open(HDR).read()))
    assert len(names) == 5
    assert not [n for n in names if not hasattr(lib, n)]


def test_structures_are_laid_out_as_the_bindings_have_them(tmp_path):
    """sizeof and offsetof of every field, from a C compiler, against the structures here and the packing in vosk.ops."""
    from vosk import ops
    kinds = {"VamdQuantizeRows": Rows, "VamdFrameMap": Map, "VamdLinearInt8": Linear}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "%s"' % HDR, "int main(void) {"]
    for name, kind in kinds.items():
        lines.append('printf("%%zu ", sizeof(%s));' % name)
        lines += ['printf("%%zu ", offsetof(%s, %s));' % (name, f.rstrip("_")) for f, _ in kind._fields_]
    (tmp_path / "a.c").write_text("\n".join(lines) + "return 0; }\n")
    subprocess.run(["gcc", str(tmp_path / "a.c"), "-o", str(tmp_path / "a")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "a")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for kind in kinds.values():
        want += [C.sizeof(kind)] + [getattr(kind, f).offset for f, _ in kind._fields_]
    assert got == want
    assert len(ops._ROWS(*range(15))) == C.sizeof(Rows)
    assert len(ops._MAP(*range(33))) == C.sizeof(Map)
    packed = ops._LINEAR(*range(1, 35), 0.5)
    assert C.sizeof(Linear) - 8 < len(packed) <= C.sizeof(Linear)
    back = Linear.from_buffer_copy(packed.ljust(C.sizeof(Linear), b"\0"))
    assert [getattr(back, f) for f, _ in Linear._fields_] == [*range(1, 35), 0.5]


@pytest.mark.parametrize("k,want", [(1, 64), (64, 64), (65, 128), (1 << 17, 1 << 17), (0, -1), (-3, -1), ((1 << 17) + 1, -1)])
def test_code_bytes(lib, k, want):
    assert lib.vamd_op_code_bytes(k) == want


def test_workspace(lib):
    assert lib.vamd_op_linear_workspace(1000, 500, 65, 1, 1000) == 1000 * (128 + 4)
    assert lib.vamd_op_linear_workspace(1000, 500, 65, 3, 77) == 77 * (128 + 4)
    assert lib.vamd_op_linear_workspace(1, 500, 65, 3, 77) == 0
    assert lib.vamd_op_linear_workspace(0, 5, 65, 1, 0) == 0
    assert lib.vamd_op_linear_workspace(-1, 5, 65, 1, 4) < 0
    assert lib.vamd_op_linear_workspace(1, -5, 65, 1, 4) < 0
    assert lib.vamd_op_linear_workspace(1, 5, 65, 0, 4) < 0
    assert lib.vamd_op_linear_workspace(1, 5, 65, 17, 4) < 0
    assert lib.vamd_op_linear_workspace(1, 5, 65, 1, -4) < 0
    assert lib.vamd_op_linear_workspace(1, 5, 0, 1, 4) < 0
    assert lib.vamd_op_linear_workspace((1 << 30) + 1, 5, 64, 1, 4) < 0


def test_no_arguments(lib):
    for name in ("vamd_op_quantize_rows", "vamd_op_frame_map", "vamd_op_linear_int8"):
        assert getattr(lib, name)(0, None, None) < 0
        assert "null" in _err(lib)


ROWS = dict(x=P, m=4, k=100, ldx=100, cache_rows=4, codes=P, ldc=128, scales=P)


@pytest.mark.parametrize("change,what", [
    (dict(type=3), "element type"), (dict(m=-1), "rows"), (dict(k=0), "k has"), (dict(k=(1 << 17) + 1), "k has"),
    (dict(x=None), "null"), (dict(codes=None), "null"), (dict(scales=None), "null"), (dict(ldx=99), "overlap"),
    (dict(x=P + 2), "aligned"), (dict(codes=P + 8), "16-byte"), (dict(ldc=120), "16-byte"), (dict(ldc=64), "shorter"),
    (dict(cache_rows=3), "fewer"), (dict(rows=P, cache_rows=-1), "fewer"), (dict(m=1, from_=P, ldx=99), "overlap"), (dict(from_=P, x_rows=-1), "rows"),
])
def test_quantize_rows_refuses(lib, change, what):
    assert _call(lib, "vamd_op_quantize_rows", Rows, **{**ROWS, **change}) < 0
    assert what in _err(lib)


def test_nothing_to_do_is_no_error(lib):
    assert _call(lib, "vamd_op_quantize_rows", Rows, **{**ROWS, "m": 0}) == 0
    assert _call(lib, "vamd_op_linear_int8", Linear, **{**LINEAR, "m": 0}) == 0
    assert _call(lib, "vamd_op_linear_int8", Linear, **{**FLOAT, "n": 0}) == 0


MAP = dict(lengths=P, first=P, streams=2, table=P, ldt=3, pages=3, page=8, page_stride=8, frame_stride=1, taps=2, step=1, clamp=1, starts=P, rows=P, cap=10)


@pytest.mark.parametrize("change,what", [
    (dict(streams=-1), "sizes"), (dict(cap=-1), "sizes"), (dict(cap=1 << 31), "sizes"), (dict(pages=0), "pages"),
    (dict(page=0), "pages"), (dict(pages=1 << 16, page=1 << 15), "pages"), (dict(taps=0), "offsets"), (dict(taps=17), "offsets"),
    (dict(step=0), "step"), (dict(starts=None), "null"), (dict(lengths=None), "null"),
    (dict(first=None), "null"), (dict(table=None), "null"), (dict(rows=None), "null"), (dict(ldt=2), "overlap"), (dict(page_stride=-1), "strides"), (dict(frame_stride=-2), "strides"),
])
def test_frame_map_refuses(lib, change, what):
    assert _call(lib, "vamd_op_frame_map", Map, **{**MAP, **change}) < 0
    assert what in _err(lib)


LINEAR = dict(codes=P, lda=128, scale=P, cache_rows=5, rows=P, ldrows=2, taps=2, w=P, ldw=256, wscale=P, m=7, n=9, k=100, residual_scale=1.0,
              out=P, ldo=9)


@pytest.mark.parametrize("change,what", [
    (dict(m=-1), "sizes"), (dict(n=-1), "sizes"), (dict(m=(1 << 30) + 1), "sizes"), (dict(n=(1 << 23) + 1), "sizes"),
    (dict(ldo=(1 << 23) + 1), "2^23"), (dict(residual=P, ldr=(1 << 23) + 1), "2^23"), (dict(residual=P, ldr=8), "overlap"),
    (dict(k=0), "k has"),
    (dict(k=(1 << 17) + 1), "k has"), (dict(taps=0), "taps"), (dict(taps=17), "taps"), (dict(out_type=-1), "output type"),
    (dict(codes=None), "null"), (dict(scale=None), "null"), (dict(w=None), "null"), (dict(wscale=None), "null"),
    (dict(out=None), "null"), (dict(codes=P + 1), "16-byte"), (dict(lda=136), "16-byte"), (dict(w=P + 4), "16-byte"),
    (dict(ldw=264), "16-byte"), (dict(cache_rows=0), "shorter"), (dict(lda=64), "shorter"), (dict(ldw=128), "shorter"),
    (dict(rows=None), "row map"), (dict(rows=None, taps=1, cache_rows=6), "fewer"), (dict(gain=P), "together"),
    (dict(shift=P), "together"), (dict(ldo=8), "overlap"), (dict(out=P + 2), "aligned"),
    (dict(residual=P, residual_type=5), "residual type"), (dict(residual=P + 2, ldr=9), "residual is not aligned"),
    (dict(x=P), "without codes"), (dict(ldrows=1), "row map overlap"), (dict(out_to=P, out_rows=-1), "sizes"),
    (dict(out_to=P, out_rows=1 << 26), "2^31"), (dict(residual=P, ldr=9, res_from=P, res_rows=1 << 26), "2^31"),
    (dict(m=1, out_to=P, out_rows=3, ldo=8), "overlap"), (dict(m=1, residual=P, res_from=P, res_rows=3, ldr=8), "overlap"),
])
def test_linear_int8_refuses(lib, change, what):
    assert _call(lib, "vamd_op_linear_int8", Linear, **{**LINEAR, **change}) < 0
    assert what in _err(lib)


FLOAT = dict(x=P, ldx=100, workspace=P, w=P, ldw=128, wscale=P, m=700, n=9, k=100, taps=1, residual_scale=1.0, out=P, ldo=9)


@pytest.mark.parametrize("change,what", [
    (dict(k=0), "k has"), (dict(x_type=7), "element type"), (dict(ldx=50), "overlap"), (dict(x=P + 1), "aligned"),
    (dict(workspace=None), "null"), (dict(workspace=P + 4), "16-byte"), (dict(ldw=64), "shorter"), (dict(m=-2), "sizes"),
    (dict(codes=P), "without codes"), (dict(scale=P), "without codes"), (dict(taps=2, ldw=256), "row map"), (dict(taps=0), "taps"),
    (dict(rows=P, ldrows=1), "bad number"),
])
def test_linear_of_floats_refuses(lib, change, what):
    assert _call(lib, "vamd_op_linear_int8", Linear, **{**FLOAT, **change}) < 0
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


def test_plan_of_the_8_bit_layers(synth_model):
    """Which layers of the TDNN-F model run as 8-bit products, and through how many maps."""
    from vosk import engine
    lines = engine.plan_describe_int8(synth_model, 51).splitlines()
    assert lines[-1] == "24 products, 5 maps"
    ops = {ln.split(":")[0]: ln.split(": ", 1)[1] for ln in lines[:-1]}
    # the spliced bottleneck layer reads two frames of the layer before, the layer after it adds the bypass
    assert ops["tdnnf2.linear"].startswith("product of tdnn1.dropout x 2 -> codes")
    assert ops["tdnnf2.noop"].startswith("product of tdnnf2.linear x 2 + 0.75 * tdnn1.dropout -> codes")
    assert ops["output.affine"].startswith("product of prefinal-chain.batchnorm2 x 1 (")
    # 32 bits: the layers before and the one that reads the features and the
    # i-vector, and tdnnf4.linear, whose frames are not evenly spaced
    assert not {"spec-augment", "delta", "input2", "tdnnf4.linear"} & set(ops)
    assert ops["tdnn1.dropout"].startswith("-> codes")
    assert "-> codes" not in ops["tdnnf3.noop"]  # read by tdnnf4.linear and a bypass alone
    assert engine.plan_describe_int8(synth_model, 21).splitlines()[-1].startswith("24 products")
    # chunks of one output frame: tdnnf4.linear has two frames a chunk, evenly spaced as two always are, and tdnnf4.noop reads it
    assert engine.plan_describe_int8(synth_model, 3).splitlines()[-1].startswith("26 products")


def test_precision_names():
    from vosk import engine
    with pytest.raises(ValueError, match="precision"):
        engine.Engine("nowhere", precision="int4")


# 7 output rows of 9 floats in a matrix of 20 columns and 50 rows
IN_PLACE = {**LINEAR, "ldo": 20, "residual": P, "ldr": 20}


@pytest.mark.parametrize("change", [
    dict(out_to=P, ldout_to=1, out_rows=50), dict(res_from=P, ldres_from=1, res_rows=50),
    dict(out_to=P, ldout_to=1, out_rows=50, res_from=P + 4, ldres_from=1, res_rows=50),
    dict(out_to=P, ldout_to=1, out_rows=50, res_from=P, ldres_from=2, res_rows=50),
    dict(residual_type=1), dict(out_type=2), dict(ldr=19), dict(ldo=19), dict(ldo=9, ldr=18), dict(residual=P + 4), dict(out=P + 20 * 4),
    dict(residual=P + 8 * 4), dict(out=P + 8 * 4), dict(residual=P + 12 * 4), dict(residual=P + 26 * 4), dict(residual=P + 20 * 6 * 4 + 32),
    dict(m=1, residual=P + 4), dict(m=1, ldo=9, out_to=P, out_rows=50, ldr=0),
    dict(out=P + 49 * 80, residual=P, res_from=P, ldres_from=1, res_rows=50), dict(out=P + 6 * 80 - 4, out_to=P, ldout_to=1, out_rows=9),
])
def test_out_that_overlaps_the_residual_otherwise_than_row_by_row_is_refused(lib, change):
    """One row's residual would be read while another's output is written over it: in place goes row by row, through no
    maps or through the same map."""
    assert _call(lib, "vamd_op_linear_int8", Linear, **{**IN_PLACE, **change}) < 0
    assert "overlap" in _err(lib) and "residual" in _err(lib)


@pytest.mark.parametrize("change", [
    dict(out_to=P, out_rows=1 << 62, ldo=9), dict(out_to=P, out_rows=(1 << 60) // 9, ldo=18), dict(out_to=P, out_rows=(1 << 62) + 5, ldo=64),
    dict(out_to=P, out_rows=(1 << 31) // 36 + 1, ldo=9), dict(residual=P, ldr=9, res_from=P, res_rows=1 << 62),
    dict(residual=P, ldr=64, res_from=P, res_rows=1 << 58), dict(residual=P, ldr=1 << 61, res_from=P, res_rows=8, m=1),
    dict(out_to=P, out_rows=8, ldo=1 << 61, m=1),
])
def test_mapped_matrices_whose_size_passes_64_bits_are_refused(lib, change):
    assert _call(lib, "vamd_op_linear_int8", Linear, **{**LINEAR, **change}) < 0
    assert "2^31" in _err(lib)


def test_kernels_use_m0_for_loads_to_lds_alone(tmp_path):
    """load_to_lds sets m0 unknown to the compiler: every instruction of the kernels' assembly that names m0 (or reads it
    unnamed) is one of its own.  Built with the flags of the library; no packed fp32 instruction either."""
    pkg = os.path.join(REPO, "vosk-api_amd")
    made = subprocess.run(["make", "-C", pkg, "-n", "-B", "build/int8_ops.o"], capture_output=True, text=True, check=True).stdout
    cmd = [ln for ln in made.splitlines() if "-c csrc/int8_ops.hip" in ln][0].split()
    cmd[cmd.index("-c")] = "-S"
    cmd[cmd.index("-o") + 1] = str(tmp_path / "a.s")
    subprocess.run(cmd + ["--cuda-device-only"], cwd=pkg, check=True, capture_output=True)
    code = [ln.split(";")[0].split("//")[0].strip() for ln in open(tmp_path / "a.s")]
    code = [ln for ln in code if ln and not ln.startswith(".")]
    sets = 0
    for i, ln in enumerate(code):
        if re.search(r"\bm0\b", ln):
            assert re.fullmatch(r"s_mov_b32 m0, s\d+", ln), ln
            assert code[i + 1] == "s_nop 0" and code[i + 2].startswith("global_load_lds_dwordx4 "), code[i:i + 3]
            sets += 1
        assert not re.match(r"(v_pk_\w+_f32|[sv]_movrel|v_interp|ds_gws|ds_append|ds_consume|s_sendmsg|buffer_load_\w+.*\blds\b)", ln), ln
    assert sets == sum(ln.startswith("global_load_lds") for ln in code) > 0


def test_forward_mode_tangents_are_refused_like_gradients():
    """A dual tensor has an address and requires no gradient, but its tangent would be lost; under no_grad as well, which
    is for reverse mode alone."""
    import torch.autograd.forward_ad as fw
    from vosk import ops
    x = torch.ones(3, 4)
    ops._no_grad(x, None, 1.0)
    with fw.dual_level():
        d = fw.make_dual(x, x)
        ops._no_grad(x, None)
        for t in (d, d[1:], d * 2):
            with pytest.raises(ValueError, match="gradient"):
                ops._no_grad(x, None, t)
        with torch.no_grad(), pytest.raises(ValueError, match="gradient"):
            ops._no_grad(d)
    ops._no_grad(d, x)
