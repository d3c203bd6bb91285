"""The 8-bit operators of libvosk.so on torch tensors (include/vosk_amd_ops.h).

  quantize_rows    rows of floats -> 8-bit codes and a scale for each row
  quantize_weight  the same for a weight matrix, laid out for linear_int8
  frame_map        which rows of a paged frame cache each output row reads
  linear_int8      the matrix product over codes, with scales for each row
                   and column and a fused bias / ReLU / affine / bypass

They are what the engine's 8-bit acoustic model runs (engine.Engine(...,
precision="int8")), on tensors of the caller's.  Calls go to the current
stream of the tensors' device, wait for nothing and may be captured into a
graph.  A tensor used on another stream than the one it was allocated on has
to be kept by the caller as torch asks (Tensor.record_stream).  A wrong
argument raises ValueError before anything is enqueued.  There is no backward
and no forward mode: tensors that require gradients or carry tangents are refused.

libvosk.so and torch have to share one HIP runtime, which they do when torch
is imported first; importing this module after vosk alone raises ImportError.
"""
from __future__ import annotations

import ctypes as C
import functools
import struct

import torch
import torch.autograd.forward_ad as _forward

from . import _c


def _one_runtime():
    try:
        with open("/proc/self/maps") as f:
            found = {line.split()[-1] for line in f if "libamdhip64" in line}
    except OSError:
        return
    if len(found) > 1:
        raise ImportError("vosk was imported before torch and the two have loaded a HIP runtime each (%s): "
                          "import torch before vosk" % ", ".join(sorted(found)))


_one_runtime()

_SIGS = {
    "vamd_op_code_bytes": (C.c_int, [C.c_int]),
    "vamd_op_quantize_rows": (C.c_int, [C.c_int, C.c_void_p, C.c_char_p]),
    "vamd_op_frame_map": (C.c_int, [C.c_int, C.c_void_p, C.c_char_p]),
    "vamd_op_linear_int8": (C.c_int, [C.c_int, C.c_void_p, C.c_char_p]),
    "vamd_op_linear_workspace": (C.c_longlong, [C.c_int, C.c_int, C.c_int, C.c_int, C.c_longlong]),
    "vamd_last_error": (C.c_char_p, []),
}
for _name, (_res, _args) in _SIGS.items():
    _fn = getattr(_c, _name)
    _fn.restype = _res
    _fn.argtypes = _args

# the structures of vosk_amd_ops.h, packed in one call (a ctypes argument
# costs 0.1 us, and the smallest operators take three)
_ROWS = struct.Struct("@6P7q2i").pack
_MAP = struct.Struct("@7P2q8i16i").pack
_LINEAR = struct.Struct("@15P11q8if").pack

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
PAD = 64          # code rows are a multiple of this many bytes
MAX_K = 1 << 17   # columns of one tap
MAX_TAPS = 16
_ZEROS = (0,) * MAX_TAPS
_i8, _i32, _f32 = torch.int8, torch.int32, torch.float32
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
    (lambda d: torch.cuda.current_stream(d).cuda_stream)


def _refuse(what):
    raise ValueError(what)


def _chk(r):
    if r < 0:
        raise ValueError((_c.vamd_last_error() or b"").decode())
    return r


def _on(t, name):
    """The GPU that a tensor is on."""
    if not isinstance(t, torch.Tensor):
        _refuse(name + " has to be a tensor")
    d = t.get_device() if t.is_cuda else -1
    if d < 0:
        _refuse(name + " has to be on the GPU")
    return d


def _vector(t, name, dtype, n, dev):
    """The address of n contiguous elements (None: 0)."""
    if t is None:
        return 0
    try:
        if t.dtype is dtype and t.numel() == n and t.get_device() == dev and t.is_contiguous():
            return t.data_ptr()
    except AttributeError:
        pass
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype:
        _refuse("%s has to be a tensor of %s" % (name, dtype))
    if t.get_device() != dev:
        _refuse(name + " is on another device")
    if t.numel() != n:
        _refuse("%s has to have %d elements" % (name, n))
    _refuse(name + " has to be contiguous")


def _matrix(t, name, dev):
    """Address, rows, columns and row stride of a matrix whose rows are contiguous and do not overlap."""
    try:
        m, n = t.shape
        ld, sc = t.stride()
        if sc == 1 and ld >= n and m > 1 and t.get_device() == dev:
            return t.data_ptr(), m, n, ld
    except (AttributeError, TypeError, ValueError):
        if not isinstance(t, torch.Tensor):
            _refuse(name + " has to be a tensor")
        _refuse(name + " has to be a matrix")
    if t.get_device() != dev:
        _refuse(name + " is on another device")
    if sc != 1 and n > 1 and m:
        _refuse("rows of %s have to be contiguous" % name)
    if m > 1 and ld < n:
        _refuse("rows of %s overlap" % name)
    return t.data_ptr(), m, n, ld if m > 1 else -(-n // 16) * 16  # (of one row any stride will do)


def _ints(t, name, n, dev):
    """Address and stride of a vector of n int32, any stride (None: 0, 0)."""
    if t is None:
        return 0, 0
    if not isinstance(t, torch.Tensor) or t.dtype is not _i32:
        _refuse(name + " has to be a tensor of torch.int32")
    if t.get_device() != dev:
        _refuse(name + " is on another device")
    if t.dim() != 1 or t.shape[0] != n:
        _refuse("%s has to have %d elements" % (name, n))
    return t.data_ptr(), t.stride(0)


def _no_grad(*ts):
    if torch.is_grad_enabled():
        for t in ts:
            if getattr(t, "requires_grad", False):
                _refuse("a tensor requires a gradient: the 8-bit operators have no backward")
    if _forward._current_level >= 0:  # (no_grad is for reverse mode alone)
        for t in ts:
            if isinstance(t, torch.Tensor) and _forward.unpack_dual(t).tangent is not None:
                _refuse("a tensor has a forward-mode gradient: the 8-bit operators have none")


@functools.lru_cache(maxsize=4096)
def _workspace(m, n, k, taps, rows):
    return _chk(_c.vamd_op_linear_workspace(m, n, k, taps, rows))


def code_bytes(k):
    """Bytes of a code row of k values: k rounded up to a multiple of 64."""
    return _chk(_c.vamd_op_code_bytes(k))


def quantize_rows(x, codes=None, scales=None, rows=None, count=None, from_rows=None):
    """Codes and scales of the rows of x (float32, float16 or bfloat16 [M, K];
    contiguous rows, any row stride):

      scale = fl32(max |x| / 127), code = x / scale rounded half to even,

    decided exactly.  A row of zeros gets scale 0 (a row so small that its
    scale is no normal float as well, or codes that end at +-127); a row holding
    an Inf or a NaN gets scale NaN and codes 0.  Returns (codes int8 [M, code_bytes(K)],
    scales float32 [M]); columns from K on are zero.

    codes and scales may be given (codes [C, >= code_bytes(K)], its rows
    16-byte aligned, C >= M), and with them rows, int32 [M]: row i is written
    to row rows[i], an entry outside [0, C) is skipped.  Entries inside have
    to be distinct (frame_map's are, without limits), rows not named are left
    as they were.  count (int32, one element, on the GPU): rows of x from there
    on are skipped; what frame_map leaves behind its last row names old frames,
    so a map's total belongs here.  from_rows, int32 [M]: row i is row
    from_rows[i] of x (skipped outside x), with rows as long; codes and scales
    are then given.
    """
    dev = _on(x, "x")
    t = _TYPES.get(x.dtype)
    if t is None:
        _refuse("x has to be float32, float16 or bfloat16")
    _no_grad(x)
    xp, m, k, ldx = _matrix(x, "x", dev)
    if not 1 <= k <= MAX_K:
        _refuse("x has to have 1 to %d columns" % MAX_K)
    kb = -(-k // PAD) * PAD
    if codes is None or scales is None:
        if codes is not scales:
            _refuse("codes and scales go together")
        if rows is not None or from_rows is not None:
            _refuse("rows and from_rows need codes and scales to write into")
        xr = m
        codes = torch.empty(m, kb, dtype=_i8, device=x.device)
        scales = torch.empty(m, dtype=_f32, device=x.device)
        cp, sp, c, ldc, rp, ldi, fp, ldf = codes.data_ptr(), scales.data_ptr(), m, kb, 0, 0, 0, 0
    else:
        cp, c, cols, ldc = _matrix(codes, "codes", dev)
        if codes.dtype is not _i8:
            _refuse("codes has to be int8")
        if cols < kb:
            _refuse("codes has to have %d columns" % kb)
        _no_grad(scales)
        sp = _vector(scales, "scales", _f32, c, dev)
        xr = m
        if from_rows is not None:
            m = from_rows.numel()
        fp, ldf = _ints(from_rows, "from_rows", m, dev)
        rp, ldi = _ints(rows, "rows", m, dev)
    if _c.vamd_op_quantize_rows(dev, _raw_stream(dev), _ROWS(xp, rp, fp, _vector(count, "count", _i32, 1, dev), cp, sp,
                                                             m, ldx, c, ldc, ldi, ldf, xr, t, k)) < 0:
        _chk(-1)
    return codes, scales


def quantize_weight(w, taps=1):
    """A weight matrix [N, taps * K] (one block of K columns for each spliced
    frame) as linear_int8 takes it: (codes int8 [N, taps * code_bytes(K)],
    scales float32 [N]), one scale for each output column n, the rounding of
    quantize_rows (and its limit: taps * K is at most 131 072)."""
    _on(w, "w")
    if w.dim() != 2 or taps < 1 or w.shape[1] % taps:
        _refuse("w has to be [N, taps * K]")
    n, k = w.shape[0], w.shape[1] // taps
    codes, scales = quantize_rows(w)
    kb = code_bytes(k)
    out = torch.zeros(n, taps, kb, dtype=_i8, device=w.device)
    out[:, :, :k] = codes[:, :taps * k].view(n, taps, k)
    return out.view(n, taps * kb), scales


def frame_map(lengths, first, table, page, rows, starts=None, offsets=(0,), step=1, low=None, high=None, clamp=True,
              strides=None):
    """Which rows of a frame cache the output rows of a step read.

    lengths, first: int32 [R], every stream's new frames and the time of the
    first; a stream gives ceil(length / step) output rows, at times first +
    step * i, packed stream after stream.  table: int32 [R, G], the pages of
    each stream, page frames each, used as a ring of G * page frames: frame t
    lies in row table[r, (t mod ring) // page] * page + t mod page.
    rows: int32 [cap, J], filled: entry j is the cache row of the frame at
    the row's time + offsets[j].  starts: int32 [R + 1], the streams' first
    output rows and the total (its last element is linear_int8's count).

    low, high (int32 [R], optional): the first and last frame a stream has; a
    frame outside is replaced by the nearest one inside (clamp) or is absent.
    Entry -1: absent, a negative page number, a frame the ring cannot hold
    beside the newest one that the stream's rows name, a row past 2^31 - 1.  Rows from the total
    on are left as they were; rows past cap are not written.
    strides = (page_stride, frame_stride), by default (page, 1): frame t lies in
    row table[...] * page_stride + (t mod page) * frame_stride.
    Returns (starts, rows).
    """
    dev = _on(lengths, "lengths")
    r = lengths.numel()
    lp = _vector(lengths, "lengths", _i32, r, dev)
    fp = _vector(first, "first", _i32, r, dev) or (r and _refuse("first is missing"))
    tp, tr, pages, ldt = _matrix(table, "table", dev)
    rp, cap, taps, ldr = _matrix(rows, "rows", dev)
    if table.dtype is not _i32 or rows.dtype is not _i32:
        _refuse("table and rows have to be int32")
    if tr != r:
        _refuse("table has to have a row for each stream")
    if not 1 <= len(offsets) <= MAX_TAPS:
        _refuse("1 to %d offsets" % MAX_TAPS)
    if taps != len(offsets) or (cap > 1 and ldr != taps):
        _refuse("rows has to be contiguous, [cap, %d]" % len(offsets))
    if starts is None:
        starts = torch.empty(r + 1, dtype=_i32, device=lengths.device)
    try:
        args = _MAP(lp, fp, tp, _vector(low, "low", _i32, r, dev), _vector(high, "high", _i32, r, dev),
                    _vector(starts, "starts", _i32, r + 1, dev), rp, ldt, cap, r, pages, page, *(strides or (page, 1)), taps, step,
                    1 if clamp else 0,
                    *offsets, *_ZEROS[taps:])
    except struct.error:
        _refuse("offsets, page, step and strides have to be 32-bit whole numbers")
    if _c.vamd_op_frame_map(dev, _raw_stream(dev), args) < 0:
        _chk(-1)
    return starts, rows


def linear_int8(x, weight, weight_scale, *, scale=None, rows=None, count=None, bias=None, relu=False, gain=None,
                shift=None, residual=None, residual_scale=1.0, out=None, dtype=None, out_rows=None, residual_rows=None):
    """Matrix product in 8-bit codes, with a scale for each row and column:

      out[i, n] = weight_scale[n] * sum_j scale[r(i, j)] * sum_k x[r(i, j), k] * weight[n, j, k]

    then + bias, ReLU, * gain + shift, + residual_scale * residual, each
    optional.  The inner sums are exact, the rest is 32-bit floats, rounded
    once to out's type.

    weight: int8 [N, J * code_bytes(K)] in -127 .. 127, weight_scale: float32 [N]
    (quantize_weight).  x is either int8 codes [C, code_bytes(K)] with scale
    float32 [C] (quantize_rows), or float rows [C, K] that are quantised in
    the call, to the same codes (all C rows, but for the smallest calls: float
    rows that a map reads few of are better quantised before, with from_rows).
    rows (int32 [M, J], frame_map) says which rows of x are read; an entry
    outside [0, C) adds nothing.  Without it row
    i reads row i.  count (int32, one element, on the GPU): output rows from there on
    are left as they were (or, where the call makes out, have no value).

    out [M, N] may be given, else it is made, of `dtype` (float32).  It may be
    residual itself, if out_rows and residual_rows are both absent or one and
    the same tensor; it must not overlap residual otherwise (refused) nor
    another input.  out_rows (int32 [M]):
    output row i goes to row out_rows[i] of a given out [O, N], skipped outside
    it; entries inside have to be distinct.  residual_rows (int32 [M]): its
    residual is row residual_rows[i] of residual [R, N], none outside it.  (A
    matrix with mapped rows is smaller than 2^31 bytes.)
    """
    dev = _on(x, "x")
    xp, m, k, ldx = _matrix(x, "x", dev)
    wp, n, wk, ldw = _matrix(weight, "weight", dev)
    if weight.dtype is not _i8:
        _refuse("weight has to be a tensor of int8")
    if not 1 <= k <= MAX_K:
        _refuse("x has to have 1 to %d columns" % MAX_K)
    kb = -(-k // PAD) * PAD
    taps, rp, ldi, wsp, c = 1, 0, 0, 0, m
    if x.dtype is _i8:
        if scale is None:
            _refuse("codes need their scales")
        if k != kb:
            _refuse("codes have to have a multiple of %d columns" % PAD)
        xt, sp, cp, lda, xp, ldx = 0, _vector(scale, "scale", _f32, m, dev), xp, ldx, 0, 0
    else:
        xt = _TYPES.get(x.dtype)
        if xt is None:
            _refuse("x has to be int8 codes, float32, float16 or bfloat16")
        if scale is not None:
            _refuse("scale belongs to codes")
        sp = cp = lda = 0
    if rows is not None:
        rp, m, taps, ldi = _matrix(rows, "rows", dev)
        if rows.dtype is not _i32:
            _refuse("rows has to be int32 [M, J]")
        if not 1 <= taps <= MAX_TAPS:
            _refuse("rows has to have 1 to %d columns" % MAX_TAPS)
    if wk != taps * kb:
        _refuse("weight has to have %d columns" % (taps * kb))
    _no_grad(x, scale, weight_scale, residual, out, bias, gain, shift)
    qp = ldr = rt = ep = lde = rr = 0
    if residual is not None:
        qp, rm, rn, ldr = _matrix(residual, "residual", dev)
        rt = _TYPES.get(residual.dtype)
        rr = rm
        if residual_rows is not None:
            ep, lde = _ints(residual_rows, "residual_rows", m, dev)
            rm = m
        if rt is None or rm != m or rn != n:
            _refuse("residual has to be [%d, %d] floats" % (m, n))
    elif residual_rows is not None:
        _refuse("residual_rows needs a residual")
    tp = ldto = 0
    if out is None:
        if out_rows is not None:
            _refuse("out_rows needs an out to write into")
        if dtype is None:
            dtype = _f32
        if dtype not in _TYPES:
            _refuse("dtype has to be float32, float16 or bfloat16")
        out = torch.empty(m, n, dtype=dtype, device=x.device)
        op, ldo, orows = out.data_ptr(), n, m
    else:
        op, om, on, ldo = _matrix(out, "out", dev)
        orows = om
        if out_rows is not None:
            tp, ldto = _ints(out_rows, "out_rows", m, dev)
            om = m
        if om != m or on != n or out.dtype not in _TYPES or (dtype is not None and dtype is not out.dtype):
            _refuse("out has to be [%d, %d] float32, float16 or bfloat16" % (m, n))
    if m == 0 or n == 0:
        return out
    if xp:
        size = _workspace(m, n, k, taps, c)
        if size:
            ws = torch.empty(size, dtype=_i8, device=x.device)
            wsp = ws.data_ptr()
    try:
        args = _LINEAR(cp, sp, rp, _vector(count, "count", _i32, 1, dev), xp, wsp, wp,
                       _vector(weight_scale, "weight_scale", _f32, n, dev), _vector(bias, "bias", _f32, n, dev),
                       _vector(gain, "gain", _f32, n, dev), _vector(shift, "shift", _f32, n, dev), qp, op, tp, ep,
                       c, lda, ldx, ldw, ldr, ldo, ldi, ldto, orows, lde, rr, m, n, k, taps, 1 if relu else 0, xt, rt,
                       _TYPES[out.dtype], residual_scale)
    except struct.error:
        _refuse("residual_scale has to be a number")
    if _c.vamd_op_linear_int8(dev, _raw_stream(dev), args) < 0:
        _chk(-1)
    return out
