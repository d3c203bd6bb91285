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
argument raises ValueError before anything is enqueued.  There is no backward:
tensors that require gradients are refused.

libvosk.so and torch have to share one HIP runtime, which they do when torch
is imported first; importing this module after vosk alone raises ImportError.
"""
from __future__ import annotations

import ctypes as C

import torch

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

_vp, _i, _ll, _f = C.c_void_p, C.c_int, C.c_longlong, C.c_float
_SIGS = {
    "vamd_op_code_bytes": (_i, [_i]),
    "vamd_op_quantize_rows": (_i, [_i, _vp, _vp, _i, _ll, _i, _ll, _vp, _vp, _ll, _vp, _ll, _vp]),
    "vamd_op_frame_map": (_i, [_i, _vp, _vp, _vp, _i, _vp, _ll, _i, _i, _vp, _i, _i, _vp, _vp, _i, _vp, _vp, _ll]),
    "vamd_op_linear_int8": (_i, [_i, _vp, _vp, _ll, _vp, _ll, _vp, _i, _vp, _vp, _ll, _vp, _i, _i, _i, _vp, _i, _vp, _vp,
                                 _vp, _ll, _i, _f, _vp, _ll, _i]),
    "vamd_op_linear_workspace": (_ll, [_i, _i]),
    "vamd_op_linear_float": (_i, [_i, _vp, _vp, _i, _ll, _vp, _vp, _vp, _ll, _vp, _i, _i, _i, _vp, _i, _vp, _vp, _vp, _ll,
                                  _i, _f, _vp, _ll, _i]),
    "vamd_last_error": (C.c_char_p, []),
}
for _name, (_res, _args) in _SIGS.items():
    _fn = getattr(_c, _name)
    _fn.restype = _res
    _fn.argtypes = _args

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
PAD = 64          # code rows are a multiple of this many bytes
MAX_K = 1 << 17   # columns of one tap
MAX_TAPS = 16


def _chk(r):
    if r < 0:
        raise ValueError((_c.vamd_last_error() or b"").decode())
    return r


def _want(ok, what):
    if not ok:
        raise ValueError(what)


def code_bytes(k):
    """Bytes of a code row of k values: k rounded up to a multiple of 64."""
    return _chk(_c.vamd_op_code_bytes(k))


def _device(t, name):
    _want(isinstance(t, torch.Tensor), name + " has to be a tensor")
    d = t.device
    _want(d.type == "cuda", name + " has to be on the GPU")
    return d


def _vector(t, name, dtype, n, device):
    """The pointer of an optional vector of n elements."""
    if t is None:
        return None
    _want(isinstance(t, torch.Tensor) and t.dtype is dtype, "%s has to be a tensor of %s" % (name, dtype))
    _want(t.device == device, name + " is on another device")
    _want(t.dim() == 1 and t.shape[0] == n, "%s has to have %d elements" % (name, n))
    _want(n <= 1 or t.stride(0) == 1, name + " has to be contiguous")
    _no_grad(t, name)
    return t.data_ptr()


def _no_grad(t, name):
    _want(not (t.requires_grad and torch.is_grad_enabled()), name + " requires a gradient: the 8-bit operators have none")


def _matrix(t, name, device):
    """(pointer, row stride) of a matrix whose rows are contiguous and do not overlap."""
    _want(t.device == device, name + " is on another device")
    _want(t.dim() == 2, name + " has to be a matrix")
    m, n = t.shape
    ld, sc = t.stride()
    _want(n <= 1 or sc == 1, "rows of %s have to be contiguous" % name)
    _want(m <= 1 or ld >= n, "rows of %s overlap" % name)
    return t.data_ptr(), (ld if m > 1 else max(ld, n))


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def quantize_rows(x, codes=None, scales=None, rows=None, count=None):
    """Codes and scales of the rows of x (float32, float16 or bfloat16 [M, K];
    contiguous rows, any row stride):

      scale = fl32(max |x| / 127), code = x / scale rounded half to even,

    decided exactly.  A row of zeros gets scale 0; a row holding an Inf or a
    NaN gets scale NaN and codes 0.  Returns (codes int8 [M, code_bytes(K)],
    scales float32 [M]); columns from K on are zero.

    codes and scales may be given (codes [C, >= code_bytes(K)], its rows
    16-byte aligned, C >= M), and with them rows, int32 [M]: row i is written
    to row rows[i], an entry outside [0, C) is skipped.  Entries inside have
    to be distinct (frame_map's are, without limits), rows not named are left
    as they were.  count (int32, one element, on the GPU): rows of x from there
    on are skipped; what frame_map leaves behind its last row names old frames,
    so a map's total belongs here.
    """
    dev = _device(x, "x")
    _want(x.dtype in _TYPES, "x has to be float32, float16 or bfloat16")
    _no_grad(x, "x")
    xp, ldx = _matrix(x, "x", dev)
    m, k = x.shape
    _want(1 <= k <= MAX_K, "x has to have 1 to %d columns" % MAX_K)
    kb = -(-k // PAD) * PAD
    _want((codes is None) == (scales is None), "codes and scales go together")
    if codes is None:
        _want(rows is None, "rows needs codes and scales to write into")
        codes = torch.empty(m, kb, dtype=torch.int8, device=dev)
        scales = torch.empty(m, dtype=torch.float32, device=dev)
    _want(codes.dtype is torch.int8, "codes has to be int8")
    cp, ldc = _matrix(codes, "codes", dev)
    c = codes.shape[0]
    _want(codes.shape[1] >= kb, "codes has to have %d columns" % kb)
    sp = _vector(scales, "scales", torch.float32, c, dev)
    rp = _vector(rows, "rows", torch.int32, m, dev)
    np_ = _vector(count, "count", torch.int32, 1, dev)
    _chk(_c.vamd_op_quantize_rows(dev.index, _stream(dev), xp, _TYPES[x.dtype], m, k, ldx, rp, np_, c, cp, ldc, sp))
    return codes, scales


def quantize_weight(w, taps=1):
    """A weight matrix [N, taps * K] (one block of K columns for each spliced
    frame) as linear_int8 takes it: (codes int8 [N, taps * code_bytes(K)],
    scales float32 [N]), one scale for each output column n, the rounding of
    quantize_rows."""
    dev = _device(w, "w")
    _want(w.dim() == 2 and taps >= 1 and w.shape[1] % taps == 0, "w has to be [N, taps * K]")
    n, k = w.shape[0], w.shape[1] // taps
    codes, scales = quantize_rows(w)
    kb = code_bytes(k)
    out = torch.zeros(n, taps, kb, dtype=torch.int8, device=dev)
    out[:, :, :k] = codes[:, :taps * k].view(n, taps, k)
    return out.view(n, taps * kb), scales


def frame_map(lengths, first, table, page, rows, starts=None, offsets=(0,), step=1, low=None, high=None, clamp=True):
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
    Entry -1: absent, a negative page number, or a frame the ring cannot hold
    beside the newest one that the stream's rows name.  Rows from the total
    on are left as they were; rows past cap are not written.
    Returns (starts, rows).
    """
    dev = _device(lengths, "lengths")
    _want(lengths.dim() == 1, "lengths has to be a vector")
    r = lengths.shape[0]
    lp = _vector(lengths, "lengths", torch.int32, r, dev)
    fp = _vector(first, "first", torch.int32, r, dev)
    _want(fp is not None, "first is missing")
    _want(isinstance(table, torch.Tensor) and table.dtype is torch.int32, "table has to be a tensor of int32")
    tp, ldt = _matrix(table, "table", dev)
    _want(table.shape[0] == r, "table has to have a row for each stream")
    _want(isinstance(rows, torch.Tensor) and rows.dtype is torch.int32, "rows has to be a tensor of int32")
    taps = len(offsets)
    _want(1 <= taps <= MAX_TAPS, "1 to %d offsets" % MAX_TAPS)
    _want(rows.device == dev and rows.dim() == 2 and rows.shape[1] == taps and rows.is_contiguous(),
          "rows has to be contiguous, [cap, %d], on the device of lengths" % taps)
    if starts is None:
        starts = torch.empty(r + 1, dtype=torch.int32, device=dev)
    sp = _vector(starts, "starts", torch.int32, r + 1, dev)
    _chk(_c.vamd_op_frame_map(dev.index, _stream(dev), lp, fp, r, tp, ldt, table.shape[1], page,
                              (_i * taps)(*offsets), taps, step, _vector(low, "low", torch.int32, r, dev),
                              _vector(high, "high", torch.int32, r, dev), 1 if clamp else 0, sp, rows.data_ptr(),
                              rows.shape[0]))
    return starts, rows


def linear_int8(x, weight, weight_scale, *, scale=None, rows=None, count=None, bias=None, relu=False, gain=None,
                shift=None, residual=None, residual_scale=1.0, out=None, dtype=None):
    """Matrix product in 8-bit codes, with a scale for each row and column:

      out[i, n] = weight_scale[n] * sum_j scale[r(i, j)] * sum_k x[r(i, j), k] * weight[n, j, k]

    then + bias, ReLU, * gain + shift, + residual_scale * residual, each
    optional.  The inner sums are exact, the rest is 32-bit floats, rounded
    once to out's type.

    weight: int8 [N, J * code_bytes(K)], weight_scale: float32 [N]
    (quantize_weight).  x is either int8 codes [C, code_bytes(K)] with scale
    float32 [C] (quantize_rows), or float rows [M, K] that are quantised in
    the call.  With codes, rows (int32 [M, J], frame_map) says which code rows
    are read; an entry outside [0, C) adds nothing.  Without it row i reads
    row i.  count (int32, one element, on the GPU): output rows from there on
    are left as they were (or, where the call makes out, have no value).

    out [M, N] may be given, else it is made, of `dtype` (float32).  It may be
    residual itself; it must not overlap another input.
    """
    dev = _device(x, "x")
    _want(isinstance(weight, torch.Tensor) and weight.dtype is torch.int8, "weight has to be a tensor of int8")
    wp, ldw = _matrix(weight, "weight", dev)
    n = weight.shape[0]
    wsp = _vector(weight_scale, "weight_scale", torch.float32, n, dev)
    _want(wsp is not None, "weight_scale is missing")
    xp, ldx = _matrix(x, "x", dev)
    m, k = x.shape
    taps, rp = 1, None
    if x.dtype is torch.int8:
        _want(scale is not None, "codes need their scales")
        _want(k % PAD == 0, "codes have to have a multiple of %d columns" % PAD)
        c = m
        scp = _vector(scale, "scale", torch.float32, c, dev)
        if rows is not None:
            _want(isinstance(rows, torch.Tensor) and rows.dtype is torch.int32 and rows.device == dev and rows.dim() == 2
                  and rows.is_contiguous(), "rows has to be contiguous int32 [M, J] on the device of x")
            m, taps = rows.shape
            _want(1 <= taps <= MAX_TAPS, "rows has to have 1 to %d columns" % MAX_TAPS)
            rp = rows.data_ptr()
    else:
        _want(x.dtype in _TYPES, "x has to be int8 codes, float32, float16 or bfloat16")
        _want(scale is None and rows is None, "scale and rows belong to codes")
        _no_grad(x, "x")
    _want(1 <= k <= MAX_K, "x has to have 1 to %d columns" % MAX_K)
    kb = -(-k // PAD) * PAD
    _want(weight.shape[1] == taps * kb, "weight has to have %d columns" % (taps * kb))
    bp = _vector(bias, "bias", torch.float32, n, dev)
    gp, hp = _vector(gain, "gain", torch.float32, n, dev), _vector(shift, "shift", torch.float32, n, dev)
    _want((gp is None) == (hp is None), "gain and shift go together")
    qp, ldr, rt = None, 0, 0
    if residual is not None:
        _want(isinstance(residual, torch.Tensor) and residual.dtype in _TYPES, "residual has to be a tensor of floats")
        _want(residual.shape == (m, n), "residual has to be [%d, %d]" % (m, n))
        _no_grad(residual, "residual")
        qp, ldr = _matrix(residual, "residual", dev)
        rt = _TYPES[residual.dtype]
    cp = _vector(count, "count", torch.int32, 1, dev)
    if out is None:
        dtype = dtype or torch.float32
        _want(dtype in _TYPES, "dtype has to be float32, float16 or bfloat16")
        out = torch.empty(m, n, dtype=dtype, device=dev)
        op, ldo = out.data_ptr(), n
    else:
        _want(isinstance(out, torch.Tensor) and out.dtype in _TYPES and (dtype is None or dtype is out.dtype),
              "out has to be a tensor of float32, float16 or bfloat16")
        _want(out.shape == (m, n), "out has to be [%d, %d]" % (m, n))
        _no_grad(out, "out")
        op, ldo = _matrix(out, "out", dev)
    tail = (wp, ldw, wsp, m, n, k, bp, 1 if relu else 0, gp, hp, qp, ldr, rt, residual_scale, op, ldo, _TYPES[out.dtype])
    if x.dtype is torch.int8:
        if m == 0 or n == 0:
            return out
        _chk(_c.vamd_op_linear_int8(dev.index, _stream(dev), xp, ldx, scp, c, rp, taps, cp, *tail))
    elif m and n:
        ws = torch.empty(m * (kb + 4), dtype=torch.int8, device=dev)
        _chk(_c.vamd_op_linear_float(dev.index, _stream(dev), xp, _TYPES[x.dtype], ldx, ws.data_ptr(), cp, *tail))
    return out
